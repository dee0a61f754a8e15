"""What the loss terms answer where no launch can succeed, on the host."""

import os
import subprocess
import sys


def test_a_launch_that_fails_is_an_error():
    """In a process that sees no GPU no launch succeeds: every entry says so, and nothing is left that a later call would report."""
    code = """
from convlogic_b200 import _lib
lib, p = _lib.lib(), 1 << 20
for rows, classes in ((4, 10), (4, 1000), (64, 5000), (64, 400000), (3, 100000), (80, 400001)):
    for how in (0, 1, 2):
        assert lib.clb_distill_fwd(p, classes, p, p, None, None, p, p, p, None, p, 1 << 20, rows, classes, 3, 1.0, how, 0, None) == -3, (rows, classes, how)
        assert lib.clb_last_cuda_error() != 0
    assert lib.clb_distill_bwd(p, classes, p, p, p, p, 0, 0, p, rows, classes, 3, 1.0, 0, None) == -3
    assert lib.clb_top_logits(p, classes, p, p, p, p, 1 << 30, rows, classes, 3, 1.0, 0, None) == -3
assert lib.clb_balance_fwd(p, 10, None, p, p, p, p, 1 << 20, 4, 10, 3, 0, None) == -3 and lib.clb_balance_bwd(p, 10, None, p, p, p, 4, 10, 0, None) == -3
assert lib.clb_distill_fwd(p, 10, p, p, None, None, p, p, p, None, p, 1 << 20, 0, 10, 3, 1.0, 0, 0, None) == 0
"""
    done = subprocess.run([sys.executable, "-c", code], env={**os.environ, "CUDA_VISIBLE_DEVICES": ""}, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
