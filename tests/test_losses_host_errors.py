"""What the loss terms answer where no launch can succeed, and to lists that a data loader has put together: on the host."""

import os
import subprocess
import sys

import pytest
import torch

import convlogic_b200 as cb


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


def test_lists_that_a_data_loader_puts_together():
    """A sample's TopLogits becomes a batch's, with a temperature for each sample."""
    top = cb.TopLogits(torch.randn(6, 3), torch.zeros(6, 3, dtype=torch.int64), torch.randn(6), 2.5)
    batch = torch.utils.data.default_collate([cb.TopLogits(*(t[i] for t in top[:3]), top.temperature) for i in range(6)])
    assert isinstance(batch, cb.TopLogits) and all(torch.equal(a, b) for a, b in zip(batch[:3], top[:3]))
    with pytest.raises(RuntimeError, match="CUDA"):              # gets as far as the scores
        cb.distillation_loss(torch.zeros(6, 8), batch, temperature=2.5)
    with pytest.raises(ValueError, match="temperature"):
        cb.distillation_loss(torch.zeros(6, 8), batch, temperature=2.0)
    batch.temperature[3] = 1.0
    with pytest.raises(ValueError, match="temperature"):
        cb.distillation_loss(torch.zeros(6, 8), batch, temperature=2.5)
