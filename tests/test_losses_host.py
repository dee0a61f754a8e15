"""The loss terms on the host: names, argument checks that come before any launch, and the 64-bit restatement against differences."""

import pytest
import torch

from oracle import loss_oracle


@pytest.fixture(scope="module")
def lib():
    from convlogic_b200 import _lib

    return _lib.lib()


def test_names():
    import convlogic_b200 as cb
    from convlogic_b200 import functional, ops

    for name in ("top_logits", "distillation_loss", "balance_loss", "DistillationLoss", "BalanceLoss", "TopLogits"):
        assert name in cb.__all__ and callable(getattr(cb, name)), name
    for name in ("top_logits", "distill_fwd", "distill_bwd", "balance_fwd", "balance_bwd"):
        assert callable(getattr(ops, name)), name
    for name in ("DistillationFunction", "BalanceFunction"):
        assert issubclass(getattr(functional, name), torch.autograd.Function), name


def test_bad_arguments_are_refused_before_any_launch(lib):
    p = 1 << 20   # never looked at
    args = dict(x=p, stride=10, values=p, indices=p, rest=p, rows=4, classes=10, k=3, t=1.0, dtype=0, scratch=p, size=0)

    def top(**kw):
        a = {**args, **kw}
        return lib.clb_top_logits(a["x"], a["stride"], a["values"], a["indices"], a["rest"], a["scratch"], a["size"], a["rows"], a["classes"], a["k"], a["t"], a["dtype"], None)

    for kw, want in (({"x": None}, -1), ({"values": None}, -1), ({"rest": None}, -1), ({"rows": -1}, -1), ({"classes": 0}, -1), ({"stride": -1}, -1), ({"k": 0}, -1),
                     ({"t": 0.0}, -1), ({"t": float("nan")}, -1), ({"t": -1.0}, -1), ({"dtype": 1}, -1), ({"dtype": 7}, -1), ({"k": 11}, -2),
                     ({"k": 129, "classes": 1000}, -6), ({"classes": 1 << 31}, -6)):
        assert top(**kw) == want, kw
    assert top(rows=0) == 0 and top(classes=100000, scratch=None) == -4 and top(classes=100000, size=100) == -4
    assert lib.clb_top_logits_scratch_bytes(4, 10, 3, 0) == 0 and lib.clb_top_logits_scratch_bytes(4, 100000, 3, 0) >= 4 * 13 * 32

    def fwd(loss=p, stats=p, listed=p, scratch=p, size=1 << 20, rows=4, classes=10, k=3, t=1.0, how=1, dtype=0, scores=p):
        return lib.clb_distill_fwd(scores, 10, p, p, None, None, loss, stats, listed, None, scratch, size, rows, classes, k, t, how, dtype, None)

    for kw, want in (({"loss": None}, -1), ({"scores": None}, -1), ({"stats": None}, -1), ({"listed": None}, -1), ({"how": 3}, -1), ({"t": 0.0}, -1), ({"dtype": 1}, -1),
                     ({"k": 0}, -1), ({"rows": -1}, -1), ({"k": 129}, -6), ({"scratch": None}, -4), ({"size": 0}, -4)):
        assert fwd(**kw) == want, kw
    assert fwd(rows=0, how=0) == 0 and lib.clb_distill_scratch_bytes(0, 10, 3) == 0
    assert lib.clb_distill_bwd(p, 10, p, p, p, None, 0, 0, p, 4, 10, 3, 1.0, 0, None) == -1
    assert lib.clb_distill_bwd(p, 10, p, p, p, p, 0, 0, p, 0, 10, 3, 1.0, 0, None) == 0

    assert lib.clb_distill_bwd(p, 10, p, p, p, p, 1, 1, p, 4, 10, 3, 1.0, 0, None) == -1     # rows' own upstream gradients are nothing that a forward knows

    def bal(loss=p, scratch=p, size=1 << 20, rows=4, experts=10, k=3, dtype=0, x=p):
        return lib.clb_balance_fwd(x, 10, None, loss, p, p, scratch, size, rows, experts, k, dtype, None)

    for kw, want in (({"loss": None}, -1), ({"x": None}, -1), ({"k": 0}, -1), ({"k": 11}, -2), ({"experts": 1025}, -6), ({"experts": 100, "k": 33}, -6), ({"dtype": 1}, -1),
                     ({"rows": 1 << 31}, -6), ({"scratch": None}, -4), ({"size": 0}, -4)):
        assert bal(**kw) == want, kw
    assert lib.clb_balance_bwd(p, 10, None, None, p, p, 4, 10, 0, None) == -1


def test_tensors_of_the_host_are_refused():
    import convlogic_b200 as cb

    x, i = torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int64)
    for call in (lambda: cb.top_logits(x, 2), lambda: cb.distillation_loss(x, (x[:, :2], i)), lambda: cb.balance_loss(x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="temperature"):
        cb.distillation_loss(x, cb.TopLogits(x[:, :2], i, None, 2.0), temperature=1.0)
    with pytest.raises(ValueError, match="reduction"):
        cb.DistillationLoss(reduction="batchmean")


def test_restatement_against_differences():
    """Central differences of step h of a smooth function are off by h^2 times its third derivative, here below 1: 1e-10 at h = 1e-5, and by the rounding of
    the two values, 2^-52 / 1e-5 = 2e-11 times their size (below 40)."""
    g = torch.Generator().manual_seed(0)
    s = torch.randn(4, 9, generator=g, dtype=torch.float64)
    teacher = torch.randn(4, 9, generator=g, dtype=torch.float64)
    v, i, r = loss_oracle.top_logits(teacher, 3, 2.0)
    i[1, 2] = i[1, 0]
    i[2, 1] = -1
    w = torch.tensor([1.0, 0.5, 2.0, 0.0], dtype=torch.float64)
    h = 1e-5
    for rest in (r, None):
        f = lambda x: float(loss_oracle.distillation(x, v, i, rest, w, 2.0, "sum")["loss"])  # noqa: E731
        got = loss_oracle.distillation(s, v, i, rest, w, 2.0, "sum")["grad"]
        for a in range(4):
            for b in range(9):
                d = torch.zeros_like(s)
                d[a, b] = h
                assert abs((f(s + d) - f(s - d)) / (2 * h) - float(got[a, b])) < 2e-9
    got = loss_oracle.balance(s, 2)
    for b in range(9):
        d = torch.zeros_like(s)
        d[1, b] = h
        assert abs(float(loss_oracle.balance(s + d, 2)["loss"] - loss_oracle.balance(s - d, 2)["loss"]) / (2 * h) - float(got["grad"][1, b])) < 2e-9
