"""Top logits, distillation from them and the balance loss against their definitions in 64 bits (oracle/loss_oracle.py).

Tolerances.  EPS bounds the relative error of one probability: its exponent is a difference, rounded, times a rounded log2(e)/T, 3 * 2^-24 of at most 60 (a term
below 2^-60 of its row is covered by the floor FLOOR), 1.1e-5; the exponential 2^-22; a sum of up to 2^17 terms taken by threads of at most 512 each and then by
trees, 520 * 2^-24 = 3.1e-5.  A gradient is a sum of such terms, whose magnitudes add up to the oracle's grad_scale, and rounded to its type once
(half a step); its factors are 32-bit products, 4 * 2^-24.  A loss adds logarithms of such sums (EPS each) and their products, 8 * 2^-24 of loss_scale."""

import math

import pytest
import torch

from oracle import loss_oracle

pytestmark = pytest.mark.gpu

EPS, FLOOR = 5e-5, 2.0 ** -60
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]
SHAPES = [(1, 1, 1), (1, 2, 2), (3, 10, 4), (512, 10, 10), (257, 16, 1), (7, 33, 33), (130, 100, 7), (65, 255, 20), (31, 1000, 20), (19, 1001, 128), (9, 1024, 5),
          (8, 1025, 64), (5, 2047, 3), (6, 2049, 16), (4, 4099, 100), (3, 8192, 50), (5, 16384, 32), (4, 16385, 9), (3, 32771, 128), (2, 50257, 64), (3, 65536, 17),
          (1, 65537, 100), (2, 131072, 64), (1, 131077, 1), (1, 300001, 40)]
KINDS = ["normal", "counts", "wide"]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    return float(torch.finfo(dtype).smallest_normal) * half_step(dtype) * 2   # half the distance of subnormals


def made(n, v, dtype, kind, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * n + v)
    x = torch.randn(n, v, generator=g)
    if kind == "counts":
        x = (x * 12).round() / 4
    elif kind == "wide":
        x = x * 25
    else:
        x = x * 3
    return x.to(dtype).cuda()


def check_grad(got, want, scale, dtype):
    got, want = got.cpu().double(), want
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    bound = (EPS + 4 * 2.0 ** -24) * scale + (half_step(dtype) * (1 + EPS)) * want.abs() + smallest(dtype) + FLOOR * scale.amax(-1, keepdim=True).clamp(max=1e30)
    bad = ((got - want).abs() > bound) & ~nan & (got != want)
    assert not bad.any(), (int(bad.sum()), got[bad][:3], want[bad][:3], bound[bad][:3])


def check_loss(got, want, scale):
    got, want, scale = got.cpu().double(), want.double(), scale.double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    far = (2 * EPS + 8 * 2.0 ** -24) * scale
    over = (got == math.inf) & (want + far > torch.finfo(torch.float32).max)   # what may lie beyond the largest float may be rounded to infinity
    bad = ((got - want).abs() > far) & ~nan & (got != want) & ~over
    assert not bad.any(), (got[bad][:3], want[bad][:3])


# ------------------------------------------------------------------------------------------------ top logits
def check_top(x, k, temperature=1.0):
    import convlogic_b200 as cb

    top = cb.top_logits(x, k, temperature)
    v = x.shape[-1]
    values, indices, rest = loss_oracle.top_logits(x.reshape(-1, v), k, temperature)
    assert top.values.dtype == torch.float32 and top.indices.dtype == torch.int64 and top.rest.dtype == torch.float32
    assert top.values.shape == (*x.shape[:-1], k) and top.indices.shape == top.values.shape and top.rest.shape == x.shape[:-1]
    assert torch.equal(top.indices.cpu().reshape(-1, k), indices)
    got = top.values.cpu().double().reshape(-1, k)
    assert torch.equal(torch.isnan(got), torch.isnan(values)) and torch.equal(got.nan_to_num(0.0), values.nan_to_num(0.0))
    got = top.rest.cpu().double().reshape(-1)
    assert torch.equal(torch.isnan(got), torch.isnan(rest))
    bad = ((got - rest).abs() > 2 * EPS + 4 * 2.0 ** -24 * rest.abs()) & (got != rest) & ~torch.isnan(rest)
    assert not bad.any(), (got[bad][:3], rest[bad][:3])
    return top


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,v,k", SHAPES)
def test_top_logits(n, v, k, dtype):
    for kind in KINDS:
        check_top(made(n, v, dtype, kind), k, 1.0 if kind == "normal" else 2.5)


def odd_rows(v, dtype, low):
    """Rows in which the order of values is where a selection goes wrong; `low`: what masked places hold."""
    inf, nan = math.inf, math.nan
    g = torch.Generator().manual_seed(v)
    x = torch.randn(16, v, generator=g)
    x[0] = 1.5                                                    # all the same
    x[1] = low                                                    # everything masked
    x[2], x[2, v // 2] = torch.full((v,), low), 0.25              # one class left
    x[3, torch.randperm(v, generator=g)[: v - min(v, 5)]] = low   # fewer left than listed
    x[4] = torch.arange(v) / v
    x[5] = -torch.arange(v) / v
    x[6, v - 1] = nan
    x[7, :: 3] = nan
    x[8, v // 3] = inf
    x[9, :: 2] = inf
    x[10, torch.arange(v) % 2 == 0], x[10, torch.arange(v) % 2 == 1] = 0.0, -0.0
    x[11] = (x[11] > 0).float()                                   # two values
    x[12] = -3.0 - x[12].abs()
    x[13, : v // 2] = low
    x[14, v // 2:] = low
    x[15] = nan
    return x.clamp(min=torch.finfo(dtype).min).where((x > torch.finfo(dtype).min) | torch.isnan(x) | (x == -inf), x.clamp(min=torch.finfo(dtype).min)) \
        .where(x != -inf, torch.full_like(x, -inf)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("v,k", [(5, 5), (12, 5), (40, 20), (333, 64), (1024, 33), (2500, 100), (9001, 64), (20000, 128), (70001, 50), (140000, 64)])
def test_top_logits_of_rows_that_tie_or_are_masked(v, k, dtype):
    for low in (-math.inf, float(torch.finfo(dtype).min)):
        check_top(odd_rows(v, dtype, low), k)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("v,k", [(33, 1), (47, 20), (64, 21), (64, 64), (65, 65), (100, 10), (100, 100), (128, 32), (128, 128), (129, 33), (200, 64), (256, 5), (256, 128),
                                 (257, 128), (300, 66), (300, 70), (500, 128), (512, 113), (512, 128), (513, 128)])
def test_top_logits_of_short_rows(v, k, dtype):
    check_top(odd_rows(v, dtype, -math.inf), k)
    check_top(made(100, v, dtype, "normal"), k, 2.5)
    g = torch.Generator().manual_seed(v * k)
    check_top(torch.randint(0, 4, (50, v), generator=g).to(dtype).cuda(), k, 0.5)         # equal values in all lanes
    check_top(made(9, 2 * v + 5, dtype, "normal")[:, 3:3 + v], k)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("v,k", [(600, 20), (1001, 64), (1999, 100), (5003, 64), (40001, 128)])
def test_top_logits_of_windows(v, k, dtype):
    """All classes but some neighbours masked, or NaN, in rows that begin anywhere."""
    g = torch.Generator().manual_seed(v)
    for outside in (-math.inf, math.nan):
        wide = torch.full((24, v + 3), outside)
        for i, w in enumerate([0, 1, k - 1, k, k + 1, 2 * k, 3 * k, 5 * k] * 3):
            w = min(w, v)
            at = int(torch.randint(0, v - w + 1, (1,), generator=g)) + 1
            wide[i, at:at + w] = torch.randn(w, generator=g)
        check_top(wide.to(dtype).cuda()[:, 1:1 + v], k, 1.5)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_top_logits_of_any_layout(dtype):
    big = made(40, 1200, dtype, "normal")
    check_top(big[:, 3:1003], 9)                       # rows at a distance of their own
    check_top(big[::3, 1:12], 11)
    check_top(big[5, 7:].expand(6, -1), 20)            # the same row six times
    check_top(big.t(), 5)                              # classes at a distance: a copy is read
    check_top(big[:, ::2], 5)
    check_top(big.view(4, 10, 1200), 6)
    check_top(big.view(4, 10, 1200).transpose(0, 1), 6)
    check_top(big[0], 8)
    check_top(big[:0], 8)
    flat = made(1, 5000, dtype, "normal").reshape(-1)
    for start in range(9):                             # rows from any address
        check_top(flat[start:start + 4001], 30)
        check_top(flat[start:start + 3 * 37].view(3, 37), 12)


# ------------------------------------------------------------------------------------------------ distillation
def lists_for(x, k, temperature, seed=1):
    g = torch.Generator().manual_seed(seed + x.shape[1])
    teacher = x.detach().float().cpu().nan_to_num(0.0, 0.0, 0.0) + torch.randn(*x.shape, generator=g)
    values, indices, rest = loss_oracle.top_logits(teacher, k, temperature)
    return values.float().cuda(), indices.cuda(), rest.float().cuda()


def check_distill(x, top, temperature=1.0, weight=None, reduction="mean", upstream=None, grad=True):
    import convlogic_b200 as cb

    leaf = x.detach().requires_grad_(grad)
    loss = cb.distillation_loss(leaf, top, temperature, weight, reduction)
    assert loss.dtype == torch.float32 and loss.shape == (x.shape[:-1] if reduction == "none" else ())
    up = torch.ones_like(loss) if upstream is None else upstream
    v = x.shape[-1]
    flat = [t if t is None else t.reshape(-1, t.shape[-1]) for t in top[:2]] + [None if len(top) < 3 or top[2] is None else top[2].reshape(-1)]
    want = loss_oracle.distillation(x.reshape(-1, v), *flat, None if weight is None else weight.reshape(-1), temperature, reduction, up.reshape(-1) if up.dim() else up)
    check_loss(loss.detach().reshape(-1), want["loss"].reshape(-1), want["loss_scale"].reshape(-1))
    if grad:
        (g,) = torch.autograd.grad(loss, leaf, up)
        assert g.dtype == x.dtype and g.shape == x.shape
        check_grad(g.reshape(-1, v), want["grad"], want["grad_scale"], x.dtype)
    return loss


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,v,k", SHAPES)
def test_distillation(n, v, k, dtype):
    g = torch.Generator().manual_seed(n + v)
    for kind, temperature, reduction, with_rest, with_weight, scale in (("normal", 1.0, "mean", True, False, None), ("counts", 3.0, "sum", False, True, 1.0),
                                                                        ("wide", 2.0, "none", True, True, 0.5), ("normal", 1.5, "mean", True, True, 64.0)):
        x = made(n, v, dtype, kind)
        values, indices, rest = lists_for(x, k, temperature)
        weight = None
        if with_weight:
            weight = torch.rand(n, generator=g).cuda()
            weight[n // 2] = 0.0
        up = None
        if scale is not None:
            up = (torch.rand(n, generator=g) - 0.5).cuda() if reduction == "none" else torch.tensor(scale, device="cuda")
        check_distill(x, (values, indices, rest if with_rest else None), temperature, weight, reduction, up)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("v,k", [(6, 4), (40, 20), (1000, 64), (3000, 100), (20000, 33), (70001, 50), (140000, 64)])
def test_distillation_of_odd_lists_and_masked_rows(v, k, dtype):
    inf = math.inf
    low = float(torch.finfo(dtype).min)
    x = made(14, v, dtype, "normal")
    values, indices, rest = lists_for(x, k, 1.0)
    indices[0, 1] = indices[0, 0]                      # the same class twice, and k times
    indices[1] = indices[1, 0].clone()
    indices[2, k // 2:] = -1                           # lists of unequal lengths
    indices[3, ::2] = v + 5
    indices[3, 1] = 1 << 40
    values[4, 1:] = -inf                               # a teacher that is sure
    rest[4] = -inf
    rest[5] = 30.0                                     # almost everything is in the rest
    x[6, v // 2:] = -inf                               # masked classes
    x[7, :] = low
    x[7, v // 3] = 0.0
    x[8, indices[8, 0]] = -inf                         # a listed class that the student has masked: the loss is infinite, the gradient is not
    rest[9] = -100.0
    x[10] = low
    up = torch.rand(14, generator=torch.Generator().manual_seed(3)).cuda()
    for with_rest in (True, False):
        check_distill(x, (values, indices, rest if with_rest else None), 1.0, None, "none", up)
    check_distill(x[:6], (values[:6], indices[:6], rest[:6]), 1.0, None, "sum")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,v,k", [(64, 2049, 5), (2500, 2500, 20), (1300, 4100, 128), (700, 8200, 64), (1300, 11000, 3), (700, 20011, 64), (310, 70003, 33), (310, 131071, 64), (160, 140003, 100)])
def test_many_long_rows(n, v, k, dtype):
    """More rows than blocks, so that a block's tables serve one row after another.  The rows compared: the first of every block, some of its second and third,
    the last ones; among them rows with classes listed twice, missing entries, masked scores, weight zero and NaN."""
    import convlogic_b200 as cb

    inf, nan = math.inf, math.nan
    g = torch.Generator(device="cuda").manual_seed(n + v)
    x = (torch.randn(n, v, device="cuda", generator=g) * 3).to(dtype)
    values, indices = torch.topk(x.float() + torch.randn(n, v, device="cuda", generator=g), k, 1)
    rest = torch.rand(n, device="cuda", generator=g) * 3
    weight = torch.rand(n, device="cuda", generator=g) + 0.5
    row = torch.arange(n, device="cuda")
    indices[row % 5 == 1, k // 2] = indices[row % 5 == 1, 0]
    indices[row % 7 == 2, 0] = -1
    x[row % 6 == 3, v // 3:] = -inf
    weight[row % 9 == 4] = 0.0
    x[row % 18 == 4, 0] = nan
    x[row % 23 == 5] = -inf
    values[row % 29 == 6], rest[row % 29 == 6] = -inf, -inf
    rest[row % 11 == 7] = -inf
    up = torch.rand(n, device="cuda", generator=g) + 0.5
    some = torch.cat([row[:24], row[n // 2 - 12:n // 2 + 12], row[-24:]])
    want = loss_oracle.distillation(x[some], values[some], indices[some], rest[some], weight[some], 1.5, "none", up[some])
    x.requires_grad_(True)
    loss = cb.distillation_loss(x, (values, indices, rest), 1.5, weight, "none")
    check_loss(loss.detach()[some], want["loss"], want["loss_scale"])
    check_grad(torch.autograd.grad(loss, x, up)[0][some], want["grad"], want["grad_scale"], dtype)
    # the forward's own gradient, and the sum; a row whose loss is infinite (its student has masked what the teacher knows) is left out of that
    loss = cb.distillation_loss(x, (values, indices, rest), 1.5, weight, "sum")
    want = loss_oracle.distillation(x[some], values[some], indices[some], rest[some], weight[some], 1.5, "sum")
    check_grad(torch.autograd.grad(loss, x)[0][some], want["grad"], want["grad_scale"], dtype)


@pytest.mark.parametrize("n,v,k", [(67000, 5300, 9), (67000, 12000, 5), (530000, 1500, 5), (530000, 700, 40), (1100000, 300, 4), (2200000, 100, 3), (4300000, 9, 3), (17000000, 3, 1)])
def test_more_rows_than_a_grid_has_teams(n, v, k):
    """The first, the last and the first of the second turn."""
    import convlogic_b200 as cb

    x = torch.empty(n, v, dtype=torch.bfloat16, device="cuda")
    for part in x.split(max(1, (1 << 27) // v)):
        part.normal_(0.0, 3.0)
    top = cb.top_logits(x, k, 1.5)
    turns = [t for t in (1 << 16, 1 << 19, 1 << 20, 1 << 21, 1 << 22, 1 << 24) if t + 8 < n]
    some = torch.cat([torch.arange(8)] + [torch.arange(t - 8, t + 8) for t in turns] + [torch.arange(n - 8, n)]).cuda()
    values, indices, rest = loss_oracle.top_logits(x[some], k, 1.5)
    assert torch.equal(top.values[some].cpu().double(), values) and torch.equal(top.indices[some].cpu(), indices)
    assert ((top.rest[some].cpu().double() - rest).abs() <= 2 * EPS + 4 * 2.0 ** -24 * rest.abs()).all()
    lists = (top.values.roll(1, 1), top.indices, top.rest)
    want = loss_oracle.distillation(x[some], *(t[some] for t in lists), None, 1.5, "none", 1.0)
    x.requires_grad_(True)
    loss = cb.distillation_loss(x, lists, 1.5, None, "none")
    check_loss(loss.detach()[some], want["loss"], want["loss_scale"])
    check_grad(torch.autograd.grad(loss, x, torch.ones_like(loss))[0][some], want["grad"], want["grad_scale"], x.dtype)
    check_grad(torch.autograd.grad(cb.distillation_loss(x, lists, 1.5, None, "sum"), x)[0][some], want["grad"], want["grad_scale"], x.dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("v", [10, 1000, 20000, 140000])
def test_rows_that_count_for_nothing(v, dtype):
    """Weight zero, no teacher, no student: nothing is added and the gradient is zero, whatever stands there; NaN elsewhere stays in its row."""
    import convlogic_b200 as cb

    inf, nan = math.inf, math.nan
    x = made(8, v, dtype, "normal")
    values, indices, rest = lists_for(x, 4, 1.0)
    clean = cb.distillation_loss(x, (values, indices, rest), reduction="none")
    weight = torch.ones(8, device="cuda")
    weight[1] = weight[2] = 0.0
    x[1], x[2], values[2] = nan, inf, nan
    values[3], rest[3] = -inf, -inf
    x[4] = -inf
    indices[5], rest[5] = -1, -inf
    x[6, v - 1] = nan
    x = x.requires_grad_(True)
    loss = cb.distillation_loss(x, (values, indices, rest), weight=weight, reduction="none")
    (g,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
    assert loss[1:6].tolist() == [0.0] * 5 and not g[1:6].any()
    assert torch.isnan(loss[6]) and torch.isnan(g[6]).all()
    assert torch.equal(loss[[0, 7]], clean[[0, 7]]) and torch.isfinite(g[[0, 7]]).all() and g[[0, 7]].any(1).all()
    total = cb.distillation_loss(x[:6], (values[:6], indices[:6], rest[:6]), weight=weight[:6], reduction="sum")
    assert float(total) == float(clean[0])


def test_distillation_of_any_layout():
    big = made(40, 1200, torch.float32, "normal")
    for x in (big[:, 3:1003], big[::3, 1:12], big.t()[:, :30], big[:, ::2], big.view(4, 10, 1200)[..., :999], big.view(4, 10, 1200).transpose(0, 1), big[0]):
        v = x.shape[-1]
        values, indices, rest = lists_for(x.reshape(-1, v), 5, 1.0)
        shape = x.shape[:-1]
        check_distill(x, (values.view(*shape, 5), indices.view(*shape, 5), rest.view(shape)), reduction="none")
    values, indices, rest = lists_for(big, 5, 1.0)
    wide = torch.stack([values, values], 1)[:, 0], torch.stack([indices, indices], 2)[..., 0], torch.stack([rest, rest], 1)[:, 1]
    assert not any(t.is_contiguous() for t in wide)
    check_distill(big, wide)
    check_distill(big, (values.half(), indices))                 # values of another type
    flat = made(1, 5000, torch.bfloat16, "normal").reshape(-1)
    for start in range(9):
        check_distill(flat[start:start + 3 * 1037].view(3, 1037), tuple(t[:3] for t in lists_for(flat[:3 * 1037].view(3, 1037), 7, 1.0)))
    # one row for everybody: the gradient is the sum
    row = made(1, 300, torch.float32, "normal")
    values, indices, rest = lists_for(row.expand(6, -1) + 0, 4, 1.0)
    import convlogic_b200 as cb

    a, b = row.clone().requires_grad_(True), (row.expand(6, -1) + 0).requires_grad_(True)
    ga, = torch.autograd.grad(cb.distillation_loss(a.expand(6, -1), (values, indices, rest)), a)
    gb, = torch.autograd.grad(cb.distillation_loss(b, (values, indices, rest)), b)
    assert torch.allclose(ga, gb.sum(0, keepdim=True), rtol=1e-6, atol=1e-7)   # five additions of numbers below 0.2: 5 * 2^-24


def test_no_rows():
    import convlogic_b200 as cb

    x = torch.zeros(0, 12, device="cuda", requires_grad=True)
    top = torch.zeros(0, 3, device="cuda"), torch.zeros(0, 3, dtype=torch.int64, device="cuda"), torch.zeros(0, device="cuda")
    for how in ("mean", "sum"):
        loss = cb.distillation_loss(x, top, reduction=how)
        assert float(loss) == 0.0 and torch.autograd.grad(loss, x)[0].shape == (0, 12)
    assert cb.distillation_loss(x, top, reduction="none").shape == (0,)
    loss, counts = cb.balance_loss(x, 2)
    assert float(loss) == 0.0 and counts.tolist() == [0] * 12 and torch.autograd.grad(loss, x)[0].shape == (0, 12)


# ------------------------------------------------------------------------------------------------ balance
def check_balance(x, k=1, keep=None, upstream=1.0):
    import convlogic_b200 as cb

    leaf = x.detach().requires_grad_(True)
    loss, counts = cb.balance_loss(leaf, k, keep)
    assert loss.dtype == torch.float32 and loss.shape == () and counts.dtype == torch.int64 and not counts.requires_grad
    e = x.shape[-1]
    want = loss_oracle.balance(x.reshape(-1, e), k, None if keep is None else keep.reshape(-1), upstream)
    assert torch.equal(counts.cpu(), want["counts"])
    check_loss(loss.detach(), want["loss"], want["loss_scale"])
    (g,) = torch.autograd.grad(loss, leaf, torch.tensor(upstream, device="cuda"))
    assert g.dtype == x.dtype and g.shape == x.shape
    check_grad(g.reshape(-1, e), want["grad"], want["grad_scale"], x.dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,e,k", [(1, 1, 1), (1, 2, 1), (5, 3, 3), (1000, 16, 1), (20000, 16, 1), (100003, 16, 2), (777, 8, 2), (4097, 64, 6), (3001, 60, 4), (999, 128, 8),
                                   (500, 129, 8), (300, 256, 8), (211, 500, 32), (100, 1000, 3), (64, 1024, 32)])
def test_balance(n, e, k, dtype):
    for kind, with_keep, up in (("normal", False, 1.0), ("counts", True, 0.25)):
        x = made(n, e, dtype, kind)
        keep = torch.rand(n, generator=torch.Generator().manual_seed(n)).cuda() < 0.8 if with_keep else None
        check_balance(x, k, keep, up)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("e,k", [(4, 3), (16, 1), (16, 4), (100, 8), (600, 16)])
def test_balance_of_rows_that_tie_or_are_masked(e, k, dtype):
    x = made(50, e, dtype, "normal")
    x[0] = 2.0
    x[1] = -math.inf
    x[2], x[2, e // 2] = -math.inf, 0.0
    x[3, : e - 2] = -math.inf
    x[4] = float(torch.finfo(dtype).min)
    x[5, 1:] = float(torch.finfo(dtype).min)
    x[6, ::2] = -math.inf
    check_balance(x, k)
    keep = torch.zeros(50, dtype=torch.bool, device="cuda")
    check_balance(x, k, keep)
    keep[:3] = True
    check_balance(x, k, keep)
    keep[5:] = True
    x[4] = math.nan                                    # a padded row may hold anything
    keep[4] = False
    check_balance(x, k, keep)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("e,k", [(16, 4), (16, 5), (16, 16), (13, 7), (24, 5), (32, 4), (37, 8), (64, 32), (100, 9), (128, 4), (256, 8), (300, 32), (512, 31), (500, 8)])
def test_balance_choices_among_equal_values(e, k, dtype):
    g = torch.Generator().manual_seed(e + k)
    for levels in (1, 2, 3, e):                        # so many different values in a row
        x = torch.randint(0, levels, (301, e), generator=g).float()
        x[1::7] = torch.where(torch.rand(43, e, generator=g) < 0.7, -math.inf, x[1::7])
        x[2::7, -1] = float(torch.finfo(dtype).min)
        x[3::7] = torch.where(torch.arange(e) >= e - k, x[3::7], torch.tensor(float(torch.finfo(dtype).min)))
        x[4::7] *= -0.0 if levels < 3 else -1.0        # zeros of both signs are equal
        check_balance(x.to(dtype).cuda(), k)


def test_balance_of_any_layout():
    big = made(60, 256, torch.float32, "normal")
    check_balance(big[:, 3:19])
    check_balance(big[::2, 5:100], 3)
    check_balance(big.t(), 2)
    check_balance(big.view(3, 20, 256)[..., :17], 2, torch.rand(3, 20).cuda() < 0.5)
    check_balance(big.view(60, 16, 16))                # the gates of a block: [channels, gates of a tree, 16]
    check_balance(big[0])
    check_balance(big[:1, :16].expand(9, -1))
    flat = made(1, 5000, torch.bfloat16, "normal").reshape(-1)
    for start in range(9):
        check_balance(flat[start:start + 37 * 16].view(37, 16))
        check_balance(flat[start:start + 37 * 7].view(37, 7), 2)
