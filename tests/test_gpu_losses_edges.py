"""The loss terms where their arithmetic goes to its ends: references far from zero, lists far from zero, sizes just past a kernel's, against 64 bits.

Tolerances are those of test_gpu_losses.py unless a test derives its own."""

import pytest
import torch

from oracle import loss_oracle
from tests.test_gpu_losses import DTYPES, EPS, IDS, check_balance, check_distill, check_grad, check_loss, check_top, lists_for, made

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ references far from zero
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("temperature", [0.7, 1.0, 1.5, 2.0, 2.5, 4.0])
def test_top_logits_with_as_many_groups_as_the_list_is_long(temperature, dtype):
    """The last segment of a row has k groups of neighbours, and in one of them all values are below -2: the bound that k of them reach is far below every value."""
    k = 20
    each = 128 // torch.finfo(dtype).bits                       # classes of a group: 16 bytes
    v = 16384 + k * each
    x = made(6, v, dtype, "normal").abs()
    for i, low in enumerate((-2.5, -3.0, -7.75, -20.0, -100.0)):
        x[i, 16384 + (3 * i) * each:16384 + (3 * i + 1) * each] = low
    check_top(x, k, temperature)
    check_top(x[:, :16384 + (k - 1) * each].contiguous(), k - 1, temperature)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e20, -3e29, -1e30, -1e37])
@pytest.mark.parametrize("v,k", [(40, 12), (300, 20), (1000, 64), (2500, 100), (9001, 64), (20000, 128), (70001, 50)])
def test_top_logits_of_classes_masked_with_a_number(v, k, mask, dtype):
    x = made(9, v, dtype, "normal")
    x[0] = mask
    x[1], x[1, v // 2] = mask, 0.25
    x[2, 7:] = mask
    x[3, : v - 7] = mask
    x[4, k - 1:] = mask
    x[5, k:] = mask
    x[6, k + 1:] = mask
    x[7, : v // 2] = mask
    x[8, :: 2] = mask
    for temperature in (1.0, 1.5, 4.0):
        check_top(x, k, temperature)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e20, -3e29, -1e30, -1e37])
@pytest.mark.parametrize("n,v", [(6, 40), (6, 1000), (6, 70001), (70, 2100), (70, 20000), (66, 70001)])
def test_distillation_of_classes_masked_with_a_number(n, v, mask, dtype):
    """The first and the last classes, and all that are not listed; by few rows and by many, which take other kernels."""
    k = 9
    x = made(n, v, dtype, "normal")
    values, indices, rest = lists_for(x, k, 1.5)
    row = torch.arange(n)
    x[:, : v // 3] = torch.where((row % 5 == 0)[:, None].cuda(), mask, x[:, : v // 3].float()).to(dtype)
    x[:, v // 4:] = torch.where((row % 5 == 1)[:, None].cuda(), mask, x[:, v // 4:].float()).to(dtype)
    for i in range(2, n, 5):
        keep = x[i, indices[i]].clone()
        x[i] = mask
        x[i, indices[i]] = keep
    x[3] = mask
    up = torch.rand(n, generator=torch.Generator().manual_seed(1)).cuda() + 0.5
    for with_rest in (True, False):
        top = (values, indices, rest if with_rest else None)
        check_distill(x, top, 1.5, None, "none", up)
        check_distill(x, top, 1.5, None, "sum", None)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,v", [(6, 3), (6, 12), (6, 100), (6, 300), (6, 1000), (6, 4000), (6, 12000), (6, 70001), (6, 300001), (70, 2100), (70, 12000), (66, 70001)])
def test_infinities_in_rows_that_count_for_nothing(n, v, dtype):
    """Weight zero, a list without mass: the gradient is zero whatever stands there, whether the forward writes it or the backward."""
    import convlogic_b200 as cb

    inf, nan = float("inf"), float("nan")
    x = made(n, v, dtype, "normal")
    values, indices, rest = lists_for(x, 2, 1.0)
    weight = torch.ones(n, device="cuda")
    for i, bad in enumerate((inf, nan, -inf)):
        for j, row in enumerate((i, n - 1 - i)):
            x[row, 0] = x[row, v // 2] = bad
            x[row, :: 3 + j] = bad
    weight[0] = weight[1] = weight[2] = 0.0
    values[n - 3:], rest[n - 3:] = -inf, -inf
    indices[n - 1] = -1
    x[0, indices[0, 0]] = inf
    nothing = torch.tensor([0, 1, 2, n - 3, n - 2, n - 1]).cuda()
    for reduction in ("sum", "mean", "none"):
        for up in (1.0, 0.5):
            leaf = x.clone().requires_grad_(True)
            loss = cb.distillation_loss(leaf, (values, indices, rest), weight=weight, reduction=reduction)
            (g,) = torch.autograd.grad(loss, leaf, torch.full_like(loss, up))
            assert torch.isfinite(loss).all() and not g[nothing].any() and not torch.isnan(g).any()
            assert n == 6 or g[3:n - 3].any(1).all()


# ------------------------------------------------------------------------------------------------ lists far from zero
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shift", [0.0, 3e3, -1e4, 1e6])
@pytest.mark.parametrize("n,v", [(7, 20), (7, 1000), (7, 5000), (3, 70001), (66, 2100), (66, 20000)])
def test_lists_far_from_zero(n, v, shift, dtype):
    """A teacher's counts in the thousands: probabilities are those of the differences, and of the rest's distance from them, as the lists hold both in 32 bits."""
    x = made(n, v, dtype, "normal")
    values, indices, rest = lists_for(x, 12, 1.7)
    indices[1, 3] = indices[1, 0]                      # a class listed twice adds up both
    values = values + shift
    rest = (rest.double() + shift / 1.7).float()
    up = torch.rand(n, generator=torch.Generator().manual_seed(2)).cuda() + 0.5
    for with_rest in (True, False):
        check_distill(x, (values, indices, rest if with_rest else None), 1.7, None, "none", up)
    check_distill(x, (values, indices, rest), 1.7, None, "sum")


@pytest.mark.parametrize("temperature", [0.25, 0.5, 1.0, 3.0])
@pytest.mark.parametrize("n,v", [(6, 40), (6, 3000), (3, 70001), (66, 2100)])
def test_lists_of_the_lowest_and_the_largest_values(n, v, temperature):
    """Equal values are equal probabilities, whatever they are: the lists of zeros give the loss.  A rest beside the lowest is everything, beside the largest nothing."""
    import convlogic_b200 as cb

    x = made(n, v, torch.float32, "normal")
    _, indices, _ = lists_for(x, 4, 1.0)
    zeros, rest = torch.zeros(n, 4, device="cuda"), torch.full((n,), 2.0, device="cuda")

    def both(values, rest):
        leaf = x.clone().requires_grad_(True)
        loss = cb.distillation_loss(leaf, (values, indices, rest), temperature, reduction="none")
        return loss.detach(), torch.autograd.grad(loss, leaf, torch.ones_like(loss))[0]

    alike = both(zeros, None)
    for value in (torch.finfo(torch.float32).min, torch.finfo(torch.float32).max, -1e30, 1e30):
        values = torch.full_like(zeros, value)
        assert all(torch.equal(a, b) for a, b in zip(both(values, None), alike)), value
        loss, grad = both(values, rest)
        want = loss_oracle.distillation(x, zeros - (1e30 if value < 0 else 0.0), indices, rest if value < 0 else rest - 1e30, None, temperature, "none")
        check_loss(loss, want["loss"], want["loss_scale"])
        check_grad(grad, want["grad"], want["grad_scale"], x.dtype)


# ------------------------------------------------------------------------------------------------ losses near zero
@pytest.mark.parametrize("n,v,k", [(8, 6, 6), (8, 12, 3), (8, 100, 20), (8, 1000, 1), (8, 1000, 64), (8, 5000, 16), (3, 70001, 1), (3, 140003, 32), (66, 2100, 40), (66, 20000, 1), (66, 40001, 100)])
def test_losses_near_zero(n, v, k):
    """A student near its teacher, and lists that hold little of the mass.  A loss is sum p f(delta) with f(d) = d - 1 + exp(-d) over all classes, delta = log p - log q: an error e of a
    delta costs |p - q| e + p e^2 / 2.  Deltas are differences of logarithms of sums, 2 EPS = 1e-4 off at most; sum |p - q| is what the gradient's magnitudes add up to,
    by T; the shares themselves are products, 16 * 2^-24."""
    import convlogic_b200 as cb

    t = 4.0
    g = torch.Generator().manual_seed(v + k)
    for noise in (3.0, 0.1, 0.01):
        x = torch.randn(n, v, generator=g)
        teacher = x + noise * torch.randn(n, v, generator=g)
        values, indices, rest = loss_oracle.top_logits(teacher, k, t)
        top = (values.float().cuda(), indices.cuda(), rest.float().cuda())
        loss = cb.distillation_loss(x.cuda(), top, t, reduction="none").cpu().double()
        want = loss_oracle.distillation(x, *(s.cpu() for s in top), None, t, "none")
        off = t * want["grad"].abs().sum(1)
        bound = 2 * EPS * off + 2 * t * t * (2 * EPS) ** 2 + 16 * 2.0 ** -24 * want["loss"]
        assert ((loss - want["loss"]).abs() <= bound).all(), (noise, loss, want["loss"], bound)


@pytest.mark.parametrize("n,v,k", [(8, 12, 1), (8, 100, 2), (8, 1000, 1), (8, 5000, 16), (3, 70001, 1), (3, 140003, 32), (66, 2100, 1), (66, 20000, 1), (66, 40001, 100)])
def test_gradients_of_lists_that_hold_little(n, v, k):
    """An unlisted class's gradient is T q_j (q_r - r) / q_r.  Where r and q_r are near one their difference is that of the listed probabilities, P - Q, each EPS off, and the other
    factors are EPS off: T q_j / q_r (EPS (P + Q) + 3 EPS |P - Q|)."""
    import convlogic_b200 as cb

    t = 4.0
    g = torch.Generator().manual_seed(v * k)
    x = torch.randn(n, v, generator=g).double()
    teacher = x + torch.randn(n, v, generator=g)
    values, indices, rest = loss_oracle.top_logits(teacher, k, t)
    top = (values.float().cuda(), indices.cuda(), rest.float().cuda())
    p = torch.softmax(torch.cat([top[0].cpu().double() / t, top[2].cpu().double()[:, None]], 1), 1)[:, :-1].sum(1, keepdim=True)
    for reduction in ("sum", "none"):
        leaf = x.float().cuda().requires_grad_(True)
        loss = cb.distillation_loss(leaf, top, t, reduction=reduction)
        (grad,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
        s = torch.softmax(leaf.detach().cpu().double() / t, 1)
        q = s.gather(1, indices).sum(1, keepdim=True)
        want = t * s / (1 - q) * (p - q)
        bound = t * s / (1 - q) * EPS * ((p + q) + 3 * (p - q).abs())
        off = ((grad.cpu().double() - want).abs() - bound).scatter(1, indices, -1.0)
        assert (off <= 0).all(), (reduction, off.max())


# ------------------------------------------------------------------------------------------------ sizes just past a kernel's
def _time(call, n=5):
    """The shortest of five times of a call, each the mean of n."""
    call()
    times = []
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(n):
            call()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) / n)
    return min(times)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("v,k,more", [(257, 32, 420), (257, 57, 420), (513, 113, 640), (513, 128, 640), (540, 128, 640), (1025, 116, 1700), (1025, 128, 1700), (1100, 128, 1700), (2049, 128, 3500),
                                      (2049, 110, 3500), (4097, 128, 6500), (8193, 128, 10000), (16900, 77, 20000), (17000, 100, 20000), (33500, 110, 40000)])
def test_top_logits_just_past_a_size(v, k, more, dtype):
    """A row that is a little longer than a kernel's shorter rows has few groups of neighbours, and a list almost as long: right, and no slower than the values that it has not.
    (Where a row's values all are candidates it takes 6 to 30 times as long.)"""
    import convlogic_b200 as cb

    check_top(made(40, v, dtype, "normal"), k)
    check_top(made(40, v + 9, dtype, "wide")[:, 3:3 + v], k, 2.0)
    short, long = (torch.randn(8192 if v < 8192 else 2048, w, device="cuda").to(dtype) for w in (v, more))
    assert _time(lambda: cb.top_logits(short, k)) < 2.0 * _time(lambda: cb.top_logits(long, k))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("e", [385, 1024])
def test_balance_of_many_experts_and_rows(e, dtype):
    """All blocks that are resident take part, whatever the number of experts: twice the experts take no more than three times as long."""
    import convlogic_b200 as cb

    x = made(3000, e, dtype, "normal")
    check_balance(x, 3)
    many = torch.randn(65536, e, device="cuda").to(dtype)
    half = many[:, :e // 2].contiguous()
    assert _time(lambda: cb.balance_loss(many)) < 3.0 * _time(lambda: cb.balance_loss(half))
    assert int(cb.balance_loss(many, 8)[1].sum()) == 8 * 65536


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("e,k", [(5, 2), (16, 1), (16, 6), (60, 3), (128, 8), (700, 5)])
def test_balance_of_rows_with_nan(e, k, dtype):
    """NaN counts as +inf, by index; the loss and such a row's gradient are NaN, the other rows' are as they are.  A row with both has them chosen by index, too."""
    import convlogic_b200 as cb

    inf, nan = float("inf"), float("nan")
    x = made(40, e, dtype, "normal")
    x[3, e // 2] = nan
    x[4, 1::2] = nan
    x[5, 0], x[5, e - 1] = inf, nan
    x[6, 0], x[6, e - 1] = nan, inf
    x[7], x[7, e // 3] = -inf, nan
    x[8, e // 2] = inf
    leaf = x.clone().requires_grad_(True)
    loss, counts = cb.balance_loss(leaf, k)
    (g,) = torch.autograd.grad(loss, leaf)
    want = loss_oracle.balance(x.float().nan_to_num(inf, inf, -inf), k)["counts"]
    assert torch.equal(counts.cpu(), want) and torch.isnan(loss)
    assert torch.isnan(g[3:9]).any(1).all()
    p = torch.softmax(x.double(), 1)
    h = e / (40.0 * 40 * k) * (counts.double() - counts.double().mean())
    fine = torch.cat([torch.arange(3), torch.arange(9, 40)]).cuda()
    exact = (p * (h - (p * h).sum(1, keepdim=True)))[fine].cpu()
    scale = (p * (h.abs() + (p * h.abs()).sum(1, keepdim=True)))[fine].cpu()
    check_grad(g[fine], exact, scale, dtype)
