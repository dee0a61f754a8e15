"""The loss terms as they are used: together in a training step, twice over one graph, on other streams, captured and replayed, and what they refuse."""

import pytest
import torch

from oracle import loss_oracle
from tests.test_gpu_losses import check_grad, check_loss

pytestmark = pytest.mark.gpu


def _scores(n=96, v=1000, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, v, generator=g) * 3).to(dtype).cuda()


def _step(net, x, labels, top):
    """Cross-entropy, distillation from a teacher's lists, and the balance of every layer's gates."""
    import convlogic_b200 as cb

    flat = [m for m in net if isinstance(m, cb.LogicLayer)]
    scores = net(x)
    loss = torch.nn.functional.cross_entropy(scores, labels) + 0.5 * cb.DistillationLoss(2.0)(scores, top)
    for m in flat:
        loss = loss + 0.1 * cb.BalanceLoss()(m.weights)[0]
    return loss, torch.autograd.grad(loss, [x] + [m.weights for m in flat])


def test_a_training_step_with_all_of_them():
    """Against the same step with the terms written in torch: the gradients are sums of the same terms, and differ by their roundings, 1e-5 of the largest."""
    import convlogic_b200 as cb

    torch.manual_seed(0)
    net = torch.nn.Sequential(cb.LogicLayer(64, 400), cb.LogicLayer(400, 200), cb.GroupSum(10, 3.0)).cuda().train()
    teacher = torch.nn.Sequential(cb.LogicLayer(64, 800), cb.LogicLayer(800, 400), cb.GroupSum(10, 5.0)).cuda().eval()
    x = torch.rand(50, 64, device="cuda").requires_grad_(True)
    labels = torch.arange(50, device="cuda") % 10
    packed = teacher(cb.PackBitsTensor(x.detach() > 0.5, 32)).float() / 5.0      # the discretised teacher's counts
    top = cb.top_logits(packed, 4, temperature=2.0)
    loss, grads = _step(net, x, labels, top)

    scores = net(x)
    t, s = packed / 2.0, scores / 2.0
    at = top.indices
    p, q = torch.softmax(t, 1), torch.softmax(s, 1)
    pk, qk = p.gather(1, at), q.gather(1, at)
    r, qr = 1 - pk.sum(1), 1 - qk.sum(1)
    kl = (torch.special.xlogy(pk, pk) - pk * qk.log()).sum(1) + torch.special.xlogy(r, r) - r * qr.log()
    want = torch.nn.functional.cross_entropy(scores, labels) + 0.5 * 4.0 * kl.mean()
    weights = [net[0].weights, net[1].weights]
    for w in weights:
        pw = torch.softmax(w, 1)
        share = torch.bincount(w.argmax(1), minlength=16) / w.shape[0]
        want = want + 0.1 * 16 * (share * pw.mean(0)).sum()
    gwant = torch.autograd.grad(want, [x] + weights)
    assert abs(float(loss) - float(want)) <= 1e-5 * abs(float(want))
    for a, b in zip(grads, gwant):
        assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())
    # the counts are the operations of the discretised layer
    counts = cb.balance_loss(weights[0])[1]
    assert torch.equal(counts, torch.bincount(net[0]._gate_ids().long(), minlength=16))


def test_a_step_adds_to_the_gradients_of_a_bucket():
    import convlogic_b200 as cb

    torch.manual_seed(0)
    net = torch.nn.Sequential(cb.LogicLayer(64, 400), cb.GroupSum(10, 3.0)).cuda().train()
    x, w = torch.rand(50, 64, device="cuda"), net[0].weights
    (alone,) = torch.autograd.grad(net(x).square().mean(), w)
    (balance,) = torch.autograd.grad(cb.balance_loss(w)[0], w)
    bucket = cb.GradBucket(net)
    bucket.zero()
    (net(x).square().mean() + cb.balance_loss(w)[0]).backward()
    assert torch.allclose(bucket.flat.view_as(w), alone + balance, rtol=1e-6, atol=1e-9)
    bucket.direct()
    with pytest.raises(RuntimeError, match="direct"):
        cb.balance_loss(w)
    with torch.no_grad():
        assert int(cb.balance_loss(w)[1].sum()) == 400              # the counts alone are no gradient
    bucket.direct(False)
    cb.balance_loss(w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("v", [10, 1000, 20000, 140000])
def test_one_graph_differentiated_again_and_again(v, dtype):
    """With any upstream gradient, in any order: every result is a tensor of its own and nothing changes an earlier one."""
    import convlogic_b200 as cb

    x = _scores(6, v, dtype).requires_grad_(True)
    top = cb.top_logits(_scores(6, v, torch.float32, 1), 4)
    loss = cb.distillation_loss(x, top)
    up = [torch.tensor(u, device="cuda") for u in (1.0, 1.0, 2.0, 0.0, 1.0, -1.0, 1.0)]
    got = [torch.autograd.grad(loss, x, u, retain_graph=True)[0] for u in up]
    first = got[0].clone()
    assert first.any() and len({g.data_ptr() for g in got}) == len(got)

    def same(g, u):
        # The first gradient may come from the forward's own exponentials: it and the others are each within 5e-5 (test_gpu_losses.py) of terms that
        # a softmax and the teacher's probabilities bound by 2 / 6 a row, of their own values elsewhere, and rounded to the type once
        want, eps = first.double() * u, torch.finfo(dtype).eps / 2
        tol = 1e-4 * want.abs() + 2 * eps * want.abs() + 2.0 ** -23 * (dtype == torch.float16) * max(abs(u), 1.0)
        listed = torch.zeros_like(want).scatter_(1, top.indices, 2 / 6 * abs(u) * 1e-4)
        assert not ((g.double() - want).abs() > tol + listed).any(), u

    for u, g in zip(up, got):
        same(g, float(u))
    second = got[1].clone()
    for u, g in zip(up, got):
        if g is not got[0]:
            same(g, float(u))
            assert not float(u) == 1.0 or torch.equal(g, second)
        g.fill_(7.0)
    assert torch.equal(got[1], torch.full_like(second, 7.0))
    again = torch.autograd.grad(loss, x)[0]
    assert torch.equal(again, second)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, x)
    # an upstream gradient other than one comes first
    loss = cb.distillation_loss(x, top)
    half, one = (torch.autograd.grad(loss, x, torch.tensor(u, device="cuda"), retain_graph=True)[0] for u in (2.0, 1.0))
    assert torch.equal(one, second)
    same(half, 2.0)


def test_a_second_derivative_is_refused():
    import convlogic_b200 as cb

    x = _scores(6, 40).requires_grad_(True)
    top = cb.top_logits(_scores(6, 40, seed=1), 4)
    for loss in (cb.distillation_loss(x, top), cb.balance_loss(x)[0]):
        (g,) = torch.autograd.grad(loss, x, create_graph=True)
        assert g.abs().sum() > 0
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(g.sum(), x, retain_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            (g.sum() + x.sum()).backward()


def test_scores_written_to_before_the_backward_pass_raise():
    import convlogic_b200 as cb

    x = _scores(6, 40).requires_grad_(True)
    y = x * 1.0
    top = cb.top_logits(_scores(6, 40, seed=1), 4)
    for loss in (cb.distillation_loss(y, top), cb.balance_loss(y)[0]):
        with torch.no_grad():
            y.add_(1.0)
        with pytest.raises(RuntimeError, match="modified"):
            loss.backward()


@pytest.mark.parametrize("n,v", [(512, 10), (300, 1000), (40, 20000), (3, 140000)])
def test_the_same_bits_every_time(n, v):
    import convlogic_b200 as cb

    x = _scores(n, v).requires_grad_(True)
    teacher = _scores(n, v, seed=1)
    runs = []
    for _ in range(4):
        top = cb.top_logits(teacher, 8)
        loss = cb.distillation_loss(x, top)
        bal, counts = cb.balance_loss(x[:, :10].contiguous(), 2)
        runs.append([*top[:3], loss, *torch.autograd.grad(loss + bal, x), bal, counts])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_calls_on_two_streams():
    """Each call has workspaces of its own."""
    import convlogic_b200 as cb

    def work(x, teacher):
        x = x.detach().requires_grad_(True)
        loss = cb.distillation_loss(x, cb.top_logits(teacher, 16)) + cb.balance_loss(x[:, :64], 4)[0]
        return loss, torch.autograd.grad(loss, x)[0]

    sets = [(_scores(256, 1000 + 50 * i, seed=i), _scores(256, 1000 + 50 * i, seed=10 + i)) for i in range(4)]
    want = [work(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(5):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(work(*s))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 4]))


@pytest.mark.parametrize("n,v", [(512, 10), (300, 1000), (40, 20000), (3, 140000)])
def test_captured_and_replayed(n, v):
    """Two captured graphs, replayed in turn on new inputs, give what the calls give."""
    import convlogic_b200 as cb

    def work(x, teacher, up):
        top = cb.top_logits(teacher, 8)
        loss = cb.distillation_loss(x, top)
        bal, counts = cb.balance_loss(x[:, :10], 2)
        return [*top[:3], loss, counts, *torch.autograd.grad([loss, bal], x, [up, up])]

    x = [_scores(n, v, seed=i).requires_grad_(True) for i in range(2)]
    teacher, up = _scores(n, v, seed=5), torch.ones((), device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        work(x[0], teacher, up)
    torch.cuda.current_stream().wait_stream(st)
    graphs, outs = [], []
    for t in x:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(work(t, teacher, up))
    for round_, u in enumerate((1.0, 3.0, 1.0, 0.5)):
        up.fill_(u)
        teacher.copy_(_scores(n, v, seed=20 + round_))
        for i in range(2):
            with torch.no_grad():
                x[i].copy_(_scores(n, v, seed=40 + 2 * round_ + i))
        for g in graphs:
            g.replay()
        for i in range(2):
            for a, b in zip(outs[i], work(x[i], teacher, up)):
                assert torch.equal(a, b), (round_, i)   # the same kernels on the same inputs


def test_a_backward_pass_captured_alone():
    """The forward ran before the capture: every replay computes the gradient anew."""
    import convlogic_b200 as cb

    x = _scores(64, 1000).requires_grad_(True)
    top = cb.top_logits(_scores(64, 1000, seed=1), 8)
    up = torch.ones((), device="cuda")
    once = cb.distillation_loss(x, top)
    torch.autograd.grad(once, x, retain_graph=True)
    want = torch.autograd.grad(once, x)[0]           # from the scores, as the graph's
    del once                                         # (an eager graph of the same leaf ties its gradient to the eager stream)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        loss = cb.distillation_loss(x, top)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            (g,) = torch.autograd.grad(loss, x, up, retain_graph=True)
    for u in (1.0, 2.0, 1.0):
        up.fill_(u)
        g.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g, want * u)
    # and a forward captured alone, differentiated outside
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        loss2 = cb.distillation_loss(x, top)
    graph2.replay()
    torch.cuda.synchronize()
    (first,) = torch.autograd.grad(loss2, x, retain_graph=True)
    kept = first.clone()
    assert torch.equal(first, want)
    graph2.replay()
    torch.cuda.synchronize()
    first.fill_(5.0)
    (second,) = torch.autograd.grad(loss2, x)
    assert torch.equal(second, kept) and float(loss2) == float(cb.distillation_loss(x, top))


def test_what_torch_puts_around_a_call():
    import convlogic_b200 as cb
    import torch.autograd.forward_ad as fwad

    x = _scores(12, 40)
    top = cb.top_logits(_scores(12, 40, seed=1), 4)

    class Both(torch.nn.Module):
        def forward(self, s):
            return cb.distillation_loss(s, top) + cb.balance_loss(s, 2)[0]

    m = Both()
    traced = torch.jit.trace(m, (x,), check_trace=False)
    other = _scores(12, 40, seed=2)
    assert torch.equal(traced(other), m(other)) and not torch.equal(m(other), m(x))
    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    # (a gradient taken from the scores and one from the forward's own exponentials: each within 5e-5 of q + p <= 2, over 12 rows, of the same number)
    assert torch.allclose(torch.autograd.grad(traced(a), a)[0], torch.autograd.grad(m(b), b)[0], rtol=0.0, atol=2 * 5e-5 * 2 / 12)
    for call in (lambda s: cb.distillation_loss(s, top), lambda s: cb.balance_loss(s)[0]):
        with fwad.dual_level(), pytest.raises(NotImplementedError, match="jvp"):
            call(fwad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError):
            torch.func.grad(call)(x)
    lists = torch.jit.trace(lambda s: tuple(cb.top_logits(s, 5)[:3]), (x,), check_trace=False)
    assert all(torch.equal(p, q) for p, q in zip(lists(other), cb.top_logits(other, 5)[:3]))
    # hooks of saved tensors see what a call keeps
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        y = x.clone().requires_grad_(True)
        loss = m(y)
    assert torch.equal(torch.autograd.grad(loss, y)[0], torch.autograd.grad(m(b), b)[0])
    # the raw calls give what the autograd ones do
    from convlogic_b200 import ops

    loss, stats, listed = ops.distill_fwd(x, *top[:3])
    assert torch.equal(loss, cb.distillation_loss(x, top))
    c = x.clone().requires_grad_(True)
    twice = cb.distillation_loss(c, top)
    torch.autograd.grad(twice, c, retain_graph=True)
    assert torch.equal(ops.distill_bwd(torch.ones_like(loss), x, top.indices, stats, listed), torch.autograd.grad(twice, c)[0])
    loss, counts, share = ops.balance_fwd(x, 2)
    assert torch.equal(ops.balance_bwd(torch.ones_like(loss), x, share), torch.autograd.grad(cb.balance_loss(c, 2)[0], c)[0])


def test_refusals():
    import convlogic_b200 as cb

    x = _scores(6, 40)
    values, indices, rest, _ = cb.top_logits(x, 4)
    bad = [(ValueError, "1 to 40", lambda: cb.top_logits(x, 0)), (ValueError, "1 to 40", lambda: cb.top_logits(x, 41)),
           (ValueError, "at most 128", lambda: cb.top_logits(_scores(2, 200), 129)), (ValueError, "temperature", lambda: cb.top_logits(x, 4, 0.0)),
           (ValueError, "temperature", lambda: cb.top_logits(x, 4, float("nan"))), (RuntimeError, "float32, float16 or bfloat16", lambda: cb.top_logits(x.double(), 4)),
           (RuntimeError, "float32, float16 or bfloat16", lambda: cb.top_logits(x.int(), 4)), (ValueError, "no classes", lambda: cb.top_logits(x[:, :0], 1)),
           (RuntimeError, "classes", lambda: cb.top_logits(x[0, 0], 1)),
           (ValueError, "lists must be", lambda: cb.distillation_loss(x, (values[:5], indices[:5]))),
           (ValueError, "lists must be", lambda: cb.distillation_loss(x, (values, indices[:, :3]))),
           (ValueError, "lists must be", lambda: cb.distillation_loss(x, (values[0], indices[0]))),
           (ValueError, "empty", lambda: cb.distillation_loss(x, (values[:, :0], indices[:, :0]))),
           (ValueError, "at most 128", lambda: cb.distillation_loss(x, (values.repeat(1, 33), indices.repeat(1, 33)))),
           (RuntimeError, "int64", lambda: cb.distillation_loss(x, (values, indices.int()))),
           (RuntimeError, "floating", lambda: cb.distillation_loss(x, (indices, indices))),
           (ValueError, "rest", lambda: cb.distillation_loss(x, (values, indices, rest[:5]))),
           (RuntimeError, "must be on", lambda: cb.distillation_loss(x, (values.cpu(), indices))),
           (RuntimeError, "must be on", lambda: cb.distillation_loss(x, (values, indices.cpu()))),
           (RuntimeError, "no gradient", lambda: cb.distillation_loss(x, (values.requires_grad_(True), indices))),
           (ValueError, "weight", lambda: cb.distillation_loss(x, (values.detach(), indices), weight=torch.ones(7, device="cuda"))),
           (RuntimeError, "no gradient", lambda: cb.distillation_loss(x, (values.detach(), indices), weight=torch.ones(6, device="cuda", requires_grad=True))),
           (ValueError, "reduction", lambda: cb.distillation_loss(x, (values.detach(), indices), reduction="batch")),
           (ValueError, "temperature", lambda: cb.distillation_loss(x, (values.detach(), indices), temperature=-1.0)),
           (ValueError, "got 4", lambda: cb.distillation_loss(x, (values, indices, rest, rest))),
           (RuntimeError, "float32, float16 or bfloat16", lambda: cb.distillation_loss(x.double(), (values.detach(), indices))),
           (ValueError, "1 to 32", lambda: cb.balance_loss(x, 33)), (ValueError, "1 to 32", lambda: cb.balance_loss(x, 0)),
           (ValueError, "1024", lambda: cb.balance_loss(_scores(2, 1025))), (RuntimeError, "bool", lambda: cb.balance_loss(x, 1, torch.ones(6, device="cuda"))),
           (ValueError, "keep", lambda: cb.balance_loss(x, 1, torch.ones(5, dtype=torch.bool, device="cuda"))),
           (RuntimeError, "must be on", lambda: cb.balance_loss(x, 1, torch.ones(6, dtype=torch.bool)))]
    for kind, match, call in bad:
        with pytest.raises(kind, match=match):
            call()
    assert float(cb.distillation_loss(x, (values.detach(), indices, rest))) < 1e-5     # and nothing is left behind


@pytest.mark.parametrize("n,v", [(512, 10), (300, 1000), (3, 140000)])
def test_every_launch_is_traced(n, v):
    import convlogic_b200 as cb
    from convlogic_b200 import _lib

    x, teacher = _scores(n, v).requires_grad_(True), _scores(n, v, seed=1)
    torch.cuda.synchronize()
    _lib.trace(True)
    before = _lib.lib().clb_kernel_launches()
    loss = cb.distillation_loss(x, cb.top_logits(teacher, 4)) + cb.balance_loss(x[:, :10])[0]
    loss.backward()
    torch.cuda.synchronize()
    counted = _lib.lib().clb_kernel_launches() - before
    names = _lib.trace_report()
    _lib.trace(False)
    assert counted > 0 and sum(c for c, _ in names.values()) == counted, names


def test_a_million_rows():
    """More rows than one block adds up.  Terms of one size: each row's loss is within 2e-4 of its own, and so is their mean; 64 bits add them."""
    import convlogic_b200 as cb

    x, teacher = torch.randn(1000003, 5, device="cuda"), torch.randn(1000003, 5, device="cuda")
    top = cb.top_logits(teacher, 2)
    rows = cb.distillation_loss(x, top, reduction="none")
    total = rows.double().sum()
    for how, want in (("sum", total), ("mean", total / 1000003)):
        got = cb.distillation_loss(x, top, reduction=how)
        # rows are rounded to 2^-24 of their size before they are added; the mean's are scaled by a rounded divisor (2^-24) before that
        assert abs(float(got) - float(want)) <= 4 * 2.0 ** -24 * float(want)
    loss, counts = cb.balance_loss(x, 2)
    assert int(counts.sum()) == 2 * 1000003
    p = torch.softmax(x.double(), 1)
    want = 5 * (counts.double() / (2 * 1000003) * p.mean(0)).sum()
    assert abs(float(loss) - float(want)) <= 5e-5 * float(want)


def test_offsets_beyond_32_bits():
    """The last rows of 4.8e9 scores."""
    import convlogic_b200 as cb

    n, v = 40000, 120001
    x = torch.empty(n, v, dtype=torch.bfloat16, device="cuda")
    for part in x.split(4000):
        part.normal_(0.0, 3.0)
    top = cb.top_logits(x, 3)
    tail = cb.top_logits(x[-100:], 3)
    assert all(torch.equal(a[-100:], b) for a, b in zip(top[:3], tail[:3]))
    # (those rows begin elsewhere in their 16-byte pieces than the same rows alone, so that sums have another order: held to the definition in 64 bits)
    up = torch.rand(n, device="cuda")
    lists = (top.values.roll(1, 1), top.indices, top.rest)
    last = [t[-100:] for t in lists]
    a = x.requires_grad_(True)
    loss = cb.distillation_loss(a, lists, reduction="none")
    (grad,) = torch.autograd.grad(loss, a, up)
    want = loss_oracle.distillation(x[-100:], *last, None, 1.0, "none", up[-100:])
    check_loss(loss.detach()[-100:], want["loss"], want["loss_scale"])
    check_grad(grad[-100:], want["grad"], want["grad_scale"], x.dtype)
    del grad, loss
    (grad,) = torch.autograd.grad(cb.distillation_loss(a, lists, reduction="sum"), a)
    want = loss_oracle.distillation(x[-100:], *last, None, 1.0, "sum")
    check_grad(grad[-100:], want["grad"], want["grad_scale"], x.dtype)
    del grad
    # columns of a wide tensor: rows at a distance of 120001
    y = x.detach()[:, 119990:]
    assert torch.equal(cb.top_logits(y, 4).indices[-5:], cb.top_logits(y[-5:].clone(), 4).indices)
    assert torch.equal(cb.balance_loss(y[-100:])[1], cb.balance_loss(y[-100:].clone())[1])


def test_a_tensor_of_another_stream_and_lists_in_flight():
    """Lists made on a side stream are waited for as any tensor is; the loss's own tensors live as long as its work."""
    import convlogic_b200 as cb

    x, teacher = _scores(200, 5000).requires_grad_(True), _scores(200, 5000, seed=1)
    want = torch.autograd.grad(cb.distillation_loss(x, cb.top_logits(teacher, 20)), x)[0]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(side):
            top = cb.top_logits(teacher, 20)
        torch.cuda.current_stream().wait_stream(side)
        for t in top[:3]:
            t.record_stream(torch.cuda.current_stream())
        loss = cb.distillation_loss(x, top)
        del top
        got = torch.autograd.grad(loss, x)[0]
        assert torch.equal(got, want)
