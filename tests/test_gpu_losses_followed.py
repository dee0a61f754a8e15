"""The loss terms where something else follows the call: torch.jit.trace, a second derivative, a gradient bucket, another stream."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _scores(n=12, v=40, seed=0):
    return (torch.randn(n, v, generator=torch.Generator().manual_seed(seed)) * 3).cuda()


def _terms(top):
    """Each loss as a call of its own, as the trace of it, and as its Function."""
    import convlogic_b200 as cb
    from convlogic_b200 import functional

    plain = {"distillation": lambda s: cb.distillation_loss(s, top), "balance": lambda s: cb.balance_loss(s, 2)[0]}
    traced = {name + " traced": torch.jit.trace(f, (_scores(),), check_trace=False) for name, f in plain.items()}
    apply = {"distillation applied": lambda s: functional.DistillationFunction.apply(s, *top[:3], None, 1.0, "mean"),
             "balance applied": lambda s: functional.BalanceFunction.apply(s, 2, None)[0]}
    return {**plain, **traced, **apply}


def test_a_second_derivative_is_refused_wherever_the_first_came_from():
    """Beside another term that keeps the sum differentiable, too: nothing is left out without a word."""
    import convlogic_b200 as cb

    top = cb.top_logits(_scores(seed=1), 4)
    for name, call in _terms(top).items():
        x = _scores(seed=2).requires_grad_(True)
        (g,) = torch.autograd.grad(call(x), x, create_graph=True)
        assert g.abs().sum() > 0, name
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(g.square().sum() + x.square().sum(), x)
            pytest.fail(name)


def test_lists_and_weights_that_need_a_gradient_are_refused_in_a_trace():
    import convlogic_b200 as cb

    x, top = _scores(), cb.top_logits(_scores(seed=1), 4)

    def call(s, values, rest, weight):
        return cb.distillation_loss(s, (values, top.indices, rest), weight=weight)

    args = (x, top.values, top.rest, torch.ones(12, device="cuda"))
    traced = torch.jit.trace(call, args, check_trace=False)
    for at in range(1, 4):
        bad = list(args)
        bad[at] = bad[at].clone().requires_grad_(True)
        for run in (lambda: torch.jit.trace(call, tuple(bad), check_trace=False), lambda: traced(*bad)):
            with pytest.raises(RuntimeError, match="no gradient"):
                run()
        with torch.no_grad():
            assert torch.equal(traced(*bad), call(*args))


def _direct():
    """A layer whose gradient is written straight into a bucket."""
    import convlogic_b200 as cb

    net = torch.nn.Sequential(cb.LogicLayer(64, 400), cb.GroupSum(10, 3.0)).cuda().train()
    bucket = cb.GradBucket(net)
    return net, bucket, net[0].weights


def test_a_trace_does_not_lose_a_balance_loss_beside_direct_gradients():
    import convlogic_b200 as cb

    net, bucket, w = _direct()

    class Balance(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = w

        def forward(self, scale):
            return cb.balance_loss(self.w)[0] * scale

    one = torch.ones((), device="cuda")
    early = torch.jit.trace(Balance(), (one,), check_trace=False)
    bucket.direct()
    for call in (lambda: torch.jit.trace(Balance(), (one,), check_trace=False), lambda: early(one)):
        with pytest.raises(RuntimeError, match="direct"):
            call()
    with torch.no_grad():
        early(one)
    bucket.direct(False)
    assert torch.equal(early(one), cb.balance_loss(w)[0])


def test_views_of_a_parameter_are_refused_beside_direct_gradients():
    import convlogic_b200 as cb

    net, bucket, w = _direct()
    views = (lambda: w.view(40, 10, 16), lambda: w[:100], lambda: w.view(-1, 16)[3:].unsqueeze(0), lambda: w.t(), lambda: w.detach().requires_grad_(True))
    before = [cb.balance_loss(v())[0].detach() for v in views]
    bucket.direct()
    for v in views[:-1]:
        with pytest.raises(RuntimeError, match="direct"):
            cb.balance_loss(v())
        with torch.no_grad():
            cb.balance_loss(v())
    assert torch.equal(cb.balance_loss(views[-1]())[0].detach(), before[-1])     # no longer the parameter's
    scores = net(torch.rand(50, 64, device="cuda"))
    cb.balance_loss(scores)[0].backward()                                        # logits that a layer has made
    bucket.direct(False)
    for v, b in zip(views, before):
        assert torch.equal(cb.balance_loss(v())[0].detach(), b)
