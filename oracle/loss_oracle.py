"""The loss terms on rows of scores, restated in 64 bits on the CPU: top logits, distillation from lists of them, balance over experts.

Gradients come from autograd over the definition, not from a formula.  Beside each result stands what its rounding errors scale with:
``..._scale`` tensors of the result's shape, the sum of the magnitudes that are added up to it."""

import numpy as np
import torch

INF = float("inf")


def top_logits(x, k, temperature=1.0):
    """(values, indices, rest) of rows [N, V]: descending, NaN first, equal values by index."""
    x = x.detach().cpu().double()
    n, v = x.shape
    a = x.numpy()
    nan = np.isnan(a)
    order = np.stack([np.lexsort((np.arange(v), -np.where(m, 0.0, r), ~m)) for r, m in zip(a, nan)]) if n else np.zeros((0, v), dtype=np.int64)
    indices = torch.from_numpy(order[:, :k].astype(np.int64))
    rest = x.scatter(1, indices, -INF) / temperature
    return x.gather(1, indices), indices, torch.logsumexp(rest, 1) if n else torch.zeros(0, dtype=torch.float64)


def distillation(scores, values, indices, rest=None, weight=None, temperature=1.0, reduction="mean", upstream=1.0):
    """{"loss", "grad", "loss_scale", "grad_scale"} for scores [N, V] and lists [N, k]."""
    s = scores.detach().cpu().double().requires_grad_(True)
    n, v = s.shape
    t = temperature
    idx = indices.detach().cpu()
    there = (idx >= 0) & (idx < v)
    safe = torch.where(there, idx, torch.zeros_like(idx))
    tv = torch.where(there, values.detach().cpu().double() / t, torch.tensor(-INF, dtype=torch.float64))
    rs = torch.full((n,), -INF, dtype=torch.float64) if rest is None else rest.detach().cpu().double()
    w = torch.ones(n, dtype=torch.float64) if weight is None else weight.detach().cpu().double()
    mass = torch.logsumexp(torch.cat([tv, rs[:, None]], 1), 1)
    on = (w != 0) & (mass != -INF) & ~(s.detach() == -INF).all(1)
    s1 = torch.where(on[:, None], s, torch.zeros_like(s))
    log_p, log_r = tv - torch.where(on, mass, torch.zeros_like(mass))[:, None], rs - torch.where(on, mass, torch.zeros_like(mass))
    p, r = torch.where(on[:, None], log_p.exp(), torch.zeros_like(log_p)), torch.where(on, log_r.exp(), torch.zeros_like(log_r))
    log_q = torch.log_softmax(s1 / t, 1)
    listed = torch.zeros(n, v, dtype=torch.bool)
    for i in range(idx.shape[1]):
        listed[torch.arange(n)[there[:, i]], idx[there[:, i], i]] = True

    def term(prob, log_prob, log_other):  # nothing where prob is nothing
        use = (prob > 0) | torch.isnan(prob)
        return torch.where(use, prob * (torch.where(use, log_prob, torch.zeros_like(log_prob)) - torch.where(use, log_other, torch.zeros_like(log_other))),
                           torch.zeros_like(prob))

    lq = log_q.gather(1, safe)
    unlisted = log_q.masked_fill(listed, -INF)
    with_rest = ((r > 0) | torch.isnan(r)) & ~(unlisted.detach() == -INF).all(1)
    lqr = torch.logsumexp(torch.where(with_rest[:, None], unlisted, torch.zeros_like(unlisted)), 1)
    lqr = torch.where(with_rest, lqr, torch.full_like(lqr, -INF))
    rows = term(p, log_p, lq).sum(1) + term(r, log_r, lqr)
    factor = t * t * w / (n if reduction == "mean" else 1)
    loss = torch.where(on, rows * torch.where(on, factor, torch.ones_like(factor)), torch.zeros_like(rows))
    up = torch.as_tensor(upstream).detach().cpu().double()
    (grad,) = torch.autograd.grad((loss * up).sum(), s) if n else (torch.zeros_like(s),)
    q = log_q.detach().exp()
    dense = torch.zeros(n, v, dtype=torch.float64).scatter_add_(1, safe, torch.where(there, p, torch.zeros_like(p)))
    ratio = torch.where(r > 0, r * torch.exp(-lqr.detach()), torch.zeros_like(r))
    scale = torch.where(listed, q + dense, q * (1 + ratio)[:, None]) * (factor / t * up.abs()).abs()[:, None]
    size = torch.where(p > 0, p * (log_p.abs() + lq.detach().abs()), torch.zeros_like(p)).sum(1) + torch.where(r > 0, r * (log_r.abs() + lqr.detach().abs()), torch.zeros_like(r))
    row_scale = torch.where(on, factor.abs() * (1 + size), torch.zeros_like(size))
    grad = torch.where(on[:, None], grad, torch.zeros_like(grad))
    if reduction == "none":
        return {"loss": loss.detach(), "grad": grad, "loss_scale": row_scale, "grad_scale": scale}
    return {"loss": loss.detach().sum(), "grad": grad, "loss_scale": row_scale.sum(), "grad_scale": scale}


def balance(x, k=1, keep=None, upstream=1.0):
    """{"loss", "counts", "grad", "loss_scale", "grad_scale"} of rows [R, E]."""
    x = x.detach().cpu().double()
    n, e = x.shape
    kept = ~(x == -INF).all(1) if n else torch.zeros(0, dtype=torch.bool)
    if keep is not None:
        kept &= keep.cpu()
    a = x[kept].clone().requires_grad_(True)
    m = a.shape[0]
    _, order, _ = top_logits(a, k)
    chosen = a.detach().gather(1, order) != -INF
    counts = torch.zeros(e, dtype=torch.int64).index_add_(0, order.reshape(-1), chosen.reshape(-1).long())
    grad, scale = torch.zeros(n, e, dtype=torch.float64), torch.zeros(n, e, dtype=torch.float64)
    if m == 0:
        return {"loss": torch.zeros((), dtype=torch.float64), "counts": counts, "grad": grad, "loss_scale": torch.zeros(()), "grad_scale": scale}
    p = torch.softmax(a, 1)
    f = counts.double() / (m * k)
    loss = e * (f * p.mean(0)).sum()
    (g,) = torch.autograd.grad(loss * upstream, a)
    grad[kept] = g
    h = (f - f.mean()).abs() * e / m * abs(upstream)
    pd = p.detach()
    h = h + 2.0 ** -36 * f.max() * e / m * abs(upstream)   # the roundings here, 2^-52 of what cancels, against a tolerance of 2^-15
    scale[kept] = pd * (h + (pd * h).sum(1, keepdim=True))
    return {"loss": loss.detach(), "counts": counts, "grad": grad, "loss_scale": loss.detach(), "grad_scale": scale}
