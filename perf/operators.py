"""The loss terms of a training step beside its cross-entropy, as cases that can be timed and compared.

Three operators: ``top`` (a teacher's largest logits per row and the mass of the others), ``distill`` (the loss of a student against such
lists and its gradient) and ``balance`` (counts per expert, the balance loss and its gradient; the experts of a gate layer are its 16
operations).  With ``own`` false each is computed from elementary torch operations in 32 bits, with ``own`` true by the calls of this
package.
"""

import math

import torch

own = False
DEV = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


def listed():
    return [
        # class sums of a discretised teacher on one training batch: ten classes, whole counts divided by tau, many ties
        {"name": "top 512x10 f32", "op": "top", "rows": 512, "classes": 10, "k": 4, "dtype": "float32", "T": 4.0, "values": "counts"},
        # one row of a large head: the answer to a single request
        {"name": "top 1x50257 f32", "op": "top", "rows": 1, "classes": 50257, "k": 100, "dtype": "float32", "T": 1.0, "values": "logits"},
        # a teacher's pass over a shard of images, 1000 classes
        {"name": "top 16384x1000 bf16", "op": "top", "rows": 16384, "classes": 1000, "k": 20, "dtype": "bfloat16", "T": 2.0, "values": "logits"},
        # long rows, a head padded to whole tiles whose padding is masked
        {"name": "top 1024x128000 bf16", "op": "top", "rows": 1024, "classes": 128000, "k": 64, "dtype": "bfloat16", "T": 1.0, "values": "masked"},
        # training step of a small network: class sums of ten classes
        {"name": "distill 512x10 f32", "op": "distill", "rows": 512, "classes": 10, "k": 4, "dtype": "float32", "T": 4.0, "rest": True,
         "weight": False, "reduction": "mean", "upstream": 1.0, "values": "logits"},
        # 1000 classes, lists without the rest's mass, rows weighted
        {"name": "distill 8192x1000 f32", "op": "distill", "rows": 8192, "classes": 1000, "k": 16, "dtype": "float32", "T": 2.0, "rest": False,
         "weight": True, "reduction": "sum", "upstream": 1.0, "values": "logits"},
        # odd long rows in half precision, the loss scaled as in mixed-precision training
        {"name": "distill 1000x50257 f16", "op": "distill", "rows": 1000, "classes": 50257, "k": 32, "dtype": "float16", "T": 1.0, "rest": True,
         "weight": True, "reduction": "mean", "upstream": 1024.0, "values": "logits"},
        # the largest step: a padded head, padded rows
        {"name": "distill 2048x131072 bf16", "op": "distill", "rows": 2048, "classes": 131072, "k": 64, "dtype": "bfloat16", "T": 1.0, "rest": True,
         "weight": True, "reduction": "sum", "upstream": 1.0, "values": "masked"},
        # a few long rows with a gradient for each row's own loss
        {"name": "distill 7x128001 f32", "op": "distill", "rows": 7, "classes": 128001, "k": 50, "dtype": "float32", "T": 1.5, "rest": True,
         "weight": False, "reduction": "none", "upstream": 1.0, "values": "logits"},
        # gates of a small flat layer
        {"name": "balance 20480x16 f32", "op": "balance", "rows": 20480, "experts": 16, "k": 1, "dtype": "float32", "keep": False, "values": "gates"},
        # gates of a large flat layer
        {"name": "balance 2621440x16 f32", "op": "balance", "rows": 2621440, "experts": 16, "k": 1, "dtype": "float32", "keep": False, "values": "gates"},
        # a router of many experts over a padded batch
        {"name": "balance 65536x128 bf16", "op": "balance", "rows": 65536, "experts": 128, "k": 8, "dtype": "bfloat16", "keep": True, "values": "logits"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["top", "distill", "distill", "balance"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "balance":
        experts = 16 if rng.random() < 0.3 else _log(rng, 2, 512)
        rows = _log(rng, 1, 40_000_000 // experts)
        return {"op": op, "rows": rows, "experts": experts, "k": min(experts, _log(rng, 1, 8)), "dtype": dtype, "keep": rng.random() < 0.5,
                "values": rng.choice(["gates", "logits", "masked"])}
    classes = _log(rng, 2, 131072)
    rows = _log(rng, 1, min(65536, 130_000_000 // classes))
    case = {"op": op, "rows": rows, "classes": classes, "k": min(classes, _log(rng, 1, 128)), "dtype": dtype,
            "T": rng.choice([1.0, 1.0, 1.5, 2.0, 4.0]), "values": rng.choice(["logits", "logits", "counts", "masked"])}
    if op == "distill":
        case |= {"rest": rng.random() < 0.6, "weight": rng.random() < 0.5, "reduction": rng.choice(["mean", "sum", "none"]),
                 "upstream": rng.choice([1.0, 1.0, 0.25, 1024.0])}
    return case


def _values(kind, rows, cols, gen):
    """Scores of a head, float32: noise of an untrained one, or whole counts, or with the last classes masked."""
    x = torch.randn(rows, cols, device=DEV, generator=gen)
    if kind == "counts":
        return x.mul_(12.0).round_().div_(4.0)
    if kind == "gates":
        x[:, min(3, cols - 1)] += 2.0  # the operation that layers start from
        return x
    x.mul_(3.0)
    if kind == "masked":
        x[:, cols - cols // 16:] = -math.inf
    return x


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rows, dtype = case["rows"], DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "balance":
        state["x"] = _values(case["values"], rows, case["experts"], gen).to(dtype).requires_grad_(True)
        state["keep"] = torch.rand(rows, device=DEV, generator=gen) < 0.9 if case["keep"] else None
        return state
    x = _values(case["values"], rows, case["classes"], gen).to(dtype)
    if case["op"] == "top":
        state["x"] = x
        return state
    # a teacher that the student resembles
    teacher = _values(case["values"], rows, case["classes"], gen).mul_(0.7).add_(x, alpha=0.7)
    values, indices = torch.topk(teacher, case["k"], dim=1)
    state["rest_mass"] = None
    if case["rest"]:
        teacher.scatter_(1, indices, -math.inf)
        state["rest_mass"] = torch.logsumexp(teacher.div_(case["T"]), 1)
    state["x"], state["top_values"], state["indices"] = x.requires_grad_(True), values, indices
    state["weights"] = None
    if case["weight"]:
        w = torch.rand(rows, device=DEV, generator=gen)
        state["weights"] = torch.where(w < 0.1, torch.zeros_like(w), w)
    shape = (rows,) if case["reduction"] == "none" else ()
    up = torch.rand(shape, device=DEV, generator=gen) + 0.5 if shape else torch.ones((), device=DEV)
    state["up"] = up * case["upstream"]
    return state


# ---- plain forms
def _plain_top(x, k, T):
    x = x.float()
    order = torch.sort(x, dim=1, descending=True, stable=True)
    values, indices = order.values[:, :k].contiguous(), order.indices[:, :k].contiguous()
    others = order.values[:, k:] / T
    if others.shape[1] == 0:
        return values, indices, torch.full_like(values[:, 0], -math.inf)
    return values, indices, _log_sum(others)


def _log_sum(a):
    """log sum exp over the rows; -inf for a row of nothing else."""
    top = a.amax(1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    return top[:, 0] + torch.log(torch.exp(a - top).sum(1))


def _times_log(p, log_ratio):
    """p * log_ratio, nothing where p is nothing."""
    return torch.where(p > 0, p * torch.where(p > 0, log_ratio, torch.zeros_like(log_ratio)), torch.zeros_like(p))


def _plain_distill(x, values, indices, rest, weights, T, reduction, up):
    a = x.float() / T
    t = values / T
    both = t if rest is None else torch.cat([t, rest[:, None]], 1)
    mass = _log_sum(both)[:, None]
    log_p, p = t - mass, torch.exp(t - mass)
    unlisted = a.scatter(1, indices, -math.inf)
    of_rest = _log_sum(unlisted)[:, None]
    whole = _log_sum(torch.cat([a.gather(1, indices), of_rest], 1))[:, None]
    log_q = a.gather(1, indices) - whole
    loss = _times_log(p, log_p - log_q).sum(1)
    if rest is None:
        r, log_r = torch.zeros_like(mass), mass
    else:
        log_r = rest[:, None] - mass
        r = torch.exp(log_r)
    loss = loss + _times_log(r, log_r - (of_rest - whole))[:, 0]
    factor = (T * (weights if weights is not None else torch.ones_like(loss)) / (x.shape[0] if reduction == "mean" else 1))
    loss = loss * factor * T
    scale = (factor * up)[:, None]
    shift = torch.where(of_rest == -math.inf, torch.zeros_like(of_rest), of_rest)
    grad = torch.exp(unlisted - shift) * (torch.exp(of_rest - whole) - r) * scale
    grad.scatter_(1, indices, (torch.exp(log_q) - p) * scale)
    return (loss if reduction == "none" else loss.sum()), grad.to(x.dtype)


def _plain_balance(x, k, keep):
    rows, experts = x.shape
    a = x.float()
    there = a.amax(1) > -math.inf
    if keep is not None:
        there = there & keep
    p = torch.exp(a - torch.where(there, a.amax(1), torch.zeros_like(a[:, 0]))[:, None])
    p = torch.where(there[:, None], p / p.sum(1, keepdim=True), torch.zeros_like(p))
    order = torch.sort(a, dim=1, descending=True, stable=True)
    chosen = (order.values[:, :k] > -math.inf) & there[:, None]
    counts = torch.zeros(experts, dtype=torch.int64, device=x.device)
    counts.index_add_(0, order.indices[:, :k].reshape(-1), chosen.reshape(-1).to(torch.int64))
    m = there.sum().double()
    c = counts.double()
    factor = torch.where(m > 0, experts / (m * m * k), torch.zeros_like(m))
    loss = (factor * (c * p.sum(0, dtype=torch.float64)).sum()).float()
    share = (counts.double() * factor).float()
    grad = p * (share - (p * share).sum(1, keepdim=True))
    return loss, counts, grad.to(x.dtype)


def run(state):
    x = state["x"]
    if state["op"] == "top":
        if own:
            import convlogic_b200 as cb

            top = cb.top_logits(x, state["k"], temperature=state["T"])
            return {"values": top.values, "indices": top.indices, "rest": top.rest}
        return dict(zip(("values", "indices", "rest"), _plain_top(x, state["k"], state["T"])))
    if state["op"] == "balance":
        if own:
            import convlogic_b200 as cb

            loss, counts = cb.balance_loss(x, state["k"], keep=state["keep"])
            (grad,) = torch.autograd.grad(loss, x)
            return {"loss": loss, "counts": counts, "grad": grad}
        return dict(zip(("loss", "counts", "grad"), _plain_balance(x.detach(), state["k"], state["keep"])))
    args = (state["top_values"], state["indices"], state["rest_mass"])
    if own:
        import convlogic_b200 as cb

        loss = cb.distillation_loss(x, args, temperature=state["T"], weight=state["weights"], reduction=state["reduction"])
        (grad,) = torch.autograd.grad(loss, x, state["up"])
        return {"loss": loss, "grad": grad}
    return dict(zip(("loss", "grad"), _plain_distill(x.detach(), *args, state["weights"], state["T"], state["reduction"], state["up"])))


def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "balance":
        n = case["rows"] * case["experts"]
        return {"bytes": 2 * n * b + case["experts"] * 8 + 4 + (case["rows"] if case["keep"] else 0), "flops": 8 * n}
    rows, n = case["rows"], case["rows"] * case["classes"]
    lists = rows * (12 * case["k"] + 4)
    if case["op"] == "top":
        return {"bytes": n * b + lists, "flops": 4 * n}
    if not case["rest"]:
        lists -= 4 * rows
    return {"bytes": 2 * n * b + lists + (4 * rows if case["weight"] else 0) + 4, "flops": 8 * n}


# ---- from the definitions, in 64 bits
def exact(case, seed):
    if case["rows"] * case.get("classes", case.get("experts")) > 300_000_000:
        return None
    state = prepare(case, seed)
    x = state["x"].detach()
    if case["op"] == "top":
        return _exact_top(x, case["k"], case["T"])
    if case["op"] == "balance":
        return _exact_balance(x, case["k"], state["keep"])
    parts = []
    step = max(1, 40_000_000 // case["classes"])
    for lo in range(0, case["rows"], step):  # a few rows at a time: 64 bits take four times the memory
        cut = lambda t: None if t is None else t[lo:lo + step]  # noqa: E731
        parts.append(_exact_distill(cut(x), cut(state["top_values"]), cut(state["indices"]), cut(state["rest_mass"]), cut(state["weights"]), case["T"],
                                    state["up"] if state["up"].dim() == 0 else cut(state["up"]), case["rows"] if case["reduction"] == "mean" else 1))
    loss, grad = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
    return {"loss": loss if case["reduction"] == "none" else loss.sum(), "grad": grad}


def _exact_top(x, k, T):
    values, rest = [], []
    step = max(1, 40_000_000 // x.shape[1])
    for part in x.split(step):
        part = part.double()
        got = torch.topk(part, k, dim=1)
        values.append(got.values)
        rest.append(torch.logsumexp(part.scatter(1, got.indices, -math.inf) / T, 1))
    return {"values": torch.cat(values), "indices": None, "rest": torch.cat(rest)}


def _exact_distill(x, values, indices, rest, weights, T, up, share):
    a = x.double() / T
    listed_here = torch.zeros_like(a, dtype=torch.bool).scatter_(1, indices, True)
    teacher = torch.zeros_like(a).scatter_(1, indices, torch.softmax(
        values.double() / T if rest is None else torch.cat([values.double() / T, rest.double()[:, None]], 1), 1)[:, :values.shape[1]])
    log_q = torch.log_softmax(a, 1)
    q = log_q.exp()
    r = (1.0 - teacher.sum(1)).clamp(min=0.0) if rest is None else torch.softmax(torch.cat([values.double() / T, rest.double()[:, None]], 1), 1)[:, -1]
    if rest is None:
        r = torch.zeros_like(r)
    of_rest = torch.logsumexp(log_q.masked_fill(listed_here, -math.inf), 1)
    xlogy = torch.special.xlogy
    loss = (xlogy(teacher, teacher) - torch.where(teacher > 0, teacher * log_q, torch.zeros_like(q))).sum(1)
    loss = loss + xlogy(r, r) - torch.where(r > 0, r * of_rest, torch.zeros_like(r))
    ratio = torch.where(r > 0, r * torch.exp(-of_rest), torch.zeros_like(r))
    grad = torch.where(listed_here, q - teacher, q * (1.0 - ratio)[:, None])
    w = T / share * (weights.double() if weights is not None else torch.ones_like(loss))
    return loss * w * T, grad * (w * up.double())[:, None]


def _exact_balance(x, k, keep):
    x = x.double()
    rows, experts = x.shape
    there = torch.isfinite(x).any(1)
    if keep is not None:
        there &= keep
    p = torch.softmax(x[there], 1)
    m = p.shape[0]
    if m == 0:
        return {"loss": 0.0, "counts": None, "grad": torch.zeros_like(x)}
    # an expert is chosen where fewer than k experts are before it in order of value, then of index
    chosen = torch.zeros(experts, dtype=torch.float64, device=x.device)
    left = x[there].clone()
    for _ in range(k):
        at = left.argmax(1, keepdim=True)
        best = left.amax(1, keepdim=True)
        at = torch.where(left == best, torch.arange(experts, device=x.device), experts).amin(1, keepdim=True)
        chosen.index_add_(0, at[:, 0], (best[:, 0] > -math.inf).double())
        left.scatter_(1, at, -math.inf)
    f = chosen / (m * k)
    loss = experts * (f * p.mean(0)).sum()
    grad = torch.zeros_like(x)
    grad[there] = experts / m * p * (f - (p * f).sum(1, keepdim=True))
    return {"loss": loss, "counts": None, "grad": grad}
