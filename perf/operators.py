"""Timed cases of the sparse-MLP and dropout operators of :mod:`resihp.ops.functional`.

Five operators, in the order a sparse (mixture-of-experts) block of a decoder calls them:

* ``route``    router logits -> the k chosen experts of every token, their weights, and the
               plan that sorts the (token, choice) pairs by expert;
* ``dispatch`` token rows copied into the plan's order, one copy per choice;
* ``grouped``  one linear layer per expert over its run of the sorted rows;
* ``combine``  every token's weighted sum of its k expert rows, plus the residual stream;
* ``dropout``  inverted dropout whose mask is recomputed from a counter, plus the residual.

``own`` selects what :func:`run` calls: the package's operators, or the same mathematics in
elementary torch operations in 32 bits. :func:`exact` states each operator once more, in 64
bits. Inputs depend on the case and the seed alone.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------


def listed():
    return [
        # a router on the few tokens of one short sequence: launch latency is what counts
        dict(name="route 64x8 top2", op="route", tokens=64, experts=8, k=2, dtype="bf16", normalize=True, masked=False),
        # many fine-grained experts over a long batch, softmax over all of them, some experts masked
        dict(name="route 32768x64 top4", op="route", tokens=32768, experts=64, k=4, dtype="fp32", normalize=False,
             masked=True),
        # the micro-batch of the 1.3B decoder (2 x 2048 tokens, width 2048), forward and backward
        dict(name="dispatch 4096x2048 top2", op="dispatch", tokens=4096, dim=2048, experts=8, k=2, dropped=False),
        # odd numbers of tokens and channels, some choices routed nowhere (another rank's experts)
        dict(name="dispatch 1021x1003 top6", op="dispatch", tokens=1021, dim=1003, experts=61, k=6, dropped=True),
        # gate and up projection of eight experts at the 1.3B widths, forward, input and weight gradient
        dict(name="grouped 8192 2048>11008 step", op="grouped", rows=8192, experts=8, inner=2048, outer=11008,
             skew=False, mode="step"),
        # down projection at the 13B widths, forward: the largest product
        dict(name="grouped 16384 13824>5120", op="grouped", rows=16384, experts=8, inner=13824, outer=5120, skew=True,
             mode="forward"),
        # eight tokens with two experts each: every expert's weights are read for two rows
        dict(name="grouped 16 2048>11008", op="grouped", rows=16, experts=8, inner=2048, outer=11008, skew=False,
             mode="forward"),
        # many small experts, very uneven, some without rows; weight gradients written, not accumulated
        dict(name="grouped 6001 1024>1416 fresh", op="grouped", rows=6001, experts=64, inner=1024, outer=1416,
             skew=True, mode="fresh"),
        # the 1.3B micro-batch with its residual stream, forward and backward
        dict(name="combine 4096x2048 top2", op="combine", tokens=4096, dim=2048, experts=8, k=2, dropped=False,
             residual=True),
        # a few tokens at the 13B width, eight choices each, some routed nowhere
        dict(name="combine 37x5120 top8", op="combine", tokens=37, dim=5120, experts=64, k=8, dropped=True,
             residual=False),
        # the 1.3B micro-batch: a block's output dropped out and added to the residual stream
        dict(name="dropout 4096x2048", op="dropout", rows=4096, dim=2048, p=0.1, dtype="bf16", residual=True),
        # a long batch at the 13B width without a residual, as after an embedding
        dict(name="dropout 16384x5120", op="dropout", rows=16384, dim=5120, p=0.25, dtype="bf16", residual=False),
    ]


def _log(rng, low, high):
    """A whole number spread evenly over the logarithm of low..high."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("route", "dispatch", "grouped", "grouped", "combine", "dropout"))
    if op == "route":
        experts = _log(rng, 2, 256)
        return dict(op=op, tokens=_log(rng, 1, 65536), experts=experts, k=min(experts, rng.randint(1, 8)),
                    dtype=rng.choice(("bf16", "fp32")), normalize=rng.random() < 0.5, masked=rng.random() < 0.3)
    if op in ("dispatch", "combine"):
        experts = _log(rng, 2, 256)
        k = min(experts, rng.randint(1, 8))
        dim = _log(rng, 64, 8192)
        if rng.random() < 0.75:  # most widths are a whole number of 16-byte vectors
            dim = max(64, dim // 8 * 8)
        tokens = _log(rng, 1, max(1, min(32768, (1 << 28) // (dim * k))))
        case = dict(op=op, tokens=tokens, dim=dim, experts=experts, k=k, dropped=rng.random() < 0.3)
        if op == "combine":
            case["residual"] = rng.random() < 0.7
        return case
    if op == "grouped":
        experts = _log(rng, 1, 128)
        mode = rng.choice(("forward", "step", "fresh"))
        most = 180_000_000 if mode == "forward" else 60_000_000  # elements of all experts' weights
        inner = _log(rng, 64, 8192) // 8 * 8
        outer = _log(rng, 64, max(72, min(14336, most // (inner * experts)))) // 8 * 8
        products = 5e11 if mode == "forward" else 1.5e11  # multiply-adds of one product
        rows = _log(rng, 1, max(2, min(32768, int(products / (inner * outer)))))
        return dict(op=op, rows=rows, experts=experts, inner=inner, outer=outer, skew=rng.random() < 0.5, mode=mode)
    dim = _log(rng, 64, 14336)
    if rng.random() < 0.75:
        dim = max(64, dim // 8 * 8)
    return dict(op=op, rows=_log(rng, 1, min(32768, 84_000_000 // dim)), dim=dim, p=round(rng.uniform(0.0, 0.6), 3),
                dtype=rng.choice(("bf16", "bf16", "fp32")), residual=rng.random() < 0.6)


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------


def _sizes(case, seed):
    """Rows of every expert: near even, or uneven with every eighth expert left without rows."""
    n, e = case["rows"], case["experts"]
    rng = np.random.default_rng(seed)
    if not case["skew"]:
        base = np.full(e, n // e)
        base[rng.permutation(e)[: n % e]] += 1
        spread = rng.integers(0, np.maximum(1, base // 8 + 1))  # some rows of each move to the next expert
        return (base - spread + np.roll(spread, 1)).tolist()
    share = 1.0 / (1.0 + np.arange(e))
    share[7::8] = 0.0
    return rng.multinomial(n, rng.permutation(share / share.sum())).tolist()


def _choices(case, seed):
    """``[tokens, k]`` distinct experts of every token, popular ones first, some of them -1."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    t, e, k = case["tokens"], case["experts"], case["k"]
    score = torch.rand(t, e, generator=g, device=DEVICE) + 0.3 * torch.rand(e, generator=g, device=DEVICE)
    ids = score.argsort(dim=1, descending=True, stable=True)[:, :k].to(torch.int32)
    if case["dropped"]:
        ids[torch.rand(t, k, generator=g, device=DEVICE) < 0.25] = -1
    return ids


def _plan(ids, experts):
    """Offsets of every expert's run and the sorted place of every choice; -1 goes to the end."""
    flat = ids.reshape(-1).long()
    key = torch.where(flat < 0, torch.full_like(flat, experts), flat)
    order = key.argsort(stable=True)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(flat.numel(), device=flat.device)
    counts = (key[:, None] == torch.arange(experts, device=flat.device)).sum(0)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=flat.device)
    offsets[1:] = counts.cumsum(0)
    return offsets, slots.to(torch.int32).view(ids.shape)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, scale=1.0):
        return (torch.randn(*shape, generator=g, device=DEVICE) * scale).to(dtype)

    op, s = case["op"], dict(case=case)
    if op == "route":
        t, e = case["tokens"], case["experts"]
        logits = torch.randn(t, e, generator=g, device=DEVICE) + 0.5 * torch.randn(e, generator=g, device=DEVICE)
        if case["masked"]:  # a quarter of all choices is not allowed, and some tokens are padding
            logits[torch.rand(t, e, generator=g, device=DEVICE) < 0.25] = float("-inf")
            logits[torch.rand(t, generator=g, device=DEVICE) < 0.02] = float("-inf")
        s["logits"] = logits.to(DTYPES[case["dtype"]])
        s["dweights"] = normal(t, case["k"], dtype=torch.float32)
    elif op in ("dispatch", "combine"):
        t, d, k = case["tokens"], case["dim"], case["k"]
        s["ids"] = _choices(case, seed)
        s["offsets"], s["slots"] = _plan(s["ids"], case["experts"])
        if op == "dispatch":
            s["x"], s["dy"] = normal(t, d), normal(t * k, d)
        else:
            s["y"], s["dout"] = normal(t * k, d), normal(t, d)
            s["weights"] = torch.rand(t, k, generator=g, device=DEVICE)
            s["residual"] = normal(t, d) if case["residual"] else None
    elif op == "grouped":
        n, e, i, o = case["rows"], case["experts"], case["inner"], case["outer"]
        s["sizes"] = _sizes(case, seed)
        s["offsets"] = torch.tensor([0] + np.cumsum(s["sizes"]).tolist(), dtype=torch.int32, device=DEVICE)
        s["x"] = normal(n, i)
        s["w"] = torch.empty(e, o, i, dtype=torch.bfloat16, device=DEVICE)
        for k in range(e):
            s["w"][k] = normal(o, i, scale=0.02)
        if case["mode"] != "forward":
            s["dy"] = normal(n, o)
        if case["mode"] == "step":  # what earlier micro-batches left in the accumulator
            s["main_grad"] = normal(e, o, i, dtype=torch.float32)
    else:
        dtype = DTYPES[case["dtype"]]
        s["x"], s["dout"] = normal(case["rows"], case["dim"], dtype=dtype), normal(case["rows"], case["dim"], dtype=dtype)
        s["residual"] = normal(case["rows"], case["dim"], dtype=dtype) if case["residual"] else None
        s["seed"], s["offset"] = 0x5EED_0000_0000 + seed, 7 * seed + 3
    if own:  # leaves of the training graph
        for name in ("logits", "x", "y", "weights", "residual"):
            if s.get(name) is not None and not (op == "grouped" and case["mode"] == "forward"):
                s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    return (_OWN if own else _PLAIN)[op](s)


def _own_route(s):
    from resihp.ops import functional as fn

    c = s["case"]
    weights, ids, plan = fn.moe_route(s["logits"], c["k"], normalize=c["normalize"])
    (dlogits,) = torch.autograd.grad(weights, s["logits"], s["dweights"])
    return {"weights": weights.detach(), "ids": ids, "offsets": plan.offsets, "slots": plan.slots, "dlogits": dlogits}


def _own_dispatch(s):
    from resihp.ops import functional as fn

    y = fn.moe_dispatch(s["x"], fn.MoePlan(s["offsets"], s["slots"]))
    (dx,) = torch.autograd.grad(y, s["x"], s["dy"])
    return {"y": y.detach(), "dx": dx}


def _own_grouped(s):
    from resihp.ops import functional as fn

    mode = s["case"]["mode"]
    if mode == "forward":
        return {"y": fn.grouped_linear(s["x"], s["w"], s["offsets"])}
    if mode == "step":
        y = fn.grouped_linear(s["x"], s["w"], s["offsets"], main_grad=s["main_grad"])
        (dx,) = torch.autograd.grad(y, s["x"], s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": s["main_grad"]}
    y = fn.grouped_linear(s["x"], s["w"], s["offsets"])
    (dx,) = torch.autograd.grad(y, s["x"], s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": fn.grouped_wgrad(s["dy"], s["x"].detach(), s["offsets"])}


def _own_combine(s):
    from resihp.ops import functional as fn

    out = fn.moe_combine(s["y"], s["weights"], fn.MoePlan(s["offsets"], s["slots"]), residual=s["residual"])
    leaves = [s["y"], s["weights"]] + ([s["residual"]] if s["residual"] is not None else [])
    grads = torch.autograd.grad(out, leaves, s["dout"])
    return {"out": out.detach(), **dict(zip(("dy", "dweights", "dresidual"), grads))}


def _own_dropout(s):
    from resihp.ops import functional as fn

    out = fn.dropout(s["x"], s["case"]["p"], s["seed"], s["offset"], residual=s["residual"])
    leaves = [s["x"]] + ([s["residual"]] if s["residual"] is not None else [])
    grads = torch.autograd.grad(out, leaves, s["dout"])
    return {"out": out.detach(), **dict(zip(("dx", "dresidual"), grads))}


_OWN = {"route": _own_route, "dispatch": _own_dispatch, "grouped": _own_grouped, "combine": _own_combine,
        "dropout": _own_dropout}


# --- the plain forms ---------------------------------------------------------------------


def _plain_route(s):
    """The k largest logits of every token, the lowest index first among equal ones. A logit of
    -inf is an expert that the token may not use: it is never chosen, and where fewer than k are
    left the remaining choices are -1 with weight 0. Weights are the softmax over all experts, or
    with ``normalize`` over the chosen ones."""
    c = s["case"]
    x = s["logits"].float()
    top, ids = x.sort(dim=1, descending=True, stable=True)
    top, ids = top[:, : c["k"]], ids[:, : c["k"]]
    allowed = top != float("-inf")
    m = x.max(dim=1, keepdim=True).values
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    e = (x - m).exp()
    chosen = torch.where(allowed, (top - m).exp(), torch.zeros_like(top))
    total = (chosen if c["normalize"] else e).sum(1, keepdim=True)
    total = torch.where(total == 0, torch.ones_like(total), total)
    weights = chosen / total
    ids_out = torch.where(allowed, ids, torch.full_like(ids, -1)).to(torch.int32)
    offsets, slots = _plan(ids_out, c["experts"])
    # d weights_j / d logit_e = weights_j (1[e is choice j] - p_e), p the softmax that was taken
    dot = (weights * s["dweights"]).sum(1, keepdim=True)
    dlogits = torch.zeros_like(x) if c["normalize"] else -(e / total) * dot
    dlogits.scatter_add_(1, ids, weights * (s["dweights"] - dot) if c["normalize"] else weights * s["dweights"])
    return {"weights": weights, "ids": ids_out, "offsets": offsets, "slots": slots,
            "dlogits": dlogits.to(s["logits"].dtype)}


def _plain_dispatch(s):
    t, k = s["slots"].shape
    slots = s["slots"].long()
    kept = s["ids"] >= 0
    y = torch.zeros(t * k, s["case"]["dim"], device=DEVICE)
    dx = torch.zeros(t, s["case"]["dim"], device=DEVICE)
    for j in range(k):
        y[slots[:, j]] = s["x"].float() * kept[:, j, None]
        dx += s["dy"][slots[:, j]].float() * kept[:, j, None]
    return {"y": y.to(s["x"].dtype), "dx": dx.to(s["x"].dtype)}


def _plain_grouped(s):
    mode = s["case"]["mode"]
    y = torch.empty(s["case"]["rows"], s["case"]["outer"], dtype=torch.bfloat16, device=DEVICE)
    out = {"y": y}
    if mode != "forward":
        out["dx"] = torch.empty_like(s["x"])
        out["dw"] = s["main_grad"] if mode == "step" else torch.empty(s["w"].shape, dtype=torch.float32, device=DEVICE)
    at = 0
    for e, n in enumerate(s["sizes"]):
        x, w = s["x"][at: at + n].float(), s["w"][e].float()
        y[at: at + n] = (x @ w.t()).to(y.dtype)
        if mode != "forward":
            dy = s["dy"][at: at + n].float()
            out["dx"][at: at + n] = (dy @ w).to(y.dtype)
            if mode == "step":
                out["dw"][e] += dy.t() @ x
            else:
                out["dw"][e] = dy.t() @ x
        at += n
    return out


def _plain_combine(s):
    k = s["slots"].shape[1]
    slots = s["slots"].long()
    kept = s["ids"] >= 0
    dout = s["dout"].float()
    out = torch.zeros_like(dout) if s["residual"] is None else s["residual"].float()
    dy = torch.zeros_like(s["y"])
    dweights = torch.zeros_like(s["weights"])
    for j in range(k):
        rows = torch.where(kept[:, j, None], s["y"][slots[:, j]].float(), torch.zeros((), device=DEVICE))
        w = s["weights"][:, j, None]
        out = out + w * rows
        dy[slots[:, j]] = (w * dout * kept[:, j, None]).to(dy.dtype)
        dweights[:, j] = (rows * dout).sum(1)
    grads = {"out": out.to(s["y"].dtype), "dy": dy, "dweights": dweights}
    return grads if s["residual"] is None else {**grads, "dresidual": s["dout"]}


def _mul32(a, b):
    """High and low 32 bits of the product of two 32-bit numbers held in int64."""
    a0, a1 = a & 0xFFFF, a >> 16
    b0, b1 = b & 0xFFFF, b >> 16
    low = a0 * b0
    mid = a1 * b0 + (low >> 16)
    mid2 = a0 * b1 + (mid & 0xFFFF)
    return a1 * b1 + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | (low & 0xFFFF)


def _keep(s):
    """Philox4x32-10 (Salmon et al., SC 2011) with key ``seed`` and counter (block, offset); the
    eight 16-bit numbers of block b belong to the elements 8b..8b+7, and one is kept where its
    number is at least p * 65536."""
    n = s["x"].numel()
    block = torch.arange(-(-n // 8), device=DEVICE)
    c0, c1 = block & 0xFFFFFFFF, block >> 32
    c2 = torch.full_like(block, s["offset"] & 0xFFFFFFFF)
    c3 = torch.full_like(block, (s["offset"] >> 32) & 0xFFFFFFFF)
    k0, k1 = s["seed"] & 0xFFFFFFFF, (s["seed"] >> 32) & 0xFFFFFFFF
    for _ in range(10):
        hi0, lo0 = _mul32(c0, 0xD2511F53)
        hi1, lo1 = _mul32(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = hi1 ^ c1 ^ k0, lo1, hi0 ^ c3 ^ k1, lo0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    halves = [h for c in (c0, c1, c2, c3) for h in (c & 0xFFFF, c >> 16)]
    u = torch.stack([h.to(torch.int32) for h in halves], 1).reshape(-1)[:n]
    drop = round(s["case"]["p"] * 65536)
    return (u >= drop).view(s["x"].shape), 65536.0 / (65536 - drop)


def _plain_dropout(s):
    keep, scale = _keep(s)
    zero = torch.zeros((), device=DEVICE)
    out = torch.where(keep, s["x"].float() * scale, zero)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    grads = {"out": out.to(s["x"].dtype), "dx": torch.where(keep, s["dout"].float() * scale, zero).to(s["x"].dtype)}
    return grads if s["residual"] is None else {**grads, "dresidual": s["dout"]}


_PLAIN = {"route": _plain_route, "dispatch": _plain_dispatch, "grouped": _plain_grouped, "combine": _plain_combine,
          "dropout": _plain_dropout}


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        size = 2 if case["dtype"] == "bf16" else 4
        # logits read, weights, ids, places and offsets written; weights' gradient read, the logits' written
        return {"bytes": 2 * t * e * size + t * k * 16 + 4 * (e + 1), "flops": 8 * t * e}
    if op == "dispatch":
        t, d, k = case["tokens"], case["dim"], case["k"]
        return {"bytes": 2 * (t * d * 2 + t * k * d * 2) + t * k * 4, "flops": t * k * d}
    if op == "combine":
        t, d, k = case["tokens"], case["dim"], case["k"]
        rows, row = t * k * d * 2, t * d * 2
        # forward and backward of one pass: y, the residual, dout read; out, dy and weight gradients written
        return {"bytes": 2 * rows + (3 if case["residual"] else 2) * row + t * k * 12, "flops": 5 * t * k * d}
    if op == "grouped":
        n, e, i, o = case["rows"], case["experts"], case["inner"], case["outer"]
        used = e - e // 8 if case["skew"] else e
        weights = min(used, n) * i * o
        total = 2 * (weights + n * i + n * o)
        products = 1
        if case["mode"] != "forward":
            total += 2 * (n * i + n * o) + (8 * weights if case["mode"] == "step" else 4 * e * i * o)
            products = 3
        return {"bytes": total, "flops": products * 2.0 * n * i * o}
    size = 2 if case["dtype"] == "bf16" else 4
    n = case["rows"] * case["dim"]
    return {"bytes": n * size * (5 if case["residual"] else 4), "flops": 4 * n}


# ---------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach() if torch.is_tensor(v) else v for k, v in s.items()}
    return _EXACT[case["op"]](case, s)


def _exact_route(c, s):
    x = s["logits"].double()
    t, e = x.shape
    left = x.clone()
    picked = torch.zeros(t, e, dtype=torch.bool, device=DEVICE)
    index = torch.arange(e, device=DEVICE)
    ids = torch.full((t, c["k"]), -1, dtype=torch.int64, device=DEVICE)
    for j in range(c["k"]):  # the largest that is left, and the first of those
        best = left.amax(1, keepdim=True)
        first = torch.where(left == best, index, e).amin(1)
        some = best[:, 0] > float("-inf")
        ids[:, j] = torch.where(some, first, torch.full_like(first, -1))
        here = (index == first[:, None]) & some[:, None]
        picked |= here
        left[here] = float("-inf")
    among = picked if c["normalize"] else x > float("-inf")
    p = torch.where(among, x, torch.full_like(x, float("-inf"))).softmax(1).nan_to_num(0.0)
    at = ids.clamp_min(0)
    weights = p.gather(1, at) * (ids >= 0)
    up = torch.zeros_like(p).scatter_add_(1, at, s["dweights"].double() * (ids >= 0))
    dlogits = p * (up - (p * up).sum(1, keepdim=True))
    return {"weights": weights, "ids": None, "offsets": None, "slots": None, "dlogits": dlogits}


def _rows_of(s):
    """For every sorted place: the token it belongs to, and whether it holds a routed choice."""
    t, k = s["slots"].shape
    token = torch.empty(t * k, dtype=torch.int64, device=DEVICE)
    token[s["slots"].reshape(-1).long()] = torch.arange(t, device=DEVICE).repeat_interleave(k)
    return token, torch.arange(t * k, device=DEVICE) < int(s["offsets"][-1])


def _exact_dispatch(c, s):
    token, used = _rows_of(s)
    y = s["x"].double()[token] * used[:, None]
    dx = torch.zeros(c["tokens"], c["dim"], dtype=torch.float64, device=DEVICE)
    dx.index_add_(0, token[used], s["dy"].double()[used])
    return {"y": y, "dx": dx}


def _exact_grouped(c, s):
    owner = torch.repeat_interleave(torch.arange(c["experts"]), torch.tensor(s["sizes"])).to(DEVICE)
    out = {"y": torch.empty(c["rows"], c["outer"], dtype=torch.float64, device=DEVICE)}
    if c["mode"] != "forward":
        out["dx"] = torch.empty(c["rows"], c["inner"], dtype=torch.float64, device=DEVICE)
        out["dw"] = torch.empty(c["experts"], c["outer"], c["inner"], dtype=torch.float64, device=DEVICE)
    for e in range(c["experts"]):
        rows = (owner == e).nonzero()[:, 0]
        x, w = s["x"][rows].double(), s["w"][e].double()
        out["y"][rows] = torch.einsum("ri,oi->ro", x, w)
        if c["mode"] != "forward":
            dy = s["dy"][rows].double()
            out["dx"][rows] = torch.einsum("ro,oi->ri", dy, w)
            dw = torch.einsum("ro,ri->oi", dy, x)
            out["dw"][e] = dw + s["main_grad"][e].double() if c["mode"] == "step" else dw
    return out


def _exact_combine(c, s):
    token, used = _rows_of(s)
    flat = torch.empty(token.numel(), dtype=torch.float64, device=DEVICE)
    flat[s["slots"].reshape(-1).long()] = s["weights"].double().reshape(-1)
    y = torch.where(used[:, None], s["y"].double(), torch.zeros((), dtype=torch.float64, device=DEVICE))
    dout = s["dout"].double()
    out = torch.zeros_like(dout) if s["residual"] is None else s["residual"].double()
    out = out.index_add(0, token, y * flat[:, None])
    dots = torch.einsum("rd,rd->r", y, dout[token])
    grads = {"out": out, "dy": flat[:, None] * dout[token] * used[:, None],
             "dweights": dots[s["slots"].reshape(-1).long()].view(s["slots"].shape)}
    return grads if s["residual"] is None else {**grads, "dresidual": dout}


def _exact_dropout(c, s):
    n = s["x"].numel()
    mask = np.uint64(0xFFFFFFFF)
    c0 = np.arange(-(-n // 8), dtype=np.uint64)
    c = [c0 & mask, c0 >> np.uint64(32), np.full_like(c0, s["offset"] & 0xFFFFFFFF),
         np.full_like(c0, (s["offset"] >> 32) & 0xFFFFFFFF)]
    key = [s["seed"] & 0xFFFFFFFF, (s["seed"] >> 32) & 0xFFFFFFFF]
    for r in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        ka = np.uint64((key[0] + r * 0x9E3779B9) & 0xFFFFFFFF)
        kb = np.uint64((key[1] + r * 0xBB67AE85) & 0xFFFFFFFF)
        c = [(b >> np.uint64(32)) ^ c[1] ^ ka, b & mask, (a >> np.uint64(32)) ^ c[3] ^ kb, a & mask]
    words = np.stack([v.astype(np.uint32) for v in c], 1)
    u = words.view(np.uint16).reshape(-1)[:n].astype(np.int32)  # little endian: the low half first
    p = round(s["case"]["p"] * 65536) / 65536
    keep = torch.from_numpy(u >= p * 65536).to(DEVICE).view(s["x"].shape).double()
    out = s["x"].double() * keep / (1 - p)
    dx = s["dout"].double() * keep / (1 - p)
    if s["residual"] is None:
        return {"out": out, "dx": dx}
    return {"out": out + s["residual"].double(), "dx": dx, "dresidual": s["dout"].double()}


_EXACT = {"route": _exact_route, "dispatch": _exact_dispatch, "grouped": _exact_grouped, "combine": _exact_combine,
          "dropout": _exact_dropout}
