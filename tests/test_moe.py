"""Sparse MLP operators (routing, dispatch, per-expert products, combine) against 64-bit forms.

Tolerances count roundings: a value rounded to a type is off by at most ``eps / 2`` of it, and
an fp32 sum of ``n`` terms by at most ``n`` steps of ``2**-23`` of the sum of magnitudes (the
tensor cores' additions may truncate, hence a whole step per term).
"""

import itertools

import pytest
import torch

from resihp.ops import KernelError, check_device_errors, grouped_dgrad, grouped_linear, grouped_wgrad
from resihp.ops import functional as fn

BF = 2.0**-8   # one rounding to bf16
F32 = 2.0**-24  # one rounding to fp32
gpu = pytest.mark.gpu
NINF = float("-inf")


def near(got, want, tol, what=""):
    """Elementwise |got - want| <= tol, everything in 64 bits; NaN nowhere."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    tol = tol.detach().double().cpu() if torch.is_tensor(tol) else torch.full_like(want, tol)
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what} {int(bad.sum())} of {bad.numel()} off, first at {at}: {got[at]} for {want[at]} +- {tol[at]}")


# ---------------------------------------------------------------------------------------
# the definitions, in 64 bits on the CPU
# ---------------------------------------------------------------------------------------


def route64(logits, k, normalize):
    x = logits.detach().double().cpu()
    t, e = x.shape
    ids = torch.full((t, k), -1, dtype=torch.int64)
    weights = torch.zeros(t, k, dtype=torch.float64)
    probs = torch.zeros(t, e, dtype=torch.float64)
    for r in range(t):
        order = sorted((i for i in range(e) if x[r, i] != NINF), key=lambda i: (-x[r, i].item(), i))[:k]
        if not order:
            continue
        among = order if normalize else [i for i in range(e) if x[r, i] != NINF]
        probs[r, among] = torch.softmax(x[r, among], 0)
        ids[r, : len(order)] = torch.tensor(order)
        weights[r, : len(order)] = probs[r, order]
    return weights, ids, probs


def plan64(ids, experts, start=0):
    flat = ids.reshape(-1).tolist()
    key = [v - start if 0 <= v - start < experts else experts for v in flat]
    order = sorted(range(len(flat)), key=lambda i: (key[i], i))
    slots = torch.empty(len(flat), dtype=torch.int64)
    for place, i in enumerate(order):
        slots[i] = place
    counts = [key.count(e) for e in range(experts)]
    return [0] + list(itertools.accumulate(counts)), slots.view(ids.shape)


def ragged(sizes, device="cpu"):
    return torch.tensor([0] + list(itertools.accumulate(sizes)), dtype=torch.int32, device=device)


def owners(sizes, rows):
    own = torch.full((rows,), -1)
    at = 0
    for g, n in enumerate(sizes):
        own[at: at + n] = g
        at += n
    return own


def make_ids(t, e, k, seed, dropped=0.2):
    g = torch.Generator().manual_seed(seed)
    ids = torch.rand(t, e, generator=g).argsort(1)[:, :k].to(torch.int32)
    ids[torch.rand(t, k, generator=g) < dropped] = -1
    return ids.contiguous()


# ---------------------------------------------------------------------------------------
# CPU: the plain path and the refusals
# ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("t,e,k", [(7, 8, 2), (1, 1, 1), (0, 4, 2), (5, 33, 16)])
def test_route_on_the_cpu(t, e, k, normalize):
    g = torch.Generator().manual_seed(3)
    logits = torch.randn(t, e, generator=g)
    logits[torch.rand(t, e, generator=g) < 0.3] = NINF
    if t > 2:
        logits[2] = NINF       # padding: no expert allowed
        logits[1] = logits[1, 0].clamp_min(-1.0)  # all equal
    logits.requires_grad_()
    weights, ids, plan = fn.moe_route(logits, k, normalize)
    w64, i64, p64 = route64(logits, k, normalize)
    assert torch.equal(ids.long(), i64)
    near(weights, w64, (70 + e) * F32 * w64)
    offsets, slots = plan64(ids, e)
    assert plan.offsets.tolist() == offsets and torch.equal(plan.slots.long(), slots)
    dw = torch.randn(t, k, generator=g)
    if t:
        weights.backward(dw)
        up = torch.zeros_like(p64).scatter_add_(1, i64.clamp_min(0), dw.double() * (i64 >= 0))
        want = p64 * (up - (p64 * up).sum(1, keepdim=True))
        near(logits.grad, want, (200 + 4 * e) * F32 * p64 * (up.abs() + (p64 * up.abs()).sum(1, keepdim=True)))


def test_plan_keeps_order_and_drops_foreign_experts():
    ids = torch.tensor([[2, 0], [0, 5], [-1, 2], [1, 0]], dtype=torch.int32)
    plan = fn.moe_plan(ids, 3)
    assert plan.offsets.tolist() == [0, 3, 4, 6]
    assert plan.slots.tolist() == [[4, 0], [1, 6], [7, 5], [3, 2]]
    local = fn.moe_plan(ids, 2, start=1)  # the experts 1 and 2 of this rank
    assert local.offsets.tolist() == [0, 1, 3]
    assert local.slots.tolist() == [[1, 3], [4, 5], [6, 2], [0, 7]]


def test_dispatch_combine_on_the_cpu_undo_each_other():
    ids = make_ids(9, 6, 3, 1, dropped=0.3)
    plan = fn.moe_plan(ids, 6)
    x = torch.randn(9, 5, requires_grad=True)
    rows = fn.moe_dispatch(x, plan)
    assert torch.equal(rows[plan.offsets[-1]:], torch.zeros(27 - int(plan.offsets[-1]), 5))
    out = fn.moe_combine(rows, torch.ones(9, 3), plan)
    times = (ids >= 0).sum(1, keepdim=True)
    near(out, x.double() * times, 3 * F32 * x.abs().double() * times)
    out.sum().backward()
    assert torch.equal(x.grad, times.float().expand(9, 5))


def test_grouped_products_on_the_cpu():
    sizes = [3, 0, 4]
    x = torch.randn(9, 6, requires_grad=True)
    w = torch.randn(3, 5, 6, requires_grad=True)
    y = fn.grouped_linear(x, w, ragged(sizes))
    assert torch.equal(y[7:], torch.zeros(2, 5))
    near(y[3:7], x[3:7].double() @ w[2].double().t(), 1e-5)
    dy = torch.randn(9, 5)
    y.backward(dy)
    near(w.grad, grouped_wgrad(dy, x.detach(), ragged(sizes)), 1e-5)
    near(x.grad, grouped_dgrad(dy, w.detach(), ragged(sizes)), 1e-5)
    assert torch.equal(x.grad[7:], torch.zeros(2, 6))
    acc = torch.ones(3, 5, 6)
    grouped_wgrad(dy, x.detach(), ragged(sizes), out=acc, accumulate=True)
    near(acc, w.grad.double() + 1, 1e-5)
    # offsets that decrease or pass the rows are clamped to 0, 5, 5, 9
    bad = torch.tensor([2, 5, 3, 20], dtype=torch.int32)
    near(grouped_linear(x.detach(), w.detach(), bad)[:5], x[:5].double() @ w[0].double().t(), 1e-5)


REFUSALS = {
    "logits of another type": lambda d: fn.moe_route(torch.zeros(2, 4, dtype=torch.float16, device=d), 1),
    "one-dimensional logits": lambda d: fn.moe_route(torch.zeros(4, device=d), 1),
    "more choices than experts": lambda d: fn.moe_route(torch.zeros(2, 4, device=d), 5),
    "no choice": lambda d: fn.moe_route(torch.zeros(2, 4, device=d), 0),
    "more choices than the limit": lambda d: fn.moe_route(torch.zeros(2, 64, device=d), 17),
    "too many experts": lambda d: fn.moe_route(torch.zeros(2, 1025, device=d), 2),
    "ids of another type": lambda d: fn.moe_plan(torch.zeros(2, 2, dtype=torch.int64, device=d), 4),
    "flat ids": lambda d: fn.moe_plan(torch.zeros(4, dtype=torch.int32, device=d), 4),
    "no experts": lambda d: fn.moe_plan(torch.zeros(2, 2, dtype=torch.int32, device=d), 0),
    "a start past 32 bits": lambda d: fn.moe_plan(torch.zeros(2, 2, dtype=torch.int32, device=d), 4, start=2**31),
    "rows for another plan": lambda d: fn.moe_dispatch(torch.zeros(3, 8, device=d), _plan(d)),
    "rows of another type": lambda d: fn.moe_dispatch(torch.zeros(2, 8, device=d, dtype=torch.float16), _plan(d))
    if d != "cpu" else _refuse(),
    "flat rows": lambda d: fn.moe_dispatch(torch.zeros(2, device=d), _plan(d)),
    "a plan of another type": lambda d: fn.moe_dispatch(torch.zeros(2, 8, device=d), fn.MoePlan(*(p.long() for p in _plan(d)))),
    "expert rows for another plan": lambda d: fn.moe_combine(torch.zeros(5, 8, device=d), torch.zeros(2, 2, device=d), _plan(d)),
    "weights of another shape": lambda d: fn.moe_combine(torch.zeros(4, 8, device=d), torch.zeros(2, 3, device=d), _plan(d)),
    "weights of another type": lambda d: fn.moe_combine(torch.zeros(4, 8, device=d),
                                                        torch.zeros(2, 2, device=d, dtype=torch.bfloat16), _plan(d)),
    "residual of another shape": lambda d: fn.moe_combine(torch.zeros(4, 8, device=d), torch.zeros(2, 2, device=d), _plan(d),
                                                          torch.zeros(2, 9, device=d)),
    "offsets of another length": lambda d: grouped_linear(torch.zeros(4, 8, device=d), torch.zeros(3, 8, 8, device=d), ragged([4], d)),
    "offsets of another type": lambda d: grouped_linear(torch.zeros(4, 8, device=d), torch.zeros(1, 8, 8, device=d),
                                                        torch.zeros(2, dtype=torch.int64, device=d)),
    "weights of another width": lambda d: grouped_linear(torch.zeros(4, 8, device=d), torch.zeros(1, 8, 16, device=d), ragged([4], d)),
    "two-dimensional weights": lambda d: grouped_linear(torch.zeros(4, 8, device=d), torch.zeros(8, 8, device=d), ragged([4], d)),
    "types that differ": lambda d: grouped_linear(torch.zeros(4, 8, device=d), torch.zeros(1, 8, 8, device=d).bfloat16(), ragged([4], d)),
    "an accumulator of another shape": lambda d: fn.grouped_linear(torch.zeros(4, 8, device=d), torch.zeros(1, 8, 8, device=d),
                                                                   ragged([4], d), main_grad=torch.zeros(8, 8, device=d)),
    "an accumulator of another type": lambda d: grouped_wgrad(torch.zeros(4, 8, device=d), torch.zeros(4, 8, device=d), ragged([4], d),
                                                              out=torch.zeros(1, 8, 8, device=d).bfloat16()),
    "rows that differ": lambda d: grouped_wgrad(torch.zeros(4, 8, device=d), torch.zeros(5, 8, device=d), ragged([4], d)),
}


def _plan(d):
    return fn.MoePlan(torch.tensor([0, 2, 4], dtype=torch.int32, device=d),
                      torch.tensor([[0, 2], [1, 3]], dtype=torch.int32, device=d))


def _refuse():
    raise ValueError


@pytest.mark.parametrize("what", sorted(REFUSALS))
def test_refusals(what):
    with pytest.raises(ValueError):
        REFUSALS[what]("cpu")


@gpu
@pytest.mark.parametrize("what", sorted(REFUSALS))
def test_refusals_on_the_gpu(what):
    with pytest.raises(ValueError):
        REFUSALS[what]("cuda")


@gpu
@pytest.mark.parametrize("n,k", [(12, 16), (16, 12)])
def test_kernels_refuse_widths_without_16_byte_vectors(n, k):
    x = torch.zeros(4, k, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(1, n, k, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="multiples of 8"):
        fn.grouped_linear(x, w, ragged([4], "cuda"))


# ---------------------------------------------------------------------------------------
# GPU: routing
# ---------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 8, 8), (5, 2, 1), (64, 8, 2), (333, 13, 4), (200, 16, 16), (97, 32, 3),
                                   (130, 61, 6), (301, 128, 8), (77, 256, 5), (40, 1000, 16), (0, 8, 2)])
def test_route(t, e, k, normalize, dtype):
    g = torch.Generator().manual_seed(t * 1000 + e)
    logits = (2 * torch.randn(t, e, generator=g)).to(dtype)
    logits[torch.rand(t, e, generator=g) < 0.2] = NINF
    if t > 10:
        logits[3] = NINF                              # padding
        logits[4] = torch.finfo(dtype).min            # a mask of lowest values: all equal, all allowed
        logits[5] = torch.where(torch.arange(e) % 2 == 0, 0.0, -0.0)  # zeros tie whatever their sign
        logits[6] = 1.5                               # ties: lowest experts first
        logits[7, 1:] = NINF                          # one expert left (or none)
    x = logits.cuda().requires_grad_()
    weights, ids, plan = fn.moe_route(x, k, normalize)
    w64, i64, p64 = route64(logits, k, normalize)
    assert torch.equal(ids.cpu().long(), i64)
    assert weights.dtype == torch.float32
    # exp of a difference: its rounding counts |x - max| steps (at most 40 here, or the result
    # is exactly 0 or 1), exp itself two; numerator and sum each, e additions, one division
    near(weights, w64, (90 + e) * F32 * w64 + 1e-37)
    offsets, slots = plan64(ids.cpu(), e)
    assert plan.offsets.tolist() == offsets and torch.equal(plan.slots.cpu().long(), slots)
    if t == 0:
        return
    dw = torch.randn(t, k, generator=g)
    weights.backward(dw.cuda())
    up = torch.zeros_like(p64).scatter_add_(1, i64.clamp_min(0), dw.double() * (i64 >= 0))
    want = p64 * (up - (p64 * up).sum(1, keepdim=True))
    size = p64 * (up.abs() + (p64 * up.abs()).sum(1, keepdim=True))
    near(x.grad, want, (BF * want.abs() if dtype == torch.bfloat16 else 0) + (300 + 4 * e) * F32 * size + 1e-37)


@gpu
@pytest.mark.parametrize("normalize", [True, False])
def test_route_gradient_against_differences(normalize):
    """Central differences of step h: off by h^2 / 6 of a third derivative (at most 1 per unit of
    the weights' gradient) and by the weights' rounding over h."""
    torch.manual_seed(0)
    h, x, dw = 2.0**-7, torch.randn(6, 9, device="cuda"), torch.randn(6, 3, device="cuda")
    x.requires_grad_()
    weights, ids, _ = fn.moe_route(x, 3, normalize)
    weights.backward(dw)
    gap = x.detach().sort(dim=1).values.diff(dim=1).min()
    assert gap > 0  # the choice must not change within h: only entries that keep it are compared
    checked = 0
    for r, e in itertools.product(range(6), range(9)):
        lo, hi = x.detach().clone(), x.detach().clone()
        lo[r, e] -= h
        hi[r, e] += h
        (wl, il, _), (wh, ih, _) = fn.moe_route(lo, 3, normalize), fn.moe_route(hi, 3, normalize)
        if not (torch.equal(il, ids) and torch.equal(ih, ids)):
            continue
        diff = ((wh - wl).double() * dw.double()).sum() / (2 * h)
        near(x.grad[r, e], diff, (h * h / 6 + 200 * F32 / h) * dw[r].abs().sum().item())
        checked += 1
    assert checked > 40


@gpu
def test_route_with_nan_stays_in_range():
    x = torch.randn(50, 12, device="cuda")
    x[7, 3] = float("nan")
    x[9] = float("nan")
    x[11, 5] = float("inf")
    weights, ids, plan = fn.moe_route(x, 4)
    assert ids[7, 0] == 3 and ids[9].tolist() == [0, 1, 2, 3] and ids[11, 0] == 5
    assert weights[7].isnan().all() and weights[9].isnan().all() and weights[11].isnan().all()
    clean = torch.ones(50, dtype=torch.bool)
    clean[[7, 9, 11]] = False
    assert weights.cpu()[clean].isfinite().all()
    assert int(plan.offsets[-1]) == 200 and sorted(plan.slots.reshape(-1).tolist()) == list(range(200))


@gpu
def test_route_takes_strided_logits():
    base = torch.randn(100, 40, device="cuda")
    for view in (base[:, 3:20], base[::3, :17], base.t()[:17], base[:, ::2]):
        got, want = fn.moe_route(view, 3), fn.moe_route(view.contiguous(), 3)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2].slots, want[2].slots)


@gpu
@pytest.mark.parametrize("t,e,k,start", [(1, 1, 1, 0), (700, 8, 2, 0), (4099, 61, 6, 0), (5000, 16, 4, 24), (33, 1024, 3, 0),
                                         (40000, 5, 2, 0), (0, 3, 2, 0), (9, 4, 2, -7)])
def test_plan(t, e, k, start):
    ids = (make_ids(t, max(e, k) + 8, k, 5) + start - 4).contiguous()
    plan = fn.moe_plan(ids.cuda(), e, start)
    offsets, slots = plan64(ids, e, start)
    assert plan.offsets.tolist() == offsets
    assert torch.equal(plan.slots.cpu().long(), slots)


@gpu
def test_plan_of_extreme_ids():
    ids = torch.tensor([[2**31 - 1, -(2**31)], [0, 3], [-1, 1]], dtype=torch.int32, device="cuda")
    assert fn.moe_plan(ids, 2).offsets.tolist() == [0, 1, 2]
    assert fn.moe_plan(ids, 2, start=-(2**31)).offsets.tolist() == [0, 1, 1]
    assert fn.moe_plan(ids, 2, start=2**31 - 1).offsets.tolist() == [0, 1, 1]


# ---------------------------------------------------------------------------------------
# GPU: dispatch and combine
# ---------------------------------------------------------------------------------------

MOVES = [(1, 8, 1, 8), (37, 64, 8, 5120), (333, 61, 6, 1003), (64, 4, 4, 64), (100, 8, 2, 2048), (50, 3, 1, 1), (29, 16, 16, 200),
         (130, 16, 3, 8 * 257), (0, 4, 2, 64)]


@gpu
@pytest.mark.parametrize("t,e,k,d", MOVES)
def test_dispatch(t, e, k, d):
    torch.manual_seed(t + d)
    ids = make_ids(t, max(e, k), k, t)
    plan = fn.moe_plan(ids.cuda(), e)
    x = torch.randn(t, d, device="cuda").bfloat16().requires_grad_()
    y = fn.moe_dispatch(x, plan)
    kept = (plan.slots.cpu() < int(plan.offsets[-1]))
    want = torch.zeros(t * k, d, dtype=torch.float64)
    for r, j in itertools.product(range(t), range(k)):
        if kept[r, j]:
            want[plan.slots[r, j]] = x[r].detach().double().cpu()
    assert torch.equal(y.detach().double().cpu(), want)
    if t == 0:
        return
    dy = torch.randn_like(y)
    y.backward(dy)
    rows = dy.double().cpu()[plan.slots.cpu().long()] * kept[..., None]
    total = rows.sum(1)
    near(x.grad, total, BF * total.abs() + (k + 1) * F32 * rows.abs().sum(1))
    check_device_errors()


@gpu
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("t,e,k,d", MOVES)
def test_combine(t, e, k, d, with_residual):
    torch.manual_seed(t + d + 1)
    ids = make_ids(t, max(e, k), k, t + 1)
    plan = fn.moe_plan(ids.cuda(), e)
    y = torch.randn(t * k, d, device="cuda").bfloat16()
    y[int(plan.offsets[-1]):] = float("nan")  # rows of no expert are never read
    y.requires_grad_()
    w = torch.rand(t, k, device="cuda").requires_grad_()
    r = torch.randn(t, d, device="cuda").bfloat16().requires_grad_() if with_residual else None
    out = fn.moe_combine(y, w, plan, residual=r)
    kept = (plan.slots.cpu() < int(plan.offsets[-1]))
    rows = torch.nan_to_num(y.detach().double().cpu())[plan.slots.cpu().long()] * kept[..., None]
    terms = rows * w.detach().double().cpu()[..., None]
    want, size = terms.sum(1), terms.abs().sum(1)
    if with_residual:
        want, size = want + r.detach().double().cpu(), size + r.detach().double().cpu().abs()
    near(out, want, BF * want.abs() + 2 * (2 * k + 2) * F32 * size)
    if t == 0:
        return
    dout = torch.randn_like(out)
    out.backward(dout)
    d64 = dout.double().cpu()
    dots = (rows * d64[:, None, :])
    near(w.grad, dots.sum(2), (d + 8) * F32 * dots.abs().sum(2))
    dy = torch.zeros(t * k, d, dtype=torch.float64)
    dy[plan.slots.cpu().long().reshape(-1)] = (w.detach().double().cpu()[..., None] * d64[:, None, :] * kept[..., None]).reshape(-1, d)
    near(y.grad, dy, (BF + 2 * F32) * dy.abs())
    if with_residual:
        assert torch.equal(r.grad, dout)
    check_device_errors()


@gpu
def test_rows_at_odd_addresses_and_with_strides():
    """Views that are not 16-byte aligned, strided rows and an expanded gradient."""
    torch.manual_seed(2)
    plan = fn.moe_plan(make_ids(40, 5, 2, 9).cuda(), 5)
    flat = torch.randn(40 * 64 + 3, device="cuda").bfloat16()
    x = flat[3:].view(40, 64)  # contiguous, six bytes behind an aligned address
    assert torch.equal(fn.moe_dispatch(x, plan), fn.moe_dispatch(x.clone(), plan))
    wide = torch.randn(40, 128, device="cuda").bfloat16()
    assert torch.equal(fn.moe_dispatch(wide[:, 5:69], plan), fn.moe_dispatch(wide[:, 5:69].clone(), plan))
    y = torch.randn(80, 64, device="cuda").bfloat16().requires_grad_()
    w = torch.rand(40, 2, device="cuda").requires_grad_()
    fn.moe_combine(y, w, plan).sum().backward()  # the gradient is one value with stride 0
    kept = (plan.slots < plan.offsets[-1])
    near(w.grad, (y.detach().double()[plan.slots.long()] * kept[..., None]).sum(2), 72 * F32 * 64 * 4)


@gpu
def test_places_outside_the_rows_are_skipped_and_reported():
    plan = fn.MoePlan(torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda"),
                      torch.tensor([[0, 99], [-5, 3]], dtype=torch.int32, device="cuda"))
    check_device_errors()
    y = torch.ones(4, 16, device="cuda", dtype=torch.bfloat16)
    out = fn.moe_combine(y, torch.ones(2, 2, device="cuda"), plan)
    with pytest.raises(KernelError):
        check_device_errors()
    assert torch.equal(out, torch.ones_like(out))
    fn.moe_dispatch(torch.ones(2, 16, device="cuda", dtype=torch.bfloat16), plan)
    with pytest.raises(KernelError):
        check_device_errors()
    check_device_errors()


# ---------------------------------------------------------------------------------------
# GPU: products grouped by expert
# ---------------------------------------------------------------------------------------

# group sizes, rows behind the last group, N, K
GROUPED = [
    ([1], 0, 8, 8),
    ([0], 5, 16, 24),
    ([3, 0, 4], 2, 72, 136),
    ([0, 0, 17, 0], 0, 128, 64),
    ([64, 64], 0, 256, 128),
    ([65, 63, 1, 0, 127, 129], 7, 200, 328),
    ([16, 15, 33, 48, 80, 2], 0, 136, 72),
    ([300, 1, 900, 257], 0, 520, 264),
    ([255, 256, 257, 512], 300, 264, 520),
    ([5] * 70, 0, 64, 40),
    ([2000], 0, 640, 1096),
    ([1023, 1, 2048], 129, 1032, 712),
]


def _grouped_case(sizes, tail, n, k, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = sum(sizes) + tail
    x = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
    w = torch.randn(len(sizes), n, k, generator=g, device="cuda").bfloat16()
    dy = torch.randn(rows, n, generator=g, device="cuda").bfloat16()
    return x, w, dy, ragged(sizes, "cuda")


def _check_grouped(sizes, x, w, dy, y, dx, dw, dw0=None):
    rows, k = x.shape
    n = w.shape[1]
    own = owners(sizes, rows)
    for g in range(len(sizes)):
        at = (own == g).cuda()
        xg, wg, dg = x[at].double(), w[g].double(), dy[at].double()
        # sums of K (N, group rows) products: one step of 2^-23 of the magnitudes per term
        want, size = xg @ wg.t(), xg.abs() @ wg.abs().t()
        near(y[at], want, BF * want.abs() + 1.01 * 2 * k * F32 * size, "y")
        want, size = dg @ wg, dg.abs() @ wg.abs()
        near(dx[at], want, BF * want.abs() + 1.01 * 2 * n * F32 * size, "dx")
        want, size = dg.t() @ xg, dg.abs().t() @ xg.abs()
        if dw0 is not None:
            want, size = want + dw0[g].double(), size + dw0[g].double().abs()
        near(dw[g], want, 2 * (len(xg) + 1) * F32 * size, "dw")
    rest = (own == -1).cuda()
    assert not y[rest].any() and not dx[rest].any()


@gpu
@pytest.mark.parametrize("sizes,tail,n,k", GROUPED)
def test_grouped_products(sizes, tail, n, k):
    x, w, dy, offsets = _grouped_case(sizes, tail, n, k)
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    acc = torch.randn(w.shape, device="cuda")
    start = acc.clone()
    y = fn.grouped_linear(xr, wr, offsets, main_grad=acc)
    y.backward(dy)
    assert wr.grad is None
    dw = grouped_wgrad(dy, x, offsets, out=torch.full(w.shape, float("nan"), device="cuda"))  # every element is written
    _check_grouped(sizes, x, w, dy, y, xr.grad, acc, start)
    _check_grouped(sizes, x, w, dy, y, grouped_dgrad(dy, w, offsets), dw)
    check_device_errors()


@gpu
def test_grouped_weights_get_a_gradient_without_an_accumulator():
    x, w, dy, offsets = _grouped_case([10, 0, 30], 0, 64, 48)
    w.requires_grad_()
    fn.grouped_linear(x, w, offsets).backward(dy)
    assert w.grad.dtype == torch.bfloat16
    assert torch.equal(w.grad, grouped_wgrad(dy, x, offsets).bfloat16())


@gpu
def test_grouped_neighbours_do_not_leak():
    """Infinities and NaN in one group's rows and weights stay in that group; so do those behind
    the last group's rows."""
    sizes, n, k = [37, 50, 9, 100], 72, 136
    x, w, dy, offsets = _grouped_case(sizes, 20, n, k, seed=4)
    for t in (x, dy):
        t[37:87] = float("nan")
        t[40, :] = float("inf")
        t[196:] = float("nan")
    w[1] = float("inf")
    y = grouped_linear(x, w, offsets)
    dx = grouped_dgrad(dy, w, offsets)
    dw = grouped_wgrad(dy, x, offsets)
    own = owners(sizes, 216).cuda()
    for g in (0, 2, 3):
        at = own == g
        assert y[at].isfinite().all() and dx[at].isfinite().all() and dw[g].isfinite().all(), g
        want, size = dy[at].double().t() @ x[at].double(), dy[at].double().abs().t() @ x[at].double().abs()
        near(dw[g], want, 2 * 101 * F32 * size)
    assert not y[own == -1].any() and not dx[own == -1].any()
    check_device_errors()


@gpu
def test_grouped_takes_views():
    """Rows and weights inside larger tensors, a transposed weight, odd addresses, stride-0 rows."""
    sizes, n, k = [20, 0, 45], 40, 64
    x, w, dy, offsets = _grouped_case(sizes, 3, n, k, seed=5)
    want = grouped_linear(x, w, offsets)
    big = torch.randn(68, 3 * k, device="cuda").bfloat16()
    big[:, k: 2 * k] = x
    assert torch.equal(grouped_linear(big[:, k: 2 * k], w, offsets), want)
    bigw = torch.randn(3, 2 * n, k + 8, device="cuda").bfloat16()
    bigw[:, n:, :k] = w
    assert torch.equal(grouped_linear(x, bigw[:, n:, :k], offsets), want)
    assert torch.equal(grouped_linear(x, w.transpose(1, 2).contiguous().transpose(1, 2), offsets), want)
    odd = torch.empty(68 * k + 1, device="cuda", dtype=torch.bfloat16)[1:].view(68, k).copy_(x)
    assert torch.equal(grouped_linear(odd, w, offsets), want)
    one = torch.randn(1, k, device="cuda").bfloat16().expand(68, k)
    assert torch.equal(grouped_linear(one, w, offsets), grouped_linear(one.contiguous(), w, offsets))
    single = torch.randn(1, k + 1, device="cuda").bfloat16()[:, :k]  # one row of an odd stride
    assert torch.equal(grouped_linear(single, w, ragged([0, 1, 0], "cuda")),
                       grouped_linear(single.clone(), w, ragged([0, 1, 0], "cuda")))
    dw = grouped_wgrad(dy, x, offsets)
    assert torch.equal(grouped_wgrad(dy, big[:, k: 2 * k], offsets), dw)
    check_device_errors()


@gpu
def test_grouped_without_rows():
    w = torch.randn(3, 16, 24, device="cuda").bfloat16()
    none = ragged([0, 0, 0], "cuda")
    x = torch.empty(0, 24, device="cuda", dtype=torch.bfloat16).requires_grad_()
    y = fn.grouped_linear(x, w, none)
    assert y.shape == (0, 16)
    y.backward(torch.empty_like(y))
    assert x.grad.shape == (0, 24)
    dw = grouped_wgrad(y.detach(), x.detach(), none, out=torch.ones(3, 16, 24, device="cuda"))
    assert not dw.any()
    acc = grouped_wgrad(y.detach(), x.detach(), none, out=torch.ones(3, 16, 24, device="cuda"), accumulate=True)
    assert torch.equal(acc, torch.ones_like(acc))


@gpu
@pytest.mark.parametrize("values", [[2, 5, 3, 20], [-4, 5, 5, 9], [0, 100, 200, 300], [0, 9, -2**31, 2**31 - 1]])
def test_offsets_out_of_order_are_clamped_and_reported(values):
    torch.manual_seed(1)
    x, w, dy, _ = _grouped_case([9], 0, 16, 24)
    w = torch.randn(3, 16, 24, device="cuda").bfloat16()
    offsets = torch.tensor(values, dtype=torch.int32, device="cuda")
    check_device_errors()
    y, dw = grouped_linear(x, w, offsets), grouped_wgrad(dy, x, offsets)
    with pytest.raises(KernelError):
        check_device_errors()
    clamped, last = [0], 0
    for v in values[1:]:
        last = max(last, min(max(v, 0), 9))
        clamped.append(last)
    fixed = torch.tensor(clamped, dtype=torch.int32, device="cuda")
    assert torch.equal(y, grouped_linear(x, w, fixed)) and torch.equal(dw, grouped_wgrad(dy, x, fixed))
    check_device_errors()


@gpu
def test_grouped_is_deterministic():
    x, w, dy, offsets = _grouped_case([700, 3, 1500, 0, 333], 0, 264, 520, seed=6)
    first = (grouped_linear(x, w, offsets), grouped_dgrad(dy, w, offsets), grouped_wgrad(dy, x, offsets))
    for _ in range(3):
        again = (grouped_linear(x, w, offsets), grouped_dgrad(dy, w, offsets), grouped_wgrad(dy, x, offsets))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


# ---------------------------------------------------------------------------------------
# GPU: together, on streams, in graphs, far into memory
# ---------------------------------------------------------------------------------------


def _block(seed=0, t=300, d=128, f=72, e=8, k=2):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).bfloat16()

    return normal(t, d), normal(e, d, scale=d**-0.5), normal(e, 2 * f, d, scale=d**-0.5), normal(e, d, f, scale=f**-0.5)


def _grads(*weights):
    return tuple(torch.zeros(w.shape, device="cuda") for w in weights)


@gpu
@pytest.mark.parametrize("normalize", [True, False])
def test_sparse_block_with_dropout(normalize):
    """The whole block forward and backward against the FP32 path on the CPU. Roundings on a
    path: logits, gate/up, swiglu (twice: both factors), y, combine and dropout forward, as
    many backward: 14 of 2^-8 relative to each tensor's norm."""
    x, wr, wgu, wd = _block()
    grads = _grads(wr, wgu, wd)
    xr = x.clone().requires_grad_()
    mlp = fn.moe_swiglu(xr, wr, wgu, wd, 2, normalize=normalize, grads=grads)
    out = fn.dropout(mlp, 0.2, 77, 5, residual=xr)
    dout = torch.randn_like(out)
    out.backward(dout)
    ref = [t.detach().float().cpu().requires_grad_() for t in (x, wr, wgu, wd)]
    # the choice of experts is the bf16 router's: a near tie may fall either way in FP32
    logits = fn.linear(x, wr)
    ids = fn.moe_route(logits, 2, normalize)[1].cpu()
    own = torch.nn.functional.linear(ref[0], ref[1])
    p = own.gather(1, ids.long()) if normalize else own
    weights = p.softmax(1) if normalize else p.softmax(1).gather(1, ids.long())
    plan = fn.moe_plan(ids, 8)
    gu = fn.grouped_linear(fn.moe_dispatch(ref[0], plan), ref[2], plan.offsets)
    mid = fn.moe_combine(fn.grouped_linear(fn.swiglu(gu), ref[3], plan.offsets), weights, plan)
    want = fn.dropout(mid, 0.2, 77, 5, residual=ref[0])
    want.backward(dout.float().cpu())
    for got, exact, what in ((out, want, "out"), (xr.grad, ref[0].grad, "x"), *zip(grads, (r.grad for r in ref[1:]), ("router", "gate_up", "down"))):
        err = ((got.detach().float().cpu() - exact.detach()).norm() / exact.detach().norm()).item()
        assert err <= 14 * BF, (what, err)
    check_device_errors()


@gpu
def test_block_is_its_steps():
    x, wr, wgu, wd = _block(1)
    out = fn.moe_swiglu(x, wr, wgu, wd, 3, residual=x)
    weights, _, plan = fn.moe_route(fn.linear(x, wr), 3)
    rows = fn.swiglu(fn.grouped_linear(fn.moe_dispatch(x, plan), wgu, plan.offsets))
    assert torch.equal(out, fn.moe_combine(fn.grouped_linear(rows, wd, plan.offsets), weights, plan, x))


@gpu
def test_expert_shards_add_up():
    """Two ranks with four experts each (``start``) give the whole block's sum."""
    x, wr, wgu, wd = _block(2)
    weights, ids, plan = fn.moe_route(fn.linear(x, wr), 2)
    y = fn.grouped_linear(fn.swiglu(fn.grouped_linear(fn.moe_dispatch(x, plan), wgu, plan.offsets)), wd, plan.offsets)
    rows = y.double()[plan.slots.long()] * weights.double()[..., None]
    total = torch.zeros_like(x, dtype=torch.float64)
    for rank in range(2):
        part = fn.moe_plan(ids, 4, start=4 * rank)
        lo = slice(4 * rank, 4 * rank + 4)
        z = fn.grouped_linear(fn.swiglu(fn.grouped_linear(fn.moe_dispatch(x, part), wgu[lo], part.offsets)), wd[lo], part.offsets)
        total += fn.moe_combine(z, weights, part).double()
    near(total, rows.sum(1), 2 * BF * rows.abs().sum(1))


@gpu
def test_another_stream():
    x, wr, wgu, wd = _block(3)
    want = fn.moe_swiglu(x, wr, wgu, wd, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fn.moe_swiglu(x, wr, wgu, wd, 2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@gpu
def test_captured_step_replays_on_new_rows():
    """Forward and backward of the block in a graph, replayed on other inputs with other row
    counts per expert; two graphs of the same step keep apart."""
    static, wr, wgu, wd = _block(4)
    leaf = static.clone().requires_grad_()
    acc = _grads(wr, wgu, wd)

    def step(into):
        out = fn.moe_swiglu(leaf, wr, wgu, wd, 2, residual=leaf, grads=into)
        (dx,) = torch.autograd.grad(out, leaf, out.detach())
        return out, dx

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(acc)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(acc)
        graphs.append((g, outs))
    for seed in (10, 11, 12):
        with torch.no_grad():
            leaf.copy_(_block(seed)[0])
        for a in acc:
            a.zero_()
        for g, _ in graphs:
            g.replay()
        twice = [a.clone() for a in acc]
        fresh = _grads(wr, wgu, wd)
        want = step(fresh)
        step(fresh)
        for _, outs in graphs:
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert all(torch.equal(a, b) for a, b in zip(twice, fresh))
    check_device_errors()


@gpu
def test_rows_far_into_memory():
    """More than 2^31 elements of sorted rows: places and products past 32-bit element offsets."""
    t, k, d, n = 70_000, 8, 4096, 64
    plan = fn.MoePlan(torch.tensor([0, t * k - 5, t * k - 2], dtype=torch.int32, device="cuda"),
                      torch.arange(t * k, dtype=torch.int32, device="cuda").view(t, k))
    assert t * k * d > 2**31
    x = torch.randn(t, d, device="cuda").bfloat16()
    rows = fn.moe_dispatch(x, plan)
    for r in (0, t // 2, t - 1):
        assert torch.equal(rows[r * k], x[r])
    assert torch.equal(rows[-3], x[-1]) and not rows[-2:].any()
    w = torch.randn(2, n, d, device="cuda").bfloat16()
    y = grouped_linear(rows, w, plan.offsets)
    for g, at in ((0, slice(0, 40)), (0, slice(t * k - 45, t * k - 5)), (1, slice(t * k - 5, t * k - 2))):
        want, size = rows[at].double() @ w[g].double().t(), rows[at].double().abs() @ w[g].double().abs().t()
        near(y[at], want, BF * want.abs() + 1.01 * 2 * d * F32 * size)
    assert not y[-2:].any()
    back = grouped_dgrad(y, w, plan.offsets)
    want, size = y[-45:-5].double() @ w[0].double(), y[-45:-5].double().abs() @ w[0].double().abs()
    near(back[-45:-5], want, BF * want.abs() + 1.01 * 2 * n * F32 * size)
    out = fn.moe_combine(rows, torch.full((t, k), 0.125, device="cuda"), plan)
    want = x[-1].double() * 0.125 * 6  # the last token's last two choices have no expert
    near(out[-1], want, BF * want.abs() + 20 * F32 * want.abs())
    check_device_errors()


# ---------------------------------------------------------------------------------------
# GPU: calls that the documentation allows and nothing above makes
# ---------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("t,k,d", [(5000, 40, 256), (5000, 31, 264), (5000, 32, 256), (9, 40, 512)])
def test_more_choices_than_a_warp_has_lanes(t, k, d):
    """A plan of ids chosen elsewhere has no limit on k, and may name an expert twice."""
    torch.manual_seed(k)
    ids = torch.randint(-1, 6, (t, k), dtype=torch.int32, device="cuda")
    plan = fn.moe_plan(ids, 6)
    y = torch.randn(t * k, d, device="cuda").bfloat16().requires_grad_()
    w = torch.rand(t, k, device="cuda").requires_grad_()
    out = fn.moe_combine(y, w, plan)
    kept = (ids >= 0)
    for a in range(0, t, 1000):  # in parts: the rows in 64 bits are large
        rows = y.detach()[plan.slots[a: a + 1000].long()].double() * kept[a: a + 1000, :, None]
        terms = rows * w.detach()[a: a + 1000, :, None].double()
        want = terms.sum(1)
        near(out[a: a + 1000], want, BF * want.abs() + 2 * (2 * k + 2) * F32 * terms.abs().sum(1))
    (dw,) = torch.autograd.grad(out, w, torch.ones_like(out))
    near(dw[-50:], (y.detach()[plan.slots[-50:].long()].double() * kept[-50:, :, None]).sum(2), (d + 8) * F32 * 6 * d)
    check_device_errors()


@gpu
def test_long_weight_gradients_do_not_drift():
    """One group of 30000 rows: the tensor cores' truncating additions alone would be 3e-5 off in
    the 2-norm. Partial sums of 512 rows, each of 32 truncated additions of 16 products, bound
    the drift by 32 steps of 2^-23 of a partial sum; their fp32 sum rounds 59 times."""
    torch.manual_seed(0)
    x = torch.randn(30000, 256, device="cuda").bfloat16()
    dy = torch.randn(30000, 264, device="cuda").bfloat16()
    dw = grouped_wgrad(dy, x, ragged([30000], "cuda"))[0].double()
    want = dy.double().t() @ x.double()
    assert ((dw - want).norm() / want.norm()).item() < (32 * 2 + 59) * F32


@gpu
def test_gradients_have_no_second_derivative():
    x = torch.randn(6, 16, device="cuda").bfloat16().requires_grad_()
    logits = torch.randn(6, 4, device="cuda").requires_grad_()
    weights, _, plan = fn.moe_route(logits, 2)
    w = torch.randn(4, 8, 16, device="cuda").bfloat16().requires_grad_()
    out = fn.moe_combine(fn.grouped_linear(fn.moe_dispatch(x, plan), w, plan.offsets), weights, plan)
    (dx,) = torch.autograd.grad(out.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        dx.float().sum().backward()


@gpu
def test_launch_counter_counts_backward_kernels():
    from resihp.ops import _ext

    counter = _ext.launch_counter()
    before = (counter.launches, counter.enabled)
    counter.launches, counter.enabled = 0, True
    try:
        x = torch.randn(40, 64, device="cuda").bfloat16().requires_grad_()
        plan = fn.moe_plan(make_ids(40, 4, 2, 1).cuda(), 4)          # 2 kernels
        y = fn.dropout(fn.moe_dispatch(x, plan), 0.1, 1)             # 2
        torch.autograd.grad(y, x, torch.ones_like(y))                # 2
        assert counter.launches == 6
        counter.enabled = False
        fn.moe_dispatch(x, plan)
        assert counter.launches == 6
    finally:
        counter.launches, counter.enabled = before


@gpu
def test_fp32_rows_take_the_torch_path_on_the_gpu():
    """Places out of range are left out there too, without a device-side index error."""
    plan = fn.MoePlan(torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda"),
                      torch.tensor([[0, 99], [-5, 3]], dtype=torch.int32, device="cuda"))
    x = torch.randn(2, 7, device="cuda")
    rows = fn.moe_dispatch(x, plan)
    assert torch.equal(rows[0], x[0]) and torch.equal(rows[3], x[1]) and not rows[1:3].any()
    out = fn.moe_combine(torch.ones(4, 7, device="cuda"), torch.ones(2, 2, device="cuda"), plan)
    assert torch.equal(out, torch.ones(2, 7, device="cuda"))  # each token's other choice has no place
    w = torch.randn(2, 5, 7, device="cuda")
    near(grouped_linear(rows, w, plan.offsets)[0], x[0].double() @ w[0].double().t(), 1e-5)
    torch.cuda.synchronize()


@gpu
def test_no_tokens_at_all():
    x, wr, wgu, wd = _block(5)
    grads = _grads(wr, wgu, wd)
    none = x[:0].clone().requires_grad_()
    out = fn.moe_swiglu(none, wr, wgu, wd, 2, residual=none, grads=grads)
    assert out.shape == (0, 128)
    out.sum().backward()
    assert none.grad.shape == (0, 128) and not any(g.any() for g in grads)


@gpu
def test_padding_takes_no_rows():
    """Tokens whose logits are all -inf get no expert's row, weight or gradient, only the residual."""
    x, wr, wgu, wd = _block(6)
    pad = torch.zeros(300, dtype=torch.bool, device="cuda")
    pad[250:] = True
    x = x.clone()
    x[pad] = float("nan")  # what lies in padded rows does not matter
    logits = torch.where(pad[:, None], torch.full((), NINF, device="cuda"), fn.linear(torch.nan_to_num(x), wr).float())
    weights, ids, plan = fn.moe_route(logits, 2)
    assert int(plan.offsets[-1]) == 500 and (ids[pad] == -1).all() and not weights[pad].any()
    rows = fn.moe_dispatch(x, plan)
    y = fn.grouped_linear(fn.swiglu(fn.grouped_linear(rows, wgu, plan.offsets)), wd, plan.offsets)
    out = fn.moe_combine(y, weights, plan)
    assert out.isfinite().all() and not out[pad].any()
    dw = grouped_wgrad(y, rows, plan.offsets)
    assert dw.isfinite().all()


@gpu
def test_captured_large_products_replay():
    """Products of many tiles per CTA pair in a graph, replayed with other offsets."""
    x, w, dy, _ = _grouped_case([1500, 2596], 0, 2056, 520, seed=8)
    offsets = ragged([1500, 2596], "cuda")
    acc = torch.zeros(w.shape, device="cuda")

    def step():
        return grouped_linear(x, w, offsets), grouped_dgrad(dy, w, offsets), grouped_wgrad(dy, x, offsets, out=acc, accumulate=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for sizes in ([4096, 0], [1, 4095], [777, 3000]):
        offsets.copy_(ragged(sizes, "cuda"))
        acc.zero_()
        graph.replay()
        got = [t.clone() for t in outs]
        assert torch.equal(got[0], grouped_linear(x, w, offsets)) and torch.equal(got[1], grouped_dgrad(dy, w, offsets))
        assert torch.equal(got[2], grouped_wgrad(dy, x, offsets))
    check_device_errors()


@gpu
def test_two_streams_at_once():
    """The same operators on two streams at the same time, on their own rows."""
    cases = [_block(s, t=700) for s in (20, 21)]
    want = [fn.moe_swiglu(x, wr, wgu, wd, 2) for x, wr, wgu, wd in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, (x, wr, wgu, wd) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(fn.moe_swiglu(x, wr, wgu, wd, 2))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


@gpu
def test_paced_products_in_graphs_and_on_two_streams():
    """Products deep and large enough that their CTA pairs keep step: alone, two at once (not all
    pairs resident) and replayed from a graph they give the same rows."""
    rows, n, k = 4200, 2568, 7176
    x, w, dy, offsets = _grouped_case([3000, 1100], 100, n, k, seed=9)
    y = grouped_linear(x, w, offsets)
    for g, at in ((0, slice(0, 300)), (0, slice(2900, 3000)), (1, slice(3000, 3100)), (1, slice(4000, 4100))):
        want, size = x[at].double() @ w[g].double().t(), x[at].double().abs() @ w[g].double().abs().t()
        near(y[at], want, BF * want.abs() + 1.01 * 2 * k * F32 * size)
    assert not y[4100:].any()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(grouped_linear(x, w, offsets))
    torch.cuda.synchronize()
    assert all(torch.equal(o, y) for o in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = grouped_linear(x, w, offsets)
    for sizes in ([3000, 1100], [17, 4183], [0, 4200]):
        offsets.copy_(ragged(sizes, "cuda"))
        graph.replay()
        assert torch.equal(out, grouped_linear(x, w, offsets))
    check_device_errors()


@gpu
def test_grouped_gradient_of_a_sum():
    """The gradient arrives as one value with stride 0, and goes to a view of a larger leaf."""
    big = torch.randn(60, 2, 64, device="cuda").bfloat16().requires_grad_()
    w = torch.randn(2, 40, 64, device="cuda").bfloat16()
    offsets = ragged([25, 35], "cuda")
    fn.grouped_linear(big[:, 1], w, offsets).sum().backward()
    own = owners([25, 35], 60).cuda()
    want = w.double().sum(1)[own]
    near(big.grad[:, 1], want, BF * want.abs() + 2 * 40 * F32 * w.double().abs().sum(1)[own])
    assert not big.grad[:, 0].any()


@gpu
def test_recomputed_block_gives_the_same_gradients():
    from torch.utils.checkpoint import checkpoint

    x, wr, wgu, wd = _block(7)
    results = []
    for recompute in (False, True):
        grads, leaf = _grads(wr, wgu, wd), x.clone().requires_grad_()
        wr.requires_grad_(), wgu.requires_grad_(), wd.requires_grad_()

        def layer(t):
            return fn.dropout(fn.moe_swiglu(t, wr, wgu, wd, 2, grads=grads), 0.1, 3, 4, residual=t)

        out = checkpoint(layer, leaf, use_reentrant=False) if recompute else layer(leaf)
        out.backward(torch.ones_like(out))
        results.append((out.detach(), leaf.grad, *grads))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@gpu
@pytest.mark.parametrize("op", ["dropout", "route", "dispatch", "combine", "residual", "grouped", "behind"])
def test_capture_beside_an_eager_graph_is_refused(op):
    """While a graph of the same leaf, recorded on the default stream, is alive, a captured backward
    pass raises; without it the pass is captured and replays."""
    x = torch.randn(64, 64, device="cuda").bfloat16().requires_grad_()
    w = torch.randn(2, 16, 64, device="cuda").bfloat16()
    _, ids, plan = fn.moe_route(torch.randn(64, 2, device="cuda"), 1)
    weights = torch.rand(64, 1, device="cuda")
    rows = torch.randn(64, 64, device="cuda").bfloat16()
    call = {
        "dropout": lambda: fn.dropout(x, 0.25, 3),
        "route": lambda: fn.moe_route(x, 2)[0],
        "dispatch": lambda: fn.moe_dispatch(x, plan),
        "combine": lambda: fn.moe_combine(x, weights, plan),
        "residual": lambda: fn.moe_combine(rows, weights, plan, residual=x),
        "grouped": lambda: fn.grouped_linear(x, w, plan.offsets),
        "behind": lambda: fn.dropout(x.view(32, 128) * 2, 0.25, 3),
    }[op]

    def step():
        out = call()
        return torch.autograd.grad(out, x, out.detach())[0]

    want = step()
    alive = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
        with pytest.raises(RuntimeError, match="default stream"):
            torch.autograd.grad(out, x, out.detach())
    del alive, out, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert torch.equal(got, want)
    check_device_errors()


@gpu
def test_capture_past_a_leaf_of_an_eager_graph():
    """Weights in a living eager graph: a captured pass that asks for the rows' gradient alone does
    not reach them and is captured, main gradient included; one that reaches them raises."""
    x = torch.randn(64, 64, device="cuda").bfloat16()
    w = torch.randn(2, 16, 64, device="cuda").bfloat16().requires_grad_()
    offsets = ragged([40, 24], "cuda")
    acc = torch.zeros(2, 16, 64, device="cuda")
    alive = fn.grouped_linear(x, w, offsets, main_grad=acc)
    alive.backward(alive.detach(), retain_graph=True)
    want = acc.clone()
    leaf = x.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn.grouped_linear(leaf, w, offsets, main_grad=acc)
        (dx,) = torch.autograd.grad(out, leaf, out.detach(), retain_graph=True)
        with pytest.raises(RuntimeError, match="default stream"):
            out.backward(out.detach())
    acc.zero_()
    graph.replay()
    assert torch.equal(acc, want) and torch.equal(dx, grouped_dgrad(alive.detach(), w, offsets))
    assert w.grad is None and leaf.grad is None
    check_device_errors()


@gpu
@pytest.mark.parametrize("sizes, n, k", [([3, 0, 70], 40, 72), ([600, 1, 1500], 264, 328), ([0, 0], 16, 8),
                                         ([130] * 9, 512, 1096), ([], 8, 8)])
def test_grouped_weight_gradient_in_the_weights_type(sizes, n, k):
    """Without a main gradient the weights' bf16 gradient is the fp32 sum rounded once, everywhere
    (groups without rows get zeros)."""
    x, w, dy, _ = _grouped_case(sizes or [0], 3, n, k, seed=5)
    offsets = ragged(sizes or [0], "cuda")
    w.requires_grad_()
    fn.grouped_linear(x, w, offsets).backward(dy)
    assert w.grad.dtype == torch.bfloat16
    assert torch.equal(w.grad, grouped_wgrad(dy, x, offsets).bfloat16())
    check_device_errors()


@gpu
@pytest.mark.parametrize("buffers", [(), (0,), (1, 2)])
def test_block_trains_every_weight(buffers):
    """A weight without a main gradient gets its own, the same fp32 sum rounded once; one with a
    main gradient does not."""
    x, wr, wgu, wd = _block(12)
    weights = (wr, wgu, wd)
    dout = torch.randn(300, 128, device="cuda").bfloat16()
    acc = _grads(*weights)
    fn.moe_swiglu(x.clone().requires_grad_(), *weights, 2, grads=acc).backward(dout)
    leaves = [w.clone().requires_grad_() for w in weights]
    into = _grads(*weights)
    grads = tuple(into[i] if i in buffers else None for i in range(3)) if buffers else None
    fn.moe_swiglu(x, *leaves, 2, grads=grads).backward(dout)
    for i, leaf in enumerate(leaves):
        if i in buffers:
            assert leaf.grad is None and torch.equal(into[i], acc[i]), i
        else:
            assert leaf.grad.dtype == torch.bfloat16 and torch.equal(leaf.grad, acc[i].bfloat16()), i
            assert not into[i].any()
    check_device_errors()


@gpu
def test_linear_weight_gets_a_gradient_without_an_accumulator():
    x = torch.randn(70, 64, device="cuda").bfloat16()
    w = torch.randn(40, 64, device="cuda").bfloat16().requires_grad_()
    dy = torch.randn(70, 40, device="cuda").bfloat16()
    fn.linear(x, w).backward(dy)
    want, size = dy.double().t() @ x.double(), dy.double().abs().t() @ x.double().abs()
    assert w.grad.dtype == torch.bfloat16
    near(w.grad, want, BF * want.abs() + 1.01 * 2 * 70 * F32 * size)


_MISFITS = r"""
import torch
from resihp.ops import _ext
from resihp.ops import functional as fn

def bf(*shape):
    return torch.zeros(*shape, device="cuda", dtype=torch.bfloat16)

ids = torch.zeros(1, 2, dtype=torch.int32, device="cuda").expand(2**30, 2)
out, k = bf(4, 8), _ext.require()
calls = (lambda: k.moe_route(torch.zeros(1, 2, device="cuda").expand(2**30, 2), 2, True),
         lambda: k.moe_scatter(bf(4, 8), ids[0], ids[:4, ::2]),
         lambda: k.gemm(bf(4, 16), False, bf(8, 24), False, out, 0),
         lambda: k.gemm(bf(4, 16), False, bf(8, 16), False, out, 9),
         lambda: k.swiglu_bwd(bf(4, 16), bf(4, 16)))
for call in calls:
    try:
        call()
    except RuntimeError as error:
        print("raised", error)
torch.cuda.synchronize()
"""


@gpu
def test_refusals_of_the_extension_raise():
    """A refusal whose message holds numbers is an exception, not the end of the process."""
    import os
    import subprocess
    import sys

    done = subprocess.run([sys.executable, "-c", _MISFITS], capture_output=True, text=True, timeout=600,
                          cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert done.returncode == 0 and done.stdout.count("raised") == 5, (done.stdout, done.stderr[-2000:])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_block_without_tokens_stays_in_the_graph(device, with_residual):
    """A rank that got no tokens: the output is a new tensor, and every leaf gets zeros."""
    dtype = torch.bfloat16 if device == "cuda" else torch.float32
    leaves = [torch.randn(s, device=device).to(dtype).requires_grad_() for s in ((0, 16), (8, 16), (8, 48, 16), (8, 16, 24))]
    residual = torch.zeros(0, 16, device=device, dtype=dtype).requires_grad_() if with_residual else None
    out = fn.moe_swiglu(*leaves, 2, residual=residual)
    assert out.shape == (0, 16) and out is not residual and not out.is_leaf
    out.sum().backward()
    for leaf in leaves + ([residual] if with_residual else []):
        assert leaf.grad.shape == leaf.shape and not leaf.grad.any()


@gpu
def test_linear_products_without_rows():
    x, w = torch.empty(0, 16, device="cuda").bfloat16(), torch.randn(24, 16, device="cuda").bfloat16()
    dy = torch.empty(0, 24, device="cuda").bfloat16()
    assert fn.linear(x, w).shape == fn.linear(x, w, residual=dy).shape == (0, 24)
    assert fn.linear_dgrad(dy, w).shape == (0, 16)
    assert torch.equal(fn.linear_wgrad(dy, x), torch.zeros(24, 16, device="cuda"))
    kept = torch.ones(24, 16, device="cuda")
    assert fn.linear_wgrad(dy, x, out=kept, accumulate=True).all() and not fn.linear_wgrad(dy, x, out=kept).any()


def _fp32_block(d, x=(4, 16), router=(8, 16), gate_up=(8, 48, 16), down=(8, 16, 24), dtype=torch.float32):
    return [torch.zeros(s, device=d, dtype=dtype) for s in (x, router, gate_up, down)]


BLOCK_REFUSALS = {
    "flat rows": lambda d: fn.moe_swiglu(*_fp32_block(d, x=(16,)), 2),
    "rows of a batch": lambda d: fn.moe_swiglu(*_fp32_block(d, x=(2, 4, 16)), 2),
    "rows of another width": lambda d: fn.moe_swiglu(*_fp32_block(d, x=(4, 24)), 2),
    "a router of another width": lambda d: fn.moe_swiglu(*_fp32_block(d, router=(8, 24)), 2),
    "gate and up of another count": lambda d: fn.moe_swiglu(*_fp32_block(d, gate_up=(7, 48, 16)), 2),
    "gate and up of an odd height": lambda d: fn.moe_swiglu(*_fp32_block(d, gate_up=(8, 49, 16)), 2),
    "down of another width": lambda d: fn.moe_swiglu(*_fp32_block(d, down=(8, 16, 16)), 2),
    "down of another height": lambda d: fn.moe_swiglu(*_fp32_block(d, down=(8, 24, 24)), 2),
    "two-dimensional weights": lambda d: fn.moe_swiglu(*_fp32_block(d, down=(16, 24)), 2),
    "half precision": lambda d: fn.moe_swiglu(*_fp32_block(d, dtype=torch.float16), 2),
    "types that differ": lambda d: fn.moe_swiglu(torch.zeros(4, 16, device=d).bfloat16(), *_fp32_block(d)[1:], 2),
    "more choices than experts": lambda d: fn.moe_swiglu(*_fp32_block(d), 9),
    "no choice": lambda d: fn.moe_swiglu(*_fp32_block(d), 0),
    "a residual of another shape": lambda d: fn.moe_swiglu(*_fp32_block(d), 2, residual=torch.zeros(1, 16, device=d)),
    "a residual of another type": lambda d: fn.moe_swiglu(*_fp32_block(d), 2, residual=torch.zeros(4, 16, device=d).bfloat16()),
    "two accumulators": lambda d: fn.moe_swiglu(*_fp32_block(d), 2, grads=_fp32_block(d)[1:3]),
    "a router's accumulator of another shape": lambda d: fn.moe_swiglu(
        *_fp32_block(d), 2, grads=(torch.zeros(16, 8, device=d), None, None)),
    "an accumulator of another type": lambda d: fn.moe_swiglu(
        *_fp32_block(d), 2, grads=(None, None, torch.zeros(8, 16, 24, device=d).bfloat16())),
    "an accumulator with gaps": lambda d: fn.moe_swiglu(
        *_fp32_block(d), 2, grads=(None, torch.zeros(8, 48, 32, device=d)[..., :16], None)),
}
KERNEL_BLOCK_REFUSALS = {
    "12 experts": dict(router=(12, 16), gate_up=(12, 48, 16), down=(12, 16, 24)),
    "rows of width 20": dict(x=(4, 20), router=(8, 20), gate_up=(8, 48, 20), down=(8, 20, 24)),
    "an inner width of 20": dict(gate_up=(8, 40, 16), down=(8, 16, 20)),
}


@pytest.mark.parametrize("what", sorted(BLOCK_REFUSALS))
def test_block_refusals(what):
    with pytest.raises(ValueError):
        BLOCK_REFUSALS[what]("cpu")


@gpu
@pytest.mark.parametrize("what", sorted(BLOCK_REFUSALS))
def test_block_refusals_on_the_gpu(what):
    with pytest.raises(ValueError):
        BLOCK_REFUSALS[what]("cuda")


@gpu
@pytest.mark.parametrize("what", sorted(KERNEL_BLOCK_REFUSALS))
def test_block_refusals_of_the_kernels(what):
    """Before anything is launched; fp32 takes the same sizes."""
    from resihp.ops import _ext

    counter = _ext.launch_counter()
    before, (counter.launches, counter.enabled) = (counter.launches, counter.enabled), (0, True)
    try:
        with pytest.raises(ValueError, match="multiples of 8"):
            fn.moe_swiglu(*_fp32_block("cuda", dtype=torch.bfloat16, **KERNEL_BLOCK_REFUSALS[what]), 2)
        assert counter.launches == 0
    finally:
        counter.launches, counter.enabled = before
    assert fn.moe_swiglu(*_fp32_block("cuda", **KERNEL_BLOCK_REFUSALS[what]), 2).shape[0] == 4


@gpu
def test_block_refuses_a_router_accumulator_off_16_bytes():
    x, wr, wgu, wd = _block(13)
    odd = torch.zeros(8 * 128 + 1, device="cuda")[1:].view(8, 128)
    with pytest.raises(ValueError, match="aligned"):
        fn.moe_swiglu(x, wr, wgu, wd, 2, grads=(odd, None, None))


@gpu
def test_block_takes_views():
    """Rows and router weights at odd addresses, strided and transposed, as the other steps take them."""
    x, wr, wgu, wd = _block(14)
    want = fn.moe_swiglu(x, wr, wgu, wd, 2)
    odd = torch.empty(x.numel() + 3, device="cuda", dtype=torch.bfloat16)[3:].view(300, 128).copy_(x)
    wide = torch.zeros(300, 133, device="cuda", dtype=torch.bfloat16)
    wide[:, 5:] = x
    views = (odd, wide[:, 5:], x.t().contiguous().t())
    router = wr.t().contiguous().t()
    for view in views:
        assert torch.equal(fn.moe_swiglu(view, router, wgu, wd, 2), want)
    leaf, wleaf = x.t().contiguous().requires_grad_(), wr.t().contiguous().requires_grad_()
    fn.moe_swiglu(leaf.t(), wleaf.t(), wgu, wd, 2).backward(want)
    xr, wrr = x.clone().requires_grad_(), wr.clone().requires_grad_()
    fn.moe_swiglu(xr, wrr, wgu, wd, 2).backward(want)
    assert torch.equal(leaf.grad.t(), xr.grad) and torch.equal(wleaf.grad.t(), wrr.grad)
    check_device_errors()


@gpu
def test_weight_gradients_off_16_bytes_are_refused():
    """Before the forward pass, not in the backward pass; fp32 rows take such an accumulator."""
    x, w, dy, offsets = _grouped_case([3, 6], 0, 16, 24)
    odd = torch.zeros(w.numel() + 1, device="cuda")[1:].view(w.shape)
    with pytest.raises(ValueError, match="aligned"):
        fn.grouped_linear(x.requires_grad_(), w, offsets, main_grad=odd)
    with pytest.raises(ValueError, match="aligned"):
        grouped_wgrad(dy, x.detach(), offsets, out=odd, accumulate=True)
    assert not odd.any()
    grouped_wgrad(dy.float(), x.detach().float(), offsets, out=odd)
    near(odd, grouped_wgrad(dy, x.detach(), offsets), 1e-4)
    check_device_errors()


def _many(d, *shape, dtype=torch.float32):
    """2^30 rows or more that are one row."""
    return torch.zeros(1, *shape[1:], device=d, dtype=dtype).expand(*shape)


SIZE_REFUSALS = {
    "logits": lambda d: fn.moe_route(_many(d, 2**30, 2), 2),
    "ids": lambda d: fn.moe_plan(_many(d, 2**30, 2, dtype=torch.int32), 4),
    "a plan of rows": lambda d: fn.moe_dispatch(_many(d, 2**30, 8), fn.MoePlan(ragged([4], d), _many(d, 2**30, 2, dtype=torch.int32))),
    "a plan of expert rows": lambda d: fn.moe_combine(
        _many(d, 2**31, 8), _many(d, 2**30, 2), fn.MoePlan(ragged([4], d), _many(d, 2**30, 2, dtype=torch.int32))),
    "a block": lambda d: fn.moe_swiglu(_many(d, 2**30, 16), *_fp32_block(d)[1:], 2),
}


@pytest.mark.parametrize("what", sorted(SIZE_REFUSALS))
def test_refusals_of_more_pairs_than_31_bits_count(what):
    with pytest.raises(ValueError, match="pairs"):
        SIZE_REFUSALS[what]("cpu")


@gpu
@pytest.mark.parametrize("what", sorted(SIZE_REFUSALS))
def test_refusals_of_more_pairs_than_31_bits_count_on_the_gpu(what):
    with pytest.raises(ValueError, match="pairs"):
        SIZE_REFUSALS[what]("cuda")


@gpu
def test_refusals_of_more_rows_than_31_bits_count():
    x, w = _many("cuda", 2**31, 8, dtype=torch.bfloat16), torch.zeros(1, 8, 8, device="cuda").bfloat16()
    for call in (lambda: fn.grouped_linear(x, w, ragged([4], "cuda")), lambda: grouped_dgrad(x, w, ragged([4], "cuda")),
                 lambda: grouped_wgrad(x, x, ragged([4], "cuda"))):
        with pytest.raises(ValueError, match="rows and columns"):
            call()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals_of_counts_that_are_not_whole(device):
    logits, ids = torch.zeros(4, 8, device=device), torch.zeros(4, 2, dtype=torch.int32, device=device)
    for call in (lambda: fn.moe_route(logits, 2.0), lambda: fn.moe_route(logits, "2"), lambda: fn.moe_plan(ids, 4.0),
                 lambda: fn.moe_plan(ids, 4, start=0.5), lambda: fn.moe_swiglu(*_fp32_block(device), 2.0)):
        with pytest.raises(ValueError, match="whole number"):
            call()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_route_takes_one_expert_with_strides(dtype):
    row = torch.randn(1, 37, device="cuda").to(dtype)
    row[0, 3] = NINF
    leaf = row.clone().requires_grad_()
    weights, ids, plan = fn.moe_route(leaf.t(), 1)
    want = fn.moe_route(row.t().clone(memory_format=torch.contiguous_format).reshape(-1, 1), 1)
    assert torch.equal(weights, want[0]) and torch.equal(ids, want[1]) and torch.equal(plan.slots, want[2].slots)
    assert ids[3] == -1 and weights.sum() == 36 and plan.offsets.tolist() == [0, 36]
    weights.backward(torch.randn_like(weights))
    assert not leaf.grad.any()  # the only expert's weight is 1 whatever its logit


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_what_lies_at_choices_without_an_expert_counts_for_nothing(device):
    """Infinite or NaN weights, and gradients of them, at choices that no expert takes."""
    dtype = torch.bfloat16 if device == "cuda" else torch.float32
    plan = fn.moe_plan(torch.tensor([[0, -1], [7, 1]], dtype=torch.int32, device=device), 2)
    y = torch.ones(4, 8, device=device, dtype=dtype).requires_grad_()
    w = torch.tensor([[0.5, float("nan")], [float("inf"), 2.0]], device=device).requires_grad_()
    out = fn.moe_combine(y, w, plan)
    assert out[:, 0].tolist() == [0.5, 2.0]
    out.sum().backward()
    assert w.grad.tolist() == [[8.0, 0.0], [0.0, 8.0]] and y.grad[:, 0].tolist() == [0.5, 2.0, 0.0, 0.0]
    for normalize in (True, False):
        logits = torch.tensor([[1.0, NINF, NINF], [NINF] * 3], device=device, requires_grad=True)
        weights, ids, _ = fn.moe_route(logits, 2, normalize)
        assert ids.tolist() == [[0, -1], [-1, -1]] and weights.tolist() == [[1.0, 0.0], [0.0, 0.0]]
        weights.backward(torch.tensor([[1.0, float("nan")], [float("inf"), float("nan")]], device=device))
        assert not logits.grad.any()


@gpu
@pytest.mark.parametrize("spoil", ["outside", "twice", "whole"])
@pytest.mark.parametrize("t,k,d", [(1, 1, 8), (2, 2, 512), (37, 5, 1003), (500, 3, 72), (4001, 5, 128), (9000, 2, 1024),
                                   (4100, 4, 1027), (2500, 2, 2048)])
def test_rows_that_no_pair_names_are_zeros(t, k, d, spoil):
    """A plan made elsewhere that leaves rows out: what lay in memory is in no output."""
    g = torch.Generator().manual_seed(t + d)
    n = t * k
    places = torch.randperm(n, generator=g).to(torch.int32)
    if spoil != "whole":
        hit = torch.randperm(n, generator=g)[: max(1, n // 50)]
        places[hit] = torch.tensor([-1, n, 2**31 - 1, -(2**31)], dtype=torch.int32)[torch.arange(len(hit)) % 4] if spoil == "outside" \
            else places[torch.randperm(n, generator=g)[: len(hit)]]
    slots = torch.empty(n + 1, dtype=torch.int32, device="cuda")[1:].view(t, k)  # four bytes behind an aligned address
    slots.copy_(places.view(t, k))
    used = n - n // 10
    plan = fn.MoePlan(torch.tensor([0, n // 2, used], dtype=torch.int32, device="cuda"), slots)
    at, token = places.long().cuda(), torch.arange(n, device="cuda") // k
    inside = (at >= 0) & (at < n)
    times = torch.zeros(n, device="cuda").index_add_(0, at[inside], torch.ones(int(inside.sum()), device="cuda"))
    once = torch.zeros(n, dtype=torch.bool, device="cuda")
    once[at[inside]] = True
    once &= (times == 1) & (torch.arange(n, device="cuda") < used)
    owner = torch.zeros(n, dtype=torch.int64, device="cuda")
    owner[at[inside]] = token[inside]
    check_device_errors()

    def poison():
        torch.full((n, d), float("nan"), device="cuda", dtype=torch.bfloat16)  # and freed: the next output's memory

    x = torch.randn(t, d, device="cuda").bfloat16()
    poison()
    rows = fn.moe_dispatch(x, plan)
    assert torch.equal(rows[once], x[owner[once]]) and not rows[times == 0].any() and not rows[used:].any()
    assert rows.isfinite().all()
    y = torch.randn(n, d, device="cuda").bfloat16().requires_grad_()
    out = fn.moe_combine(y, torch.ones(t, k, device="cuda"), plan)
    poison()
    out.backward(x)
    assert torch.equal(y.grad[once], x[owner[once]]) and not y.grad[times == 0].any() and not y.grad[used:].any()
    assert y.grad.isfinite().all()
    if spoil == "outside":
        with pytest.raises(KernelError):
            check_device_errors()
    check_device_errors()


def _check_moves(t, k, d, with_residual, seed):
    """Dispatch and combine with their gradients, all rows, against 64-bit sums (on the GPU, by rows)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = make_ids(t, max(k, 6), k, seed).cuda()
    plan = fn.moe_plan(ids, max(k, 6))
    at, kept = plan.slots.long(), (ids >= 0)[..., None]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").bfloat16()

    x, dy = normal(t, d).requires_grad_(), normal(t * k, d)
    rows = fn.moe_dispatch(x, plan)
    assert torch.equal(rows.detach()[at.reshape(-1)].view(t, k, d), torch.where(kept, x.detach()[:, None], torch.zeros_like(x[:, None])))
    rows.backward(dy)
    total, size = torch.zeros(2, t, d, device="cuda", dtype=torch.float64)
    for j in range(k):
        part = dy[at[:, j]].double() * kept[:, j]
        total += part
        size += part.abs()
    near(x.grad, total, BF * total.abs() + (k + 1) * F32 * size)
    y, w, dout = normal(t * k, d).requires_grad_(), torch.rand(t, k, generator=g, device="cuda").requires_grad_(), normal(t, d)
    r = normal(t, d).requires_grad_() if with_residual else None
    out = fn.moe_combine(y, w, plan, residual=r)
    out.backward(dout)
    want = r.detach().double() if with_residual else torch.zeros(t, d, device="cuda", dtype=torch.float64)
    size = want.abs()
    for j in range(k):
        row, weight = y.detach()[at[:, j]].double() * kept[:, j], w.detach()[:, j, None].double()
        want, size = want + weight * row, size + (weight * row).abs()
        dots = row * dout.double()
        near(w.grad[:, j], dots.sum(1), (d + 8) * F32 * dots.abs().sum(1))
        back = weight * dout.double() * kept[:, j]
        near(y.grad[at[:, j]], back, (BF + 2 * F32) * back.abs())
    near(out, want, BF * want.abs() + 2 * (2 * k + 2) * F32 * size)
    if with_residual:
        assert torch.equal(r.grad, dout)
    check_device_errors()


@gpu
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("t,k,d", [(2400, 2, 256), (2400, 1, 2048), (4096, 2, 1032), (2401, 5, 520), (2400, 3, 64),
                                   (2500, 2, 1003), (8200, 2, 128)])
def test_moves_of_many_tokens(t, k, d, with_residual):
    """A warp per token or pair: row widths of one and several rounds of a warp, even and odd counts
    of choices."""
    _check_moves(t, k, d, with_residual, t + d)


@gpu
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("t,e,k,dtype", [(5000, 8, 2, torch.bfloat16), (4097, 61, 6, torch.float32), (30000, 64, 4, torch.bfloat16),
                                         (100_003, 16, 1, torch.float32), (3000, 300, 16, torch.bfloat16), (2000, 1024, 3, torch.float32)])
def test_route_of_many_tokens(t, e, k, dtype, normalize):
    """More rows than one block takes, and more blocks than one."""
    g = torch.Generator().manual_seed(t)
    logits = (2 * torch.randn(t, e, generator=g)).to(dtype)
    logits[torch.rand(t, e, generator=g) < 0.3] = NINF
    logits[::97] = NINF
    leaf = logits.cuda().requires_grad_()
    weights, ids, plan = fn.moe_route(leaf, k, normalize)
    x = logits.double()
    top, order = x.sort(dim=1, descending=True, stable=True)
    chosen = torch.where(top[:, :k] == NINF, -1, order[:, :k])
    assert torch.equal(ids.cpu().long(), chosen)
    among = torch.zeros(t, e, dtype=torch.bool).scatter_(1, order[:, :k], True) & (x != NINF) if normalize else x != NINF
    probs = torch.where(among, x, torch.full_like(x, NINF)).softmax(1).nan_to_num(0.0)
    w64 = probs.gather(1, chosen.clamp_min(0)) * (chosen >= 0)
    near(weights, w64, (90 + e) * F32 * w64 + 1e-37)
    key = torch.where(chosen < 0, e, chosen).reshape(-1)
    slots = torch.empty(t * k, dtype=torch.int64)
    slots[key.argsort(stable=True)] = torch.arange(t * k)
    assert torch.equal(plan.slots.cpu().long().reshape(-1), slots)
    assert plan.offsets.tolist() == [0] + torch.bincount(key, minlength=e + 1)[:e].cumsum(0).tolist()
    again = fn.moe_plan(ids, e)
    assert torch.equal(again.slots, plan.slots) and torch.equal(again.offsets, plan.offsets)
    dw = torch.randn(t, k, generator=g)
    weights.backward(dw.cuda())
    up = torch.zeros_like(probs).scatter_add_(1, chosen.clamp_min(0), dw.double() * (chosen >= 0))
    want = probs * (up - (probs * up).sum(1, keepdim=True))
    size = probs * (up.abs() + (probs * up.abs()).sum(1, keepdim=True))
    near(leaf.grad, want, (BF * want.abs() if dtype == torch.bfloat16 else 0) + (300 + 4 * e) * F32 * size + 1e-37)


@gpu
def test_linear_products_without_rows_are_checked():
    x, w = torch.empty(0, 16, device="cuda").bfloat16(), torch.randn(24, 8, device="cuda").bfloat16()
    rows = torch.randn(8, 16, device="cuda").bfloat16()
    for call in (lambda: fn.linear(x, w), lambda: fn.linear_dgrad(x, w), lambda: fn.linear_wgrad(x, rows),
                 lambda: fn.linear_wgrad(x, x[:, :8], out=torch.zeros(16, 16, device="cuda"))):
        with pytest.raises(RuntimeError):
            call()


@gpu
def test_captured_block_without_accumulators():
    """Every weight's own gradient in a graph, replayed on other rows."""
    leaves = [t.requires_grad_() for t in _block(15)]

    def step():
        out = fn.moe_swiglu(*leaves, 2, residual=leaves[0])
        return (out.detach(), *torch.autograd.grad(out, leaves, out.detach()))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (16, 17):
        with torch.no_grad():
            leaves[0].copy_(_block(seed)[0])
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    check_device_errors()


@gpu
@pytest.mark.parametrize("d", [128, 256])
def test_captured_moves_of_plans_that_change(d):
    """The places are read at each replay, whole or with rows left out (both ways to zero those)."""
    t, k = 9000, 2
    x, y = torch.randn(t, d, device="cuda").bfloat16(), torch.randn(t * k, d, device="cuda").bfloat16().requires_grad_()
    slots = torch.arange(t * k, dtype=torch.int32, device="cuda").view(t, k).clone()
    plan = fn.MoePlan(torch.tensor([0, t * k], dtype=torch.int32, device="cuda"), slots)
    weights = torch.rand(t, k, device="cuda")

    def step():
        out = fn.moe_combine(y, weights, plan)
        return fn.moe_dispatch(x, plan), torch.autograd.grad(out, y, x)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows, dy = step()
    for left_out in (0, 700, 0):
        slots.copy_(torch.randperm(t * k, device="cuda").view(t, k))
        if left_out:
            gone = slots.view(-1)[:left_out].long()
            slots.view(-1)[:left_out] = slots.view(-1)[left_out: 2 * left_out]  # named twice, so others not at all
        rows.fill_(float("nan")), dy.fill_(float("nan"))
        graph.replay()
        assert rows.isfinite().all() and dy.isfinite().all()
        last = slots.view(-1)[2 * left_out:].long()
        token = torch.arange(2 * left_out, t * k, device="cuda") // k
        assert torch.equal(rows[last], x[token])
        if left_out:
            assert not rows[gone].any() and not dy[gone].any()
    check_device_errors()
