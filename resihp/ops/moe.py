"""Sparse (mixture-of-experts) MLP: routing, row movements and per-expert linear layers.

The steps of one block, in order, over ``T`` tokens, ``E`` experts and ``k`` choices per token::

    weights, ids, plan = moe_route(logits, k)                 # logits [T, E]
    rows = moe_dispatch(x, plan)                              # [T * k, d], sorted by expert
    gu = grouped_linear(rows, w_gate_up, plan.offsets, g)     # one linear layer per expert
    y = grouped_linear(swiglu(gu), w_down, plan.offsets, g)
    out = moe_combine(y, weights, plan, residual=x)           # [T, d]

:func:`moe_swiglu` is that block in one call. Nothing waits for the host: the experts' row
counts stay on the device, and every kernel reads them there. A choice that no expert takes
(``-inf`` logits, ids outside ``start .. start + experts``) moves no weight: its place lies
behind the last expert's rows, which are zero, and :func:`moe_combine` leaves it out.

As elsewhere in this package bf16 CUDA tensors run the kernels (``csrc/moe.cu``,
``csrc/grouped.cu``) and FP32 rows the plain torch expressions; the router's logits run its
kernel on every CUDA device in bf16 or FP32. FP32 grouped products read ``offsets`` on the
host, so a step of theirs cannot be captured. (No counterpart in the reference, whose blocks
are dense.)
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _ext
from .gemm import MAX_GROUPS, _cuda, check_aligned, check_groups, whole
from .gemm import grouped_linear as _grouped_linear

MAX_CHOICES = 16
MAX_PAIRS = 0x7FFF0000  # tokens * k: places are int32, with room for a block's rows


class MoePlan(NamedTuple):
    """Where the ``T * k`` (token, choice) pairs go when sorted by expert, token, choice.

    ``offsets`` (int32 ``[E + 1]``): expert ``e`` owns the rows ``offsets[e] .. offsets[e + 1]``.
    ``slots`` (int32 ``[T, k]``): each pair's row; pairs of no expert have the rows from
    ``offsets[E]`` on. Every row belongs to exactly one pair; a plan made elsewhere has to keep
    that. Where it does not, rows without a pair are zeros, of two pairs with one place either
    may win, and places outside the rows are left out and on the kernels reported by
    :func:`resihp.ops.check_device_errors`.
    """

    offsets: torch.Tensor
    slots: torch.Tensor


# ---------------------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------------------


def _plan_torch(ids, experts: int, start: int) -> MoePlan:
    local = ids.reshape(-1).long() - start
    key = torch.where((local < 0) | (local >= experts), experts, local)
    order = key.argsort(stable=True)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device=ids.device)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=ids.device)
    offsets[1:] = torch.bincount(key, minlength=experts + 1)[:experts].cumsum(0)
    return MoePlan(offsets, slots.to(torch.int32).view(ids.shape))


def _route_torch(logits, k: int, normalize: bool):
    x = logits.float()
    top, ids = x.sort(dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    allowed = top != float("-inf")
    among = top if normalize else x
    m = among.amax(1, keepdim=True).detach()
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    total = (among - m).exp().sum(1, keepdim=True)
    # (chosen after the division: a gradient at a choice that was not made does not reach ``total``)
    weights = torch.where(allowed, (top - m).exp() / total.masked_fill(total == 0, 1.0), torch.zeros_like(top))
    return weights, torch.where(allowed, ids, torch.full_like(ids, -1)).to(torch.int32)


def _check_pairs(tokens: int, k: int) -> None:
    if tokens * k > MAX_PAIRS:
        raise ValueError(f"a plan takes up to {MAX_PAIRS} (token, choice) pairs, got {tokens} x {k}")


def _check_choices(experts: int, k) -> int:
    k = whole(k, "the number of choices")
    if not 1 <= experts <= MAX_GROUPS or not 1 <= k <= min(experts, MAX_CHOICES):
        raise ValueError(f"{k} choices of {experts} experts: 1 to {MAX_CHOICES} choices, no more than experts, "
                         f"of 1 to {MAX_GROUPS} experts")
    return k


def moe_route(logits, k: int, normalize: bool = True):
    """The ``k`` experts of every token: ``(weights, ids, plan)`` from router logits ``[T, E]``.

    Choice ``j`` is the token's ``j``-th largest logit, the lowest expert first among equal
    ones. ``weights`` (FP32 ``[T, k]``) are the softmax over the chosen experts (``normalize``)
    or the chosen experts' part of the softmax over all; gradients flow through them. A logit
    of ``-inf`` is an expert the token may not use: it is never chosen, and where fewer than
    ``k`` are left the remaining choices are ``-1`` with weight 0 -- a token without any
    allowed expert (padding) takes no row. ``ids`` is int32 ``[T, k]``, ``plan`` sorts the
    choices (:class:`MoePlan`). NaN sorts above everything, and its token's weights are NaN.
    """
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"router logits must be bf16 or fp32 [T, E], got {logits.dtype} {list(logits.shape)}")
    experts = logits.shape[1]
    k = _check_choices(experts, k)
    _check_pairs(logits.shape[0], k)
    if logits.is_cuda:
        weights, ids, offsets, slots = _ext.require().moe_route_ad(logits, k, normalize)
        return weights, ids, MoePlan(offsets, slots)
    weights, ids = _route_torch(logits, k, normalize)
    return weights, ids, _plan_torch(ids, experts, 0)


def moe_plan(ids, experts: int, start: int = 0) -> MoePlan:
    """The plan of choices made elsewhere: ``ids`` int32 ``[T, k]``, the experts ``start ..
    start + experts`` (this rank's); any other id is a choice that no expert here takes."""
    if ids.dim() != 2 or ids.dtype != torch.int32 or ids.shape[1] < 1:
        raise ValueError(f"expert ids must be int32 [T, k], got {ids.dtype} {list(ids.shape)}")
    experts, start = whole(experts, "the number of experts"), whole(start, "the first expert")
    if not 1 <= experts <= MAX_GROUPS or not -(2**31) <= start < 2**31:
        raise ValueError(f"a plan takes 1 to {MAX_GROUPS} experts from a 32-bit start, got {experts} from {start}")
    _check_pairs(*ids.shape)
    if ids.is_cuda:
        return MoePlan(*_ext.require().moe_plan(ids.contiguous(), experts, start))
    return _plan_torch(ids, experts, start)


# ---------------------------------------------------------------------------------------
# row movements
# ---------------------------------------------------------------------------------------


def _check_plan(rows, plan: MoePlan) -> tuple[torch.Tensor, torch.Tensor]:
    offsets, slots = plan
    if slots.dim() != 2 or slots.shape[1] < 1 or offsets.dim() != 1 or offsets.numel() < 2:
        raise ValueError("a plan is offsets [E + 1] and slots [T, k]")
    _check_pairs(*slots.shape)
    if slots.dtype != torch.int32 or offsets.dtype != torch.int32:
        raise ValueError("a plan's offsets and slots must be int32")
    if slots.device != rows.device or offsets.device != rows.device:
        raise ValueError("a plan must lie on its rows' device")
    if rows.dim() != 2 or rows.shape[1] < 1:
        raise ValueError(f"rows must be [rows, d] with d of at least 1, got {list(rows.shape)}")
    if rows.is_cuda and rows.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"rows move in bf16 or fp32, not {rows.dtype}")
    return offsets.contiguous(), slots.contiguous()


def moe_dispatch(x, plan: MoePlan):
    """Token rows ``x [T, d]`` in the plan's order ``[T * k, d]``: ``y[slots[t, j]] = x[t]``, zeros
    in the rows of choices that no expert takes."""
    offsets, slots = _check_plan(x, plan)
    if x.shape[0] != slots.shape[0]:
        raise ValueError(f"{x.shape[0]} rows for a plan of {slots.shape[0]} tokens")
    if _cuda(x):
        return _ext.require().moe_dispatch_ad(x, offsets, slots)
    at = slots.long().reshape(-1)
    count = at.numel()
    kept = (at < offsets[-1])[:, None]
    rows = torch.where(kept, x.repeat_interleave(slots.shape[1], 0), torch.zeros((), dtype=x.dtype, device=x.device))
    at = torch.where((at >= 0) & (at < count), at, torch.full_like(at, count))  # places out of range go nowhere
    return x.new_zeros(count + 1, x.shape[1]).index_copy(0, at, rows)[:count]


def moe_combine(y, weights, plan: MoePlan, residual=None):
    """``out[t] = residual[t] + sum_j weights[t, j] * y[slots[t, j]]`` over the choices that an
    expert takes, in FP32 and rounded once; ``y [T * k, d]``, ``weights`` FP32 ``[T, k]``."""
    offsets, slots = _check_plan(y, plan)
    if y.shape[0] != slots.numel():
        raise ValueError(f"{y.shape[0]} rows for a plan of {slots.numel()} choices")
    if weights.shape != slots.shape or weights.dtype != torch.float32 or weights.device != y.device:
        raise ValueError(f"weights must be fp32 {list(slots.shape)} beside the rows")
    if residual is not None and (residual.shape != (slots.shape[0], y.shape[1]) or residual.dtype != y.dtype
                                 or residual.device != y.device):
        raise ValueError("the residual must be [T, d] in the rows' dtype, beside them")
    if _cuda(y):
        return _ext.require().moe_combine_ad(y, weights, offsets, slots, residual)
    at = slots.long()
    kept = ((at >= 0) & (at < offsets[-1].clamp_max(at.numel())))[..., None]
    rows = y[torch.where(kept[..., 0], at, torch.zeros_like(at)).reshape(-1)].view(*at.shape, y.shape[1])
    zero = torch.zeros((), device=y.device)  # (in both factors: what lies at a choice without an expert counts for nothing)
    out = (torch.where(kept, rows, zero.to(y.dtype)) * torch.where(kept, weights[..., None], zero)).sum(1)
    return (out if residual is None else residual + out).to(y.dtype)


# ---------------------------------------------------------------------------------------
# per-expert linear layers
# ---------------------------------------------------------------------------------------


def grouped_linear(x, w, offsets, main_grad=None):
    """One linear layer per expert: ``y[r] = w[e(r)] @ x[r]`` for the rows ``offsets[e] ..
    offsets[e + 1]`` of ``x [R, K]``, ``w [E, N, K]``; zeros behind the last expert's rows.

    CUDA bf16: tcgen05 products, widths multiples of 8; the weight gradient is accumulated
    into ``main_grad`` (FP32 ``[E, N, K]``) where one is given, as :func:`linear` does, and
    is ``w``'s gradient otherwise. Rows behind the last expert get a zero gradient.
    """
    check_groups(x, w, offsets)
    if main_grad is not None and (main_grad.shape != w.shape or main_grad.dtype != torch.float32
                                  or main_grad.device != w.device or not main_grad.is_contiguous()):
        raise ValueError(f"main_grad must be a contiguous fp32 {list(w.shape)} beside the weights")
    if main_grad is not None:
        check_aligned(x, main_grad)
    if not _cuda(x):
        return _grouped_linear(x, w, offsets)
    return _ext.require().grouped_linear_ad(x, w, offsets.contiguous(), main_grad)


def check_block(x, w_router, w_gate_up, w_down, k: int, residual, grads) -> None:
    """Refuse operands of a sparse block before its first step is launched."""
    if x.dim() != 2 or w_router.dim() != 2 or w_gate_up.dim() != 3 or w_down.dim() != 3:
        raise ValueError("a sparse block takes x [T, d], w_router [E, d], w_gate_up [E, 2F, d] and w_down [E, d, F]")
    (experts, d), f = w_router.shape, w_down.shape[2]
    if x.shape[1] != d or w_gate_up.shape != (experts, 2 * f, d) or w_down.shape != (experts, d, f) or d < 1 or f < 1:
        raise ValueError(f"x {list(x.shape)}, w_router {list(w_router.shape)}, w_gate_up {list(w_gate_up.shape)} and "
                         f"w_down {list(w_down.shape)} are not [T, d], [E, d], [E, 2F, d] and [E, d, F]")
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"a sparse block runs in bf16 or fp32, not {x.dtype}")
    weights = (w_router, w_gate_up, w_down)
    if any(w.dtype != x.dtype or w.device != x.device for w in weights):
        raise ValueError(f"the weights must match x ({x.dtype}, {x.device})")
    _check_pairs(x.shape[0], _check_choices(experts, k))
    if _cuda(x) and (experts % 8 or d % 8 or f % 8):
        raise ValueError(f"the bf16 kernels need experts and widths that are multiples of 8, got {experts} experts, "
                         f"{d} and {f}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("the residual must match x in shape, dtype and device")
    if grads is None:
        return
    if len(grads) != 3:
        raise ValueError("grads are the main gradients of the router's, gate / up's and down's weights")
    for w, g in zip(weights, grads):
        if g is not None and (g.shape != w.shape or g.dtype != torch.float32 or g.device != w.device):
            raise ValueError(f"main gradients must be fp32 {list(w.shape)} beside their weights")
        if g is not None and _cuda(w) and (g.stride(-1) != 1 or g.data_ptr() % 16 or g.stride(0) % 8):
            raise ValueError("main gradients must be 16-byte aligned rows")
        if g is not None and w.dim() == 3 and not g.is_contiguous():
            raise ValueError("the experts' main gradients must be contiguous")
