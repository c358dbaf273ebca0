"""Dropout whose mask is recomputed from a counter instead of stored (``csrc/dropout.cu``).

A run that is replanned after a failure, recomputes its activations or shards its tokens has
to drop the same elements every time. The mask is therefore a function of a key (``seed``), a
64-bit stream number (``offset``: one per call site, layer, micro-batch and step) and an
element's index in the whole tensor; the backward pass evaluates it again. (No counterpart in
the reference, whose blocks have no dropout.)
"""

from __future__ import annotations

import torch

from . import _ext
from .gemm import whole

_M32 = 0xFFFFFFFF


def _mul32(a: torch.Tensor, b: int) -> tuple[torch.Tensor, torch.Tensor]:
    """High and low words of the product of 32-bit numbers (in int64, whose own product wraps)."""
    a0, a1, b0, b1 = a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16
    mid = a1 * b0 + (a0 * b0 >> 16)
    mid2 = a0 * b1 + (mid & 0xFFFF)
    return a1 * b1 + (mid >> 16) + (mid2 >> 16), (mid2 & 0xFFFF) << 16 | (a0 * b0 & 0xFFFF)


def philox(block: torch.Tensor, offset: int, seed: int) -> list[torch.Tensor]:
    """The four words of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011) with the counter
    ``(block, offset)`` and the key ``seed``, as int64 tensors."""
    c = [block & _M32, (block >> 32) & _M32, torch.full_like(block, offset & _M32),
         torch.full_like(block, (offset >> 32) & _M32)]
    k0, k1 = seed & _M32, (seed >> 32) & _M32
    for _ in range(10):
        h0, l0 = _mul32(c[0], 0xD2511F53)
        h1, l1 = _mul32(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return c


def dropout_threshold(p: float) -> int:
    """Of 65536 equally likely numbers, how many drop an element."""
    return round(p * 65536)


def dropout_mask(n: int, p: float, seed: int, offset: int = 0, first: int = 0, device=None) -> torch.Tensor:
    """Which of the elements ``first .. first + n`` are kept (the plain torch form of the mask)."""
    b0 = first // 8
    block = torch.arange(b0, (first + n + 7) // 8, dtype=torch.int64, device=device)
    words = philox(block, offset, seed)
    halves = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], dim=1).reshape(-1)
    return (halves >= dropout_threshold(p))[first - 8 * b0: first - 8 * b0 + n]


def _signed(v: int) -> int:
    return v - (1 << 64) if v >> 63 else v


def dropout(x, p: float, seed, offset: int = 0, residual=None, first_row: int = 0):
    """``x`` with a share ``p`` of its elements set to 0 and the others scaled, plus ``residual``.

    ``p`` in ``[0, 1]`` counts in steps of ``2**-16``; what is kept is scaled by the inverse of
    the share that is kept after that rounding, so the expectation is exact. ``seed`` and
    ``offset`` are unsigned 64-bit numbers; equal ones give equal masks on every device.
    ``seed`` may be an int64 CUDA tensor ``[seed, offset]`` instead (then ``offset`` is left at
    0): a captured graph reads it at each replay, and the backward pass reads it again, so it
    must not change between the two. ``first_row`` is the place of ``x``'s first row in the
    whole tensor (a token shard draws its part of that tensor's mask); rows are the last
    dimension of ``x``. A dropped infinity or NaN gives 0.
    """
    try:
        p = float(p * 1.0)  # (a number's product; a text has none)
    except (TypeError, OverflowError):
        raise ValueError(f"dropout probability must be a number, got {p!r}") from None
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must lie in [0, 1], got {p}")
    if x.dtype not in (torch.bfloat16, torch.float32) or x.dim() < 1:
        raise ValueError(f"dropout takes bf16 or fp32 rows, got {x.dtype} {list(x.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("the residual must match x in shape, dtype and device")
    offset, first_row, state = whole(offset, "the offset"), whole(first_row, "first_row"), None
    if torch.is_tensor(seed):
        if seed.dtype != torch.int64 or seed.shape != (2,) or seed.device != x.device or offset:
            raise ValueError("a seed tensor is int64 [seed, offset] beside x, with no other offset")
        state, seed = seed.contiguous(), 0
    else:
        seed = whole(seed, "the seed")
        if not 0 <= seed < 1 << 64:
            raise ValueError("the seed must be an unsigned 64-bit number")
    if not 0 <= offset < 1 << 64:
        raise ValueError("the offset must be an unsigned 64-bit number")
    first = first_row * x.shape[-1]
    if first_row < 0 or first + x.numel() >= 1 << 62:
        raise ValueError("first_row must not be negative, and indices must stay below 2**62")
    if x.is_cuda:
        return _ext.require().dropout_ad(x, dropout_threshold(p), _signed(seed), _signed(offset), first, state, residual)
    if state is not None:
        seed, offset = (int(v) % (1 << 64) for v in state)
    drop = dropout_threshold(p)
    keep = dropout_mask(x.numel(), p, seed, offset, first).view(x.shape)
    out = torch.where(keep, x.float() * (65536.0 / max(1, 65536 - drop)), torch.zeros(()))
    return (out if residual is None else out + residual.float()).to(x.dtype)
