"""Linear-layer products on the tcgen05 GEMM (``csrc/gemm.cu``).

All three products of a bias-free linear layer ``y = x w^T`` read their operands in
place (no transposes): the kernel takes each operand K-major or MN-major. (Reference:
``F.linear`` at ``resihp/parallel/tp.py:235-248,272`` and its autograd products.)

bf16 CUDA tensors always run the hand-written kernel; FP32 tensors (CPU or CUDA)
compute in plain torch, the FP32 reference path.
"""

from __future__ import annotations

import operator
import os

import torch

from . import _ext

EPI_BF16 = 0
EPI_F32 = 1
EPI_ACC_F32 = 2
EPI_ADD_BF16 = 3
EPI_RED_F32 = 4

#: Weight-gradient accumulation through ``red.global.add`` (no load in the epilogue)
#: instead of load-add-store; same sums except that subnormals flush to zero. Each
#: element receives exactly one addition per launch, so the result is deterministic.
#: Measured 14-25 % faster on the 1.3B weight-gradient shapes (``bench_kernels.py
#: gemm_time``); ``RESIHP_WGRAD_RED=0`` selects load-add-store.
WGRAD_RED = os.environ.get("RESIHP_WGRAD_RED", "1") == "1"


def whole(value, what: str) -> int:
    """``value`` as an int (of any integer type); refuses what is none."""
    try:
        return operator.index(value)
    except TypeError:
        raise ValueError(f"{what} must be a whole number, got {value!r}") from None


def _cuda(*tensors) -> bool:
    return tensors[0].is_cuda and tensors[0].dtype == torch.bfloat16


def linear(x: torch.Tensor, w: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ w.T`` (+ ``residual``), x: [..., K], w: [N, K]."""
    if not _cuda(x):
        y = torch.nn.functional.linear(x, w)
        return y if residual is None else y + residual
    lead = x.shape[:-1]
    x2 = x.reshape(-1, x.shape[-1])
    out = torch.empty((x2.shape[0], w.shape[0]), dtype=torch.bfloat16, device=x.device)
    if not out.shape[0] and x2.shape[1] == w.shape[1]:
        pass  # no rows: nothing to launch
    elif residual is None:
        _ext.require().gemm(x2, False, w, False, out, EPI_BF16)
    else:
        r2 = residual.reshape(-1, w.shape[0])
        _ext.require().gemm(x2, False, w, False, out, EPI_ADD_BF16, 1.0, r2)
    return out.view(*lead, w.shape[0])


def linear_dgrad(dy: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """``dy @ w``: the input gradient of ``x @ w.T``; dy: [..., N], w: [N, K]."""
    if not _cuda(dy):
        return dy @ w
    lead = dy.shape[:-1]
    d2 = dy.reshape(-1, dy.shape[-1])
    out = torch.empty((d2.shape[0], w.shape[1]), dtype=torch.bfloat16, device=dy.device)
    if out.shape[0] or d2.shape[1] != w.shape[0]:
        _ext.require().gemm(d2, False, w, True, out, EPI_BF16)
    return out.view(*lead, w.shape[1])


def linear_wgrad(dy: torch.Tensor, x: torch.Tensor, out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """``dy^T @ x`` in FP32: the weight gradient of ``x @ w.T``.

    With ``accumulate`` the product is added into ``out`` (an FP32 main-grad buffer),
    which is how gradients of successive micro-batches accumulate without a separate
    add kernel.
    """
    d2 = dy.reshape(-1, dy.shape[-1])
    x2 = x.reshape(-1, x.shape[-1])
    if not _cuda(dy):
        g = d2.t().float() @ x2.float()
        if out is None:
            return g
        if accumulate:
            out.add_(g)
        else:
            out.copy_(g)
        return out
    if out is None:
        out = torch.empty((d2.shape[1], x2.shape[1]), dtype=torch.float32, device=dy.device)
        accumulate = False
    if d2.shape[0] == x2.shape[0] == 0 and out.shape == (d2.shape[1], x2.shape[1]):  # a sum of nothing
        return out if accumulate else out.zero_()
    _ext.require().gemm(d2, True, x2, True, out, ((EPI_RED_F32 if WGRAD_RED else EPI_ACC_F32) if accumulate
                                                 else EPI_F32))
    return out


# ---------------------------------------------------------------------------------------
# products grouped by expert (``csrc/grouped.cu``)
# ---------------------------------------------------------------------------------------

MAX_GROUPS = 1024
MAX_SIZE = 2**31 - 1 - 512  # rows and widths: leaves room for a tile in 31 bits


def check_groups(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> None:
    """Refuse operands of a grouped product ``x [R, K]``, ``w [E, N, K]``, ``offsets [E + 1]``."""
    if x.dim() != 2 or w.dim() != 3 or x.shape[1] != w.shape[2]:
        raise ValueError(f"a grouped product takes rows [R, K] and weights [E, N, K], got {list(x.shape)} and {list(w.shape)}")
    if x.dtype != w.dtype or x.device != w.device:
        raise ValueError(f"rows ({x.dtype}, {x.device}) and weights ({w.dtype}, {w.device}) must match")
    _check_offsets(x, offsets, w.shape[0])
    _check_widths(x, w.shape[1], w.shape[2])


def _check_offsets(x: torch.Tensor, offsets: torch.Tensor, groups: int) -> None:
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.device != x.device:
        raise ValueError("offsets must be an int32 vector on the rows' device")
    if offsets.numel() != groups + 1 or not 1 <= groups <= MAX_GROUPS:
        raise ValueError(f"{groups} groups need {groups + 1} offsets (1 to {MAX_GROUPS} groups), got {offsets.numel()}")


def _check_widths(x: torch.Tensor, n: int, k: int) -> None:
    if n < 1 or k < 1:
        raise ValueError("a grouped product needs widths of at least 1")
    if _cuda(x) and (n % 8 or k % 8):
        raise ValueError(f"the bf16 kernels need widths that are multiples of 8, got {n} and {k}")
    if _cuda(x) and max(x.shape[0], n, k) > MAX_SIZE:
        raise ValueError(f"the bf16 kernels take up to {MAX_SIZE} rows and columns, got {x.shape[0]}, {n} and {k}")
    if x.is_cuda and x.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"grouped products run in bf16 or fp32, not {x.dtype}")


def check_aligned(rows: torch.Tensor, out: torch.Tensor) -> None:
    """The kernels write a weight gradient in 16-byte units."""
    if _cuda(rows) and out.data_ptr() % 16:
        raise ValueError("the bf16 kernels need a weight gradient at a 16-byte aligned address")


def _tiles(t: torch.Tensor) -> torch.Tensor:
    """``t`` as TMA reads it: unit inner stride, 16-byte aligned base and outer strides (which
    no two rows may share); anything else is copied."""
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s > 0 and s % 8 == 0 for s in t.stride()[:-1]):
        return t
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def _bounds(offsets: torch.Tensor, rows: int) -> list[int]:
    """The groups' first rows on the host, clamped like the kernels do (FP32 path)."""
    out, last = [0], 0
    for v in offsets.tolist()[1:]:
        last = max(last, min(max(v, 0), rows))
        out.append(last)
    return out


def grouped_linear(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """``y[r] = w[g(r)] @ x[r]``: rows ``offsets[g] .. offsets[g + 1]`` of ``x [R, K]`` times the
    group's ``w[g] [N, K]``; rows behind the last group give zeros. ``offsets`` (int32, first
    entry 0, not decreasing) stays on the device: lengths, empty groups among them, are read
    by the kernel. Entries that decrease or pass ``R`` are clamped and reported by
    :func:`check_device_errors`."""
    check_groups(x, w, offsets)
    if _cuda(x):
        return _ext.require().grouped_rows(_tiles(x), _tiles(w), False, offsets.contiguous())
    at = _bounds(offsets, x.shape[0])
    parts = [torch.nn.functional.linear(x[a:b], w[g]) for g, (a, b) in enumerate(zip(at, at[1:]))]
    return torch.cat(parts + [x.new_zeros(x.shape[0] - at[-1], w.shape[1])])


def grouped_dgrad(dy: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """``dx[r] = w[g(r)]^T @ dy[r]``: the input gradient of :func:`grouped_linear`."""
    check_groups(dy, w.transpose(1, 2) if w.dim() == 3 else w, offsets)
    if _cuda(dy):
        return _ext.require().grouped_rows(_tiles(dy), _tiles(w), True, offsets.contiguous())
    at = _bounds(offsets, dy.shape[0])
    parts = [dy[a:b] @ w[g] for g, (a, b) in enumerate(zip(at, at[1:]))]
    return torch.cat(parts + [dy.new_zeros(dy.shape[0] - at[-1], w.shape[2])])


def grouped_wgrad(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor, out: torch.Tensor | None = None,
                  accumulate: bool = False) -> torch.Tensor:
    """``dw[g] = sum over the group's rows of dy[r] x[r]^T`` in FP32 ``[E, N, K]``: the weight
    gradient of :func:`grouped_linear`, added into ``out`` with ``accumulate``."""
    groups = offsets.numel() - 1
    if dy.dim() != 2 or x.dim() != 2 or dy.shape[0] != x.shape[0] or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError("a grouped weight gradient takes dy [R, N] and x [R, K] of one dtype and device")
    _check_offsets(dy, offsets, groups)
    _check_widths(dy, dy.shape[1], x.shape[1])
    shape = (groups, dy.shape[1], x.shape[1])
    if out is None:
        out, accumulate = torch.empty(shape, dtype=torch.float32, device=dy.device), False
    elif out.shape != shape or out.dtype != torch.float32 or out.device != dy.device or not out.is_contiguous():
        raise ValueError(f"the weight gradient goes into a contiguous fp32 {list(shape)} on the rows' device")
    else:
        check_aligned(dy, out)
    if _cuda(dy):
        _ext.require().grouped_wgrad(_tiles(dy), _tiles(x), offsets.contiguous(), out, accumulate)
        return out
    at = _bounds(offsets, dy.shape[0])
    for g, (a, b) in enumerate(zip(at, at[1:])):
        product = dy[a:b].t().float() @ x[a:b].float()
        if accumulate:
            out[g].add_(product)
        else:
            out[g].copy_(product)
    return out


#: Codes a kernel records in its device's error word (``ErrorCode`` in csrc/common.cuh).
ERROR_CODES = {
    1: "TMA producer waited past its budget for a free shared-memory stage",
    2: "MMA issuer waited past its budget for a filled stage or a free accumulator",
    3: "epilogue waited past its budget for a finished accumulator",
    4: "a wait on another GPU's flag ran out its budget (peer never arrived)",
    5: "a bounds check skipped an access (offsets or places of a sparse MLP out of range, or the checked build)",
}
PEER_WAIT = 4


class KernelError(RuntimeError):
    """A kernel reported an error code (a bounded wait that ran out, a failed bounds
    check) instead of hanging or faulting; ``code`` is the recorded code."""

    def __init__(self, code: int, device_index: int):
        self.code = int(code)
        self.device_index = int(device_index)
        what = ERROR_CODES.get(self.code, "unknown error code")
        super().__init__(f"resihp kernel reported error code {self.code} on cuda:{self.device_index}: {what}")


def check_device_errors(device: torch.device | int | None = None) -> None:
    """Raise :class:`KernelError` if any kernel on ``device`` reported a timed-out wait
    or a bounds error since the last check (the word is cleared by the read)."""
    if not torch.cuda.is_available():
        return
    index = torch.cuda.current_device() if device is None else torch.device("cuda", device).index if isinstance(device, int) else (device.index or 0)
    code = _ext.require().read_and_clear_error(index)
    if code:
        raise KernelError(code, index)
