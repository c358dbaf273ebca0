"""Counter-based dropout: the generator's published vectors, the mask on both devices, gradients.

Tolerances count roundings: ``x * scale + residual`` is two fp32 roundings of its terms and one
of the result to its type.
"""

import math

import pytest
import torch

from resihp.ops import functional as fn
from resihp.ops.dropout import dropout_mask, dropout_threshold, philox

gpu = pytest.mark.gpu
F32 = 2.0**-24
HALF = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}


def _expect(x, keep, p, residual=None):
    drop = dropout_threshold(p)
    y = torch.where(keep, x.double() * (65536 / max(1, 65536 - drop)), torch.zeros((), dtype=torch.float64))
    size = y.abs()
    if residual is not None:
        y, size = y + residual.double(), size + residual.double().abs()
    return y, size


def _check(got, x, keep, p, residual=None):
    want, size = _expect(x.detach().cpu(), keep.cpu(), p, None if residual is None else residual.detach().cpu())
    off = (got.detach().double().cpu() - want).abs()
    assert bool((off <= HALF[got.dtype] * want.abs() + 3 * F32 * size).all())


def test_generator_vectors():
    """Philox4x32-10 of the zero, all-ones and pi-digit counters and keys (the paper's library's
    known answers)."""
    def words(c01, c23, key):
        block = torch.tensor([c01 - (1 << 64) if c01 >> 63 else c01])
        return [int(w) for w in philox(block, c23, key)]

    assert words(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = (1 << 64) - 1
    assert words(ones, ones, ones) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert words(0x85A308D3243F6A88, 0x0370734413198A2E, 0x299F31D0A4093822) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_share_and_independence_on_the_cpu():
    """The kept share of n draws is within six standard deviations; other seeds and offsets give
    other masks that agree as often as chance says."""
    n, p = 1 << 18, 0.3
    a = dropout_mask(n, p, 11)
    q = dropout_threshold(p) / 65536
    sigma = math.sqrt(q * (1 - q) / n)
    assert abs(1 - a.double().mean().item() - q) < 6 * sigma
    agree = q * q + (1 - q) * (1 - q)
    for other in (dropout_mask(n, p, 12), dropout_mask(n, p, 11, offset=1), dropout_mask(n, p, 11, offset=1 << 40),
                  dropout_mask(n, p, 11, first=8), dropout_mask(n, p, 11, first=1)):
        assert abs((a == other).double().mean().item() - agree) < 6 * math.sqrt(agree * (1 - agree) / n)


@pytest.mark.parametrize("first", [0, 1, 8, 13, 2**34 + 5])
def test_mask_is_a_window_of_one_sequence(first):
    whole = dropout_mask(200, 0.5, 3, 9, first=first)
    assert torch.equal(dropout_mask(90, 0.5, 3, 9, first=first + 57), whole[57:147])


def test_cpu_forward_and_gradient():
    x = torch.randn(6, 10, requires_grad=True)
    r = torch.randn(6, 10, requires_grad=True)
    y = fn.dropout(x, 0.4, 5, 6, residual=r, first_row=3)
    keep = dropout_mask(60, 0.4, 5, 6, first=30).view(6, 10)
    _check(y, x, keep, 0.4, r)
    dy = torch.randn(6, 10)
    y.backward(dy)
    _check(x.grad, dy, keep, 0.4)
    assert torch.equal(r.grad, dy)
    state = torch.tensor([5, 6])
    assert torch.equal(fn.dropout(x, 0.4, state, residual=r, first_row=3), y)


def test_ends_of_the_range():
    x = torch.randn(4, 8)
    assert torch.equal(fn.dropout(x, 0.0, 1), x)
    assert not fn.dropout(x, 1.0, 1).any()
    assert fn.dropout(torch.zeros(0, 8), 0.5, 1).shape == (0, 8)


REFUSALS = {
    "p above 1": lambda d: fn.dropout(torch.zeros(2, 8, device=d), 1.5, 1),
    "p below 0": lambda d: fn.dropout(torch.zeros(2, 8, device=d), -0.1, 1),
    "p not a number": lambda d: fn.dropout(torch.zeros(2, 8, device=d), float("nan"), 1),
    "half precision": lambda d: fn.dropout(torch.zeros(2, 8, device=d, dtype=torch.float16), 0.5, 1),
    "a scalar": lambda d: fn.dropout(torch.zeros((), device=d), 0.5, 1),
    "residual of another shape": lambda d: fn.dropout(torch.zeros(2, 8, device=d), 0.5, 1, residual=torch.zeros(8, device=d)),
    "residual of another type": lambda d: fn.dropout(torch.zeros(2, 8, device=d), 0.5, 1, residual=torch.zeros(2, 8, device=d).bfloat16()),
    "a negative seed": lambda d: fn.dropout(torch.zeros(2, 8, device=d), 0.5, -1),
    "a seed past 64 bits": lambda d: fn.dropout(torch.zeros(2, 8, device=d), 0.5, 1 << 64),
    "a negative offset": lambda d: fn.dropout(torch.zeros(2, 8, device=d), 0.5, 1, -1),
    "a seed tensor of another type": lambda d: fn.dropout(torch.zeros(2, 8, device=d), 0.5, torch.zeros(2, device=d)),
    "a seed tensor and an offset": lambda d: fn.dropout(torch.zeros(2, 8, device=d), 0.5, torch.zeros(2, dtype=torch.int64, device=d), 1),
    "a negative row": lambda d: fn.dropout(torch.zeros(2, 8, device=d), 0.5, 1, first_row=-1),
    "a row past 62 bits": lambda d: fn.dropout(torch.zeros(2, 8, device=d), 0.5, 1, first_row=1 << 60),
}


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
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,p,first_row", [((1, 1), 0.5, 0), ((3, 5), 0.1, 0), ((3, 5), 0.1, 7), ((64, 128), 0.25, 0),
                                               ((64, 128), 0.25, 3), ((33, 1003), 0.1, 0), ((33, 1003), 0.6, 2**33 // 1003),
                                               ((2, 7, 40), 0.3, 1), ((1000, 1000), 0.0, 0), ((20, 64), 1.0, 0),
                                               ((301, 2048), 0.1, 2**24 + 1), ((0, 16), 0.5, 0)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_kernel_mask_and_gradient(shape, p, first_row, dtype, with_residual):
    g = torch.Generator().manual_seed(0)
    seed, offset = (1 << 63) + 12345, (1 << 40) + 3
    x = torch.randn(shape, generator=g).to(dtype).cuda().requires_grad_()
    r = torch.randn(shape, generator=g).to(dtype).cuda().requires_grad_() if with_residual else None
    y = fn.dropout(x, p, seed, offset, residual=r, first_row=first_row)
    keep = dropout_mask(x.numel(), p, seed, offset, first=first_row * shape[-1]).view(shape)
    _check(y, x, keep, p, r)
    dy = torch.randn(shape, generator=g).to(dtype).cuda()
    y.backward(dy)
    _check(x.grad, dy, keep, p)
    if with_residual:
        assert torch.equal(r.grad, dy)


@gpu
def test_token_shards_draw_the_whole_mask():
    x = torch.randn(96, 72, device="cuda").bfloat16()
    whole = fn.dropout(x, 0.3, 8, 9)
    parts = [fn.dropout(x[a: a + 32], 0.3, 8, 9, first_row=a) for a in (0, 32, 64)]
    assert torch.equal(torch.cat(parts), whole)


@gpu
def test_dropped_infinities_give_zero():
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.full((50, 40), float("nan"), device="cuda", dtype=dtype)
        x[::2] = float("inf")
        keep = dropout_mask(2000, 0.5, 2).view(50, 40)
        y = fn.dropout(x, 0.5, 2).cpu()
        assert not y[~keep].any() and not y[keep].isfinite().any()


@gpu
def test_views_and_odd_addresses():
    base = torch.randn(40, 200, device="cuda").bfloat16()
    for x in (base[:, 7:107], base.t()[:96], base.reshape(-1)[3: 3 + 6400].view(40, 160), base[:, :1].expand(40, 64)):
        r = torch.randn(x.shape, device="cuda").bfloat16()
        assert torch.equal(fn.dropout(x, 0.3, 1, residual=r), fn.dropout(x.clone(), 0.3, 1, residual=r))
    x = torch.randn(30, 16, device="cuda").bfloat16().requires_grad_()
    fn.dropout(x, 0.3, 4).sum().backward()  # a stride-0 gradient
    _check(x.grad, torch.ones(30, 16), dropout_mask(480, 0.3, 4).view(30, 16), 0.3)


@gpu
def test_more_elements_than_32_bits():
    rows, d = 2**20 + 3, 2056
    x = torch.ones(rows, d, device="cuda", dtype=torch.bfloat16)
    assert x.numel() > 2**31
    y = fn.dropout(x, 0.5, 6, 7)
    for r in (0, rows // 2, rows - 1):
        keep = dropout_mask(d, 0.5, 6, 7, first=r * d)
        assert torch.equal(y[r].cpu() != 0, keep)
    del y


@gpu
def test_graph_replays_draw_new_masks_from_a_seed_tensor():
    x = torch.randn(64, 256, device="cuda").bfloat16().requires_grad_()
    state = torch.tensor([42, 0], device="cuda")

    def step():
        y = fn.dropout(x, 0.2, state)
        return y, torch.autograd.grad(y, x, torch.ones_like(y))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step()
    for offset in (1, 2, (1 << 62) + 5):
        state[1] = offset
        graph.replay()
        assert torch.equal(y, fn.dropout(x, 0.2, 42, offset))
        keep = dropout_mask(x.numel(), 0.2, 42, offset).view(64, 256)
        assert torch.equal(dx.cpu() != 0, keep)


@gpu
def test_a_seed_tensor_must_not_change_before_the_backward_pass():
    x = torch.randn(8, 16, device="cuda").bfloat16().requires_grad_()
    state = torch.tensor([1, 2], device="cuda")
    y = fn.dropout(x, 0.2, state)
    state.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@gpu
def test_recomputed_activations_drop_the_same_elements():
    from torch.utils.checkpoint import checkpoint

    x = torch.randn(32, 64, device="cuda").bfloat16().requires_grad_()

    def layer(t):
        return fn.dropout(t * 2, 0.3, 9, 1, residual=t)

    y = checkpoint(layer, x, use_reentrant=False)
    y.backward(torch.ones_like(y))
    z = x.detach().clone().requires_grad_()
    layer(z).backward(torch.ones_like(y))
    assert torch.equal(x.grad, z.grad)


@gpu
def test_gradient_has_no_second_derivative():
    x = torch.randn(4, 16, device="cuda").bfloat16().requires_grad_()
    (dx,) = torch.autograd.grad(fn.dropout(x, 0.5, 1).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        dx.float().sum().backward()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_against_differences(dtype):
    """Dropout is linear: the difference of two inputs that are apart by h in one element equals
    the gradient times h, up to the outputs' roundings."""
    x = torch.randn(9, 24, device="cuda").to(dtype)
    h = 0.5
    keep = dropout_mask(216, 0.25, 3, 4).view(9, 24)
    leaf = x.clone().requires_grad_()
    fn.dropout(leaf, 0.25, 3, 4).backward(torch.ones_like(x))
    for r, c in ((0, 0), (3, 7), (8, 23)):
        moved = x.clone()
        moved[r, c] += h
        step = (moved - x)[r, c].double().item()
        diff = (fn.dropout(moved, 0.25, 3, 4) - fn.dropout(x, 0.25, 3, 4)).double().sum().item()
        size = abs(moved[r, c].item()) + abs(x[r, c].item())
        assert abs(diff - leaf.grad[r, c].item() * step) <= 4 * HALF[dtype] * (size + h) * 65536 / (65536 - 16384)
        assert (leaf.grad[r, c] != 0).item() == keep[r, c].item()


NOT_NUMBERS = {
    "a fractional seed": lambda x: fn.dropout(x, 0.5, 1.5),
    "a seed of text": lambda x: fn.dropout(x, 0.5, "1"),
    "a fractional offset": lambda x: fn.dropout(x, 0.5, 1, 2.5),
    "a fractional row": lambda x: fn.dropout(x, 0.5, 1, first_row=1.0),
    "p of text": lambda x: fn.dropout(x, "0.5", 1),
    "no p": lambda x: fn.dropout(x, None, 1),
}


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("what", sorted(NOT_NUMBERS))
def test_refusals_of_what_is_no_number(what, device):
    with pytest.raises(ValueError, match="number"):
        NOT_NUMBERS[what](torch.zeros(2, 8, device=device))


def test_numbers_of_any_type():
    import numpy as np

    x = torch.ones(4, 9)
    want = fn.dropout(x, 0.25, 3, 4, first_row=2)
    assert torch.equal(fn.dropout(x, np.float64(0.25), np.uint64(3), np.int32(4), first_row=np.int64(2)), want)
    assert torch.equal(fn.dropout(x, np.float32(0.25), True + 2, 4, first_row=2), want)
