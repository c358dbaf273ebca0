"""The bounds-checked build (``-DRESIHP_BOUNDS_CHECK``, ``resihp/_C_checked.so``).

CPU: the variant is built from the same sources with the one extra define, into its own
build directory and library, and ``RESIHP_CHECKED=1`` makes the loader pick it.
GPU (runs last in the GPU tier): the checked library runs a forward GEMM, a
weight-gradient GEMM and causal attention forward + backward with every check passing
(no error recorded) and produces bit-identical results to the default library -- the
checks only test addresses, they never change the arithmetic.
"""

import json
import os
import subprocess
import sys

import pytest

from resihp.ops import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_checked_variant_is_the_same_sources_with_one_define():
    assert build.cuda_flags(checked=True) == build.CUDA_FLAGS + ["-DRESIHP_BOUNDS_CHECK"] + build.cuda_flags()[
        len(build.CUDA_FLAGS):]
    assert build.library_path(checked=True).endswith("_C_checked.so") and build.library_path().endswith("_C.so")


def test_loader_switch_names_the_checked_library():
    code = ("import json, resihp.ops._ext as e; print(json.dumps([e.CHECKED, e._LIB]))")
    for env, want in (({"RESIHP_CHECKED": "1"}, "_C_checked.so"), ({"RESIHP_CHECKED": "0"}, "_C.so")):
        out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT,
                             env={**os.environ, **env}, check=True)
        checked, lib = json.loads(out.stdout.strip().splitlines()[-1])
        assert checked == (env["RESIHP_CHECKED"] == "1") and lib.endswith(want)


_WORKLOAD = r"""
import hashlib, json, sys
import torch
from resihp.ops import _ext, check_device_errors
from resihp.ops import functional as fn
from resihp.ops.gemm import linear_wgrad
torch.manual_seed(0)
x = torch.randn(512, 256, device="cuda").bfloat16()
w = torch.randn(384, 256, device="cuda").bfloat16()
y = fn.linear(x, w)
dw = torch.zeros(384, 256, device="cuda")
linear_wgrad(y, x, out=dw, accumulate=True)
hq, hkv, d, seq = 4, 2, 128, 256
qkv = (0.5 * torch.randn(2 * seq, (hq + 2 * hkv) * d, device="cuda")).bfloat16().requires_grad_()
cs = fn.rope_table(seq, d, 10000.0, device="cuda")
o = fn.rope_attention(qkv.clone(), cs, seq, hq, hkv, d)
o.backward(torch.randn_like(o))
torch.cuda.synchronize()
check_device_errors(0)
digest = {n: hashlib.sha256(t.detach().float().cpu().numpy().tobytes()).hexdigest()
          for n, t in (("y", y), ("dw", dw), ("o", o), ("dqkv", qkv.grad))}
print(json.dumps({"lib": _ext._LIB, "digest": digest}))
"""


@pytest.mark.gpu
def test_checked_library_passes_its_checks_and_matches_bitwise():
    results = {}
    for flag in ("0", "1"):
        out = subprocess.run([sys.executable, "-c", _WORKLOAD], capture_output=True, text=True, cwd=ROOT,
                             env={**os.environ, "RESIHP_CHECKED": flag}, timeout=600)
        assert out.returncode == 0, out.stderr[-2000:]
        results[flag] = json.loads(out.stdout.strip().splitlines()[-1])
    assert results["1"]["lib"].endswith("_C_checked.so") and results["0"]["lib"].endswith("_C.so")
    assert results["1"]["digest"] == results["0"]["digest"]


_GROUPED_WORKLOAD = r"""
import hashlib, itertools, json
import torch
from resihp.ops import _ext, check_device_errors, grouped_dgrad, grouped_linear, grouped_wgrad
from resihp.ops import functional as fn
torch.manual_seed(0)
digest = {}

def keep(name, t):
    digest[name] = hashlib.sha256(t.detach().float().cpu().numpy().tobytes()).hexdigest()

# empty groups, groups cut at every remainder of a step and a tile, rows behind the last group, tiles
# past the matrices' edges; the last case is one whose CTA pairs keep step
for sizes, tail, n, k in (([3, 0, 4], 2, 72, 136), ([65, 63, 1, 0, 127, 129, 16, 15], 7, 200, 328), ([5] * 70, 0, 64, 40),
                          ([700, 1, 900, 257], 129, 1032, 520), ([3000, 1100], 100, 2568, 7176)):
    offsets = torch.tensor([0, *itertools.accumulate(sizes)], dtype=torch.int32, device="cuda")
    rows = sum(sizes) + tail
    x, dy = torch.randn(rows, k, device="cuda").bfloat16(), torch.randn(rows, n, device="cuda").bfloat16()
    w = torch.randn(len(sizes), n, k, device="cuda").bfloat16()
    acc = torch.randn(w.shape, device="cuda")
    name = f"{len(sizes)} {n} {k} "
    keep(name + "y", grouped_linear(x, w, offsets))
    keep(name + "dx", grouped_dgrad(dy, w, offsets))
    keep(name + "dw", grouped_wgrad(dy, x, offsets))
    keep(name + "accumulated", grouped_wgrad(dy, x, offsets, out=acc, accumulate=True))
    leaf = w.clone().requires_grad_()
    fn.grouped_linear(x, leaf, offsets).backward(dy)
    keep(name + "bf16", leaf.grad)
torch.cuda.synchronize()
check_device_errors(0)
print(json.dumps({"lib": _ext._LIB, "digest": digest}))
"""


@pytest.mark.gpu
def test_checked_library_passes_its_checks_of_grouped_products():
    results = {}
    for flag in ("0", "1"):
        out = subprocess.run([sys.executable, "-c", _GROUPED_WORKLOAD], capture_output=True, text=True, cwd=ROOT,
                             env={**os.environ, "RESIHP_CHECKED": flag}, timeout=600)
        assert out.returncode == 0, out.stderr[-2000:]
        results[flag] = json.loads(out.stdout.strip().splitlines()[-1])
    assert results["1"]["lib"].endswith("_C_checked.so") and results["0"]["lib"].endswith("_C.so")
    assert results["1"]["digest"] == results["0"]["digest"] and len(results["0"]["digest"]) == 25
