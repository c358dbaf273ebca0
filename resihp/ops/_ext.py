"""Loader for the in-tree sm_100a extension ``resihp/_C.so``.

The bf16 CUDA path has no fallback: a missing or unloadable extension is an error
(``require()`` raises), never a silent switch to torch kernels. FP32 tensors (CPU, or
CUDA in a reference-semantics run) take the plain-torch FP32 path of each op, which is
what the CPU test tier and the reference-semantics runs use.
"""

from __future__ import annotations

import importlib.util
import os

_PKG = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
#: ``RESIHP_CHECKED=1`` loads the bounds-checked build of the same kernels instead.
CHECKED = os.environ.get("RESIHP_CHECKED", "0") == "1"
_NAME = "_C_checked" if CHECKED else "_C"
_LIB = os.path.join(_PKG, _NAME + ".so")
_module = None
_error: Exception | None = None


def _load():
    global _module, _error
    if _module is not None or _error is not None:
        return _module
    try:
        import torch  # noqa: F401  (libtorch must be loaded before the extension)

        spec = importlib.util.spec_from_file_location("resihp." + _NAME, _LIB)
        if spec is None or not os.path.exists(_LIB):
            raise ImportError(f"extension not built: {_LIB} (run python -m resihp.ops.build"
                              f"{' --checked' if CHECKED else ''})")
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        _module = module
    except Exception as exc:  # kept and re-raised by require()
        _error = exc
    return _module


# Kernels each extension entry point launches (for the benchmark's launch count).
KERNELS_PER_CALL = {
    "gemm": 1, "rmsnorm_fwd": 1, "rmsnorm_bwd": 2, "rope": 1, "swiglu_fwd": 1, "swiglu_bwd": 1,
    "adamw": 1, "embedding_fwd": 1, "embedding_bwd": 2, "xent_stats": 1, "xent_grad": 1,
    "attn_fwd": 1, "attn_bwd": 3, "ag_gemm": 1, "gemm_rs": 1, "dp_allreduce_adamw": 1, "reshard_gather": 1,
}


class _Counting:
    """Proxy over the extension module that counts kernel launches per entry point.

    Entry points whose backward passes run in C++ (dropout, the sparse MLP) are counted by the
    module itself: Python does not see every launch of theirs.
    """

    def __init__(self, module):
        self._module = module
        self._called = 0
        self._native = 0      # the module's count when counting began
        self._enabled = False

    @property
    def enabled(self) -> bool:
        return self._enabled

    @enabled.setter
    def enabled(self, on: bool) -> None:
        self.launches = self.launches  # what the module counted so far, folded in
        self._enabled = bool(on)

    @property
    def launches(self) -> int:
        native = self._module.native_launches() - self._native if self._enabled else 0
        return self._called + native

    @launches.setter
    def launches(self, value: int) -> None:
        self._called = value
        self._native = self._module.native_launches()

    def __getattr__(self, name):
        fn = getattr(self._module, name)
        per = KERNELS_PER_CALL.get(name)
        if per is None:
            return fn

        def counted(*args, **kwargs):
            if self._enabled:
                self._called += per
            return fn(*args, **kwargs)

        setattr(self, name, counted)  # looked up once
        return counted


_counting = None


def launch_counter() -> "_Counting":
    """The counting proxy; set ``.enabled`` and read ``.launches``."""
    require()
    return _counting


def available() -> bool:
    return _load() is not None


def require():
    """The loaded extension module; raises if it cannot be loaded."""
    global _counting
    module = _load()
    if module is None:
        raise RuntimeError(f"resihp CUDA extension unavailable: {_error}")
    if _counting is None:
        _counting = _Counting(module)
    return _counting


def library_path() -> str:
    return _LIB
