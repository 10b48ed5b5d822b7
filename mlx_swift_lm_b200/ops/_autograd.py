"""Loader of the autograd module of the training operators (csrc/torch): argument
checks and differentiable entry points in C++ over the kernel library's C entry
points, whose addresses it is given here."""
from __future__ import annotations

import ctypes as C
import glob
import importlib.util
import os

from . import _lib

_ENTRIES = ("b200_dropout", "b200_block_norms", "b200_block_norms_bwd", "b200_block_norms_max_width",
            "b200_block_norms_bwd_grid", "b200_lce_saved_bytes", "b200_lce_forward_bytes", "b200_lce_backward_bytes",
            "b200_lce_forward", "b200_lce_backward")
_module = None
_bound = False
_lib.register_signatures({}, status_tags=("dropout", "block_norms", "linear_ce"))


class _Unbuilt:
    """Stands in for the module on CPU where nothing has been built: the oracles answer,
    and refuse what they cannot compute."""

    @staticmethod
    def dropout(x, p, *rest):
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability {p} is not in [0, 1]")

    @staticmethod
    def block_norms(x, delta, *rest):
        if delta.shape != x.shape:
            raise ValueError(f"block_norms: delta {tuple(delta.shape)} for x {tuple(x.shape)}")

    @staticmethod
    def linear_cross_entropy(h, w, targets, softcap, ignore_index, reduction, *rest):
        if reduction not in ("none", "sum", "mean"):
            raise ValueError(f"linear_cross_entropy: reduction '{reduction}'")


def _path():
    return glob.glob(os.path.join(os.path.dirname(_lib.LIB_PATH), "_b200torch*.so"))


def module():
    """The module, loaded once. Calls on CPU tensors check their arguments and return None."""
    global _module
    if _module is None:
        path = _path()
        if not path:
            raise _lib.KernelLibraryMissing("_b200torch is missing: build it with `python mlx_swift_lm_b200/_build.py`")
        spec = importlib.util.spec_from_file_location("_b200torch", path[0])
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        mod.raise_as(_lib.KernelError)
        _module = mod
    return _module


def cuda_module():
    """The module with the kernel library's entry points in place."""
    global _bound
    m = module()
    if not _bound:
        lib = _lib.lib()
        m.bind({n: C.cast(getattr(lib, n), C.c_void_p).value for n in _ENTRIES})
        _bound = True
    return m


def for_device(t):
    if t.is_cuda:
        return cuda_module()
    return module() if _module is not None or _path() else _Unbuilt
