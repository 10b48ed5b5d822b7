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


def module():
    """The module, loaded once. Calls on CPU tensors check their arguments and return None."""
    global _module
    if _module is None:
        path = glob.glob(os.path.join(os.path.dirname(_lib.LIB_PATH), "_b200torch*.so"))
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
    return cuda_module() if t.is_cuda else module()
