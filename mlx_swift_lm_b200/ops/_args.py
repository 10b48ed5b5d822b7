"""Argument checks and row views shared by the elementwise training ops."""
from __future__ import annotations

import torch

# element types the row kernels know (ElemType in csrc/include/b200_elem.cuh)
ELEM = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def elem_code(t: torch.Tensor, what: str) -> int:
    code = ELEM.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be bfloat16, float16 or float32, not {t.dtype}")
    return code


def same_device(what: str, first: torch.Tensor, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"{what}: tensors on {first.device} and {t.device}")


def rows2d(t: torch.Tensor, width: int) -> torch.Tensor:
    """`t` [..., width] as [rows, width] with neighbouring columns: a view where
    the strides allow it, else a copy."""
    t = t if t.dim() == 2 else t.reshape(-1, width)
    return t if width <= 1 or t.stride(1) == 1 else t.contiguous()
