"""Dropout from a counter-based generator: the mask is a function of (seed,
offset, row, column), so the backward pass draws it again and nothing is stored
(csrc/kernels/dropout.cu on CUDA, the same stream in numpy on CPU).

Parity: LoRALinear's dropout before the A product (LoRA+Layers.swift:109).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from . import reference as ref
from ._args import ELEM, elem_code, rows2d, same_device
from .linear import num_sms

_lib.register_signatures({
    "b200_dropout": (_lib.i32, [_lib.vp, _lib.i64, _lib.vp, _lib.i64, _lib.vp, _lib.i64, _lib.i64, _lib.i32, _lib.i32,
                                _lib.u64, _lib.u64, _lib.vp, _lib.i32, _lib.f32, _lib.i32, _lib.vp]),
}, status_tags=("dropout",))


def _launch(x, p, seed, offset, residual):
    cut = ref.dropout_cut(p)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    if x.numel() == 0:
        return y
    K = x.shape[-1] if x.dim() else 1
    x2 = rows2d(x, K)
    r2 = None if residual is None else rows2d(residual, K)
    host_offset, dev_offset = (0, offset.data_ptr()) if isinstance(offset, torch.Tensor) else (offset, None)
    rc = _lib.launch(_lib.lib().b200_dropout, x.device, x2.data_ptr(), x2.stride(0),
                     None if r2 is None else r2.data_ptr(), 0 if r2 is None else r2.stride(0), y.data_ptr(), K,
                     x2.shape[0], K, ELEM[x.dtype], seed, host_offset, dev_offset, cut, ref.dropout_scale(cut),
                     num_sms(x.device))
    _lib.check(rc, "dropout")
    _lib.count(1)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.p, ctx.seed = p, seed
        # a device counter may have moved on by the time the gradient is taken: keep its value, not the tensor
        ctx.offset = offset.clone() if isinstance(offset, torch.Tensor) else offset
        return _launch(x, p, seed, ctx.offset, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = _launch(dy, ctx.p, ctx.seed, ctx.offset, None) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, seed: int, offset: int | torch.Tensor = 0,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """Inverted dropout of x [..., K] (+ `residual` of x's shape), differentiable
    in both.

    The mask is a function of (seed, offset, row, column) alone: the same call
    gives the same mask whatever the dtype, strides or device, and each (seed,
    offset) pair gives its own. Rows are numbered over the leading dimensions.
    `offset` may be an int64 CUDA tensor of one element that the kernel reads,
    so that a captured graph draws a new mask whenever the tensor has moved on
    between replays. p is rounded to a multiple of 2^-16; kept elements are
    scaled by 1 / (1 - that). Dropped elements are 0 whatever they held (inf
    and NaN included). One rounding, after the residual is added.
    """
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability {p} is not in [0, 1]")
    elem_code(x, "dropout")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"dropout: residual {tuple(residual.shape)} {residual.dtype} for x {tuple(x.shape)} {x.dtype}")
    if isinstance(offset, torch.Tensor):
        if offset.dtype != torch.int64 or offset.numel() != 1:
            raise ValueError("dropout: a tensor offset is one int64 element")
        same_device("dropout", x, residual, offset)
    else:
        same_device("dropout", x, residual)
        offset = int(offset) & 0xFFFFFFFFFFFFFFFF
    seed = int(seed) & 0xFFFFFFFFFFFFFFFF
    if not x.is_cuda:
        off = int(offset) & 0xFFFFFFFFFFFFFFFF
        return ref.dropout_ref(x, p, seed, off, residual)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, p, seed, offset)
    return _launch(x, p, seed, offset, residual)
