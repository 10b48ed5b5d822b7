"""Dropout from a counter-based generator: the mask is a function of (seed,
offset, row, column), so the backward pass draws it again and nothing is stored
(csrc/kernels/dropout.cu on CUDA, the same stream in numpy on CPU).

Parity: LoRALinear's dropout before the A product (LoRA+Layers.swift:109).
"""
from __future__ import annotations

import torch

from . import _autograd, _lib
from . import reference as ref

_MASK64 = 0xFFFFFFFFFFFFFFFF


def dropout(x: torch.Tensor, p: float, seed: int, offset: int | torch.Tensor = 0,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """Inverted dropout of x [..., K] (+ `residual` of x's shape and dtype),
    differentiable in both. x is bf16, fp16 or fp32.

    The mask is a function of (seed, offset, row, column) alone: the same call
    gives the same mask whatever the dtype, strides or device, and each (seed,
    offset) pair gives its own. Rows are numbered over the leading dimensions.
    `offset` may be an int64 tensor of one element on x's device that the kernel
    reads, so that a captured graph draws a new mask whenever the tensor has
    moved on between replays. p is rounded to a multiple of 2^-16; kept elements
    are scaled by 1 / (1 - that). Dropped elements are 0 whatever they held (inf
    and NaN included). One rounding, after the residual is added.
    """
    if isinstance(offset, torch.Tensor):
        offset, offset_t = 0, offset
    else:
        offset, offset_t = int(offset) & _MASK64, None
    seed = int(seed) & _MASK64
    y = _autograd.for_device(x).dropout(x, p, seed, offset, offset_t, residual)
    if y is None:
        return ref.dropout_ref(x, p, seed, offset if offset_t is None else int(offset_t) & _MASK64, residual)
    _lib.count(1)
    return y
