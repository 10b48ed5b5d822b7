"""Cross entropy of a linear head without its logits
(csrc/kernels/linear_ce.cu on CUDA, plain torch on CPU).

Parity: the loss of LoRATrain (MLXLLM/LoraTrain.swift:134-433), whose logits
are a full [tokens, vocabulary] tensor there.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from . import reference as ref
from ._args import rows2d, same_device
from .linear import num_sms

_lib.register_signatures({
    "b200_lce_saved_bytes": (_lib.i64, [_lib.i32, _lib.i32]),
    "b200_lce_forward_bytes": (_lib.i64, [_lib.i32, _lib.i32]),
    "b200_lce_backward_bytes": (_lib.i64, [_lib.i32, _lib.i32, _lib.i32, _lib.i32, _lib.i32]),
    "b200_lce_forward": (_lib.i32, [_lib.vp, _lib.i64, _lib.vp, _lib.i64, _lib.vp, _lib.i64, _lib.i32, _lib.i32,
                                    _lib.i32, _lib.i32, _lib.f32, _lib.vp, _lib.vp, _lib.vp, _lib.vp, _lib.i32,
                                    _lib.i32, _lib.vp]),
    "b200_lce_backward": (_lib.i32, [_lib.vp, _lib.vp, _lib.i64, _lib.vp, _lib.i64, _lib.i32, _lib.i32, _lib.i32,
                                     _lib.i32, _lib.i32, _lib.f32, _lib.i32, _lib.vp, _lib.vp, _lib.vp, _lib.i64,
                                     _lib.i32, _lib.vp]),
}, status_tags=("linear_ce",))

_TILE = 256  # columns of a tile; pieces of the vocabulary are whole tiles
# Bytes of one piece of the logits' gradient. Larger pieces mean fewer passes over the
# fp32 sums of dh; a piece is never narrower than MIN_PIECE columns.
PIECE_BYTES = 256 << 20
MIN_PIECE = 8192


def _aligned_head(w: torch.Tensor) -> torch.Tensor:
    """The head as TMA reads it (16-byte aligned rows of neighbouring columns):
    itself, or a copy in padded rows."""
    V, K = w.shape
    if (K == 1 or w.stride(1) == 1) and w.stride(0) % 8 == 0 and w.stride(0) >= K and w.data_ptr() % 16 == 0:
        return w
    out = torch.empty((V, (K + 7) // 8 * 8), dtype=w.dtype, device=w.device)[:, :K]
    out.copy_(w)
    return out


def _forward(h2, w, targets, softcap, ignore_index, reduction):
    """(losses or their total, what the backward pass needs)."""
    T, K = h2.shape
    V = w.shape[0]
    Kp = (K + 7) // 8 * 8
    dev = h2.device
    w = _aligned_head(w)
    L = _lib.lib()
    saved = torch.empty(L.b200_lce_saved_bytes(T, Kp), dtype=torch.uint8, device=dev)
    part = torch.empty(L.b200_lce_forward_bytes(T, V), dtype=torch.uint8, device=dev)
    loss = torch.empty(T, dtype=torch.float32, device=dev)
    total = None if reduction == "none" else torch.empty((), dtype=torch.float32, device=dev)
    rc = _lib.launch(L.b200_lce_forward, dev, h2.data_ptr(), h2.stride(0), w.data_ptr(), w.stride(0),
                     targets.data_ptr(), ignore_index, T, V, K, Kp, softcap, saved.data_ptr(), part.data_ptr(),
                     loss.data_ptr(), _lib.ptr(total), 1 if reduction == "mean" else 0, num_sms(dev))
    _lib.check(rc, f"linear_cross_entropy T={T} V={V} K={K}")
    _lib.count(3)
    return loss if total is None else total, saved


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h2, w, targets, softcap, ignore_index, reduction):
        out, saved = _forward(h2, w, targets, softcap, ignore_index, reduction)
        ctx.save_for_backward(w, saved)
        ctx.shape, ctx.softcap, ctx.mean = h2.shape, softcap, reduction == "mean"
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        w, saved = ctx.saved_tensors
        (T, K), (V, _), dev = ctx.shape, w.shape, w.device
        need_h, need_w = ctx.needs_input_grad[:2]
        Kp = (K + 7) // 8 * 8
        w2 = _aligned_head(w)
        piece = max(MIN_PIECE, PIECE_BYTES // (2 * T) // _TILE * _TILE)
        piece = min(piece, (V + _TILE - 1) // _TILE * _TILE)
        L, sms = _lib.lib(), num_sms(dev)
        scratch = torch.empty(L.b200_lce_backward_bytes(T, K, piece, 1 if need_h else 0, sms), dtype=torch.uint8,
                              device=dev)
        dh = torch.empty((T, K), dtype=torch.bfloat16, device=dev) if need_h else None
        dw = torch.empty((V, Kp), dtype=torch.bfloat16, device=dev)[:, :K] if need_w else None  # rows as TMA stores them
        g = dloss.reshape(-1)
        rc = _lib.launch(L.b200_lce_backward, dev, saved.data_ptr(), w2.data_ptr(), w2.stride(0), g.data_ptr(),
                         g.stride(0) if T > 1 and g.numel() == T else 0, 1 if ctx.mean else 0, T, V, K, Kp, ctx.softcap,
                         piece, scratch.data_ptr(), _lib.ptr(dh), _lib.ptr(dw), Kp, sms)
        _lib.check(rc, f"linear_cross_entropy backward T={T} V={V} K={K}")
        _lib.count(-(-V // piece) * (1 + need_h + need_w) + need_h)
        return dh, dw, None, None, None, None


def linear_cross_entropy(h: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, softcap: float = 0.0,
                         ignore_index: int = -100, reduction: str = "none") -> torch.Tensor:
    """Softmax cross entropy of the logits h @ w.T against `targets`, without
    forming them: fp32 losses, differentiable in h and w.

    h [..., K] and w [V, K] (bf16 on CUDA), targets [...] int64. `softcap` c > 0
    caps the logits as c tanh(z / c). Positions whose target is `ignore_index`
    have loss 0, take no part in any gradient and cost nothing (only the others
    are computed). `reduction`: "none" (a loss per position), "sum", or "mean"
    over the scored positions (0 where there are none). Any other target outside
    [0, V) gives a NaN loss and a status bit on CUDA, and raises on CPU.
    """
    if reduction not in ("none", "sum", "mean"):
        raise ValueError(f"linear_cross_entropy: reduction {reduction!r}")
    if h.dim() < 1 or w.dim() != 2 or w.shape[1] != h.shape[-1] or w.shape[0] < 1 or w.shape[1] < 1:
        raise ValueError(f"linear_cross_entropy: hidden rows {tuple(h.shape)}, head {tuple(w.shape)}")
    if targets.shape != h.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: targets {tuple(targets.shape)} for hidden rows {tuple(h.shape)}")
    if targets.dtype != torch.int64:
        raise TypeError(f"linear_cross_entropy: targets {targets.dtype}, int64 needed")
    if h.dtype != w.dtype or not h.is_floating_point():
        raise TypeError(f"linear_cross_entropy: hidden rows {h.dtype}, head {w.dtype}")
    softcap = float(softcap)
    if not 0.0 <= softcap < float("inf"):
        raise ValueError(f"linear_cross_entropy: softcap {softcap}")
    same_device("linear_cross_entropy", h, w, targets)
    T = targets.numel()
    if not h.is_cuda:
        return ref.linear_cross_entropy_ref(h, w, targets, softcap, ignore_index, reduction)
    if h.dtype != torch.bfloat16:
        raise TypeError(f"linear_cross_entropy: {h.dtype}; the CUDA kernels take bfloat16")
    if T == 0:
        zero = h.float().sum() + w[:0].float().sum()  # sums of nothing: both stay in the graph, with zero gradients
        return zero.expand(targets.shape) if reduction == "none" else zero
    h2, t1 = rows2d(h, h.shape[-1]), targets.reshape(-1).contiguous()
    if torch.is_grad_enabled() and (h.requires_grad or w.requires_grad):
        out = _LinearCrossEntropy.apply(h2, w, t1, softcap, int(ignore_index), reduction)
    else:
        out = _forward(h2, w, t1, softcap, int(ignore_index), reduction)[0]
    return out.reshape(targets.shape) if reduction == "none" else out
