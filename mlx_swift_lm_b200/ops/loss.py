"""Cross entropy of a linear head without its logits
(csrc/kernels/linear_ce.cu on CUDA, plain torch on CPU).

Parity: the loss of LoRATrain (MLXLLM/LoraTrain.swift:134-433), whose logits
are a full [tokens, vocabulary] tensor there.
"""
from __future__ import annotations

import torch

from . import _autograd, _lib
from . import reference as ref

# Bytes of one piece of the logits' gradient. Larger pieces mean fewer passes over the
# fp32 sums of dh (4096 rows of a 151936 x 4096 head, both gradients: 64 MB 15.5 ms,
# 128 MB 15.2, 256 MB 15.0, 1 GB 14.7; frozen head, 2048 rows: 4.85, 4.70, 4.65, 4.60):
# four times the memory for 2 % is not taken. A piece is never narrower than MIN_PIECE columns.
PIECE_BYTES = 256 << 20
MIN_PIECE = 8192


def linear_cross_entropy(h: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, softcap: float = 0.0,
                         ignore_index: int = -100, reduction: str = "none") -> torch.Tensor:
    """Softmax cross entropy of the logits h @ w.T against `targets`, without
    forming them: fp32 losses, differentiable in h and w.

    h [..., K] and w [V, K] (bf16 on CUDA), targets [...] int64. `softcap` c > 0
    (2^-126 to 2^126) caps the logits as c tanh(z / c). Positions whose target is `ignore_index`
    have loss 0, take no part in any gradient and cost nothing (only the others
    are computed). `reduction`: "none" (a loss per position), "sum", or "mean"
    over the scored positions (0 where there are none). Any other target outside
    [0, V) gives a NaN loss and a status bit on CUDA, and raises on CPU.
    """
    out = _autograd.for_device(h).linear_cross_entropy(h, w, targets, softcap, ignore_index, reduction, PIECE_BYTES,
                                                       MIN_PIECE)
    if out is None:
        return ref.linear_cross_entropy_ref(h, w, targets, softcap, ignore_index, reduction)
    _lib.count(3)
    return out
