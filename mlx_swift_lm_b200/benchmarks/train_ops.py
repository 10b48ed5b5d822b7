"""Times of the training operators (CUDA events, inputs larger than L2).

    python -m mlx_swift_lm_b200.benchmarks.train_ops --op ce --tokens 4096 --vocab 151936 --hidden 4096
    python -m mlx_swift_lm_b200.benchmarks.train_ops --op dropout --tokens 8192 --hidden 4096
    python -m mlx_swift_lm_b200.benchmarks.train_ops --op norms --tokens 8192 --hidden 4096
"""
from __future__ import annotations

import argparse

import torch

from .. import ops


def _time(f, reps: int) -> float:
    """Microseconds a call, the median of `reps` after three untimed ones."""
    for _ in range(3):
        f()
    out = []
    for _ in range(reps):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        out.append(a.elapsed_time(b) * 1e3)
    return sorted(out)[len(out) // 2]


def main(argv=None):
    p = argparse.ArgumentParser()
    p.add_argument("--op", choices=("ce", "dropout", "norms"), required=True)
    p.add_argument("--tokens", type=int, default=4096)
    p.add_argument("--hidden", type=int, default=4096)
    p.add_argument("--vocab", type=int, default=151936)
    p.add_argument("--frozen-head", action="store_true")
    p.add_argument("--reps", type=int, default=10)
    a = p.parse_args(argv)
    T, H, V = a.tokens, a.hidden, a.vocab
    rows = lambda: torch.randn(T, H, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    x = rows().requires_grad_()
    dy = rows()
    if a.op == "ce":
        w = (torch.randn(V, H, device="cuda", dtype=torch.bfloat16) / H ** 0.5).requires_grad_(not a.frozen_head)
        t = torch.randint(0, V, (T,), device="cuda")
        leaves = [x] if a.frozen_head else [x, w]
        us = _time(lambda: torch.autograd.grad(ops.linear_cross_entropy(x, w, t, reduction="mean"), leaves), a.reps)
        flops = 2.0 * T * V * H * (1 + len(leaves))
        print(f"linear_cross_entropy T={T} V={V} K={H} {len(leaves)} gradient(s): {us:.0f} us, "
              f"{flops / us / 1e6:.0f} TFLOP/s of the operator's own products")
        return
    if a.op == "dropout":
        us = _time(lambda: torch.autograd.grad(ops.dropout(x, 0.1, 1), x, dy), a.reps)
        moved = 4 * 2.0 * T * H
    else:
        d, w = rows().requires_grad_(), torch.ones(H, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        us = _time(lambda: torch.autograd.grad(ops.block_norms(x, d, w, w), [x, d, w], [dy, dy]), a.reps)
        moved = 10 * 2.0 * T * H
    print(f"{a.op} {T} x {H} bf16 forward + backward: {us:.1f} us, {moved / us / 1e6:.2f} TB/s")


if __name__ == "__main__":
    main()
