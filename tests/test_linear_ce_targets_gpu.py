"""ops.linear_cross_entropy: the targets' entries of G reach dW unrounded, however many rows are scored."""
import math

import pytest
import torch

from mlx_swift_lm_b200 import ops
from mlx_swift_lm_b200.ops import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _targets(kind, T, V, g):
    if kind == "distinct":
        return torch.randperm(V, generator=g)[:T]
    if kind == "one":
        return torch.full((T,), V - 1)
    if kind == "runs":  # a frequent target in a stretch, others around it
        t = torch.randint(0, V, (T,), generator=g)
        t[T // 4:T // 2] = 3
        return t
    t = torch.randint(0, max(1, V // 50), (T,), generator=g)  # few different ones
    t[torch.rand(T, generator=g) < 0.3] = -100
    return t


@pytest.mark.parametrize("kind", ["distinct", "one", "runs", "few"])
@pytest.mark.parametrize("T,V,K,cap", [(65, 300, 64, 0.0), (130, 2000, 100, 5.0), (1000, 5000, 264, 0.0), (700, 1500, 2056, 0.0),
                                       (2100, 2500, 72, 0.0)])
def test_rows_of_targets(T, V, K, cap, kind):
    g = torch.Generator().manual_seed(T + V)
    w = (torch.randn(V, K, generator=g) * 1.3 / math.sqrt(K)).bfloat16().to(DEV).requires_grad_()
    h = torch.randn(T, K, generator=g).bfloat16().to(DEV)
    t = _targets(kind, T, V, g).to(DEV)
    weights = (torch.rand(T, generator=g) + 0.5).to(DEV)
    dw, = torch.autograd.grad(ops.linear_cross_entropy(h, w, t, softcap=cap), [w], weights)
    keep = t != -100
    hd, y, wts = h.double()[keep], t[keep], weights.double()[keep]
    n = y.numel()
    u = hd @ w.detach().double().t()
    z = cap * torch.tanh(u / cap) if cap else u
    slope = 1 - (z / cap) ** 2 if cap else torch.ones_like(u)
    p = torch.softmax(z, 1)
    G = p.clone()
    G[torch.arange(n, device=DEV), y] -= 1
    G *= slope * wts[:, None]
    want = G.t() @ hd
    rows = torch.unique(y)
    others = G.abs()
    others[torch.arange(n, device=DEV), y] = 0
    half_step = torch.finfo(torch.bfloat16).eps / 2
    # an entry's exponent: two logits' errors, (K / 16 + 16) 2^-23 of their terms each, the sums' 2^-22 (32 + tiles / 8) and,
    # with a cap, its 2^-20; the target's entry p - 1 shares that error of p. The contraction adds (n / 16 + 80) 2^-23.
    ex = 2 * (K / 16 + 16) * 2 ** -23 * (hd.abs() @ w.detach().double().abs().t()).amax(1) + 2 ** -22 * (32 + V / 2048) \
        + (8 * 2 ** -20 * cap if cap else 0.0)
    entry = half_step * others + (ex * wts)[:, None] * p * slope + 2 ** -20 * wts[:, None] * (p + (G != 0)) * (cap > 0)
    off = (entry.t() @ hd.abs() + (n / 16 + 80) * 2 ** -23 * (G.abs().t() @ hd.abs()))[rows]
    limit = off + half_step * (want[rows].abs() + off)
    err = (dw.double() - want)[rows].abs()
    assert (err <= limit).all(), f"{(err / limit).max().item():.2f} of the tolerance"
    assert _lib.read_status()["linear_ce"] == 0


def test_repeats_bit_for_bit():
    g = torch.Generator().manual_seed(0)
    w = torch.randn(900, 520, generator=g).bfloat16().to(DEV).requires_grad_()
    h = torch.randn(3000, 520, generator=g).bfloat16().to(DEV)
    t = _targets("few", 3000, 900, g).to(DEV)
    runs = [torch.autograd.grad(ops.linear_cross_entropy(h, w, t, reduction="mean"), w)[0] for _ in range(3)]
    assert all(torch.equal(r, runs[0]) for r in runs)


def test_a_target_out_of_range_among_many_rows():
    g = torch.Generator().manual_seed(0)
    w = torch.randn(400, 64, generator=g).bfloat16().to(DEV).requires_grad_()
    h = torch.randn(200, 64, generator=g).bfloat16().to(DEV)
    t = torch.randint(0, 400, (200,), generator=g).to(DEV)
    t[50] = 400
    loss = ops.linear_cross_entropy(h, w, t)
    weights = torch.ones(200, device=DEV)
    torch.autograd.grad(loss, w, weights)  # NaN, as the loss is
    assert loss[50].isnan() and loss.isnan().sum() == 1 and _lib.read_status()["linear_ce"] == 8
