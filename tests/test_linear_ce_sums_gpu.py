"""ops.linear_cross_entropy: how the logits' sums are rounded, on operands for which tensor cores
that truncate would be off by much, by little, or not at all."""
import math

import pytest
import torch

from mlx_swift_lm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
T, V = 96, 3000


def _operands(kind, K):
    g = torch.Generator().manual_seed(K)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    w, t = n(V, K) * 1.3 / math.sqrt(K), torch.randint(0, V, (T,), generator=g)
    if kind == "one-hot":
        h = torch.zeros(T, K)
        h[torch.arange(T), torch.randint(0, K, (T,), generator=g)] = 1.0
        w = n(V, K) * 5
    elif kind == "eighths":  # every sum is a whole number of 64ths below 2^18 of them
        h, w = (torch.randint(-2, 3, s, generator=g).float() / 8 for s in ((T, K), (V, K)))
    elif kind == "positive":
        h, w = n(T, K).abs() * 3.2, n(V, K).abs() * 10 / K
    elif kind == "cancelling":
        a, b = n(T, K // 2), n(V, K // 2)
        h, w = torch.cat([a, -a + 0.02 * n(T, K // 2)], 1) * 8, torch.cat([b, b + 0.02 * n(V, K // 2)], 1) * 4 / math.sqrt(K)
    else:
        h = n(T, K)
    return h.bfloat16().to(DEV), w.bfloat16().to(DEV), t.to(DEV)


@pytest.mark.parametrize("K", [64, 512, 520, 1000, 4096, 8192])
@pytest.mark.parametrize("kind", ["one-hot", "eighths"])
def test_exact_sums_stay_exact(kind, K):
    h, w, t = _operands(kind, K)
    got = ops.linear_cross_entropy(h, w, t).double()
    z = h.double() @ w.double().t()
    want = torch.nn.functional.cross_entropy(z, t, reduction="none")
    # 2^-22 (32 + tiles / 8) for the exponentials and their sums, 2^-22 of the loss, and the exponents' own: a logit is scaled
    # to base 2 in fp32 with the largest subtracted, three roundings of it
    limit = 2 ** -22 * (32 + V / 2048 + want.abs()) + 3 * 2 ** -23 * z.abs().amax(1)
    assert ((got - want).abs() <= limit).all(), f"{((got - want).abs() / limit).max().item():.2f} of the tolerance"


@pytest.mark.parametrize("K", [64, 512, 520, 1000, 4096, 8192])
@pytest.mark.parametrize("kind", ["normal", "positive", "cancelling"])
def test_errors_do_not_grow_with_the_products_length(kind, K):
    h, w, t = _operands(kind, K)
    got = ops.linear_cross_entropy(h, w, t).double()
    hd, wd = h.double(), w.double()
    z = hd @ wd.t()
    want = torch.nn.functional.cross_entropy(z, t, reduction="none")
    # a logit: 512 / 16 steps of a chunk truncated, its K / 512 chunks rounded, the 16 products of a step, 2^-23 of the terms'
    # magnitudes each; two logits for a loss (the target's is a sum of K / 32 terms a lane, rounded, and 5 more)
    S = (hd.abs() @ wd.abs().t()).amax(1)
    limit = (32 + K / 512 + 16 + (K / 32 + 5) / 2) * 2 ** -23 * S + 2 ** -22 * (32 + V / 2048 + want.abs()) \
        + 3 * 2 ** -23 * z.abs().amax(1)
    assert ((got - want).abs() <= limit).all(), f"{((got - want).abs() / limit).max().item():.2f} of the tolerance"
    # and on average the truncation: half a step of what the sum had reached, half of it on the way, 32 times
    mean = (32 / 4 * 2 ** -23 * S.mean() if kind == "positive" else 32 / 4 * 2 ** -23 * z.abs().amax()) + 2 ** -22 * 4
    assert abs((got - want).mean()) <= 2 * mean
