"""The softcap of ops.linear_cross_entropy over the range it may have, on the GPU."""
import math

import pytest
import torch

from mlx_swift_lm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("cap", [30.0, 250.0, 260.0, 1e3, 1e4, 1e6, 1e12, 1e30])
@pytest.mark.parametrize("T,V,K", [(5, 300, 64), (130, 3000, 256)])
def test_gradients_of_logits_far_below_the_cap(T, V, K, cap):
    """Logits of up to about 20: a cap far above them changes little, and its error must not grow with it."""
    g = torch.Generator().manual_seed(0)
    w = (torch.randn(V, K, generator=g) * 4 / math.sqrt(K)).bfloat16().to(DEV).requires_grad_()
    h = torch.randn(T, K, generator=g).bfloat16().to(DEV).requires_grad_()
    t = torch.randint(0, V, (T,), generator=g).to(DEV)
    loss = ops.linear_cross_entropy(h, w, t, softcap=cap)
    got = torch.autograd.grad(loss.sum(), [h, w])
    hd, wd = h.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    want = torch.nn.functional.cross_entropy(cap * torch.tanh(hd @ wd.t() / cap), t, reduction="none")
    # a logit's error: (K / 16 + 16) 2^-23 of its terms (truncation counted as a whole step) and 8 roundings of itself;
    # the loss has two logits' and 2^-22 (32 + tiles / 8) of the sums
    S = (hd.detach().abs() @ wd.detach().abs().t()).amax(1)
    ez = (K / 16 + 16 + 8) * 2 ** -23 * S
    assert ((loss.detach().double() - want.detach()).abs() <= 2 * ez + 2 ** -22 * (32 + V / 2048 + want.detach())).all()
    for a, b in zip(got, torch.autograd.grad(want.sum(), [hd, wd])):
        # G's entries are off by their bf16 rounding and the exponent's error (2^-14 of the fast tanh and ez), the
        # outputs by theirs: 2^-8 each at most, in norm
        assert (a.double() - b).norm() <= (2 * 2 ** -8 + 2 ** -13 + 2 * ez.amax()) * b.norm()


@pytest.mark.parametrize("cap", [2.0 ** 126, 2.0 ** -126])
def test_the_ends_of_the_range(cap):
    g = torch.Generator().manual_seed(0)
    h, w = torch.randn(5, 64, generator=g).bfloat16().to(DEV), torch.randn(300, 64, generator=g).bfloat16().to(DEV)
    t = torch.tensor([0, 3, 299, -100, 7], device=DEV)
    with pytest.raises(ValueError, match="softcap"):
        ops.linear_cross_entropy(h, w, t, softcap=cap * cap)
    a, b = h.requires_grad_(), w.requires_grad_()
    got = ops.linear_cross_entropy(a, b, t, softcap=cap)
    grads = torch.autograd.grad(got.sum(), [a, b])
    if cap < 1:  # all logits 0, and tanh flat
        want = torch.where(t == -100, 0.0, math.log(300))
        assert torch.allclose(got, want, rtol=1e-6) and all((x == 0).all() for x in grads)
    else:
        # none: logits of up to 40, whose rounding z = c tanh(u / c) adds some 2^-22 of each
        want = ops.linear_cross_entropy(a, b, t)
        assert torch.allclose(got, want, rtol=1e-5, atol=4e-5)
        for x, y in zip(grads, torch.autograd.grad(want.sum(), [a, b])):
            assert (x - y).norm() <= 2 * 2 ** -8 * y.norm()
