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
