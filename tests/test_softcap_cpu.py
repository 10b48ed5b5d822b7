"""The softcap of ops.linear_cross_entropy: the range it may have."""
import pytest
import torch

from mlx_swift_lm_b200 import ops


def _inputs():
    g = torch.Generator().manual_seed(0)
    return torch.randn(4, 8, generator=g), torch.randn(10, 8, generator=g), torch.tensor([0, 3, 9, -100])


@pytest.mark.parametrize("cap", [1e39, 1e38, 1e-39, 1e-46, 1e300, 5e-324, float("inf"), float("nan"), -2.0])
def test_caps_that_32_bits_do_not_hold(cap):
    with pytest.raises(ValueError, match="softcap"):
        ops.linear_cross_entropy(*_inputs(), softcap=cap)


@pytest.mark.parametrize("cap", [2.0 ** 126, 2.0 ** -126, 1e30])
def test_the_ends_of_the_range(cap):
    h, w, t = _inputs()
    got = ops.linear_cross_entropy(h, w, t, softcap=cap)
    want = ops.linear_cross_entropy(h, w * (cap > 1), t)  # far above the logits: none; far below: all logits 0
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)  # fp32 sums of ten terms of order one
