"""ops.dropout on CPU: the generator against published vectors, its mask's
rate and independence of layout, gradients, and what the op refuses."""
import numpy as np
import pytest
import torch

from mlx_swift_lm_b200 import ops
from mlx_swift_lm_b200.ops import reference as ref


def test_philox_matches_the_known_answers():
    # known-answer vectors of Philox-4x32-10 published with the generator (Salmon et al., SC'11)
    cases = [((0, 0, 0, 0), 0, (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
             ((0xffffffff,) * 4, 0xffffffffffffffff, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
             ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), 0x299f31d0a4093822,
              (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))]
    for counter, key, want in cases:
        got = ref.philox_4x32([np.array(c) for c in counter], key)
        assert tuple(int(w) for w in got) == want


def test_mask_rate_and_dependence():
    rows, K = 512, 1000
    for p in (0.05, 0.3, 0.9):
        keep = ref.dropout_keep_ref(rows, K, p, seed=7, offset=3)
        n, q = rows * K, 1 - ref.dropout_cut(p) / 65536
        # six standard deviations of a binomial count
        assert abs(keep.sum().item() - n * q) < 6 * (n * q * (1 - q)) ** 0.5
    a = ref.dropout_keep_ref(rows, K, 0.5, 7, 3)
    assert torch.equal(a[:100, :77], ref.dropout_keep_ref(100, 77, 0.5, 7, 3))  # row and column alone decide
    for seed, off in ((8, 3), (7, 4), (7 + (1 << 40), 3), (7, 3 + (1 << 40))):
        b = ref.dropout_keep_ref(rows, K, 0.5, seed, off)
        agree = (a == b).sum().item()
        assert abs(agree - rows * K / 2) < 6 * (rows * K / 4) ** 0.5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_values_and_gradient(dtype):
    x = torch.randn(5, 3, 37, dtype=dtype, requires_grad=True)
    r = torch.randn(5, 3, 37, dtype=dtype, requires_grad=True)
    y = ops.dropout(x, 0.25, seed=11, offset=5, residual=r)
    keep = ref.dropout_keep_ref(15, 37, 0.25, 11, 5).reshape(5, 3, 37)
    want = (torch.where(keep, x.double() / 0.75, 0.0) + r.double())
    # one rounding of the exact value, plus two fp32 roundings of the product and the sum
    # (half a step below the smallest normal number n is eps / 2 * n)
    fi = torch.finfo(dtype)
    tol = fi.eps / 2 * want.abs().clamp_min(fi.smallest_normal) + 3 * 2 ** -24 * (x.double().abs() / 0.75 + r.double().abs())
    assert ((y.double() - want).abs() <= tol).all()
    dy = torch.randn_like(y)
    dx, dr = torch.autograd.grad(y, [x, r], dy)
    assert torch.equal(dr, dy)
    want = torch.where(keep, dy.double() / 0.75, 0.0)
    assert ((dx.double() - want).abs() <= fi.eps * want.abs().clamp_min(fi.smallest_normal)).all()
    assert (dx[~keep] == 0).all()


def test_dropped_places_hold_anything():
    x = torch.randn(4, 64)
    keep = ref.dropout_keep_ref(4, 64, 0.5, 1, 0)
    x = torch.where(keep, x, torch.tensor([float("nan"), float("inf")]).repeat(32))
    y = ops.dropout(x, 0.5, 1)
    assert torch.isfinite(y).all() and (y[~keep] == 0).all()


def test_edges():
    x = torch.randn(3, 10)
    assert torch.equal(ops.dropout(x, 0.0, 5), x)
    assert torch.equal(ops.dropout(x, 1.0, 5), torch.zeros_like(x))
    assert torch.equal(ops.dropout(x, 1.0, 5, residual=x), x)
    for shape in ((0, 10), (3, 0), (0,)):
        assert ops.dropout(torch.empty(shape), 0.5, 5).shape == torch.Size(shape)
    assert torch.equal(ops.dropout(x, 0.5, 5, torch.tensor([9])), ops.dropout(x, 0.5, 5, 9))
    assert torch.equal(ops.dropout(x, 0.5, -1), ops.dropout(x, 0.5, (1 << 64) - 1))


def test_refusals():
    x = torch.randn(3, 10)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            ops.dropout(x, p, 0)
    with pytest.raises(TypeError):
        ops.dropout(x.double(), 0.5, 0)
    with pytest.raises(ValueError):
        ops.dropout(x, 0.5, 0, residual=torch.randn(3, 9))
    with pytest.raises(ValueError):
        ops.dropout(x, 0.5, 0, residual=torch.randn(3, 10).half())
    with pytest.raises(ValueError):
        ops.dropout(x, 0.5, 0, torch.tensor([1, 2]))
    with pytest.raises(ValueError):
        ops.dropout(x, 0.5, 0, torch.tensor([1], dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.dropout(x, 0.5, 0, residual=torch.empty(3, 10, device="meta"))
