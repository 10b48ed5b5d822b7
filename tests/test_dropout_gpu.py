"""ops.dropout on the GPU: the mask equals the CPU stream's bit for bit in every
layout, gradients draw it again, graphs and streams."""
import pytest
import torch

from mlx_swift_lm_b200 import ops
from mlx_swift_lm_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rows(T, K, slack, start, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    buf = torch.randn(T, K + slack + start, generator=g).to(dtype).to(DEV)
    return buf[:, start:start + K]


def _check(y, x, keep, p, residual=None):
    s = ref.dropout_scale(ref.dropout_cut(p))
    want = torch.where(keep.to(DEV), x.double() * s, 0.0)
    mag = x.double().abs() * s
    if residual is not None:
        want = want + residual.double()
        mag = mag + residual.double().abs()
    # one rounding to the type, and at most three fp32 roundings (scale, product, sum). Below the type's
    # smallest normal number n the steps stay those at n, eps * n, so half a step is eps / 2 * max(|v|, n)
    fi = torch.finfo(x.dtype)
    tol = fi.eps / 2 * want.abs().clamp_min(fi.smallest_normal) + 3 * 2 ** -24 * mag
    assert ((y.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K", [(1, 1), (1, 7), (1, 8), (3, 9), (5, 255), (4, 256), (7, 257), (33, 1000), (300, 4096)])
@pytest.mark.parametrize("slack,start", [(0, 0), (8, 8), (3, 1)])
@pytest.mark.parametrize("with_res", [False, True])
def test_forward_and_backward(dtype, T, K, slack, start, with_res):
    p, seed, off = 0.3, 0x1234567890ABCDEF, (5 << 33) + 17
    x = _rows(T, K, slack, start, dtype).detach().requires_grad_()
    r = _rows(T, K, slack, start, dtype, 1).detach().requires_grad_() if with_res else None
    keep = ref.dropout_keep_ref(T, K, p, seed, off)
    y = ops.dropout(x, p, seed, off, residual=r)
    _check(y, x.detach(), keep, p, None if r is None else r.detach())
    dy = _rows(T, K, start, slack, dtype, 2)
    got = torch.autograd.grad(y, [x, r] if with_res else [x], dy)
    _check(got[0], dy, keep, p)
    if with_res:
        assert torch.equal(got[1], dy)
    assert torch.equal(ops.dropout(x.detach(), p, seed, off, residual=None if r is None else r.detach()), y)


def test_masked_places_hold_anything_and_extremes():
    T, K, p = 64, 512, 0.5
    keep = ref.dropout_keep_ref(T, K, p, 3, 0).to(DEV)
    x = torch.randn(T, K, device=DEV)
    bad = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float32).min], device=DEV)
    y = ops.dropout(torch.where(keep, x, bad.repeat(K // 4)), p, 3)
    assert torch.equal(y, ops.dropout(x, p, 3)) and (y[~keep] == 0).all()
    assert torch.equal(ops.dropout(x, 0.0, 3), x)
    assert torch.equal(ops.dropout(x, 1.0, 3), torch.zeros_like(x))
    for shape in ((0, 10), (3, 0), (0,)):
        assert ops.dropout(torch.empty(shape, device=DEV), 0.5, 5).shape == torch.Size(shape)


def test_layouts():
    x = torch.randn(6, 40, 24, device=DEV)
    want = ops.dropout(x, 0.4, 9)
    assert torch.equal(want.reshape(240, 24), ops.dropout(x.reshape(240, 24), 0.4, 9))
    assert torch.equal(ops.dropout(x.transpose(0, 1).contiguous().transpose(0, 1), 0.4, 9), want)
    t = torch.randn(24, 240, device=DEV).t()  # columns apart
    assert torch.equal(ops.dropout(t, 0.4, 9), ops.dropout(t.contiguous(), 0.4, 9))
    e = torch.randn(1, 24, device=DEV).expand(240, 24)  # one row for all, each with its own mask
    assert torch.equal(ops.dropout(e, 0.4, 9), ops.dropout(e.contiguous(), 0.4, 9))
    v = torch.randn(100, device=DEV)
    assert torch.equal(ops.dropout(v, 0.4, 9), ops.dropout(v[None], 0.4, 9)[0])


def test_gradient_of_an_expanded_gradient():
    x = torch.randn(9, 30, device=DEV, requires_grad=True)
    ops.dropout(x, 0.4, 2).sum().backward()
    keep = ref.dropout_keep_ref(9, 30, 0.4, 2).to(DEV)
    s = ref.dropout_scale(ref.dropout_cut(0.4))
    assert torch.allclose(x.grad, keep.float() * s, rtol=2 ** -22, atol=0)


def test_captured_graph_draws_a_new_mask_as_the_offset_moves():
    x = torch.randn(32, 320, device=DEV)
    off = torch.zeros(1, dtype=torch.int64, device=DEV)
    ops.dropout(x, 0.5, 4, off)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.dropout(x, 0.5, 4, off)
    for step in (0, 1, 1 << 35):
        off.fill_(step)
        g.replay()
        assert torch.equal(y, ops.dropout(x, 0.5, 4, step))


def test_backward_uses_the_offset_of_its_forward():
    x = torch.randn(16, 64, device=DEV, requires_grad=True)
    off = torch.full((1,), 3, dtype=torch.int64, device=DEV)
    y = ops.dropout(x, 0.5, 4, off)
    off.add_(1)
    dx, = torch.autograd.grad(y, [x], torch.ones_like(y))
    assert torch.equal(dx != 0, ref.dropout_keep_ref(16, 64, 0.5, 4, 3).to(DEV))


def test_side_stream():
    x = torch.randn(256, 4096, device=DEV)
    want = ops.dropout(x, 0.5, 4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = ops.dropout(x, 0.5, 4)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want)
