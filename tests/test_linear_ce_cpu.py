"""ops.linear_cross_entropy on CPU: the definition in 64 bits, gradients against
differences, ignored rows, and what the op refuses."""
import math

import pytest
import torch

from mlx_swift_lm_b200 import ops


def _definition(h, w, t, cap, ignore):
    z = h @ w.t()
    if cap:
        z = cap * torch.tanh(z / cap)
    keep = t != ignore
    lse = torch.logsumexp(z, 1)
    return torch.where(keep, lse - z.gather(1, t.clamp_min(0)[:, None])[:, 0], torch.zeros_like(lse)), keep.sum()


def _inputs(T, V, K, seed=0, ignored=0.3):
    g = torch.Generator().manual_seed(seed)
    h, w = torch.randn(T, K, generator=g), torch.randn(V, K, generator=g) / math.sqrt(K)
    t = torch.randint(0, V, (T,), generator=g)
    t[torch.rand(T, generator=g) < ignored] = -100
    return h, w, t


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("cap", [0.0, 2.0])
@pytest.mark.parametrize("T,V,K", [(1, 2, 1), (7, 33, 5), (20, 300, 16)])
def test_definition_and_gradients(reduction, cap, T, V, K):
    h, w, t = _inputs(T, V, K)
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    out = ops.linear_cross_entropy(a, b, t, softcap=cap, reduction=reduction)
    hd, wd = h.double().requires_grad_(), w.double().requires_grad_()
    each, n = _definition(hd, wd, t, cap, -100)
    want = {"none": each, "sum": each.sum(), "mean": each.sum() / n.clamp_min(1)}[reduction]
    assert out.dtype == torch.float32 and out.shape == want.shape
    # fp32 sums of up to 300 terms of order one
    assert torch.allclose(out.double(), want, rtol=1e-5, atol=1e-5)
    cot = torch.rand(out.shape, generator=torch.Generator().manual_seed(1))
    ga = torch.autograd.grad(out, [a, b], cot)
    gd = torch.autograd.grad(want, [hd, wd], cot.double())
    for x, y in zip(ga, gd):
        assert torch.allclose(x.double(), y, rtol=1e-4, atol=2e-5)
    # the 64-bit gradient against central differences along a random direction
    dh, dw = torch.randn_like(hd), torch.randn_like(wd)
    e = 1e-5

    def value(s):
        v, _ = _definition(h.double() + s * e * dh, w.double() + s * e * dw, t, cap, -100)
        v = {"none": v, "sum": v.sum(), "mean": v.sum() / n.clamp_min(1)}[reduction]
        return (v * cot.double()).sum()

    slope = (value(1) - value(-1)) / (2 * e)
    along = (gd[0] * dh).sum() + (gd[1] * dw).sum()
    assert abs(slope - along) <= 1e-6 * (1 + abs(along))


def test_ignored_rows_hold_anything():
    h, w, t = _inputs(12, 50, 8)
    t[:] = torch.arange(12)
    t[3:6] = 7
    clean = h.clone()
    for bad in (float("nan"), float("inf"), torch.finfo(torch.float32).min):
        h[3:6] = bad
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        loss = ops.linear_cross_entropy(a, b, t, ignore_index=7, reduction="sum")
        loss.backward()
        c, d = clean.clone().requires_grad_(), w.clone().requires_grad_()
        want = ops.linear_cross_entropy(c, d, t, ignore_index=7, reduction="sum")
        want.backward()
        assert loss == want and torch.equal(b.grad, d.grad) and torch.equal(a.grad, c.grad)
        assert (a.grad[3:6] == 0).all()


def test_nothing_scored_and_no_rows():
    h, w, t = _inputs(4, 10, 8)
    t[:] = -100
    for reduction in ("none", "sum", "mean"):
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        out = ops.linear_cross_entropy(a, b, t, reduction=reduction)
        assert (out == 0).all()
        out.sum().backward()
        assert (a.grad == 0).all() and (b.grad == 0).all()
        assert ops.linear_cross_entropy(h[:0], w, t[:0], reduction=reduction).numel() == (reduction != "none")


def test_batched_shape():
    h, w, t = _inputs(12, 10, 8)
    a = ops.linear_cross_entropy(h.reshape(3, 4, 8), w, t.reshape(3, 4))
    assert torch.equal(a.reshape(-1), ops.linear_cross_entropy(h, w, t))


def test_refusals():
    h, w, t = _inputs(4, 10, 8)
    for args, kw in [((h, w[:, :4], t), {}), ((h, w, t[:3]), {}), ((h, w[0], t), {}), ((h, w[:0], t), {}),
                     ((h, w, t), dict(reduction="max")), ((h, w, t), dict(softcap=-1.0)),
                     ((h, w, t), dict(softcap=float("nan"))), ((h, w.to("meta"), t), {})]:
        with pytest.raises(ValueError):
            ops.linear_cross_entropy(*args, **kw)
    with pytest.raises(TypeError):
        ops.linear_cross_entropy(h, w.bfloat16(), t)
    with pytest.raises(TypeError):
        ops.linear_cross_entropy(h, w, t.int())
    with pytest.raises((IndexError, RuntimeError)):
        ops.linear_cross_entropy(h, w, torch.full((4,), 10))
