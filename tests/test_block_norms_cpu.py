"""ops.block_norms on CPU: the formula in 64 bits, gradients against
differences, and what the op refuses."""
import pytest
import torch

from mlx_swift_lm_b200 import ops


def _formula(x, delta, post, pre, gate, scale, eps, one=0.0):
    def rms(v, w):
        return v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * (w + one)

    u = delta if post is None else rms(delta, post)
    y = x + scale * (u if gate is None else u * gate)
    return y, None if pre is None else rms(y, pre)


def _inputs(T, H, gate, seed=0):
    g = torch.Generator().manual_seed(seed)
    shape = {"": None, "channel": (H,), "row": (T, 1), "element": (T, H)}[gate]
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return n(T, H), n(T, H), 1 + 0.1 * n(H), 1 + 0.1 * n(H), None if shape is None else n(*shape)


@pytest.mark.parametrize("gate", ["", "channel", "row", "element"])
@pytest.mark.parametrize("use_post,use_pre", [(True, True), (True, False), (False, True), (False, False)])
def test_formula_and_gradients(gate, use_post, use_pre):
    T, H, scale, eps = 5, 19, 0.3, 1e-5
    x, delta, post, pre, gt = _inputs(T, H, gate)
    ins = [x, delta, post if use_post else None, pre if use_pre else None, gt]
    leaves = [None if t is None else t.clone().requires_grad_() for t in ins]
    y, h = ops.block_norms(leaves[0], leaves[1], leaves[2], leaves[3], eps, leaves[4], scale)
    dbl = [None if t is None else t.double().requires_grad_() for t in ins]
    yd, hd = _formula(*dbl, scale, eps)
    outs, outd = [y] + ([h] if use_pre else []), [yd] + ([hd] if use_pre else [])
    for a, b in zip(outs, outd):  # 2^-24 a rounding, fewer than 32 of them, on values of order one
        assert torch.allclose(a.double(), b, rtol=32 * 2 ** -24, atol=32 * 2 ** -24)
    cot = [torch.randn_like(o) for o in outs]
    ga = torch.autograd.grad(outs, [t for t in leaves if t is not None], cot)
    gd = torch.autograd.grad(outd, [t for t in dbl if t is not None], [c.double() for c in cot])
    for a, b in zip(ga, gd):  # sums of up to 19 terms of order one
        assert torch.allclose(a.double(), b, rtol=1e-5, atol=64 * 2 ** -24 * 8)
    # and the 64-bit formula's gradients against central differences along a random direction
    dirs = [None if t is None else torch.randn_like(t) for t in dbl]
    e = 1e-5

    def value(sign):
        moved = [None if t is None else t.detach() + sign * e * d for t, d in zip(dbl, dirs)]
        o = _formula(*moved, scale, eps)
        return sum((c.double() * v).sum() for c, v in zip(cot, o))

    slope = (value(1) - value(-1)) / (2 * e)
    along = sum((g * d).sum() for g, d in zip(gd, [d for d in dirs if d is not None]))
    assert abs(slope - along) <= 1e-6 * (1 + abs(along))  # truncation e^2 and 1e-16 / e


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset_one", [False, True])
def test_round_branch_is_norm_then_add_norm(dtype, offset_one):
    x, delta, post, pre, _ = (None if t is None else t.to(dtype) for t in _inputs(7, 64, ""))
    x2 = x.clone()
    want = ops.add_rmsnorm(x2, ops.rmsnorm(delta, post, 1e-6, offset_one), pre, 1e-6, offset_one=offset_one)
    y, h = ops.block_norms(x, delta, post, pre, 1e-6, offset_one=offset_one, round_branch=True, inplace=True)
    assert y is x and torch.equal(x, x2) and torch.equal(h, want)


def test_refusals():
    x, delta, post, pre, _ = _inputs(4, 16, "")
    bad = [dict(delta=delta[:3]), dict(delta=delta.half()), dict(post_w=post[:8]), dict(pre_w=pre[None]),
           dict(gate=torch.randn(4)), dict(gate=torch.randn(4, 8)), dict(gate=torch.randn(16, device="meta"))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.block_norms(x, kw.pop("delta", delta), **kw)
    with pytest.raises(TypeError):
        ops.block_norms(x.double(), delta.double())
    with pytest.raises(TypeError):
        ops.block_norms(x, delta, gate=torch.randn(16).half())
    with pytest.raises(TypeError):
        ops.block_norms(x, delta, post, pre.half())
    with pytest.raises(ValueError):
        ops.block_norms(x, delta, post.requires_grad_(), inplace=True)
    post.requires_grad_(False)
    with pytest.raises(ValueError):
        ops.block_norms(torch.randn(1, 16).expand(4, 16), delta, post, inplace=True)
    with pytest.raises(ValueError):
        ops.block_norms(torch.empty(4, 0), torch.empty(4, 0))
