"""Lazily negated views (what complex numbers' .conj().imag are) count as the values they stand for on CUDA."""
import pytest
import torch

from mlx_swift_lm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _calls():
    """(tensor, call of it) for each input of each operator."""
    x, d, v = torch.randn(4, 32, device=DEV), torch.randn(4, 32, device=DEV), torch.randn(32, device=DEV)
    hb, w = x.bfloat16(), torch.randn(40, 32, device=DEV).bfloat16()
    t = torch.arange(4, device=DEV)
    return [(x, lambda a: ops.dropout(a, 0.5, 1)), (x, lambda a: ops.dropout(d, 0.5, 1, residual=a)),
            (torch.ones(1, dtype=torch.int64, device=DEV), lambda a: ops.dropout(d, 0.5, 1, offset=a)),
            (x, lambda a: ops.block_norms(a, d, v, v)[1]), (d, lambda a: ops.block_norms(x, a, v, v)[1]),
            (v, lambda a: ops.block_norms(x, d, a, v)[1]), (v, lambda a: ops.block_norms(x, d, v, a)[1]),
            (v, lambda a: ops.block_norms(x, d, v, v, gate=a)[1]), (x, lambda a: ops.block_norms(x, d, v, v, gate=a)[1]),
            (hb, lambda a: ops.linear_cross_entropy(a, w, t)), (w, lambda a: ops.linear_cross_entropy(hb, a, t)),
            (-t, lambda a: ops.linear_cross_entropy(hb, w, a))]


@pytest.mark.parametrize("which", range(12))
def test_inputs(which):
    x, call = _calls()[which]
    v = torch._neg_view(x)
    assert v.is_neg()
    want = call(-x)
    assert torch.equal(call(v), want)
    if x.is_floating_point():  # and through the saved tensors
        grads = []
        for a in (torch._neg_view(x.detach().requires_grad_()), (-x).requires_grad_()):
            leaf = a.detach().requires_grad_()
            grads.append(torch.autograd.grad(call(leaf).sum(), leaf)[0])
        assert torch.equal(*grads)


@pytest.mark.parametrize("which", [0, 3, 4, 9, 10])
def test_gradients_that_come_in(which):
    x, call = _calls()[which]
    x.requires_grad_()
    out = call(x)
    dy = torch.randn_like(out)
    got, = torch.autograd.grad(out, x, torch._neg_view(dy), retain_graph=True)
    want, = torch.autograd.grad(out, x, -dy)
    assert torch.equal(got, want)


def test_in_place():
    x, d, v = torch.randn(4, 32, device=DEV), torch.randn(4, 32, device=DEV), torch.ones(32, device=DEV)
    with pytest.raises(ValueError, match="negated"):
        ops.block_norms(torch._neg_view(x), d, v, inplace=True)
    want = ops.block_norms(x, -d, v)[0]
    assert torch.equal(ops.block_norms(x, torch._neg_view(d), v, inplace=True)[0], want)
