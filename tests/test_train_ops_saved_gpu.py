"""Saved tensors that the caller's hooks replace: the backward passes read them by the sizes, type and device they had."""
import pytest
import torch

from mlx_swift_lm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _calls():
    g = torch.Generator().manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=g).to(DEV).requires_grad_()  # noqa: E731
    x, d, v, e, g0, hb, w = n(4, 32), n(4, 32), n(32), n(32), n(4, 32), n(4, 32), n(40, 32)
    hb, w = (t.detach().bfloat16().requires_grad_() for t in (hb, w))
    t = torch.arange(4, device=DEV)
    return [([x, d, v, e], lambda: ops.block_norms(x, d, v, e)[1]), ([x, d], lambda: ops.block_norms(x, d)[0]),
            ([x, d, v, g0], lambda: ops.block_norms(x, d, v, gate=g0)[0]), ([hb, w], lambda: ops.linear_cross_entropy(hb, w, t))]


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("unpack", [lambda t: t.cpu(), lambda t: t[:1], lambda t: t.half(), lambda t: t.reshape(-1)[:0]])
def test_changed_ones_are_refused(which, unpack):
    leaves, call = _calls()[which]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        out = call()
    with pytest.raises(RuntimeError, match="came back changed"):
        torch.autograd.grad(out.sum(), leaves)


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("pack,unpack", [(lambda t: t.cpu(), lambda t: t.to(DEV)), (lambda t: t, lambda t: t.clone()),
                                         (lambda t: t, lambda t: torch.stack([t, t], -1)[..., 0])])
def test_equal_ones_give_the_same_gradients(which, pack, unpack):
    leaves, call = _calls()[which]
    want = torch.autograd.grad(call().sum(), leaves)
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        out = call()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out.sum(), leaves), want))


def test_a_storage_that_was_given_back():
    x = torch.randn(4, 32, device=DEV)
    x.untyped_storage().resize_(0)
    with pytest.raises(TypeError, match="without memory"):
        ops.dropout(x, 0.5, 1)
    with pytest.raises(TypeError, match="without memory"):
        ops.block_norms(torch.randn(4, 32, device=DEV), x)
