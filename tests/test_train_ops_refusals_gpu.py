"""Forms of autograd that the training operators' kernels do not carry are refused on CUDA, where
a result without them would pass for one."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from mlx_swift_lm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _calls():
    """(tensor, call of it) for each floating input of each operator."""
    x, d, v = torch.randn(4, 32, device=DEV), torch.randn(4, 32, device=DEV), torch.randn(32, device=DEV)
    hb, w = x.bfloat16(), torch.randn(40, 32, device=DEV).bfloat16()
    t = torch.arange(4, device=DEV)
    return [(x, lambda a: ops.dropout(a, 0.5, 1)), (x, lambda a: ops.dropout(d, 0.5, 1, residual=a)),
            (x, lambda a: ops.block_norms(a, d, v, v)[1]), (d, lambda a: ops.block_norms(x, a, v, v)[1]),
            (v, lambda a: ops.block_norms(x, d, a, v)[1]), (v, lambda a: ops.block_norms(x, d, v, a)[1]),
            (v, lambda a: ops.block_norms(x, d, v, v, gate=a)[1]),
            (x, lambda a: ops.block_norms(a, d, v, v, inplace=True)[1]),
            (hb, lambda a: ops.linear_cross_entropy(a, w, t)), (w, lambda a: ops.linear_cross_entropy(hb, a, t))]


@pytest.mark.parametrize("which", range(10))
def test_forward_mode(which):
    x, call = _calls()[which]
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(fwd.make_dual(x, torch.ones_like(x)))
        call(x)


@pytest.mark.parametrize("which", [0, 2, 8])
def test_forward_mode_over_the_gradient(which):
    x, call = _calls()[which]
    x.requires_grad_()
    out = call(x)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, x, fwd.make_dual(torch.ones_like(out), torch.ones_like(out)))


@pytest.mark.parametrize("which", [0, 2, 8])
def test_function_transforms(which):
    x, call = _calls()[which]
    for run in (lambda: torch.func.jvp(call, (x,), (torch.ones_like(x),)), lambda: torch.func.vmap(call)(x[None])):
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            run()


@pytest.mark.parametrize("which", [0, 2, 8])
def test_traces(which):
    x, call = _calls()[which]
    with pytest.raises(NotImplementedError, match="jit.trace"):
        torch.jit.trace(call, x)
    call(x)
