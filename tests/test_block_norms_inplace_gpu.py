"""ops.block_norms(inplace=True) on the GPU: what autograd sees of the write."""
import pytest
import torch

from mlx_swift_lm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _graph_then_inplace(dev):
    x, d = torch.randn(4, 64, device=dev), torch.randn(4, 64, device=dev)
    w = torch.randn(64, device=dev, requires_grad=True)
    z = x * w  # saves x for w's gradient
    with torch.no_grad():
        ops.block_norms(x, d, None, torch.ones(64, device=dev), inplace=True)
    return z


def test_a_saved_x_is_seen_to_have_changed():
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        _graph_then_inplace(DEV).sum().backward()


def test_views_share_the_version():
    x = torch.randn(2, 3, 64, device=DEV)
    before = x._version
    ops.block_norms(x.view(6, 64), torch.randn(6, 64, device=DEV), torch.ones(64, device=DEV), inplace=True)
    assert x._version > before
    before = x._version
    ops.block_norms(x, torch.randn(2, 3, 64, device=DEV), torch.ones(64, device=DEV))
    assert x._version == before


def test_inference_tensors():
    with torch.inference_mode():
        x, d = torch.randn(4, 64, device=DEV), torch.randn(4, 64, device=DEV)
        want = ops.block_norms(x.clone(), d, torch.ones(64, device=DEV))[0]
        assert torch.equal(ops.block_norms(x, d, torch.ones(64, device=DEV), inplace=True)[0], want) and torch.equal(x, want)
