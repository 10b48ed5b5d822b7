"""Captured training steps beside eager graphs: what the operators refuse before autograd's thread meets it."""
import pytest
import torch

from mlx_swift_lm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _calls(x):
    ones, w = torch.ones(32, device=DEV), torch.randn(40, 32, device=DEV).bfloat16()
    t = torch.arange(6, device=DEV)
    return {"dropout": lambda a: ops.dropout(a, 0.5, 1), "block_norms": lambda a: ops.block_norms(a, a, None, ones)[1],
            "linear_cross_entropy": lambda a: ops.linear_cross_entropy(a.bfloat16(), w, t)}


@pytest.mark.parametrize("op", ["dropout", "block_norms", "linear_cross_entropy"])
def test_an_input_made_from_a_leaf_of_a_living_eager_graph(op):
    x = torch.randn(6, 32, device=DEV, requires_grad=True)
    call = _calls(x)[op]
    kept = x * 2  # an eager graph of the leaf on the default stream
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call(x * 1)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call(kept)  # the eager graph's own output
    del kept
    want, = torch.autograd.grad(call(x * 1).sum(), x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got, = torch.autograd.grad(call(x * 1).sum(), x)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_a_stream_that_joined_the_capture_is_no_other_graph():
    x = torch.randn(6, 32, device=DEV, requires_grad=True)
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            h = ops.dropout(x, 0.5, 1)
        main.wait_stream(side)
        with torch.no_grad():
            h0 = ops.dropout(x, 0.5, 1)
        y = ops.dropout(h, 0.25, 2)  # its input's node lies on the other stream of the same capture
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(h, h0) and torch.equal(y, ops.dropout(h0, 0.25, 2))
