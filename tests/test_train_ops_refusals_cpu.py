"""Tensors that the training operators' kernels cannot answer for, refused before any launch."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from mlx_swift_lm_b200 import ops


def _calls(dev):
    x = torch.empty(4, 32, device=dev)
    w, t = torch.empty(40, 32, device=dev, dtype=torch.bfloat16), torch.empty(4, device=dev, dtype=torch.int64)
    return [lambda: ops.dropout(x, 0.5, 1), lambda: ops.block_norms(x, x, x[0], x[0]),
            lambda: ops.linear_cross_entropy(x.bfloat16(), w, t)]


@pytest.mark.parametrize("which", range(3))
def test_fake_cuda_tensors(which):
    with FakeTensorMode(), pytest.raises(TypeError, match="without memory"):
        _calls("cuda")[which]()


def test_fake_cpu_tensors_pass():
    with FakeTensorMode():
        x = torch.empty(4, 32)
        y, h = ops.block_norms(x, torch.empty(4, 32), x.new_empty(32), x.new_empty(32), inplace=True)
        assert y.shape == h.shape == (4, 32)
