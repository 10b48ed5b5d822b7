"""ops._lib.stream_ptr names a device in each way that torch does."""
import pytest
import torch

from mlx_swift_lm_b200.ops import _lib


@pytest.mark.parametrize("device,index", [(None, 5), (2, 2), ("cuda:3", 3), ("cuda", 5), (torch.device("cuda", 1), 1),
                                          (torch.device("cuda"), 5)])
def test_devices(monkeypatch, device, index):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 5)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    assert _lib.stream_ptr(device) == 100 + index
