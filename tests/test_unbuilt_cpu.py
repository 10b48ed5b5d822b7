"""CPU tensors need nothing built: the oracles answer where the autograd module is missing."""
import pytest
import torch

from mlx_swift_lm_b200 import DecoderLM, ops
from mlx_swift_lm_b200.models.config import tiny_qwen3
from mlx_swift_lm_b200.ops import _autograd, _lib


@pytest.fixture
def unbuilt(monkeypatch, tmp_path):
    monkeypatch.setattr(_autograd, "_module", None)
    monkeypatch.setattr(_lib, "LIB_PATH", str(tmp_path / "libb200kernels.so"))


def _outs():
    g = torch.Generator().manual_seed(0)
    x, d, w = torch.randn(5, 32, generator=g), torch.randn(5, 32, generator=g), torch.randn(40, 32, generator=g)
    t = torch.tensor([1, 2, -100, 39, 0])
    x.requires_grad_()
    y, h = ops.block_norms(x, d, w[0], w[1])
    outs = [y, h, ops.dropout(x, 0.3, 5), ops.linear_cross_entropy(x, w, t, reduction="mean")]
    grad, = torch.autograd.grad(sum(o.sum() for o in outs), x)
    return [o.detach() for o in outs] + [grad]


def test_operators(unbuilt, monkeypatch):
    got = _outs()
    assert _autograd._module is None
    with pytest.raises(ValueError):
        ops.dropout(torch.ones(4), 1.5, 0)
    with pytest.raises(ValueError):
        ops.block_norms(torch.ones(4, 8), torch.ones(1, 8))
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(torch.ones(1, 8), torch.ones(4, 8), torch.zeros(1, dtype=torch.int64), reduction="max")
    with pytest.raises(_lib.KernelLibraryMissing):
        _autograd.module()
    monkeypatch.undo()
    assert all(torch.equal(a, b) for a, b in zip(got, _outs()))


def test_serving_with_output_norms(unbuilt):
    m = DecoderLM(tiny_qwen3(), "cpu", torch.float32).init_random(0, std=0.2)
    for L in m.layers:
        L.post_attn_norm = L.post_ffn_norm = torch.ones(m.cfg.hidden_size)
    assert torch.isfinite(m.forward_dense(torch.arange(3, 25), m.new_cache())).all()
    assert _autograd._module is None
