"""The stock-PyTorch comparison build's single-sequence path."""
import pytest
import torch

from mlx_swift_lm_b200 import DecoderLM
from mlx_swift_lm_b200.baseline import TorchDecoderLM
from mlx_swift_lm_b200.models.config import tiny_qwen3


@pytest.mark.parametrize("sandwich", [False, True])
def test_baseline_dense_forward(sandwich):
    """The single-sequence path runs the baseline's own norms, with and without output norms."""
    cfg = tiny_qwen3()
    models = [cls(cfg, "cpu", torch.float32).init_random(5, std=0.2) for cls in (DecoderLM, TorchDecoderLM)]
    if sandwich:
        for m in models:
            g = torch.Generator().manual_seed(3)
            for L in m.layers:
                L.post_attn_norm = 1 + 0.1 * torch.randn(cfg.hidden_size, generator=g)
                L.post_ffn_norm = 1 + 0.1 * torch.randn(cfg.hidden_size, generator=g)
    toks = torch.arange(3, 25)
    want, got = (m.forward_dense(toks, m.new_cache()) for m in models)
    torch.testing.assert_close(got, want, atol=2e-4, rtol=2e-4)
