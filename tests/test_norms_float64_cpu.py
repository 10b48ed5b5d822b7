"""Decoders with output norms in float64 on CPU: the fused block norms do not take that
type, and the separate norms run in their place."""
import pytest
import torch

from mlx_swift_lm_b200 import DecoderLM
from mlx_swift_lm_b200.models.config import tiny_qwen3
from mlx_swift_lm_b200.models.families import build_config

LT = ["sliding_attention", "sliding_attention", "full_attention"] * 2
ROPE = {"sliding_attention": {"rope_type": "default", "rope_theta": 10000.0},
        "full_attention": {"rope_type": "proportional", "partial_rotary_factor": 0.25, "rope_theta": 1000000.0}}
GEMMA4 = dict(model_type="gemma4_text", vocab_size=300, hidden_size=64, intermediate_size=128, num_hidden_layers=6,
              num_attention_heads=2, num_key_value_heads=1, head_dim=32, global_head_dim=64, sliding_window=8, layer_types=LT,
              num_kv_shared_layers=2, hidden_size_per_layer_input=16, vocab_size_per_layer_input=300,
              use_double_wide_mlp=True, final_logit_softcapping=30.0, rope_parameters=ROPE, rms_norm_eps=1e-6,
              max_position_embeddings=512)


def _sandwich():
    m = DecoderLM(tiny_qwen3(), "cpu", torch.float32).init_random(0, std=0.05)
    g = torch.Generator().manual_seed(3)
    for L in m.layers:
        L.post_attn_norm = 1 + 0.1 * torch.randn(m.cfg.hidden_size, generator=g)
        L.post_ffn_norm = 1 + 0.1 * torch.randn(m.cfg.hidden_size, generator=g)
    return m


@pytest.mark.parametrize("which", ["sandwich", "gemma4"])
def test_float64_models_run(which):
    m = _sandwich() if which == "sandwich" else DecoderLM(build_config(GEMMA4), "cpu", torch.float32).init_random(0, std=0.05)
    d = m.clone_to("cpu", torch.float64)
    toks = torch.arange(3, 25)
    got, want = (v.forward_dense(toks, v.new_cache()) for v in (d, m))
    # the oracles compute in fp32 either way; a float64 model differs by what fp32 rounds in between
    torch.testing.assert_close(got.float(), want.float(), atol=1e-3, rtol=1e-3)
