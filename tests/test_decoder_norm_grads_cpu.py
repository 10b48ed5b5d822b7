"""A paged forward pass that autograd records, through a decoder with output norms."""
import torch

from mlx_swift_lm_b200 import DecoderLM
from mlx_swift_lm_b200.kv.paged import PagedKVCache
from mlx_swift_lm_b200.models.batch import ForwardBatch
from mlx_swift_lm_b200.models.config import tiny_qwen3


def test_output_norms_take_gradients():
    m = DecoderLM(tiny_qwen3(), "cpu", torch.float32).init_random(0, std=0.2)
    for L in m.layers:
        L.post_attn_norm = torch.full((m.cfg.hidden_size,), 1.1)
        L.post_ffn_norm = torch.full((m.cfg.hidden_size,), 0.9)

    def logits():
        kv = PagedKVCache.for_model(m, max_tokens=256)
        pages = kv.pool.alloc(4)
        slots = torch.tensor([pages[i // 16] * 16 + i % 16 for i in range(40)], dtype=torch.int64)
        fb = ForwardBatch(input_ids=torch.arange(40, dtype=torch.int32), positions=torch.arange(40, dtype=torch.int32),
                          slots=slots, pf_cu_q=torch.tensor([0, 40], dtype=torch.int32), pf_cu_q_host=[0, 40],
                          pf_pos0=torch.zeros(1, dtype=torch.int32), pf_pos0_host=[0],
                          pf_page_table=torch.tensor([pages], dtype=torch.int32))
        return m.forward(fb, kv)

    want = logits()
    w = m.layers[-1].post_attn_norm.requires_grad_()
    got = logits()
    assert torch.equal(got.detach(), want)
    grad, = torch.autograd.grad(got.double().sum(), w)
    # the gradient along a direction against a central difference: fp32 logits of order 10 step by 2^-20,
    # 20480 of them by 2^-20 sqrt(20480) < 2e-4 in all at random, and the difference divides that by 2 e
    d, e = torch.randn(w.shape, generator=torch.Generator().manual_seed(1)), 1e-2
    vals = []
    for s in (1, -1):
        m.layers[-1].post_attn_norm = w.detach() + s * e * d
        vals.append(logits().double().sum())
    slope = (vals[0] - vals[1]) / (2 * e)
    assert abs(slope - (grad * d).sum()) <= 2e-2 * (1 + abs(slope))
