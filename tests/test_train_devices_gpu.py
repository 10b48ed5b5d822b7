"""The fused training loss takes its targets from the CPU or the model's device, as the plain one does."""
import pytest
import torch

from mlx_swift_lm_b200 import DecoderLM
from mlx_swift_lm_b200.api.tokenizer import ByteTokenizer
from mlx_swift_lm_b200.models.config import tiny_qwen3
from mlx_swift_lm_b200.train import iterate_batches, loss_fn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fused", [False, True])
def test_targets_on_the_models_device(fused):
    m = DecoderLM(tiny_qwen3(), torch.device("cuda"), torch.bfloat16).init_random(0, std=0.1)
    x, y, ln = next(iterate_batches(["hello adapters", "abc"], ByteTokenizer(m.cfg.vocab_size), 2, train=False))
    with torch.no_grad():
        want, n = loss_fn(m, None, x, y, ln, training=False, fused=fused)
        got, k = loss_fn(m, None, x.cuda(), y.cuda(), ln, training=False, fused=fused)
    assert torch.equal(got, want) and n == k
