"""Adapter training on the training operators (TrainParameters.fused): the same loss
and gradients as the plain forward, dropout masks that follow from the step, and the
sandwich-norm decoders' serving path over the fused block norms."""
import pytest
import torch

from mlx_swift_lm_b200 import DecoderLM, ops
from mlx_swift_lm_b200.adapters import LoRAConfiguration, LoRAContainer, LoRAParameters
from mlx_swift_lm_b200.api.tokenizer import ByteTokenizer
from mlx_swift_lm_b200.models.config import tiny_qwen3
from mlx_swift_lm_b200.train import (MaskStream, TrainableLoRA, TrainParameters, evaluate, iterate_batches, loss_fn, train,
                                     train_forward, train_hidden)

KEYS = ["self_attn.q_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.down_proj"]
TEXT = ["the quick brown fox jumps over the lazy dog", "hello world", "hello adapters, hello", "abc def"]


def _model(seed=0, **over):
    cfg = tiny_qwen3()
    for k, v in over.items():
        setattr(cfg, k, v)
    m = DecoderLM(cfg, "cpu", torch.float32).init_random(seed, std=0.2)
    return m


def _sandwich(m, seed=3):
    g = torch.Generator().manual_seed(seed)
    for L in m.layers:
        L.post_attn_norm = 1 + 0.1 * torch.randn(m.cfg.hidden_size, generator=g)
        L.post_ffn_norm = 1 + 0.1 * torch.randn(m.cfg.hidden_size, generator=g)
    return m


def _adapter(m, dropout=0.0, seed=0):
    conf = LoRAConfiguration(num_layers=2, lora_parameters=LoRAParameters(rank=4, scale=2.0, dropout=dropout, keys=KEYS))
    ad = LoRAContainer.init_for(m, conf, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    for ent in ad.tensors.values():
        ent["b"] = torch.randn(ent["b"].shape, generator=g) * 0.05
    return ad


def _batch(m):
    return next(iterate_batches(TEXT, ByteTokenizer(m.cfg.vocab_size), 4, train=False))


@pytest.mark.parametrize("over", [{}, {"final_logit_softcap": 8.0}, {"norm_offset_one": True}])
@pytest.mark.parametrize("sandwich", [False, True])
def test_fused_loss_and_gradients_equal_the_plain_ones(over, sandwich):
    m = _model(**over)
    if sandwich:
        _sandwich(m)
    x, y, ln = _batch(m)
    grads = []
    for fused in (False, True):
        lora = TrainableLoRA(_adapter(m), "cpu")
        loss, n = loss_fn(m, lora, x, y, ln, fused=fused)
        loss.backward()
        grads.append((loss.detach(), n, [p.grad for p in lora.parameters()]))
    (l0, n0, g0), (l1, n1, g1) = grads
    # both in fp32: the sums differ in their order only
    assert n0 == n1 and abs(l0 - l1) <= 1e-5 * l0
    for a, b in zip(g0, g1):
        assert (a - b).norm() <= 1e-4 * a.norm()


def test_hidden_rows_give_the_plain_logits():
    m = _sandwich(_model())
    x, _, _ = _batch(m)
    a = train_forward(m, x, None, training=False)
    h = train_hidden(m, x, None, training=False)
    assert torch.allclose(h @ m.lm_head.t(), a, rtol=1e-4, atol=2e-4)


def test_masks_follow_from_the_step():
    m = _model()
    x, y, ln = _batch(m)
    ad = _adapter(m, dropout=0.3)
    lora = TrainableLoRA(ad, "cpu")

    def loss(seed, step, training=True):
        lora.masks = MaskStream(seed, step)
        return float(loss_fn(m, lora, x, y, ln, training=training, fused=True)[0].detach())

    torch.manual_seed(1)
    a = loss(5, 7)
    torch.manual_seed(2)
    assert loss(5, 7) == a and loss(5, 8) != a and loss(6, 7) != a
    assert loss(5, 7, training=False) == loss(9, 1, training=False)
    s = MaskStream(5, 7)
    t = torch.ones(4, 64)
    assert not torch.equal(s.dropout(t, 0.5), s.dropout(t, 0.5))  # each call its own mask


def test_a_resumed_run_takes_the_steps_it_would_have_taken():
    m = _model()
    tok = ByteTokenizer(m.cfg.vocab_size)
    data = TEXT[:1] * 4  # every batch is the same, whatever order an iterator deals
    sgd = lambda ps: torch.optim.SGD(ps, lr=1e-2)  # noqa: E731  (no state of its own to resume)

    def run(ad, **kw):
        p = TrainParameters(batch_size=4, steps_per_eval=100, validation_batches=1, fused=True, seed=3, **kw)
        return train(m, ad, tok, data, [], p, optimizer_factory=sgd)

    whole = run(_adapter(m, dropout=0.2), iterations=4)
    parts = run(_adapter(m, dropout=0.2), iterations=2)
    assert not all(torch.equal(whole.tensors[k]["b"], parts.tensors[k]["b"]) for k in whole.tensors)
    parts = run(parts, iterations=4, completed_iterations=2)
    for k in whole.tensors:
        assert torch.equal(whole.tensors[k]["a"], parts.tensors[k]["a"])
        assert torch.equal(whole.tensors[k]["b"], parts.tensors[k]["b"])


def test_fused_training_runs_and_evaluates():
    m = _model(seed=1)
    tok = ByteTokenizer(m.cfg.vocab_size)
    events = []
    p = TrainParameters(batch_size=2, iterations=4, steps_per_report=2, steps_per_eval=2, validation_batches=1,
                        learning_rate=1e-3, fused=True)
    train(m, _adapter(m, dropout=0.1), tok, TEXT, TEXT[:2], p, progress=lambda e: events.append(e) or True)
    assert {e.kind for e in events} == {"train", "validation"}
    a = evaluate(m, None, TEXT, tok, 2, fused=True)
    b = evaluate(m, None, TEXT, tok, 2)
    assert abs(a - b) <= 1e-5 * b


def test_fused_refuses_what_the_plain_forward_refuses():
    m = _model()
    m.lm_head = object()
    x, y, ln = _batch(m)
    with pytest.raises(ValueError):
        loss_fn(m, None, x, y, ln, fused=True)


@pytest.mark.parametrize("pre_norms", [True, False])
def test_serving_forward_of_sandwich_norms(pre_norms):
    """The dense forward with the norms fused equals the norms taken one by one, bit for bit."""
    m = _sandwich(_model())
    if not pre_norms:
        m.cfg.pre_norms = False
        for L in m.layers:
            L.ln1 = L.ln2 = None
    toks = torch.arange(3, 25)
    fused = m.forward_dense(toks, m.new_cache())
    calls = []

    def one_by_one(x, delta, post_w, pre_w, eps, **kw):
        calls.append(1)
        d = ops.rmsnorm(delta, post_w, eps, kw["offset_one"])
        if pre_w is None:
            x.add_(d)
            return x, None
        return x, ops.add_rmsnorm(x, d, pre_w, eps, offset_one=kw["offset_one"])

    real, ops.block_norms = ops.block_norms, one_by_one
    try:
        want = m.forward_dense(toks, m.new_cache())
    finally:
        ops.block_norms = real
    assert len(calls) == 2 * len(m.layers) and torch.equal(fused, want)
