"""The training operators together, as an adapter step uses them: block norms, dropout
and the loss from hidden rows, eager and in a captured step, and the training path."""
import math

import pytest
import torch

from mlx_swift_lm_b200 import DecoderLM, ops
from mlx_swift_lm_b200.adapters import LoRAConfiguration, LoRAContainer, LoRAParameters
from mlx_swift_lm_b200.api.tokenizer import ByteTokenizer
from mlx_swift_lm_b200.models.config import tiny_qwen3
from mlx_swift_lm_b200.ops import _lib
from mlx_swift_lm_b200.ops import reference as ref
from mlx_swift_lm_b200.train import MaskStream, TrainableLoRA, TrainParameters, iterate_batches, loss_fn, train, train_hidden

pytestmark = pytest.mark.gpu
DEV = "cuda"
KEYS = ["self_attn.q_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.down_proj"]
TEXT = ["the quick brown fox jumps over the lazy dog", "hello world", "hello adapters, hello", "abc def"]


def _step(x, delta, post, pre, w, t, p, seed, offset, dtype):
    y, h = ops.block_norms(x, delta, post, pre)
    y2, h2 = ops.block_norms(y, ops.dropout(h, p, seed, offset), post, pre)
    return ops.linear_cross_entropy(h2.to(dtype), w, t, reduction="mean")


def _inputs(T=70, H=96, V=700, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = torch.randint(0, V, (T,), generator=g)
    t[::5] = -100
    return [n(T, H), n(T, H), 1 + 0.1 * n(H), 1 + 0.1 * n(H)], (n(V, H) / math.sqrt(H)).bfloat16(), t


def test_a_run_of_the_operators():
    leaves, w, t = _inputs()
    dev = [v.to(DEV).requires_grad_() for v in leaves]
    loss = _step(*dev, w.to(DEV), t.to(DEV), 0.2, 9, 4, torch.bfloat16)
    got = torch.autograd.grad(loss, dev)
    # the same run in 64 bits, with the head's rows rounded to bf16 as the step rounds them
    dbl = [v.double().requires_grad_() for v in leaves]
    keep = ref.dropout_keep_ref(70, 96, 0.2, 9, 4)

    def rms(v, s):
        return v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * s

    y = dbl[0] + rms(dbl[1], dbl[2])
    h = rms(y, dbl[3])
    y = y + rms(torch.where(keep, h * ref.dropout_scale(ref.dropout_cut(0.2)), 0.0), dbl[2])
    h = rms(y, dbl[3])
    h = h + (h.detach().bfloat16().double() - h.detach())
    z = h @ w.double().t()
    want = torch.nn.functional.cross_entropy(z, t, ignore_index=-100)
    # a logit may be off where h rounds to the other neighbour (2^-7 of an entry, where fp32 and 64 bits
    # fall on different sides: at most once in 2^13 entries) and by the product's own 2^-20
    assert abs(loss.item() - want.item()) <= 1e-3 * want.item()
    wanted = torch.autograd.grad(want, dbl)
    for a, b in zip(got, wanted):
        # bf16 rounds G and then dh: at most 2^-8 of each, which the chain of norms carries on linearly
        assert (a.double().cpu() - b).norm() <= 2 * 2 ** -8 * b.norm()


def test_a_captured_step_replays_with_new_inputs_and_masks():
    leaves, w, t = _inputs()
    dev = [v.to(DEV).requires_grad_() for v in leaves]
    w, t, off = w.to(DEV), t.to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV)

    def step(offset):
        loss = _step(*dev, w, t, 0.2, 9, offset, torch.bfloat16)
        return (loss.detach(),) + torch.autograd.grad(loss, dev)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(off)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(off)
    for k in range(3):
        off.fill_(k)
        with torch.no_grad():
            for v, new in zip(dev, _inputs(seed=k)[0]):
                v.copy_(new)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step(k)))


def test_two_captured_steps_do_not_share_workspaces():
    graphs = []
    for seed in (1, 2):
        leaves, w, t = _inputs(seed=seed)
        dev = [v.to(DEV).requires_grad_() for v in leaves]
        args = (w.to(DEV), t.to(DEV), 0.3, seed, 0, torch.bfloat16)

        def step(dev=dev, args=args):
            loss = _step(*dev, *args)
            return (loss.detach(),) + torch.autograd.grad(loss, dev)

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            want = step()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got, want))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (g, _, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, got, want in graphs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_steps_leave_no_memory_behind():
    leaves, w, t = _inputs()
    dev = [v.to(DEV).requires_grad_() for v in leaves]
    w, t = w.to(DEV), t.to(DEV)

    def step():
        loss = _step(*dev, w, t, 0.2, 9, 4, torch.bfloat16)
        torch.autograd.grad(loss, dev)
        _step(*dev, w, t, 0.2, 9, 4, torch.bfloat16)  # and a graph that is dropped

    step()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(20):
        step()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before


def test_the_same_leaf_twice():
    x = torch.randn(6, 32, device=DEV, requires_grad=True)
    w = torch.ones(32, device=DEV, requires_grad=True)
    y, h = ops.block_norms(x, x, w, w)
    gx, gw = torch.autograd.grad(y.sum() + (h * h).sum(), [x, w])
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    rms = lambda v: v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * wd  # noqa: E731
    yd = xd + rms(xd)
    want = torch.autograd.grad(yd.sum() + rms(yd).square().sum(), [xd, wd])
    assert torch.allclose(gx.double(), want[0], rtol=1e-4, atol=1e-4) and torch.allclose(gw.double(), want[1], rtol=1e-4, atol=1e-4)
    a = torch.randn(6, 32, device=DEV)
    b, c = a.clone(), a.clone()
    y, _ = ops.block_norms(b, b, w.detach(), None, inplace=True)
    assert torch.equal(y, ops.block_norms(a, c, w.detach(), None)[0])
    z = ops.dropout(x, 0.5, 3, residual=x)
    keep = ref.dropout_keep_ref(6, 32, 0.5, 3).to(DEV)
    assert torch.equal(torch.autograd.grad(z.sum(), x)[0], 1 + 2.0 * keep)


def test_a_capture_beside_a_living_eager_graph_is_refused():
    x = torch.randn(6, 32, device=DEV, requires_grad=True)
    w = torch.randn(40, 32, device=DEV).bfloat16()
    hb = torch.randn(6, 32, device=DEV).bfloat16().requires_grad_()
    t = torch.arange(6, device=DEV)
    calls = [(x, lambda: ops.dropout(x, 0.5, 1)), (x, lambda: ops.block_norms(x, x, None, torch.ones(32, device=DEV))[1]),
             (hb, lambda: ops.linear_cross_entropy(hb, w, t))]
    for leaf, call in calls:
        kept = call()  # an eager graph on the default stream
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(g):
                call()
        want, = torch.autograd.grad(kept.sum(), leaf)
        del kept
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got, = torch.autograd.grad(call().sum(), leaf)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_gradients_are_taken_once():
    x = torch.randn(4, 32, device=DEV, requires_grad=True)
    w = torch.randn(40, 32, device=DEV).bfloat16()
    t = torch.arange(4, device=DEV)
    for out in (ops.dropout(x, 0.5, 1).sum(), ops.block_norms(x, x, None, torch.ones(32, device=DEV))[1].sum(),
                ops.linear_cross_entropy(x.bfloat16(), w, t).sum()):
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out, x, create_graph=True)


def _model(dtype=torch.bfloat16):
    return DecoderLM(tiny_qwen3(), torch.device(DEV), dtype).init_random(0, std=0.1)


def _adapter(m, dropout=0.0):
    conf = LoRAConfiguration(num_layers=2, lora_parameters=LoRAParameters(rank=4, scale=2.0, dropout=dropout, keys=KEYS))
    ad = LoRAContainer.init_for(m, conf, seed=0)
    g = torch.Generator().manual_seed(1)
    for ent in ad.tensors.values():
        ent["b"] = torch.randn(ent["b"].shape, generator=g) * 0.05
    return ad


def test_training_loss_and_gradients():
    m = _model()
    x, y, ln = next(iterate_batches(TEXT, ByteTokenizer(m.cfg.vocab_size), 4, train=False))
    res = []
    for fused in (False, True):
        lora = TrainableLoRA(_adapter(m), torch.device(DEV))
        loss, n = loss_fn(m, lora, x, y, ln, fused=fused)
        loss.backward()
        res.append((loss.item(), n, [p.grad for p in lora.parameters()]))
    (l0, n0, g0), (l1, n1, g1) = res
    with torch.no_grad():
        h = train_hidden(m, x, TrainableLoRA(_adapter(m), torch.device(DEV)), training=False).reshape(-1, m.cfg.hidden_size)
        # rounding the head's rows moves a logit by at most 2^-8 sum |h w|, a loss by two logits' worth
        bound = 2 * 2 ** -8 * (h.abs() @ m.lm_head.float().abs().t()).amax().item()
    assert n0 == n1 and abs(l0 - l1) <= bound
    assert all(torch.isfinite(g).all() and g.abs().sum() > 0 for g in g1)
    assert _lib.read_status()["linear_ce"] == 0


def test_fused_training_runs():
    m = _model()
    p = TrainParameters(batch_size=2, iterations=3, steps_per_report=1, steps_per_eval=2, validation_batches=1, fused=True)
    events = []
    train(m, _adapter(m, dropout=0.1), ByteTokenizer(m.cfg.vocab_size), TEXT, TEXT[:2], p,
          progress=lambda e: events.append(e) or True)
    assert {e.kind for e in events} == {"train", "validation"}
    assert all(math.isfinite(e.loss) for e in events)


def test_masks_equal_the_cpu_streams():
    x = torch.randn(40, 100, device=DEV)
    a = MaskStream(3, 5).dropout(x, 0.3)
    assert torch.equal(a.cpu(), MaskStream(3, 5).dropout(x.cpu(), 0.3))
