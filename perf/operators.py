"""Cases of the adapter-training operators and of the block norms that serving shares with them.

Three operators that one training step of a decoder's adapters runs next to each other:

* ``linear_cross_entropy``: the vocabulary head and its softmax cross entropy in one operator that never
  holds the logits of the whole vocabulary, with the gradients of the hidden rows and of the head;
* ``dropout``: inverted dropout from a counter-based generator (Philox-4x32-10 keyed by the seed, counting
  columns, rows and the call's offset), whose mask is drawn again by the backward pass instead of stored;
* ``block_norms``: the norm after a block, its gate and residual scale, the residual add and the norm before
  the next block as one pass, forward and backward. Decoding runs its forward pass on a few rows.

A case's plain form is written in elementary torch operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORE = -100
EPS = 1e-6
M32 = 0xFFFFFFFF


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # scoring a single position of a small vocabulary (the tiny test model's head): latency alone
        dict(name="ce_one_token", op="ce", T=1, V=4096, K=256, ignored=0.0, softcap=0.0, reduction="mean", dh=True, dw=False),
        # validation loss of one 512-token sample, nothing differentiable: one pass over the head
        dict(name="ce_eval", op="ce", T=512, V=151936, K=4096, ignored=0.0, softcap=0.0, reduction="none", dh=False, dw=False),
        # adapter step of four 512-token samples, a quarter of it padding; the head is frozen
        dict(name="ce_adapter_step", op="ce", T=2048, V=151936, K=4096, ignored=0.25, softcap=0.0, reduction="mean", dh=True, dw=False),
        # full step of 4096 tokens with a trained head
        dict(name="ce_full_step", op="ce", T=4096, V=151936, K=4096, ignored=0.0, softcap=0.0, reduction="mean", dh=True, dw=True),
        # odd vocabulary and row count, capped logits, weighted tokens
        dict(name="ce_softcap_odd", op="ce", T=1001, V=50257, K=2560, ignored=0.1, softcap=30.0, reduction="none", dh=True, dw=True),
        # the tiny test model's rows in 32 bits
        dict(name="dropout_small", op="dropout", T=33, K=256, dtype="fp32", p=0.1, residual=False, slack=0),
        # adapter dropout over the hidden rows of 8192 tokens
        dict(name="dropout_step", op="dropout", T=8192, K=4096, dtype="bf16", p=0.05, residual=False, slack=0),
        # residual dropout over odd rows that are a slice of a wider buffer
        dict(name="dropout_residual_odd", op="dropout", T=2047, K=5001, dtype="fp16", p=0.3, residual=True, slack=7),
        # one decode step of 64 streams: forward only
        dict(name="norms_decode", op="norms", T=64, H=4096, dtype="bf16", post=True, pre=True, gate="", scale=1.0, grad=False, slack=0),
        # training step of 8192 tokens through a sandwich-norm block
        dict(name="norms_step", op="norms", T=8192, H=4096, dtype="bf16", post=True, pre=True, gate="", scale=1.0, grad=True, slack=0),
        # gate for each channel and a residual scale, no norm after the block, 32 bits, odd width
        dict(name="norms_channel_gate_odd", op="norms", T=1023, H=2561, dtype="fp32", post=False, pre=True, gate="channel", scale=0.22, grad=True, slack=3),
        # gate for each element (modulated blocks), both norms
        dict(name="norms_element_gate", op="norms", T=2048, H=2304, dtype="bf16", post=True, pre=True, gate="element", scale=0.5, grad=True, slack=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ce", "ce", "dropout", "norms"])
    if op == "ce":
        dh = rng.random() < 0.8
        return dict(op="ce", T=_log(rng, 1, 4096), V=_log(rng, 200, 151936),
                    K=rng.choice([8 * _log(rng, 8, 512), _log(rng, 64, 4096)]), ignored=rng.choice([0.0, 0.0, 0.3, 0.9]),
                    softcap=rng.choice([0.0, 0.0, 30.0]), reduction=rng.choice(["none", "mean", "sum"]), dh=dh,
                    dw=dh and rng.random() < 0.5)
    T = _log(rng, 1, 8192)
    width = min(16384, 8192 * 4096 // T)
    if op == "dropout":
        return dict(op="dropout", T=T, K=_log(rng, 1, width), dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    p=round(rng.uniform(0.01, 0.9), 3), residual=rng.random() < 0.5, slack=rng.choice([0, 0, 5, 64]))
    post, pre = rng.choice([(True, True), (True, True), (True, False), (False, True)])
    return dict(op="norms", T=T, H=rng.choice([8 * _log(rng, 1, max(1, width // 8)), _log(rng, 8, max(8, width))]),
                dtype=rng.choice(["bf16", "fp16", "fp32"]), post=post, pre=pre,
                gate=rng.choice(["", "", "channel", "row", "element"]), scale=rng.choice([1.0, 0.22, -1.5]),
                grad=rng.random() < 0.7, slack=rng.choice([0, 0, 3, 64]))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def rows(T, C, slack, dtype):  # a [T, C] matrix whose rows lie `slack` elements apart
        buf = torch.empty(T, C + slack, device=DEV, dtype=dtype)
        buf[:, :C] = normal(T, C)
        return buf[:, :C]

    if case["op"] == "ce":
        T, V, K = case["T"], case["V"], case["K"]
        # final-normed rows (unit RMS) leaning towards their target's head row, as a trained model's do:
        # the target's probability runs from next to nothing to about a half over the tokens
        w = torch.empty(V, K, device=DEV, dtype=torch.bfloat16).normal_(0.0, 1.3 / math.sqrt(K), generator=g)
        targets = torch.randint(0, V, (T,), generator=g, device=DEV)
        lean = torch.rand(T, 1, generator=g, device=DEV) * 8.0
        h = (normal(T, K) + lean * w[targets].float()).to(torch.bfloat16)
        drop = torch.rand(T, generator=g, device=DEV) < case["ignored"]
        targets = torch.where(drop, torch.full_like(targets, IGNORE), targets)
        dloss = torch.rand(T, generator=g, device=DEV) if case["reduction"] == "none" else torch.ones((), device=DEV)
        return dict(case=case, h=h, w=w, targets=targets, dloss=dloss)
    dtype = TYPES[case["dtype"]]
    if case["op"] == "dropout":
        T, K = case["T"], case["K"]
        key = int(torch.randint(0, 1 << 62, (1,), generator=g, device=DEV))
        return dict(case=case, x=rows(T, K, case["slack"], dtype), dy=rows(T, K, 0, dtype),
                    residual=rows(T, K, case["slack"], dtype) if case["residual"] else None, seed=key, offset=key % 1000003)
    T, H = case["T"], case["H"]
    shape = {"": None, "channel": (H,), "row": (T, 1), "element": (T, H)}[case["gate"]]
    return dict(case=case, x=rows(T, H, case["slack"], dtype).mul_(3.0), delta=rows(T, H, case["slack"], dtype),
                post=(1 + 0.2 * normal(H)).to(dtype) if case["post"] else None,
                pre=(1 + 0.2 * normal(H)).to(dtype) if case["pre"] else None,
                gate=None if shape is None else (0.5 + 0.5 * normal(*shape)).to(dtype),
                dy=rows(T, H, 0, dtype) if case["grad"] else None,
                dh=rows(T, H, 0, dtype) if case["grad"] and case["pre"] else None)


def run(state):
    case = state["case"]
    if own:
        return _OWN[case["op"]](state)
    return _PLAIN[case["op"]](state)


def work(case):
    if case["op"] == "ce":
        n = round(case["T"] * (1 - case["ignored"]))
        products = 1 + (1 if case["dh"] else 0) + (1 if case["dw"] else 0)
        rows, head = 2 * n * case["K"], 2 * case["V"] * case["K"]
        return {"bytes": rows + head + 12 * case["T"] + (2 * case["T"] * case["K"] if case["dh"] else 0) + (head if case["dw"] else 0),
                "flops": 2 * n * case["V"] * case["K"] * products}
    size = 2 if case["dtype"] != "fp32" else 4
    if case["op"] == "dropout":
        n = case["T"] * case["K"]
        return {"bytes": size * n * (5 if case["residual"] else 4), "flops": 4 * n}
    n, elem = case["T"] * case["H"], case["gate"] == "element"
    reads = (2 + elem) * n
    moved = reads + (2 if case["pre"] else 1) * n
    if case["grad"]:  # the incoming gradients and the residual's, the block's and the gate's
        moved += (2 if case["pre"] else 1) * n + (2 + elem) * n
    return {"bytes": size * moved, "flops": (30 if case["grad"] else 10) * n}


# ---------------------------------------------------------------------------------------------- the framework's operators
def _own_ce(s):
    from mlx_swift_lm_b200 import ops

    case = s["case"]
    if not case["dh"]:
        return (ops.linear_cross_entropy(s["h"], s["w"], s["targets"], softcap=case["softcap"], ignore_index=IGNORE,
                                         reduction=case["reduction"]),)
    h = s["h"].detach().requires_grad_()
    w = s["w"].detach().requires_grad_(case["dw"])
    loss = ops.linear_cross_entropy(h, w, s["targets"], softcap=case["softcap"], ignore_index=IGNORE, reduction=case["reduction"])
    return (loss.detach(),) + torch.autograd.grad(loss, [h, w] if case["dw"] else [h], s["dloss"])


def _own_dropout(s):
    from mlx_swift_lm_b200 import ops

    x = s["x"].detach().requires_grad_()
    y = ops.dropout(x, s["case"]["p"], s["seed"], s["offset"], residual=s["residual"])
    return (y.detach(),) + torch.autograd.grad(y, [x], s["dy"])


def _own_norms(s):
    from mlx_swift_lm_b200 import ops

    case = s["case"]
    leaves = [s["x"], s["delta"], s["post"], s["pre"], s["gate"]]
    if case["grad"]:
        leaves = [None if t is None else t.detach().requires_grad_() for t in leaves]
    x, delta, post, pre, gate = leaves
    y, h = ops.block_norms(x, delta, post_w=post, pre_w=pre, eps=EPS, gate=gate, scale=case["scale"])
    outs = [y] if h is None else [y, h]
    if not case["grad"]:
        return tuple(outs)
    grads = torch.autograd.grad(outs, [t for t in leaves if t is not None], [s["dy"], s["dh"]][:len(outs)])
    return tuple(o.detach() for o in outs) + grads


_OWN = {"ce": _own_ce, "dropout": _own_dropout, "norms": _own_norms}


# ---------------------------------------------------------------------------------------------- plain forms
def _plain_ce(s):
    case, targets = s["case"], s["targets"]
    h, w, cap = s["h"].float(), s["w"].float(), case["softcap"]
    scored = targets != IGNORE
    at = torch.where(scored, targets, torch.zeros_like(targets))
    z = h @ w.t()
    if cap > 0:
        z = cap * torch.tanh(z / cap)
    # the target stands apart from the others' sum, so that a loss near zero keeps its digits:
    # loss = log(1 + exp(d)) with d = log sum_{v != t} exp(z_v) - z_t
    zt = z.gather(1, at[:, None])
    others = z.scatter(1, at[:, None], -math.inf)
    top = others.amax(1, keepdim=True)
    d = top + torch.log(torch.exp(others - top).sum(1, keepdim=True)) - zt
    each = torch.clamp_min(d, 0) + torch.log1p(torch.exp(-d.abs()))
    loss = torch.where(scored, each[:, 0], torch.zeros_like(each[:, 0]))
    n = scored.sum().clamp_min(1)
    out = {"none": loss, "sum": loss.sum(), "mean": loss.sum() / n}[case["reduction"]]
    if not case["dh"]:
        return (out,)
    d = s["dloss"].float() / (n if case["reduction"] == "mean" else 1)
    d = torch.where(scored, d.expand(targets.shape[0]), torch.zeros_like(loss))
    G = torch.exp(z - (zt + each)).scatter(1, at[:, None], torch.expm1(-each))
    G = G * d[:, None]
    if cap > 0:
        G = G * (1 - (z / cap) ** 2)
    dh = (G @ w).to(s["h"].dtype)
    return (out, dh, (G.t() @ h).to(s["w"].dtype)) if case["dw"] else (out, dh)


def _mulhilo(m, c):
    """(high, low) 32 bits of m * c for 32-bit values held in 64: the product by halves of m."""
    lo, hi = c * (m & 0xFFFF), c * (m >> 16)
    return ((lo >> 16) + hi) >> 16, (lo + ((hi & 0xFFFF) << 16)) & M32


def _keep(T, K, p, seed, offset):
    """The mask [T, K]: one Philox-4x32-10 block for 8 neighbouring columns of a row, 16 bits each."""
    blocks = (K + 7) // 8
    c0 = torch.arange(blocks, device=DEV)[None, :].expand(T, blocks)
    c1 = torch.arange(T, device=DEV)[:, None].expand(T, blocks)
    c2 = torch.full_like(c0, offset & M32)
    c3 = torch.full_like(c0, (offset >> 32) & M32)
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(10):
        h0, l0 = _mulhilo(0xD2511F53, c0)
        h1, l1 = _mulhilo(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    words = torch.stack([c0, c1, c2, c3], -1)
    halves = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(T, blocks * 8)
    return halves[:, :K] >= math.floor(p * 65536 + 0.5)


def _plain_dropout(s):
    case = s["case"]
    keep = _keep(case["T"], case["K"], case["p"], s["seed"], s["offset"])
    scale = 65536.0 / (65536 - math.floor(case["p"] * 65536 + 0.5))
    zero = torch.zeros((), device=DEV)
    y = torch.where(keep, s["x"].float() * scale, zero)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype), torch.where(keep, s["dy"].float() * scale, zero).to(s["x"].dtype)


def _rms_grad(g, hat, rstd):
    return rstd * (g - hat * (g * hat).mean(1, keepdim=True))


def _plain_norms(s):
    case, dtype = s["case"], s["x"].dtype
    x, delta = s["x"].float(), s["delta"].float()
    post, pre, gate = (None if t is None else t.float() for t in (s["post"], s["pre"], s["gate"]))
    u = delta
    if post is not None:
        r1 = torch.rsqrt((delta * delta).mean(1, keepdim=True) + EPS)
        dhat = delta * r1
        u = dhat * post
    branch = u if gate is None else u * gate
    y = (x + case["scale"] * branch).to(dtype)  # the residual stream is held in its own type
    outs = [y]
    if pre is not None:
        r2 = torch.rsqrt((y.float() * y.float()).mean(1, keepdim=True) + EPS)
        yhat = y.float() * r2
        outs.append((yhat * pre).to(dtype))
    if not case["grad"]:
        return tuple(outs)
    dx, grads = s["dy"].float(), {}
    if pre is not None:
        dh = s["dh"].float()
        dx = dx + _rms_grad(dh * pre, yhat, r2)
        grads["pre"] = (dh * yhat).sum(0)
    du = case["scale"] * dx
    if gate is not None:
        dgate = du * u
        grads["gate"] = {"channel": lambda: dgate.sum(0), "row": lambda: dgate.sum(1, keepdim=True), "element": lambda: dgate}[case["gate"]]()
        du = du * gate
    if post is not None:
        grads["post"] = (du * dhat).sum(0)
        du = _rms_grad(du * post, dhat, r1)
    order = [dx, du] + [grads[k] for k in ("post", "pre", "gate") if k in grads]
    return tuple(outs) + tuple(t.to(dtype) for t in order)


_PLAIN = {"ce": _plain_ce, "dropout": _plain_dropout, "norms": _plain_norms}


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_ce(case, s):
    """Cross entropy from its definition, a few thousand head rows at a time: -log softmax(z)[target], with
    the gradient (softmax(z) - indicator) dloss carried through the cap z = c tanh(u / c)."""
    T, V, cap = case["T"], case["V"], case["softcap"]
    h, t = s["h"].double(), s["targets"]
    scored = (t >= 0).double()
    step = 8192
    pieces = [(a, min(V, a + step)) for a in range(0, V, step)]

    def logits(a, b):
        u = torch.einsum("tk,vk->tv", h, s["w"][a:b].double())
        return u if cap <= 0 else torch.tanh(u / cap) * cap

    lse = torch.full((T,), -math.inf, dtype=torch.float64, device=DEV)
    zt = torch.zeros(T, dtype=torch.float64, device=DEV)
    for a, b in pieces:
        z = logits(a, b)
        lse = torch.logaddexp(lse, torch.logsumexp(z, 1))
        mine = (t >= a) & (t < b)
        zt[mine] = z[mine, t[mine] - a]
    each = (lse - zt) * scored
    count = max(1.0, float(scored.sum()))
    out = {"none": each, "sum": each.sum(), "mean": each.sum() / count}[case["reduction"]]
    if not case["dh"]:
        return (out,)
    d = scored * s["dloss"].double() / (count if case["reduction"] == "mean" else 1.0)
    dh, dw = torch.zeros_like(h), []
    for a, b in pieces:
        z = logits(a, b)
        G = torch.exp(z - lse[:, None])
        mine = (t >= a) & (t < b)
        G[mine, t[mine] - a] -= 1.0
        G *= d[:, None]
        if cap > 0:
            G *= 1.0 - torch.square(z / cap)
        dh += torch.einsum("tv,vk->tk", G, s["w"][a:b].double())
        if case["dw"]:
            dw.append(torch.einsum("tv,tk->vk", G, h))
    return (out, dh, torch.cat(dw)) if case["dw"] else (out, dh)


def _exact_dropout(case, s):
    T, K = case["T"], case["K"]
    blocks = -(-K // 8)
    u64 = np.uint64
    low, sh = u64(M32), u64(32)
    c = [np.broadcast_to(np.arange(blocks, dtype=u64), (T, blocks)), np.broadcast_to(np.arange(T, dtype=u64)[:, None], (T, blocks)),
         np.full((T, blocks), s["offset"] & M32, u64), np.full((T, blocks), s["offset"] >> 32, u64)]
    key = [s["seed"] & M32, s["seed"] >> 32]
    for _ in range(10):
        p, q = u64(0xD2511F53) * c[0], u64(0xCD9E8D57) * c[2]
        c = [(q >> sh) ^ c[1] ^ u64(key[0]), q & low, (p >> sh) ^ c[3] ^ u64(key[1]), p & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    drawn = np.empty((T, blocks, 8), np.uint16)
    for j in range(4):
        drawn[..., 2 * j] = c[j] & u64(0xFFFF)
        drawn[..., 2 * j + 1] = c[j] >> u64(16)
    cut = int(case["p"] * 65536 + 0.5)
    keep = torch.from_numpy(drawn.reshape(T, -1)[:, :K].astype(np.int32)).to(DEV) >= cut
    factor = keep.double() * (65536.0 / (65536 - cut))
    y = s["x"].double() * factor
    if s["residual"] is not None:
        y += s["residual"].double()
    return y, s["dy"].double() * factor


def _exact_norms(case, s):
    """The definition by torch's own operations in 64 bits, nothing rounded on the way, and autograd's
    gradients of it."""
    names = [k for k in ("x", "delta", "post", "pre", "gate") if s[k] is not None]
    leaf = {k: s[k].double().requires_grad_() for k in names}

    def rms(v, w):
        return v / torch.sqrt(torch.square(v).mean(-1, keepdim=True) + EPS) * w

    branch = rms(leaf["delta"], leaf["post"]) if "post" in leaf else leaf["delta"] * 1.0
    if "gate" in leaf:
        branch = branch * leaf["gate"]
    y = torch.add(leaf["x"], branch, alpha=case["scale"])
    outs = [y] + ([rms(y, leaf["pre"])] if "pre" in leaf else [])
    if not case["grad"]:
        return tuple(o.detach() for o in outs)
    grads = torch.autograd.grad(outs, [leaf[k] for k in names], [s["dy"].double(), s["dh"].double() if "pre" in leaf else None][:len(outs)])
    return tuple(o.detach() for o in outs) + grads


def exact(case, seed):
    return {"ce": _exact_ce, "dropout": _exact_dropout, "norms": _exact_norms}[case["op"]](case, prepare(case, seed))
