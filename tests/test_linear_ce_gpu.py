"""ops.linear_cross_entropy on the GPU against the definition in 64 bits, with
tolerances counted from the roundings."""
import math

import pytest
import torch

from mlx_swift_lm_b200 import ops
from mlx_swift_lm_b200.ops import _lib
from mlx_swift_lm_b200.ops import loss as loss_mod

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(T, V, K, ignored=0.3, lean=8.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, K, generator=g) * 1.3 / math.sqrt(K)).bfloat16()
    t = torch.randint(0, V, (T,), generator=g)
    h = (torch.randn(T, K, generator=g) + torch.rand(T, 1, generator=g) * lean * w[t].float()).bfloat16()
    t[torch.rand(T, generator=g) < ignored] = -100
    return h.to(DEV), w.to(DEV), t.to(DEV)


def _expect(h, w, t, cap, reduction, dloss):
    """((loss, tolerance), (dh, tolerance), (dw, tolerance)) in 64 bits.

    A product of K terms accumulates in fp32, 16 at a time: its error is at most
    (K / 16 + 16) 2^-23 of the terms' magnitudes S (truncation counted as a whole
    step). A loss adds two logits' errors, 2^-22 (32 + tiles / 8) for the
    exponentials and the sums of sums, and 2^-22 of d itself. An entry of G is
    then off by its bf16 rounding 2^-9, by its relative error (the exponent's
    absolute one), or at the target by the loss's; dh and dW add the second
    product's accumulation and the output's rounding."""
    T, K = h.shape
    V = w.shape[0]
    hd, wd = h.double(), w.double()
    keep = t != -100
    hd = torch.where(keep[:, None], hd, 0.0)
    y = t.clamp(0, V - 1)
    u = hd @ wd.t()
    S = hd.abs() @ wd.abs().t()
    ez = (K / 16 + 16) * 2 ** -23 * S
    if cap:
        z = cap * torch.tanh(u / cap)
        ez = ez + 8 * 2 ** -23 * cap
        slope = 1 - (z / cap) ** 2
    else:
        z, slope = u, torch.ones_like(u)
    zt = z.gather(1, y[:, None])
    d = torch.logsumexp(z.scatter(1, y[:, None], -math.inf), 1, keepdim=True) - zt
    each = torch.where(d > 0, d + torch.log1p(torch.exp(-d)), torch.log1p(torch.exp(d)))
    tiles = -(-V // 256)
    el = 2 * ez.amax(1, keepdim=True) + 2 ** -22 * (32 + tiles / 8) + 2 ** -22 * torch.where(d.isinf(), 0.0, d.abs())
    n = keep.sum().clamp_min(1)
    k1 = keep[:, None].double()
    each, el = each * k1, el * k1
    out = {"none": (each[:, 0], el[:, 0] + 2 ** -23 * each[:, 0]), "sum": (each.sum(), el.sum() + T * 2 ** -23 * each.sum()),
           "mean": (each.sum() / n, (el.sum() + T * 2 ** -23 * each.sum()) / n)}[reduction]
    dl = (dloss.double() / (n if reduction == "mean" else 1)).expand(T)[:, None] * k1
    x = torch.exp(z - zt - each)
    ex = x * (ez + el + ez.gather(1, y[:, None]) + 2 ** -20 * (1 + (z.abs() + zt.abs() + each) / 8))
    x.scatter_(1, y[:, None], torch.expm1(-each))
    ex.scatter_(1, y[:, None], el + 2 ** -22 * each)
    G = dl * x * slope
    E = 2 ** -8 * G.abs() + dl.abs() * (ex * slope + (2 * x.abs() * (ez / cap + 2 ** -21) if cap else 0.0)) + 2 ** -22 * G.abs()
    out_r = torch.finfo(torch.bfloat16).eps / 2

    def product(a, ea, b, terms):
        v, m = a @ b, a.abs() @ b.abs()
        before = ea @ b.abs() + (terms / 16 + 80) * 2 ** -23 * m
        return v, before + out_r * (v.abs() + before) + 1e-38

    return out, product(G, E, wd, V), product(G.t(), E.t(), hd, T)


def _within(got, want, what):
    v, tol = want
    err = (got.double() - v).abs()
    assert (err <= tol).all(), f"{what}: {(err / tol.clamp_min(1e-300)).max().item():.3f} of the tolerance"


def _check(T, V, K, cap=0.0, reduction="none", ignored=0.3, dh=True, dw=True, seed=0, layout=None):
    h, w, t = _inputs(T, V, K, ignored, seed=seed)
    if layout is not None:
        h, w = layout(h), layout(w)
    h, w = h.detach().requires_grad_(dh), w.detach().requires_grad_(dw)
    out = ops.linear_cross_entropy(h, w, t, softcap=cap, reduction=reduction)
    dloss = torch.rand(out.shape, generator=torch.Generator().manual_seed(3)).to(DEV)
    wl, wh, ww = _expect(h.detach(), w.detach(), t, cap, reduction, dloss)
    _within(out.detach(), wl, "loss")
    if dh or dw:
        got = list(torch.autograd.grad(out, [x for x, need in ((h, dh), (w, dw)) if need], dloss))
        if dh:
            g = got.pop(0)
            _within(g, wh, "dh")
            assert (g[t == -100] == 0).all()
        if dw:
            _within(got.pop(0), ww, "dW")
    assert _lib.read_status()["linear_ce"] == 0


SIZES = [(1, 1, 8), (1, 2, 1), (1, 300, 64), (2, 256, 13), (5, 4096, 256), (64, 257, 100), (127, 1000, 72), (128, 512, 64),
         (129, 255, 512), (300, 700, 320), (257, 5000, 1000), (70, 50257, 128)]


@pytest.mark.parametrize("T,V,K", SIZES)
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_sizes(T, V, K, reduction):
    _check(T, V, K, reduction=reduction)


@pytest.mark.parametrize("T,V,K", [(5, 300, 64), (200, 3000, 136)])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("ignored", [0.0, 0.9])
@pytest.mark.parametrize("dh,dw", [(True, False), (False, True), (False, False)])
def test_directions(T, V, K, reduction, ignored, dh, dw):
    _check(T, V, K, reduction=reduction, ignored=ignored, dh=dh, dw=dw)


@pytest.mark.parametrize("ignored", [0.0, 0.5, 0.95])
def test_many_rows(ignored):
    """More row tiles than one walk's column of them, and few scored rows among many."""
    _check(4700, 600, 64, ignored=ignored)


@pytest.mark.parametrize("T", [1, 7, 300])
def test_one_upstream_gradient_for_all(T):
    h, w, t = _inputs(T, 900, 128)
    h, w = h.requires_grad_(), w.requires_grad_()
    out = ops.linear_cross_entropy(h, w, t)
    got = torch.autograd.grad(out, [h, w], torch.full((1,), 0.37, device=DEV).expand(T))
    _, wh, ww = _expect(h.detach(), w.detach(), t, 0.0, "none", torch.full((T,), 0.37, device=DEV))
    _within(got[0], wh, "dh")
    _within(got[1], ww, "dW")


def test_the_targets_rows_lose_little_to_rounding():
    """With one upstream gradient and unsure rows the target's entries are near -1, whose rounding to bf16 does not
    show: dW is off by its own rounding, not by a second one that all rows share (which 1 / 1365 would add)."""
    h, w, t = _inputs(1365, 4000, 256, ignored=0.0, lean=0.0)
    h, w = h.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(h, w, t, reduction="mean")
    dh, dw = torch.autograd.grad(loss, [h, w])
    hd, wd = h.detach().double(), w.detach().double()
    G = torch.softmax(hd @ wd.t(), 1)
    G[torch.arange(1365, device=DEV), t] -= 1
    # rms of a bf16 rounding: at most 2^-8 / sqrt(3) of a value; twice that leaves no room for a second one of 2^-8
    for got, want in ((dh, G @ wd / 1365), (dw, G.t() @ hd / 1365)):
        assert (got.double() - want).norm() <= 1.25 * 2 ** -8 / 3 ** 0.5 * want.norm()


@pytest.mark.parametrize("T,V,K", [(1, 257, 256), (2, 3, 100), (33, 9000, 72), (64, 300, 520)])
def test_few_rows_keep_their_targets_entries(T, V, K):
    """Up to 64 rows the targets' entries of G reach dW unrounded: what is left is dW's own rounding
    (half a step) and that of other rows' entries in the same column."""
    h, w, t = _inputs(T, V, K, ignored=0.0, lean=0.0)
    t = t % max(1, V // 2)  # some rows share a target
    h, w = h.requires_grad_(), w.requires_grad_()
    weights = torch.rand(T, device=DEV) + 0.5
    dw, = torch.autograd.grad(ops.linear_cross_entropy(h, w, t), [w], weights)
    hd, wd = h.detach().double(), w.detach().double()
    G = torch.softmax(hd @ wd.t(), 1)
    G[torch.arange(T, device=DEV), t] -= 1
    want = (G * weights[:, None].double()).t() @ hd
    rows = torch.unique(t)
    half_step = torch.finfo(torch.bfloat16).eps / 2
    others = G.clone()
    others[torch.arange(T, device=DEV), t] = 0
    off = half_step * ((others.abs() * weights[:, None].double()).t() @ hd.abs())[rows]
    limit = half_step * want[rows].abs() + off + 1e-6 * (G.abs().t() @ hd.abs())[rows]
    assert ((dw.double() - want)[rows].abs() <= limit).all()


@pytest.mark.parametrize("T,V,K", [(3, 300, 64), (140, 2000, 200), (64, 50257, 96)])
def test_softcap(T, V, K):
    _check(T, V, K, cap=5.0)


@pytest.mark.parametrize("piece", [256, 768])
@pytest.mark.parametrize("T,V,K", [(40, 2000, 64), (300, 2048, 264), (9, 700, 40)])
def test_pieces_of_the_vocabulary(monkeypatch, piece, T, V, K):
    monkeypatch.setattr(loss_mod, "PIECE_BYTES", 0)
    monkeypatch.setattr(loss_mod, "MIN_PIECE", piece)
    _check(T, V, K)


@pytest.mark.parametrize("layout", [
    lambda x: torch.cat([x, torch.full_like(x[:, :8], float("nan"))], 1)[:, :x.shape[1]],  # slack behind aligned rows
    lambda x: torch.cat([torch.full_like(x[:, :3], float("nan")), x], 1)[:, 3:],  # rows that start anywhere
    lambda x: x.t().contiguous().t(),  # columns apart
])
def test_layouts(layout):
    _check(33, 600, 72, layout=layout)


def test_expanded_rows_share_their_gradient():
    h, w, t = _inputs(1, 500, 64, ignored=0.0)
    t = torch.arange(6, device=DEV)
    one = h.detach().requires_grad_()
    ops.linear_cross_entropy(one.expand(6, 64), w, t, reduction="sum").backward()
    many = h.repeat(6, 1).requires_grad_()
    ops.linear_cross_entropy(many, w, t, reduction="sum").backward()
    # the sum of six bf16 gradients, rounded
    want = many.grad.double().sum(0)
    assert ((one.grad[0].double() - want).abs() <= 6 * 2 ** -8 * many.grad.double().abs().sum(0)).all()


def test_ignored_rows_hold_anything():
    h, w, t = _inputs(300, 900, 128, ignored=0.4)
    bad = torch.tensor([float("nan"), float("inf"), torch.finfo(torch.bfloat16).min], device=DEV).bfloat16()
    dirty = torch.where((t == -100)[:, None], bad[torch.arange(300, device=DEV) % 3][:, None], h)
    runs = []
    for x in (h, dirty):
        x, v = x.detach().requires_grad_(), w.detach().requires_grad_()
        out = ops.linear_cross_entropy(x, v, t)
        runs.append((out.detach(),) + torch.autograd.grad(out.sum(), [x, v]))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_a_bad_row_stays_alone_in_the_losses():
    h, w, t = _inputs(200, 900, 128, ignored=0.0)
    good = ops.linear_cross_entropy(h, w, t)
    h = h.clone()
    h[17] = float("nan")
    h[18, 3] = float("inf")
    out = ops.linear_cross_entropy(h, w, t)
    assert out[17].isnan() and not out[18].isfinite()
    rest = torch.ones(200, dtype=torch.bool, device=DEV)
    rest[17:19] = False
    assert torch.equal(out[rest], good[rest])


@pytest.mark.parametrize("gap", [60.0, 1e4, 3e38])
def test_a_target_far_below_the_others(gap):
    """A head row of very low logits as the target: the others' probabilities keep their digits."""
    h, w, t = _inputs(40, 500, 64, ignored=0.0, lean=0.0)
    h[:, 0] = 1.0
    w[7] = 0.0
    w[7, 0] = -gap
    t[:] = 7
    a, b = h.detach().requires_grad_(), w.detach().requires_grad_()
    dh, dw = torch.autograd.grad(ops.linear_cross_entropy(a, b, t, reduction="sum"), [a, b])
    hd, wd = h.double(), w.double()
    p = torch.softmax(hd @ wd.t(), 1)
    p[:, 7] -= 1
    rest = torch.arange(500, device=DEV) != 7
    # bf16 G and the output's rounding: 2^-8 each of the terms
    want = p.t() @ hd
    assert ((dw.double() - want).abs() <= 2 * 2 ** -8 * (p.abs().t() @ hd.abs()) + 1e-6)[rest].all()
    want = p[:, rest] @ wd[rest]
    assert ((dh.double() - want)[:, 1:].abs() <= 3 * 2 ** -8 * (p[:, rest].abs() @ wd[rest].abs())[:, 1:] + 1e-6).all()


def test_targets_out_of_range_are_reported():
    h, w, t = _inputs(10, 300, 64, ignored=0.0)
    good = ops.linear_cross_entropy(h, w, t)
    for bad in (300, -1, 1 << 40, -(1 << 40)):
        t2 = t.clone()
        t2[4] = bad
        out = ops.linear_cross_entropy(h, w, t2)
        assert out[4].isnan() and torch.equal(out[:4], good[:4]) and torch.equal(out[5:], good[5:])
        assert _lib.read_status()["linear_ce"] == 8
    t2 = t.clone()
    t2[4] = 299  # the last column, and an ignore index inside the vocabulary
    assert ops.linear_cross_entropy(h, w, t2, ignore_index=299)[4] == 0


def test_nothing_scored_and_no_rows():
    h, w, t = _inputs(130, 600, 64)
    t[:] = -100
    for reduction in ("none", "sum", "mean"):
        a, b = h.detach().requires_grad_(), w.detach().requires_grad_()
        out = ops.linear_cross_entropy(a, b, t, reduction=reduction)
        out.sum().backward()
        assert (out == 0).all() and (a.grad == 0).all() and (b.grad == 0).all()
        a, b = h[:0].detach().requires_grad_(), w.detach().requires_grad_()
        out = ops.linear_cross_entropy(a, b, t[:0], reduction=reduction)
        out.sum().backward()
        assert (out == 0).all() and (b.grad == 0).all()


def test_repeats_bit_for_bit_and_does_not_depend_on_ignored_rows():
    h, w, t = _inputs(500, 3000, 256, ignored=0.0)
    pad = torch.arange(500, device=DEV) % 3 == 1
    runs = []
    for _ in range(3):
        a, b = h.detach().requires_grad_(), w.detach().requires_grad_()
        out = ops.linear_cross_entropy(a, b, torch.where(pad, -100, t), reduction="mean")
        runs.append((out.detach(),) + torch.autograd.grad(out, [a, b]))
    for r in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, runs[0]))
    out = ops.linear_cross_entropy(h[~pad], w, t[~pad], reduction="mean")
    assert torch.equal(out, runs[0][0])


def test_captured_step_with_other_inputs_and_targets():
    h, w, t = _inputs(70, 1200, 128)
    a, b = h.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    tt = t.clone()

    def step():
        out = ops.linear_cross_entropy(a, b, tt, reduction="mean")
        return (out.detach(),) + torch.autograd.grad(out, [a, b])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed, ignored in ((1, 0.0), (2, 0.9), (3, 0.5)):
        h2, w2, t2 = _inputs(70, 1200, 128, ignored, seed=seed)
        with torch.no_grad():
            a.copy_(h2), b.copy_(w2), tt.copy_(t2)
        g.replay()
        c, d = h2.requires_grad_(), w2.requires_grad_()
        out = ops.linear_cross_entropy(c, d, t2, reduction="mean")
        want = (out.detach(),) + torch.autograd.grad(out, [c, d])
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_two_streams_at_once():
    h, w, t = _inputs(256, 4000, 512)
    want = ops.linear_cross_entropy(h, w, t)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append([ops.linear_cross_entropy(h, w, t) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for k in outs for o in k)


def test_refuses_other_types():
    with pytest.raises(TypeError):
        ops.linear_cross_entropy(torch.randn(3, 8, device=DEV), torch.randn(9, 8, device=DEV),
                                 torch.zeros(3, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(torch.randn(3, 8, device=DEV).bfloat16(), torch.randn(9, 8).bfloat16(),
                                 torch.zeros(3, dtype=torch.int64, device=DEV))
