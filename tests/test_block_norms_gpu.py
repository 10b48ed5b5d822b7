"""ops.block_norms on the GPU against the formula in 64 bits."""
import pytest
import torch

from mlx_swift_lm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
E32 = 2.0 ** -24


def _inputs(T, H, dtype, gate, slack=0, seed=0):
    g = torch.Generator().manual_seed(seed)

    def rows(scale=1.0):
        return (torch.randn(T, H + slack, generator=g) * scale).to(dtype).to(DEV)[:, :H]

    shape = {"": None, "channel": (H,), "row": (T, 1), "element": (T, H)}[gate]
    vec = lambda: (1 + 0.2 * torch.randn(H, generator=g)).to(dtype).to(DEV)  # noqa: E731
    gt = None if shape is None else torch.randn(*shape, generator=g).to(dtype).to(DEV)
    return dict(x=rows(3.0), delta=rows(), post_w=vec(), pre_w=vec(), gate=gt), rows(), rows()


def _half_ulp(t, dtype):
    # below the smallest normal number n the steps stay those at n: half a step is eps / 2 * max(|v|, n)
    fi = torch.finfo(dtype)
    return fi.eps / 2 * t.abs().clamp_min(fi.smallest_normal)


def _check(T, H, dtype, gate, use_post, use_pre, slack, scale, with_dy=True, offset_one=False):
    ins, dy, dh = _inputs(T, H, dtype, gate, slack)
    eps, one = 1e-6, 1.0 if offset_one else 0.0
    if not use_post:
        ins["post_w"] = None
    if not use_pre:
        ins["pre_w"] = None
    leaf = {k: None if t is None else t.detach().requires_grad_() for k, t in ins.items()}
    y, h = ops.block_norms(**leaf, eps=eps, scale=scale, offset_one=offset_one)
    d = {k: None if t is None else t.double() for k, t in ins.items()}
    g = 1.0 if d["gate"] is None else d["gate"]
    r1 = (d["delta"].square().mean(-1, keepdim=True) + eps).rsqrt() if use_post else 1.0
    dhat = d["delta"] * r1
    wp = d["post_w"] + one if use_post else torch.ones((), dtype=torch.float64, device=DEV)
    u = dhat * wp
    # a reduction adds at most 8 + 10 (+ 4 groups) terms deep and halves through the root; 32 roundings bound a value
    N = 32
    want = d["x"] + scale * g * u
    tol = _half_ulp(want, dtype) + N * E32 * (d["x"].abs() + (scale * g * u).abs())
    assert ((y.double() - want).abs() <= tol).all()
    yd = y.detach().double()  # the stream as it is held: what h and the gradients are functions of
    if use_pre:
        r2 = (yd.square().mean(-1, keepdim=True) + eps).rsqrt()
        yhat, wq = yd * r2, d["pre_w"] + one
        want = yhat * wq
        assert ((h.double() - want).abs() <= _half_ulp(want, dtype) + N * E32 * want.abs()).all()
    outs, cot = ([y, h] if with_dy else [h], [dy, dh] if with_dy else [dh]) if use_pre else ([y], [dy])
    names = [k for k in leaf if leaf[k] is not None]
    got = dict(zip(names, torch.autograd.grad(outs, [leaf[k] for k in names], cot)))
    dt = dy.double() if with_dy or not use_pre else torch.zeros_like(yd)
    mag = dt.abs()
    if use_pre:
        G = dh.double() * wq
        m = (G * yhat).mean(-1, keepdim=True)
        dt = dt + r2 * (G - yhat * m)
        mag = mag + r2 * (G.abs() + yhat.abs() * (G * yhat).abs().mean(-1, keepdim=True))
    assert ((got["x"].double() - dt).abs() <= _half_ulp(dt, dtype) + 2 * N * E32 * mag).all()
    du, dumag = scale * dt * g, abs(scale) * mag * (g if isinstance(g, float) else g.abs())
    B, Bmag = du * wp, dumag * wp.abs()
    if use_post:
        m1 = (B * dhat).mean(-1, keepdim=True)
        dd = r1 * (B - dhat * m1)
        ddmag = r1 * (Bmag + dhat.abs() * (Bmag * dhat.abs()).mean(-1, keepdim=True))
    else:
        dd, ddmag = B, Bmag
    assert ((got["delta"].double() - dd).abs() <= _half_ulp(dd, dtype) + 4 * N * E32 * ddmag).all()

    def total(name, term, tmag, dim):  # a sum over rows (or columns): the terms' errors and the additions'
        want = term.sum(dim)
        tol = _half_ulp(want, dtype) + (4 * N + term.shape[dim]) * E32 * tmag.sum(dim)
        assert ((got[name].double().reshape(want.shape) - want).abs() <= tol).all(), name

    if use_pre:
        total("pre_w", dh.double() * yhat, (dh.double() * yhat).abs(), 0)
    if use_post:
        total("post_w", du * dhat, dumag * dhat.abs(), 0)
    dg, dgmag = scale * dt * u, abs(scale) * mag * u.abs()
    if gate == "channel":
        total("gate", dg, dgmag, 0)
    elif gate == "row":
        total("gate", dg, dgmag, 1)
    elif gate == "element":
        assert ((got["gate"].double() - dg).abs() <= _half_ulp(dg, dtype) + 4 * N * E32 * dgmag).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H", [(1, 1), (3, 7), (2, 8), (5, 256), (4, 257), (9, 2561), (64, 4096), (3, 8192), (2, 8200),
                                 (3, 16384), (2, 20001), (2, 32768)])
def test_formula_and_gradients(dtype, T, H):
    _check(T, H, dtype, "", True, True, 0, 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gate", ["channel", "row", "element"])
@pytest.mark.parametrize("use_post,use_pre", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("T,H,slack", [(700, 320, 0), (37, 513, 3), (6, 1024, 8)])
def test_gates(dtype, gate, use_post, use_pre, T, H, slack):
    _check(T, H, dtype, gate, use_post, use_pre, slack, -0.22)


@pytest.mark.parametrize("offset_one", [False, True])
def test_only_the_normed_output_has_a_gradient(offset_one):
    _check(40, 384, torch.bfloat16, "channel", True, True, 0, 0.5, with_dy=False, offset_one=offset_one)


@pytest.mark.parametrize("H", [8, 256, 2304, 4096, 8192, 12160])
@pytest.mark.parametrize("offset_one", [False, True])
def test_round_branch_equals_norm_then_add_norm(H, offset_one):
    # add_rmsnorm holds a row in 48 KB of shared memory beside its 128 bytes: 12256 columns at most
    for T in (1, 3, 64, 600):
        ins, _, _ = _inputs(T, H, torch.bfloat16, "", seed=T)
        x, delta, post, pre = ins["x"].contiguous(), ins["delta"], ins["post_w"], ins["pre_w"]
        want_x = x.clone()
        want = ops.add_rmsnorm(want_x, ops.rmsnorm(delta, post, 1e-6, offset_one), pre, 1e-6, offset_one=offset_one)
        y, h = ops.block_norms(x, delta, post, pre, 1e-6, offset_one=offset_one, round_branch=True)
        assert torch.equal(y, want_x) and torch.equal(h, want)
        y2, h2 = ops.block_norms(x, delta, post, pre, 1e-6, offset_one=offset_one, round_branch=True, inplace=True)
        assert y2 is x and torch.equal(x, want_x) and torch.equal(h2, want)


def test_a_row_does_not_depend_on_its_batch():
    for H in (2304, 4096):
        ins, _, _ = _inputs(2000, H, torch.bfloat16, "")
        y, h = ops.block_norms(**ins)
        for n in (1, 7, 64, 300):
            part = {k: t[:n] if t is not None and t.dim() == 2 else t for k, t in ins.items()}
            yn, hn = ops.block_norms(**part)
            assert torch.equal(yn, y[:n]) and torch.equal(hn, h[:n])


@pytest.mark.parametrize("T,H,gate,kind", [(300, 512, "channel", 0), (300, 511, "row", 1), (40, 1024, "element", 2)])
def test_each_gradient_by_itself(T, H, gate, kind):
    ins, dy, dh = _inputs(T, H, torch.bfloat16, gate)
    leaf = {k: t.detach().requires_grad_() for k, t in ins.items()}
    all_of = dict(zip(leaf, torch.autograd.grad(ops.block_norms(**leaf), list(leaf.values()), [dy, dh])))
    for name in ins:
        one = {k: t.detach().requires_grad_(k == name) for k, t in ins.items()}
        got, = torch.autograd.grad(ops.block_norms(**one), [one[name]], [dy, dh])
        assert torch.equal(got, all_of[name]), name


def test_bad_rows_stay_alone_and_repeat_bit_for_bit():
    ins, dy, dh = _inputs(50, 640, torch.bfloat16, "")
    ins["x"] = ins["x"].clone()
    ins["x"][3] = float("nan")
    ins["x"][4] = float("inf")
    y, h = ops.block_norms(**ins)
    ok = torch.ones(50, dtype=torch.bool, device=DEV)
    ok[3:5] = False
    assert torch.isfinite(y[ok]).all() and torch.isfinite(h[ok]).all() and not torch.isfinite(h[3]).any()
    leaf = {k: None if t is None else t.detach().requires_grad_() for k, t in _inputs(900, 640, torch.bfloat16, "")[0].items()}
    _, dy, dh = _inputs(900, 640, torch.bfloat16, "")
    names = [k for k in leaf if leaf[k] is not None]
    runs = [torch.autograd.grad(ops.block_norms(**leaf), [leaf[k] for k in names], [dy, dh]) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_no_rows_and_expanded_gradients():
    w = torch.ones(64, device=DEV, requires_grad=True)
    x = torch.randn(0, 64, device=DEV, requires_grad=True)
    y, h = ops.block_norms(x, x, w, w)
    (y.sum() + h.sum()).backward()
    assert x.grad.shape == (0, 64) and (w.grad == 0).all()
    x = torch.randn(6, 5, 64, device=DEV, requires_grad=True)
    d = torch.randn(5, 6, 64, device=DEV).transpose(0, 1).requires_grad_()
    y, h = ops.block_norms(x, d, None, w)
    y.sum().backward()
    assert torch.equal(x.grad, torch.ones_like(x))


def test_captured_forward_and_backward():
    ins, dy, dh = _inputs(48, 512, torch.bfloat16, "channel")
    leaf = {k: None if t is None else t.detach().requires_grad_() for k, t in ins.items()}
    names = list(leaf)

    def step():
        return torch.autograd.grad(ops.block_norms(**leaf), [leaf[k] for k in names], [dy, dh])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for t in got:
        t.fill_(7)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_width_limit():
    with pytest.raises(ValueError):
        ops.block_norms(torch.empty(1, 32769, device=DEV), torch.empty(1, 32769, device=DEV))
