"""ops.block_norms(inplace=True) on CPU: what autograd sees of the write."""
import pytest
import torch

from mlx_swift_lm_b200 import ops

DEV = "cpu"


def _graph_then_inplace(dev):
    x, d = torch.randn(4, 64, device=dev), torch.randn(4, 64, device=dev)
    w = torch.randn(64, device=dev, requires_grad=True)
    z = x * w  # saves x for w's gradient
    with torch.no_grad():
        ops.block_norms(x, d, None, torch.ones(64, device=dev), inplace=True)
    return z


def test_a_saved_x_is_seen_to_have_changed():
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        _graph_then_inplace(DEV).sum().backward()


def test_views_share_the_version():
    x = torch.randn(2, 3, 64, device=DEV)
    before = x._version
    ops.block_norms(x.view(6, 64), torch.randn(6, 64, device=DEV), torch.ones(64, device=DEV), inplace=True)
    assert x._version > before
    before = x._version
    ops.block_norms(x, torch.randn(2, 3, 64, device=DEV), torch.ones(64, device=DEV))
    assert x._version == before


def test_inference_tensors():
    with torch.inference_mode():
        x, d = torch.randn(4, 64, device=DEV), torch.randn(4, 64, device=DEV)
        want = ops.block_norms(x.clone(), d, torch.ones(64, device=DEV))[0]
        assert torch.equal(ops.block_norms(x, d, torch.ones(64, device=DEV), inplace=True)[0], want) and torch.equal(x, want)


def test_memory_that_x_shares_is_refused_or_harmless():
    T, H = 6, 32
    ones = torch.ones(H, device=DEV)

    def buf():
        g = torch.Generator().manual_seed(0)
        return torch.randn(T + 1, 3 * H, generator=g).to(DEV)

    def run(make):
        args = make(buf())
        want = ops.block_norms(args[0].clone(), *(None if a is None else a.clone() for a in args[1:4]), gate=args[4].clone() if len(args) > 4 else None)
        got = ops.block_norms(*args[:4], gate=args[4] if len(args) > 4 else None, inplace=True)
        assert got[0] is args[0] and all(torch.equal(a, b) for a, b in zip(got, want))

    flat = lambda b: b.reshape(-1)[:(T + 1) * H].view(T + 1, H)  # noqa: E731  (packed rows)
    fine = [lambda b: (b[:T, :H], b[:T, H:2 * H], ones, ones),           # columns of one buffer
            lambda b: (b[:T, H:2 * H], b[:T, :H], ones, ones, b[:T, 2 * H:]),
            lambda b: (b[1:, :H], b[:T, H:2 * H], ones, ones),
            lambda b: (b[:T, :H], b[:T, :H], ones, ones),                # x itself
            lambda b: (b[:T, :H], b[:T, :H], ones, ones, b[:T, :H]),
            lambda b: (flat(b)[:T], flat(b)[:T], ones, ones),
            lambda b: (b[:T, :H], b[:T, H:2 * H], b[2, H:2 * H], b[0, 2 * H:])]
    for make in fine:
        run(make)
    bad = [lambda b: (flat(b)[:T], flat(b)[1:], ones, ones),             # one row further
           lambda b: (flat(b)[1:], flat(b)[:T], ones, ones),
           lambda b: (b[:T, :H], b[:T, 1:H + 1], ones, ones),            # one column further
           lambda b: (b[:T, 2 * H:], b.reshape(-1)[3 * H - 1:3 * H - 1 + 3 * H * T].view(T, 3 * H)[:, :H], ones, ones),
           lambda b: (flat(b)[:T], b.reshape(-1)[-T * H:].view(T, H), flat(b)[2], ones),
           lambda b: (flat(b)[:T], b.reshape(-1)[-T * H:].view(T, H), ones, flat(b)[0]),
           lambda b: (flat(b)[:T], b.reshape(-1)[-T * H:].view(T, H), ones, ones, flat(b)[3]),
           lambda b: (flat(b)[:T], b.reshape(-1)[-T * H:].view(T, H), ones, ones, flat(b)[1:]),
           lambda b: (flat(b)[:T], b.reshape(-1)[-T * H:].view(T, H), ones, ones, flat(b)[0, :T, None])]
    for make in bad:
        b = buf()
        args = make(b)
        with pytest.raises(ValueError, match="shares"):
            ops.block_norms(*args[:4], gate=args[4] if len(args) > 4 else None, inplace=True)
        assert torch.equal(b, buf())
        ops.block_norms(*args[:4], gate=args[4] if len(args) > 4 else None)  # out of place all of them run


def test_one_row_that_shares_memory():
    b = torch.randn(40, device=DEV)
    x, ones = b[:32].expand(1, 32).as_strided((1, 32), (0, 1)), torch.ones(32, device=DEV)
    with pytest.raises(ValueError, match="shares"):
        ops.block_norms(x, b[8:][None], ones, inplace=True)
    with pytest.raises(ValueError, match="shares"):
        ops.block_norms(x, torch.zeros(1, 32, device=DEV), b[1:33], inplace=True)
    want = ops.block_norms(x.clone(), x.clone(), ones)[0]
    assert torch.equal(ops.block_norms(x, x, ones, inplace=True)[0], want)
