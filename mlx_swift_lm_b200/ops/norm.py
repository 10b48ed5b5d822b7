"""RMSNorm / residual / RoPE / KV-append / embedding ops."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from . import reference as ref
from ._args import ELEM, elem_code, rows2d, same_device
from .linear import num_sms

_lib.register_signatures({
    "b200_block_norms": (_lib.i32, [_lib.vp, _lib.i64, _lib.vp, _lib.i64, _lib.vp, _lib.vp, _lib.i32, _lib.vp, _lib.i64,
                                    _lib.i32, _lib.vp, _lib.i64, _lib.vp, _lib.i64, _lib.vp, _lib.vp, _lib.i64,
                                    _lib.i32, _lib.i32, _lib.f32, _lib.f32, _lib.i32, _lib.i32, _lib.i32, _lib.vp]),
    "b200_block_norms_bwd": (_lib.i32, [_lib.vp, _lib.i64, _lib.vp, _lib.i64, _lib.vp, _lib.vp, _lib.i32, _lib.vp,
                                        _lib.i64, _lib.i32, _lib.vp, _lib.vp, _lib.vp, _lib.i64, _lib.vp, _lib.i64,
                                        _lib.vp, _lib.vp, _lib.vp, _lib.vp, _lib.vp, _lib.vp, _lib.i64, _lib.i32,
                                        _lib.i32, _lib.f32, _lib.i32, _lib.i32, _lib.vp]),
    "b200_block_norms_max_width": (_lib.i32, []),
    "b200_block_norms_bwd_grid": (_lib.i32, [_lib.i64, _lib.i32, _lib.i32]),
}, status_tags=("block_norms",))


def add_rmsnorm(x: torch.Tensor, delta: torch.Tensor | None, w: torch.Tensor, eps: float,
                out: torch.Tensor | None = None, offset_one: bool = False) -> torch.Tensor:
    """x <- x + delta (in place, rounded to x.dtype); returns RMSNorm(x) * w."""
    if not x.is_cuda:
        r, y = ref.add_rmsnorm_ref(x, delta, w, eps, offset_one)
        if delta is not None:
            x.copy_(r)
        if out is not None:
            out.copy_(y)
            return out
        return y
    T, H = x.shape
    if out is None:
        out = torch.empty_like(x)
    rc = _lib.lib().b200_add_rmsnorm(x.data_ptr(), _lib.ptr(delta), w.data_ptr(), out.data_ptr(), T, H,
                                     x.stride(0), delta.stride(0) if delta is not None else 0, out.stride(0),
                                     float(eps), 1 if offset_one else 0, _lib.stream_ptr(x.device))
    _lib.check(rc, "add_rmsnorm")
    _lib.count(1)
    return out


def add_layernorm(x: torch.Tensor, delta: torch.Tensor | None, w: torch.Tensor, b: torch.Tensor | None, eps: float,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """x <- x + delta (in place, rounded to x.dtype); returns LayerNorm(x) * w + b
    (`out` may be x itself: the post-norm residual of BERT-family encoders)."""
    if not x.is_cuda:
        if delta is not None:
            x.copy_((x.float() + delta.float()).to(x.dtype))
        y = torch.nn.functional.layer_norm(x.float(), (x.shape[-1],), w.float(),
                                           None if b is None else b.float(), eps).to(x.dtype)
        if out is not None:
            out.copy_(y)
            return out
        return y
    T, H = x.shape
    if out is None:
        out = torch.empty_like(x)
    rc = _lib.lib().b200_add_layernorm(x.data_ptr(), _lib.ptr(delta), w.data_ptr(), _lib.ptr(b), out.data_ptr(), T, H,
                                       x.stride(0), delta.stride(0) if delta is not None else 0, out.stride(0),
                                       float(eps), _lib.stream_ptr(x.device))
    _lib.check(rc, "add_layernorm")
    _lib.count(1)
    return out


def rmsnorm(x, w, eps, offset_one=False):
    return add_rmsnorm(x, None, w, eps, offset_one=offset_one)


_GATE_NONE, _GATE_CHANNEL, _GATE_ROW, _GATE_ELEMENT = range(4)


def _gate_kind(gate, x) -> int:
    if gate is None:
        return _GATE_NONE
    if gate.shape == x.shape[-1:]:
        return _GATE_CHANNEL
    if gate.shape == x.shape[:-1] + (1,):
        return _GATE_ROW
    if gate.shape == x.shape:
        return _GATE_ELEMENT
    raise ValueError(f"block_norms: gate {tuple(gate.shape)} is neither {tuple(x.shape[-1:])}, "
                     f"{tuple(x.shape[:-1]) + (1,)} nor {tuple(x.shape)}")


def _block_norms_fwd(x, delta, post_w, pre_w, gate, kind, eps, scale, offset_one, round_branch, y, save):
    """(y, h, r1, r2); y is written in place when given. r1 / r2 (fp32 [T], the
    reciprocal RMS of delta and y) are kept for the backward pass with `save`."""
    H = x.shape[-1]
    dev = x.device
    if y is None:
        y = torch.empty_like(x, memory_format=torch.contiguous_format)
    h = None if pre_w is None else torch.empty_like(x, memory_format=torch.contiguous_format)
    x2, d2, y2 = rows2d(x, H), rows2d(delta, H), rows2d(y, H)
    T = x2.shape[0]
    r1 = torch.empty(T, dtype=torch.float32, device=dev) if save and post_w is not None else None
    r2 = torch.empty(T, dtype=torch.float32, device=dev) if save and pre_w is not None else None
    post_w, pre_w = (None if w is None else w.contiguous() for w in (post_w, pre_w))
    g = None if gate is None else rows2d(gate, H) if kind == _GATE_ELEMENT else gate.contiguous()
    w = post_w if post_w is not None else pre_w
    if T:
        rc = _lib.launch(
            _lib.lib().b200_block_norms, dev, x2.data_ptr(), x2.stride(0), d2.data_ptr(), d2.stride(0),
            _lib.ptr(post_w), _lib.ptr(pre_w), ELEM[x.dtype if w is None else w.dtype], _lib.ptr(g),
            g.stride(0) if kind == _GATE_ELEMENT else 0, kind, y2.data_ptr(), y2.stride(0), _lib.ptr(h), H,
            _lib.ptr(r1), _lib.ptr(r2), T, H, ELEM[x.dtype], float(eps), float(scale), 1 if offset_one else 0,
            1 if round_branch else 0, num_sms(dev))
        _lib.check(rc, "block_norms")
        _lib.count(1)
    return y, h, r1, r2


class _BlockNorms(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, post_w, pre_w, gate, kind, eps, scale, offset_one, round_branch):
        ctx.set_materialize_grads(False)
        y, h, r1, r2 = _block_norms_fwd(x, delta, post_w, pre_w, gate, kind, eps, scale, offset_one, round_branch,
                                        None, True)
        ctx.save_for_backward(y, delta, post_w, pre_w, gate, r1, r2)
        ctx.kind, ctx.scale, ctx.offset_one = kind, float(scale), bool(offset_one)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        y, delta, post_w, pre_w, gate, r1, r2 = ctx.saved_tensors
        need_x, need_d, need_post, need_pre, need_gate = ctx.needs_input_grad[:5]
        none = (None,) * 5
        if dy is None and dh is None:
            return (None,) * 5 + none
        dev, H, kind = y.device, y.shape[-1], ctx.kind

        def like(t, need):
            return torch.empty_like(t, memory_format=torch.contiguous_format) if need else None

        y2, d2 = rows2d(y, H), rows2d(delta, H)
        T = y2.shape[0]
        dx, dd, dgate, dpost, dpre = (like(y, need_x), like(delta, need_d), like(gate, need_gate),
                                      like(post_w, need_post), like(pre_w, need_pre and dh is not None))
        if T == 0:
            for t in (dgate, dpost, dpre):
                if t is not None:
                    t.zero_()
            return (dx, dd, dpost, dpre, dgate) + none
        dy2 = None if dy is None else rows2d(dy, H)
        dh2 = None if dh is None else rows2d(dh, H)
        pw, qw = (None if w is None else w.contiguous() for w in (post_w, pre_w))
        g = None if gate is None else rows2d(gate, H) if kind == _GATE_ELEMENT else gate.contiguous()
        w = pw if pw is not None else qw
        n_part = sum(t is not None for t in (dpost, dpre, dgate if kind == _GATE_CHANNEL else None))
        L, sms = _lib.lib(), num_sms(dev)
        part = (torch.empty(n_part * L.b200_block_norms_bwd_grid(T, H, sms) * H, dtype=torch.float32, device=dev)
                if n_part else None)
        rc = _lib.launch(
            L.b200_block_norms_bwd, dev, y2.data_ptr(), y2.stride(0), d2.data_ptr(), d2.stride(0), _lib.ptr(pw),
            _lib.ptr(qw), ELEM[y.dtype if w is None else w.dtype], _lib.ptr(g), g.stride(0) if kind == _GATE_ELEMENT else 0,
            kind, _lib.ptr(r1), _lib.ptr(r2), _lib.ptr(dy2), 0 if dy2 is None else dy2.stride(0), _lib.ptr(dh2),
            0 if dh2 is None else dh2.stride(0), _lib.ptr(dx), _lib.ptr(dd), _lib.ptr(dgate), _lib.ptr(dpost),
            _lib.ptr(dpre), _lib.ptr(part), T, H, ELEM[y.dtype], ctx.scale, 1 if ctx.offset_one else 0, sms)
        _lib.check(rc, "block_norms backward")
        _lib.count(2 if n_part else 1)
        return (dx, dd, dpost, dpre, dgate) + none


def block_norms(x: torch.Tensor, delta: torch.Tensor, post_w: torch.Tensor | None = None,
                pre_w: torch.Tensor | None = None, eps: float = 1e-6, gate: torch.Tensor | None = None,
                scale: float = 1.0, offset_one: bool = False, round_branch: bool = False, inplace: bool = False):
    """The norms around a block with its gate and residual scale, in one pass:

        u = RMSNorm(delta) * post_w   (delta itself without post_w)
        y = x + scale * gate * u      (rounded to x's dtype)
        h = RMSNorm(y) * pre_w        (None without pre_w)

    Returns (y, h), differentiable in x, delta, the weights and the gate. x and
    delta [..., H] (bf16, fp16 or fp32, H up to 32768); gate of x's dtype with
    shape [H], [..., 1] or [..., H]; post_w and pre_w [H] of one dtype, x's or fp32.
    `offset_one`: the weights are stored minus one. `round_branch`: u is rounded
    to x's dtype before the gate, as a separate norm and add would (bit-equal to
    ``add_rmsnorm(x, rmsnorm(delta, post_w), pre_w)``). `inplace`: y is written
    into x (no gradients).
    """
    H = x.shape[-1] if x.dim() else 0
    if x.dim() == 0 or H == 0:
        raise ValueError("block_norms: x needs at least one column")
    elem_code(x, "block_norms")
    if delta.shape != x.shape or delta.dtype != x.dtype:
        raise ValueError(f"block_norms: delta {tuple(delta.shape)} {delta.dtype} for x {tuple(x.shape)} {x.dtype}")
    kind = _gate_kind(gate, x)
    if gate is not None and gate.dtype != x.dtype:
        raise TypeError(f"block_norms: gate {gate.dtype} for x {x.dtype}")
    for w in (post_w, pre_w):
        if w is not None and w.shape != (H,):
            raise ValueError(f"block_norms: weight {tuple(w.shape)} for rows of {H}")
        if w is not None and w.dtype != x.dtype and w.dtype != torch.float32:
            raise TypeError(f"block_norms: weight {w.dtype} for x {x.dtype}")
    if post_w is not None and pre_w is not None and post_w.dtype != pre_w.dtype:
        raise TypeError(f"block_norms: post_w {post_w.dtype}, pre_w {pre_w.dtype}")
    same_device("block_norms", x, delta, post_w, pre_w, gate)
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, delta, post_w, pre_w, gate))
    if inplace:
        if grad:
            raise ValueError("block_norms: inplace takes no gradients")
        rows = x.view(-1, H)
        if x.numel() and ((H > 1 and rows.stride(1) != 1) or (rows.shape[0] > 1 and rows.stride(0) < H)):
            raise ValueError("block_norms: inplace needs rows of neighbouring columns that do not overlap")
    if not x.is_cuda:
        y, h = ref.block_norms_ref(x, delta, post_w, pre_w, eps, gate, scale, offset_one, round_branch)
        return (x.copy_(y) if inplace else y), h
    if H > _lib.lib().b200_block_norms_max_width():
        raise ValueError(f"block_norms: {H} columns, at most {_lib.lib().b200_block_norms_max_width()}")
    if grad:
        return _BlockNorms.apply(x, delta, post_w, pre_w, gate, kind, eps, scale, offset_one, round_branch)
    return _block_norms_fwd(x, delta, post_w, pre_w, gate, kind, eps, scale, offset_one, round_branch,
                            x if inplace else None, False)[:2]


def qk_norm_rope_kv(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor | None, cos_sin: torch.Tensor,
                    rot_dim: int, interleaved: bool, q_norm: torch.Tensor | None, k_norm: torch.Tensor | None,
                    eps: float, k_cache: torch.Tensor | None, v_cache: torch.Tensor | None, H: int, KVH: int, D: int,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    q_out: torch.Tensor | None = None, return_kv: bool = False):
    """Split fused qkv [T, (H+2KVH)*D], qk-norm, RoPE, and append K/V to the
    paged cache at `slots` (page*16+offset; -1 skips). Returns q [T, H, D]
    (and k, v [T, KVH, D] when return_kv)."""
    T = qkv.shape[0]
    if not qkv.is_cuda:
        q, k, v = ref.qk_norm_rope_kv_ref(qkv, positions, slots, cos_sin, rot_dim, interleaved, q_norm, k_norm, eps,
                                          k_cache, v_cache, H, KVH, D, k_scale, v_scale)
        if q_out is not None:
            q_out.copy_(q)
            q = q_out
        return (q, k, v) if return_kv else q
    if q_out is None:
        q_out = torch.empty((T, H, D), dtype=qkv.dtype, device=qkv.device)
    k_out = v_out = None
    if return_kv:
        k_out = torch.empty((T, KVH, D), dtype=qkv.dtype, device=qkv.device)
        v_out = torch.empty((T, KVH, D), dtype=qkv.dtype, device=qkv.device)
    kv_fp8 = k_cache is not None and k_cache.dtype == torch.float8_e4m3fn
    num_slots = k_cache.shape[0] * 16 if k_cache is not None else 0
    rc = _lib.lib().b200_qk_norm_rope_kv(
        qkv.data_ptr(), T, qkv.stride(0), positions.data_ptr(), _lib.ptr(slots), cos_sin.data_ptr(), rot_dim,
        1 if interleaved else 0, _lib.ptr(q_norm), _lib.ptr(k_norm), float(eps), q_out.data_ptr(),
        _lib.ptr(k_cache), _lib.ptr(v_cache), 1 if kv_fp8 else 0, _lib.ptr(k_scale), _lib.ptr(v_scale), H, KVH, D,
        num_slots, _lib.ptr(k_out), _lib.ptr(v_out), _lib.stream_ptr(qkv.device))
    _lib.check(rc, "qk_norm_rope_kv")
    _lib.count(1)
    return (q_out, k_out, v_out) if return_kv else q_out


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, out: torch.Tensor | None = None):
    if not ids.is_cuda:
        y = table[ids.long()]
        if scale != 1.0:
            y = (y.float() * scale).to(table.dtype)
        if out is not None:
            out.copy_(y)
            return out
        return y
    T = ids.shape[0]
    H = table.shape[1]
    if out is None:
        out = torch.empty((T, H), dtype=table.dtype, device=table.device)
    rc = _lib.lib().b200_embedding(ids.data_ptr(), table.data_ptr(), out.data_ptr(), T, H, table.shape[0],
                                   float(scale), _lib.stream_ptr(ids.device))
    _lib.check(rc, "embedding")
    _lib.count(1)
    return out


def silu_mul(gu: torch.Tensor, out: torch.Tensor | None = None):
    """[T, 2F] laid out [gate | up] -> silu(gate) * up."""
    T, F2 = gu.shape
    F = F2 // 2
    if not gu.is_cuda:
        y = (torch.nn.functional.silu(gu[:, :F].float()) * gu[:, F:].float()).to(gu.dtype)
        if out is not None:
            out.copy_(y)
            return out
        return y
    if out is None:
        out = torch.empty((T, F), dtype=gu.dtype, device=gu.device)
    rc = _lib.lib().b200_silu_mul(gu.data_ptr(), out.data_ptr(), T, F, gu.stride(0), out.stride(0),
                                  _lib.stream_ptr(gu.device))
    _lib.check(rc, "silu_mul")
    _lib.count(1)
    return out


def xielu(x: torch.Tensor, params: torch.Tensor) -> torch.Tensor:
    """xIELU activation in place (Apertus MLPs). params = raw (alpha_p,
    alpha_n, beta, eps) of the layer (fp32 [4]); see xielu_ref."""
    if not x.is_cuda:
        x.copy_(ref.xielu_ref(x, params))
        return x
    assert x.dtype == torch.bfloat16 and x.is_contiguous()
    rc = _lib.lib().b200_xielu(x.data_ptr(), x.numel(), params.data_ptr(), _lib.stream_ptr(x.device))
    _lib.check(rc, "xielu")
    _lib.count(1)
    return x


_lib.register_signatures({"b200_xielu": (_lib.i32, [_lib.vp, _lib.i64, _lib.vp, _lib.vp])})
