"""Norm and position rotation of queries and keys: host side of fa_norm_rope,
fa_norm_rope_bwd and fa_norm_rope_and_cache.

The reference has neither: its callers norm and rotate q and k before they
call it.  Here the two steps are one pass over q and k, and in serving the same
pass writes the keys and values into the paged cache that
tilelang_paged_forward and tilelang_decode_forward read.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, _native
from ._checks import require_cuda, require_half, require_same, rows_ready, strides


def _check_heads(q, k, dims):
    for name, t in (("q", q), ("k", k)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
        require_half(t, name)
    require_same({"q": q, "k": k}, "dtype")
    if q.dim() not in dims or k.dim() != q.dim() or q.shape[:-2] != k.shape[:-2] or \
            q.shape[-1] != k.shape[-1]:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must be "
                         "[..., heads, head_dim] of the same tokens and head_dim")
    D = q.shape[-1]
    if D % 8 != 0 or not 16 <= D <= 512:
        raise ValueError(f"head_dim {D} must be a multiple of 8 in [16, 512]")
    if q.shape[-2] == 0 or k.shape[-2] == 0:
        raise ValueError("q and k need at least one head")


def _check_tables(cos, sin, D):
    for name, t in (("cos", cos), ("sin", sin)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
        if t.dtype != torch.float32:
            raise TypeError(f"{name} must be float32, got {t.dtype}")
        if t.requires_grad:
            raise ValueError(f"{name} gets no gradient: pass {name}.detach()")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[0] == 0:
        raise ValueError("cos / sin must both be [num_positions, rotary_dim / 2]")
    R = 2 * cos.shape[1]
    if R % 16 != 0 or not 16 <= R <= D:
        raise ValueError(f"rotary_dim {R} must be a multiple of 16 in [16, head_dim {D}]")
    return R


def _check_weights(q, q_weight, k_weight):
    D = q.shape[-1]
    given = [(n, w) for n, w in (("q_weight", q_weight), ("k_weight", k_weight)) if w is not None]
    for name, w in given:
        if not isinstance(w, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor or None, got {type(w).__name__}")
        if w.dtype not in (torch.float32, q.dtype):
            raise TypeError(f"{name} must be float32 or {q.dtype}, got {w.dtype}")
        if w.shape != (D,):
            raise ValueError(f"{name} must have shape ({D},), got {tuple(w.shape)}")
    if len(given) == 2:
        require_same(dict(given), "dtype")


def _check_positions(positions, shape, name="positions"):
    if not isinstance(positions, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(positions).__name__}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be an integer tensor, got {positions.dtype}")
    if positions.shape not in (shape, shape[-1:]):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(positions.shape)}")


def _require_place(named):
    for name, t in named.items():
        require_cuda(t, name)
    require_same(named, "device")


def _table_ready(t):
    """t, or a contiguous copy where the kernels cannot read 16 bytes of a row at a time."""
    ok = t.stride(1) == 1 and t.data_ptr() % 16 == 0 and \
        (t.shape[0] == 1 or (t.stride(0) >= 0 and t.stride(0) % 4 == 0))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _weight_ready(w):
    if w is None or (w.is_contiguous() and w.data_ptr() % 16 == 0):
        return w
    return w.clone(memory_format=torch.contiguous_format)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _strides4(t):
    """{batch, seq, head} strides of [B, S, H, D] or [T, H, D]."""
    return strides(t, 3) if t.dim() == 4 else (0, *strides(t, 2))


def _fill(a, q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved):
    """The fields fa_norm_rope and its backward share; returns what must stay alive."""
    cos, sin = _table_ready(cos), _table_ready(sin)
    q_weight, k_weight = _weight_ready(q_weight), _weight_ready(k_weight)
    a.q_weight, a.k_weight = _ptr(q_weight), _ptr(k_weight)
    a.cos, a.sin = cos.data_ptr(), sin.data_ptr()
    a.table_stride[:] = (strides(cos, 1)[0], strides(sin, 1)[0])
    if positions is not None:
        positions = positions.to(device=q.device, dtype=torch.int64)
        a.positions = positions.data_ptr()
        s = positions.stride()
        a.pos_stride[:] = (s[0], s[1]) if positions.dim() == 2 else (0, s[0])
    a.num_positions = cos.shape[0]
    a.batch, a.seqlen = (q.shape[0], q.shape[1]) if q.dim() == 4 else (1, q.shape[0])
    a.num_heads, a.num_heads_k, a.head_dim = q.shape[-2], k.shape[-2], q.shape[-1]
    a.rotary_dim = 2 * cos.shape[1]
    a.interleaved = int(bool(interleaved))
    a.weight_f32 = int((q_weight if q_weight is not None else k_weight).dtype == torch.float32) \
        if q_weight is not None or k_weight is not None else 0
    a.dtype = _lib.dtype_code(q.dtype)
    a.eps = float(eps)
    return cos, sin, q_weight, k_weight, positions


def _forward(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved):
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    if q.numel() == 0:
        return q_out, k_out
    q, k = rows_ready(q), rows_ready(k)
    a = _lib.NormRopeArgs()
    keep = _fill(a, q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved)
    a.q, a.k, a.q_out, a.k_out = q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr()
    a.q_stride[:], a.k_stride[:] = _strides4(q), _strides4(k)
    a.qo_stride[:], a.ko_stride[:] = _strides4(q_out), _strides4(k_out)
    lib = _lib.load()
    _lib.check(_lib.call_on(q.device, lambda st: lib.fa_norm_rope(ctypes.byref(a), st)),
               "fa_norm_rope")
    del keep
    return q_out, k_out


def _backward(q, k, dq_out, dk_out, cos, sin, q_weight, k_weight, positions, eps, interleaved):
    """q / k (None where the weight is None) and the outputs' gradients -> the gradients."""
    done = _native.norm_rope_bwd(q, k, dq_out, dk_out, cos, sin, q_weight, k_weight, positions,
                                 eps, interleaved)
    if done is not None:
        return done
    dq_out, dk_out = rows_ready(dq_out), rows_ready(dk_out)
    dq = torch.empty(dq_out.shape, dtype=dq_out.dtype, device=dq_out.device)
    dk = torch.empty(dk_out.shape, dtype=dk_out.dtype, device=dk_out.device)
    dqw, dkw = (torch.empty(w.shape, dtype=w.dtype, device=w.device) if w is not None else None
                for w in (q_weight, k_weight))
    if dq_out.numel() == 0:
        return dq, dk, *(w.zero_() if w is not None else None for w in (dqw, dkw))
    a = _lib.NormRopeBwdArgs()
    keep = _fill(a, dq_out, dk_out, cos, sin, q_weight, k_weight, positions, eps, interleaved)
    if q is not None:
        q = rows_ready(q)
        a.q, a.q_stride[:] = q.data_ptr(), _strides4(q)
    if k is not None:
        k = rows_ready(k)
        a.k, a.k_stride[:] = k.data_ptr(), _strides4(k)
    a.dq_out, a.dk_out, a.dq, a.dk = (t.data_ptr() for t in (dq_out, dk_out, dq, dk))
    a.dqo_stride[:], a.dko_stride[:] = _strides4(dq_out), _strides4(dk_out)
    a.dq_stride[:], a.dk_stride[:] = _strides4(dq), _strides4(dk)
    a.dq_weight, a.dk_weight = _ptr(dqw), _ptr(dkw)
    lib = _lib.load()

    def run(stream):
        # The size depends on the current device (its CU count).
        nbytes = lib.fa_norm_rope_bwd_workspace_bytes(ctypes.byref(a))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dq.device) if nbytes else None
        return lib.fa_norm_rope_bwd(ctypes.byref(a), _ptr(ws), nbytes, stream)

    _lib.check(_lib.call_on(dq.device, run), "fa_norm_rope_bwd")
    del keep
    return dq, dk, dqw, dkw


class QkNormRopeFunc(torch.autograd.Function):
    """qk_norm_rope under autograd, where the native node does not take the call: saves
    its inputs alone (q and k only where they are normed; a rotation's gradient needs
    neither)."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved):
        q_out, k_out = _norm_rope(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved)
        ctx.save_for_backward(q if q_weight is not None else None,
                              k if k_weight is not None else None,
                              cos, sin, q_weight, k_weight, positions)
        ctx.shapes = q.shape, k.shape
        ctx.like = q.dtype, q.device
        ctx.eps, ctx.interleaved = eps, interleaved
        ctx.set_materialize_grads(False)
        return q_out, k_out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, cos, sin, q_weight, k_weight, positions = ctx.saved_tensors
        dtype, device = ctx.like
        grads = [torch.zeros(s, dtype=dtype, device=device) if g is None else g.to(dtype)
                 for g, s in zip((dq_out, dk_out), ctx.shapes)]
        dq, dk, dqw, dkw = _backward(q, k, *grads, cos, sin, q_weight, k_weight, positions,
                                     ctx.eps, ctx.interleaved)
        return dq, dk, None, None, dqw, dkw, None, None, None


def _norm_rope(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved):
    done = _native.norm_rope(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved,
                             False)
    if done is not None:
        return done
    _check_heads(q, k, (3, 4))
    _check_tables(cos, sin, q.shape[-1])
    _check_weights(q, q_weight, k_weight)
    if positions is not None:
        _check_positions(positions, q.shape[:-2])
    named = {"q": q, "k": k, "cos": cos, "sin": sin, "q_weight": q_weight, "k_weight": k_weight}
    _require_place({n: t for n, t in named.items() if t is not None})
    return _forward(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved)


def qk_norm_rope(q, k, cos, sin, q_weight=None, k_weight=None, positions=None, eps=1e-6,
                 interleaved=False):
    """Per-head RMS norm and position rotation of queries and keys, in one pass.

    Args:
        q, k: [B, S, H, D] and [B, S, Hk, D], or [T, H, D] and [T, Hk, D]; fp16
            or bf16, D a multiple of 8 in [16, 512].
        cos, sin: [num_positions, R / 2] fp32, the rotation of each position;
            R a multiple of 16 up to D, components from R on are not rotated.
        q_weight, k_weight: [D] in fp32 or q's dtype, the norms' weights; None:
            that tensor is rotated without a norm.
        positions: [B, S], [S] or [T] integers, the rows of cos and sin; None:
            0 .. S - 1 (0 .. T - 1).  A negative position marks padding: its
            rows come out zero.  One beyond the tables gives NaN.
        eps: added to the mean of the squares.
        interleaved: components 2i and 2i + 1 form a pair instead of i and
            i + R / 2.
    Returns:
        (q_out, k_out), new contiguous tensors.  Differentiable with respect to
        q, k and the weights.  Computed in fp32, rounded once.
    """
    done = _native.norm_rope(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved,
                             None)
    if done is not None:
        return done
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad
                                       for t in (q, k, q_weight, k_weight)):
        _native.refuse_foreign_leaves({"q": q, "k": k, "q_weight": q_weight,
                                       "k_weight": k_weight})
        done = _native.norm_rope(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved,
                                 True)
        if done is not None:
            return done
        return QkNormRopeFunc.apply(q, k, cos, sin, q_weight, k_weight, positions, eps,
                                    interleaved)
    return _norm_rope(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved)


def norm_rope_and_cache(q, k, v, key_cache, value_cache, slot_mapping, positions, cos, sin,
                        q_weight=None, k_weight=None, eps=1e-6, interleaved=False):
    """qk_norm_rope on new tokens, with the keys and values written to the paged cache.

    Args:
        q: [T, H, D]; k, v: [T, Hkv, D] (views of one projection's output are
            taken as they are).
        key_cache, value_cache: [num_pages, page_size, Hkv, D], modified in place.
        slot_mapping: [T] integers; token t's normed and rotated key and its
            value go to page slot // page_size, slot slot % page_size.  A slot
            outside the caches (negative: padding) is skipped, as in
            reshape_and_cache.  Slots inside them must be distinct.
        positions: [T] integers, rows of cos and sin.
        cos, sin, q_weight, k_weight, eps, interleaved: as for qk_norm_rope.
    Returns:
        The normed and rotated q, a new [T, H, D] tensor.  No gradients.
    """
    done = _native.norm_rope_cache(q, k, v, key_cache, value_cache, slot_mapping, positions, cos,
                                   sin, q_weight, k_weight, eps, interleaved)
    if done is not None:
        return done
    _check_heads(q, k, (3,))
    for name, t in (("v", v), ("key_cache", key_cache), ("value_cache", value_cache)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    require_same({"q": q, "v": v, "key_cache": key_cache, "value_cache": value_cache}, "dtype")
    T, Hkv, D = k.shape
    if v.shape != k.shape:
        raise ValueError(f"v {tuple(v.shape)} must have k's shape {tuple(k.shape)}")
    if key_cache.dim() != 4 or value_cache.shape != key_cache.shape or \
            key_cache.shape[2:] != (Hkv, D):
        raise ValueError("key_cache / value_cache must both be "
                         f"[num_pages, page_size, {Hkv}, {D}]")
    if key_cache.shape[1] == 0:
        raise ValueError("page_size must be positive")
    _check_tables(cos, sin, D)
    _check_weights(q, q_weight, k_weight)
    _check_positions(slot_mapping, (T,), "slot_mapping")
    _check_positions(positions, (T,))
    named = {"q": q, "k": k, "v": v, "key_cache": key_cache, "value_cache": value_cache,
             "cos": cos, "sin": sin, "q_weight": q_weight, "k_weight": k_weight}
    _require_place({n: t for n, t in named.items() if t is not None})
    for t in (key_cache, value_cache):
        if rows_ready(t) is not t:
            raise ValueError("key_cache / value_cache must have a contiguous head_dim, 16-byte "
                             "aligned rows and strides that are multiples of 8 (they are written "
                             "in place)")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if T == 0:
        return out
    slots = slot_mapping.to(device=q.device, dtype=torch.int64).contiguous()
    pos = positions.to(device=q.device, dtype=torch.int64).contiguous()
    q, k, v = rows_ready(q), rows_ready(k), rows_ready(v)
    cos, sin = _table_ready(cos), _table_ready(sin)
    q_weight, k_weight = _weight_ready(q_weight), _weight_ready(k_weight)
    a = _lib.NormRopeCacheArgs()
    a.q, a.k, a.v, a.q_out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.k_cache, a.v_cache = key_cache.data_ptr(), value_cache.data_ptr()
    a.slot_mapping, a.positions = slots.data_ptr(), pos.data_ptr()
    a.q_weight, a.k_weight = _ptr(q_weight), _ptr(k_weight)
    a.cos, a.sin = cos.data_ptr(), sin.data_ptr()
    a.q_stride[:], a.key_stride[:] = strides(q, 2), strides(k, 2)
    a.value_stride[:], a.qo_stride[:] = strides(v, 2), strides(out, 2)
    a.k_stride[:], a.v_stride[:] = strides(key_cache, 3), strides(value_cache, 3)
    a.table_stride[:] = (strides(cos, 1)[0], strides(sin, 1)[0])
    a.num_positions = cos.shape[0]
    a.num_tokens, a.num_heads, a.num_kv_heads, a.head_dim = T, q.shape[1], Hkv, D
    a.rotary_dim = 2 * cos.shape[1]
    a.num_pages, a.page_size = key_cache.shape[:2]
    a.interleaved = int(bool(interleaved))
    weight = q_weight if q_weight is not None else k_weight
    a.weight_f32 = int(weight is not None and weight.dtype == torch.float32)
    a.dtype = _lib.dtype_code(q.dtype)
    a.eps = float(eps)
    lib = _lib.load()
    _lib.check(_lib.call_on(q.device, lambda st: lib.fa_norm_rope_and_cache(ctypes.byref(a), st)),
               "fa_norm_rope_and_cache")
    return out
