"""Linear attention with a decay for each head: host side of fa_linear_fwd,
fa_linear_bwd and fa_linear_decode.

    S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,    o_t = scale q_t S_t

The reference has softmax attention only; this is the attention whose memory is
one [D, D] matrix a head instead of a cache of keys and values.  Tensors have
the layouts of the softmax entry points: [B, S, H, D] in training, packed
[T, H, D] with query_start_loc in prefill, [B, H, D] in decode.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, _native
from ._checks import (HEAD_DIMS, as_int32, require_cuda, require_half, require_same, rows_ready,
                      strides)


def _check_qkv(q, k, v, layout):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
        require_half(t, name)
    require_same({"q": q, "k": k, "v": v}, "dtype")
    if q.dim() != len(layout) or k.dim() != q.dim() or k.shape != v.shape or \
            k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} must be "
                         f"[{', '.join(layout)}] of the same tokens and head_dim, k and v with "
                         "num_heads_k heads")
    H, Hk, D = q.shape[-2], k.shape[-2], q.shape[-1]
    if D not in HEAD_DIMS:
        raise ValueError(f"head_dim {D} not supported (expected one of {HEAD_DIMS})")
    if Hk == 0 or H == 0 or H % Hk != 0:
        raise ValueError(f"num_heads {H} is not a multiple of num_heads_k {Hk}")
    return H, Hk, D


def _check_decay(log_decay, H):
    if not isinstance(log_decay, torch.Tensor):
        raise TypeError(f"log_decay must be a torch.Tensor, got {type(log_decay).__name__}")
    if log_decay.dtype != torch.float32:
        raise TypeError(f"log_decay must be float32, got {log_decay.dtype}")
    if log_decay.shape != (H,):
        raise ValueError(f"log_decay must have shape ({H},), got {tuple(log_decay.shape)}")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError("log_decay gets no gradient: pass log_decay.detach()")


def _check_state(state, name, shape):
    if not isinstance(state, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(state).__name__}")
    if state.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {state.dtype}")
    if state.dim() != 4 or state.shape[1:] != shape[1:] or (shape[0] is not None
                                                            and state.shape[0] != shape[0]):
        raise ValueError(f"{name} must have shape {tuple('N' if s is None else s for s in shape)}, "
                         f"got {tuple(state.shape)}")


def _state_ready(t):
    """Whether the kernels can address it: contiguous 16-byte aligned matrices."""
    D = t.shape[-1]
    return t.stride(-1) == 1 and t.stride(-2) == D and t.data_ptr() % 16 == 0 and all(
        n == 1 or (s >= 0 and s % 4 == 0) for n, s in zip(t.shape[:2], t.stride()[:2]))


def _state_rows(t):
    return t if _state_ready(t) else t.clone(memory_format=torch.contiguous_format)


def _check_pool(state, H, D):
    _check_state(state, "state", (None, H, D, D))
    if state.shape[0] == 0:
        raise ValueError("state must hold at least one slot")
    if not _state_ready(state) or any(n > 1 and s < D * D
                                      for n, s in zip(state.shape[:2], state.stride()[:2])):
        raise ValueError("state must be made of contiguous, 16-byte aligned [head_dim, head_dim] "
                         "matrices that do not overlap (it is updated in place)")


def _require_place(named):
    for name, t in named.items():
        require_cuda(t, name)
    require_same(named, "device")


def _rows(t):
    """rows_ready, and a copy where the sequence stride is 2^24 elements or more."""
    t = rows_ready(t)
    return t if t.stride(-3) < 1 << 24 or t.shape[-3] == 1 else t.contiguous()


def _scale(scale, D):
    return float(scale) if scale is not None else D ** -0.5


def _strides3(t):
    """{batch, seq, head} strides of [B, S, H, D] or [T, H, D]."""
    return strides(t, 3) if t.dim() == 4 else (0, *strides(t, 2))


def _set_qkv(a, q, k, v, log_decay, scale):
    a.q, a.k, a.v, a.log_decay = (t.data_ptr() for t in (q, k, v, log_decay))
    a.num_heads, a.num_heads_k, a.head_dim = q.shape[-2], k.shape[-2], q.shape[-1]
    a.scale = scale
    a.dtype = _lib.dtype_code(q.dtype)


def _launch_fwd(a, device):
    lib = _lib.load()

    def run(stream):
        # The size depends on the current device (its CU count).
        nbytes = lib.fa_linear_fwd_workspace_bytes(ctypes.byref(a))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        return lib.fa_linear_fwd(ctypes.byref(a), ws.data_ptr() if ws is not None else None,
                                 nbytes, stream)

    _lib.check(_lib.call_on(device, run), "fa_linear_fwd")


# ------------------------------------------------------------------ training

def _forward(q, k, v, log_decay, scale, initial_state, want_final):
    done = _native.linear_dense_fwd(q, k, v, log_decay, scale, initial_state, want_final, False)
    if done is not None:
        return done
    H, Hk, D = _check_qkv(q, k, v, ("batch", "seqlen", "heads", "head_dim"))
    B, S = q.shape[:2]
    _check_decay(log_decay, H)
    if initial_state is not None:
        _check_state(initial_state, "initial_state", (B, H, D, D))
    named = {"q": q, "k": k, "v": v, "log_decay": log_decay, "initial_state": initial_state}
    _require_place({n: t for n, t in named.items() if t is not None})
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if B == 0 or S == 0:
        final = None
        if want_final:
            final = initial_state.clone() if initial_state is not None else \
                torch.zeros((B, H, D, D), dtype=torch.float32, device=q.device)
        return out, final
    final = torch.empty((B, H, D, D), dtype=torch.float32, device=q.device) if want_final else None
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    a = _lib.LinearArgs()
    _set_qkv(a, q, k, v, log_decay, scale)
    a.out = out.data_ptr()
    a.q_stride[:], a.k_stride[:] = strides(q, 3), strides(k, 3)
    a.v_stride[:], a.o_stride[:] = strides(v, 3), strides(out, 3)
    a.batch, a.seqlen, a.num_states = B, S, B
    if initial_state is not None:
        initial_state = _state_rows(initial_state)
        a.initial_state, a.is_stride[:] = initial_state.data_ptr(), strides(initial_state, 2)
    if final is not None:
        a.final_state, a.fs_stride[:] = final.data_ptr(), strides(final, 2)
    _launch_fwd(a, q.device)
    return out, final


def _backward(q, k, v, dout, log_decay, scale, initial_state, d_final, want_d_initial):
    """(dq, dk, dv, d_initial_state or None)."""
    done = _native.linear_dense_bwd(q, k, v, dout, log_decay, scale, initial_state, d_final,
                                    want_d_initial)
    if done is not None:
        return done
    B, S, H, D = q.shape
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    if B == 0 or S == 0:
        d_initial = None
        if want_d_initial:
            d_initial = d_final.clone() if d_final is not None else \
                torch.zeros((B, H, D, D), dtype=torch.float32, device=q.device)
        return dq, dk, dv, d_initial
    d_initial = torch.empty((B, H, D, D), dtype=torch.float32, device=q.device) \
        if want_d_initial else None
    q, k, v, dout = _rows(q), _rows(k), _rows(v), _rows(dout)
    log_decay = log_decay.contiguous()
    a = _lib.LinearBwdArgs()
    _set_qkv(a, q, k, v, log_decay, scale)
    a.dout, a.dq, a.dk, a.dv = (t.data_ptr() for t in (dout, dq, dk, dv))
    for name, t in (("q", q), ("k", k), ("v", v), ("do", dout), ("dq", dq), ("dk", dk),
                    ("dv", dv)):
        getattr(a, f"{name}_stride")[:] = strides(t, 3)
    a.batch, a.seqlen = B, S
    if initial_state is not None:
        initial_state = _state_rows(initial_state)
        a.initial_state, a.is_stride[:] = initial_state.data_ptr(), strides(initial_state, 2)
    if d_final is not None:
        d_final = _state_rows(d_final)
        a.d_final_state, a.fs_stride[:] = d_final.data_ptr(), strides(d_final, 2)
    if d_initial is not None:
        a.d_initial_state, a.dis_stride[:] = d_initial.data_ptr(), strides(d_initial, 2)
    lib = _lib.load()

    def run(stream):
        nbytes = lib.fa_linear_bwd_workspace_bytes(ctypes.byref(a))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        return lib.fa_linear_bwd(ctypes.byref(a), ws.data_ptr() if ws is not None else None,
                                 nbytes, stream)

    _lib.check(_lib.call_on(q.device, run), "fa_linear_bwd")
    return dq, dk, dv, d_initial


class LinearAttnFunc(torch.autograd.Function):
    """linear_attn_func under autograd, where the native node does not take the call:
    saves its inputs alone."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, scale, initial_state, want_final):
        out, final = _forward(q, k, v, log_decay, scale, initial_state, want_final)
        ctx.save_for_backward(q, k, v, log_decay, initial_state)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (out, final) if want_final else out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, d_final=None):
        q, k, v, log_decay, initial_state = ctx.saved_tensors
        dout = torch.zeros_like(q) if dout is None else dout.to(q.dtype)
        if d_final is not None:
            d_final = d_final.float()
        dq, dk, dv, ds = _backward(q, k, v, dout, log_decay, ctx.scale, initial_state, d_final,
                                   ctx.needs_input_grad[5])
        return dq, dk, dv, None, None, ds, None


def linear_attn_func(q, k, v, log_decay, scale=None, initial_state=None,
                     return_final_state=False):
    """Causal linear attention with a decay for each head.

    Args:
        q: [B, S, H, D]; k, v: [B, S, Hk, D] with H % Hk == 0 (consecutive
            groups of H / Hk query heads share k and v); fp16 or bf16, D 64,
            128 or 256.
        log_decay: [H] fp32, the natural logarithm of each head's decay, <= 0
            (0: no decay, -inf: a token sees itself alone).  No gradient.
        scale: default 1/sqrt(D).
        initial_state: [B, H, D, D] fp32 (key component, value component), the
            state before the first token; None: zeros.
        return_final_state: also return the state after the last token.
    Returns:
        out [B, S, H, D] in q's dtype, or (out, final_state [B, H, D, D] fp32).
        Differentiable with respect to q, k, v and initial_state.

    Sums and states are fp32; a value that is not finite reaches the outputs of
    its chunk of 64 tokens, those before it in the chunk too.
    """
    scale = _scale(scale, q.shape[-1] if isinstance(q, torch.Tensor) and q.dim() else 1)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad
                                       for t in (q, k, v, log_decay, initial_state)):
        if isinstance(log_decay, torch.Tensor) and log_decay.requires_grad:
            raise ValueError("log_decay gets no gradient: pass log_decay.detach()")
        _native.refuse_foreign_leaves({"q": q, "k": k, "v": v, "initial_state": initial_state})
        done = _native.linear_dense_fwd(q, k, v, log_decay, scale, initial_state,
                                        bool(return_final_state), True)
        if done is not None:
            return done if return_final_state else done[0]
        return LinearAttnFunc.apply(q, k, v, log_decay, scale, initial_state,
                                    bool(return_final_state))
    out, final = _forward(q, k, v, log_decay, scale, initial_state, bool(return_final_state))
    return (out, final) if return_final_state else out


# ------------------------------------------------------------------ serving

def _check_index(t, name, n):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be an integer tensor, got {t.dtype}")
    if t.shape != (n,):
        raise ValueError(f"{name} must have shape ({n},), got {tuple(t.shape)}")


def linear_attn_prefill(q, k, v, log_decay, state, query_start_loc, prefix_kv_lens,
                        state_indices=None, scale=None, out=None):
    """linear_attn_func on packed sequences, with their states in a pool.

    Args:
        q: [T, H, D]; k, v: [T, Hk, D]; log_decay: [H]; scale: as for
            linear_attn_func.
        state: [N, H, D, D] fp32, updated in place.
        query_start_loc: [B + 1] integers; sequence b's new tokens are rows
            query_start_loc[b] .. query_start_loc[b + 1] - 1.
        prefix_kv_lens: [B] integers, the tokens before them: with 0 the
            sequence starts from zeros whatever its slot holds, otherwise from
            its slot's state.  (The index tensors of tilelang_paged_forward.)
        state_indices: [B] integers, each sequence's slot, distinct; None:
            0 .. B - 1.  A sequence whose slot is not in the pool (negative:
            padding) starts from zeros and keeps no state.
        out: written in place when given; may be q, must not overlap k or v.
    Returns:
        out [T, H, D].  Rows of no sequence are not written, and a sequence of
        no tokens leaves its slot as it was.  No gradients.
    """
    if out is None:
        done = _native.linear_prefill(q, k, v, log_decay, state, query_start_loc, prefix_kv_lens,
                                      state_indices, scale)
        if done is not None:
            return done
    H, Hk, D = _check_qkv(q, k, v, ("num_tokens", "heads", "head_dim"))
    _check_decay(log_decay, H)
    _check_pool(state, H, D)
    if not isinstance(prefix_kv_lens, torch.Tensor) or prefix_kv_lens.dim() != 1:
        raise ValueError("prefix_kv_lens must be a [batch] tensor")
    B = prefix_kv_lens.shape[0]
    _check_index(prefix_kv_lens, "prefix_kv_lens", B)
    _check_index(query_start_loc, "query_start_loc", B + 1)
    if state_indices is not None:
        _check_index(state_indices, "state_indices", B)
    elif B > state.shape[0]:
        raise ValueError(f"{B} sequences need as many slots, state has {state.shape[0]}")
    named = {"q": q, "k": k, "v": v, "log_decay": log_decay, "state": state}
    _require_place(named)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif not isinstance(out, torch.Tensor) or out.shape != q.shape or out.dtype != q.dtype or \
            out.device != q.device:
        raise ValueError("out must match q in shape, dtype and device")
    if B == 0 or q.shape[0] == 0:
        return out
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    target = _rows(out)
    starts = as_int32(query_start_loc, q.device, "query_start_loc")
    prefix = as_int32(prefix_kv_lens, q.device, "prefix_kv_lens")
    slots = as_int32(state_indices, q.device, "state_indices") \
        if state_indices is not None else None
    a = _lib.LinearArgs()
    _set_qkv(a, q, k, v, log_decay, _scale(scale, D))
    a.out = target.data_ptr()
    a.q_stride[:], a.k_stride[:] = _strides3(q), _strides3(k)
    a.v_stride[:], a.o_stride[:] = _strides3(v), _strides3(target)
    a.initial_state = a.final_state = state.data_ptr()
    a.is_stride[:] = strides(state, 2)
    a.fs_stride[:] = strides(state, 2)
    a.query_start_loc, a.prefix_kv_lens = starts.data_ptr(), prefix.data_ptr()
    a.state_indices = slots.data_ptr() if slots is not None else None
    a.batch, a.seqlen, a.num_states = B, q.shape[0], state.shape[0]
    _launch_fwd(a, q.device)
    if target is not out:
        out.copy_(target)
    return out


def linear_attn_decode(q, k, v, log_decay, state, state_indices=None, scale=None):
    """One token for each sequence: its state is updated in place, then read.

    Args:
        q: [B, H, D]; k, v: [B, Hk, D]; log_decay: [H]; scale: as for
            linear_attn_func.
        state: [N, H, D, D] fp32, updated in place.
        state_indices: [B] integers, each sequence's slot, distinct; None:
            0 .. B - 1.  A sequence whose slot is not in the pool (negative:
            padding) sees its own token alone and keeps no state.
    Returns:
        out [B, H, D] in q's dtype.  fp32 arithmetic.  No gradients.
    """
    done = _native.linear_decode(q, k, v, log_decay, state, state_indices, scale)
    if done is not None:
        return done
    H, Hk, D = _check_qkv(q, k, v, ("batch", "heads", "head_dim"))
    _check_decay(log_decay, H)
    _check_pool(state, H, D)
    B = q.shape[0]
    if state_indices is not None:
        _check_index(state_indices, "state_indices", B)
    elif B > state.shape[0]:
        raise ValueError(f"{B} sequences need as many slots, state has {state.shape[0]}")
    _require_place({"q": q, "k": k, "v": v, "log_decay": log_decay, "state": state})
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if B == 0:
        return out
    q, k, v, log_decay = rows_ready(q), rows_ready(k), rows_ready(v), log_decay.contiguous()
    slots = as_int32(state_indices, q.device, "state_indices") \
        if state_indices is not None else None
    a = _lib.LinearDecodeArgs()
    _set_qkv(a, q, k, v, log_decay, _scale(scale, D))
    a.out, a.state = out.data_ptr(), state.data_ptr()
    a.state_indices = slots.data_ptr() if slots is not None else None
    a.q_stride[:], a.k_stride[:] = strides(q, 2), strides(k, 2)
    a.v_stride[:], a.o_stride[:] = strides(v, 2), strides(out, 2)
    a.s_stride[:] = strides(state, 2)
    a.batch, a.num_states = B, state.shape[0]
    lib = _lib.load()
    _lib.check(_lib.call_on(q.device, lambda st: lib.fa_linear_decode(ctypes.byref(a), st)),
               "fa_linear_decode")
    return out
