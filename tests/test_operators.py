"""CPU tests of the operators around attention: struct layouts, refusals before any
launch, and the 64-bit references against independent forms."""
import ctypes
import os
import subprocess

import pytest
import torch

import tilelang_fa_v100 as fa
from oracle import operators_ref as ref
from tilelang_fa_v100 import _lib, _native

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"fa_norm_rope_args": _lib.NormRopeArgs, "fa_norm_rope_bwd_args": _lib.NormRopeBwdArgs,
           "fa_norm_rope_cache_args": _lib.NormRopeCacheArgs, "fa_linear_args": _lib.LinearArgs,
           "fa_linear_bwd_args": _lib.LinearBwdArgs,
           "fa_linear_decode_args": _lib.LinearDecodeArgs}


def test_ctypes_structs_match_c_layout(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "fa355.h"', "int main(void){"]
    for cname, py in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        for fname, _ in py._fields_:
            lines.append(f'printf("{cname} {fname} %zu\\n", offsetof({cname}, {fname}));')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{REPO}/include", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    for line in out.splitlines():
        cname, field, val = line.split()
        py = STRUCTS[cname]
        got = ctypes.sizeof(py) if field == "size" else getattr(py, field).offset
        assert got == int(val), (cname, field)


def rope_args(**over):
    a = _lib.NormRopeArgs()
    a.q = a.k = a.q_out = a.k_out = a.cos = a.sin = 0x1000
    for s in (a.q_stride, a.k_stride, a.qo_stride, a.ko_stride):
        s[:] = (0, 1024, 128)
    a.table_stride[:] = (64, 64)
    a.num_positions, a.batch, a.seqlen, a.num_heads, a.num_heads_k = 10, 1, 4, 8, 8
    a.head_dim, a.rotary_dim, a.eps = 128, 128, 1e-6
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,status", [
    (dict(q=None), _lib.FA_E_INVALID), (dict(cos=None), _lib.FA_E_INVALID),
    (dict(dtype=5), _lib.FA_E_UNSUPPORTED), (dict(head_dim=520), _lib.FA_E_UNSUPPORTED),
    (dict(head_dim=100), _lib.FA_E_UNSUPPORTED), (dict(rotary_dim=24), _lib.FA_E_UNSUPPORTED),
    (dict(rotary_dim=144), _lib.FA_E_UNSUPPORTED), (dict(num_positions=0), _lib.FA_E_INVALID),
    (dict(seqlen=-1), _lib.FA_E_INVALID), (dict(k_out=0x1008), _lib.FA_E_UNSUPPORTED),
    (dict(q_weight=0x1004), _lib.FA_E_UNSUPPORTED), (dict(positions=0x1004), _lib.FA_E_INVALID),
    (dict(batch=1 << 20, seqlen=1 << 11), _lib.FA_E_UNSUPPORTED)])
def test_norm_rope_abi_rejects_bad_arguments(over, status):
    lib = _lib.load()
    assert lib.fa_norm_rope(ctypes.byref(rope_args(**over)), None) == status
    assert lib.fa_last_error_message()
    assert lib.fa_norm_rope(None, None) == _lib.FA_E_INVALID


def test_norm_rope_bwd_abi_rejects_bad_arguments():
    lib = _lib.load()
    a = _lib.NormRopeBwdArgs()
    a.dq_out = a.dk_out = a.dq = a.dk = a.cos = a.sin = 0x1000
    a.num_positions, a.batch, a.seqlen, a.num_heads, a.num_heads_k = 10, 1, 4, 8, 8
    a.head_dim, a.rotary_dim = 128, 128
    assert lib.fa_norm_rope_bwd_workspace_bytes(ctypes.byref(a)) == 0
    a.q_weight = 0x1000  # without its gradient, and without q
    assert lib.fa_norm_rope_bwd(ctypes.byref(a), None, 0, None) == _lib.FA_E_INVALID
    a.q = 0x1000
    assert lib.fa_norm_rope_bwd(ctypes.byref(a), None, 0, None) == _lib.FA_E_INVALID


def linear_args(cls=_lib.LinearArgs, **over):
    a = cls()
    for n, t in cls._fields_:
        if t is ctypes.c_void_p:
            setattr(a, n, 0x1000)
    a.batch, a.num_heads, a.num_heads_k, a.head_dim = 1, 4, 2, 128
    for n, v in dict(seqlen=100, num_states=1).items():
        if hasattr(a, n):
            setattr(a, n, v)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,status", [
    (dict(q=None), _lib.FA_E_INVALID), (dict(log_decay=None), _lib.FA_E_INVALID),
    (dict(dtype=9), _lib.FA_E_UNSUPPORTED), (dict(head_dim=96), _lib.FA_E_UNSUPPORTED),
    (dict(num_heads_k=3), _lib.FA_E_INVALID), (dict(batch=-1), _lib.FA_E_INVALID),
    (dict(v=0x1008), _lib.FA_E_UNSUPPORTED), (dict(batch=1 << 30), _lib.FA_E_UNSUPPORTED)])
def test_linear_abi_rejects_bad_arguments(over, status):
    lib = _lib.load()
    assert lib.fa_linear_fwd(ctypes.byref(linear_args(**over)), None, 0, None) == status
    assert lib.fa_linear_fwd_workspace_bytes(ctypes.byref(linear_args(**over))) == 0
    b = linear_args(_lib.LinearBwdArgs, **over)
    assert lib.fa_linear_bwd(ctypes.byref(b), None, 0, None) == status
    d = linear_args(_lib.LinearDecodeArgs, **over)
    assert lib.fa_linear_decode(ctypes.byref(d), None) == status
    for fn, n in ((lib.fa_linear_fwd, 4), (lib.fa_linear_bwd, 4), (lib.fa_linear_decode, 2)):
        assert fn(*([None, None, 0, None] if n == 4 else [None, None])) == _lib.FA_E_INVALID


def test_linear_abi_rejects_bad_states():
    lib = _lib.load()
    for field in ("initial_state", "final_state"):
        a = linear_args(**{field: 0x1004})
        assert lib.fa_linear_fwd(ctypes.byref(a), None, 0, None) == _lib.FA_E_UNSUPPORTED
    a = linear_args()
    a.fs_stride[1] = 2
    assert lib.fa_linear_fwd(ctypes.byref(a), None, 0, None) == _lib.FA_E_UNSUPPORTED
    d = linear_args(_lib.LinearDecodeArgs, state=None)
    assert lib.fa_linear_decode(ctypes.byref(d), None) == _lib.FA_E_INVALID


# ------------------------------------------------------------------ Python

def h(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def test_qk_norm_rope_refusals():
    q, k, t, w = h(4, 2, 64), h(4, 1, 64), torch.zeros(8, 32), torch.ones(64)
    call = fa.qk_norm_rope
    for bad in (dict(q=q.float()), dict(k=k.bfloat16()), dict(cos=t.half()), dict(q=[1]),
                dict(q_weight=w.double()), dict(q_weight=w, k_weight=w.half()),
                dict(positions=torch.zeros(4)), dict(sin=None)):
        with pytest.raises(TypeError):
            call(**{**dict(q=q, k=k, cos=t, sin=t), **bad})
    for bad in (dict(q=h(4, 2, 60)), dict(k=h(5, 1, 64)), dict(k=h(4, 1, 128)), dict(q=h(4, 64)),
                dict(cos=t[:, :4], sin=t[:, :4]), dict(sin=t[:3]), dict(cos=t[:0], sin=t[:0]),
                dict(cos=torch.zeros(8, 64), sin=torch.zeros(8, 64)), dict(q_weight=w[:32]),
                dict(positions=torch.zeros(3, dtype=torch.long)),
                dict(cos=t.clone().requires_grad_()), dict(k=h(4, 0, 64))):
        with pytest.raises(ValueError):
            call(**{**dict(q=q, k=k, cos=t, sin=t), **bad})
    with pytest.raises(ValueError, match="GPU"):
        call(q, k, t, t, w, w)
    with pytest.raises(ValueError, match="GPU"):
        call(q.clone().requires_grad_(), k, t, t)


def test_norm_rope_and_cache_refusals():
    ok = dict(q=h(4, 2, 64), k=h(4, 1, 64), v=h(4, 1, 64), key_cache=h(3, 16, 1, 64),
              value_cache=h(3, 16, 1, 64), slot_mapping=torch.arange(4), positions=torch.arange(4),
              cos=torch.zeros(8, 32), sin=torch.zeros(8, 32))
    for bad in (dict(v=h(4, 1, 64).float()), dict(key_cache=h(3, 16, 1, 64).bfloat16()),
                dict(slot_mapping=torch.zeros(4)), dict(positions=None)):
        with pytest.raises(TypeError):
            fa.norm_rope_and_cache(**{**ok, **bad})
    for bad in (dict(v=h(4, 2, 64)), dict(value_cache=h(3, 8, 1, 64)),
                dict(key_cache=h(3, 16, 2, 64), value_cache=h(3, 16, 2, 64)),
                dict(slot_mapping=torch.arange(3)), dict(positions=torch.arange(5)),
                dict(q=h(1, 4, 2, 64))):
        with pytest.raises(ValueError):
            fa.norm_rope_and_cache(**{**ok, **bad})
    with pytest.raises(ValueError, match="GPU"):
        fa.norm_rope_and_cache(**ok)


def test_linear_refusals():
    q, k, g = h(1, 8, 4, 64), h(1, 8, 2, 64), torch.zeros(4)
    s = torch.zeros(1, 4, 64, 64)
    ok = dict(q=q, k=k, v=k, log_decay=g)
    for bad in (dict(q=q.float()), dict(v=k.bfloat16()), dict(log_decay=g.double()),
                dict(log_decay=0.5), dict(initial_state=s.half())):
        with pytest.raises(TypeError):
            fa.linear_attn_func(**{**ok, **bad})
    for bad in (dict(v=h(1, 8, 4, 64)), dict(q=h(1, 8, 3, 64), log_decay=g[:3]),
                dict(q=h(1, 7, 4, 64)), dict(q=h(8, 4, 64)), dict(log_decay=g[:2]),
                dict(initial_state=s[:, :2]), dict(log_decay=g.clone().requires_grad_()),
                dict(q=h(1, 8, 4, 96), k=h(1, 8, 2, 96), v=h(1, 8, 2, 96))):
        with pytest.raises(ValueError):
            fa.linear_attn_func(**{**ok, **bad})
    with pytest.raises(ValueError, match="GPU"):
        fa.linear_attn_func(**ok)
    ints = dict(query_start_loc=torch.tensor([0, 8]), prefix_kv_lens=torch.tensor([0]))
    pre = dict(q=q[0], k=k[0], v=k[0], log_decay=g, state=s, **ints)
    for bad in (dict(state=s.half()), dict(query_start_loc=torch.zeros(2))):
        with pytest.raises(TypeError):
            fa.linear_attn_prefill(**{**pre, **bad})
    for bad in (dict(state=s[:0]), dict(state=s.transpose(2, 3)), dict(state=s[..., :32]),
                dict(state=s[:, :1].expand(1, 4, 64, 64)),
                dict(query_start_loc=torch.tensor([0, 4, 8])), dict(prefix_kv_lens=[0]),
                dict(prefix_kv_lens=torch.tensor([0, 0]), query_start_loc=torch.tensor([0, 4, 8])),
                dict(state_indices=torch.tensor([0, 1])), dict(q=q)):
        with pytest.raises(ValueError):
            fa.linear_attn_prefill(**{**pre, **bad})
    with pytest.raises(ValueError, match="GPU"):
        fa.linear_attn_prefill(**pre)
    dec = dict(q=q[0, :1], k=k[0, :1], v=k[0, :1], log_decay=g, state=s)
    for bad in (dict(q=q[0, :2], k=k[0, :2], v=k[0, :2]), dict(state=s[0])):
        with pytest.raises(ValueError):
            fa.linear_attn_decode(**{**dec, **bad})
    with pytest.raises(ValueError, match="GPU"):
        fa.linear_attn_decode(**dec)


def test_native_hands_back_what_is_not_plain():
    m, t = _native.load(), h(2, 4, 64)
    assert m.norm_rope(t, t, t, t, None, None, None, 1e-6, False, False, 0, 0) is None
    assert m.norm_rope_cache(t, t, t, t, t, t, t, t, t, None, None, 1e-6, False, 0, 0) is None
    assert m.linear_prefill(t, t, t, t, t, t, t, None, None, 0, 0) is None
    assert m.linear_decode(t, t, t, t, t, None, None, 0, 0) is None
    for name in ("norm_rope", "norm_rope_cache", "linear_prefill", "linear_decode"):
        assert getattr(m, name)() is None


# ------------------------------------------------------------------ the references

def test_linear_reference_is_the_sum_over_pairs():
    gen = torch.Generator().manual_seed(0)
    S, H, Hk, D = 30, 4, 2, 8
    q = torch.randn(S, H, D, generator=gen)
    k, v = (torch.randn(S, Hk, D, generator=gen) for _ in range(2))
    g, s0 = -torch.rand(H, generator=gen), torch.randn(H, D, D, generator=gen)
    out, final = ref.linear_attention(q, k, v, g, 0.3, s0)
    kk, vv = (t.repeat_interleave(2, 1).double() for t in (k, v))
    for h_ in range(H):
        for i in range(S):
            o = torch.exp(g[h_].double() * (i + 1)) * (q[i, h_].double() @ s0[h_].double())
            for j in range(i + 1):
                o = o + torch.exp(g[h_].double() * (i - j)) * (q[i, h_].double() @ kk[j, h_]) * vv[j, h_]
            torch.testing.assert_close(out[i, h_], 0.3 * o, rtol=1e-12, atol=1e-12)
    half, full, size = ref.linear_attention_bounds(q, k, v, g, 0.3, s0, chunk=7)
    assert (full + 1e-12 >= out.abs()).all() and (full + 1e-12 >= half).all()
    assert (size + 1e-12 >= final.abs()).all()


def test_norm_rope_reference_keeps_norms_and_pairs():
    gen = torch.Generator().manual_seed(1)
    x, w = torch.randn(6, 2, 32, generator=gen), torch.ones(32)
    angle = torch.rand(6, 8, generator=gen, dtype=torch.float64)
    pos = torch.arange(6)
    y = ref.norm_rope(x, w, angle.cos(), angle.sin(), pos, eps=0.0)
    z = ref.norm_rope(x, w, angle.cos(), angle.sin(), pos, eps=0.0, interleaved=True)
    for t in (y, z):
        torch.testing.assert_close((t * t).mean(-1), torch.ones(6, 2, dtype=torch.float64))
    perm = [*range(0, 16, 2), *range(1, 16, 2), *range(16, 32)]
    torch.testing.assert_close(
        ref.norm_rope(x[..., perm], w, angle.cos(), angle.sin(), pos, eps=0.0), z[..., perm])
