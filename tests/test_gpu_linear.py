"""GPU parity: linear attention (training, packed prefill, decode) against the
64-bit recurrence of oracle/operators_ref.py.

Tolerances, from linear_attention_bounds on the same inputs.  A 16-bit output
carries half a step (eps / 2) of its own value and of `half`, the terms whose
score or state is rounded to the inputs' type once; and the fp32 arithmetic: a
sum of n products is within n 2^-24 of `full` in any order, n at most the row's
keys and components (S + 2 D), and every factor (decay, scale) adds a few
roundings, 8 2^-24.  A state: its fp32 sums, (S + 16) 2^-24 of `states`, with
16 for the decay factors and the split of the values.  fp16 adds its subnormal
step.
"""
import pytest
import torch

import tilelang_fa_v100 as fa
from helpers import randn
from oracle import operators_ref as ref
from tilelang_fa_v100 import _native

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E24 = 2.0 ** -24


def slopes(H, kind="mixed"):
    if kind == "none":
        return torch.zeros(H)
    g = -torch.exp2(-8 * torch.arange(1, H + 1).float() / H)
    if kind == "hard":
        g = -torch.tensor([float("inf"), 30.0, 1e-4, 0.0, 3.0])[torch.arange(H) % 5]
    return g


def assert_out(got, want, bounds, dtype, S, D, extra=0.0):
    half, full = bounds
    eps = torch.finfo(dtype).eps / 2
    tol = eps * (want.abs() + half) + (S + 2 * D + 8) * E24 * full + 2.0 ** -24 + extra
    err = (got.double().cpu() - want).abs()
    assert not got.isnan().any()
    assert (err <= tol).all(), f"worst {(err / tol).max():.3g}"


def assert_state(got, want, size, S):
    tol = (S + 16) * E24 * size + 1e-30
    err = (got.double().cpu() - want).abs()
    assert not got.isnan().any()
    assert (err <= tol).all(), f"worst {(err / tol).max():.3g}"


def inputs(seed, B, S, H, Hk, D, dtype, state):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (randn(g, B, S, h, D, dtype=dtype) for h in (H, Hk, Hk))
    s = torch.randn(B, H, D, D, generator=g) if state else None
    return g, q, k, v, s


CASES = [  # B, S, H, Hk, D, dtype, state, slopes
    (1, 1, 1, 1, 64, torch.float16, False, "mixed"),
    (2, 1, 2, 1, 128, torch.bfloat16, True, "mixed"),
    (1, 63, 2, 2, 128, torch.float16, True, "none"),
    (2, 64, 3, 3, 64, torch.bfloat16, True, "mixed"),
    (1, 65, 2, 2, 256, torch.bfloat16, False, "mixed"),
    (1, 257, 5, 5, 128, torch.bfloat16, True, "hard"),
    (2, 300, 4, 2, 64, torch.float16, False, "mixed"),
    (1, 513, 4, 1, 128, torch.float16, True, "mixed"),
    (1, 700, 2, 2, 256, torch.float16, True, "mixed"),
    (3, 129, 5, 5, 256, torch.float16, False, "hard"),
]
IDS = [f"B{c[0]}_S{c[1]}_H{c[2]}_{c[3]}_D{c[4]}_{str(c[5])[6:]}_{'s' if c[6] else 'z'}_{c[7]}"
       for c in CASES]


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_forward_matches_reference(case):
    B, S, H, Hk, D, dtype, state, kind = case
    _, q, k, v, s0 = inputs(S + D, B, S, H, Hk, D, dtype, state)
    g = slopes(H, kind)
    dev = [t.to(DEV) if t is not None else None for t in (q, k, v, g, s0)]
    out, final = fa.linear_attn_func(*dev[:4], initial_state=dev[4], return_final_state=True)
    assert out.dtype == dtype and out.shape == q.shape and final.dtype == torch.float32
    alone = fa.linear_attn_func(*dev[:4], initial_state=dev[4])
    assert torch.equal(alone, out)
    for b in range(B):
        args = (q[b], k[b], v[b], g, D ** -0.5, s0[b] if state else None)
        want, want_s = ref.linear_attention(*args)
        half, full, size = ref.linear_attention_bounds(*args)
        assert_out(out[b], want, (half, full), dtype, S, D)
        assert_state(final[b], want_s, size, S)


def grad_bounds(q, k, v, do, g, scale, s0, ds):
    """Bounds of dq, dk, dv and of the initial state's gradient, from the three
    forms the gradients are (scale on the carried sums; the states' gradients
    carry none)."""
    t = lambda x: None if x is None else x.transpose(-1, -2) / scale  # noqa: E731
    H, Hk = q.shape[1], k.shape[1]
    kk, vv = (x.repeat_interleave(H // Hk, 1) for x in (k, v))
    bq = ref.linear_attention_bounds(do, vv, kk, g, scale,
                                     None if s0 is None else s0.transpose(-1, -2))
    bk = ref.linear_attention_bounds(vv, do, q, g, scale, t(ds), reverse=True)
    bv = ref.linear_attention_bounds(kk, q, do, g, scale, None if ds is None else ds / scale,
                                     reverse=True)
    return bq, bk, bv


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_gradients_match_reference(case):
    B, S, H, Hk, D, dtype, state, kind = case
    gen, q, k, v, s0 = inputs(S + D + 1, B, S, H, Hk, D, dtype, state)
    do = randn(gen, B, S, H, D, dtype=dtype)
    ds = torch.randn(B, H, D, D, generator=gen) if state else None
    g, scale = slopes(H, kind), D ** -0.5
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, s0) if t is not None]
    out = fa.linear_attn_func(*leaves[:3], g.to(DEV), initial_state=leaves[3] if state else None,
                              return_final_state=state)
    grads = torch.autograd.grad(out, leaves, [t.to(DEV) for t in (do, ds) if t is not None])
    for b in range(B):
        ins = [t[b].double().requires_grad_() for t in (q, k, v)]
        first = s0[b].double().requires_grad_() if state else None
        o, final = ref.linear_attention(*ins, g, scale, first)
        loss = (o * do[b].double()).sum()
        if state:
            loss = loss + (final * ds[b].double()).sum()
        want = torch.autograd.grad(loss, ins + ([first] if state else []))
        bounds = grad_bounds(q[b], k[b], v[b], do[b], g, scale, s0[b] if state else None,
                             ds[b] if state else None)
        for n, name in enumerate("qkv"):
            half, full, size = bounds[n]
            if n and H != Hk:
                # heads that share k and v: their parts are summed in fp32
                half, full = (x.reshape(S, Hk, H // Hk, D).sum(2) for x in (half, full))
            assert grads[n].dtype == dtype
            assert_out(grads[n][b], want[n], (half, full), dtype, S + H, D)
        if state:
            assert_state(grads[3][b], want[3], scale * bounds[2][2], S)


def test_gradient_against_differences():
    """Along a random direction, the gradients against the central difference of
    the 64-bit loss.  Each gradient is within 2^-10 of its value and of what it
    rounds (half), here twice its size at most: 3 2^-10 sum |g d| bounds them all;
    the differences' own error is 1e-8 of terms of order 1e3."""
    gen, q, k, v, s0 = inputs(3, 1, 90, 2, 2, 64, torch.float16, True)
    do, ds = randn(gen, 1, 90, 2, 64), torch.randn(1, 2, 64, 64, generator=gen)
    g, scale = slopes(2), 0.125
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, s0)]
    out = fa.linear_attn_func(*leaves[:3], g.to(DEV), initial_state=leaves[3],
                              return_final_state=True)
    grads = torch.autograd.grad(out, leaves, (do.to(DEV), ds.to(DEV)))

    def loss(ts):
        o, f = ref.linear_attention(ts[0], ts[1], ts[2], g, scale, ts[3])
        return (o * do[0].double()).sum() + (f * ds[0].double()).sum()

    base = [t[0].double() for t in (q, k, v, s0)]
    for n in range(4):
        d = [torch.zeros_like(t) for t in base]
        d[n] = torch.randn(base[n].shape, generator=gen, dtype=torch.float64)
        diff = (loss([b + 1e-4 * x for b, x in zip(base, d)])
                - loss([b - 1e-4 * x for b, x in zip(base, d)])) / 2e-4
        terms = grads[n][0].double().cpu() * d[n]
        assert (diff - terms.sum()).abs() <= 3 * 2.0 ** -10 * terms.abs().sum() + 1e-3


def test_long_memory_keeps_fp32():
    """A decay so slow that 4096 tokens all count: the state's decay is taken 64
    times, and what it loses in all stays in the sums' own bound."""
    S, H, D = 4096, 2, 64
    _, q, k, v, _ = inputs(8, 1, S, H, H, D, torch.bfloat16, False)
    g = torch.tensor([-1e-5, -1e-3])
    out, final = fa.linear_attn_func(*(t.to(DEV) for t in (q, k, v, g)), return_final_state=True)
    j = torch.arange(S, dtype=torch.float64)
    w = torch.exp(g.double()[:, None] * (S - 1 - j)).T[:, :, None]
    want = torch.einsum("shd,she->hde", k[0].double() * w, v[0].double())
    rel = (final[0].double().cpu() - want).norm() / want.norm()
    assert rel < 1e-6  # random sums: far below (S + 16) 2^-24 = 2.5e-4 of the absolute values


@pytest.mark.parametrize("size", [1e-3, 300.0])
def test_fp16_state_range(size):
    """fp16 with states far beyond 65504 and with values near its smallest ones:
    the copy of the state that meets q is scaled."""
    S, H, D = 400, 2, 128
    _, q, k, v, _ = inputs(21, 1, S, H, H, D, torch.float16, False)
    q, k, v = q * 1e-2 if size > 1 else q, (k * size).half(), (v * size).half()
    q = q.half()
    g, scale = slopes(H, "none"), 1e-4 if size > 1 else 0.1
    if size > 1:  # one key direction: the state grows with every token
        k, v = k.abs(), v.abs()
    out, final = fa.linear_attn_func(*(t.to(DEV) for t in (q, k, v, g)), scale=scale,
                                     return_final_state=True)
    args = (q[0], k[0], v[0], g, scale)
    want, want_s = ref.linear_attention(*args)
    half, full, sz = ref.linear_attention_bounds(*args)
    if size > 1:
        assert want_s.abs().max() > 65504
    # scores below fp16's normal range lose up to half its subnormal step, 2^-25,
    # against each v of the chunk
    extra = 2.0 ** -25 * 64 * v.double().abs().max()
    assert_out(out[0], want, (half, full), torch.float16, S, D, extra)


def packed(seed, lens, H, Hk, D, dtype, tail=0):
    gen = torch.Generator().manual_seed(seed)
    T = sum(lens) + tail
    q, k, v = (randn(gen, T, h, D, dtype=dtype) for h in (H, Hk, Hk))
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    return gen, q, k, v, torch.tensor(starts, dtype=torch.int32)


PACKED = [  # lens, H, Hk, D, dtype
    ([1], 2, 2, 64, torch.float16),
    ([5, 0, 64, 1, 130, 0], 4, 2, 128, torch.bfloat16),
    ([600, 1, 1, 1, 700, 300], 2, 2, 128, torch.float16),
    ([1] * 70 + [400], 2, 1, 64, torch.bfloat16),
    ([90, 290], 3, 3, 256, torch.bfloat16),
]


@pytest.mark.parametrize("lens,H,Hk,D,dtype", PACKED)
def test_prefill_matches_reference(lens, H, Hk, D, dtype):
    """Every sequence from its slot's state or from zeros, rows behind the last
    sequence and unused slots as they were, one sequence without a slot."""
    B, tail = len(lens), 3
    gen, q, k, v, starts = packed(len(lens) + D, lens, H, Hk, D, dtype, tail)
    g = slopes(H)
    pool = torch.randn(B + 2, H, D, D, generator=gen)
    slots = torch.randperm(B + 2, generator=gen)[:B].int()
    prefix = torch.tensor([7 * (i % 2) for i in range(B)], dtype=torch.int32)
    if B > 3:
        slots[3] = -1
        slots[2] = B + 2
    dev_pool = pool.to(DEV)
    out = torch.full_like(q, 9.0).to(DEV)
    args = [t.to(DEV) for t in (q, k, v, g)]
    got = fa.linear_attn_prefill(*args, dev_pool, starts.to(DEV), prefix.to(DEV), slots.to(DEV),
                                 out=out)
    assert got is out and (out[sum(lens):] == 9.0).all()
    again = pool.to(DEV)
    fresh = fa.linear_attn_prefill(*args, again, starts.to(DEV), prefix.to(DEV), slots.to(DEV))
    assert torch.equal(fresh[:sum(lens)], out[:sum(lens)]) and torch.equal(again, dev_pool)
    want_pool = pool.double()
    for b, n in enumerate(lens):
        rows, slot = slice(int(starts[b]), int(starts[b + 1])), int(slots[b])
        kept = 0 <= slot < B + 2
        if n == 0:
            assert not kept or torch.equal(dev_pool[slot].cpu(), pool[slot])
            continue
        first = pool[slot] if kept and prefix[b] > 0 else None
        a = (q[rows], k[rows], v[rows], g, D ** -0.5, first)
        want, want_s = ref.linear_attention(*a)
        half, full, size = ref.linear_attention_bounds(*a)
        assert_out(out[rows], want, (half, full), dtype, n, D)
        if kept:
            assert_state(dev_pool[slot], want_s, size, n)
            want_pool[slot] = dev_pool[slot].double().cpu()
    assert torch.equal(want_pool, dev_pool.double().cpu())


@pytest.mark.parametrize("B,H,Hk,D,dtype", [
    (1, 1, 1, 64, torch.float16), (3, 4, 2, 128, torch.bfloat16), (2, 3, 1, 256, torch.float16),
    (40, 8, 8, 128, torch.float16), (150, 2, 2, 256, torch.bfloat16), (300, 1, 1, 64, torch.bfloat16)])
def test_decode_matches_reference(B, H, Hk, D, dtype):
    gen = torch.Generator().manual_seed(B + D)
    q, k, v = (randn(gen, B, h, D, dtype=dtype) for h in (H, Hk, Hk))
    g = slopes(H)
    pool = torch.randn(B + 3, H, D, D, generator=gen)
    slots = torch.randperm(B + 3, generator=gen)[:B].int()
    if B > 2:
        slots[1], slots[2] = -5, B + 3
    dev_pool = pool.to(DEV)
    out = fa.linear_attn_decode(*(t.to(DEV) for t in (q, k, v, g)), dev_pool, slots.to(DEV))
    used = set()
    for b in range(B):
        slot = int(slots[b])
        kept = 0 <= slot < B + 3
        a = (q[b][None], k[b][None], v[b][None], g, D ** -0.5, pool[slot] if kept else None)
        want, want_s = ref.linear_attention(*a)
        _, full, size = ref.linear_attention_bounds(*a)
        assert_out(out[b][None], want, (torch.zeros(()), full), dtype, 1, D)
        if kept:
            used.add(slot)
            assert_state(dev_pool[slot], want_s, size, 1)
    for slot in set(range(B + 3)) - used:
        assert torch.equal(dev_pool[slot].cpu(), pool[slot])


def test_prefill_then_decode_is_the_whole_sequence():
    """norm and rotation, prefill of a prompt, then tokens one by one: the outputs
    of the whole sequence in one training call."""
    gen = torch.Generator().manual_seed(12)
    S, P, H, D, dtype = 100, 70, 4, 64, torch.float16
    q, k, v = (randn(gen, S, H, D, dtype=dtype).to(DEV) for _ in range(3))
    w = torch.ones(D, device=DEV)
    angle = torch.arange(S).double()[:, None] * 0.3
    cos, sin = (t.float().expand(S, 32).contiguous().to(DEV) for t in (angle.cos(), angle.sin()))
    q, k = fa.qk_norm_rope(q, k, cos, sin, w, w)
    g = slopes(H).to(DEV)
    whole, final = fa.linear_attn_func(q[None], k[None], v[None], g, return_final_state=True)
    state = torch.full((2, H, D, D), float("nan"), device=DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    outs = [fa.linear_attn_prefill(q[:P], k[:P], v[:P], g, state, i32(0, P), i32(0), i32(1))]
    for t in range(P, S):
        outs.append(fa.linear_attn_decode(q[t:t + 1], k[t:t + 1], v[t:t + 1], g, state, i32(1)))
    args = [t.cpu() for t in (q, k, v, g)]
    half, full, size = ref.linear_attention_bounds(*args, D ** -0.5)
    want, want_s = ref.linear_attention(*args, D ** -0.5)
    assert_out(torch.cat(outs), want, (half, full), dtype, S, D)
    assert_out(whole[0], want, (half, full), dtype, S, D)
    assert_state(state[1], want_s, size, S)
    assert_state(final[0], want_s, size, S)
    assert state[0].isnan().all()


def test_strides_and_views():
    """q, k, v as views of one projection, transposed and misaligned tensors, an
    initial state that is a transposed view, expanded gradients."""
    gen = torch.Generator().manual_seed(17)
    B, S, H, D = 2, 150, 3, 64
    qkv = randn(gen, B, S, 3 * H, D).to(DEV)
    q, k, v = qkv.split(H, 2)
    g = slopes(H).to(DEV)
    s0 = torch.randn(B, H, D, D, generator=gen).to(DEV)
    plain = [t.contiguous().requires_grad_() for t in (q, k, v)]
    s = s0.clone().requires_grad_()
    want, want_s = fa.linear_attn_func(*plain, g, initial_state=s, return_final_state=True)
    ones = (torch.ones_like(want), torch.ones_like(want_s))
    want_g = torch.autograd.grad((want, want_s), (*plain, s), ones)
    leaf = qkv.detach().clone().requires_grad_()
    views = leaf.split(H, 2)
    kt = views[1].transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.zeros(v.numel() + 1, dtype=v.dtype, device=DEV)[1:].view(v.shape).copy_(v)
    st = s0.transpose(2, 3).contiguous().transpose(2, 3).requires_grad_()
    got, got_s = fa.linear_attn_func(views[0], kt, odd, g, initial_state=st,
                                     return_final_state=True)
    assert torch.equal(got, want) and torch.equal(got_s, want_s)
    (got.sum() + got_s.sum()).backward()
    assert torch.equal(st.grad, want_g[3])
    assert torch.equal(leaf.grad[:, :, :2 * H], torch.cat(want_g[:2], 2))


def test_repeats_empty_and_no_grad():
    gen = torch.Generator().manual_seed(2)
    q, k, v = (randn(gen, 1, 1000, 8, 128, dtype=torch.bfloat16).to(DEV).requires_grad_()
               for _ in range(3))
    g = slopes(8).to(DEV)
    runs = [(o, *torch.autograd.grad(o, (q, k, v), torch.ones_like(o)))
            for o in (fa.linear_attn_func(q, k, v, g) for _ in range(3))]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))
    e = q[:, :0]
    s0 = torch.ones(1, 8, 128, 128, device=DEV, requires_grad=True)
    out, final = fa.linear_attn_func(e, e, e, g, initial_state=s0, return_final_state=True)
    assert out.shape == e.shape and torch.equal(final, s0)
    (final.sum() + out.sum()).backward()
    assert (s0.grad == 1).all()
    with torch.no_grad():
        assert not fa.linear_attn_func(q, k, v, g).requires_grad


def test_offsets_that_do_not_fit_the_rows():
    """Offsets beyond the rows, decreasing or overlapping ones: no access outside
    the tensors (what the rows get is not defined)."""
    gen, q, k, v, _ = packed(1, [300], 2, 2, 64, torch.float16)
    pool = torch.zeros(4, 2, 64, 64, device=DEV)
    args = [t.to(DEV) for t in (q, k, v, slopes(2))]
    for starts in ([-5, 10, 1 << 30, 4, 200], [0, 300, 0, 300, 0], [500, 600, 700, 800, 900]):
        fa.linear_attn_prefill(*args, pool, torch.tensor(starts, dtype=torch.int32, device=DEV),
                               torch.zeros(4, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert pool.isfinite().all()


def test_native_and_python_paths_agree(monkeypatch):
    gen, q, k, v, starts = packed(4, [100, 5], 4, 2, 128, torch.bfloat16)
    args = [t.to(DEV) for t in (q, k, v, slopes(4))]
    pool = torch.randn(2, 4, 128, 128, generator=gen).to(DEV)
    prefix = torch.tensor([3, 0], dtype=torch.int32, device=DEV)

    def call():
        p = pool.clone()
        o = fa.linear_attn_prefill(*args, p, starts.to(DEV), prefix)
        d = fa.linear_attn_decode(*(t[:2] if t.dim() == 3 else t for t in args), p)
        return o, d, p

    p = pool.clone()
    assert _native.linear_prefill(*args, p, starts.to(DEV), prefix, None, None) is not None
    assert _native.linear_decode(*(t[:2] if t.dim() == 3 else t for t in args), p, None,
                                 0.1) is not None
    native = call()
    monkeypatch.setattr(_native, "_missing", True)
    assert all(torch.equal(a, b) for a, b in zip(native, call()))


def test_streams_and_graphs():
    """A training step and a decode step captured and replayed between eager calls."""
    gen, q, k, v, s0 = inputs(31, 1, 200, 2, 2, 64, torch.bfloat16, True)
    g = slopes(2).to(DEV)
    q, k, v, s0 = (t.to(DEV) for t in (q, k, v, s0))

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, s0)]
        out = fa.linear_attn_func(*leaves[:3], g, initial_state=leaves[3], return_final_state=True)
        grads = torch.autograd.grad(out, leaves, [torch.ones_like(t) for t in out])
        return [*out, *grads]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    state = torch.zeros(1, 2, 64, 64, device=DEV)
    tok = [t[:, 0].contiguous() for t in (q, k, v)]
    dec = torch.cuda.CUDAGraph()
    with torch.cuda.graph(dec):
        tok_out = fa.linear_attn_decode(*tok, g, state)
    for n in range(3):
        q.copy_(randn(gen, *q.shape, dtype=q.dtype).to(DEV))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(step(), kept))
        state.normal_()
        mine = state.clone()
        dec.replay()
        torch.cuda.synchronize()
        got, got_s = tok_out.clone(), state.clone()
        assert torch.equal(fa.linear_attn_decode(*tok, g, mine), got) and torch.equal(mine, got_s)


# One or two heads want more segments than the main launch adds up: their states
# are joined before it.
JOINED = [
    (1, 2053, 1, 1, 128, torch.float16, True, "mixed"),
    (2, 1300, 2, 1, 64, torch.bfloat16, True, "mixed"),
    (1, 2500, 2, 2, 64, torch.float16, False, "none"),
]


@pytest.mark.parametrize("case", JOINED, ids=[f"S{c[1]}_H{c[2]}_{c[3]}_D{c[4]}" for c in JOINED])
def test_many_segments(case):
    test_forward_matches_reference(case)
    test_gradients_match_reference(case)


@pytest.mark.parametrize("lens", [(9000, 0, 5003, 1, 2380), (16384,), (64,) * 40 + (3000, 1)],
                         ids=["long", "one", "many"])
@pytest.mark.parametrize("D", [64, 128])
def test_many_packed_segments(lens, D):
    test_prefill_matches_reference(lens, 2, 1, D, torch.bfloat16)


@pytest.mark.parametrize("D,H,S", [(64, 48, 8192), (128, 40, 5003), (256, 24, 3000)])
def test_pool_is_read_before_it_is_written(D, H, S):
    """Segments far beyond what the GPU runs at once, all starting from the state that
    the last one replaces: the same as with two tensors, several times over."""
    gen = torch.Generator().manual_seed(D)
    q, k, v = (randn(gen, 1, S, H, D, dtype=torch.bfloat16).to(DEV) for _ in range(3))
    g = slopes(H).to(DEV) / 64
    first = (32 * torch.randn(1, H, D, D, generator=gen)).to(DEV)
    want, final = fa.linear_attn_func(q, k, v, g, initial_state=first, return_final_state=True)
    starts, prefix = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, S], [9]))
    for _ in range(4):
        pool = first.clone()
        out = fa.linear_attn_prefill(q[0], k[0], v[0], g, pool, starts, prefix)
        assert torch.equal(out, want[0]) and torch.equal(pool, final)


def test_overlapping_offsets_stay_in_bounds():
    """Sequences that claim the same rows have more segments than the workspace has
    slots: no result is promised, the rows and slots of others are left alone."""
    D, H, T = 64, 1, 4096
    gen = torch.Generator().manual_seed(5)
    q, k, v = (randn(gen, T, H, D, dtype=torch.float16).to(DEV) for _ in range(3))
    starts = torch.tensor([0, T, 0, T, 0, T], dtype=torch.int32, device=DEV)
    pool = torch.zeros(8, H, D, D, device=DEV)
    fa.linear_attn_prefill(q, k, v, slopes(H).to(DEV), pool, starts,
                           torch.ones(5, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert (pool[5:] == 0).all()
