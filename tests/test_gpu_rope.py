"""GPU parity: qk_norm_rope, its gradients, and norm_rope_and_cache against the
64-bit reference.

Tolerances: one rounding to the output's type (half a step, eps / 2 of the
value) and the fp32 arithmetic before it.  A forward component sums at most 20
squares in a row and in a tree, so r is within 12 roundings of 2^-24; the
products and the rotation add 6: 2^-19 of |a| + |b|, the pair that is turned.
fp16 adds half its subnormal step, 2^-25.
"""
import pytest
import torch

import tilelang_fa_v100 as fa
from helpers import randn
from oracle import operators_ref as ref
from tilelang_fa_v100 import _native

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32 = 2.0 ** -19


def table(P, R, seed=0):
    inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    angle = torch.arange(P, dtype=torch.float64)[:, None] * inv + seed
    return angle.cos().float(), angle.sin().float()


def assert_turned(got, want, normed, dtype, R, interleaved):
    """normed [T, H, D]: the values before the rotation."""
    half = R // 2
    pair = normed.abs()
    a, b = ((slice(0, R, 2), slice(1, R, 2)) if interleaved
            else (slice(0, half), slice(half, R)))
    size = pair.clone()
    size[..., a] = size[..., b] = pair[..., a] + pair[..., b]
    tol = torch.finfo(dtype).eps / 2 * want.abs() + F32 * size + 2.0 ** -25
    got = got.double().cpu().reshape(want.shape)
    assert torch.equal(got.isnan(), want.isnan())
    bad = ((got - want).abs() > tol) & ~want.isnan()
    assert not bad.any(), f"{bad.sum()} of {bad.numel()}, worst {((got - want).abs() / tol).nan_to_num().max()}"


def normed(x, w, eps):
    x = x.double()
    return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()


CASES = [  # T, H, Hk, D, R, interleaved, dtype, weights
    (1, 1, 1, 64, 64, False, torch.float16, "half"),
    (37, 5, 1, 128, 128, False, torch.bfloat16, "f32"),
    (300, 32, 8, 128, 64, True, torch.float16, "f32"),
    (65, 3, 3, 256, 256, True, torch.bfloat16, "half"),
    (33, 4, 2, 80, 32, False, torch.float16, "q"),
    (7, 2, 2, 16, 16, False, torch.bfloat16, "k"),
    (129, 7, 7, 96, 96, True, torch.float16, None),
    (50, 2, 1, 512, 128, False, torch.bfloat16, "half"),
    (9, 3, 2, 24, 16, True, torch.float16, "f32"),
    (40, 2, 2, 192, 192, False, torch.float16, "half"),
]
IDS = [f"T{c[0]}_H{c[1]}_{c[2]}_D{c[3]}_R{c[4]}_{'i' if c[5] else 'h'}_{str(c[6])[6:]}_{c[7]}"
       for c in CASES]


def weights(g, D, dtype, kind):
    w = [(1 + 0.2 * torch.randn(D, generator=g)) for _ in range(2)]
    if kind != "f32":
        w = [x.to(dtype) for x in w]
    if kind is None:
        return None, None
    return (w[0] if kind != "k" else None), (w[1] if kind != "q" else None)


def on(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_forward_matches_reference(case):
    T, H, Hk, D, R, inter, dtype, kind = case
    g = torch.Generator().manual_seed(T + D)
    q, k = randn(g, T, H, D, dtype=dtype), randn(g, T, Hk, D, dtype=dtype)
    qw, kw = weights(g, D, dtype, kind)
    cos, sin = table(500, R)
    pos = torch.randint(0, 500, (T,), generator=g)
    got = fa.qk_norm_rope(*on(DEV, q, k, cos, sin, qw, kw, pos), eps=1e-5, interleaved=inter)
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        assert y.dtype == dtype and y.is_contiguous()
        want = ref.norm_rope(x, w, cos, sin, pos, 1e-5, inter)
        assert_turned(y, want, normed(x, w, 1e-5), dtype, R, inter)


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_gradients_match_reference(case):
    """Against autograd through the 64-bit reference.  A component's fp32 error:
    2^-19 of the terms it sums, r (|h| + |x r| mean |h x r|); a weight's: that of
    its terms, and N + 64 additions of 2^-24."""
    T, H, Hk, D, R, inter, dtype, kind = case
    g = torch.Generator().manual_seed(T + D + 1)
    q, k = randn(g, T, H, D, dtype=dtype), randn(g, T, Hk, D, dtype=dtype)
    dq, dk = randn(g, T, H, D, dtype=dtype), randn(g, T, Hk, D, dtype=dtype)
    qw, kw = weights(g, D, dtype, kind)
    cos, sin = table(500, R)
    pos = torch.randint(0, 500, (T,), generator=g)
    pos[T // 2] = -1 if T > 1 else 3
    dev = on(DEV, q, k, qw, kw)
    for t in dev:
        if t is not None:
            t.requires_grad_()
    out = fa.qk_norm_rope(dev[0], dev[1], *on(DEV, cos, sin), dev[2], dev[3], pos.to(DEV), 1e-5,
                          inter)
    torch.autograd.backward(out, on(DEV, dq, dk))
    for i, (x, w, dy) in enumerate(((q, qw, dq), (k, kw, dk))):
        xd = x.double().requires_grad_()
        wd = w.double().requires_grad_() if w is not None else None
        y = ref.norm_rope(xd, wd, cos, sin, pos, 1e-5, inter)
        y.backward(dy.double())
        live = (pos >= 0)[:, None, None]
        # |R^T dy| is at most sqrt(2) of the row's largest |dy|
        size = torch.where(live, dy.double().abs().amax(-1, keepdim=True) * 1.5, 0.0)
        got = dev[i].grad
        assert got.dtype == dtype and got.shape == x.shape
        if w is None:
            terms = size
        else:
            r = 1 / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-5)
            h = size * w.double().abs().max()
            terms = r * (h + (x.double() * r).abs() * (h * (x.double() * r).abs().mean(-1, keepdim=True)))
            gw = dev[2 + i].grad
            assert gw.dtype == w.dtype
            sums = (size * (x.double() * r).abs()).sum((0, 1))
            n = T * x.shape[1] + 64
            tol = torch.finfo(w.dtype).eps / 2 * wd.grad.abs() + (F32 + n * 2.0 ** -24) * sums + 2.0 ** -25
            worst = ((gw.double().cpu() - wd.grad).abs() / tol).max()
            assert worst <= 1, f"weight gradient: worst {worst}"
        tol = torch.finfo(dtype).eps / 2 * xd.grad.abs() + F32 * terms + 2.0 ** -25
        worst = ((got.double().cpu() - xd.grad).abs() / tol).max()
        assert worst <= 1, f"worst {worst}"


def test_gradient_against_differences():
    """Along a random direction: the sum of gradient times direction against the
    central difference of the 64-bit loss.  The gradients carry half a step of
    fp16 each, 2^-11 of their value: over N of them at most 2^-11 sum |g d|; the
    difference's own error is O(h^2) = 1e-8 of terms of order one."""
    g = torch.Generator().manual_seed(5)
    T, H, D, R = 40, 3, 64, 32
    q, k = randn(g, T, H, D), randn(g, T, H, D)
    qw, kw = weights(g, D, torch.float16, "f32")
    cos, sin = table(T, R)
    pos = torch.arange(T)
    dq, dk = randn(g, T, H, D), randn(g, T, H, D)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, qw, kw)]
    out = fa.qk_norm_rope(leaves[0], leaves[1], *on(DEV, cos, sin), leaves[2], leaves[3])
    grads = [t.double().cpu() for t in torch.autograd.grad(out, leaves, on(DEV, dq, dk))]

    def loss(ts):
        y = ref.norm_rope(ts[0], ts[2], cos, sin, pos)
        z = ref.norm_rope(ts[1], ts[3], cos, sin, pos)
        return (y * dq.double()).sum() + (z * dk.double()).sum()

    base = [t.double() for t in (q, k, qw, kw)]
    for n in range(4):
        d = [torch.zeros_like(t) for t in base]
        d[n] = torch.randn(base[n].shape, generator=g, dtype=torch.float64)
        h = 1e-4
        diff = (loss([b + h * x for b, x in zip(base, d)])
                - loss([b - h * x for b, x in zip(base, d)])) / (2 * h)
        along = (grads[n] * d[n]).sum()
        tol = 2.0 ** -11 * (grads[n] * d[n]).abs().sum() + 1e-4
        assert (diff - along).abs() <= tol


def test_dense_positions_strides_and_defaults():
    """[B, S, H, D] with no positions, [S] positions and [B, S] positions that say
    the same; q and k as views of one projection; tables as column slices."""
    g = torch.Generator().manual_seed(9)
    B, S, H, Hk, D, R = 2, 45, 4, 2, 128, 128
    qkv = randn(g, B, S, H + 2 * Hk, D).to(DEV)
    q, k = qkv[:, :, :H], qkv[:, :, H:H + Hk]
    cos, sin = (t.to(DEV) for t in table(S + 3, R))
    both = torch.cat((cos, sin), 1)
    w = torch.ones(D, dtype=torch.float16, device=DEV)
    want = fa.qk_norm_rope(q.reshape(B * S, H, D), k.reshape(B * S, Hk, D), cos, sin, w, w,
                           torch.arange(S, device=DEV).repeat(B))
    pos = torch.arange(S, device=DEV)
    for p in (None, pos, pos.int(), pos.expand(B, S), pos.repeat(B, 1)):
        got = fa.qk_norm_rope(q, k, both[:, :R // 2], both[:, R // 2:], w, w, p)
        assert torch.equal(got[0].reshape(want[0].shape), want[0])
        assert torch.equal(got[1].reshape(want[1].shape), want[1])
    # transposed heads and tokens, a misaligned base (copied)
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.zeros(k.numel() + 1, dtype=k.dtype, device=DEV)[1:].view(k.shape).copy_(k)
    got = fa.qk_norm_rope(qt, odd, cos, sin, w, w)
    assert torch.equal(got[0].reshape(want[0].shape), want[0])
    assert torch.equal(got[1].reshape(want[1].shape), want[1])


def test_positions_outside_the_table():
    g = torch.Generator().manual_seed(1)
    q, k = randn(g, 5, 2, 64), randn(g, 5, 1, 64)
    cos, sin = table(10, 32)
    pos = torch.tensor([-1, 9, 10, -(1 << 40), 1 << 40])
    w = torch.ones(64)
    dev = [t.to(DEV) for t in (q, k)]
    for t in dev:
        t.requires_grad_()
    out = fa.qk_norm_rope(*dev, *on(DEV, cos, sin, w, w, pos))
    for y in out:
        assert (y[[0, 3]] == 0).all()
        assert y[[2, 4], :, :32].isnan().all()
        assert y[[2, 4], :, 32:].isfinite().all() and y[1].isfinite().all()
    grads = torch.autograd.grad(out, dev, [torch.ones_like(y) for y in out])
    assert (grads[0][[0, 3]] == 0).all() and grads[0][1].isfinite().all()


def test_zero_rows_and_broadcast_gradients():
    """A row of zeros has r = 1 / sqrt(eps); a gradient expanded from one value."""
    cos, sin = (t.to(DEV) for t in table(4, 64))
    q = torch.zeros(4, 2, 64, dtype=torch.float16, device=DEV, requires_grad=True)
    k = torch.ones(4, 2, 64, dtype=torch.float16, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    out = fa.qk_norm_rope(q, k, cos, sin, w, w)
    assert (out[0] == 0).all()
    (out[0].sum() + out[1].sum()).backward()
    assert q.grad.isfinite().all() and w.grad.isfinite().all()
    # one output unused: its gradient is zero
    q2, k2 = q.detach().requires_grad_(), k.detach().requires_grad_()
    a, _ = fa.qk_norm_rope(q2, k2, cos, sin)
    a.sum().backward()
    assert (k2.grad == 0).all()


def test_empty_and_repeatable():
    cos, sin = (t.to(DEV) for t in table(4, 64))
    w = torch.ones(64, device=DEV, requires_grad=True)
    q = torch.zeros(2, 0, 3, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    out = fa.qk_norm_rope(q, q, cos, sin, w, w)
    assert out[0].shape == q.shape
    (out[0].sum() + out[1].sum()).backward()
    assert (w.grad == 0).all() and q.grad.shape == q.shape
    g = torch.Generator().manual_seed(2)
    q = randn(g, 700, 16, 128, dtype=torch.bfloat16).to(DEV).requires_grad_()
    cos, sin = (t.to(DEV) for t in table(700, 128))
    w = torch.ones(128, device=DEV, requires_grad=True)
    runs = [torch.autograd.grad(fa.qk_norm_rope(q, q, cos, sin, w, w), (q, w),
                                [torch.ones_like(q)] * 2) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(runs[0], r))


# ------------------------------------------------------------------ the cache

@pytest.mark.parametrize("case", CASES, ids=IDS)
@pytest.mark.parametrize("page", [16, 5])
def test_cache_form_matches_dense_bit_for_bit(case, page):
    """q and the written keys are qk_norm_rope's, values are copied, and every
    slot that no token names keeps its sentinel."""
    T, H, Hk, D, R, inter, dtype, kind = case
    g = torch.Generator().manual_seed(T + D + page)
    qkv = randn(g, T, (H + 2 * Hk) * D, dtype=dtype).to(DEV)
    q, k, v = (t.view(T, -1, D) for t in qkv.split([H * D, Hk * D, Hk * D], 1))
    qw, kw = on(DEV, *weights(g, D, dtype, kind))
    cos, sin = (t.to(DEV) for t in table(900, R))
    pos = torch.randint(0, 900, (T,), generator=g).to(DEV)
    P = -(-T // page) + 3
    slots = (torch.randperm(P * page + 6, generator=g)[:T] - 3).to(DEV)  # some outside
    slots[::5] = -1
    caches = [torch.full((P, page, Hk, D), x, dtype=dtype, device=DEV) for x in (3.5, -2.5)]
    want = [c.clone() for c in caches]
    out = fa.norm_rope_and_cache(q, k, v, *caches, slots, pos, cos, sin, qw, kw, interleaved=inter)
    qn, kn = fa.qk_norm_rope(q, k, cos, sin, qw, kw, pos, interleaved=inter)
    ok = (slots >= 0) & (slots < P * page)
    want[0].view(-1, Hk, D)[slots[ok]] = kn[ok]
    want[1].view(-1, Hk, D)[slots[ok]] = v[ok]
    assert torch.equal(out, qn)
    assert torch.equal(caches[0], want[0]) and torch.equal(caches[1], want[1])


def test_many_rows_a_group():
    """Enough rows for the unrolled kernel, an odd count of them."""
    g = torch.Generator(device=DEV).manual_seed(3)
    T, H, Hk, D = 8191, 33, 3, 64
    q, k = (torch.randn(T, h, D, generator=g, device=DEV, dtype=torch.float16) for h in (H, Hk))
    cos, sin = (t.to(DEV) for t in table(T, D))
    w = torch.linspace(0.5, 2, D, device=DEV)
    got = fa.qk_norm_rope(q, k, cos, sin, w, w)
    for t in (0, 1, 4095, 8190):
        one = fa.qk_norm_rope(q[t:t + 1], k[t:t + 1], cos, sin, w, w,
                              torch.tensor([t], device=DEV))
        assert torch.equal(got[0][t], one[0][0]) and torch.equal(got[1][t], one[1][0])
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[1]).all()


def test_native_and_python_paths_agree(monkeypatch):
    g = torch.Generator().manual_seed(4)
    q, k = randn(g, 2, 30, 4, 128).to(DEV), randn(g, 2, 30, 2, 128).to(DEV)
    cos, sin = (t.to(DEV) for t in table(30, 64))
    w = torch.ones(128, device=DEV)
    assert _native.norm_rope(q, k, cos, sin, w, None, None, 1e-6, False, False) is not None
    kc, vc = (torch.zeros(5, 16, 2, 128, dtype=q.dtype, device=DEV) for _ in range(2))
    slots = torch.arange(60, device=DEV)
    flat = [t.reshape(60, -1, 128) for t in (q, k)]
    call = lambda: (*fa.qk_norm_rope(q, k, cos, sin, w, None),  # noqa: E731
                    fa.norm_rope_and_cache(*flat, flat[1], kc, vc, slots, slots % 30, cos, sin, w,
                                           None), kc.clone())
    native = call()
    monkeypatch.setattr(_native, "_missing", True)
    kc.zero_()
    assert all(torch.equal(a, b) for a, b in zip(native, call()))


def test_other_stream_and_graph():
    """On a side stream, and captured with replays between eager calls."""
    g = torch.Generator().manual_seed(6)
    T, H, Hk, D = 64, 8, 2, 128
    q, k, v = (randn(g, T, h, D, dtype=torch.bfloat16).to(DEV) for h in (H, Hk, Hk))
    cos, sin = (t.to(DEV) for t in table(64, D))
    w = torch.ones(D, dtype=torch.bfloat16, device=DEV)
    kc, vc = (torch.zeros(5, 16, Hk, D, dtype=q.dtype, device=DEV) for _ in range(2))
    slots = torch.arange(T, device=DEV)
    step = lambda: fa.norm_rope_and_cache(q, k, v, kc, vc, slots, slots, cos, sin, w, w)  # noqa: E731
    want, want_k = step(), kc.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kc.zero_()
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(kc, want_k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(3):
        q.copy_(randn(g, T, H, D, dtype=torch.bfloat16).to(DEV))
        kc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, got_k = out.clone(), kc.clone()
        kc.zero_()
        assert torch.equal(step(), got) and torch.equal(kc, got_k)
