"""The operators together, as a training step and a serving loop use them: norm and
rotation before dense attention and before linear attention, with gradients through
both; prompts and single tokens through norm_rope_and_cache, paged prefill and
paged decode."""
import pytest
import torch

import tilelang_fa_v100 as fa
from helpers import randn
from oracle import attention_ref as attn
from oracle import operators_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def table(P, R):
    inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    angle = torch.arange(P, dtype=torch.float64)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def rel(got, want):
    return ((got.double().cpu() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("attention", ["softmax", "linear"])
def test_training_step(attention):
    """loss = <attention(norm_rope(q, k), v), w>, every gradient against 64-bit autograd.
    Relative 2-norms: each of the two stages rounds its output and its gradients to
    bf16 (2^-9 of a value, uniform: 2^-9 / sqrt(3) in the norm) and its products'
    operands (P, dS or the state) once more; at most eight such roundings of the
    terms meet in one gradient: 8 * 2^-9 / sqrt(3) = 9e-3."""
    g = torch.Generator().manual_seed(3)
    B, S, H, Hk, D, dtype = 1, 150, 4, 2, 64, torch.bfloat16
    q, k, v = (randn(g, B, S, h, D, dtype=dtype) for h in (H, Hk, Hk))
    do = randn(g, B, S, H, D, dtype=dtype)
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=g)) for _ in range(2))
    decay = -torch.exp2(-8 * torch.arange(1, H + 1).float() / H)
    cos, sin = table(S, D)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, qw, kw)]
    qn, kn = fa.qk_norm_rope(leaves[0], leaves[1], cos.to(DEV), sin.to(DEV), *leaves[3:])
    if attention == "softmax":
        out = fa.tilelang_flash_attn_func(qn, kn, leaves[2], causal=True)
    else:
        out = fa.linear_attn_func(qn, kn, leaves[2], decay.to(DEV))
    grads = torch.autograd.grad(out, leaves, do.to(DEV))

    ins = [t.double().requires_grad_() for t in (q[0], k[0], v[0], qw, kw)]
    pos = torch.arange(S)
    a = ref.norm_rope(ins[0], ins[3], cos, sin, pos)
    b = ref.norm_rope(ins[1], ins[4], cos, sin, pos)
    if attention == "softmax":
        kk, vv = (t.repeat_interleave(H // Hk, 1) for t in (b, ins[2]))
        s = torch.einsum("ihd,jhd->hij", a, kk) * D ** -0.5
        s = s.masked_fill(torch.ones(S, S).triu(1).bool(), float("-inf"))
        want = torch.einsum("hij,jhd->ihd", s.softmax(-1), vv)
    else:
        want, _ = ref.linear_attention(a, b, ins[2], decay, D ** -0.5)
    want_g = torch.autograd.grad(want, ins, do[0].double())
    assert rel(out[0], want.detach()) < 9e-3
    for x, y in zip(grads, want_g):
        assert rel(x.reshape(y.shape), y) < 9e-3


def test_serving_loop():
    """Two prompts into the cache and through paged prefill, then four tokens each
    through the cache and paged decode: every output against dense attention over the
    sequence so far, computed from the normed and rotated rows in 64 bits.  Outputs
    are averages of v: the keys' and queries' rounding to fp16 moves a score by
    2 * 2^-11 of the sum of its terms' sizes (|q| |k| <= 64 * 0.125 * 4, below 32:
    3e-2 at the very most, 2e-3 for sums of random signs), and so an output by
    about that share of |v|; the existing bound of outputs, 2e-3 + 1e-2 |ref|,
    holds the whole."""
    g = torch.Generator().manual_seed(8)
    H, Hk, D, page, dtype = 8, 2, 64, 16, torch.float16
    lens, steps = [37, 90], 4
    total = [n + steps for n in lens]
    pages = [-(-n // page) for n in total]
    perm = torch.randperm(sum(pages) + 2, generator=g)
    bt = torch.full((2, max(pages)), -1, dtype=torch.int32)
    bt[0, :pages[0]] = perm[:pages[0]].int()
    bt[1, :pages[1]] = perm[pages[0]:sum(pages)].int()
    rows = [randn(g, n, (H + 2 * Hk) * D, dtype=dtype) for n in total]
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=g)).to(dtype) for _ in range(2))
    cos, sin = table(128, D)
    kc, vc = (torch.full((len(perm), page, Hk, D), float("nan"), dtype=dtype, device=DEV)
              for _ in range(2))
    dev = [t.to(DEV) for t in (cos, sin, qw, kw)]

    def append(parts):
        """parts: (sequence, first, end); returns q of all their rows."""
        x = torch.cat([rows[b][i:j] for b, i, j in parts]).to(DEV)
        pos = torch.cat([torch.arange(i, j) for _, i, j in parts])
        slots = torch.cat([bt[b, torch.arange(i, j) // page].long() * page
                           + torch.arange(i, j) % page for b, i, j in parts])
        q, k, v = (t.reshape(len(pos), -1, D) for t in x.split([H * D, Hk * D, Hk * D], 1))
        return fa.norm_rope_and_cache(q, k, v, kc, vc, slots.to(DEV), pos.to(DEV), *dev)

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    got = [[], []]
    q = append([(0, 0, lens[0]), (1, 0, lens[1])])
    out, _ = fa.tilelang_paged_forward(q, kc, vc, bt.to(DEV), i32(lens),
                                       i32([0, lens[0], sum(lens)]), i32([0, 0]),
                                       block_size=page)
    got[0].append(out[:lens[0]])
    got[1].append(out[lens[0]:])
    for t in range(steps):
        q = append([(b, lens[b] + t, lens[b] + t + 1) for b in range(2)])
        out = fa.tilelang_decode_forward(q, kc, vc, bt.to(DEV), i32([n + t + 1 for n in lens]),
                                         block_size=page)
        for b in range(2):
            got[b].append(out[b:b + 1])
    for b in range(2):
        n = total[b]
        x = rows[b].view(n, H + 2 * Hk, D)
        pos = torch.arange(n)
        qn = ref.norm_rope(x[:, :H], qw, cos, sin, pos)
        kn = ref.norm_rope(x[:, H:H + Hk], kw, cos, sin, pos)
        want, _ = attn.dense_attention(qn[None].float(), kn[None].float(),
                                       x[None, :, H + Hk:].float(), causal=True)
        err = (torch.cat(got[b]).float().cpu() - want[0]).abs()
        assert (err <= 2e-3 + 1e-2 * want[0].abs()).all(), err.max()
