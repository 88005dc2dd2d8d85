"""The measured operators around and beside the attention kernels.

* rope: `qk_norm_rope`, the per-head norm of queries and keys and the position rotation that
  stand before dense attention, forward only or forward and backward;
* append: `norm_rope_and_cache`, the serving form: queries and keys are normed and rotated and
  the keys and values go into the paged cache;
* train: `linear_attn_func`, linear attention with a decay for each head, forward and backward;
* prefill: `linear_attn_prefill`, the same on packed prompts with a pool of states;
* decode: `linear_attn_decode`, one token for each sequence.

`listed()` names twelve cases, `draw()` gives others from the same ranges.  `run()` computes an
operator in its plain form, or through the package's entry points where `own` is set.
"""
import math
import os
import random
import sys

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
CHUNK = 64  # rows of a chunk in the plain linear attention


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "tilelang-fa-v100_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import tilelang_fa_v100
    return tilelang_fa_v100


# ------------------------------------------------------------------ cases

def rope(name, batch, seq, heads, kv_heads, dim, rotary, dtype, interleaved, backward):
    return dict(name=name, kind="rope", batch=batch, seq=seq, heads=heads, kv_heads=kv_heads,
                dim=dim, rotary=rotary, dtype=dtype, interleaved=interleaved, backward=backward)


def append(name, tokens, heads, kv_heads, dim, rotary, page, dtype, interleaved, norm):
    return dict(name=name, kind="append", tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                rotary=rotary, page=page, dtype=dtype, interleaved=interleaved, norm=norm)


def train(name, batch, seq, heads, kv_heads, dim, dtype, state, backward):
    """state: the call starts from an initial state and returns the final one."""
    return dict(name=name, kind="train", batch=batch, seq=seq, heads=heads, kv_heads=kv_heads,
                dim=dim, dtype=dtype, state=state, backward=backward)


def prefill(name, seqs, len_lo, len_hi, singles, heads, kv_heads, dim, dtype, lens_seed):
    """`seqs` sequences of len_lo..len_hi new tokens, the last `singles` of them one token; every
    second one goes on from a cached state."""
    return dict(name=name, kind="prefill", seqs=seqs, len_lo=len_lo, len_hi=len_hi,
                singles=singles, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                lens_seed=lens_seed)


def decode(name, seqs, heads, kv_heads, dim, dtype):
    return dict(name=name, kind="decode", seqs=seqs, heads=heads, kv_heads=kv_heads, dim=dim,
                dtype=dtype)


def listed():
    return [
        # A short encoder block at inference: a small call, forward only.
        rope("rope_512_d64", 1, 512, 16, 16, 64, 64, "fp16", False, False),
        # The training step of the repository's benchmark, queries and keys before attention.
        rope("rope_train_2k_d128", 4, 2048, 16, 16, 128, 128, "bf16", False, True),
        # Long-sequence training of a grouped-query model.
        rope("rope_train_8k_gqa", 2, 8192, 32, 8, 128, 128, "bf16", False, True),
        # Serving: a decode step of a few sequences.
        append("append_4", 4, 32, 8, 128, 128, 16, "bf16", False, True),
        # Serving: chunked prefill, 16 chunks of 512 new tokens.
        append("append_8192", 8192, 64, 8, 128, 128, 16, "bf16", False, True),
        # Serving: a ragged batch of prompts, half of each head rotated in neighbouring pairs.
        append("append_5003_partial", 5003, 32, 8, 128, 64, 16, "fp16", True, False),
        # Training a linear-attention layer at the benchmark's sizes.
        train("linear_train_2k_d128", 4, 2048, 16, 16, 128, "bf16", False, True),
        # Long-sequence training, the largest case: a segment that takes over a state.
        train("linear_train_8k_d128", 2, 8192, 16, 16, 128, "fp16", True, True),
        # Serving: whole prompts.
        prefill("linear_prompts_8", 8, 512, 4096, 0, 16, 16, 128, "fp16", 3),
        # Serving: continuous batching, two prompt chunks among 30 decoding sequences.
        prefill("linear_mixed_32", 32, 256, 512, 30, 32, 32, 64, "bf16", 7),
        # Serving: a large decode batch.
        decode("linear_decode_64", 64, 32, 32, 128, "bf16"),
        # Serving: a decode step of a few sequences.
        decode("linear_decode_4", 4, 16, 16, 128, "fp16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["rope", "append", "train", "prefill", "decode"])
    dtype = rng.choice(["fp16", "bf16"])
    dim = rng.choice([64, 128, 128, 256])
    heads, kv_heads = rng.choice([(32, 8), (64, 8), (16, 2), (16, 16), (28, 4), (8, 8), (5, 5)])
    rotary = rng.choice([dim, dim, dim // 2])
    if kind == "rope":
        c = rope("", rng.choice([1, 2, 3, 4]), _log_int(rng, 60, 8192), heads, kv_heads, dim,
                 rotary, dtype, rng.random() < 0.3, rng.random() < 0.7)
    elif kind == "append":
        c = append("", _log_int(rng, 1, 8192), heads, kv_heads, dim, rotary,
                   rng.choice([16, 16, 32, 64]), dtype, rng.random() < 0.3, rng.random() < 0.7)
    elif kind == "train":
        heads, kv_heads = rng.choice([(16, 16), (16, 16), (32, 32), (8, 8), (5, 5), (16, 4)])
        c = train("", rng.choice([1, 2, 3, 4]), _log_int(rng, 60, 8192), heads, kv_heads, dim,
                  dtype, rng.random() < 0.3, rng.random() < 0.7)
    elif kind == "prefill":
        heads, kv_heads = rng.choice([(16, 16), (16, 16), (32, 32), (8, 8), (5, 5), (16, 4)])
        seqs = _log_int(rng, 1, 48)
        lo = _log_int(rng, 16, 2048)
        c = prefill("", seqs, lo, 2 * lo, rng.choice([0, rng.randint(0, seqs - 1)]), heads,
                    kv_heads, dim, dtype, rng.randrange(1 << 20))
    else:
        c = decode("", _log_int(rng, 1, 128), heads, kv_heads, dim, dtype)
    c.pop("name")
    return c


def draw(rng):
    # No more than the largest listed case of the kind, by what it reads, writes and computes.
    most = {}
    for c in listed():
        w = work(c)
        b, f = most.get(c["kind"], (0, 0))
        most[c["kind"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        c = _draw(rng)
        w = work(c)
        b, f = most[c["kind"]]
        if w["bytes"] <= b and w["flops"] <= f:
            return c


def _lens(case):
    """New tokens of every sequence of a prefill case."""
    r = random.Random(case["lens_seed"])
    n = case["seqs"] - case["singles"]
    return [r.randint(case["len_lo"], case["len_hi"]) for _ in range(n)] + [1] * case["singles"]


def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once."""
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "rope":
        rows = case["batch"] * case["seq"] * (H + Hk)
        passes = 8 if case["backward"] else 4  # x, y and, backward, dy, dx: 2 bytes an element
        return {"bytes": rows * D * passes + case["seq"] * case["rotary"] * 4,
                "flops": rows * D * (24 if case["backward"] else 8)}
    if case["kind"] == "append":
        T = case["tokens"]
        return {"bytes": T * (H + 2 * Hk) * D * 4 + T * (case["rotary"] * 4 + 12),
                "flops": T * (H + Hk) * D * 8}
    if case["kind"] == "train":
        rows, states = case["batch"] * case["seq"], case["batch"] * H * D * D
        n = (2 * H + 2 * Hk) * D * 2  # q, out, k, v; and again dq, dout, dk, dv
        both = case["backward"]
        return {"bytes": rows * n * (2 if both else 1)
                + (states * 4 * (4 if both else 2) if case["state"] else 0),
                "flops": rows * H * D * D * (14 if both else 4)}
    if case["kind"] == "prefill":
        T, states = sum(_lens(case)), case["seqs"] * H * D * D
        return {"bytes": T * (2 * H + 2 * Hk) * D * 2 + states * 6, "flops": T * H * D * D * 4}
    B = case["seqs"]
    return {"bytes": B * H * D * D * 8 + B * (2 * H + 2 * Hk) * D * 2, "flops": B * H * D * D * 5}


# ------------------------------------------------------------------ inputs

def _table(positions, rotary):
    """cos and sin of every position and frequency, [positions, rotary / 2] fp32."""
    inv = 10000.0 ** (-torch.arange(0, rotary, 2, device=DEVICE, dtype=torch.float64) / rotary)
    angle = torch.arange(positions, device=DEVICE, dtype=torch.float64)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _log_decay(heads):
    """Slopes that halve from head to head, as linear-attention models fix them."""
    h = torch.arange(1, heads + 1, device=DEVICE, dtype=torch.float64)
    return (-torch.exp2(-8 * h / heads)).float()


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]

    def randn(*shape, dtype=dtype):
        return torch.randn(*shape, generator=gen, device=DEVICE).to(dtype)

    s = {"case": case}
    if case["kind"] == "rope":
        B, S = case["batch"], case["seq"]
        s["q"], s["k"] = randn(B, S, H, D), randn(B, S, Hk, D)
        s["cos"], s["sin"] = _table(S, case["rotary"])
        # A training program holds the norms' weights in fp32.
        wt = torch.float32 if case["backward"] else dtype
        s["qw"] = (1 + 0.1 * randn(D, dtype=torch.float32)).to(wt)
        s["kw"] = (1 + 0.1 * randn(D, dtype=torch.float32)).to(wt)
        if case["backward"]:
            s["dq"], s["dk"] = randn(B, S, H, D), randn(B, S, Hk, D)
            for name in ("q", "k", "qw", "kw"):
                s[name].requires_grad_()
    elif case["kind"] == "append":
        T, page = case["tokens"], case["page"]
        # The fused projection's output; a user takes q, k and v as views of it.
        s["qkv"] = randn(T, (H + 2 * Hk) * D)
        pages = -(-T // page) + 4
        s["k_cache"], s["v_cache"] = (randn(pages, page, Hk, D) for _ in range(2))
        s["slots"] = torch.randperm(pages * page, generator=gen, device=DEVICE)[:T]
        s["positions"] = torch.randint(0, 32768, (T,), generator=gen, device=DEVICE)
        s["cos"], s["sin"] = _table(32768, case["rotary"])
        s["qw"], s["kw"] = ((1 + 0.1 * randn(D, dtype=torch.float32)).to(dtype)
                            if case["norm"] else None for _ in range(2))
    elif case["kind"] == "train":
        B, S = case["batch"], case["seq"]
        s["q"], s["k"], s["v"] = randn(B, S, H, D), randn(B, S, Hk, D), randn(B, S, Hk, D)
        s["log_decay"] = _log_decay(H)
        s["state"] = randn(B, H, D, D, dtype=torch.float32) if case["state"] else None
        if case["backward"]:
            s["dout"] = randn(B, S, H, D)
            s["dstate"] = randn(B, H, D, D, dtype=torch.float32) if case["state"] else None
            for name in ("q", "k", "v", "state"):
                if s[name] is not None:
                    s[name].requires_grad_()
    elif case["kind"] == "prefill":
        lens = _lens(case)
        T, B = sum(lens), len(lens)
        s["q"], s["k"], s["v"] = randn(T, H, D), randn(T, Hk, D), randn(T, Hk, D)
        s["log_decay"] = _log_decay(H)
        s["pool"] = randn(B + 2, H, D, D, dtype=torch.float32)
        s["slots"] = torch.randperm(B + 2, generator=gen, device=DEVICE)[:B].int()
        starts = [sum(lens[:i]) for i in range(B + 1)]
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE)
        s["prefix"] = torch.tensor([100 * (i % 2) for i in range(B)], dtype=torch.int32,
                                   device=DEVICE)
        s["longest"] = max(lens)
    else:
        B = case["seqs"]
        s["q"], s["k"], s["v"] = randn(B, H, D), randn(B, Hk, D), randn(B, Hk, D)
        s["log_decay"] = _log_decay(H)
        s["pool"] = randn(B + 2, H, D, D, dtype=torch.float32)
        s["slots"] = torch.randperm(B + 2, generator=gen, device=DEVICE)[:B].int()
    return s


# ------------------------------------------------------------------ the framework's calls

def _leaves(s, *names):
    return [s[n] for n in names if s[n] is not None]


def _own(s):
    fa, case = _package(), s["case"]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "rope":
        out = fa.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["qw"], s["kw"], eps=EPS,
                              interleaved=case["interleaved"])
        if not case["backward"]:
            return out
        return out, torch.autograd.grad(out, _leaves(s, "q", "k", "qw", "kw"), (s["dq"], s["dk"]))
    if case["kind"] == "append":
        T = case["tokens"]
        q, k, v = s["qkv"].split([H * D, Hk * D, Hk * D], dim=1)
        q = fa.norm_rope_and_cache(q.view(T, H, D), k.view(T, Hk, D), v.view(T, Hk, D),
                                   s["k_cache"], s["v_cache"], s["slots"], s["positions"],
                                   s["cos"], s["sin"], s["qw"], s["kw"], eps=EPS,
                                   interleaved=case["interleaved"])
        return q, s["k_cache"], s["v_cache"]
    if case["kind"] == "train":
        out = fa.linear_attn_func(s["q"], s["k"], s["v"], s["log_decay"],
                                  initial_state=s["state"], return_final_state=case["state"])
        if not case["backward"]:
            return out
        grads = (s["dout"], s["dstate"]) if case["state"] else (s["dout"],)
        return out, torch.autograd.grad(out, _leaves(s, "q", "k", "v", "state"), grads)
    if case["kind"] == "prefill":
        out = fa.linear_attn_prefill(s["q"], s["k"], s["v"], s["log_decay"], s["pool"],
                                     s["starts"], s["prefix"], state_indices=s["slots"])
        return out, s["pool"]
    out = fa.linear_attn_decode(s["q"], s["k"], s["v"], s["log_decay"], s["pool"],
                                state_indices=s["slots"])
    return out, s["pool"]


# ------------------------------------------------------------------ the plain forms

def _plain_norm(x, weight):
    x = x.float()
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()


def _plain_rotate(x, cos, sin, rotary, interleaved):
    """x [..., heads, D]; cos, sin [..., 1, rotary / 2]."""
    turned, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = turned[..., : rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, rest), -1)


def _plain_linear(q, k, v, log_decay, scale):
    """Chunked linear attention from a zero state, fp32 [B, H, L, D] with L a multiple of CHUNK
    and k, v of H heads: (out, final state).  Decay factors are formed in fp64."""
    B, H, L, D = q.shape
    C, N = CHUNK, L // CHUNK
    g = log_decay.double()[:, None, None]
    n = torch.arange(C, device=q.device, dtype=torch.float64)
    m = torch.arange(N + 1, device=q.device, dtype=torch.float64)
    gap = n[:, None] - n
    inner = torch.where(gap >= 0, torch.exp(g * gap.clamp(min=0)), 0.0).float()
    gap = m[:, None] - 1 - m[:N]
    outer = torch.where(gap >= 0, torch.exp(g * C * gap.clamp(min=0)), 0.0).float()
    before = torch.exp(g * (n[:, None] + 1)).float()[:, None]
    after = torch.exp(g * (C - 1 - n[:, None])).float()[:, None]
    qc, kc, vc = (t.reshape(B, H, N, C, D) for t in (q, k, v))
    scores = (qc @ kc.transpose(-1, -2)) * inner[:, None]
    update = (kc * after).transpose(-1, -2) @ vc
    states = (outer @ update.reshape(B, H, N, D * D)).reshape(B, H, N + 1, D, D)
    out = scores @ vc + (qc * before) @ states[:, :, :N]
    return (scale * out).reshape(B, H, L, D), states[:, :, N]


def _plain_rope(s, rows, cos, sin, weight):
    c = s["case"]
    return _plain_rotate(_plain_norm(rows, weight), cos, sin, c["rotary"], c["interleaved"])


def _plain_train(s):
    case = s["case"]
    q, k, v = (s[n].float().transpose(1, 2) for n in ("q", "k", "v"))
    group, S, D = case["heads"] // case["kv_heads"], case["seq"], case["dim"]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    pad = -S % CHUNK  # zero rows in front: they add nothing to a state
    q, k, v = (torch.nn.functional.pad(t, (0, 0, pad, 0)) for t in (q, k, v))
    scale = D ** -0.5
    out, final = _plain_linear(q, k, v, s["log_decay"], scale)
    out = out[:, :, pad:]
    if case["state"]:
        g = s["log_decay"].double()[:, None, None]
        i = torch.arange(1, S + 1, device=q.device, dtype=torch.float64)[:, None]
        out = out + scale * torch.exp(g * i).float() * (q[:, :, pad:] @ s["state"])
        final = final + torch.exp(g * S).float() * s["state"]
    out = out.transpose(1, 2).to(s["q"].dtype)
    return (out, final) if case["state"] else out


def _plain_prefill(s):
    case = s["case"]
    H, D, pool = case["heads"], case["dim"], s["pool"]
    starts, slots = s["starts"].long(), s["slots"].long()
    lens = starts[1:] - starts[:-1]
    L = s["longest"] + -s["longest"] % CHUNK
    # Sequences end at the last column; rows in front of them are zeros.
    col = torch.arange(L, device=pool.device) - (L - lens)[:, None]
    there = col >= 0
    at = (starts[:-1, None] + col).clamp(min=0)
    group = H // case["kv_heads"]
    q, k, v = (torch.where(there[:, :, None, None], s[n].float()[at], 0.0).transpose(1, 2)
               for n in ("q", "k", "v"))
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    scale = D ** -0.5
    out, final = _plain_linear(q, k, v, s["log_decay"], scale)
    g = s["log_decay"].double()[:, None, None]
    first = torch.where((s["prefix"] > 0)[:, None, None, None], pool[slots], 0.0)
    past = torch.exp(g * (col + 1).clamp(min=0)[:, None, :, None].double()).float()
    out = out + scale * past * (q @ first)
    pool[slots] = final + torch.exp(g * lens[:, None, None, None].double()).float() * first
    rows = torch.arange(s["q"].shape[0], device=pool.device)
    seq = torch.searchsorted(starts, rows, right=True) - 1
    out = out[seq, :, rows - starts[seq] + L - lens[seq]]
    return out.to(s["q"].dtype), pool


def _plain_decode(s):
    case, slots = s["case"], s["slots"].long()
    group, D = case["heads"] // case["kv_heads"], case["dim"]
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    state = s["pool"][slots] * torch.exp(s["log_decay"])[:, None, None]
    state = state + k[..., :, None] * v[..., None, :]
    s["pool"][slots] = state
    out = D ** -0.5 * (q[..., None, :] @ state)[..., 0, :]
    return out.to(s["q"].dtype), s["pool"]


def run(s):
    if own:
        return _own(s)
    case = s["case"]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "rope":
        cos, sin = s["cos"][:, None], s["sin"][:, None]
        out = (_plain_rope(s, s["q"], cos, sin, s["qw"]).to(s["q"].dtype),
               _plain_rope(s, s["k"], cos, sin, s["kw"]).to(s["k"].dtype))
        if not case["backward"]:
            return out
        return out, torch.autograd.grad(out, _leaves(s, "q", "k", "qw", "kw"), (s["dq"], s["dk"]))
    if case["kind"] == "append":
        T, dtype = case["tokens"], s["qkv"].dtype
        q, k, v = s["qkv"].split([H * D, Hk * D, Hk * D], dim=1)
        cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
        q = _plain_rope(s, q.view(T, H, D), cos, sin, s["qw"]).to(dtype)
        k = _plain_rope(s, k.view(T, Hk, D), cos, sin, s["kw"]).to(dtype)
        s["k_cache"].view(-1, Hk, D)[s["slots"]] = k
        s["v_cache"].view(-1, Hk, D)[s["slots"]] = v.view(T, Hk, D)
        return q, s["k_cache"], s["v_cache"]
    if case["kind"] == "train":
        out = _plain_train(s)
        if not case["backward"]:
            return out
        grads = (s["dout"], s["dstate"]) if case["state"] else (s["dout"],)
        return out, torch.autograd.grad(out, _leaves(s, "q", "k", "v", "state"), grads)
    if case["kind"] == "prefill":
        return _plain_prefill(s)
    return _plain_decode(s)


# ------------------------------------------------------------------ exact values

def _exact_turn(x, cos, sin, rotary, interleaved, back=False):
    """The rotation as a complex product; back: its transpose."""
    half = rotary // 2
    a, b = ((x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved
            else (x[..., :half], x[..., half:rotary]))
    z = torch.complex(a, b) * torch.complex(cos, -sin if back else sin)
    y = x.clone()
    if interleaved:
        y[..., 0:rotary:2], y[..., 1:rotary:2] = z.real, z.imag
    else:
        y[..., :half], y[..., half:rotary] = z.real, z.imag
    return y


def _exact_rope(case, x, w, cos, sin, dy=None):
    """(y, dx, dw) in fp64; dy None: y alone.  w None: no norm."""
    x = x.detach().double()
    turn = (cos.double()[..., None, :], sin.double()[..., None, :], case["rotary"],
            case["interleaved"])
    if w is None:
        return _exact_turn(x, *turn)
    w = w.detach().double()
    r = (x.pow(2).mean(-1, keepdim=True) + EPS).pow(-0.5)
    y = _exact_turn(x * r * w, *turn)
    if dy is None:
        return y
    unit = x * r
    g = _exact_turn(dy.double(), *turn, back=True)
    h = g * w
    dx = r * (h - unit * (h * unit).mean(-1, keepdim=True))
    return y, dx, (g * unit).reshape(-1, x.shape[-1]).sum(0)


def _exact_pairs(q, k, v, g, scale, state, dout=None, dstate=None):
    """Linear attention over all pairs in fp64, [B, H, S, D]: (out, final) and with dout
    (dq, dk, dv, dstate0) too; rows in blocks."""
    S = q.shape[2]
    j = torch.arange(S, device=q.device, dtype=torch.float64)
    g = g[:, None, None]
    out, dq = torch.empty_like(q), torch.empty_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for lo in range(0, S, 512):
        hi = min(S, lo + 512)
        gap = j[lo:hi, None] - j[:hi]
        w = scale * torch.where(gap >= 0, torch.exp(g * gap.clamp(min=0)), 0.0)
        a = w * (q[:, :, lo:hi] @ k[:, :, :hi].transpose(-1, -2))
        out[:, :, lo:hi] = a @ v[:, :, :hi]
        if dout is not None:
            d = w * (dout[:, :, lo:hi] @ v[:, :, :hi].transpose(-1, -2))
            dq[:, :, lo:hi] = d @ k[:, :, :hi]
            dk[:, :, :hi] += d.transpose(-1, -2) @ q[:, :, lo:hi]
            dv[:, :, :hi] += a.transpose(-1, -2) @ dout[:, :, lo:hi]
    past, ahead = torch.exp(g * (j[:, None] + 1)), torch.exp(g * (S - 1 - j[:, None]))
    final = (k * ahead).transpose(-1, -2) @ v
    if state is not None:
        out += scale * past * (q @ state)
        final += torch.exp(g * S) * state
    if dout is None:
        return out, final
    dfirst = scale * (q * past).transpose(-1, -2) @ dout
    if state is not None:
        dq += scale * past * (dout @ state.transpose(-1, -2))
        dk += ahead * (v @ dstate.transpose(-1, -2))
        dv += ahead * (k @ dstate)
        dfirst += torch.exp(g * S) * dstate
    return out, final, dq, dk, dv, dfirst


def exact(case, seed):
    s = prepare(case, seed)
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    group, scale = H // Hk, D ** -0.5
    if case["kind"] == "rope":
        both = [_exact_rope(case, s[n], s[n + "w"], s["cos"], s["sin"], s.get("d" + n))
                for n in ("q", "k")]
        if not case["backward"]:
            return both
        (y, dy, dyw), (z, dz, dzw) = both
        return [[y, z], [dy, dz, dyw, dzw]]
    if case["kind"] == "append":
        T, at = case["tokens"], s["slots"]
        x = s["qkv"].view(T, H + 2 * Hk, D)
        cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
        caches = [s[n].double() for n in ("k_cache", "v_cache")]
        caches[0].view(-1, Hk, D)[at] = _exact_rope(case, x[:, H:H + Hk], s["kw"], cos, sin)
        caches[1].view(-1, Hk, D)[at] = x[:, H + Hk:].double()
        return [_exact_rope(case, x[:, :H], s["qw"], cos, sin), *caches]
    g = s["log_decay"].double()
    if case["kind"] == "train":
        q, k, v, do = (s[n].detach().double().transpose(1, 2) if n in s else None
                       for n in ("q", "k", "v", "dout"))
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        state, dstate = (s[n].detach().double() if s.get(n) is not None else None
                         for n in ("state", "dstate"))
        r = _exact_pairs(q, k, v, g, scale, state, do, dstate)
        out = [r[0].transpose(1, 2), r[1]] if case["state"] else r[0].transpose(1, 2)
        if not case["backward"]:
            return out
        B, S = case["batch"], case["seq"]
        dk, dv = (t.reshape(B, Hk, group, S, D).sum(2).transpose(1, 2) for t in r[3:5])
        grads = [r[2].transpose(1, 2), dk, dv] + ([r[5]] if case["state"] else [])
        return [out, grads]
    pool, slots = s["pool"].double(), s["slots"].tolist()
    if case["kind"] == "prefill":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
        starts, prefix = s["starts"].tolist(), s["prefix"].tolist()
        for b, slot in enumerate(slots):
            rows = slice(starts[b], starts[b + 1])
            q, k, v = (s[n][rows].double().transpose(0, 1)[None] for n in ("q", "k", "v"))
            k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
            first = pool[slot][None] if prefix[b] else None
            o, final = _exact_pairs(q, k, v, g, scale, first)
            out[rows] = o[0].transpose(0, 1)
            pool[slot] = final[0]
        return [out, pool]
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    lam = torch.exp(g)
    for b, slot in enumerate(slots):
        pool[slot] = lam[:, None, None] * pool[slot] + k[b][:, :, None] * v[b][:, None, :]
    out = scale * (q[..., None] * pool[s["slots"].long()]).sum(-2)
    return [out, pool]
