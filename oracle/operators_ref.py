"""64-bit references of the operators around attention, on the CPU.

Every function takes tensors of any type, computes in float64 from their
values and returns float64.  The linear attention runs its recurrence token by
token, and its gradients come from autograd through that loop.
"""
from __future__ import annotations

import torch


def norm_rope(x, weight, cos, sin, positions, eps=1e-6, interleaved=False):
    """x [T, H, D], cos / sin [P, R / 2], positions [T]; weight None: no norm.

    A negative position gives zero rows, one at or beyond P NaN in the rotated
    components."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    P, half = cos.shape
    inside = positions < P  # (padding rows are masked below: finite here, for their gradient)
    at = positions.clamp(0, P - 1).long()
    c = torch.where(inside[:, None], cos.double()[at], torch.nan)[:, None]
    s = torch.where(inside[:, None], sin.double()[at], torch.nan)[:, None]
    y = x.clone()
    if interleaved:
        first, second = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
    else:
        first, second = slice(0, half), slice(half, 2 * half)
    a, b = x[..., first], x[..., second]
    y[..., first] = a * c - b * s
    y[..., second] = a * s + b * c
    return torch.where((positions < 0)[:, None, None], 0.0, y)


def linear_attention(q, k, v, log_decay, scale, state=None):
    """q [S, H, D], k / v [S, Hk, D], log_decay [H], state [H, D, D] or None:
    (out [S, H, D], final state)."""
    S, H, D = q.shape
    group = H // k.shape[1]
    q = q.double()
    k, v = (t.double().repeat_interleave(group, 1) for t in (k, v))
    decay = torch.exp(log_decay.double())[:, None, None]
    state = torch.zeros(H, D, D, dtype=torch.float64) if state is None else state.double()
    outs = []
    for t in range(S):
        state = decay * state + k[t, :, :, None] * v[t, :, None, :]
        outs.append(scale * (q[t, :, None, :] @ state)[:, 0])
    out = torch.stack(outs) if outs else torch.zeros(0, H, D, dtype=torch.float64)
    return out, state


def linear_attention_bounds(q, k, v, log_decay, scale, state=None, chunk=64, reverse=False):
    """What the chunked form rounds, in absolute values: (half, full, states).

    half [S, H, D]: the sum of |terms| that carry one rounding to the inputs'
    type each: the rounded scores times v within a chunk, q times the rounded
    state before it.  full: the sum over all products' absolute values, for the
    fp32 sums.  states [H, D, D]: the same for the final state.
    reverse: time runs backwards, and a row sees the carried state without its
    own decay (the gradients of k and v).  state: the one before the first row."""
    if reverse:
        q, k, v = (t.flip(0) for t in (q, k, v))
    S, H, D = q.shape
    group = H // k.shape[1]
    q = q.double()
    k, v = (t.double().repeat_interleave(group, 1) for t in (k, v))
    g = log_decay.double().clamp(min=-1e30)[:, None, None]  # (-inf times 0 rows is 0 here)
    late = 0 if reverse else 1
    before = torch.zeros(H, D, D, dtype=torch.float64) if state is None else state.double()
    size = before.abs()
    half, full = torch.zeros(S, H, D, dtype=torch.float64), torch.zeros(S, H, D, dtype=torch.float64)
    for c in range(0, S, chunk):
        n = min(chunk, S - c)
        i = torch.arange(n, dtype=torch.float64)
        qc, kc, vc = (t[c:c + n].transpose(0, 1) for t in (q, k, v))
        gap = i[:, None] - i
        w = torch.where(gap >= 0, torch.exp(g * gap.clamp(min=0)), 0.0)
        past = torch.exp(g * (i[:, None] + late))
        scores = qc @ kc.transpose(1, 2)
        h = (w * scores).abs() @ vc.abs() + past * (qc.abs() @ before.abs())
        f = (w * (qc.abs() @ kc.abs().transpose(1, 2))) @ vc.abs() + past * (qc.abs() @ size)
        half[c:c + n], full[c:c + n] = h.transpose(0, 1), f.transpose(0, 1)
        after = torch.exp(g * (n - late - i[:, None]))
        keep = torch.exp(g * n)
        before = keep * before + (kc * after).transpose(1, 2) @ vc
        size = keep * size + (kc.abs() * after).transpose(1, 2) @ vc.abs()
    if reverse:
        half, full = half.flip(0), full.flip(0)
    return abs(scale) * half, abs(scale) * full, size
