"""Attention block in 64 bits on the host: rotation with norms and cache store, attention over packed or paged keys, and how
far a computation in fewer bits may be off.  Written from the definitions, one row at a time."""

from __future__ import annotations

import math

import torch

HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def rotate(x, positions, cos_sin, weight=None, eps=1e-6, interleaved=False):
    """x [T, heads, D] -> (result, bound of its error before the last rounding) in 64 bits."""
    x, table = x.double(), cos_sin.double()
    dim, rotary = x.size(-1), cos_sin.size(1)
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    out, size = x.clone(), x.abs()
    for t, p in enumerate(positions.tolist()):
        for i in range(rotary // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)
            c, s = (table[p, i], table[p, rotary // 2 + i]) if 0 <= p < table.size(0) else (math.nan, math.nan)
            out[t, :, a], out[t, :, b] = x[t, :, a] * c - x[t, :, b] * s, x[t, :, a] * s + x[t, :, b] * c
            size[t, :, a] = size[t, :, b] = x[t, :, a].abs() + x[t, :, b].abs()
    # fp32: the mean of D squares (D roundings, halved by the root), root, quotient, weight (5), two products and a sum (3)
    return out, size * (dim / 2 + 8) * 2.0**-24


def visible(position, total, causal, window, sinks):
    """Keys that the row at `position` of a sequence of `total` keys sees."""
    if not causal:
        return list(range(total))
    return [j for j in range(min(position + 1, total)) if window == 0 or j > position - window or j < sinks]


def attend(q, k, v, causal=True, window=0, sinks=0, scale=None, dtype=torch.float32, hidden=()):
    """q [Lq, heads, D] at the end of k, v [Lk, kv_heads, D] -> (result, bound of its error with `dtype` outputs), 64 bits.
    `hidden`: keys that no row sees."""
    rows, heads, dim = q.shape
    total, kv_heads = k.shape[:2]
    scale = dim**-0.5 if scale is None else scale
    out = torch.zeros(rows, heads, dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    step = HALF_STEP[dtype]
    k, v, q = k.double(), v.double(), q.double()
    for i in range(rows):
        seen = [j for j in visible(total - rows + i, total, causal, window, sinks) if j not in hidden]
        if not seen:
            continue
        for g in range(kv_heads):
            kk, vv = k[seen, g], v[seen, g]
            qq = q[i, g * (heads // kv_heads) : (g + 1) * (heads // kv_heads)]
            scores = qq @ kk.T * scale
            p = torch.softmax(scores, dim=-1)
            o, a = p @ vv, p @ vv.abs()
            # a score's D products and sums in fp32 (D + 2 roundings) times its terms, and exp2's argument once more: that much is p's
            # relative error, twice with the sum l; then n additions of p v and of p; p's own rounding; the result's
            terms = (qq.abs() @ kk.abs().T * abs(scale)).amax(-1, keepdim=True)
            wrong = 2 * ((dim + 6) * 2.0**-24 * terms + 2.0**-21) + 2 * (len(seen) + 8) * 2.0**-24
            rows_of = slice(g * (heads // kv_heads), (g + 1) * (heads // kv_heads))
            out[i, rows_of] = o
            # (fp16: the weights below its least normal number are off by 2^-25 each, of a largest of one)
            # (element by element of v: sum_j 2^-25 |v_je| <= n 2^-25 max_j |v_je|, and a NaN in one element is no bound of another's)
            tiny = len(seen) * 2.0**-25 * vv.abs().amax(0) if dtype == torch.float16 else 0.0
            # sum l may be of the rounded weights: o = (sum p (1 + e) v) / (sum p (1 + e)) with |e| <= step, off by at most step (a + |o|) to
            # first order, and by that times 2 step beyond it; then the result's own rounding
            bound[i, rows_of] = (wrong + step * (1 + 2 * step)) * a + tiny + step * o.abs() * (2 + 3 * step)
    return out, bound
