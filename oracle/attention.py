"""The attention half of a decoder layer in float64 on the CPU, from the formulas.

Test infrastructure only.  Norm and rotation of head rows, the paged cache as
plain indexing, and softmax attention one (query, head) at a time over exactly
the keys that the query sees, with the error that the device kernels' roundings
can cause beside each value.
"""

from __future__ import annotations

import math

import torch

F64 = torch.float64
BF16_HALF_STEP = 2.0 ** -8     # rounding to bf16: at most this, relative
F32_HALF_STEP = 2.0 ** -24


def norm_rope(x, positions, freq=None, *, interleaved=False, rot_first=0, mscale=1.0, gamma=None, norm=True, eps=1e-6):
    """(y, tol) [T, heads, D] float64 for x of any float type.

    tol: one rounding to bf16 of y, and float32 arithmetic before it: a norm's value carries at most D / 8 + 8
    roundings of its mean (8 a lane, then a tree), halved by the root, and 6 more; a rotated one is the sum of
    two products whose factors have 4 half steps each (the angle's fraction, sine or cosine, mscale, gamma):
    16 + D / 8 half steps of the pair's magnitude bound both."""
    x = x.to(F64)
    d = x.shape[-1]
    y = x.clone()
    if norm:
        y = y / torch.sqrt((x * x).sum(-1, keepdim=True) / d + eps)
        if gamma is not None:
            y = y * gamma.to(F64)
    mag = y.abs()
    if freq is not None:
        r = freq.numel()
        i = torch.arange(r)
        a, b = (rot_first + 2 * i, rot_first + 2 * i + 1) if interleaved else (rot_first + i, rot_first + i + r)
        t = positions.to(F64)[:, None] * freq.to(F64).cpu()
        c, s = (mscale * torch.cos(t))[:, None], (mscale * torch.sin(t))[:, None]
        ya, yb = y[..., a].clone(), y[..., b].clone()
        y[..., a], y[..., b] = ya * c - yb * s, yb * c + ya * s
        both = (ya.abs() + yb.abs()) * max(1.0, abs(mscale))
        mag[..., a], mag[..., b] = both, both
        # the angle itself: float32 holds a fraction of a turn to 2^-25, 2 pi of it in radians,
        # and positions * freq in float64 to 2^-52
    tol = BF16_HALF_STEP * y.abs() + (16 + d / 8) * F32_HALF_STEP * mag * 1.01
    return y, tol + 1e-38


def rows_of(cache, pages, n):
    """Rows 0..n-1 of a sequence whose pages are given: [n, kv heads, D]."""
    page = cache.shape[2]
    at = torch.arange(n)
    return cache[pages.long()[at // page], :, at % page]


def attention(q, k, v, last, scale):
    """(o, tol) of q [Lq, heads, D] over k, v [Lk, kv heads, D]; query i sees the keys 0..last[i] (none: zeros).

    Roundings: p (the weight before normalisation) to bf16, 2^-8 of each term; the scores' sums of D products and
    the sums over the keys in float32, at most n and D steps of them; the result to bf16.  Where the kernels divide by the
    sum of the rounded weights, a term's rounding counts with |v - o| instead of |v|: less, but where nearly all of the value is
    that of keys of little weight, and all roundings fall the worst way, up to o's half step more."""
    q, k, v = q.to(F64), k.to(F64), v.to(F64)
    heads, kv = q.shape[1], k.shape[1]
    o, tol = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(q.shape[0]):
        n = min(int(last[i]) + 1, k.shape[0])
        if n <= 0:
            continue
        for h in range(heads):
            kh, vh = k[:n, h * kv // heads], v[:n, h * kv // heads]
            s = scale * (kh @ q[i, h])
            w = torch.softmax(s, 0)
            o[i, h] = w @ vh
            size = scale * float((kh.abs() @ q[i, h].abs()).max())
            slack = 4.0 * (n + q.shape[2] * size + 16) * F32_HALF_STEP
            tol[i, h] = (w @ vh.abs()) * (BF16_HALF_STEP + slack) + o[i, h].abs() * BF16_HALF_STEP * (1 + 2.0 ** -6)
    return o, tol + 1e-38


def prompt(q, k, v, cu_q, cu_k, causal=True, scale=None):
    """(o, tol) over packed sequences; rows of no sequence are NaN in o."""
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[2])
    o, tol = torch.full(q.shape, math.nan, dtype=F64), torch.zeros(q.shape, dtype=F64)
    for b in range(len(cu_q) - 1):
        q0, q1, k0, k1 = cu_q[b], cu_q[b + 1], cu_k[b], cu_k[b + 1]
        lq, lk = q1 - q0, k1 - k0
        last = torch.arange(lq) + lk - lq if causal else torch.full((lq,), lk - 1)
        o[q0:q1], tol[q0:q1] = attention(q[q0:q1], k[k0:k1], v[k0:k1], last, scale)
    return o, tol


def paged(q, k_cache, v_cache, table, lens, prefix=None, prefix_len=0, scale=None):
    """(o, tol) of q [batch, q_len, heads, D]: query i sees the prefix and the own keys 0 .. lens - q_len + i."""
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[3])
    o, tol = torch.zeros(q.shape, dtype=F64), torch.zeros(q.shape, dtype=F64)
    for b in range(q.shape[0]):
        n = max(0, int(lens[b]))
        k, v = rows_of(k_cache, table[b], n), rows_of(v_cache, table[b], n)
        if prefix_len:
            k = torch.cat([rows_of(k_cache, prefix, prefix_len), k])
            v = torch.cat([rows_of(v_cache, prefix, prefix_len), v])
        own = torch.arange(q.shape[1]) + n - q.shape[1]
        last = prefix_len + torch.clamp(own, min=-1)
        o[b], tol[b] = attention(q[b], k, v, last, scale)
    return o, tol
