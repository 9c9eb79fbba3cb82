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
        # positions [T], or [T, pairs] where pairs turn by axes of their own
        t = (positions if positions.dim() == 2 else positions[:, None]).to(F64) * freq.to(F64).cpu()
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


def attention_of_many(q, k, v, last, scale):
    """``attention`` with the rows of a key head at once, for long sequences."""
    heads, kv, n = q.shape[1], k.shape[1], k.shape[0]
    o, tol = torch.zeros(q.shape, dtype=F64), torch.zeros(q.shape, dtype=F64)
    hidden = torch.arange(n)[:, None] > last.repeat_interleave(heads // kv)[None]
    seen = (last + 1).clamp(0, n).repeat_interleave(heads // kv)[:, None]
    for g in range(kv):
        mine = slice(g * heads // kv, (g + 1) * heads // kv)
        rows, kh, vh = q[:, mine].to(F64).flatten(0, 1), k[:, g].to(F64).contiguous(), v[:, g].to(F64).contiguous()
        w = torch.softmax((kh @ rows.t()).mul_(scale).masked_fill_(hidden, -math.inf), 0).nan_to_num_(0.0).t()
        size = scale * (kh.abs() @ rows.abs().t()).masked_fill_(hidden, 0.0).amax(0)[:, None]
        y = w @ vh
        slack = 4.0 * (seen + q.shape[2] * size + 16) * F32_HALF_STEP
        bound = (w @ vh.abs()) * (BF16_HALF_STEP + slack) + y.abs() * BF16_HALF_STEP * (1 + 2.0 ** -6)
        o[:, mine], tol[:, mine] = y.view(q.shape[0], -1, q.shape[2]), bound.view(q.shape[0], -1, q.shape[2])
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


def key_weights(q, k, last, scale):
    """(w, tol) [Lk, kv heads]: softmax weight that each key receives from q [Lq, heads, D], in all.

    A weight is 2 to a float32 score: its relative error is the score's absolute one, D products and their sums
    of at most |q| |k| each, with the logarithm of the sum taken off (n terms); one rounding for every addition."""
    q, k = q.to(F64), k.to(F64)
    heads, kv = q.shape[1], k.shape[1]
    w, tol = torch.zeros(k.shape[:2], dtype=F64), torch.zeros(k.shape[:2], dtype=F64)
    for i in range(q.shape[0]):
        n = min(int(last[i]) + 1, k.shape[0])
        if n <= 0:
            continue
        for h in range(heads):
            g = h * kv // heads
            kh = k[:n, g]
            p = torch.softmax(scale * (kh @ q[i, h]), 0)
            size = scale * float((kh.abs() @ q[i, h].abs()).max())
            w[:n, g] += p
            tol[:n, g] += p * 4.0 * (n + q.shape[2] * size + 16) * F32_HALF_STEP
    return w, tol + w * q.shape[0] * heads * F32_HALF_STEP


# ------------------------------------------------------------------ the cache in 8 bits
BLOCK = 16
LEAST, MOST = 27, 246

_CODES = torch.tensor([[(-1.0) ** (c >> 7) * ((c & 7) / 8 * 2.0 ** -6 if not c >> 3 & 15 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3 & 15) - 7)),
                        math.nan][c & 127 == 127] for c in range(256)], dtype=F64)


def to_codes(x, byte):
    """uint8 e4m3 codes of x (float64) in the scale of byte (same shape), nearest, ties to the even code."""
    y = x / 2.0 ** (byte.to(F64) - 127)
    size = y.abs().nan_to_num(0.0).clamp(max=448.0)
    positive = _CODES[:127]
    hi = torch.searchsorted(positive, size).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    low, high = size - positive[lo], positive[hi] - size
    code = torch.where((low < high) | ((low == high) & (lo % 2 == 0)), lo, hi)
    code = torch.where(torch.signbit(y), code + 128, code)
    return torch.where(torch.isfinite(x), code, torch.full_like(code, 127)).to(torch.uint8)


def values(codes, byte):
    """float64 values of uint8 codes [pages, kv heads, page, D] with scales [pages, kv heads, page / 16]."""
    return _CODES[codes.long()] * 2.0 ** (byte.to(F64).repeat_interleave(BLOCK, -1)[..., None] - 127)


def scale_byte(top):
    """Least b with top <= 448 * 2^(b - 127) (a float), in range."""
    if top == 0:
        return LEAST
    m, e = math.frexp(top / 448.0)
    return min(max((e if m > 0.5 else e - 1) + 127, LEAST), MOST)


def append_codes(x, codes, byte, slots):
    """codes and byte (changed in place) after a call whose token t brings the rows x[t] [kv heads, D] to
    (page, row) = slots[t] (None: not kept)."""
    blocks = {}
    for t, at in enumerate(slots):
        if at is not None:
            blocks.setdefault((at[0], at[1] // BLOCK), []).append((t, at[1]))
    for (page, sub), rows in blocks.items():
        for h in range(x.shape[1]):
            brought = torch.stack([x[t, h] for t, _ in rows]).to(F64)
            b = scale_byte(float(torch.where(torch.isfinite(brought), brought.abs(), torch.zeros_like(brought)).max()))
            if not any(r % BLOCK == 0 for _, r in rows):
                old = int(byte[page, h, sub])
                b = max(b, old)
                if b > old:
                    block = codes[page, h, sub * BLOCK:(sub + 1) * BLOCK]
                    block[:] = rescale(block, old, b)
            byte[page, h, sub] = b
            for t, r in rows:
                codes[page, h, r] = to_codes(x[t, h].to(F64), torch.tensor(b))


def rescale(codes, old, new):
    """Codes of the scale of byte old in that of new; a NaN stays one."""
    got = to_codes(_CODES[codes.long()] * 2.0 ** (old - new), torch.tensor(127))
    return torch.where((codes & 127) == 127, codes, got)


def evict(caches, weights, table, lens, keep, first, recent, page):
    """New lengths; caches (a list of (rows [pages, kv heads, page, D], scales or None)) and weights are changed in place.

    Row by row from the definition: an item's whole order first, then all of its rows at once."""
    new = []
    n_pages = weights.shape[0]
    for b, n in enumerate(lens):
        if n <= keep or n > table.shape[1] * page:
            new.append(n)
            continue
        new.append(keep)
        place = [(int(table[b, j // page]), j % page) for j in range(n)]
        ok = [0 <= p < n_pages for p, _ in place]
        for h in range(weights.shape[1]):
            def order(j):
                w = float(weights[place[j][0], h, place[j][1]]) if ok[j] else None
                return (0 if w is None else 2 if math.isnan(w) else 1, 0.0 if w is None or math.isnan(w) else w)
            free = sorted(range(first, n - recent), key=order, reverse=True)      # (stable: of equal ones the earlier)
            stay = set(free[:keep - first - recent]) | set(range(first))
            middle = keep - recent
            src = list(range(middle)) + [n - recent + i for i in range(recent)]
            fills = iter(sorted(j for j in stay if j >= middle))
            for j in range(middle):
                if j not in stay:
                    src[j] = next(fills)
            assert next(fills, None) is None
            src = [s if ok[s] else j for j, s in enumerate(src)]
            moved = [j for j in range(keep) if src[j] != j and ok[j]]
            had = {j: (weights[place[src[j]][0], h, place[src[j]][1]].clone(),
                       [(r[place[src[j]][0], h, place[src[j]][1]].clone(), None if s is None else int(s[place[src[j]][0], h, place[src[j]][1] // BLOCK]))
                        for r, s in caches])
                   for j in range(keep) if ok[j]}
            # in 8 bits a block is touched as a whole, also where the row that should come is not there
            want = {j // BLOCK for j in range(middle) if j not in stay} | ({j // BLOCK for j in range(middle, keep)} if recent else set())
            for j in moved:
                weights[place[j][0], h, place[j][1]] = had[j][0]
            for c, (rows, scales) in enumerate(caches):
                if scales is None:
                    for j in moved:
                        rows[place[j][0], h, place[j][1]] = had[j][1][c][0]
                    continue
                for block in sorted(want):
                    js = [j for j in range(block * BLOCK, min((block + 1) * BLOCK, keep)) if ok[j]]
                    if not js:
                        continue
                    top = max(had[j][1][c][1] for j in js)
                    for j in js:
                        code, byte = had[j][1][c]
                        rows[place[j][0], h, place[j][1]] = rescale(code, byte, top) if byte != top else code
                    scales[place[js[0]][0], h, place[js[0]][1] // BLOCK] = top
    return new
