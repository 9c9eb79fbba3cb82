"""The attention operators at the sizes where other forms of their kernels run
than for a few rows: norm and rotation by whole tokens, prompts whose row tiles
come to a CU twice, long runs of keys.  Every row is looked at.

Long sums hide a lost key (each weighs 1 / n of inputs drawn alike), so the
long cases are built to show one: keys that a query finds alone among all of
them, and equal weights over values that mark a range of keys, whose exact
fraction then comes out."""

from __future__ import annotations

import math

import pytest
import torch

import dsk_moe
from oracle import attention as O
from test_gpu_attention import BF16, DEV, F32, I32, INF, NAN, assert_within, cumulative, gen, ints, normal, paged_setup

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ norm, rotation, append by whole tokens
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,first,inter", [(2047, 9, 5, 64, 64, 0, False), (2048, 9, 5, 64, 32, 8, True),
                                                                 (2051, 33, 7, 128, 128, 0, False), (2049, 5, 5, 128, 64, 64, True),
                                                                 (2048, 0, 3, 64, 64, 0, False)])
def test_whole_token_append(dtype, tokens, heads, kv, dim, rot, first, inter):
    """Views of one projection's rows into a cache: some tokens are padding (their rows stay), some have no page, row or
    sequence (their q and k are still written)."""
    print(f"append {dtype} {tokens}x{heads},{kv} of {dim}", flush=True)
    g = gen(tokens + heads)
    page, prefix, width = 32, 11, 12
    qkv = normal(g, tokens, (heads + 2 * kv) * dim, dtype=dtype) * 2
    split = lambda t: [p.unflatten(1, (-1, dim)) if p.shape[1] else None for p in t.split([heads * dim, kv * dim, kv * dim], 1)]  # noqa: E731
    q, k, v = split(qkv)
    n_seqs = -(-tokens // 300)
    row = torch.arange(tokens) % 300
    seq = (torch.arange(tokens) // 300).to(I32)
    table, kc, vc = paged_setup(g, [10] * n_seqs, width, 4, kv, page, dim)
    table[0, 3], table[1, 9] = 1 << 30, -2                       # pages outside the cache
    order = torch.randperm(tokens, generator=g)
    row, seq = row[order], seq[order]
    pos = (row + prefix).to(I32)
    pos[::37] = -1                                               # padding
    pos[5::91] = 3                                               # before the prefix's end
    pos[7::101] = prefix + width * page                          # behind the table row
    seq[9::97] = n_seqs
    seq[11::89] = -1
    at = pos.long() - prefix
    ok = (pos >= 0) & (at >= 0) & (at < width * page) & (seq >= 0) & (seq < n_seqs)
    ids = table[seq.long().clamp(0, n_seqs - 1), (at // page).clamp(0, width - 1)].long()
    ok &= (ids >= 0) & (ids < kc.shape[0])
    freq = dsk_moe.rope_frequencies(rot, device="cpu")[0]
    gq, gk = torch.rand(dim, generator=g) + 0.5, torch.rand(dim, generator=g) + 0.5
    kw = dict(interleaved=inter, rot_first=first, mscale=1.25)
    kd, vd = kc.to(DEV), vc.to(DEV)
    qd, kk, vv = split(qkv.to(DEV))
    qo = torch.full((tokens, heads, dim), 9.0, dtype=BF16, device=DEV) if heads else None
    ko = torch.full((tokens, kv, dim), 8.0, dtype=BF16, device=DEV)
    dsk_moe.kv_append(qd, kk, vv, pos.to(DEV), seq.to(DEV), table.to(DEV), kd, vd, freq.to(DEV), prefix_len=prefix, q_out=qo, k_out=ko,
                      q_gamma=gq.to(DEV) if heads else None, k_gamma=gk.to(DEV), **kw)
    live = pos >= 0
    for x, out, gamma, fill in ((q, qo, gq, 9.0), (k, ko, gk, 8.0)):
        if x is not None:
            want, tol = O.norm_rope(x[live], pos[live], freq, gamma=gamma, **kw)
            assert_within(out.cpu()[live], want, tol)
            assert (out.cpu()[~live] == fill).all()
    r = (at % page)[ok]
    kc[ids[ok], :, r] = ko.cpu()[ok]
    vc[ids[ok], :, r] = v[ok].to(BF16)
    assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), vc)
    # without the copy of the keys, the same in the cache and in q
    kd2, vd2 = torch.full_like(kd, 3.0), torch.full_like(vd, 3.0)
    q2 = torch.full_like(qo, 9.0) if heads else None
    dsk_moe.kv_append(qd, kk, vv, pos.to(DEV), seq.to(DEV), table.to(DEV), kd2, vd2, freq.to(DEV), prefix_len=prefix, q_out=q2,
                      q_gamma=gq.to(DEV) if heads else None, k_gamma=gk.to(DEV), **kw)
    assert q2 is None or torch.equal(q2, qo)
    assert torch.equal(kd2[ids[ok].to(DEV), :, r.to(DEV)], kd[ids[ok].to(DEV), :, r.to(DEV)])
    assert int((kd2 != 3.0).any(-1).sum()) <= int(ok.sum()) * kv


@pytest.mark.parametrize("tokens", [2047, 2048, 2051])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("heads,kv,dim", [(9, 5, 64), (20, 3, 128)])
def test_whole_token_rotation_in_place(tokens, inter, heads, kv, dim):
    g = gen(tokens + dim)
    qkv = normal(g, tokens, (heads + 2 * kv) * dim)
    pos = torch.randint(0, 100000, (tokens,), generator=g, dtype=I32)
    pos[3::50] = -1
    freq = dsk_moe.rope_frequencies(dim, device="cpu")[0]
    live = pos >= 0
    dev = qkv.to(DEV)
    q, k, v = (p.unflatten(1, (-1, dim)) for p in dev.split([heads * dim, kv * dim, kv * dim], 1))
    dsk_moe.qk_norm_rope(q, k, pos.to(DEV), freq.to(DEV), interleaved=inter, q_out=q, k_out=k)
    q0, k0, v0 = (p.unflatten(1, (-1, dim)) for p in qkv.split([heads * dim, kv * dim, kv * dim], 1))
    for got, x in ((q, q0), (k, k0)):
        want, tol = O.norm_rope(x[live], pos[live], freq, interleaved=inter)
        # positions * freq / (2 pi) in float64: 2^-52 of 2^17 radians, far below float32's half step
        assert_within(got.cpu()[live], want, tol)
        assert torch.equal(got.cpu()[~live], x[~live])
    assert torch.equal(v.cpu(), v0)


# ------------------------------------------------------------------ prompts
def prompt_on_device(q, k, v, lens, lens_k, causal):
    """(o, tol) of every row in float64 on the device, head by head, with the oracle's tolerance (its largest |q||k| over
    a head in the place of a row's); rows of no sequence are zero with no tolerance."""
    o = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(o)
    heads, kv, dim = q.shape[1], k.shape[1], q.shape[2]
    cu, ck = cumulative(lens), cumulative(lens_k)
    for b in range(len(lens)):
        n, nk = lens[b], lens_k[b]
        if not n or not nk:
            continue
        hidden = torch.arange(nk, device=DEV)[None] > torch.arange(n, device=DEV)[:, None] + (nk - n if causal else nk)
        none = hidden.all(1, keepdim=True)
        for h in range(heads):
            qh = q[cu[b]:cu[b + 1], h].double()
            kh, vh = (x[ck[b]:ck[b + 1], h * kv // heads].double() for x in (k, v))
            w = torch.softmax((qh @ kh.T / dim ** 0.5).masked_fill(hidden, -INF), -1).masked_fill(none, 0.0)
            want = w @ vh
            slack = 4 * (nk + dim * float((qh.abs() @ kh.abs().T).max()) / dim ** 0.5 + 16) * 2.0 ** -24
            o[cu[b]:cu[b + 1], h] = want
            tol[cu[b]:cu[b + 1], h] = (w @ vh.abs()) * (2.0 ** -8 + slack) + want.abs() * 2.0 ** -8 * (1 + 2.0 ** -6) + 1e-38
    return o, tol


@pytest.mark.parametrize("heads,kv,dim,lens,before,causal", [
    (10, 5, 128, [4000, 17, 0, 2500, 483], 0, True),             # 128-row tiles, 51 a CU row of 5 heads: 110 of them
    (10, 5, 64, [4000, 17, 0, 2500, 483], 0, True),
    (12, 12, 64, [1500, 1, 2200, 300], 0, True),                 # 64-row tiles: 64 of 21 at once
    (12, 12, 128, [1500, 1, 2200, 300], 0, True),
    (24, 12, 128, [3000, 900, 45], 0, True),                     # 62 of 21
    (16, 2, 64, [900, 0, 1300, 2], 513, True),
    (8, 8, 128, [5000], 0, True),                                # 40 of 32
    (8, 8, 64, [4500, 100], 0, False)])
def test_prompts_of_many_row_tiles(heads, kv, dim, lens, before, causal):
    print(f"prompts {heads},{kv} of {dim}: {lens} behind {before}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(sum(lens) + dim)
    lens_k = [n + before for n in lens]
    t, tk = sum(lens) + 3, sum(lens_k)
    q, k, v = (torch.randn((n, h, dim), generator=g, device=DEV).to(BF16) for n, h in ((t, heads), (tk, kv), (tk, kv)))
    out = torch.full((t, heads, dim), NAN, dtype=BF16, device=DEV)
    dsk_moe.prompt_attention(q, k, v, ints(cumulative(lens)), ints(cumulative(lens_k)), causal=causal, out=out)
    want, tol = prompt_on_device(q, k, v, lens, lens_k, causal)
    assert out[-3:].isnan().all()
    got = out[:-3].double()
    assert not got.isnan().any()
    assert ((got - want[:-3]).abs() <= tol[:-3]).all()


# ------------------------------------------------------------------ keys that are found, keys that are counted
def codes(g, n, dim):
    """n rows of random signs: a row's product with itself is dim, with another one 0 +- sqrt(dim)."""
    return (torch.randint(0, 2, (n, dim), generator=g) * 2 - 1).to(BF16)


def scale_that_finds(q, k, wanted):
    """A scale with which each row's wanted key outweighs all others together 2^40 times, in exponents below 2^10."""
    s = q.float() @ k.float().T
    own = s.gather(1, wanted[:, None])
    rest = s.scatter(1, wanted[:, None], -INF).amax(1, keepdim=True)
    gap = float((own - rest).min())
    assert gap > 0
    return (40.0 + math.log2(k.shape[0])) * math.log(2.0) / gap


EDGES = [0, 15, 16, 31, 32, 63, 64, 127, 128, 255, 256, 1023, 1024, 4095, 4096, 4223, 8191, 8192, 16383, 16384, 20479]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,lens_k", [([300], [20500]), ([40, 3, 70], [9000, 4100, 131]), ([5000], [5000])])
def test_prompt_finds_every_key(dim, lens, lens_k):
    """Each row asks for one key: those at the edges of tiles, its own last one, and others at random; the first key that
    it does not see answers to it even louder."""
    g = gen(dim + sum(lens_k))
    heads, kv = 4, 2
    cu, ck = cumulative(lens), cumulative(lens_k)
    k = torch.stack([codes(g, ck[-1], dim) for _ in range(kv)], 1)
    v = normal(g, ck[-1], kv, dim)
    q = torch.zeros(cu[-1], heads, dim, dtype=BF16)
    target = torch.zeros(cu[-1], heads, dtype=torch.long)
    for b in range(len(lens)):
        n, nk = lens[b], lens_k[b]
        last = torch.arange(n) + nk - n
        for h in range(heads):
            t = (torch.rand(n, generator=g) * (last + 1)).long()
            t[1::5] = last[1::5]
            t[2::5] = (last[2::5] // 64 * 64 - 1).clamp(min=0)
            e = torch.tensor([x for x in EDGES if x < nk])
            at = torch.arange(0, n, 5)
            t[at] = torch.minimum(e[torch.arange(len(at)) % len(e)], last[at])
            target[cu[b]:cu[b + 1], h] = ck[b] + t
            q[cu[b]:cu[b + 1], h] = k[ck[b] + t, h * kv // heads]
    # the gap between a code's product with itself and with any of the others, over the heads
    scale = max(scale_that_finds(q[cu[b]:cu[b + 1], h].to(DEV), k[ck[b]:ck[b + 1], h * kv // heads].to(DEV),
                                 (target[cu[b]:cu[b + 1], h] - ck[b]).to(DEV)) for b in range(len(lens)) for h in range(heads))
    assert scale * dim * math.log2(math.e) < 1024
    want = torch.stack([v[target[:, h], h * kv // heads] for h in range(heads)], 1)
    got = dsk_moe.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), ints(cu), ints(ck), scale=scale)
    assert torch.equal(got.cpu(), want)
    # the rows whose target is the key before their last one, and the last one's bits
    q2, k2 = q.clone(), k.clone()
    b, nk = 0, lens_k[0]
    k2[ck[0] + nk - 1] = 2 * k2[ck[0] + nk - 2]                   # louder, and for the last row alone
    q2[cu[1] - 2] = k[ck[0] + nk - 2].repeat_interleave(heads // kv, 0)
    q2[cu[1] - 1] = q2[cu[1] - 2]
    got = dsk_moe.prompt_attention(q2.to(DEV), k2.to(DEV), v.to(DEV), ints(cu), ints(ck), scale=scale).cpu()
    assert torch.equal(got[cu[1] - 2], v[ck[0] + nk - 2].repeat_interleave(heads // kv, 0))
    assert torch.equal(got[cu[1] - 1], v[ck[0] + nk - 1].repeat_interleave(heads // kv, 0))


def fractions(n, dim, first=0):
    """Values [n, dim] that mark ranges: element d is 1 for the keys of range first + d of 64, 0 for others; and how
    many keys each range has."""
    at = torch.arange(n) // 64 - first
    v = torch.zeros(n, dim, dtype=BF16)
    rows = (at >= 0) & (at < dim)
    v[torch.arange(n)[rows], at[rows]] = 1.0
    return v, v.float().sum(0).double()


@pytest.mark.parametrize("dim,lens,nk", [(64, 48, 40000), (128, 300, 20500), (64, 5000, 5000), (128, 3000, 9100)])
def test_prompt_counts_every_key(dim, lens, nk):
    """q of zeros weighs all visible keys alike: a row that sees m keys has fraction (keys of the range) / m at each range of
    64, within one rounding of the result: 64 keys or 63 differ by 2^-6."""
    heads, kv = 4, 4
    q = torch.zeros(lens, heads, dim, dtype=BF16, device=DEV)
    k = normal(gen(1), nk, kv, dim).to(DEV)
    ranges = -(-nk // 64)
    m = (torch.arange(lens) + nk - lens + 1).double()
    for first in range(0, ranges, dim * kv):
        v = torch.stack([fractions(nk, dim, first + dim * h)[0] for h in range(kv)], 1)
        got = dsk_moe.prompt_attention(q, k, v.to(DEV), ints([0, lens]), ints([0, nk])).cpu().double()
        for h in range(kv):
            lo = 64.0 * (first + dim * h + torch.arange(dim).double())
            want = (m[:, None] - lo).clamp(0.0, 64.0) / m[:, None]
            assert ((got[:, h] - want).abs() <= want * (2.0 ** -8 + 2.0 ** -12)).all(), (first, h)


@pytest.mark.parametrize("dim,heads,kv,q_len,page,width_keys,prefix", [
    (128, 8, 2, 1, 64, 20500, 0), (64, 4, 1, 2, 16, 20500, 0), (128, 4, 2, 1, 16, 500, 0), (64, 8, 2, 4, 32, 1000, 0),
    (128, 8, 2, 1, 64, 4300, 9000), (64, 4, 2, 2, 16, 600, 4230), (128, 40, 1, 1, 64, 5000, 0)])
def test_paged_finds_every_key(dim, heads, kv, q_len, page, width_keys, prefix):
    """Each query row asks for one key of its sequence or of the prefix and gets its value, bit for bit; a key behind the
    sequence's end answers louder and is not heard."""
    print(f"paged {heads},{kv} of {dim}, {q_len} tokens, page {page}, {width_keys} keys behind {prefix}", flush=True)
    g = gen(dim + page + q_len)
    lens = [width_keys - 3, 1 + q_len, 129, 64, width_keys // 2, 130 if width_keys > 200 else 33]
    used = [-(-width_keys // page)] * len(lens)
    shared = -(-prefix // page)
    table, kc, vc = paged_setup(g, used + [shared], max(used[0], shared), 0, kv, page, dim)
    pre, table = table[-1, :shared], table[:-1, :used[0]].contiguous()
    kc.copy_(codes(g, kc[..., 0].numel(), dim).view(kc.shape))
    group = heads // kv
    q = torch.zeros(len(lens), q_len, heads, dim, dtype=BF16)
    want = torch.zeros_like(q)
    scale = 0.0
    for b, n in enumerate(lens):
        k, v = O.rows_of(kc, table[b], n), O.rows_of(vc, table[b], n)
        if prefix:
            k = torch.cat([O.rows_of(kc, pre, prefix), k])
            v = torch.cat([O.rows_of(vc, pre, prefix), v])
        edges = [x for x in [prefix - 1, prefix, 4095, 4096, 4159, 4223, 4224] + [prefix + x for x in EDGES] if 0 <= x]
        at = torch.zeros(q_len, heads, dtype=torch.long)
        for i in range(q_len):
            last = prefix + n - q_len + i
            own = [min(x, last) for x in edges] + [last, last, max(0, last - 1)] + [int(x) for x in torch.randint(0, last + 1, (8,), generator=g)]
            at[i] = torch.tensor([own[(7 * b + 3 * i + h) % len(own)] for h in range(heads)])
        for h in range(heads):
            q[b, :, h] = k[at[:, h], h // group]
            want[b, :, h] = v[at[:, h], h // group]
            scale = max(scale, scale_that_finds(q[b, :, h], k[:, h // group], at[:, h]))
    assert scale * dim * math.log2(math.e) < 1024
    kw = dict(prefix=pre.to(DEV), prefix_len=prefix) if prefix else {}
    # behind the end: what the last head's rows ask for, three times as loud
    for b, n in enumerate(lens):
        if n < width_keys:
            kc[table[b, n // page], :, n % page] = 3 * q[b, -1].view(kv, group, dim)[:, -1]
            vc[table[b, n // page], :, n % page] = 77.0
    got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), table.to(DEV), ints(lens), scale=scale, **kw)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dim,page,n,prefix,heads,q_len", [(64, 16, 40000, 0, 4, 1), (128, 64, 9100, 0, 4, 2), (128, 64, 500, 0, 8, 1), (64, 64, 77, 17000, 4, 1),
                                                           (128, 16, 130, 6000, 80, 1)])
def test_paged_counts_every_key(dim, page, n, prefix, heads, q_len):
    """As for prompts: equal weights over values that mark ranges of 64 keys, of the prefix and of the own keys."""
    kv = 2
    g = gen(n + prefix)
    used, shared = -(-n // page), -(-prefix // page)
    lens = [n, 0 if prefix else 70, max(q_len, n // 3)]
    table, kc, vc = paged_setup(g, [used] * 3 + [shared], max(used, shared), 0, kv, page, dim)
    pre, table = table[-1, :shared], table[:-1, :used].contiguous()
    q = torch.zeros(3, q_len, heads, dim, dtype=BF16, device=DEV)
    kd = kc.to(DEV)
    kw = dict(prefix=pre.to(DEV), prefix_len=prefix) if prefix else {}
    at = torch.arange(used * page)
    for first in range(0, -(-(n + prefix) // 64), dim * kv):
        for h in range(kv):
            v, _ = fractions(prefix + used * page, dim, first + dim * h)
            for b in range(3):
                vc[table[b].long()[at // page], h, at % page] = v[prefix:]
            if prefix:
                ap = torch.arange(prefix)
                vc[pre.long()[ap // page], h, ap % page] = v[:prefix]
        got = dsk_moe.paged_attention(q, kd, vc.to(DEV), table.to(DEV), ints(lens), **kw).cpu().double()
        for b in range(3):
            for i in range(q_len):
                m = prefix + max(0, lens[b] - q_len + i + 1)
                for h in range(heads):
                    lo = 64.0 * (first + dim * (h * kv // heads) + torch.arange(dim).double())
                    want = (m - lo).clamp(0.0, 64.0) / m
                    assert ((got[b, i, h] - want).abs() <= want * (2.0 ** -8 + 2.0 ** -12)).all(), (first, b, i, h)
