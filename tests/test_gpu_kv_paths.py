"""GPU parity of the cache in 8 bits and the keys' weights where only certain sizes and values lead: sums of a prefix
whose weights all round alike; parts of a prefix of many tiles; shares of so many steps that the pages held at once change
under way; tables on both sides of the width that one workgroup takes; an append on its own inputs."""

from __future__ import annotations

import math

import pytest
import torch

import dsk_moe
from oracle import attention as O
from test_gpu_attention import assert_within, gen, ints, normal
from test_gpu_kv_extra import BF16, DEV, I32, U8, code_cache, dev8, paged8_setup, run_paged8, weights_want

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ weights behind a prefix
@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv,q_len", [(2, 1, 1), (8, 2, 4), (8, 1, 2), (8, 1, 8)])
@pytest.mark.parametrize("prefix", [640, 1400])
def test_key_weights_behind_a_prefix_whose_weights_round_alike(codes, dim, heads, kv, q_len, prefix):
    """One key of every 64 has the largest score; the weights of all others are 0.5 (1 + 0.9 * 2^-8) of its own, which bf16
    rounds down by that 0.9 * 2^-8.  The sum that divides the own keys' weights is of the weights themselves: with |q||k| = 1
    the bound on a float32 score leaves a tenth of such a share."""
    print(f"weights of alike codes={codes} {dim} {heads},{kv} q {q_len} prefix {prefix}", flush=True)
    g = gen(dim + heads + prefix)
    lens = [40, 100, 17, 0]
    lens = [n if n == 0 else max(n, q_len) for n in lens]
    pre, table, kc, ks, vc, vs = paged8_setup(g, lens, kv, 64, dim, 1, prefix)
    kc[:], ks[:] = 0, 127
    at = torch.arange(0, prefix, 64)
    kc[pre.long()[at // 64], :, at % 64, 0] = 0x38               # the code of 1
    q = torch.zeros(len(lens), q_len, heads, dim, dtype=BF16)
    q[..., 0] = 1.0
    scale = -math.log(0.5 * (1 + 0.9 * 2.0 ** -8))               # exp(0 - scale)
    k64, v64 = O.values(kc, ks), O.values(vc, vs)
    w = torch.zeros(kc.shape[:3])
    wd = w.to(DEV)
    more = dict(prefix=pre.to(DEV), prefix_len=prefix, scale=scale)
    if codes:
        got = run_paged8(q, table, lens, kc, ks, vc, vs, key_weights=wd, **more)
    else:
        v64 = v64.to(BF16).double()
        got = dsk_moe.paged_attention(q.to(DEV), k64.to(BF16).to(DEV), v64.to(BF16).to(DEV), table.to(DEV), ints(lens), key_weights=wd, **more)
    want, tol = O.paged(q, k64, v64, table, lens, pre, prefix, scale=scale)
    assert_within(got, want, tol)
    want, tol = weights_want(w, q, k64, table, lens, 64, scale, pre, prefix)
    own = want > 0
    assert own.any() and float((tol[own] / want[own]).max()) < 0.2 * 0.9 * 2.0 ** -8
    assert_within(wd, want, tol + 1e-38, "weights")


# ------------------------------------------------------------------ a prefix in few parts
@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tiles,last", [(2, 36), (3, 64), (4, 1), (17, 46), (67, 6)])
def test_paged_codes_prefix_in_one_piece(dim, tiles, last, weigh):
    """So many rows (264 tiles of 128) that the prefix is not split: its tiles of 64 keys come one after the other through two
    buffers, and 67 are more than the 64 whose places a wave holds at once."""
    heads, kv, page, batch, q_len, prefix = 64, 8, 64, 130, 4, 64 * (tiles - 1) + last
    print(f"prefix in one piece {dim} {prefix} weigh={weigh}", flush=True)
    g = gen(dim + tiles)
    lens = [0] * batch
    lens[7], lens[64] = 9, 70
    pre, table, kc, ks, vc, vs = paged8_setup(g, lens, kv, page, dim, 1, prefix)
    q = normal(g, batch, q_len, heads, dim)
    w = torch.rand(kc.shape[:3], generator=g)
    wd = w.to(DEV)
    got = run_paged8(q, table, lens, kc, ks, vc, vs, prefix=pre, prefix_len=prefix, **(dict(key_weights=wd) if weigh else {}))
    rows = [0, 7, 31, 64, 129]
    k64, v64 = O.values(kc, ks), O.values(vc, vs)
    for b in rows:
        n = lens[b]
        k, v = (torch.cat([O.rows_of(x, pre, prefix), O.rows_of(x, table[b], n)]) for x in (k64, v64))
        last_key = prefix + torch.clamp(torch.arange(q_len) + n - q_len, min=-1)
        want, tol = O.attention_of_many(q[b], k, v, last_key, dim ** -0.5)
        assert_within(got[b], want, tol, f"sequence {b}")
    if weigh:
        want, tol = weights_want(w, q, k64, table, lens, page, dim ** -0.5, pre, prefix)
        assert_within(wd, want, tol + 1e-38, "weights")


# ------------------------------------------------------------------ long shares
@pytest.mark.parametrize("dim,heads,kv,q_len,lens", [(128, 128, 8, 4, [75000]), (64, 128, 8, 4, [300, 140000]), (64, 256, 16, 1, [140000])])
def test_paged_codes_of_more_steps_than_pages_held(dim, heads, kv, q_len, lens):
    """A share of 37, 69 or 34 steps of 128 keys; a wave holds the page ids and scales of 32.  Every row wants one key of its own,
    anywhere, so its output is that key's value and tells which scale it was read with (512 or 256 rows, of which one in 37, 69 or 34 meets
    any one step); then an even call's weights tell of every key."""
    print(f"long shares {dim} {heads},{kv} q {q_len} {lens}", flush=True)
    g = gen(dim + heads + q_len)
    _, table, kc, ks, vc, vs = paged8_setup(g, lens, kv, 64, dim)
    ks = torch.randint(126, 128, ks.shape, generator=g).to(U8)   # keys of like size, values of very different ones
    group, batch = heads // kv, len(lens)
    q = torch.empty(batch, q_len, heads, dim)
    target = torch.empty(batch, q_len, heads, dtype=torch.long)
    for b, n in enumerate(lens):
        target[b] = torch.randint(0, n - q_len, (q_len, heads), generator=g)
        for h in range(heads):
            one = slice(h // group, h // group + 1)
            at = target[b, :, h]
            p, r = table[b].long()[at // 64], at % 64
            values = O._CODES[kc[p, one.start, r].long()] * 2.0 ** (ks[p, one.start, r // 16].double()[:, None] - 127)
            q[b, :, h] = (values / values.norm(dim=-1, keepdim=True)).float()
    q = q.to(BF16)
    got = run_paged8(q, table, lens, kc, ks, vc, vs, scale=0.25)
    w = torch.zeros(kc.shape[:3], device=DEV)
    flat = normal(g, batch, q_len, heads, dim)
    run_paged8(flat, table, lens, kc, ks, vc, vs, key_weights=w, scale=0.002)
    wanted = 0
    for h in range(kv):
        k64, v64 = (O.values(c[:, h:h + 1], s[:, h:h + 1]) for c, s in ((kc, ks), (vc, vs)))
        mine = slice(h * group, (h + 1) * group)
        for b, n in enumerate(lens):
            k, v = (O.rows_of(x, table[b], n) for x in (k64, v64))
            last = torch.arange(q_len) + n - q_len
            want, tol = O.attention_of_many(q[b, :, mine], k, v, last, 0.25)
            assert_within(got[b, :, mine], want, tol, f"head {h} of sequence {b}")
            near = (want - v[target[b, :, mine], 0]).norm(dim=-1) < 0.1 * want.norm(dim=-1)
            wanted += int(near.sum())
            if h % 3:
                continue
            want, tol = O.key_weights(flat[b, :, mine], k, last, 0.002)
            at = torch.arange(n)
            have = w.cpu()[table[b].long()[at // 64], h, at % 64]
            assert_within(have, want[:, 0], tol[:, 0] + 1e-38, "weights")
    assert wanted > batch * q_len * heads // 2                   # most rows are of one key indeed


# ------------------------------------------------------------------ one workgroup an item, or shares
@pytest.mark.parametrize("dim,heads,kv,q_len", [(128, 8, 2, 1), (64, 6, 2, 3), (128, 16, 1, 4)])
@pytest.mark.parametrize("places", [640, 1008, 1024, 1040])
def test_paged_codes_on_both_sides_of_a_table_s_width(dim, heads, kv, q_len, places):
    """Up to 1024 places a workgroup takes an item alone, four steps of 256 keys; beyond, shares of it are joined."""
    g = gen(dim + heads + places)
    lens = [places, 600, 529, 1, 0, places - 9]
    lens = [n if n == 0 else max(n, q_len) for n in lens]
    _, table, kc, ks, vc, vs = paged8_setup(g, lens, kv, 16, dim, 0)
    assert table.shape[1] * 16 == places
    q = normal(g, len(lens), q_len, heads, dim) * 2
    w = torch.rand(kc.shape[:3], generator=g)
    wd = w.to(DEV)
    k64, v64 = O.values(kc, ks), O.values(vc, vs)
    want, tol = O.paged(q, k64, v64, table, lens)
    assert_within(run_paged8(q, table, lens, kc, ks, vc, vs), want, tol)
    assert_within(run_paged8(q, table, lens, kc, ks, vc, vs, key_weights=wd), want, tol)
    want, tol = weights_want(w, q, k64, table, lens, 16, dim ** -0.5)
    assert_within(wd, want, tol + 1e-38, "weights")


# ------------------------------------------------------------------ an append on its own inputs
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,start,dim,kv", [(1, 5, 128, 8), (23, 9, 64, 3), (150, 3, 128, 5), (2100, 0, 64, 2)])
def test_append_codes_in_place(tokens, start, dim, kv, interleaved):
    """q_out that is q and k_out that is k, with a cache in 8 bits; keys that are the values too."""
    g = gen(tokens + dim)
    heads, page = 2 * kv, 32
    pages = (start + tokens) // page + 2
    qkv = normal(g, tokens, (heads + kv) * dim).to(DEV)
    freq = dsk_moe.rope_frequencies(dim)[0]
    rows = torch.arange(start, start + tokens, dtype=I32, device=DEV)
    table = torch.randperm(pages, generator=g).to(I32)[None].to(DEV)
    kc, ks = code_cache(g, pages, kv, page, dim)
    outs = []
    for in_place in (False, True):
        q, k = (p.unflatten(1, (-1, dim)) for p in qkv.clone().split([heads * dim, kv * dim], 1))
        v = k.clone() if in_place else k                         # (in place the keys change: the values may not be they)
        (kd, vd), ksd, vsd = dev8(kc.clone(), kc.clone()), ks.to(DEV), ks.to(DEV)
        ko = k if in_place else torch.empty((tokens, kv, dim), dtype=BF16, device=DEV)
        got = dsk_moe.kv_append(q, k, v, rows, torch.zeros_like(rows), table, kd, vd, freq, k_scale=ksd, v_scale=vsd,
                                interleaved=interleaved, q_out=q if in_place else None, k_out=ko)
        outs.append((got.clone(), ko.clone(), kd.view(U8), vd.view(U8), ksd, vsd))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and a.any()
