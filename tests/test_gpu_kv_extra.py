"""GPU parity of the cache in 8 bits, the keys' weights, eviction and several rotary axes with the restatement in
64 bits (``oracle/attention.py``), value by value within the roundings that it derives; codes, scales and what
eviction moves are equal.  Then runs of them together, as a server would make them, eager and captured."""

from __future__ import annotations

import math

import pytest
import torch

import dsk_moe
from dsk_moe import _lib
from oracle import attention as O
from test_gpu_attention import assert_within, cumulative, gen, ints, make_decoder, normal, paged_setup

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32, F64, I32, F8, U8 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.float8_e4m3fn, torch.uint8
NAN, INF = math.nan, math.inf


def code_cache(g, pages, kv, page, dim):
    """(codes uint8, scale bytes) of random rows whose blocks differ in size, on the CPU."""
    codes = torch.randint(0, 256, (pages, kv, page, dim), generator=g, dtype=U8)
    codes[(codes & 127) == 127] = 0
    # the exponents of a normal sample rather than of random bytes
    x = torch.randn((pages, kv, page, dim), generator=g) * 60
    byte = torch.randint(118, 126, (pages, kv, page // 16), generator=g).to(U8)
    return x.to(F8).view(U8), byte


def same_codes(a, b):
    """Equal codes; a NaN has two (its sign says nothing)."""
    a, b = (torch.where((x & 127) == 127, torch.full_like(x, 127), x) for x in (a, b))
    return torch.equal(a, b)


def dev8(*codes):
    return tuple(c.to(DEV).view(F8) for c in codes)


# ------------------------------------------------------------------ several axes
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,rot,first,inter,sections,kw", [
    (128, 128, 0, False, [16, 24, 24], {}), (128, 128, 0, True, [20, 20, 24], dict(in_turn=True)), (64, 64, 0, False, [16, 16], dict(each=True)),
    (64, 32, 16, True, [5, 5, 3, 3], dict(in_turn=True, each=True)), (128, 64, 8, False, [32], {}), (64, 16, 48, False, [1] * 8, {})])
@pytest.mark.parametrize("tokens,heads,kv", [(1, 5, 1), (37, 3, 3), (2050, 9, 2)])
def test_axes(dtype, dim, rot, first, inter, sections, kw, tokens, heads, kv):
    print(f"axes {dtype} {dim} {rot}+{first} {sections} {kw} {tokens}x{heads},{kv}", flush=True)
    g = gen(dim + rot + tokens)
    q, k = normal(g, tokens, heads, dim, dtype=dtype), normal(g, tokens, kv, dim, dtype=dtype) * 2
    n = len(sections)
    pos = torch.randint(0, 70000, (n, tokens), generator=g, dtype=I32)
    gq, gk = torch.rand(dim, generator=g) + 0.5, torch.randn(dim, generator=g)
    freq, axis = dsk_moe.rope_axes(sections, device="cpu", **kw)
    more = dict(interleaved=inter, rot_first=first, mscale=0.9)
    # rows of the positions further apart than tokens
    wide = torch.full((n, tokens + 3), -5, dtype=I32)
    wide[:, :tokens] = pos
    got_q, got_k = dsk_moe.qk_norm_rope(q.to(DEV), k.to(DEV), wide.to(DEV)[:, :tokens], freq.to(DEV), axis=axis.to(DEV), q_gamma=gq.to(DEV),
                                        k_gamma=gk.to(DEV), **more)
    at = pos[axis.long()].t()
    assert_within(got_q, *O.norm_rope(q, at, freq, gamma=gq, **more), "q")
    assert_within(got_k, *O.norm_rope(k, at, freq, gamma=gk, **more), "k")


def test_equal_axes_are_one_axis():
    g = gen(2)
    q, k = normal(g, 50, 4, 128).to(DEV), normal(g, 50, 2, 128).to(DEV)
    pos = torch.randint(0, 1 << 30, (50,), generator=g, dtype=I32).to(DEV)
    freq, axis = dsk_moe.rope_axes([16, 24, 24], base=1e6)
    one = dsk_moe.qk_norm_rope(q, k, pos, freq)
    for same in (pos.expand(3, 50).contiguous(), pos.expand(3, 50)):
        for got, want in zip(dsk_moe.qk_norm_rope(q, k, same, freq, axis=axis), one):
            assert torch.equal(got, want)
    for got, want in zip(dsk_moe.qk_norm_rope(q, k, pos[None], freq, axis=torch.zeros_like(axis)), one):
        assert torch.equal(got, want)


def test_axes_that_are_none_and_tokens_left_out():
    """A pair of no axis does not turn; a token that is negative on any axis is left out."""
    g = gen(3)
    k = normal(g, 5, 2, 64)
    pos = torch.tensor([[3, -1, 5, 0, 9], [4, 2, -7, 0, 9]], dtype=I32)
    freq, axis = dsk_moe.rope_axes([16, 16], device="cpu")
    bad = axis.clone()
    bad[[0, 20]] = torch.tensor([2, -1], dtype=I32)
    ko = torch.full((5, 2, 64), 7.0, dtype=BF16, device=DEV)
    dsk_moe.qk_norm_rope(None, k.to(DEV), pos.to(DEV), freq.to(DEV), axis=bad.to(DEV), k_out=ko)
    at = pos[axis.long()].t().clone()
    at[:, [0, 20]] = 0
    want, tol = O.norm_rope(k, at, freq)
    live = torch.tensor([True, False, False, True, True])
    assert_within(ko.cpu()[live], want[live], tol[live])
    assert (ko.cpu()[~live] == 7.0).all()


# ------------------------------------------------------------------ rows, weights of a bf16 cache
@pytest.mark.parametrize("tokens", [3, 40, 2100])
def test_append_rows_and_new_weights(tokens):
    """Rows given apart from positions, as for several axes; kept keys weigh nothing yet, other weights stay."""
    g = gen(tokens)
    kv, dim, page, pages = 3, 64, 32, 80
    rows = torch.randperm(tokens + 5, generator=g)[:tokens].to(I32)
    rows[0] = -1
    table = torch.randperm(pages, generator=g).to(I32)[None]
    k, v, q = normal(g, tokens, kv, dim), normal(g, tokens, kv, dim), normal(g, tokens, 6, dim)
    pos = torch.randint(0, 100, (2, tokens), generator=g, dtype=I32)
    freq, axis = dsk_moe.rope_axes([8, 8], device="cpu")
    kc, vc, w = normal(g, pages, kv, page, dim), normal(g, pages, kv, page, dim), torch.rand((pages, kv, page), generator=g)
    kd, vd, wd = kc.to(DEV), vc.to(DEV), w.to(DEV)
    ko = torch.empty((tokens, kv, dim), dtype=BF16, device=DEV)
    got = dsk_moe.kv_append(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), torch.zeros(tokens, dtype=I32, device=DEV), table.to(DEV), kd, vd,
                            freq.to(DEV), axis=axis.to(DEV), rows=rows.to(DEV), key_weights=wd, k_out=ko)
    at = pos[axis.long()].t()
    assert_within(got, *O.norm_rope(q, at, freq), "q")
    assert_within(ko, *O.norm_rope(k, at, freq), "k")
    r = rows[1:].long()
    p, r = table[0].long()[r // page], r % page
    kc[p, :, r], vc[p, :, r], w[p, :, r] = ko.cpu()[1:], v[1:], 0.0
    assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), vc) and torch.equal(wd.cpu(), w)


# ------------------------------------------------------------------ append in 8 bits
def slots_of(table, seq, rows, page, pages):
    out = []
    for s, r in zip(seq.tolist(), rows.tolist()):
        ok = 0 <= s < table.shape[0] and r >= 0 and r // page < table.shape[1] and 0 <= int(table[s, r // page]) < pages
        out.append((int(table[s, r // page]), r % page) if ok else None)
    return out


def check_append(g, k, v, table, seq, rows, kc, ks, vc, vs, pos=None, freq=None, weights=False, heads=2, fresh_ok=True, **kw):
    """One call against the restatement: values exactly, keys too where nothing turns."""
    pages, kv, page, dim = kc.shape
    tokens = k.shape[0]
    slots = slots_of(table, seq, rows, page, pages)
    kd, vd = dev8(kc.clone(), vc.clone())
    ksd, vsd = ks.to(DEV), vs.to(DEV)
    w = torch.rand((pages, kv, page), generator=g)
    wd = w.to(DEV)
    q = normal(g, tokens, heads, dim).to(k.dtype)
    ko = torch.empty((tokens, kv, dim), dtype=BF16, device=DEV)
    pos = rows if pos is None else pos
    got = dsk_moe.kv_append(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), seq.to(DEV), table.to(DEV), kd, vd,
                            freq.to(DEV) if freq is not None else None, rows=rows.to(DEV), k_scale=ksd, v_scale=vsd,
                            key_weights=wd if weights else None, k_out=ko, **kw)
    norm = kw.get("norm", True)
    want_q, tol = O.norm_rope(q, pos, freq, norm=norm)
    assert_within(got, want_q, tol, "q")
    want_k, k_tol = O.norm_rope(k, pos, freq, norm=norm)
    O.append_codes(v.double(), vc, vs, slots)
    assert same_codes(vd.cpu().view(U8), vc) and torch.equal(vsd.cpu(), vs)
    if not norm and freq is None:
        O.append_codes(k.double(), kc, ks, slots)
        assert same_codes(kd.cpu().view(U8), kc) and torch.equal(ksd.cpu(), ks)
    else:
        # a scale may be the next one where the largest magnitude is float32's roundings from its border
        before = kc.clone()
        O.append_codes(want_k, kc, ks, slots)
        assert torch.equal(ksd.cpu(), ks)
        mine = torch.zeros((pages, page), dtype=torch.bool)
        for at in slots:
            if at is not None:
                mine[at] = True
        have = kd.cpu().view(U8)
        others = ~mine[:, None, :, None].expand_as(kc)
        assert torch.equal(have[others], kc[others])
        assert before.shape == have.shape
        real, size = O.values(have, ks), 2.0 ** (ks.double().repeat_interleave(16, -1)[..., None] - 127)
        for t, at in enumerate(slots):
            if at is not None:
                y = want_k[t]
                # half a step of e4m3 (2^-4, or 2^-10 of the scale below its normal codes) and what float32 does before it
                arithmetic = k_tol[t] - O.BF16_HALF_STEP * y.abs()
                tol = torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * size[at[0], :, at[1]]) + arithmetic * (1 + 2.0 ** -4)
                assert ((real[at[0], :, at[1]] - y).abs() <= tol).all()
    for t, at in enumerate(slots):
        if at is not None and weights:
            w[at[0], :, at[1]] = 0.0
    assert torch.equal(wd.cpu(), w)
    return ko


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,page,kv", [(128, 64, 3), (64, 16, 2), (128, 16, 1), (64, 256, 5), (128, 32, 8)])
@pytest.mark.parametrize("turned", [False, True])
def test_append_codes(dtype, dim, page, kv, turned):
    """Sequences from one token to a few blocks, begun anywhere in a block."""
    print(f"append codes {dtype} {dim} {page} {kv} {turned}", flush=True)
    g = gen(dim + page + kv)
    lens, starts = [70, 1, 33, 2, 16, 15, 5, 1, 1, 40], [0, 500, 15, 255, 16, 3, 12, 31, 32, 7]
    used = [(a + n - 1) // page + 1 for a, n in zip(starts, lens)]
    table, _, _ = paged_setup(g, used, max(used) + 1, 2, 1, 16, 16)
    pages = sum(used) + 2
    kc, ks = code_cache(g, pages, kv, page, dim)
    vc, vs = code_cache(g, pages, kv, page, dim)
    rows = torch.tensor([a + i for a, n in zip(starts, lens) for i in range(n)], dtype=I32)
    seq = torch.tensor([b for b, n in enumerate(lens) for _ in range(n)], dtype=I32)
    t = len(rows)
    # sizes from below the blocks' to above them
    k, v = ((torch.randn((t, kv, dim), generator=g) * torch.exp2(torch.randint(-4, 5, (t, 1, 1), generator=g).float())).to(dtype) for _ in range(2))
    freq = dsk_moe.rope_frequencies(dim // 2, device="cpu")[0] if turned else None
    pos = torch.randint(0, 3000, (t,), generator=g, dtype=I32)
    check_append(g, k, v, table, seq, rows, kc, ks, vc, vs, pos, freq, weights=True, norm=turned)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,rot,first,inter", [(128, 128, 0, True), (128, 64, 32, False), (64, 32, 16, True), (64, 64, 0, False)])
def test_append_codes_turned(dtype, dim, rot, first, inter):
    """Both kinds of pairs, a part of the head turned, gammas, three axes: the values within their one rounding, as k_out's."""
    g = gen(dim + rot + first)
    kv, page, t = 3, 32, 90
    table = torch.randperm(8, generator=g)[:6].view(2, 3).to(I32)
    rows = torch.cat([torch.arange(5, 60), torch.arange(35)]).to(I32)
    seq = torch.tensor([0] * 55 + [1] * 35, dtype=I32)
    q, k, v = (normal(g, t, n, dim, dtype=dtype) for n in (5, kv, kv))
    pos = torch.randint(0, 9000, (3, t), generator=g, dtype=I32)
    freq, axis = dsk_moe.rope_axes([rot // 2 - 2 * (rot // 8), rot // 8, rot // 8], in_turn=inter, device="cpu")
    gq, gk = torch.rand(dim, generator=g) + 0.5, torch.randn(dim, generator=g)
    more = dict(interleaved=inter, rot_first=first, mscale=1.1)
    kd, vd = dev8(torch.zeros(8, kv, page, dim, dtype=U8), torch.zeros(8, kv, page, dim, dtype=U8))
    ks, vs = (torch.zeros(8, kv, page // 16, dtype=U8, device=DEV) for _ in range(2))
    ko = torch.empty((t, kv, dim), dtype=BF16, device=DEV)
    got = dsk_moe.kv_append(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), seq.to(DEV), table.to(DEV), kd, vd, freq.to(DEV), axis=axis.to(DEV),
                            rows=rows.to(DEV), k_scale=ks, v_scale=vs, q_gamma=gq.to(DEV), k_gamma=gk.to(DEV), k_out=ko, **more)
    at = pos[axis.long()].t()
    assert_within(got, *O.norm_rope(q, at, freq, gamma=gq, **more), "q")
    want, tol = O.norm_rope(k, at, freq, gamma=gk, **more)
    assert_within(ko, want, tol, "k")
    real, byte = O.values(kd.cpu().view(U8), ks.cpu()), ks.cpu()
    p, r = table[seq.long(), rows.long() // page].long(), rows.long() % page
    size = 2.0 ** (byte[p, :, r // 16].double()[..., None] - 127)
    arithmetic = tol - O.BF16_HALF_STEP * want.abs()
    # (each block comes in one call: one rounding, of a scale that is at most twice the least)
    bound = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * size) + arithmetic * (1 + 2.0 ** -4)
    assert ((real[p, :, r] - want).abs() <= bound).all()
    # both sequences' blocks: the least scale for their largest, up to float32's roundings at a border
    for b, lo, hi in ((0, 5, 60), (1, 0, 35)):
        for block in range(lo // 16, -(-hi // 16)):
            mine = (seq == b) & (rows // 16 == block)
            if bool((rows[mine] % 16 == 0).any()):
                top = want[mine].abs().amax((0, 2))
                have = byte[int(table[b, block * 16 // page]), :, block * 16 % page // 16]
                for h in range(kv):
                    assert int(have[h]) in {O.scale_byte(float(top[h]) * f) for f in (1 - 1e-6, 1.0, 1 + 1e-6)}


@pytest.mark.parametrize("tokens,batch", [(1, 1), (64, 64), (130, 65), (2060, 2)])
def test_append_codes_of_few_and_many(tokens, batch):
    """Decode steps, verify steps and prompts: as many workgroups for a token as for 16."""
    g = gen(tokens)
    kv, dim, page, each = 4, 128, 64, tokens // batch
    starts = [int(x) for x in torch.randint(0, 60, (batch,), generator=g)]
    used = [(a + each - 1) // page + 1 for a in starts]
    table, _, _ = paged_setup(g, used, max(used), 1, 1, 16, 16)
    kc, ks = code_cache(g, sum(used) + 1, kv, page, dim)
    vc, vs = code_cache(g, sum(used) + 1, kv, page, dim)
    rows = torch.tensor([a + i for a in starts for i in range(each)], dtype=I32)
    seq = torch.arange(batch, dtype=I32).repeat_interleave(each)
    k, v = normal(g, tokens, kv, dim) * 9, normal(g, tokens, kv, dim)
    check_append(g, k, v, table, seq, rows, kc, ks, vc, vs, norm=False, heads=33)


@pytest.mark.parametrize("dim", [64, 128])
def test_append_codes_in_any_order_of_a_block(dim):
    """A block's tokens next to each other, in any order; the last block's rows backwards."""
    g = gen(11)
    table = torch.tensor([[3, 1, 0]], dtype=I32)
    kc, ks = code_cache(g, 4, 2, 32, dim)
    vc, vs = code_cache(g, 4, 2, 32, dim)
    rows = torch.tensor([20, 19, 31, 40, 36, 47, 32, 63, 62, 61, 60, 59, 58, 57, 56, 55, 54, 53, 52, 51, 50, 49, 48], dtype=I32)
    k, v = normal(g, 23, 2, dim) * 5, normal(g, 23, 2, dim) * 5
    check_append(g, k, v, table, torch.zeros(23, dtype=I32), rows, kc, ks, vc, vs, norm=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_append_codes_of_special_values(dtype):
    """NaN and infinities, zeros, the largest and the least numbers, and rows of one magnitude at a border of a scale."""
    g = gen(12)
    kc, ks = code_cache(g, 3, 1, 64, 64)
    vc, vs = code_cache(g, 3, 1, 64, 64)
    k = torch.randn((64, 1, 64), generator=g)
    v = torch.zeros(64, 1, 64)
    k[1, 0, 3], k[17, 0, 5], k[18, 0, 6] = NAN, INF, -INF
    k[32:48] = 0.0
    k[33, 0, 0] = -0.0
    k[48:, :, :] *= 1e-38
    k[50, 0, 7] = INF
    v[:16, :, :] = 448.0
    v[16:32] = 3.0e38
    v[17, 0, 0] = -3.3e38
    v[32:48] = 1.75 * 2.0 ** -9
    v[40, 0, 9] = 1.765625 * 2.0 ** -9
    v[48:] = torch.tensor(2.0) ** -120
    k, v = k.to(dtype), v.to(dtype)
    rows = torch.arange(64, dtype=I32)
    check_append(g, k, v, torch.tensor([[2]], dtype=I32), torch.zeros(64, dtype=I32), rows, kc, ks, vc, vs, norm=False)


def test_append_codes_leaves_out_what_has_no_place():
    g = gen(13)
    kc, ks = code_cache(g, 4, 2, 16, 64)
    vc, vs = code_cache(g, 4, 2, 16, 64)
    table = torch.tensor([[0, 4, -1], [1, 2, 1 << 30]], dtype=I32)
    rows = torch.tensor([-1, 16, 32, 48, 32, 3, 3, 17, 18, -9], dtype=I32)
    seq = torch.tensor([0, 0, 0, 0, 1, 2, -1, 1, 1, 1], dtype=I32)
    k, v = normal(g, 10, 2, 64), normal(g, 10, 2, 64)
    pos = torch.arange(10, dtype=I32)
    ko = check_append(g, k, v, table, seq, rows, kc, ks, vc, vs, pos, weights=True, norm=False)
    assert torch.equal(ko.cpu(), k)
    # a token of padding writes nothing at all
    kd, vd = dev8(kc, vc)
    out, qo = torch.full((1, 2, 64), 5.0, dtype=BF16, device=DEV), torch.full((1, 2, 64), 6.0, dtype=BF16, device=DEV)
    dsk_moe.kv_append(k[:1].to(DEV), k[:1].to(DEV), v[:1].to(DEV), ints([-1]), ints([1]), table.to(DEV), kd, vd, rows=ints([3]),
                      k_scale=ks.to(DEV), v_scale=vs.to(DEV), q_out=qo, k_out=out)
    assert (out == 5.0).all() and (qo == 6.0).all() and torch.equal(kd.cpu().view(U8), kc) and torch.equal(vd.cpu().view(U8), vc)


def test_append_codes_one_by_one_as_at_once_or_nearly():
    """Sixteen tokens of a block one by one: rounded again as the scale grows, by half a least step of the last scale each time at
    most beside the one rounding; whole blocks at once are what a prompt keeps."""
    g = gen(14)
    x = torch.randn((16, 1, 128), generator=g) * torch.exp2(torch.arange(16).float()[:, None, None] / 2)
    kd, vd = dev8(torch.zeros(1, 1, 16, 128, dtype=U8), torch.zeros(1, 1, 16, 128, dtype=U8))
    ks, vs = (torch.zeros(1, 1, 1, dtype=U8, device=DEV) for _ in range(2))
    for t in range(16):
        dsk_moe.kv_append(None, x[t:t + 1].to(DEV), x[t:t + 1].to(DEV), ints([t]), ints([0]), ints([[0]]), kd, vd, norm=False, k_scale=ks, v_scale=vs)
    kc, byte = torch.zeros(1, 1, 16, 128, dtype=U8), torch.zeros(1, 1, 1, dtype=U8)
    for t in range(16):
        O.append_codes(x[t:t + 1].double(), kc, byte, [(0, t)])
    assert torch.equal(kd.cpu().view(U8), kc) and torch.equal(ks.cpu(), byte) and torch.equal(vd.cpu().view(U8), kc)
    size = 2.0 ** (int(byte) - 127)
    err = (O.values(kc, byte)[0, 0] - x[:, 0].double()).abs()
    assert (err <= torch.maximum(2.0 ** -4 * x[:, 0].double().abs(), torch.tensor(2.0 ** -10 * size)) + 2.0 ** -10 * size).all()


def test_append_codes_views_and_no_queries():
    """Views of one projection; a prefix before the rows; no queries."""
    g = gen(15)
    qkv = normal(g, 20, (2 + 2 + 2) * 64)
    _, k, v = (p.unflatten(1, (-1, 64)) for p in qkv.split([128, 128, 128], 1))
    qd, kd_in, vd_in = (p.unflatten(1, (-1, 64)) for p in qkv.to(DEV).split([128, 128, 128], 1))
    outs = []
    for kk, vv, q in ((kd_in, vd_in, None), (k.contiguous().to(DEV), v.contiguous().to(DEV), qd)):
        kd, vd = dev8(torch.zeros(2, 2, 16, 64, dtype=U8), torch.zeros(2, 2, 16, 64, dtype=U8))
        ks, vs = (torch.zeros(2, 2, 1, dtype=U8, device=DEV) for _ in range(2))
        got = dsk_moe.kv_append(q, kk, vv, torch.arange(100, 120, dtype=I32, device=DEV), torch.zeros(20, dtype=I32, device=DEV), ints([[1, 0]]),
                                kd, vd, prefix_len=100, k_scale=ks, v_scale=vs)
        assert (got is None) == (q is None)
        outs.append((kd.view(U8), vd.view(U8), ks, vs))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and a.any()


# ------------------------------------------------------------------ attention over the cache in 8 bits
def paged8_setup(g, lens, kv, page, dim, spare=1, prefix=0):
    used = [-(-max(0, n) // page) for n in lens] + [-(-prefix // page)]
    table, _, _ = paged_setup(g, used, max(used) + spare, 2, 1, 16, 16)
    n = sum(used) + 2
    kc, ks = code_cache(g, n, kv, page, dim)
    vc, vs = code_cache(g, n, kv, page, dim)
    return table[-1, :used[-1]], table[:-1], kc, ks, vc, vs


def run_paged8(q, table, lens, kc, ks, vc, vs, **kw):
    kd, vd = dev8(kc, vc)
    more = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    return dsk_moe.paged_attention(q.to(DEV), kd, vd, table.to(DEV), ints(lens), k_scale=ks.to(DEV), v_scale=vs.to(DEV), **more)


@pytest.mark.parametrize("heads,kv,dim,page,q_len", [(8, 2, 128, 64, 1), (4, 4, 64, 16, 1), (8, 1, 64, 32, 3), (16, 1, 128, 16, 4),
                                                     (6, 2, 128, 256, 2), (32, 2, 128, 32, 2), (12, 1, 64, 128, 5)])
@pytest.mark.parametrize("prefix,spare", [(0, 1), (0, 130), (1, 1), (130, 1)])
def test_paged_codes(heads, kv, dim, page, q_len, prefix, spare):
    print(f"paged codes {heads},{kv},{dim} page {page} q {q_len} prefix {prefix} spare {spare}", flush=True)
    g = gen(heads + dim + page + q_len + prefix)
    lens = [1, 0, 16, 17, 63, 64, 65, 130, 255, 256, 257, 300, -1, 520]
    lens = [n if n <= 0 else max(n, q_len) for n in lens]
    pre, table, kc, ks, vc, vs = paged8_setup(g, lens, kv, page, dim, spare, prefix)
    q = normal(g, len(lens), q_len, heads, dim) * 2
    got = run_paged8(q, table, lens, kc, ks, vc, vs, **(dict(prefix=pre, prefix_len=prefix) if prefix else {}))
    live = [i for i, n in enumerate(lens) if n >= 0]
    want, tol = O.paged(q, O.values(kc, ks), O.values(vc, vs), table, lens, pre, prefix)
    assert_within(got[live], want[live], tol[live])
    assert not got[lens.index(-1)].any()


@pytest.mark.parametrize("batch,longest,heads,kv,dim", [(1, 9000, 8, 2, 128), (3, 4100, 4, 2, 64), (70, 600, 4, 1, 128), (1, 517, 32, 8, 128)])
def test_paged_codes_long_and_many(batch, longest, heads, kv, dim):
    g = gen(batch + longest)
    lens = [max(1, longest * (i + 1) // batch - 3 * (i % 2)) for i in range(batch)]
    _, table, kc, ks, vc, vs = paged8_setup(g, lens, kv, 64, dim)
    q = normal(g, batch, heads, dim)
    got = run_paged8(q, table, lens, kc, ks, vc, vs)
    want, tol = O.paged(q[:, None], O.values(kc, ks), O.values(vc, vs), table, lens)
    assert_within(got, want[:, 0], tol[:, 0])


@pytest.mark.parametrize("spare", [1, 200])
@pytest.mark.parametrize("dim,heads,q_len", [(64, 4, 3), (128, 2, 4), (128, 32, 2)])
def test_paged_codes_unseen_values_stay_unseen(dim, heads, q_len, spare):
    """NaN codes and scales that are none in keys that a row does not see, and behind the last key; rows that see them show it."""
    g = gen(31 + dim)
    lens = [40, 64, 100, 129, 1000]
    _, table, kc, ks, vc, vs = paged8_setup(g, lens, 1, 32, dim, spare)
    q = normal(g, 5, q_len, heads, dim)
    want, tol = O.paged(q, O.values(kc, ks), O.values(vc, vs), table, lens)
    for b, n in enumerate(lens):
        last = n - 1
        vc[table[b, last // 32], 0, last % 32, 7] = 0x7f         # seen by the last token alone
        kc[table[b, last // 32], 0, last % 32, 0] = 0xff
        for r in range(n, -(-n // 32) * 32):                     # rows that nobody sees
            kc[table[b, r // 32], 0, r % 32] = 0x7f
            vc[table[b, r // 32], 0, r % 32] = 0xff
            if r % 16 == 0:                                      # blocks that nobody sees
                ks[table[b, r // 32], 0, r % 32 // 16] = 255
                vs[table[b, r // 32], 0, r % 32 // 16] = 255
    got = run_paged8(q, table, lens, kc, ks, vc, vs)
    assert_within(got[:, :-1], want[:, :-1], tol[:, :-1])
    assert got[:, -1].isnan().all()


def test_paged_codes_seen_nan_shows_and_scales_that_are_none():
    """A NaN value is seen by every token behind it; a block whose scale is none (255) gives NaN to those that see it."""
    g = gen(32)
    _, table, kc, ks, vc, vs = paged8_setup(g, [200, 200], 1, 16, 64, 1)
    q = normal(g, 2, 2, 4, 64)
    want, tol = O.paged(q, O.values(kc, ks), O.values(vc, vs), table, [200, 200])
    vc[table[0, 2], 0, 5, 9] = 0x7f
    vs[table[1, 12], 0, 0] = 255                                 # keys 192 .. 199
    got = run_paged8(q, table, [200, 200], kc, ks, vc, vs).cpu()
    rest = [i for i in range(64) if i != 9]
    assert got[0, :, :, 9].isnan().all() and not torch.isfinite(got[1]).any()
    assert_within(got[0][..., rest], want[0][..., rest], tol[0][..., rest])


@pytest.mark.parametrize("prefix", [0, 40])
def test_paged_codes_bad_pages_and_lengths_show(prefix):
    g = gen(33)
    lens = [40, 40, 40, 1000]
    pre, table, kc, ks, vc, vs = paged8_setup(g, [40, 40, 40, 40], 2, 16, 64, 1, prefix)
    q = normal(g, 4, 1, 4, 64)
    more = dict(prefix=pre, prefix_len=prefix) if prefix else {}
    want, tol = O.paged(q, O.values(kc, ks), O.values(vc, vs), table, [40] * 4, pre, prefix)
    table = table.clone()
    table[1, 1] = kc.shape[0]
    table[2, 2] = -1
    got = run_paged8(q, table, lens, kc, ks, vc, vs, **more)
    assert_within(got[:1], want[:1], tol[:1])
    assert got[1:].isnan().all()
    if prefix:
        bad = pre.clone()
        bad[1] = 1 << 20
        assert run_paged8(q, table, lens, kc, ks, vc, vs, prefix=bad, prefix_len=prefix).isnan().all()


def test_paged_codes_long_prefix():
    g = gen(34)
    lens = [0, 5, 100, 33]
    pre, table, kc, ks, vc, vs = paged8_setup(g, lens, 2, 64, 128, 1, 5000)
    q = normal(g, 4, 1, 8, 128)
    got = run_paged8(q, table, lens, kc, ks, vc, vs, prefix=pre, prefix_len=5000)
    want, tol = O.paged(q, O.values(kc, ks), O.values(vc, vs), table, lens, pre, 5000)
    assert_within(got, want, tol)


def test_paged_codes_far_pages():
    """Offsets into the cache beyond 2^32 bytes."""
    g = gen(35)
    kd, vd = (torch.empty((34000, 16, 64, 128), dtype=U8, device=DEV).view(F8) for _ in range(2))   # 4.4 GB each
    ks, vs = (torch.empty((34000, 16, 4), dtype=U8, device=DEV) for _ in range(2))
    table = torch.tensor([[33999, 33990], [2, 33950]], dtype=I32)
    lens = [100, 70]
    kc, kb = code_cache(g, 4, 16, 64, 128)
    vc, vb = code_cache(g, 4, 16, 64, 128)
    ids = table.flatten().long().to(DEV)
    kd.view(U8)[ids], vd.view(U8)[ids], ks[ids], vs[ids] = kc.to(DEV), vc.to(DEV), kb.to(DEV), vb.to(DEV)
    q = normal(g, 2, 16, 128)
    got = dsk_moe.paged_attention(q.to(DEV), kd, vd, table.to(DEV), ints(lens), k_scale=ks, v_scale=vs)
    near = torch.arange(4, dtype=I32).view(2, 2)
    want, tol = O.paged(q[:, None], O.values(kc, kb), O.values(vc, vb), near, lens)
    assert_within(got, want[:, 0], tol[:, 0])
    # and an append there
    k = normal(g, 2, 16, 128)
    dsk_moe.kv_append(None, k.to(DEV), k.to(DEV), ints([100, 71]), ints([0, 1]), table.to(DEV), kd, vd, norm=False, k_scale=ks, v_scale=vs)
    O.append_codes(k.double(), kc, kb, [(1, 36), (3, 7)])
    assert torch.equal(kd.view(U8)[ids].cpu(), kc) and torch.equal(ks[ids].cpu(), kb)
    w = torch.rand((34000, 16, 64), device=DEV)
    before = w.cpu()
    dsk_moe.kv_evict(kd, vd, w, table.to(DEV), ints([101, 72]), 50, first=3, recent=20, k_scale=ks, v_scale=vs)
    O.append_codes(k.double(), vc, vb, [(1, 36), (3, 7)])
    wn = before[table.flatten().long()]
    O.evict([(kc, kb), (vc, vb)], wn, near, [101, 72], 50, 3, 20, 64)
    assert torch.equal(kd.view(U8)[ids].cpu(), kc) and torch.equal(vd.view(U8)[ids].cpu(), vc) and torch.equal(w[ids].cpu(), wn)


# ------------------------------------------------------------------ weights
def weights_want(w, q, k, table, lens, page, scale, pre=None, prefix=0):
    """(want, tol) of the weights after a call; k [pages, kv, page, dim] float64."""
    want, tol = w.double(), torch.zeros(w.shape, dtype=F64)
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        keys = O.rows_of(k, table[b], n)
        if prefix:
            keys = torch.cat([O.rows_of(k, pre, prefix), keys])
        last = prefix + torch.clamp(torch.arange(q.shape[1]) + n - q.shape[1], min=-1)
        got, err = O.key_weights(q[b], keys, last, scale)
        at = torch.arange(n)
        p, r = table[b].long()[at // page], at % page
        want[p, :, r] += got[prefix:]
        tol[p, :, r] += err[prefix:] + want[p, :, r] * O.F32_HALF_STEP
    return want, tol


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("heads,kv,dim,page,q_len", [(8, 2, 128, 64, 1), (3, 1, 64, 16, 1), (4, 4, 64, 32, 3), (16, 4, 128, 16, 16),
                                                     (40, 5, 128, 64, 2), (10, 2, 64, 256, 5)])
@pytest.mark.parametrize("prefix,spare", [(0, 1), (0, 100), (70, 1)])
def test_key_weights(codes, heads, kv, dim, page, q_len, prefix, spare):
    print(f"weights codes={codes} {heads},{kv},{dim} page {page} q {q_len} prefix {prefix} spare {spare}", flush=True)
    g = gen(heads + dim + page + q_len)
    lens = [0, 16, 17, 200, -1, 300, 3, 128]
    pre, table, kc, ks, vc, vs = paged8_setup(g, lens, kv, page, dim, spare, prefix)
    k64, v64 = O.values(kc, ks), O.values(vc, vs)
    q = normal(g, len(lens), q_len, heads, dim) * 2
    w = torch.rand(kc.shape[:3], generator=g)
    wd = w.to(DEV)
    more = dict(prefix=pre.to(DEV), prefix_len=prefix) if prefix else {}
    if codes:
        got = run_paged8(q, table, lens, kc, ks, vc, vs, key_weights=wd, scale=0.07, **more)
    else:
        k64, v64 = k64.to(BF16).double(), v64.to(BF16).double()
        got = dsk_moe.paged_attention(q.to(DEV), k64.to(BF16).to(DEV), v64.to(BF16).to(DEV), table.to(DEV), ints(lens), key_weights=wd,
                                      scale=0.07, **more)
    live = [i for i, n in enumerate(lens) if n >= 0]
    want, tol = O.paged(q, k64, v64, table, lens, pre, prefix, scale=0.07)
    assert_within(got[live], want[live], tol[live])
    want, tol = weights_want(w, q, k64, table, lens, page, 0.07, pre, prefix)
    assert_within(wd, want, tol + 1e-38, "weights")
    untouched = tol == 0
    assert torch.equal(wd.cpu()[untouched], w[untouched])


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv,q_len", [(4, 1, 5), (8, 1, 4), (8, 1, 8), (4, 1, 16)])
@pytest.mark.parametrize("prefix", [0, 300])
def test_many_rows_in_wide_tables(codes, dim, heads, kv, q_len, prefix):
    """More than 16 rows an item where the tables have many places (the other cases have few)."""
    g = gen(heads + q_len + dim)
    lens = [900, 40, 0]
    pre, table, kc, ks, vc, vs = paged8_setup(g, lens, kv, 256, dim, 1, prefix)
    more = dict(prefix=pre.to(DEV), prefix_len=prefix) if prefix else {}
    wide = torch.full((3, 700), -1, dtype=I32)                   # 537600 places
    wide[:, :table.shape[1]] = table
    k64, v64 = O.values(kc, ks), O.values(vc, vs)
    q = normal(g, 3, q_len, heads, dim)
    w = torch.rand(kc.shape[:3], generator=g)
    wd = w.to(DEV)
    if codes:
        got = run_paged8(q, wide, lens, kc, ks, vc, vs, key_weights=wd, **more)
        assert torch.equal(got, run_paged8(q, wide, lens, kc, ks, vc, vs, **more))
    else:
        k64, v64 = k64.to(BF16).double(), v64.to(BF16).double()
        got = dsk_moe.paged_attention(q.to(DEV), k64.to(BF16).to(DEV), v64.to(BF16).to(DEV), wide.to(DEV), ints(lens), key_weights=wd, **more)
    want, tol = O.paged(q, k64, v64, wide, lens, pre, prefix)
    assert_within(got, want, tol)
    want, tol = weights_want(w, q, k64, wide, lens, 256, dim ** -0.5, pre, prefix)
    assert_within(wd, want, tol + 1e-38, "weights")


def test_key_weights_add_up_and_repeat():
    """The same call twice gives twice the weight, bit for bit the same each time; outputs are those without weights."""
    g = gen(41)
    lens = [700, 1, 33]
    _, table, kc, ks, vc, vs = paged8_setup(g, lens, 2, 32, 128, 1)
    q = normal(g, 3, 1, 8, 128)
    a, b = (torch.zeros(kc.shape[:3], device=DEV) for _ in range(2))
    plain = run_paged8(q, table, lens, kc, ks, vc, vs)
    assert torch.equal(run_paged8(q, table, lens, kc, ks, vc, vs, key_weights=a), plain)
    run_paged8(q, table, lens, kc, ks, vc, vs, key_weights=b)
    assert torch.equal(a, b)
    run_paged8(q, table, lens, kc, ks, vc, vs, key_weights=b)
    assert torch.equal(b, 2 * a)
    # every query gives one in all
    total = sum(float(a[table[i, :-(-n // 32)].long()].double().sum()) for i, n in enumerate(lens))
    assert abs(total - 3 * 8) < 24 * 2.0 ** -15


@pytest.mark.parametrize("spare", [1, 200])
def test_key_weights_of_bad_sequences(spare):
    """A NaN query gives NaN to the keys that it sees and nothing to others; a length beyond the table row changes nothing."""
    g = gen(42)
    lens = [40, 40, 40, 100000]
    _, table, kc, ks, vc, vs = paged8_setup(g, [40] * 4, 1, 16, 64, spare)
    q = normal(g, 4, 2, 4, 64)
    q[1, 0, 2] = NAN
    w = torch.rand(kc.shape[:3], generator=g)
    wd = w.to(DEV)
    run_paged8(q, table, lens, kc, ks, vc, vs, key_weights=wd)
    got = wd.cpu()
    at = lambda b, r: got[int(table[b, r // 16]), 0, r % 16]  # noqa: E731
    assert all(bool(at(1, r).isnan()) for r in range(39)) and not at(1, 39).isnan()      # the second token alone sees it
    assert not any(bool(at(b, r).isnan()) for b in (0, 2) for r in range(40))
    for r in range(64):
        assert at(3, r) == w[int(table[3, r // 16]), 0, r % 16] if r < 48 else True


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("heads,q_len", [(2, 2), (8, 2), (8, 8)])
@pytest.mark.parametrize("spare", [1, 200])
def test_key_weights_of_endless_scores(codes, heads, q_len, spare):
    """Scores of minus infinity: a row of nothing else is NaN, as its output is, to all keys that it sees and to no others; among
    others such a key gets nothing; beside a NaN score it is NaN as well."""
    g = gen(heads + q_len)
    lens = [37, 37, 37]
    _, table, kc, ks, vc, vs = paged8_setup(g, lens, 1, 16, 64, spare)
    k64 = O.values(kc, ks) if codes else normal(g, *kc.shape).double()
    v64 = O.values(vc, vs) if codes else normal(g, *vc.shape).double()
    q = normal(g, 3, q_len, heads, 64)
    row = lambda b, r: (int(table[b, r // 16]), 0, r % 16)  # noqa: E731
    minus = 0xb8                                           # the code of -1

    def put(b, r, code, value):
        if codes:
            kc[row(b, r)][0] = code
        k64[row(b, r)][0] = value

    q[0, 0, 1, 0] = q[1, 0, 1, 0] = INF
    for r in range(37):
        for b in (0, 1):
            put(b, r, minus, -1.0)
    put(1, 3, 0x7f, NAN)
    if codes:
        k64 = O.values(kc, ks)
    else:
        k64[row(2, 5)][0] = -INF
        q[2, :, :, 0] = q[2, :, :, 0].abs() + 1
    w = torch.zeros(kc.shape[:3], dtype=F32)
    wd = w.to(DEV)
    if codes:
        out = run_paged8(q, table, lens, kc, ks, vc, vs, key_weights=wd)
    else:
        out = dsk_moe.paged_attention(q.to(DEV), k64.to(BF16).to(DEV), v64.to(BF16).to(DEV), table.to(DEV), ints(lens), key_weights=wd)
    got = wd.cpu()
    assert out[0, 0, 1].isnan().all() and out[1, 0, 1].isnan().all()
    seen = 37 - q_len + 1                                  # by the first token
    for r in range(37):
        assert bool(got[row(0, r)].isnan()) == (r < seen), r
        assert bool(got[row(1, r)].isnan()), r             # the other heads and tokens meet the NaN itself
    assert not got[table[2, :3].long()].isnan().any() and torch.isfinite(out[2]).all()
    total = q_len * heads                                  # (the first tokens see fewer keys, but some)
    assert abs(float(got[table[2, :3].long()].double().sum()) - total) < total * 2.0 ** -15
    if not codes:
        assert got[row(2, 5)] == 0


# ------------------------------------------------------------------ eviction
def evict_case(g, lens, keep, first, recent, kv, page, dim, codes, weights=None, spoil=None, spare=1, **kw):
    used = [-(-max(0, n) // page) for n in lens]
    table, kb, vb = paged_setup(g, used, max(used) + spare, 2, kv, page, dim)
    n = sum(used) + 2
    if codes:
        kc, ks = code_cache(g, n, kv, page, dim)
        vc, vs = code_cache(g, n, kv, page, dim)
        kd, vd = dev8(kc, vc)
        ksd, vsd = ks.to(DEV), vs.to(DEV)
    else:
        (kc, vc), (ks, vs, ksd, vsd) = (kb, vb), (None,) * 4
        kd, vd = kc.to(DEV), vc.to(DEV)
    w = weights(n, kv, page) if weights else torch.rand((n, kv, page), generator=g)
    table = spoil(table, n) if spoil else table
    wd, lens_d = w.to(DEV), ints(lens)
    got = dsk_moe.kv_evict(kd, vd, wd, table.to(DEV), lens_d, keep, first=first, recent=recent, k_scale=ksd, v_scale=vsd, **kw)
    want = O.evict([(kc, ks), (vc, vs)], w, table, lens, keep, first, recent, page)
    assert got.tolist() == want and lens_d.tolist() == lens
    assert torch.equal(wd.cpu().view(I32), w.view(I32))
    view = (lambda t: t.cpu().view(U8)) if codes else (lambda t: t.cpu().view(torch.int16))
    assert torch.equal(view(kd), kc if codes else kc.view(torch.int16)) and torch.equal(view(vd), vc if codes else vc.view(torch.int16))
    if codes:
        assert torch.equal(ksd.cpu(), ks) and torch.equal(vsd.cpu(), vs)


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("dim,page,kv", [(128, 64, 2), (64, 16, 3), (64, 128, 1)])
@pytest.mark.parametrize("keep,first,recent", [(1, 0, 0), (1, 0, 1), (1, 1, 0), (40, 4, 7), (64, 0, 64), (64, 64, 0), (64, 0, 32), (50, 0, 0),
                                               (49, 1, 48), (100, 4, 17)])
def test_evict(codes, dim, page, kv, keep, first, recent):
    print(f"evict codes={codes} {dim} {page} {kv} keep {keep} first {first} recent {recent}", flush=True)
    g = gen(dim + page + keep + first + recent)
    evict_case(g, [0, 1, keep, keep + 1, keep + 2, keep + 16, 2 * keep + 3, 300, -1, 129], keep, first, recent, kv, page, dim, codes)


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("lens,keep,first,recent", [([5000], 1000, 4, 200), ([2500, 1500], 1400, 0, 700), ([3000], 2999, 0, 0), ([1030, 1090], 1024, 4, 128),
                                                    ([4200], 30, 0, 10), ([40000, 17000], 16500, 3, 100)])
def test_evict_of_long_sequences(codes, lens, keep, first, recent):
    g = gen(sum(lens) + keep)
    evict_case(g, lens, keep, first, recent, 1 if lens[0] > 10000 else 2, 64, 64, codes)


@pytest.mark.parametrize("codes", [False, True])
def test_evict_of_sequences_in_wide_tables(codes):
    """Short sequences whose tables have room for many more rows."""
    evict_case(gen(50), [300, 41, 100, 40, 0], 40, 2, 9, 2, 32, 64, codes, spare=200)


@pytest.mark.parametrize("codes", [False, True])
def test_evict_ties_and_weights_that_are_no_numbers(codes):
    """Equal weights, zeros of both signs, infinities and NaN: the earlier of equal ones, NaN above all."""
    g = gen(51)

    def few(n, kv, page):
        v = torch.tensor([0.0, -0.0, 1.0, 1.0, 2.0, INF, NAN, -NAN, -1.0, -INF, 1e-42, -1e-42])
        return v[torch.randint(0, len(v), (n, kv, page), generator=g)]
    for keep, first, recent in ((60, 2, 10), (150, 0, 0), (20, 0, 0)):
        evict_case(g, [200, 170, 300, 61], keep, first, recent, 2, 32, 64, codes, weights=few)
    evict_case(g, [200, 1200], 60, 2, 10, 2, 32, 64, codes, weights=lambda n, kv, page: torch.zeros(n, kv, page))


@pytest.mark.parametrize("codes", [False, True])
def test_evict_leaves_bad_pages_and_lengths_alone(codes):
    """Rows on pages outside the cache do not move and are the first to go; a length beyond the table row is left."""
    g = gen(52)

    def spoil(table, n):
        table = table.clone()
        table[0, 1], table[1, 5], table[1, 0], table[2, 2] = n, -1, 1 << 30, -7
        return table
    for keep, first, recent in ((40, 4, 16), (70, 0, 5), (33, 0, 33)):
        evict_case(g, [100, 110, 90], keep, first, recent, 2, 16, 64, codes, spoil=spoil)
    evict_case(g, [100, 110], 40, 0, 3, 2, 16, 64, codes, spoil=lambda t, n: t[:, :6])


@pytest.mark.parametrize("codes", [False, True])
def test_evict_again_and_again_in_place(codes):
    """One row of each sequence a time, lengths in place, on a workspace of the caller's, captured and replayed."""
    g = gen(53)
    page, kv, dim, keep = 16, 2, 64, 40
    table, kb, vb = paged_setup(g, [4, 4], 5, 1, kv, page, dim)
    if codes:
        kc, ks = code_cache(g, 9, kv, page, dim)
        vc, vs = code_cache(g, 9, kv, page, dim)
        (kd, vd), ksd, vsd = dev8(kc, vc), ks.to(DEV), vs.to(DEV)
    else:
        kc, vc, ks, vs, ksd, vsd = kb, vb, None, None, None, None
        kd, vd = kc.to(DEV), vc.to(DEV)
    w = torch.rand((9, kv, page), generator=g)
    wd, lens, td = w.to(DEV), ints([41, 44]), table.to(DEV)
    ws = torch.empty(1 << 20, dtype=U8, device=DEV)
    call = lambda: dsk_moe.kv_evict(kd, vd, wd, td, lens, keep, first=2, recent=9, k_scale=ksd, v_scale=vsd, lens_out=lens, workspace=ws)  # noqa: E731
    side = torch.cuda.Stream()
    graph = None
    for step in range(6):
        if step == 2:
            saved = [t.clone() for t in (kd.view(U8) if codes else kd, vd.view(U8) if codes else vd, wd, lens)]
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                call()
            for t, s in zip((kd.view(U8) if codes else kd, vd.view(U8) if codes else vd, wd, lens), saved):
                t.copy_(s)
        now = lens.tolist()
        if graph is not None and step % 2 == 0:
            graph.replay()
        else:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                call()
            torch.cuda.current_stream().wait_stream(side)
        new = O.evict([(kc, ks), (vc, vs)], w, table, now, keep, 2, 9, page)
        assert lens.tolist() == new
        assert torch.equal(wd.cpu(), w) and torch.equal(kd.cpu().view(U8), kc.view(U8)) and torch.equal(vd.cpu().view(U8), vc.view(U8))
        lens += ints([1, 3])
        more = torch.rand(wd.shape, generator=g)
        w += more
        wd += more.to(DEV)
        assert torch.equal(wd.cpu(), w)


def test_calls_on_two_streams():
    """Appends, attention with weights and evictions of two caches at once, on streams of their own: as one after the other."""
    runs = []
    for streams in ((None, None), (torch.cuda.Stream(), torch.cuda.Stream())):
        outs = []
        states = []
        for i in range(2):
            g = gen(80 + i)
            lens = [700 - 300 * i, 90, 33]
            _, table, kc, ks, vc, vs = paged8_setup(g, [n + 16 for n in lens], 2, 32, 128, 1 + 100 * i)
            kd, vd = dev8(kc, vc)
            states.append((table.to(DEV), kd, vd, ks.to(DEV), vs.to(DEV), torch.zeros(kc.shape[:3], device=DEV),
                           [(normal(g, 3, 8, 128).to(DEV), normal(g, 3, 2, 128).to(DEV)) for _ in range(4)], lens))
        torch.cuda.synchronize()
        for t in range(4):
            for st, (table, kd, vd, ks, vs, w, qk, lens) in zip(streams, states):
                with torch.cuda.stream(st) if st is not None else torch.cuda.stream(torch.cuda.current_stream()):
                    rows = ints([n + t for n in lens])
                    extra = dict(k_scale=ks, v_scale=vs, key_weights=w)
                    q = dsk_moe.kv_append(qk[t][0], qk[t][1], qk[t][1], rows, ints([0, 1, 2]), table, kd, vd, dsk_moe.rope_frequencies(128)[0], **extra)
                    outs.append(dsk_moe.paged_attention(q, kd, vd, table, rows + 1, **extra))
                    if t == 2:
                        dsk_moe.kv_evict(kd, vd, w, table, rows + 1, 95, first=1, recent=20, k_scale=ks, v_scale=vs)
        torch.cuda.synchronize()
        runs.append(outs + [x.view(U8) if x.dtype == F8 else x for s in states for x in s[1:6]])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


# ------------------------------------------------------------------ together
def rows_and_lens(lens, q_len=1):
    return ints([n + i for n in lens for i in range(q_len)]), ints([n + q_len for n in lens])


@pytest.mark.parametrize("dtype", [BF16, F8])
def test_prompts_steps_and_evictions(dtype):
    """Prompts on three axes, decode and verify steps, an eviction, and steps behind it: every call against the restatement
    on the cache as it then is."""
    g = gen(61)
    heads, kv, dim, page, pages = 8, 2, 128, 32, 40
    f8 = dtype == F8
    kd, vd = (torch.zeros((pages, kv, page, dim), dtype=U8, device=DEV).view(F8) if f8 else torch.zeros((pages, kv, page, dim), dtype=BF16, device=DEV)
              for _ in range(2))
    ks, vs = (torch.zeros((pages, kv, page // 16), dtype=U8, device=DEV) for _ in range(2)) if f8 else (None, None)
    wd = torch.full((pages, kv, page), 99.0, device=DEV)
    extra = dict(k_scale=ks, v_scale=vs, key_weights=wd)
    freq, axis = dsk_moe.rope_axes([16, 24, 24], device="cpu")
    fd, ad = freq.to(DEV), axis.to(DEV)
    table = torch.randperm(pages, generator=g)[:30].view(3, 10).to(I32)
    td = table.to(DEV)

    def now():
        if not f8:
            return kd.cpu().double(), vd.cpu().double()
        return O.values(kd.cpu().view(U8), ks.cpu()), O.values(vd.cpu().view(U8), vs.cpu())

    def step(lens, q_len, where):
        t = 3 * q_len
        q, k, v = normal(g, t, heads, dim), normal(g, t, kv, dim), normal(g, t, kv, dim)
        rows, new = rows_and_lens(lens, q_len)
        pos = (torch.tensor(where)[:, None] + torch.arange(q_len)).flatten().to(I32).expand(3, t).contiguous()
        seq = torch.arange(3, dtype=I32).repeat_interleave(q_len).to(DEV)
        qr = dsk_moe.kv_append(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), seq, td, kd, vd, fd, axis=ad, rows=rows, **extra)
        w = wd.cpu()
        o = dsk_moe.paged_attention(qr.view(3, q_len, heads, dim), kd, vd, td, new, **extra)
        k64, v64 = now()
        lens = new.tolist()
        want, tol = O.paged(qr.cpu().view(3, q_len, heads, dim), k64, v64, table, lens)
        assert_within(o, want, tol)
        want, tol = weights_want(w, qr.cpu().view(3, q_len, heads, dim), k64, table, lens, page, dim ** -0.5)
        assert_within(wd, want, tol + 1e-38, "weights")
        for b, n in enumerate(lens):                             # fresh keys have this step's weight alone
            assert wd[int(table[b, (n - 1) // page]), :, (n - 1) % page].max() <= heads // kv * q_len * 1.001
        return lens, [x + q_len for x in where]

    lens = [60, 100, 1]
    t = sum(lens)
    q, k, v = normal(g, t, heads, dim), normal(g, t, kv, dim), normal(g, t, kv, dim)
    pos = torch.randint(0, 40, (3, t), generator=g, dtype=I32)
    rows = ints([i for n in lens for i in range(n)])
    kr = torch.empty((t, kv, dim), dtype=BF16, device=DEV)
    qr = dsk_moe.kv_append(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), ints([b for b, n in enumerate(lens) for _ in range(n)]), td, kd, vd, fd,
                           axis=ad, rows=rows, k_out=kr, **extra)
    want, tol = O.norm_rope(k, pos[axis.long()].t(), freq)
    assert_within(kr, want, tol)
    o = dsk_moe.prompt_attention(qr, kr, v.to(DEV), ints(cumulative(lens)))
    want, tol = O.prompt(qr.cpu(), kr.cpu(), v, cumulative(lens), cumulative(lens))
    assert_within(o, want, tol)
    for b, n in enumerate(lens):
        assert not wd[table[b, :-(-n // page)].long()].transpose(1, 2).flatten(0, 1)[:n].any()
    where = [200, 300, 50]
    lens, where = step(lens, 1, where)
    lens, where = step(lens, 3, where)
    assert lens == [64, 104, 5]
    caches = [(kd.cpu().view(U8), ks.cpu()), (vd.cpu().view(U8), vs.cpu())] if f8 else [(kd.cpu(), None), (vd.cpu(), None)]
    w = wd.cpu()
    new = dsk_moe.kv_evict(kd, vd, wd, td, ints(lens), 41, first=2, recent=9, k_scale=ks, v_scale=vs)
    assert O.evict(caches, w, table, lens, 41, 2, 9, page) == new.tolist() == [41, 41, 5]
    assert torch.equal(kd.cpu().view(U8), caches[0][0].view(U8)) and torch.equal(vd.cpu().view(U8), caches[1][0].view(U8)) and torch.equal(wd.cpu(), w)
    lens = new.tolist()
    for q_len in (1, 2, 1):
        lens, where = step(lens, q_len, where)


def decoder_with(seed, dtype, weigh, axis=False, n=2):
    g, stack = make_decoder(seed, n=n)
    for a in stack.attention:
        page = a.k_cache.shape[2]
        a.new_cache(a.k_cache.shape[0], page, dtype=dtype, weigh=weigh)
        if axis:
            pairs = a._rotate["freq"].numel()
            a._rotate["axis"] = torch.arange(pairs, dtype=I32, device=DEV) % 3
    return g, stack


@pytest.mark.parametrize("dtype", [BF16, F8])
def test_decoder_with_evictions_captured_and_eager(dtype):
    """A decoder's prompts, then captured steps with an eviction between them, against an eager twin, bit for bit; both follow
    the lengths, rows and positions in place."""
    runs = []
    for captured in (False, True):
        g, stack = decoder_with(71, dtype, 4)
        table = torch.randperm(60, generator=g)[:36].view(3, 12).to(I32).to(DEV)
        lens = [40, 1, 70]
        pos = ints([i for n in lens for i in range(n)])
        seq = ints([b for b, n in enumerate(lens) for _ in range(n)])
        outs = [stack(normal(g, sum(lens), 1024).to(DEV), step=dsk_moe.PromptStep(pos, seq, table, ints(cumulative(lens)))).clone()]
        assert all(a.key_weights.any() for a in stack.attention)
        lens = ints(lens + [-1])
        table = torch.cat([table, table[:1]])
        live = (lens >= 0).int()
        step = dsk_moe.DecodeStep(lens.clone(), torch.arange(4, dtype=I32, device=DEV), table, lens + live, rows=lens.clone())
        if captured:
            stack.capture(4, step=step)
        for i in range(9):
            if i in (3, 6):
                step.lens -= live                                # what is kept so far
                step.rows -= live
                stack.evict(step, 24, first=2, recent=8)
                assert step.lens.tolist()[0] == 24 and step.rows.tolist() == [x - 1 for x in step.lens.tolist()[:3]] + [-1]
                step.lens += live
                step.rows += live
            x = normal(g, 4, 1024).to(DEV)
            outs.append((stack.replay(x) if captured else stack(x, step=step)).clone())
            assert torch.isfinite(outs[-1].float()).all()
            for t in (step.positions, step.lens, step.rows):
                t += live
        outs += [t.view(U8) if t.dtype == F8 else t for a in stack.attention for t in a.cache_tensors() if t is not None]
        runs.append(outs)
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F8])
def test_decoder_on_several_axes_in_8_bits(dtype):
    """Text has the same position on all axes: a decoder with axes gives what one without them does, bit for bit."""
    outs = []
    for axis in (False, True):
        g, stack = decoder_with(72, dtype, None, axis)
        table = torch.randperm(60, generator=g)[:12].view(1, 12).to(I32).to(DEV)
        pos = torch.arange(50, dtype=I32, device=DEV)
        step = dsk_moe.PromptStep(pos.expand(3, 50).contiguous() if axis else pos, torch.zeros_like(pos), table, ints([0, 50]),
                                  rows=pos if axis else None)
        got = [stack(normal(g, 50, 1024).to(DEV), step=step).clone()]
        at = ints([50])
        step = dsk_moe.DecodeStep(at.expand(3, 1).contiguous() if axis else at, ints([0]), table, ints([51]), rows=at if axis else None)
        got.append(stack(normal(g, 1, 1024).to(DEV), step=step).clone())
        outs.append(got)
    for a, b in zip(*outs):
        assert torch.equal(a, b) and torch.isfinite(a.float()).all()


@pytest.mark.parametrize("dtype", [BF16, F8])
def test_captured_prompts_that_weigh(dtype):
    """A captured step of whole prompts on three axes follows its bounds, places and positions: outputs, caches and weights as
    the eager step's, every replay."""
    g, stack = decoder_with(76, dtype, 5, True)
    tokens = 60
    table = torch.randperm(60, generator=g)[:36].view(3, 12).to(I32).to(DEV)

    def fill(step, lens):
        rows = torch.full((tokens,), -1, dtype=I32)
        rows[:sum(lens)] = torch.tensor([i for n in lens for i in range(n)], dtype=I32)
        step.rows.copy_(rows)
        step.positions.copy_(torch.where(rows >= 0, torch.randint(0, 50, (3, tokens), generator=g, dtype=I32), -1))
        step.seq.copy_(torch.tensor([b for b, n in enumerate(lens) for _ in range(n)] + [0] * (tokens - sum(lens)), dtype=I32))
        step.cu.copy_(torch.tensor(cumulative(lens), dtype=I32))

    rows = torch.arange(tokens, dtype=I32, device=DEV)
    step = dsk_moe.PromptStep(rows.repeat(3, 1), torch.zeros_like(rows), table, ints([0, tokens, tokens, tokens]), rows=rows)
    stack.capture(tokens, step=step)
    caches = [c for a in stack.attention for c in a.cache_tensors() if c is not None]
    raw = [c.view(U8) if c.dtype == F8 else c for c in caches]
    for lens in ([20, 1, 30], [60, 0, 0], [3, 4, 2], [20, 20, 20]):
        fill(step, lens)
        x = normal(g, tokens, 1024).to(DEV)
        for c in raw:
            c.zero_()
        got = stack.replay(x).clone()
        held = [c.clone() for c in raw]
        assert any(a.key_weights.any() for a in stack.attention)
        for c in raw:
            c.zero_()
        want = stack(x, step=step)
        assert torch.equal(got[:sum(lens)], want[:sum(lens)]) and all(torch.equal(c, h) for c, h in zip(raw, held))


def test_8_bit_decoder_is_near_the_bf16_one():
    """Not a parity: the two agree to the rounding of keys and values (2^-4 each at most, and their signs differ)."""
    outs = []
    for dtype in (BF16, F8):
        g, stack = decoder_with(73, dtype, None, n=1)
        table = torch.arange(12, dtype=I32, device=DEV)[None]
        pos = torch.arange(100, dtype=I32, device=DEV)
        stack(normal(g, 100, 1024).to(DEV), step=dsk_moe.PromptStep(pos, torch.zeros_like(pos), table, ints([0, 100])))
        a = stack.attention[0]
        outs.append(a(normal(g, 1, 1024).to(DEV), dsk_moe.DecodeStep(ints([100]), ints([0]), table, ints([101]))).double())
    assert (outs[0] - outs[1]).norm() <= 2.0 ** -3 * outs[0].norm()


def test_stack_evict_refuses():
    g, stack = decoder_with(74, BF16, None, n=1)
    step = dsk_moe.DecodeStep(ints([0]), ints([0]), ints([[0]]), ints([1]), rows=ints([0]))
    with pytest.raises(RuntimeError, match="weigh"):
        stack.evict(step, 4)
    stack.attention[0].new_cache(8, 16, weigh=0)
    with pytest.raises(ValueError, match="rows"):
        stack.evict(dsk_moe.DecodeStep(ints([0]), ints([0]), ints([[0]]), ints([1])), 4)
    stack.evict(step, 4)
    with pytest.raises(_lib.DskError):
        stack.evict(step, 0)
    stack.capture(1, step=step)
    stack.attention[0].key_weights = stack.attention[0].key_weights.clone()
    with pytest.raises(RuntimeError, match="another cache"):
        stack.replay()


def test_refusals_on_the_device():
    g = gen(75)
    k = normal(g, 2, 2, 64).to(DEV)
    kd = torch.zeros(2, 2, 16, 64, dtype=U8, device=DEV).view(F8)
    kb = torch.zeros(2, 2, 16, 64, dtype=BF16, device=DEV)
    s, table, one = torch.zeros(2, 2, 1, dtype=U8, device=DEV), ints([[0, 1]]), ints([0, 0])
    pos = ints([0, 1])
    for kc, more, text in ((kd, {}, "bf16"), (kb, dict(k_scale=s, v_scale=s), "float8"), (kd, dict(k_scale=s), "go together"),
                           (kd, dict(k_scale=s, v_scale=s[:1]), "v_scale"), (kb, dict(key_weights=torch.zeros(2, 2, 16)), "key_weights"),
                           (kb, dict(rows=ints([0])), "rows"), (kb, dict(axis=ints([0] * 16)), "positions")):
        with pytest.raises(ValueError, match=text):
            dsk_moe.kv_append(None, k, k, pos, one, table, kc, kc, dsk_moe.rope_frequencies(32)[0], **more)
    with pytest.raises(ValueError, match="axis"):
        dsk_moe.qk_norm_rope(None, k, pos[None], dsk_moe.rope_frequencies(32)[0], axis=ints([0] * 15))
    with pytest.raises(_lib.DskError, match="prefix_len"):
        dsk_moe.kv_append(None, k, k, pos, one, table, kb, kb, rows=pos, prefix_len=1)
    q = normal(g, 1, 4, 64).to(DEV)
    with pytest.raises(ValueError, match="bf16"):
        dsk_moe.paged_attention(q, kd, kd, table, ints([3]))
    w = torch.zeros(2, 2, 16, device=DEV)
    with pytest.raises(_lib.DskError, match="ESPACE"):
        dsk_moe.paged_attention(q, kb, kb, table, ints([3]), key_weights=w, workspace=torch.empty(256, dtype=U8, device=DEV))
    with pytest.raises(_lib.DskError, match="ESPACE"):
        dsk_moe.kv_evict(kb, kb, w, table, ints([20]), 4, workspace=torch.empty(256, dtype=U8, device=DEV))
    with pytest.raises(ValueError, match="lens_out"):
        dsk_moe.kv_evict(kb, kb, w, table, ints([20]), 4, lens_out=ints([0, 0]))
    with pytest.raises(ValueError, match="key_weights"):
        dsk_moe.kv_evict(kb, kb, w[:, :1], table, ints([20]), 4)
