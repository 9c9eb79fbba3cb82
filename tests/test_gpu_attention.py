"""GPU parity of the attention kernels with the float64 restatement, value by
value within the rounding errors that it derives (``oracle/attention.py``):
norm and rotation, the append to a paged cache, prompts and decode steps, with
and without a shared prefix; then a run of them as a server would make it,
captured and eager."""

from __future__ import annotations

import math

import pytest
import torch

import dsk_moe
from dsk_moe import _lib
from oracle import attention as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
NAN, INF = math.nan, math.inf


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=BF16):
    return torch.randn(shape, generator=g).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=I32, device=DEV)


def assert_within(got, want, tol, what=""):
    got = got.detach().cpu().double()
    assert not got.isnan().any(), f"{what}: NaN"
    over = ((got - want).abs() / tol).max() if got.numel() else 0.0
    assert over <= 1.0, f"{what}: off by {float(over):.3f} of what the roundings allow"


# ------------------------------------------------------------------ norm and rotation
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,rot,first,inter", [(128, 128, 0, False), (128, 128, 0, True), (128, 64, 64, False),
                                                 (128, 32, 8, True), (64, 64, 0, False), (64, 16, 48, False),
                                                 (64, 48, 16, True), (128, 0, 0, False)])
@pytest.mark.parametrize("tokens,heads,kv", [(1, 32, 8), (5, 3, 1), (600, 9, 4)])
def test_norm_rope(dtype, dim, rot, first, inter, tokens, heads, kv):
    print(f"norm_rope {dtype} {dim} {rot}+{first} inter={inter} {tokens}x{heads},{kv}", flush=True)
    g = gen(dim + rot + first + tokens)
    q, k = normal(g, tokens, heads, dim, dtype=dtype) * 3, normal(g, tokens, kv, dim, dtype=dtype)
    pos = torch.randint(0, 5000, (tokens,), generator=g, dtype=I32)
    gq, gk = torch.rand(dim, generator=g) + 0.5, torch.randn(dim, generator=g)
    freq = dsk_moe.rope_frequencies(rot, device="cpu")[0] if rot else None
    kw = dict(interleaved=inter, rot_first=first, mscale=1.25)
    got_q, got_k = dsk_moe.qk_norm_rope(q.to(DEV), k.to(DEV), pos.to(DEV), freq.to(DEV) if rot else None, q_gamma=gq.to(DEV),
                                        k_gamma=gk.to(DEV), **kw)
    assert got_q.dtype == got_k.dtype == BF16
    assert_within(got_q, *O.norm_rope(q, pos, freq, gamma=gq, **kw), "q")
    assert_within(got_k, *O.norm_rope(k, pos, freq, gamma=gk, **kw), "k")


def test_far_positions_and_padding():
    """Angles of positions up to 2^31 - 1; tokens at negative positions keep their output rows."""
    g = gen(3)
    pos = torch.tensor([(1 << 31) - 1, 123456789, -1, 0, -(1 << 31), 1 << 20], dtype=I32)
    q, k = normal(g, 6, 4, 128), normal(g, 6, 2, 128)
    freq, mscale = dsk_moe.rope_frequencies(128, 1e6, scaling="ramp", factor=8.0, device="cpu")
    qo, ko = torch.full((6, 4, 128), 7.0, dtype=BF16, device=DEV), torch.full((6, 2, 128), 8.0, dtype=BF16, device=DEV)
    dsk_moe.qk_norm_rope(q.to(DEV), k.to(DEV), pos.to(DEV), freq.to(DEV), mscale=mscale, q_out=qo, k_out=ko)
    live = pos >= 0
    for x, o, fill in ((q, qo, 7.0), (k, ko, 8.0)):
        y, tol = O.norm_rope(x, pos, freq, mscale=mscale)
        # positions * freq / (2 pi) in float64 at 2^31: 2^-21 of a turn
        tol = tol + 2 * math.pi * 2.0 ** -21 * 2.0 ** -1 * x.double().abs().amax(-1, keepdim=True) * 4
        assert_within(o.cpu()[live], y[live], tol[live])
        assert (o.cpu()[~live] == fill).all()


@pytest.mark.parametrize("inter", [False, True])
def test_norm_rope_views_and_in_place(inter):
    """Views of one projection's rows, heads-first layouts, and the results written over the inputs."""
    g = gen(4)
    qkv = normal(g, 33, (6 + 2 + 2) * 64).to(DEV)
    q, k, _ = (p.unflatten(1, (-1, 64)) for p in qkv.split([384, 128, 128], 1))
    pos, freq = torch.arange(33, dtype=I32, device=DEV), dsk_moe.rope_frequencies(64)[0]
    want = dsk_moe.qk_norm_rope(q.contiguous(), k.contiguous(), pos, freq, interleaved=inter)
    for a, b in zip(dsk_moe.qk_norm_rope(q, k, pos, freq, interleaved=inter), want):
        assert torch.equal(a, b)
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)         # [heads][tokens] in memory
    out = torch.empty_like(qt)
    assert out.stride() == qt.stride()
    got, _ = dsk_moe.qk_norm_rope(qt, k, pos, freq, interleaved=inter, q_out=out)
    assert torch.equal(got, want[0])
    before = qkv.clone()
    dsk_moe.qk_norm_rope(q, k, pos, freq, interleaved=inter, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 512:], before[:, 512:])


def test_no_norm_is_the_rotation_alone():
    g = gen(5)
    k = normal(g, 9, 2, 64, dtype=F32) * 100
    pos = torch.arange(9, dtype=I32)
    freq = dsk_moe.rope_frequencies(32, device="cpu")[0]
    _, got = dsk_moe.qk_norm_rope(None, k.to(DEV), pos.to(DEV), freq.to(DEV), norm=False)
    assert_within(got, *O.norm_rope(k, pos, freq, norm=False))
    _, got = dsk_moe.qk_norm_rope(None, k.to(DEV), pos.to(DEV), norm=False)
    assert torch.equal(got.cpu(), k.to(BF16))


# ------------------------------------------------------------------ append
def paged_setup(g, used, width, spare, kv, page, dim, fill=None):
    """(table [len(used), width] with used[b] shuffled pages, k_cache, v_cache)."""
    n = sum(used) + spare
    ids = torch.randperm(n, generator=g)[:sum(used)].to(I32)
    table = torch.zeros((len(used), width), dtype=I32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = ids[at:at + u]
        at += u
    make = (lambda: normal(g, n, kv, page, dim)) if fill is None else (lambda: torch.full((n, kv, page, dim), fill, dtype=BF16))
    return table, make(), make()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,page,prefix,inter", [(128, 64, 0, False), (64, 16, 0, True), (128, 256, 37, False), (64, 32, 5, False)])
def test_append(dtype, dim, page, prefix, inter):
    g = gen(dim + page)
    kv, heads = 3, 6
    lens, starts = [70, 1, 33, 2], [0, 500, 15, 255]
    used = [(a + n - 1) // page + 1 for a, n in zip(starts, lens)]
    table, kc, vc = paged_setup(g, used, max(used) + 2, 2, kv, page, dim)
    t = sum(lens)
    q, k, v = normal(g, t, heads, dim, dtype=dtype), normal(g, t, kv, dim, dtype=dtype), normal(g, t, kv, dim, dtype=dtype)
    row = torch.tensor([a + i for a, n in zip(starts, lens) for i in range(n)], dtype=I32)
    seq = torch.tensor([b for b, n in enumerate(lens) for _ in range(n)], dtype=I32)
    order = torch.randperm(t, generator=g)                       # tokens in any order
    row, seq, pos = row[order], seq[order], row[order] + prefix
    freq = dsk_moe.rope_frequencies(dim // 2, device="cpu")[0]
    gamma = torch.rand(dim, generator=g) + 0.5
    kd, vd = kc.to(DEV), vc.to(DEV)
    ko = torch.empty((t, kv, dim), dtype=BF16, device=DEV)
    got = dsk_moe.kv_append(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), seq.to(DEV), table.to(DEV), kd, vd, freq.to(DEV),
                            prefix_len=prefix, interleaved=inter, k_gamma=gamma.to(DEV), k_out=ko)
    assert_within(got, *O.norm_rope(q, pos, freq, interleaved=inter), "q")
    assert_within(ko, *O.norm_rope(k, pos, freq, interleaved=inter, gamma=gamma), "k")
    at, r = table[seq.long(), row.long() // page].long(), row.long() % page
    kc[at, :, r] = ko.cpu()
    vc[at, :, r] = v.to(BF16)
    assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), vc)


def test_append_leaves_out_what_has_no_place():
    """Negative positions, rows before the prefix's end or behind the table, unknown sequences and pages outside the
    cache: nothing of the cache changes; q is still written (not at negative positions)."""
    g = gen(8)
    kc, vc = normal(g, 4, 2, 16, 64), normal(g, 4, 2, 16, 64)
    table = torch.tensor([[0, 4, -1], [1, 2, 1 << 30]], dtype=I32)
    pos = torch.tensor([-1, 2, 10 + 16, 10 + 32, 10 + 48, 10 + 32, 10 + 3, 10 + 3, 10 + 17], dtype=I32)
    seq = torch.tensor([0, 0, 0, 0, 0, 1, 2, -1, 1], dtype=I32)
    q, k, v = normal(g, 9, 2, 64), normal(g, 9, 2, 64), normal(g, 9, 2, 64)
    kd, vd = kc.to(DEV), vc.to(DEV)
    qo = torch.full((9, 2, 64), 9.0, dtype=BF16, device=DEV)
    dsk_moe.kv_append(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), seq.to(DEV), table.to(DEV), kd, vd, prefix_len=10,
                      norm=False, q_out=qo)
    kc[2, :, 1], vc[2, :, 1] = k[8], v[8]                         # the last token alone has a place
    assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), vc)
    assert torch.equal(qo.cpu()[1:], q[1:]) and (qo.cpu()[0] == 9.0).all()


def test_append_without_queries():
    g = gen(9)
    kd, vd = (torch.zeros(2, 1, 32, 128, dtype=BF16, device=DEV) for _ in range(2))
    k, v = normal(g, 3, 1, 128), normal(g, 3, 1, 128)
    assert dsk_moe.kv_append(None, k.to(DEV), v.to(DEV), ints([31, 32, 0]), ints([0, 0, 0]), ints([[1, 0]]), kd, vd, norm=False) is None
    assert torch.equal(kd[1, 0, 31].cpu(), k[0, 0]) and torch.equal(vd[0, 0, 0].cpu(), v[1, 0]) and torch.equal(kd[1, 0, 0].cpu(), k[2, 0])
    assert int((kd != 0).any(-1).sum()) == 3


# ------------------------------------------------------------------ prompts
def cumulative(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def run_prompt(q, k, v, lens, lens_k=None, **kw):
    cu, ck = cumulative(lens), cumulative(lens_k or lens)
    got = dsk_moe.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), ints(cu), ints(ck) if lens_k else None, **kw)
    return got, O.prompt(q, k, v, cu, ck, **{x: kw[x] for x in ("causal", "scale") if x in kw})


@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 2, 128), (10, 2, 64), (8, 1, 128), (3, 1, 128)])
@pytest.mark.parametrize("lens", [[1], [17], [64], [65, 1, 0, 127, 3], [0, 0, 5], [200], [128, 129]])
def test_prompt(heads, kv, dim, lens):
    print(f"prompt {heads},{kv},{dim} {lens}", flush=True)
    g = gen(sum(lens) + heads)
    t = sum(lens)
    q, k, v = normal(g, t, heads, dim), normal(g, t, kv, dim), normal(g, t, kv, dim)
    got, (want, tol) = run_prompt(q, k, v, lens)
    assert_within(got, want, tol)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,lens,lens_k", [(128, [3, 40, 1, 20], [70, 40, 130, 300]), (64, [30, 5, 7], [10, 0, 1]), (128, [64], [1])])
def test_prompt_with_other_keys(causal, dim, lens, lens_k):
    """Keys of earlier tokens before the prompt's, or fewer keys than queries (rows without a key are zero)."""
    g = gen(7 * sum(lens))
    q, k, v = normal(g, sum(lens), 4, dim), normal(g, sum(lens_k), 2, dim), normal(g, sum(lens_k), 2, dim)
    got, (want, tol) = run_prompt(q, k, v, lens, lens_k, causal=causal, scale=0.2)
    assert_within(got, want, tol)
    if min(lens_k) == 0:
        assert not got[30:35].any()


def test_prompt_views_and_padding_rows():
    """Views of a fused projection, heads-first outputs; rows behind the last sequence stay as they were."""
    g = gen(21)
    lens, t = [50, 31], 90
    qkv = normal(g, t, (6 + 2 + 2) * 64)
    q, k, v = (p.unflatten(1, (-1, 64)) for p in qkv.split([384, 128, 128], 1))
    out = torch.full((6, t, 64), 5.0, dtype=BF16, device=DEV).transpose(0, 1)
    qd, kd, vd = (p.unflatten(1, (-1, 64)) for p in qkv.to(DEV).split([384, 128, 128], 1))
    got = dsk_moe.prompt_attention(qd, kd, vd, ints(cumulative(lens)), out=out)
    want, tol = O.prompt(q[:81], k[:81], v[:81], cumulative(lens), cumulative(lens))
    assert got is out
    assert_within(out[:81], want, tol)
    assert (out[81:] == 5.0).all()


@pytest.mark.parametrize("poison", [NAN, INF, -INF])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_unseen_values_stay_unseen(dim, poison):
    """NaN and infinities in keys and values of later tokens, other sequences and padding reach no row that does not
    see them; rows that do see them show it."""
    g = gen(22)
    lens = [70, 90, 20]
    cu = cumulative(lens)
    q, k, v = normal(g, 200, 4, dim), normal(g, 200, 2, dim), normal(g, 200, 2, dim)
    want, tol = O.prompt(q[:180], k[:180], v[:180], cu, cu)
    seen = torch.ones(180, dtype=torch.bool)
    for bad in ([0], [75, 135], [180]):                          # tokens: of sequence 0, of sequence 1, of padding
        for b in bad:
            if b < 180:
                end = next(c for c in cu if c > b)
                seen[b:end] = False                              # its own row and its sequence's later ones
            v[b, 1, 3] = poison
            k[b, 0, 5] = poison if b >= 180 else k[b, 0, 5]
    got = dsk_moe.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), ints(cu)).cpu()[:180].double()
    # heads 0, 1 read key head 0, whose values are finite
    clean = torch.ones(180, 4, dim, dtype=torch.bool)
    clean[~seen, 2:, 3] = False
    assert not torch.isfinite(got[~clean]).any()
    assert ((got - want).abs() <= tol)[clean].all()


def test_prompt_poisoned_later_keys():
    g = gen(23)
    q, k, v = normal(g, 100, 2, 128), normal(g, 100, 1, 128), normal(g, 100, 1, 128)
    want, tol = O.prompt(q, k, v, [0, 100], [0, 100])
    k[60] = NAN
    got = dsk_moe.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), ints([0, 100]))
    assert_within(got[:60], want[:60], tol[:60])
    assert got[60:].isnan().all()


def test_prompt_bounds_outside_are_cut():
    """Sequence bounds that are not ascending or leave the tensors touch no row outside."""
    g = gen(24)
    q, k, v = normal(g, 40, 2, 64), normal(g, 40, 1, 64), normal(g, 40, 1, 64)
    out = torch.full((40, 2, 64), 3.0, dtype=BF16, device=DEV)
    dsk_moe.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), ints([-5, 10, 7, 30, 1 << 30]), out=out)
    want, tol = O.prompt(q, k, v, [0, 10], [0, 10])
    assert_within(out[:7], want[:7], tol[:7])
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (8, 1, 128), (3, 3, 128), (5, 1, 64)])
@pytest.mark.parametrize("lens,lens_k", [([290], [290]), ([5, 40, 0, 33], [700, 257, 300, 331]), ([90, 1], [20, 513])])
def test_prompt_of_few_rows_and_many_keys(heads, kv, dim, lens, lens_k, causal):
    g = gen(sum(lens_k) + heads)
    q, k, v = normal(g, sum(lens), heads, dim), normal(g, sum(lens_k), kv, dim), normal(g, sum(lens_k), kv, dim)
    got, (want, tol) = run_prompt(q, k, v, lens, lens_k, causal=causal)
    assert_within(got, want, tol)


@pytest.mark.parametrize("poison", [NAN, INF, -INF])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_of_many_keys_unseen_values_stay_unseen(dim, poison):
    """As above, for rows whose keys two waves share: a poisoned key in either half of a tile."""
    g = gen(26)
    cu = [0, 290, 570]
    q, k, v = normal(g, 570, 2, dim), normal(g, 570, 2, dim), normal(g, 570, 2, dim)
    want, tol = O.prompt(q, k, v, cu, cu)
    clean = torch.ones(570, 2, dim, dtype=torch.bool)
    for at, end in ((270, 290), (290 + 200, 570), (290 + 250, 570)):
        v[at, 1, 7] = poison
        clean[at:end, 1, 7] = False
    k[569, 0] = NAN                                              # seen by its own row alone
    clean[569, 0] = False
    got = dsk_moe.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), ints(cu)).cpu().double()
    assert not torch.isfinite(got[~clean]).any()
    assert ((got - want).abs() <= tol)[clean].all()


@pytest.mark.parametrize("longest", [0, 700])
def test_prompt_of_many_sequences(longest):
    """More sequences than lanes, and one whose row tiles are more than lanes."""
    lens = [(7 * i) % 10 for i in range(150)]
    lens[77] = longest
    g = gen(27)
    t = sum(lens)
    q, k, v = normal(g, t, 16, 64), normal(g, t, 1, 64), normal(g, t, 1, 64)
    got, (want, tol) = run_prompt(q, k, v, lens)
    assert_within(got, want, tol)


def test_prompt_behind_very_many_keys():
    g = gen(28)
    lens, lens_k = [3, 2], [10, 40000]
    q, k, v = normal(g, 5, 16, 64), normal(g, 40010, 1, 64), normal(g, 40010, 1, 64)
    got, (want, tol) = run_prompt(q, k, v, lens, lens_k)
    assert_within(got, want, tol)


def test_prompt_long_rows():
    """2000 tokens: every row of a few heads against float64 on the device (tolerances as the oracle's)."""
    g = torch.Generator(device=DEV).manual_seed(25)
    q, k, v = (torch.randn((2000, h, 128), generator=g, device=DEV).to(BF16) for h in (8, 2, 2))
    got = dsk_moe.prompt_attention(q, k, v, ints([0, 2000])).double()
    hidden = torch.ones((2000, 2000), dtype=torch.bool, device=DEV).triu(1)
    for h in range(8):
        qh, kh, vh = q[:, h].double(), k[:, h // 4].double(), v[:, h // 4].double()
        w = torch.softmax((qh @ kh.T / 128 ** 0.5).masked_fill(hidden, -INF), -1)
        size = float((qh.abs() @ kh.abs().T).max()) / 128 ** 0.5
        slack = 4 * (2000 + 128 * size + 16) * 2.0 ** -24
        want = w @ vh
        tol = (w @ vh.abs()) * (2.0 ** -8 + slack) + want.abs() * 2.0 ** -8 * (1 + 2.0 ** -6)
        assert ((got[:, h] - want).abs() <= tol).all()


# ------------------------------------------------------------------ decode
@pytest.mark.parametrize("heads,kv,dim,page,q_len", [(8, 2, 128, 64, 1), (4, 4, 64, 16, 1), (8, 1, 64, 32, 3), (16, 1, 128, 16, 4),
                                                     (10, 2, 128, 128, 2), (64, 1, 64, 256, 1), (3, 3, 128, 16, 16), (20, 1, 128, 32, 2)])
@pytest.mark.parametrize("prefix,spare", [(0, 1), (0, 70), (1, 1), (130, 1)])
def test_paged(heads, kv, dim, page, q_len, prefix, spare):
    print(f"paged {heads},{kv},{dim} page {page} q_len {q_len} prefix {prefix}", flush=True)
    g = gen(heads * dim + page + prefix)
    lens = [0, 1, 15, 16, 17, 127, 128, 129, 300, -1]
    used = [-(-max(n, 0) // page) for n in lens]
    shared = -(-prefix // page)
    # wide tables: the work is shared out; short ones: a workgroup for an item
    table, kc, vc = paged_setup(g, used + [shared], max(max(used) + spare, shared), 2, kv, page, dim)
    pre, table = table[-1, :shared], table[:-1]
    # what no sequence holds is NaN: rows behind the lengths, and pages of nobody
    held = torch.zeros(kc.shape[0], page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(n):
            held[table[b, j // page], j % page] = True
    for j in range(prefix):
        held[pre[j // page], j % page] = True
    for c in (kc, vc):
        c.transpose(1, 2)[~held] = NAN
    q = normal(g, len(lens), q_len, heads, dim)
    q[-1, :, 1] = NAN                                            # an unused slot's q may hold anything
    got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), table.to(DEV), ints(lens),
                                  prefix=pre.to(DEV) if prefix else None, prefix_len=prefix, scale=0.15)
    want, tol = O.paged(q[:-1], kc, vc, table, lens[:-1], pre, prefix, scale=0.15)
    assert got.shape == q.shape
    assert_within(got[:-1], want, tol)
    assert (got[-1] == 0).all()
    if not prefix:
        assert not got[0].any()


@pytest.mark.parametrize("batch,longest", [(1, 5000), (3, 2500), (150, 300)])
def test_paged_long_and_many(batch, longest):
    """Items over many shares, many items in a share."""
    g = gen(batch)
    lens = [int(x) for x in torch.randint(0, longest, (batch,), generator=g)]
    lens[batch // 2] = longest
    used = [-(-n // 64) for n in lens]
    table, kc, vc = paged_setup(g, used, max(used), 1, 2, 64, 128)
    q = normal(g, batch, 4, 128)
    got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), table.to(DEV), ints(lens))
    want, tol = O.paged(q[:, None], kc, vc, table, lens)
    assert_within(got, want[:, 0], tol[:, 0])


@pytest.mark.parametrize("batch,heads,kv,dim,q_len,width,longest,prefix", [
    (150, 8, 2, 128, 1, 80, 300, 0), (70, 4, 1, 64, 2, 80, 1200, 0), (130, 8, 8, 64, 1, 60, 960, 0), (260, 8, 2, 128, 1, 64, 1024, 0),
    (150, 8, 2, 64, 1, 80, 300, 200), (70, 8, 1, 128, 4, 80, 700, 100)])
def test_paged_many_sequences(batch, heads, kv, dim, q_len, width, longest, prefix):
    """More sequences than lanes over shares or in tables that a workgroup takes alone, long and empty ones among them;
    their tables hold the same pages in different orders."""
    page = 16
    g = gen(batch + dim + width)
    n_pages = width + 20
    kc, vc = normal(g, n_pages, kv, page, dim), normal(g, n_pages, kv, page, dim)
    table = torch.stack([torch.randperm(n_pages, generator=g)[:width] for _ in range(batch)]).to(I32)
    lens = torch.randint(0, 40, (batch,), generator=g).to(I32)
    lens[[0, 5, 63, 64, batch - 1]] = torch.tensor([longest, 0, longest, longest // 2, longest - 1], dtype=I32)
    lens[lens > 0] = lens[lens > 0].clamp(min=q_len)
    q = normal(g, batch, q_len, heads, dim)
    pre = torch.randperm(n_pages, generator=g)[:-(-prefix // page)].to(I32)
    kw = dict(prefix=pre.to(DEV), prefix_len=prefix) if prefix else {}
    got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), table.to(DEV), lens.to(DEV), **kw)
    want, tol = O.paged(q, kc, vc, table, lens.tolist(), pre, prefix)
    assert_within(got, want, tol)


def test_paged_long_prefix():
    g = gen(31)
    table, kc, vc = paged_setup(g, [3, 1, 60], 60, 1, 1, 64, 128)
    pre, table = table[2], table[:2]
    q = normal(g, 2, 40, 128)
    got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), table.to(DEV), ints([150, 0]), prefix=pre.to(DEV), prefix_len=3801)
    want, tol = O.paged(q[:, None], kc, vc, table, [150, 0], pre, 3801)
    assert_within(got, want[:, 0], tol[:, 0])


def test_paged_prefix_in_one_piece():
    """So many rows that a part of the prefix is longer than the 64 tiles whose places a wave holds at once."""
    heads, kv, dim, page, batch, q_len, prefix = 64, 8, 64, 64, 130, 4, 4230
    g = gen(23)
    n_pages = -(-prefix // page) + 3
    kc, vc = normal(g, n_pages, kv, page, dim), normal(g, n_pages, kv, page, dim)
    q = normal(g, batch, q_len, heads, dim)
    ids = torch.randperm(n_pages, generator=g)
    pre, own = ids[:-2].to(I32), ids[-1:].to(I32)
    lens = torch.zeros(batch, dtype=I32)
    lens[7] = 9
    table = own.repeat(batch, 1)
    got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), table.to(DEV), lens.to(DEV), prefix=pre.to(DEV), prefix_len=prefix)
    rows = [0, 7, 64, 129]
    want, tol = O.paged(q[rows], kc, vc, table[rows], lens[rows].tolist(), pre, prefix)
    assert_within(got[rows], want, tol)


@pytest.mark.parametrize("prefix", [0, 40])
def test_paged_bad_pages_and_lengths_show(prefix):
    """A page outside the cache or a length beyond the table: NaN rows of that sequence alone; no read outside."""
    g = gen(32)
    table, kc, vc = paged_setup(g, [4, 4, 4, 4, 3], 4, 0, 2, 16, 64)
    pre, table = table[4, :3], table[:4]
    bad = table.clone()
    bad[1, 2], bad[2, 0] = 1 << 30, -7
    lens = [50, 50, 64, 1 << 30]
    q = normal(g, 4, 4, 64)
    kw = dict(prefix=pre.to(DEV), prefix_len=prefix) if prefix else {}
    got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), bad.to(DEV), ints(lens), **kw)
    want, tol = O.paged(q[:, None], kc, vc, table, [50, 50, 64, 64], pre, prefix)
    assert_within(got[0], want[0, 0], tol[0, 0])
    assert got[1:].isnan().all()
    # the bad page lies behind the length: nobody asks for it
    got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), bad.to(DEV), ints([50, 32, 0, 64]), **kw)
    want, tol = O.paged(q[:, None], kc, vc, table, [50, 32, 0, 64], pre, prefix)
    assert_within(got, want[:, 0], tol[:, 0])
    if prefix:
        pre[1] = 1 << 20
        got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), table.to(DEV), ints([50] * 4), prefix=pre.to(DEV), prefix_len=prefix)
        assert got.isnan().all()


@pytest.mark.parametrize("dim,heads,q_len", [(64, 4, 3), (128, 2, 4), (128, 32, 2)])
@pytest.mark.parametrize("poison", [NAN, INF])
def test_paged_unseen_values_stay_unseen(dim, heads, q_len, poison):
    """In a verify step the last token's value must not reach the tokens before it."""
    g = gen(33)
    for n in (q_len, 32, 33, 130):
        table, kc, vc = paged_setup(g, [9], 9, 0, 1, 16, dim)
        q = normal(g, 1, q_len, heads, dim)
        want, tol = O.paged(q, kc, vc, table, [n])
        j = n - 1
        vc[table[0, j // 16], 0, j % 16, 9] = poison
        got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), table.to(DEV), ints([n])).cpu().double()
        assert ((got - want).abs() <= tol)[:, :-1].all()
        assert not torch.isfinite(got[0, -1, :, 9]).any()
        keep = torch.arange(dim) != 9
        assert ((got - want).abs() <= tol)[..., keep].all()


def test_paged_far_pages():
    """Pages beyond 2^31 elements and 2^32 bytes of the cache."""
    pages = (1 << 31) // (8 * 256 * 128) + 40
    kc, vc = (torch.empty((pages, 8, 256, 128), dtype=BF16, device=DEV) for _ in range(2))
    g = gen(34)
    ids = [pages - 1, pages // 2 + 1, 5]
    ks, vs = normal(g, 3, 8, 256, 128), normal(g, 3, 8, 256, 128)
    kc[ids], vc[ids] = ks.to(DEV), vs.to(DEV)
    k1, v1 = normal(g, 1, 8, 128), normal(g, 1, 8, 128)
    table = ints([[ids[1], ids[0]]])
    dsk_moe.kv_append(None, k1.to(DEV), v1.to(DEV), ints([300]), ints([0]), table, kc, vc, norm=False)
    ks[0, :, 44], vs[0, :, 44] = k1[0], v1[0]
    q = normal(g, 1, 8, 128)
    got = dsk_moe.paged_attention(q.to(DEV), kc, vc, table, ints([301]), prefix=ints([ids[2]]), prefix_len=200)
    want, tol = O.paged(q[:, None], ks, vs, torch.tensor([[1, 0]]), [301], torch.tensor([2]), 200)
    assert_within(got, want[:, 0], tol[:, 0])


@pytest.mark.parametrize("width", [8, 80])
def test_paged_views_and_scratch(width):
    """Strided queries and outputs; a workspace of the caller's, full of NaN, twice; a table row that one workgroup takes
    alone, and one that needs the workspace."""
    g = gen(35)
    table, kc, vc = paged_setup(g, [3, 7], width, 0, 2, 16, 64)
    dev = [x.to(DEV) for x in (kc, vc, table)]
    q = normal(g, 2, 2, 4, 64)
    qkv = torch.cat([q.flatten(2), normal(g, 2, 2, 256)], -1).to(DEV)
    view = qkv[..., :256].unflatten(2, (4, 64))
    out = torch.zeros((2, 2, 4, 128), dtype=BF16, device=DEV)[..., 64:]
    ws = torch.full((64 << 20,), 255, dtype=torch.uint8, device=DEV)
    want, tol = O.paged(q, kc, vc, table, [40, 111])
    for _ in range(2):
        got = dsk_moe.paged_attention(view, *dev, ints([40, 111]), out=out, workspace=ws)
        assert got is out
        assert_within(out, want, tol)
    with pytest.raises(_lib.DskError, match="DSK_ESPACE"):
        dsk_moe.paged_attention(view, *dev, ints([40, 111]), workspace=ws[:128 if width == 8 else 1024])


def test_same_call_same_bits():
    g = gen(36)
    table, kc, vc = paged_setup(g, [20, 3, 40, 9], 40, 0, 2, 16, 128)
    q = normal(g, 4, 8, 128).to(DEV)
    args = [x.to(DEV) for x in (kc, vc, table)] + [ints([320, 33, 640, 140])]
    want = dsk_moe.paged_attention(q, *args, prefix=args[2][2], prefix_len=600)
    for _ in range(5):
        assert torch.equal(dsk_moe.paged_attention(q, *args, prefix=args[2][2], prefix_len=600), want)


def test_refusals_on_the_device():
    g = gen(37)
    q, k = normal(g, 4, 8, 128).to(DEV), normal(g, 4, 2, 128).to(DEV)
    pos, cu = ints([0, 1, 2, 3]), ints([0, 4])
    kc, table, lens = torch.zeros(4, 2, 16, 128, dtype=BF16, device=DEV), ints([[0], [1], [2], [3]]), ints([1, 1, 1, 1])
    bad = [lambda: dsk_moe.qk_norm_rope(q, k, pos.long()), lambda: dsk_moe.qk_norm_rope(q, k.float(), pos),
           lambda: dsk_moe.qk_norm_rope(q, k, pos[:3]), lambda: dsk_moe.qk_norm_rope(q[..., ::2], k, pos),
           lambda: dsk_moe.qk_norm_rope(q, k, pos, torch.ones(64, device=DEV)), lambda: dsk_moe.qk_norm_rope(q.half(), k.half(), pos),
           lambda: dsk_moe.qk_norm_rope(q, k, pos, q_gamma=torch.ones(64, device=DEV)),
           lambda: dsk_moe.qk_norm_rope(q[:3], k, pos), lambda: dsk_moe.qk_norm_rope(q, k, pos.cpu()),
           lambda: dsk_moe.qk_norm_rope(q, k, pos, q_out=torch.empty_like(k)),
           lambda: dsk_moe.kv_append(q, k, k[:, :1], pos, pos, table, kc, kc), lambda: dsk_moe.kv_append(q, k, k, pos, pos, table, kc, kc[:, :1]),
           lambda: dsk_moe.kv_append(q, k, k, pos, pos, table.long(), kc, kc),
           lambda: dsk_moe.prompt_attention(q, k, k[:3], cu), lambda: dsk_moe.prompt_attention(q.float(), k, k, cu),
           lambda: dsk_moe.prompt_attention(q, k, k, cu, ints([0, 2, 4])), lambda: dsk_moe.prompt_attention(q, k, k, cu.long()),
           lambda: dsk_moe.paged_attention(q[:3], kc, kc, table, lens), lambda: dsk_moe.paged_attention(q, kc, kc, table, lens[:3]),
           lambda: dsk_moe.paged_attention(q, kc, kc, table, lens, prefix_len=3), lambda: dsk_moe.paged_attention(q, kc, kc, table, lens, prefix=lens),
           lambda: dsk_moe.paged_attention(q, kc, kc, table, lens, prefix=lens, prefix_len=65),
           lambda: dsk_moe.paged_attention(q, kc[..., :64], kc[..., :64], table, lens),
           lambda: dsk_moe.paged_attention(q, kc, kc, table, lens, workspace=torch.empty(9, device=DEV))]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("accepted", i)
    for f in (lambda: dsk_moe.prompt_attention(q[:, :7], k, k, cu), lambda: dsk_moe.prompt_attention(q, k, k, cu[:1]),
              lambda: dsk_moe.prompt_attention(q, k, k, cu, scale=-1.0),
              lambda: dsk_moe.paged_attention(q[:, None].expand(4, 17, 8, 128).contiguous(), kc, kc, table, lens)):
        with pytest.raises(_lib.DskError):
            f()


# ------------------------------------------------------------------ as a server runs them
class Server:
    """Four conversations behind a shared prefix: prompts, then steps of two tokens, on one cache."""

    def __init__(self, seed, dim=64, heads=8, kv=2, page=16, prefix=37):
        self.g = gen(seed)
        self.dim, self.heads, self.kv, self.page, self.prefix = dim, heads, kv, page, prefix
        self.freq = dsk_moe.rope_frequencies(dim // 2, device="cpu")[0]
        self.gq, self.gk = torch.rand(dim, generator=self.g) + 0.5, torch.rand(dim, generator=self.g) + 0.5
        self.shared = -(-prefix // page)
        self.table, kc, vc = paged_setup(self.g, [12, 12, 12, 12, self.shared], 12, 0, kv, page, dim, fill=NAN)
        self.pre = self.table[4, :self.shared]
        self.table = self.table[:4].contiguous()
        self.kc, self.vc = kc.to(DEV), vc.to(DEV)
        self.k = [torch.zeros(0, kv, dim, dtype=BF16) for _ in range(4)]     # as appended
        self.v = [torch.zeros(0, kv, dim, dtype=BF16) for _ in range(4)]

    def rows(self, t):
        return normal(self.g, t, (self.heads + 2 * self.kv) * self.dim)

    def split(self, qkv):
        return (p.unflatten(1, (-1, self.dim)) for p in qkv.split([self.heads * self.dim] + [self.kv * self.dim] * 2, 1))

    def append(self, qkv, pos, seq, table, prefix_len, k_out=None):
        q, k, v = self.split(qkv)
        return dsk_moe.kv_append(q, k, v, pos, seq, table, self.kc, self.vc, self.freq.to(DEV), prefix_len=prefix_len,
                                 q_gamma=self.gq.to(DEV), k_gamma=self.gk.to(DEV), k_out=k_out)


def test_prompts_then_decode_steps():
    """Shared prefix, packed prompts behind it, then two-token steps: the cache's reader sees what the appends wrote.
    Every output against attention in float64 over the rotated rows (rounded to bf16 as the cache holds them)."""
    s = Server(40)
    # the prefix as a prompt of its own
    qkv = s.rows(s.prefix)
    ar = torch.arange(s.prefix, dtype=I32, device=DEV)
    kp = torch.empty((s.prefix, s.kv, s.dim), dtype=BF16, device=DEV)
    q = s.append(qkv.to(DEV), ar, torch.zeros_like(ar), s.pre[None].to(DEV), 0, kp)
    vp = list(s.split(qkv))[2]
    got = dsk_moe.prompt_attention(q, kp, vp.to(DEV), ints([0, s.prefix]))
    want, tol = O.prompt(q.cpu(), kp.cpu(), vp, [0, s.prefix], [0, s.prefix])
    assert_within(got, want, tol, "prefix")
    # the prompts: keys and values of the prefix before their own
    lens = [5, 33, 1, 16]
    t, cu = sum(lens), cumulative(lens)
    qkv = s.rows(t)
    row = [i for n in lens for i in range(n)]
    seq = [b for b, n in enumerate(lens) for _ in range(n)]
    ko = torch.empty((t, s.kv, s.dim), dtype=BF16, device=DEV)
    q = s.append(qkv.to(DEV), ints([r + s.prefix for r in row]), ints(seq), s.table.to(DEV), s.prefix, ko)
    y, tol = O.norm_rope(list(s.split(qkv))[1], torch.tensor(row) + s.prefix, s.freq, gamma=s.gk)
    assert_within(ko, y, tol, "prompt keys")
    vo = list(s.split(qkv))[2]
    for b in range(4):
        s.k[b], s.v[b] = ko.cpu()[cu[b]:cu[b + 1]], vo[cu[b]:cu[b + 1]]
    kk = torch.cat([x for b in range(4) for x in (kp.cpu(), s.k[b])])
    vv = torch.cat([x for b in range(4) for x in (vp, s.v[b])])
    ck = cumulative([n + s.prefix for n in lens])
    got = dsk_moe.prompt_attention(q, kk.to(DEV), vv.to(DEV), ints(cu), ints(ck))
    want, tol = O.prompt(q.cpu(), kk, vv, cu, ck)
    assert_within(got, want, tol, "prompts")
    # steps of two tokens
    for step in range(3):
        at = [len(k) for k in s.k]
        qkv = s.rows(8)
        pos = ints([a + i + s.prefix for a in at for i in range(2)])
        ko = torch.empty((8, s.kv, s.dim), dtype=BF16, device=DEV)
        q = s.append(qkv.to(DEV), pos, ints([0, 0, 1, 1, 2, 2, 3, 3]), s.table.to(DEV), s.prefix, ko).view(4, 2, s.heads, s.dim)
        vo = list(s.split(qkv))[2]
        for b in range(4):
            s.k[b], s.v[b] = torch.cat([s.k[b], ko.cpu()[2 * b:2 * b + 2]]), torch.cat([s.v[b], vo[2 * b:2 * b + 2]])
        lens = [len(k) for k in s.k]
        got = dsk_moe.paged_attention(q, s.kc, s.vc, s.table.to(DEV), ints(lens), prefix=s.pre.to(DEV), prefix_len=s.prefix)
        for b in range(4):
            want, tol = O.attention(q[b].cpu(), torch.cat([kp.cpu(), s.k[b]]), torch.cat([vp, s.v[b]]),
                                    torch.tensor([s.prefix + lens[b] - 2, s.prefix + lens[b] - 1]), s.dim ** -0.5)
            assert_within(got[b], want, tol, f"step {step} sequence {b}")


@pytest.mark.parametrize("prefix", [0, 37])
def test_captured_steps_follow_the_lengths(prefix):
    """A decode step (append and attention) captured once and replayed while the sequences grow; a second graph of
    another batch between the replays, and eager work that must not disturb them."""
    def build(seed):
        s = Server(seed, prefix=prefix or 1)
        for c in (s.kc, s.vc):
            c.copy_(normal(s.g, *c.shape))
        st = dict(qkv=s.rows(4).to(DEV), pos=ints([0, 60, 15, 130]) + prefix, lens=ints([1, 61, 16, 131]), seq=ints([0, 1, 2, 3]),
                  table=s.table.to(DEV), pre=s.pre.to(DEV), freq=s.freq.to(DEV), gq=s.gq.to(DEV))

        def step():
            q, k, v = s.split(st["qkv"])
            q = dsk_moe.kv_append(q, k, v, st["pos"], st["seq"], st["table"], s.kc, s.vc, st["freq"], prefix_len=prefix, q_gamma=st["gq"])
            return dsk_moe.paged_attention(q, s.kc, s.vc, st["table"], st["lens"], prefix=st["pre"] if prefix else None, prefix_len=prefix)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        return s, st, step, graph, out

    one, two = build(41), build(42)
    for i in range(4):
        for s, st, step, graph, out in (one, two):
            st["qkv"].copy_(s.rows(4))
            st["pos"] += 1
            st["lens"] += 1
        for s, st, step, graph, out in (one, two):
            graph.replay()
        torch.cuda.synchronize()
        for s, st, step, graph, out in (one, two):
            held = out.clone()
            assert torch.equal(step(), held), i                  # the eager step writes the same rows again


@pytest.mark.parametrize("dim", [64, 128])
def test_captured_prompts_follow_their_bounds(dim):
    """A prompt step (norms, rotation, append, attention) captured once: replays on other rows and other bounds against
    the eager calls, with eager work between them."""
    g = gen(45)
    t, heads, kv = 700, 8, 2
    st = dict(qkv=normal(g, t, (heads + 2 * kv) * dim).to(DEV), pos=torch.zeros(t, dtype=I32, device=DEV),
              seq=torch.zeros(t, dtype=I32, device=DEV), cu=ints([0, t, t, t]), table=torch.arange(3 * 44, dtype=I32).view(3, 44).to(DEV))
    caches = [torch.zeros((140, kv, 16, dim), dtype=BF16, device=DEV) for _ in range(4)]
    freq, _ = dsk_moe.rope_frequencies(dim)

    def step(kc, vc):
        q, k, v = (p.unflatten(1, (-1, dim)) for p in st["qkv"].split([heads * dim, kv * dim, kv * dim], 1))
        kr = torch.zeros((t, kv, dim), dtype=BF16, device=DEV)
        q = dsk_moe.kv_append(q, k, v, st["pos"], st["seq"], st["table"], kc, vc, freq, k_out=kr, q_out=torch.zeros((t, heads, dim), dtype=BF16, device=DEV))
        return dsk_moe.prompt_attention(q, kr, v, st["cu"], out=torch.zeros_like(q))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*caches[:2])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*caches[:2])
    for lens in ([700, 0, 0], [1, 300, 399], [0, 0, 0], [64, 65, 63], [350, 350, 0]):
        n = sum(lens)
        st["qkv"].copy_(normal(g, *st["qkv"].shape))
        st["cu"].copy_(ints(cumulative(lens)))
        st["pos"].copy_(ints([i for m in lens for i in range(m)] + [-1] * (t - n)))
        st["seq"].copy_(ints([b for b, m in enumerate(lens) for _ in range(m)] + [0] * (t - n)))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        want = step(*caches[2:])
        assert torch.equal(got, want) and not got[n:].any(), lens
        assert all(torch.equal(a, b) for a, b in zip(caches[:2], caches[2:])), lens
        dsk_moe.prompt_attention(want[:50], want[:50, :kv].contiguous(), want[:50, :kv].contiguous(), ints([0, 20, 50]))   # eager work of another size


def test_calls_on_two_streams():
    """Concurrent calls on two streams, each with its own scratch memory."""
    g = gen(50)
    table, kc, vc = paged_setup(g, [30] * 8, 30, 0, 2, 16, 128)
    kc, vc, table, lens = kc.to(DEV), vc.to(DEV), table.to(DEV), ints([480, 3, 100, 250, 7, 480, 64, 128])
    q = [normal(g, 8, 8, 128).to(DEV) for _ in range(2)]
    want = [dsk_moe.paged_attention(x, kc, vc, table, lens) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(dsk_moe.paged_attention(q[i], kc, vc, table, lens))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


# ------------------------------------------------------------------ the stack
def make_decoder(seed, n=2, heads=8, kv=2, dim=64, pages=80, page=16):
    """A small MoE stack with attention sublayers (hidden 1024), and the same sublayers one by one."""
    from dsk_moe import synth as gsynth
    g = gen(seed)
    layers = [gsynth.make_layer(hidden=1024, n_experts=64, top_k=6, inter=512, inter_shared=512, seed=seed + l, device=DEV)
              for l in range(n)]
    freq, mscale = dsk_moe.rope_frequencies(dim, scaling="ramp", factor=2.0)
    att = []
    for _ in range(n):
        a = dsk_moe.Attention((normal(g, (heads + 2 * kv) * dim, 1024, dtype=F32) / 32).to(BF16).to(DEV),
                              (normal(g, 1024, heads * dim, dtype=F32) / 32).to(BF16).to(DEV), heads, kv, freq=freq,
                              mscale=mscale, q_gamma=(torch.rand(dim, generator=g) + 0.5).to(DEV),
                              k_gamma=(torch.rand(dim, generator=g) + 0.5).to(DEV))
        a.new_cache(pages, page)
        att.append(a)
    gam = [(torch.rand(1024, generator=g) + 0.5).to(DEV) for _ in range(2 * n)]
    return g, dsk_moe.MoEStack(layers, gammas=gam[:n], attention=att, attention_gammas=gam[n:])


def decoder_by_hand(stack, x, step):
    """The stack's composition from its public pieces, with the attention sublayer's own pieces apart."""
    h = x
    for l, layer in enumerate(stack.layers):
        a = stack.attention[l]
        y = dsk_moe.rmsnorm(h, stack.eps, stack.attention_gammas[l])
        qkv = torch.mm(y, a.w_qkv.t())
        q, k, v = (p.unflatten(1, (-1, a.head_dim)) for p in qkv.split([a.heads * a.head_dim] + [a.kv_heads * a.head_dim] * 2, 1))
        if isinstance(step, dsk_moe.PromptStep):
            kr = torch.empty_like(k, memory_format=torch.contiguous_format)
            q = dsk_moe.kv_append(q, k, v, step.positions, step.seq, step.table, a.k_cache, a.v_cache, k_out=kr, **a._rotate)
            o = dsk_moe.prompt_attention(q, kr, v, step.cu, out=torch.zeros_like(q))
        else:
            q = dsk_moe.kv_append(q, k, v, step.positions, step.seq, step.table, a.k_cache, a.v_cache,
                                  prefix_len=step.prefix_len, **a._rotate)
            o = dsk_moe.paged_attention(q.unflatten(0, (-1, step.q_len)), a.k_cache, a.v_cache, step.table, step.lens,
                                        prefix=step.prefix, prefix_len=step.prefix_len)
        d = torch.mm(o.reshape(x.shape[0], -1), a.w_o.t())
        h2, y = torch.empty_like(h), torch.empty_like(h)
        d = layer.forward_residual(h, d, h2, y, torch.empty_like(h), gamma=stack.gammas[l], eps=stack.eps)
        h = torch.empty_like(h)
        dsk_moe.rmsnorm(h2, stack.eps, residual=d, h_out=h, out=False)
    return h


def test_decoder_stack_prompts_and_steps():
    """Prompts, then steps of one and two tokens: the stack against its pieces, bit for bit."""
    g, stack = make_decoder(60)
    table = torch.randperm(60, generator=g)[:36].view(3, 12).to(I32).to(DEV)
    lens = [20, 1, 33]
    pos = ints([i for n in lens for i in range(n)] + [-1, -1])
    seq = ints([b for b, n in enumerate(lens) for _ in range(n)] + [0, 0])
    step = dsk_moe.PromptStep(pos, seq, table, ints(cumulative(lens)))
    x = normal(g, 56, 1024).to(DEV)
    got = stack(x, step=step).clone()
    assert torch.equal(got, decoder_by_hand(stack, x, step)) and torch.isfinite(got.float()).all()
    for q_len in (1, 2, 1):
        pos = ints([n + i for n in lens for i in range(q_len)])
        lens = [n + q_len for n in lens]
        step = dsk_moe.DecodeStep(pos, ints([b for b in range(3) for _ in range(q_len)]), table, ints(lens), q_len)
        x = normal(g, 3 * q_len, 1024).to(DEV)
        got = stack(x, step=step).clone()
        assert torch.equal(got, decoder_by_hand(stack, x, step)) and torch.isfinite(got.float()).all()


def test_decoder_steps_agree_with_the_prompt():
    """A prompt in one piece, and its last tokens in decode steps: the same attention over the same cache rows.  One
    layer without experts' routing in between: its attention output, within the roundings of both."""
    g, stack = make_decoder(61, n=1)
    a = stack.attention[0]
    table = torch.arange(12, dtype=I32, device=DEV)[None]
    y = normal(g, 40, 1024).to(DEV)
    ar = torch.arange(40, dtype=I32, device=DEV)
    zero = torch.zeros_like(ar)
    qkv = torch.mm(y, a.w_qkv.t())
    q, k, v = (p.unflatten(1, (-1, 64)) for p in qkv.split([512, 128, 128], 1))
    kr = torch.empty((40, 2, 64), dtype=BF16, device=DEV)
    q = dsk_moe.kv_append(q, k, v, ar, zero, table, a.k_cache, a.v_cache, k_out=kr, **a._rotate)
    want, tol = O.prompt(q.cpu(), kr.cpu(), v.cpu(), [0, 40], [0, 40])
    assert_within(dsk_moe.prompt_attention(q, kr, v, ints([0, 40])), want, tol, "prompt")
    for i in range(30, 40):
        got = dsk_moe.paged_attention(q[i:i + 1], a.k_cache, a.v_cache, table, ints([i + 1]))
        assert_within(got, want[i:i + 1], tol[i:i + 1], f"token {i}")


@pytest.mark.parametrize("prefix", [0, 25])
def test_captured_decoder(prefix):
    """A decode step of the stack as a graph: replays follow the step's positions and lengths, against the eager stack,
    with eager prompts between them; an unused slot stays out of it."""
    g, stack = make_decoder(62)
    for a in stack.attention:
        for c in (a.k_cache, a.v_cache):
            c.copy_(normal(g, *c.shape))
    table = torch.randperm(70, generator=g)[:48].view(4, 12).to(I32).to(DEV)
    pre = torch.arange(70, 72, dtype=I32, device=DEV)
    other = torch.randperm(70, generator=g)[:12].view(1, 12).to(I32).to(DEV)
    pos, lens = ints([3, 100, -1, 17]), ints([4, 101, -1, 18])
    pos[pos >= 0] += prefix
    step = dsk_moe.DecodeStep(pos, ints([0, 1, 2, 3]), table, lens, 1, pre if prefix else None, prefix)
    stack.capture(4, step=step)
    for rep in range(4):
        live = lens >= 0
        pos[live] += 1
        lens[live] += 1
        x = normal(g, 4, 1024).to(DEV)
        x[2] = 0
        held = [(a.k_cache.clone(), a.v_cache.clone()) for a in stack.attention]
        got = stack.replay(x).clone()
        torch.cuda.synchronize()
        after = [(a.k_cache.clone(), a.v_cache.clone()) for a in stack.attention]
        for a, (k, v) in zip(stack.attention, held):
            a.k_cache.copy_(k)
            a.v_cache.copy_(v)
        want = stack(x, step=step)
        assert torch.equal(got, want), rep
        assert torch.isfinite(got.float()).all()
        for a, (k, v) in zip(stack.attention, after):
            assert torch.equal(a.k_cache, k) and torch.equal(a.v_cache, v)
        # an eager prompt of another size, on pages of its own kind, in between
        ar = torch.arange(9, dtype=I32, device=DEV)
        stack(normal(g, 9, 1024).to(DEV), step=dsk_moe.PromptStep(ar, torch.zeros_like(ar), other, ints([0, 9])))


def test_decoder_refuses():
    g, stack = make_decoder(63, n=1)
    x = normal(g, 1, 1024).to(DEV)
    with pytest.raises(ValueError, match="go together"):
        stack(x)
    with pytest.raises(ValueError, match="go together"):
        dsk_moe.MoEStack(stack.layers)(x, step=dsk_moe.DecodeStep(None, None, None, None))
    with pytest.raises(ValueError, match="sublayers for"):
        dsk_moe.MoEStack(stack.layers, attention=[])
    a = stack.attention[0]
    with pytest.raises(ValueError, match="bfloat16"):
        a(x.float(), None)
    b = dsk_moe.Attention(a.w_qkv, a.w_o, 8, 2)
    with pytest.raises(RuntimeError, match="new_cache"):
        b(x, None)
    for heads, kv in ((8, 3), (7, 7), (0, 0)):
        with pytest.raises(ValueError):
            dsk_moe.Attention(a.w_qkv, a.w_o, heads, kv)


@pytest.mark.parametrize("width,prefix", [(16, 0), (80, 0), (16, 50)])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_shows_an_infinite_value_as_it_is(dim, width, prefix):
    """One token a sequence: an infinite value among its last keys gives that infinity whatever the length leaves
    empty of the last 32 keys, a NaN gives NaN, and the other elements stay as they were."""
    g = gen(38 + dim)
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 48, 100, 127, 128, 129, 190]
    used = [-(-n // 16) for n in lens]
    table, kc, vc = paged_setup(g, used + [4], max(max(used), width), 0, 1, 16, dim)
    pre, table = table[-1, :4], table[:-1]
    q = normal(g, len(lens), 4, dim)
    want, tol = O.paged(q[:, None], kc, vc, table, lens, pre, prefix)
    want, tol = want[:, 0], tol[:, 0]
    for b, n in enumerate(lens):                                 # at the last key, and one before it
        for j, at, x in ((n - 1, 3, INF), (n - 1, 9, -INF), (n - 1, 20, NAN), (max(0, n - 2), 5, INF)):
            vc[table[b, j // 16], 0, j % 16, at] = x
    for at, x in ((3, INF), (9, -INF), (20, NAN), (5, INF)):
        want[..., at] = x
    got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), table.to(DEV), ints(lens),
                                  prefix=pre.to(DEV) if prefix else None, prefix_len=prefix).cpu().double()
    assert torch.equal(got[..., [3, 5, 9]], want[..., [3, 5, 9]])
    assert got[..., 20].isnan().all()
    rest = [i for i in range(dim) if i not in (3, 5, 9, 20)]
    assert ((got - want).abs() <= tol)[..., rest].all()


def test_capture_leaves_the_cache_alone():
    """Prompts, then a captured decode step, as documented: the capture keeps nothing in the caches, and the replays follow
    the eager steps bit for bit.  An unused slot's table row names the page of a live sequence, which stays as it is."""
    g, stack = make_decoder(64)
    table = (torch.randperm(60, generator=g)[:48].view(4, 12) + 1).to(I32)
    table[0, 0], table[2] = 0, 0                                  # slot 2 is unused; page 0 is sequence 0's first
    table = table.to(DEV)
    rows = [20, 1, 0, 33]
    ar = torch.cat([torch.arange(n) for n in rows]).to(I32).to(DEV)
    seq = torch.repeat_interleave(torch.arange(4), torch.tensor(rows)).to(I32).to(DEV)
    stack(normal(g, 54, 1024).to(DEV), step=dsk_moe.PromptStep(ar, seq, table, ints(cumulative(rows))))
    caches = [c for a in stack.attention for c in (a.k_cache, a.v_cache)]
    held = [c.clone() for c in caches]
    xs = [normal(g, 4, 1024).to(DEV) for _ in range(3)]

    def fresh():
        return dsk_moe.DecodeStep(ints([19, 0, -1, 32]), ints([0, 1, 2, 3]), table, ints([20, 1, -1, 33]))

    def advance(step):
        live = (step.lens >= 0).int()
        step.positions += live
        step.lens += live

    step, want = fresh(), []
    for x in xs:
        advance(step)
        want.append(stack(x, step=step).clone())
    after = [c.clone() for c in caches]
    for c, h in zip(caches, held):
        c.copy_(h)
    step = fresh()
    stack.capture(4, step=step)
    torch.cuda.synchronize()
    assert all(torch.equal(c, h) for c, h in zip(caches, held)), "the capture wrote to the cache"
    assert step.positions.tolist() == [19, 0, -1, 32] and step.lens.tolist() == [20, 1, -1, 33]
    for x, w in zip(xs, want):
        advance(step)
        assert torch.equal(stack.replay(x), w)
        torch.cuda.synchronize()
    assert all(torch.equal(c, a) for c, a in zip(caches, after))


@pytest.mark.parametrize("width,prefix", [(6, 0), (80, 0), (6, 33)])
def test_paged_rows_that_need_no_bad_page(width, prefix):
    """Of a verify step's tokens, those that see a key on a page outside the cache are NaN; those before them are not,
    and those that see no key are zero."""
    g = gen(39)
    n, q_len = [50, 48, 2, 83], 4
    table, kc, vc = paged_setup(g, [6, 6, 6, 6, 3], max(width, 6), 0, 2, 16, 64)
    pre, table = table[-1, :3], table[:-1]
    bad = table.clone()
    bad[0, 3], bad[1, 2], bad[2, 0], bad[3, 5], bad[3, 1] = 1 << 30, -1, 99, 1 << 20, -5
    q = normal(g, 4, q_len, 6, 64)
    kw = dict(prefix=pre.to(DEV), prefix_len=prefix) if prefix else {}
    got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), bad.to(DEV), ints(n), **kw)
    want, tol = O.paged(q, kc, vc, table, n, pre, prefix)
    needs = torch.tensor([[False, False, True, True], [True] * 4, [False, False, True, True], [True] * 4])
    assert got[needs.to(DEV)].isnan().all()
    assert_within(got.cpu()[~needs], want[~needs], tol[~needs])
    if not prefix:
        assert not got[2, :2].any()


# ------------------------------------------------------------------ the weights' sum
def constant_values(g, dim, n, special):
    """(q [64, 2, dim], k [n, 1, dim], v [1, 1, dim]): all keys but one score 0 and that one x, up to 8, for the first head's rows
    (scale ln 2), a little more or less for the second's.  Its weight is 2^x beside the others' 1, so the reference point of the exponentials
    stays where they have put it."""
    v = normal(g, 1, 1, dim)
    v[..., :8] = torch.tensor([1.9921875, 1.0, 1.0078125, 1.984375, -1.9921875, 255.0, 0.49609375, 3.984375])
    k = torch.zeros(n, 1, dim, dtype=BF16)
    k[special, 0, 0] = 1.0
    q = torch.zeros(64, 2, dim, dtype=BF16)
    q[:, 0, 0] = torch.linspace(0.1, 7.9, 64).to(BF16)
    q[:, 1] = normal(g, 64, dim) * 0.2
    return q, k, v


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,special", [(65, 64), (200, 128), (700, 650)])
def test_prompt_gives_constant_values_as_they_are(dim, n, special):
    """Where every visible value is the same, so is the result, bit for bit, whatever the weights: their sum is that of
    the weights as the product uses them.  (Sums in float32 are off by less than 2 n 2^-24, far below the half step of
    2^-9 that would change a bf16.)"""
    q, k, v = constant_values(gen(52), dim, n, special)
    got = dsk_moe.prompt_attention(q.to(DEV), k.to(DEV), v.expand(n, 1, dim).contiguous().to(DEV), ints([0, 64]), ints([0, n]),
                                   causal=False, scale=math.log(2.0))
    assert torch.equal(got.cpu(), v.expand(64, 2, dim))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,special", [(65, 64), (200, 128), (700, 650)])
@pytest.mark.parametrize("wide,prefix", [(False, False), (True, False), (False, True)])
def test_paged_gives_constant_values_as_they_are(dim, n, special, wide, prefix):
    q, k, v = constant_values(gen(53), dim, n, special)
    pages = -(-n // 16)
    kc = torch.zeros(pages, 1, 16, dim, dtype=BF16)
    kc[special // 16, 0, special % 16] = k[special, 0]
    vc = v.view(1, 1, 1, dim).expand(pages, 1, 16, dim).contiguous()
    table = torch.zeros(64, 100 if wide else pages, dtype=I32)
    table[:, :pages] = torch.arange(pages)
    pre = dict(prefix=torch.arange(pages, dtype=I32).to(DEV), prefix_len=n) if prefix else {}
    got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), table.to(DEV), ints([3 if prefix else n] * 64), scale=math.log(2.0), **pre)
    assert torch.equal(got.cpu(), v.expand(64, 2, dim))


@pytest.mark.parametrize("heads,kv,dim,q_len,width,lens", [(8, 2, 128, 1, 40, [1, 2, 33, 500, 639]), (4, 1, 64, 2, 40, [2, 3, 33, 500, 639]),
                                                          (4, 2, 128, 1, 400, [1, 2, 33, 500, 6000]), (40, 1, 64, 1, 400, [1, 2, 33, 500, 6000])])
def test_paged_weights_keep_their_digits(heads, kv, dim, q_len, width, lens):
    """Own keys: the weights enter the product with 2^-16 of each at most left out, so the result's own rounding is nearly
    all of the error (the float32 sums as in the oracle's tolerance)."""
    g = gen(54 + dim)
    table, kc, vc = paged_setup(g, [-(-n // 16) for n in lens], width, 0, kv, 16, dim)
    q = normal(g, len(lens), q_len, heads, dim)
    got = dsk_moe.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), table.to(DEV), ints(lens)).cpu().double()
    want, tol = O.paged(q, kc, vc, table, lens)
    # without the 2^-8 of each weight that the oracle allows
    size = O.paged(q, kc, vc.abs(), table, lens)[0]
    assert ((got - want).abs() <= tol - size * (2.0 ** -8 - 2.0 ** -16)).all()


def test_numbers_given_as_tensors_are_read_at_every_call():
    g = gen(51)
    q, k = normal(g, 5, 2, 64).to(DEV), normal(g, 5, 2, 64).to(DEV)
    pos, cu, freq = torch.arange(5, dtype=I32, device=DEV), ints([0, 5]), dsk_moe.rope_frequencies(64)[0]
    table, lens = ints([[0]]), ints([5])
    cache = normal(g, 1, 2, 16, 64).to(DEV)
    number = torch.tensor(1.0)
    for x in (1.0, 0.25):
        number.fill_(x)
        for a, b in zip(dsk_moe.qk_norm_rope(q, k, pos, freq, mscale=number), dsk_moe.qk_norm_rope(q, k, pos, freq, mscale=x)):
            assert torch.equal(a, b), x
        for a, b in zip(dsk_moe.qk_norm_rope(q, k, pos, freq, eps=number), dsk_moe.qk_norm_rope(q, k, pos, freq, eps=x)):
            assert torch.equal(a, b), x
        assert torch.equal(dsk_moe.prompt_attention(q, k, k, cu, scale=number), dsk_moe.prompt_attention(q, k, k, cu, scale=x)), x
        assert torch.equal(dsk_moe.paged_attention(q[:1], cache, cache, table, lens, scale=number),
                           dsk_moe.paged_attention(q[:1], cache, cache, table, lens, scale=x)), x


def test_prompt_step_of_a_part_of_a_prompt_is_refused():
    """The sublayer's prompts attend over their own keys alone: a step that starts behind kept keys would leave those out."""
    seq, table = ints([0, 0, 0, 1, 1, 0]), ints([[0, 1], [2, 3]])

    def step(pos, cu):
        return dsk_moe.PromptStep(ints(pos), seq, table, ints(cu))

    step([0, 1, 2, 0, 1, -1], [0, 3, 5])
    step([0, 1, 2, 0, 1, -1], [0, 0, 3, 3, 5, 5])
    step([-1, 0, 1, 0, 1, -1], [1, 3, 5])
    step([-1] * 6, [0, 0, 0])
    for pos, cu in (([7, 8, 9, 0, 1, -1], [0, 3, 5]), ([0, 1, 2, 16, 17, -1], [0, 3, 5]), ([0, 2, 1, 0, 1, -1], [0, 3, 5]),
                    ([0, 1, -1, 0, 1, -1], [0, 3, 5]), ([0, 1, 2, 0, 1, 2], [0, 3, 5]), ([0, 1, 2, 0, 1, -1], [0, 3, 6]),
                    ([0, 1, 2, 0, 1, -1], [0, 3, 7]), ([0, 1, 2, 0, 1, -1], [0, 3, 2]), ([0, 1, 2, 0, 1, -1], [-1, 3, 5]),
                    ([0, 1, 2, 0, 1, -1], [1, 3, 5])):
        with pytest.raises(ValueError, match="whole prompts"):
            step(pos, cu)


def test_replay_with_another_cache_is_refused():
    """A graph writes to the caches that its layers had: a layer's new one needs a new capture."""
    g, stack = make_decoder(65, n=1)
    step = dsk_moe.DecodeStep(ints([0]), ints([0]), ints([[0]]), ints([1]))
    x = normal(g, 1, 1024).to(DEV)
    stack.capture(1, step=step)
    want = stack.replay(x).clone()
    stack.attention[0].new_cache(4, 16)
    with pytest.raises(RuntimeError, match="capture"):
        stack.replay(x)
    stack.capture(1, step=step)
    assert torch.equal(stack.replay(x), want) and stack.attention[0].k_cache[0, :, 0].any()


def test_two_captured_decoders_at_once():
    """Two stacks' graphs replayed on two streams at the same time: each gives what it gives alone."""
    stacks = []
    for seed in (70, 71):
        g, stack = make_decoder(seed)
        for a in stack.attention:
            for c in (a.k_cache, a.v_cache):
                c.copy_(normal(g, *c.shape))
        table = torch.randperm(70, generator=g)[:48].view(4, 12).to(I32).to(DEV)
        stack.capture(4, step=dsk_moe.DecodeStep(ints([3, 100, 40, 17]), ints([0, 1, 2, 3]), table, ints([4, 101, 41, 18])))
        x = normal(g, 4, 1024).to(DEV)
        stacks.append((stack, x, stack.replay(x).clone()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for (stack, x, _), s in zip(stacks, streams):
            with torch.cuda.stream(s):
                for _ in range(3):
                    stack.replay(x)
        torch.cuda.synchronize()
        for stack, x, want in stacks:
            assert torch.equal(stack._out, want)


def test_failed_capture_leaves_no_graph():
    """A capture that raises has replaced the buffers that an earlier graph used: there is nothing to replay then."""
    g, stack = make_decoder(66, n=1)
    step = dsk_moe.DecodeStep(ints([0]), ints([0]), ints([[0]]), ints([1]))
    x = normal(g, 1, 1024).to(DEV)
    stack.capture(1, step=step)
    want = stack.replay(x).clone()
    torch.cuda.synchronize()
    with pytest.raises(ValueError):
        stack.capture(2, step=step)                              # two rows for one sequence
    with pytest.raises(RuntimeError, match="capture"):
        stack.replay()
    stack.capture(1, step=step)
    assert torch.equal(stack.replay(x), want)


def test_captured_prompts_of_the_stack():
    """A prompt step captured: nothing is kept by the capture; replays follow the step's tensors, against the eager stack."""
    g, stack = make_decoder(67)
    caches = [c for a in stack.attention for c in (a.k_cache, a.v_cache)]
    table = torch.randperm(60, generator=g)[:24].view(2, 12).to(I32).to(DEV)
    step = dsk_moe.PromptStep(ints(list(range(20)) + [-1] * 20), ints([0] * 20 + [1] * 20), table, ints([0, 20, 20]))
    stack.capture(40, step=step)
    torch.cuda.synchronize()
    assert not any(c.any() for c in caches)
    for a, b in ((20, 20), (1, 30), (37, 0)):
        step.positions.copy_(ints(list(range(a)) + list(range(b)) + [-1] * (40 - a - b)))
        step.seq.copy_(ints([0] * a + [1] * (40 - a)))
        step.cu.copy_(ints([0, a, a + b]))
        x = normal(g, 40, 1024).to(DEV)
        for c in caches:
            c.zero_()
        got = stack.replay(x).clone()
        torch.cuda.synchronize()
        held = [c.clone() for c in caches]
        for c in caches:
            c.zero_()
        want = stack(x, step=step)
        assert torch.equal(got, want) and all(torch.equal(c, h) for c, h in zip(caches, held))


def test_decoder_refuses_gammas_without_their_sublayers():
    g, stack = make_decoder(68, n=2)
    for kw in (dict(attention_gammas=stack.attention_gammas), dict(attention=stack.attention, attention_gammas=stack.attention_gammas[:1])):
        with pytest.raises(ValueError, match="attention_gammas"):
            dsk_moe.MoEStack(stack.layers, **kw)


def test_replay_of_a_step_with_other_tensors_is_refused():
    """A graph reads the tensors that its step had: new ones in the step would not be seen."""
    g, stack = make_decoder(69, n=1)
    step = dsk_moe.DecodeStep(ints([0]), ints([0]), ints([[0]]), ints([1]))
    x = normal(g, 1, 1024).to(DEV)
    stack.capture(1, step=step)
    stack.replay(x)
    held = step.positions
    step.positions = step.positions + 1
    with pytest.raises(RuntimeError, match="other tensors"):
        stack.replay(x)
    step.positions = held
    held += 1
    step.lens += 1
    got = stack.replay(x).clone()
    assert torch.equal(got, stack(x, step=step))
