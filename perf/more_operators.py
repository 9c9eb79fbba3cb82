"""What a decoder's key / value cache is asked for beside plain bfloat16 rows, as cases that can be timed and compared.

A case is one call of ``qk_norm_rope`` with positions on several axes, ``kv_append`` to a
cache held in 8 bits, ``paged_attention`` over such a cache, ``paged_attention`` that
also sums up the weight that every key received, or ``kv_evict``, which keeps the keys
of most weight.  Heads of 128 with 32 query and 8 key heads fit the hidden size of
4096 that the layers here are benchmarked with; the others are generic.

A cache in 8 bits: e4m3 codes [pages, key heads, page size, dim] and a scale 2^(b - 127) for every
16 rows of a page and head, [pages, key heads, page size / 16] bytes b.  A block's scale is the least
that holds its largest magnitude (at most 448 times the scale); rows that come to a block which
has some take the larger of its scale and theirs, and the rows there are rounded to it; a call
that brings a block's first row starts it afresh.

``run`` computes either the plain form (elementary torch operations in float32, angles
in float64) or calls the package; ``exact`` is the definition in float64, sequence by
sequence.
"""

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False
DEV = "cuda"
EPS = 1e-6
BLOCK = 16                          # rows of a page that share a scale
LEAST, MOST = 27, 246               # scale bytes that are given out
F8, U8, BF16, F32, F64 = torch.float8_e4m3fn, torch.uint8, torch.bfloat16, torch.float32, torch.float64
_PKG = str(Path(__file__).resolve().parent.parent / "deepseeker-v4.1_amd")


def _package():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import dsk_moe
    return dsk_moe


# ------------------------------------------------------------------ cases
def _rope(name, tokens, heads, kv_heads, dim, rot, axes, each=False, in_turn=False, interleaved=False, dtype="bf16"):
    return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "axes": axes, "each": each, "in_turn": in_turn, "interleaved": interleaved, "dtype": dtype}


def _append(name, seqs, tokens, heads, kv_heads, dim, rot, page, axes=1, dtype="bf16", far=900):
    return {"name": name, "op": "append", "seqs": seqs, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rot": rot, "axes": axes, "each": False, "in_turn": False, "interleaved": False, "page": page, "dtype": dtype, "far": far}


def _paged(name, batch, q_len, longest, heads, kv_heads, dim, page, prefix=0, empty=False):
    return {"name": name, "op": "paged", "batch": batch, "q_len": q_len, "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "prefix": prefix, "empty": empty, "cache": "e4m3"}


def _weigh(name, batch, q_len, longest, heads, kv_heads, dim, page, cache):
    return {**_paged(name, batch, q_len, longest, heads, kv_heads, dim, page), "op": "weigh", "cache": cache}


def _evict(name, batch, longest, keep, first, recent, kv_heads, dim, page, cache, same=False):
    return {"name": name, "op": "evict", "batch": batch, "longest": longest, "keep": keep, "first": first, "recent": recent,
            "kv_heads": kv_heads, "dim": dim, "page": page, "cache": cache, "same": same}


def listed():
    return [
        # a small image's patches, float32, a bank of frequencies for each of its two axes
        _rope("axes_196", 196, 12, 12, 64, 64, 2, each=True, interleaved=True, dtype="f32"),
        # a video with text before it: time, height and width share one bank of frequencies
        _rope("axes_8192", 8192, 32, 8, 128, 128, 3),
        # one token of each conversation of a full decode batch is kept
        _append("append8_64", 64, 64, 32, 8, 128, 128, 64),
        # a prefill step: packed prompts with pictures, behind what their conversations hold already
        _append("append8_8192", 13, 8192, 32, 8, 128, 128, 64, axes=3),
        # one token of one short conversation, all latency
        _paged("paged8_1", 1, 1, 517, 32, 8, 128, 64),
        # a full decode batch of ragged conversations, one slot of it unused
        _paged("paged8_64", 64, 1, 8192, 32, 8, 128, 64, empty=True),
        # a two-token verify step of few long conversations, small pages
        _paged("paged8_8x2", 8, 2, 32768, 16, 4, 64, 16),
        # a full batch that shares a long document
        _paged("paged8_prefix", 64, 1, 600, 32, 8, 128, 64, prefix=16385),
        # a decode step over caches of bounded size that are evicted from
        _weigh("weigh_48", 48, 1, 2100, 32, 8, 128, 64, "bf16"),
        # the last 16 tokens of long prompts say which of their keys to keep
        _weigh("weigh8_4x16", 4, 16, 8000, 32, 8, 128, 64, "e4m3"),
        # a batch of full caches makes room for the next 64 tokens
        _evict("evict_64", 64, 1088, 1024, 4, 128, 8, 128, 64, "bf16", same=True),
        # long prompts are cut down to what a conversation may keep
        _evict("evict8_4", 4, 16000, 2000, 4, 250, 8, 128, 64, "e4m3"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 4, 128), (16, 4, 64), (12, 12, 64), (40, 5, 128), (24, 8, 64)])
    page = rng.choice([16, 32, 64, 128])
    rot = rng.choice([dim, dim, dim // 2])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    cache = rng.choice(["bf16", "e4m3"])
    op = rng.choice(["rope", "append", "append", "paged", "paged", "prefix", "weigh", "evict", "evict"])
    if op == "rope":
        c = _rope("", log_int(1, 8192), heads, kv_heads, dim, rot, rng.choice([2, 3, 4]), rng.random() < 0.5, rng.random() < 0.5,
                  rng.random() < 0.5, dtype)
    elif op == "append":
        tokens = log_int(1, 8192)
        c = _append("", min(tokens, log_int(1, 64)), tokens, heads, kv_heads, dim, rot, page, rng.choice([1, 1, 3]), dtype)
    elif op == "evict":
        batch = log_int(1, 64)
        longest = log_int(20, min(16000, 131072 // batch))
        keep = rng.randint(10, longest - 1)
        c = _evict("", batch, longest, keep, rng.randint(0, min(8, keep // 4)), rng.randint(0, keep // 2), kv_heads, dim, page, cache,
                   rng.random() < 0.5)
    else:
        batch = log_int(1, 64)
        q_len = rng.choice([1, 1, 1, 2, 4, 8])
        longest = log_int(q_len, min(32768, 524288 // batch))
        if op == "weigh":
            c = _weigh("", batch, q_len, max(q_len, longest // 2), heads, kv_heads, dim, page, cache)
        else:
            c = _paged("", batch, min(q_len, 4), longest, heads, kv_heads, dim, page, log_int(64, 16384) if op == "prefix" else 0,
                       rng.random() < 0.3)
    c.pop("name")
    return c


# ------------------------------------------------------------------ inputs
def _lengths(rng, n, longest):
    """n lengths of 1 to longest, spread over their logarithm, one of them the longest."""
    got = [min(longest, max(1, int(round(math.exp(rng.uniform(0.0, math.log(longest + 0.5))))))) for _ in range(n)]
    got[rng.randrange(n)] = longest
    return got


def _lens_of(case):
    """The case's lengths: they belong to the case, so that its work is the same for every seed."""
    rng = random.Random(19)
    if case["op"] == "evict":
        if case["same"]:
            return [case["longest"]] * case["batch"]
        got = [rng.randint(max(1, case["keep"] // 2), case["longest"]) for _ in range(case["batch"])]
        got[rng.randrange(len(got))] = case["longest"]
        return got
    if case["op"] == "append":
        cuts = sorted(rng.sample(range(1, case["tokens"]), case["seqs"] - 1)) if case["seqs"] > 1 else []
        return [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
    got = [max(case["q_len"], v) for v in _lengths(rng, case["batch"], case["longest"])]
    if case["empty"]:
        got[got.index(min(got))] = 0
    return got


def _axis_of(case):
    """The axis of every pair: in turn, or a run for each (of three axes the first has a quarter)."""
    pairs, n = case["rot"] // 2, case["axes"]
    if case["in_turn"]:
        return [i % n for i in range(pairs)]
    first = pairs // 4 if n == 3 else -(-pairs // n)
    return [0 if i < first else 1 + (i - first) * (n - 1) // (pairs - first) for i in range(pairs)]


def _frequencies(case):
    axis = _axis_of(case)
    if case["each"]:                # a bank for each axis
        part = [axis[:i].count(a) / axis.count(a) for i, a in enumerate(axis)]
    else:
        part = [i / len(axis) for i in range(len(axis))]
    return torch.tensor([10000.0 ** -p for p in part], dtype=F64, device=DEV)


def _places(case, n, start):
    """n tokens from `start` on: text, whose axes all count the same, and behind it pictures of 16 columns."""
    at = np.arange(n)
    text = n // 5
    grid = np.stack([text + (at - text) // 256, text + (at - text) // 16 % 16, text + (at - text) % 16, text + (at - text) // 4096])
    return start + np.where(at < text, at, grid)[:case["axes"]]


def _pages(gen, table_pages, spare):
    """A shuffled assignment of table_pages pages out of table_pages + spare."""
    return torch.randperm(table_pages + spare, generator=gen, device=DEV)[:table_pages].to(torch.int32)


def _scale_byte(top):
    """The least scale, as its byte, that holds the float32 magnitudes `top`."""
    m, e = torch.frexp(top)
    return (e - 9 + (m > 0.875).to(e.dtype) + 127).clamp(LEAST, MOST)


def _power(byte):
    return torch.exp2((byte.to(F32) - 127.0))


def _to_codes(x, byte):
    """float32 x in codes of the scale of `byte`."""
    return (x / _power(byte)).clamp(-448.0, 448.0).to(F8)


def _cache(case, pages, normal):
    """(codes, scales) of standard normal rows whose blocks differ in size, or bfloat16 rows."""
    kv, page, dim = case["kv_heads"], case["page"], case["dim"]
    x = normal(pages, kv, page // BLOCK, BLOCK, dim)
    if case["op"] != "append" and case["cache"] == "bf16":
        return x.view(pages, kv, page, dim).to(BF16), None
    x *= torch.exp2(normal(pages, kv, page // BLOCK, 1, 1) * 0.5)
    byte = _scale_byte(x.abs().amax((-1, -2)))
    return _to_codes(x, byte[..., None, None]).view(pages, kv, page, dim), byte.to(U8)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    rng = random.Random(int(seed))
    dim, kv = case["dim"], case["kv_heads"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    def ints(v):
        return torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)

    s = {"case": dict(case)}
    if case["op"] in ("rope", "append"):
        t, heads = case["tokens"], case["heads"]
        # the three are views of one projection's rows
        qkv = normal(t, (heads + 2 * kv) * dim).to(BF16 if case["dtype"] == "bf16" else F32)
        s["q"], s["k"], s["v"] = (p.unflatten(1, (-1, dim)) for p in qkv.split([heads * dim, kv * dim, kv * dim], 1))
        s["q_gamma"], s["k_gamma"] = (1.0 + 0.1 * normal(dim) for _ in range(2))
        s["freq"] = _frequencies(case)
        s["axis"] = ints(_axis_of(case)) if case["axes"] > 1 else None
    if case["op"] == "rope":
        s["pos"] = ints(_places(case, t, rng.randint(0, 500)))
        return s
    lens, page = _lens_of(case), case["page"]
    shared = 0
    if case["op"] == "append":
        where = random.Random(20)
        starts = [where.randint(0, case["far"]) for _ in lens]
        s["rows"] = ints([a + i for a, n in zip(starts, lens) for i in range(n)])
        s["seq"] = ints([b for b, n in enumerate(lens) for _ in range(n)])
        s["pos"] = ints(np.concatenate([_places(case, n, a) for a, n in zip(starts, lens)], 1))
        if case["axes"] == 1:
            s["pos"], s["rows"] = s["rows"], None     # a position is the row as well
        ends = [a + n for a, n in zip(starts, lens)]
    else:
        ends = lens
        s["lens"] = ints(lens)
        shared = -(-case.get("prefix", 0) // page)
    used = [-(-v // page) for v in ends]
    ids = _pages(gen, sum(used) + shared, 3)
    s["prefix"] = ids[:shared].contiguous()
    s["table"] = torch.zeros((len(lens), max(used) + 1), dtype=torch.int32, device=DEV)
    s["table"][torch.arange(max(used) + 1, device=DEV)[None] < torch.tensor(used, device=DEV)[:, None]] = ids[shared:]
    pages = sum(used) + shared + 3
    s["k_cache"], s["k_scale"] = _cache(case, pages, normal)
    s["v_cache"], s["v_scale"] = _cache(case, pages, normal)
    if case["op"] in ("paged", "weigh"):
        s["q"] = normal(case["batch"], case["q_len"], case["heads"], dim).to(BF16)
    if case["op"] in ("weigh", "evict"):
        # what earlier steps gave the keys: few have most of it
        s["weights"] = torch.exp(1.5 * normal(pages, kv, page)) * 1e-2
    return s


# ------------------------------------------------------------------ the plain form
def _norm_rotate(x, gamma, s):
    """[T, heads, dim] -> float32: norm of every head, then the rotation of its first elements."""
    case = s["case"]
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma
    pos = s["pos"] if s["axis"] is None else s["pos"][s["axis"].long()].t()
    angle = pos.double().view(case["tokens"], -1) * s["freq"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    rot, rest = x[..., :case["rot"]], x[..., case["rot"]:]
    if case["interleaved"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = rot.chunk(2, -1)
        rot = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([rot, rest], -1)


def _requantise(codes, old, new):
    """Codes of the scale of byte `old` in that of `new`."""
    return (codes.float() * torch.exp2(old.to(F32) - new.to(F32))).to(F8)


def _plain_keep(x, cache, scale, s, page_id, row, first):
    """The rows x [T, heads, dim] (float32) into the cache in 8 bits."""
    case = s["case"]
    kv, dim, blocks = case["kv_heads"], case["dim"], case["page"] // BLOCK
    block = page_id * blocks + row // BLOCK                                      # of every token
    by_block = cache.view(-1, kv, blocks, BLOCK, dim).transpose(1, 2)            # [pages, blocks, heads, 16, dim]
    at, sub = page_id, row // BLOCK
    top = torch.zeros(len(cache) * blocks, kv, device=DEV)
    top.scatter_reduce_(0, block[:, None].expand(-1, kv), x.abs().amax(-1), "amax")
    fresh = torch.zeros(len(cache) * blocks, dtype=torch.bool, device=DEV)
    fresh[block[first]] = True
    old = scale[at, :, sub].int()
    new = _scale_byte(top[block])
    new = torch.where(fresh[block][:, None], new, torch.maximum(new, old))
    # the rows that are there: tokens of one block write the same
    grown = (new > old) & ~fresh[block][:, None]
    there = by_block.view(U8)[at, sub].view(F8)
    moved = _requantise(there, old[..., None, None], new[..., None, None])
    by_block.view(U8)[at, sub] = torch.where(grown[..., None, None], moved.view(U8), there.view(U8))
    scale[at, :, sub] = new.to(U8)
    cache.view(U8)[at, :, row] = _to_codes(x, new[..., None]).view(U8)


def _plain_append(s):
    page = s["case"]["page"]
    rows = (s["pos"] if s["rows"] is None else s["rows"]).long()
    at, row = s["table"][s["seq"].long(), rows // page].long(), rows % page
    first = row % BLOCK == 0
    _plain_keep(_norm_rotate(s["k"], s["k_gamma"], s), s["k_cache"], s["k_scale"], s, at, row, first)
    _plain_keep(s["v"].float(), s["v_cache"], s["v_scale"], s, at, row, first)
    return _norm_rotate(s["q"], s["q_gamma"], s).to(BF16)


def _values(s, which, ids):
    """The float32 rows of the pages `ids` [..], [.., heads, page, dim]."""
    x = s[which + "_cache"]
    if x.dtype == BF16:
        return x[ids].float()
    return x.view(U8)[ids].view(F8).float() * _power(s[which + "_scale"][ids]).repeat_interleave(BLOCK, -1)[..., None]


def _plain_paged(s):
    case = s["case"]
    batch, ql, heads, kv, dim, page = (case[x] for x in ("batch", "q_len", "heads", "kv_heads", "dim", "page"))
    group, prefix = heads // kv, case["prefix"]
    table, lens = s["table"].long(), s["lens"].long()
    longest = table.shape[1] * page
    own_k, own_v = (_values(s, x, table).permute(0, 2, 1, 3, 4).reshape(batch, kv, longest, dim) for x in "kv")
    last = lens[:, None] - ql + torch.arange(ql, device=DEV)[None]              # last own key that each token sees
    seen = torch.arange(longest, device=DEV)[None, None] <= last[..., None]
    q = s["q"].float().view(batch, ql, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv, group * ql, dim)
    scores = torch.matmul(q, own_k.transpose(-1, -2)).mul_(dim ** -0.5)
    seen = seen[:, None, None].expand(batch, kv, group, ql, longest).reshape(batch, kv, group * ql, longest)
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if prefix:
        pk, pv = (_values(s, x, s["prefix"].long()).permute(1, 0, 2, 3).reshape(kv, -1, dim)[:, :prefix] for x in "kv")
        rows = q.permute(1, 0, 2, 3).reshape(kv, -1, dim)
        shared = torch.matmul(rows, pk.transpose(-1, -2)).mul_(dim ** -0.5)
        both = torch.maximum(top.permute(1, 0, 2, 3).reshape(kv, -1, 1), shared.amax(-1, keepdim=True))
        shared = shared.sub_(both).exp_()
        back = lambda t: t.view(kv, batch, group * ql, -1).permute(1, 0, 2, 3)  # noqa: E731
        more, more_sum, top = back(torch.matmul(shared, pv)), back(shared.sum(-1, keepdim=True)), back(both)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    o, total = torch.matmul(p, own_v), p.sum(-1, keepdim=True)
    if prefix:
        o, total = o + more, total + more_sum
    total = torch.where(total == 0, torch.ones_like(total), total)
    o = (o / total).view(batch, kv, group, ql, dim).permute(0, 3, 1, 2, 4).reshape(batch, ql, heads, dim).to(BF16)
    if case["op"] == "paged":
        return o
    given = p.div_(total).sum(2)                                                # [batch, heads, keys]
    rows = torch.arange(longest, device=DEV)
    b, r = (rows[None] < lens[:, None]).nonzero(as_tuple=True)
    s["weights"][table[b, r // page], :, r % page] += given[b, :, r]
    return {"o": o, "weights": s["weights"]}


def _plain_evict(s):
    """Dest row j of the first `keep` takes the row src[j] >= j: itself, or what is kept from behind."""
    case = s["case"]
    kv, page, keep, first, recent = (case[x] for x in ("kv_heads", "page", "keep", "first", "recent"))
    table, lens = s["table"].long(), s["lens"].long()
    full = (lens > keep).nonzero()[:, 0]                                        # the sequences that are cut down
    new = torch.clamp(lens, max=keep).to(torch.int32)
    table, n = table[full], lens[full][:, None, None]
    longest = table.shape[1] * page
    at = torch.arange(longest, device=DEV)
    weights = s["weights"][table].permute(0, 2, 1, 3).reshape(len(full), kv, longest)
    fixed = ((at < first) | ((at >= n - recent) & (at < n))).expand_as(weights)
    free = (at < n) & ~fixed
    # among the free rows by weight, the first of equals first; then all others
    order = torch.sort(weights, dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, torch.sort((~free.gather(-1, order)).to(U8), dim=-1, stable=True).indices)
    best = torch.zeros_like(free).scatter_(-1, order[..., :keep - first - recent], True)
    kept = fixed | best
    middle = keep - recent
    hole, spare = ~kept[..., :middle], (kept & (at < n - recent))[..., middle:]
    # the i-th of the spare rows goes to the i-th hole
    place = torch.where(spare, spare.cumsum(-1) - 1, longest)
    rank = torch.zeros(len(full), kv, longest + 1, dtype=torch.long, device=DEV).scatter_(-1, place, at[middle:].expand_as(place))
    src = at[:keep].expand(len(full), kv, keep).clone()
    src[..., :middle] = torch.where(hole, rank.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)), src[..., :middle])
    src[..., middle:] += n - keep
    head = torch.arange(kv, device=DEV)[None, :, None]
    which = torch.arange(len(full), device=DEV)[:, None, None]
    from_page, to_page = table[which, src // page], table[which, at[:keep] // page].expand_as(src)
    from_row, to_row = src % page, (at[:keep] % page).expand_as(src)
    moved = s["weights"][from_page, head, from_row]
    s["weights"][to_page, head, to_row] = moved
    for x in "kv":
        cache = s[x + "_cache"]
        rows = cache.view(U8)[from_page, head, from_row].view(cache.dtype)
        if cache.dtype != BF16:
            scale = s[x + "_scale"]
            byte = scale[from_page, head, from_row // BLOCK].int()
            # a block with a row from elsewhere takes the largest of its rows' scales
            block = (at[:keep] // BLOCK).expand_as(src)
            top = torch.zeros(len(full), kv, -(-keep // BLOCK), dtype=torch.int32, device=DEV)
            other = torch.zeros_like(top).scatter_reduce_(-1, block, (src != at[:keep]).int(), "amax")
            top = top.scatter_reduce_(-1, block, byte, "amax").gather(-1, block)
            top = torch.where(other.gather(-1, block) > 0, top, byte)
            rows = _requantise(rows, byte[..., None], top[..., None])
            scale[to_page, head, to_row // BLOCK] = top.to(U8)
        cache.view(U8)[to_page, head, to_row] = rows.view(U8)
    return new


def _state(s):
    """The caches as a user reads them."""
    case = s["case"]
    if case["op"] == "evict" and case["cache"] == "bf16":
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "k_scale": s["k_scale"].view(torch.float8_e8m0fnu),
            "v_scale": s["v_scale"].view(torch.float8_e8m0fnu)}


def _plain(s):
    op = s["case"]["op"]
    if op == "rope":
        return {"q": _norm_rotate(s["q"], s["q_gamma"], s).to(BF16), "k": _norm_rotate(s["k"], s["k_gamma"], s).to(BF16)}
    if op == "append":
        return {"q": _plain_append(s), **_state(s)}
    if op == "evict":
        return {"lens": _plain_evict(s), "weights": s["weights"], **_state(s)}
    return _plain_paged(s)


# ------------------------------------------------------------------ the package
def _own(s):
    dsk, case = _package(), s["case"]
    if case["op"] == "rope":
        q, k = dsk.qk_norm_rope(s["q"], s["k"], s["pos"], s["freq"], axis=s["axis"], interleaved=case["interleaved"],
                                q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=EPS)
        return {"q": q, "k": k}
    if case["op"] == "append":
        q = dsk.kv_append(s["q"], s["k"], s["v"], s["pos"], s["seq"], s["table"], s["k_cache"], s["v_cache"], s["freq"],
                          axis=s["axis"], rows=s["rows"], k_scale=s["k_scale"], v_scale=s["v_scale"], q_gamma=s["q_gamma"],
                          k_gamma=s["k_gamma"], eps=EPS)
        return {"q": q, **_state(s)}
    if case["op"] == "evict":
        lens = dsk.kv_evict(s["k_cache"], s["v_cache"], s["weights"], s["table"], s["lens"], case["keep"], first=case["first"],
                            recent=case["recent"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {"lens": lens, "weights": s["weights"], **_state(s)}
    shared = {"prefix": s["prefix"], "prefix_len": case["prefix"]} if case["prefix"] else {}
    if case["op"] == "paged":
        return dsk.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], k_scale=s["k_scale"],
                                   v_scale=s["v_scale"], **shared)
    o = dsk.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                            key_weights=s["weights"])
    return {"o": o, "weights": s["weights"]}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ work and definition
def work(case):
    dim, kv = case["dim"], case["kv_heads"]
    if case["op"] == "rope":
        rows = case["tokens"] * (case["heads"] + kv) * dim
        return {"bytes": rows * ((2 if case["dtype"] == "bf16" else 4) + 2), "flops": 10 * rows}
    if case["op"] == "append":
        q, rows = case["tokens"] * case["heads"] * dim, 2 * case["tokens"] * kv * dim
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": q * (size + 2) + rows * (size + 1) + rows // dim // BLOCK, "flops": 10 * (q + rows)}
    lens = _lens_of(case)
    row = 2 * dim * 2 if case["cache"] == "bf16" else 2 * dim + 2 / BLOCK       # a key and its value
    if case["op"] == "evict":
        keep, fixed = case["keep"], case["first"] + case["recent"]
        cut = [n for n in lens if n > keep]
        moved = sum(case["recent"] + (n - keep) * (keep - fixed) / max(1, n - fixed) for n in cut)
        return {"bytes": int(kv * (4 * sum(cut) + 2 * moved * (row + 4))) + 8 * len(lens), "flops": kv * sum(cut)}
    ql, prefix, heads = case["q_len"], case["prefix"], case["heads"]
    pairs = sum(max(0, n - ql + 1 + i) for n in lens for i in range(ql)) + case["batch"] * ql * prefix
    more = 8 * kv * sum(lens) if case["op"] == "weigh" else 0
    return {"bytes": int(4 * dim * heads * case["batch"] * ql + row * kv * (sum(lens) + prefix)) + more, "flops": 4 * dim * heads * pairs}


def _exact_rotate(x, gamma, s):
    case = s["case"]
    x = x.double()
    y = x / torch.sqrt(torch.mean(x ** 2, dim=-1, keepdim=True) + EPS) * gamma.double()
    i = torch.arange(case["rot"] // 2, device=DEV)
    pos = s["pos"].double().view(-1, case["tokens"])
    at = pos[s["axis"].long()] if s["axis"] is not None else pos.expand(len(i), -1)
    turn = torch.polar(torch.ones((), dtype=F64, device=DEV), (at * s["freq"][:, None]).t()[:, None])
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + case["rot"] // 2)
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_byte(top):
    """Least b with top <= 448 * 2^(b - 127), by the logarithm."""
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0))
    return (e + 127).clamp(LEAST, MOST)


def _round_e4m3(x):
    """float64 to the nearest e4m3 value (ties to even), still float64."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))).clamp(max=8) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_append(s):
    case = s["case"]
    page, blocks = case["page"], case["page"] // BLOCK
    rows = (s["pos"] if s["rows"] is None else s["rows"]).tolist()
    seq, table = s["seq"].tolist(), s["table"].tolist()
    new = {"k": _exact_rotate(s["k"], s["k_gamma"], s), "v": s["v"].double()}
    got = {}
    to = {}
    for t, (b, r) in enumerate(zip(seq, rows)):
        to.setdefault((table[b][r // page], r % page // BLOCK), []).append((t, r % BLOCK))
    # blocks with the same number of new rows together
    for x in "kv":
        codes, byte = s[x + "_cache"].double(), s[x + "_scale"].double()
        view = codes.view(len(codes), -1, blocks, BLOCK, case["dim"])
        sizes = sorted({len(v) for v in to.values()})
        for size in sizes:
            keys = [k for k, v in to.items() if len(v) == size]
            p, c = (torch.tensor([k[i] for k in keys], device=DEV) for i in (0, 1))
            tok, row = (torch.tensor([[e[i] for e in to[k]] for k in keys], device=DEV) for i in (0, 1))
            y = new[x][tok].transpose(1, 2)                                     # [block, head, new row, dim]
            want = _exact_byte(y.abs().amax((-1, -2)))
            afresh = (row == 0).any(1)[:, None]
            have = byte[p, :, c]
            b = torch.where(afresh, want, torch.maximum(want, have))
            there = view[p, :, c]                                               # [block, head, 16, dim]
            scaled = _round_e4m3(there * torch.exp2(have - b)[..., None, None])
            there = torch.where(afresh[..., None, None], there, scaled)
            index = row[:, None, :, None].expand(-1, y.shape[1], -1, y.shape[3])
            view[p, :, c] = there.scatter(2, index, _round_e4m3(y / torch.exp2(b - 127)[..., None, None]))
            byte[p, :, c] = b
        got[x + "_cache"], got[x + "_scale"] = codes, torch.exp2(byte - 127)
    return {"q": _exact_rotate(s["q"], s["q_gamma"], s), **got}


def _exact_paged(s):
    case = s["case"]
    kv, ql, page, prefix, group = case["kv_heads"], case["q_len"], case["page"], case["prefix"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=F64, device=DEV)
    weights = s["weights"].double() if case["op"] == "weigh" else None

    def rows(x, ids):
        y = s[x + "_cache"].view(U8)[ids.long()].view(s[x + "_cache"].dtype).double()
        if s[x + "_scale"] is not None:
            y = y.unflatten(2, (-1, BLOCK)) * torch.exp2(s[x + "_scale"][ids.long()].double() - 127)[..., None, None]
            y = y.flatten(2, 3)
        return y.transpose(1, 2).flatten(0, 1)                                  # [rows, heads, dim]

    for b, n in enumerate(s["lens"].tolist()):
        mine = s["table"][b][:-(-n // page)]
        k, v = (torch.cat([rows(x, s["prefix"])[:prefix], rows(x, mine)[:n]]) for x in "kv")
        if not len(k):
            continue
        last = torch.arange(ql, device=DEV) + prefix + n - ql
        hidden = torch.arange(len(k), device=DEV)[None] > last.clamp(min=prefix - 1)[:, None]
        for h in range(case["heads"]):
            w = torch.softmax((s["q"][b, :, h].double() @ k[:, h // group].T / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf), -1)
            w = w.masked_fill(hidden, 0.0)
            out[b, :, h] = w @ v[:, h // group]
            if weights is not None:
                at = torch.arange(n, device=DEV)
                weights[mine.long()[at // page], h // group, at % page] += w.sum(0)[prefix:]
    return out if weights is None else {"o": out, "weights": weights}


def _exact_evict(s):
    case = s["case"]
    page, keep, first, recent = (case[x] for x in ("page", "keep", "first", "recent"))
    weights = s["weights"].cpu().numpy()
    table, lens = s["table"].cpu().numpy(), s["lens"].tolist()
    got = {"weights": s["weights"].double()}
    for x in "kv":
        got[x + "_cache"] = s[x + "_cache"].double()
        if s[x + "_scale"] is not None:
            got[x + "_scale"] = s[x + "_scale"].double()
    for b, n in enumerate(lens):
        if n <= keep:
            continue
        at = np.arange(n)
        ids = table[b][at // page]
        for h in range(case["kv_heads"]):
            w = weights[ids, h, at % page]
            free = at[first:n - recent]
            best = free[np.lexsort((free, -w[free]))][:keep - first - recent]
            stay = np.sort(np.concatenate([at[:first], best]))
            source = np.full(keep, -1)
            near = stay[stay < keep - recent]
            source[near] = near
            source[:keep - recent][source[:keep - recent] < 0] = stay[stay >= keep - recent]
            source[keep - recent:] = at[n - recent:]
            changed = source != np.arange(keep)
            if not changed.any():
                continue
            # whole blocks, as far as the first `keep` rows go
            lo = int(np.flatnonzero(changed)[0]) // BLOCK * BLOCK
            dest = np.arange(lo, keep)
            ids_t, row_t = torch.tensor(ids[dest], device=DEV).long(), torch.tensor(dest % page, device=DEV)
            ids_f, row_f = torch.tensor(ids[source[dest]], device=DEV).long(), torch.tensor(source[dest] % page, device=DEV)
            got["weights"][ids_t, h, row_t] = got["weights"][ids_f, h, row_f]
            for x in "kv":
                cache = got[x + "_cache"]
                rows = cache[ids_f, h, row_f]
                if x + "_scale" in got:
                    scale = got[x + "_scale"]
                    byte = scale[ids_f, h, row_f // BLOCK]
                    count = -(-len(dest) // BLOCK)
                    padded = torch.zeros(count * BLOCK, dtype=F64, device=DEV)
                    padded[:len(dest)] = byte
                    other = np.zeros(count * BLOCK, dtype=bool)
                    other[:len(dest)] = changed[dest]
                    touched = torch.tensor(other.reshape(count, BLOCK).any(1), device=DEV)
                    top = padded.view(count, BLOCK).amax(1).repeat_interleave(BLOCK)[:len(dest)]
                    top = torch.where(touched.repeat_interleave(BLOCK)[:len(dest)], top, byte)
                    rows = _round_e4m3(rows * torch.exp2(byte - top)[:, None])
                    scale[ids_t, h, row_t // BLOCK] = top
                cache[ids_t, h, row_t] = rows
    for x in "kv":
        if x + "_scale" in got:
            got[x + "_scale"] = torch.exp2(got[x + "_scale"] - 127)
    return {"lens": None, **got}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return {"q": _exact_rotate(s["q"], s["q_gamma"], s), "k": _exact_rotate(s["k"], s["k_gamma"], s)}
    return {"append": _exact_append, "evict": _exact_evict}.get(case["op"], _exact_paged)(s)
