"""The attention half of a decoder layer, as cases that can be timed and compared.

A case is one call of ``qk_norm_rope`` (per-head norms and rotation of queries and
keys), ``kv_append`` (the same pass, keeping keys and values in a paged cache),
``prompt_attention`` (causal attention over packed prompts) or ``paged_attention``
(a decode or verify step over the cache, with or without a prefix that the batch
shares).  Heads of 128 with 32 query and 8 key heads fit the hidden size of 4096 that
the layers here are benchmarked with; the others are generic.

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
_PKG = str(Path(__file__).resolve().parent.parent / "deepseeker-v4.1_amd")


def _package():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import dsk_moe
    return dsk_moe


# ------------------------------------------------------------------ cases
def _rope(name, tokens, heads, kv_heads, dim, rot, interleaved=False, dtype="bf16", far=4096, scaled=False):
    return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rot": rot, "interleaved": interleaved, "dtype": dtype, "far": far, "scaled": scaled}


def _append(name, seqs, tokens, heads, kv_heads, dim, rot, page, interleaved=False, dtype="bf16", far=4096):
    return {"name": name, "op": "append", "seqs": seqs, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rot": rot, "page": page, "interleaved": interleaved, "dtype": dtype, "far": far}


def _prompt(name, seqs, longest, heads, kv_heads, dim, pad=0, before=0):
    return {"name": name, "op": "prompt", "seqs": seqs, "longest": longest, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "pad": pad, "before": before}


def _paged(name, batch, q_len, longest, heads, kv_heads, dim, page, prefix=0, empty=False):
    return {"name": name, "op": "paged", "batch": batch, "q_len": q_len, "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "prefix": prefix, "empty": empty}


def listed():
    return [
        # a few float32 rows with heads of 64, pairs next to each other, half of the head rotated
        _rope("rope_7", 7, 16, 4, 64, 32, interleaved=True, dtype="f32", far=500),
        # a long chunk at far positions, frequencies scaled for a long context
        _rope("rope_4095", 4095, 32, 8, 128, 128, far=1000000, scaled=True),
        # one token of decode goes into the cache
        _append("append_1", 1, 1, 32, 8, 128, 128, 64, far=900),
        # a prefill step: packed prompts of many requests are kept in the cache
        _append("append_8192", 13, 8192, 32, 8, 128, 128, 64),
        # one short prompt, all latency
        _prompt("prompt_17", 1, 17, 32, 8, 128),
        # a prefill step of ragged prompts with heads of 64, some rows of padding behind them
        _prompt("prompt_packed", 16, 1500, 16, 4, 64, pad=37),
        # one long prompt
        _prompt("prompt_8192", 1, 8192, 32, 8, 128),
        # one token of one short conversation, all latency
        _paged("decode_1", 1, 1, 517, 32, 8, 128, 64),
        # a full decode batch of ragged conversations, one slot of it unused
        _paged("decode_64", 64, 1, 8192, 32, 8, 128, 64, empty=True),
        # a two-token verify step of few long conversations, small pages
        _paged("verify_8x2", 8, 2, 32768, 16, 4, 64, 16),
        # a two-token verify step behind a shared instruction
        _paged("prefix_6x2", 6, 2, 300, 16, 4, 64, 16, prefix=1999),
        # a full batch that shares a long document
        _paged("prefix_64", 64, 1, 600, 32, 8, 128, 64, prefix=16385),
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 4, 128), (16, 4, 64), (12, 12, 64), (40, 5, 128), (24, 8, 64)])
    page = rng.choice([16, 32, 64, 128])
    rot = rng.choice([dim, dim, dim // 2, dim // 4])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    op = rng.choice(["rope", "append", "prompt", "prompt", "paged", "paged", "prefix", "prefix"])
    if op == "rope":
        c = _rope("", log_int(1, 8192), heads, kv_heads, dim, rot, rng.random() < 0.5, dtype, log_int(10, 1000000),
                  rng.random() < 0.5)
    elif op == "append":
        tokens = log_int(1, 8192)
        c = _append("", min(tokens, log_int(1, 64)), tokens, heads, kv_heads, dim, rot, page, rng.random() < 0.5, dtype)
    elif op == "prompt":
        seqs = log_int(1, 40)
        # padded to the longest, the scores stay below those of the longest listed prompt
        c = _prompt("", seqs, log_int(1, int(5800 / math.sqrt(seqs))), heads, kv_heads, dim,
                    rng.choice([0, 0, rng.randint(1, 99)]), rng.choice([0, 0, rng.randint(1, 900)]))
    else:
        batch = log_int(1, 64)
        q_len = rng.choice([1, 1, 1, 2, 4])
        c = _paged("", batch, q_len, log_int(q_len, min(32768, 524288 // batch)), heads, kv_heads, dim, page,
                   log_int(64, 16384) if op == "prefix" else 0, rng.random() < 0.3)
    c.pop("name")
    return c


# ------------------------------------------------------------------ inputs
def _lengths(rng, n, longest):
    """n lengths of 1 to longest, spread over their logarithm, one of them the longest."""
    got = [min(longest, max(1, int(round(math.exp(rng.uniform(0.0, math.log(longest + 0.5))))))) for _ in range(n)]
    got[rng.randrange(n)] = longest
    return got


def _lens_of(case):
    """The case's sequence lengths: they belong to the case, so that its work is the same for every seed."""
    rng = random.Random(17)
    if case["op"] == "prompt":
        return _lengths(rng, case["seqs"], case["longest"])
    if case["op"] == "paged":
        got = [max(case["q_len"], v) for v in _lengths(rng, case["batch"], case["longest"])]
        if case["empty"]:
            got[got.index(min(got))] = 0
        return got
    cuts = sorted(rng.sample(range(1, case["tokens"]), case["seqs"] - 1)) if case["seqs"] > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]


def _frequencies(rot, scaled):
    """Radians per position of each pair, float64; scaled: slow pairs turn a quarter as fast, quick ones as before."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaled:
        turns = 4096.0 * f / (2.0 * math.pi)
        keep = torch.clamp((turns - 1.0) / 31.0, 0.0, 1.0)
        f = f * (keep + (1.0 - keep) / 4.0)
    return f.to(DEV)


def _pages(gen, table_pages, spare):
    """A shuffled assignment of table_pages pages out of table_pages + spare."""
    return torch.randperm(table_pages + spare, generator=gen, device=DEV)[:table_pages].to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    rng = random.Random(int(seed))
    dim, heads, kv = case["dim"], case["heads"], case["kv_heads"]

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(shape, generator=gen, device=DEV).to(dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    s = {"case": dict(case)}
    if case["op"] in ("rope", "append"):
        t = case["tokens"]
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        # the three are views of one projection's rows
        qkv = normal(t, (heads + 2 * kv) * dim, dtype=dtype)
        s["q"], s["k"], s["v"] = (p.unflatten(1, (-1, dim)) for p in qkv.split([heads * dim, kv * dim, kv * dim], 1))
        s["q_gamma"], s["k_gamma"] = (1.0 + 0.1 * torch.randn(dim, generator=gen, device=DEV) for _ in range(2))
        s["freq"] = _frequencies(case["rot"], case.get("scaled", False))
        if case["op"] == "rope":
            s["pos"] = (torch.arange(t, device=DEV) + rng.randint(0, case["far"])).to(torch.int32)
            return s
        lens = _lens_of(case)
        where = random.Random(18)
        starts = [where.randint(0, case["far"]) for _ in lens]
        s["pos"] = ints([a + i for a, n in zip(starts, lens) for i in range(n)])
        s["seq"] = ints([b for b, n in enumerate(lens) for _ in range(n)])
        width = (case["far"] + max(lens)) // case["page"] + 1
        used = [(a + n - 1) // case["page"] + 1 for a, n in zip(starts, lens)]
        ids = _pages(gen, sum(used), 3)
        s["table"] = torch.zeros((len(lens), width), dtype=torch.int32, device=DEV)
        cols = torch.arange(width, device=DEV)[None, :] < torch.tensor(used, device=DEV)[:, None]
        s["table"][cols] = ids
        s["k_cache"], s["v_cache"] = (normal(sum(used) + 3, kv, case["page"], dim) for _ in range(2))
        return s
    lens = _lens_of(case)
    if case["op"] == "prompt":
        n, before = sum(lens), case["before"]
        s["q"] = normal(n + case["pad"], heads, dim)
        s["k"], s["v"] = (normal(n + before * len(lens) + case["pad"], kv, dim) for _ in range(2))
        s["cu"] = ints(np.concatenate([[0], np.cumsum(lens)]).tolist())
        # with earlier tokens before each prompt: its keys and values are longer than its queries
        s["cu_k"] = ints(np.concatenate([[0], np.cumsum([v + before for v in lens])]).tolist())
        s["out"] = normal(n + case["pad"], heads, dim)
        s["longest"] = case["longest"]
        return s
    page = case["page"]
    s["q"] = normal(case["batch"], case["q_len"], heads, dim)
    s["lens"] = ints(lens)
    used = [-(-v // page) for v in lens]
    shared = -(-case["prefix"] // page)
    ids = _pages(gen, sum(used) + shared, 3)
    s["prefix"] = ids[:shared].contiguous()
    width = max(used) + 1
    s["table"] = torch.zeros((case["batch"], width), dtype=torch.int32, device=DEV)
    cols = torch.arange(width, device=DEV)[None, :] < torch.tensor(used, device=DEV)[:, None]
    s["table"][cols] = ids[shared:]
    s["k_cache"], s["v_cache"] = (normal(sum(used) + shared + 3, kv, page, dim) for _ in range(2))
    return s


# ------------------------------------------------------------------ the plain form
def _norm_rotate(x, gamma, s):
    """[T, heads, dim] -> bf16: norm of every head, then the rotation of its first elements."""
    case = s["case"]
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma
    angle = s["pos"].double()[:, None] * s["freq"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    rot, rest = x[..., :case["rot"]], x[..., case["rot"]:]
    if case["interleaved"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = rot.chunk(2, -1)
        rot = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([rot, rest], -1).to(torch.bfloat16)


def _softmax_product(scores, seen, v):
    """scores [.., rows, keys], seen [.., rows, keys], v [.., keys, dim] -> [.., rows, dim]; zero where nothing is seen."""
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)


def _plain_prompt(s):
    case = s["case"]
    heads, kv, dim, group = case["heads"], case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    cu, cu_k, lq = s["cu"].long(), s["cu_k"].long(), s["longest"]
    lk = lq + case["before"]
    n, nk = cu[1:] - cu[:-1], cu_k[1:] - cu_k[:-1]
    iq, ik = torch.arange(lq, device=DEV), torch.arange(lk, device=DEV)
    at_q = cu[:-1, None] + torch.minimum(iq[None], n[:, None] - 1)
    at_k = cu_k[:-1, None] + torch.minimum(ik[None], nk[:, None] - 1)
    q = s["q"][at_q].float().view(-1, lq, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(-1, kv, group * lq, dim)
    k, v = (s[x][at_k].float().permute(0, 2, 1, 3) for x in ("k", "v"))
    seen = (ik[None, None] < nk[:, None, None]) & (ik[None, None] <= iq[None, :, None] + (nk - n)[:, None, None])
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(dim ** -0.5).view(-1, kv, group, lq, lk)
    o = _softmax_product(scores, seen[:, None, None], v[:, :, None])
    o = o.permute(0, 3, 1, 2, 4).reshape(-1, lq, heads, dim).to(torch.bfloat16)
    real = iq[None] < n[:, None]
    s["out"][at_q[real]] = o[real]
    return s["out"]


def _plain_paged(s):
    case = s["case"]
    batch, ql, heads, kv, dim, page = (case[x] for x in ("batch", "q_len", "heads", "kv_heads", "dim", "page"))
    group, prefix = heads // kv, case["prefix"]
    lens = s["lens"].long()
    longest = s["table"].shape[1] * page
    at = torch.arange(longest, device=DEV)
    own_k, own_v = (s[x][s["table"].long()].float().permute(0, 2, 1, 3, 4).reshape(batch, kv, longest, dim)
                    for x in ("k_cache", "v_cache"))
    last = lens[:, None] - ql + torch.arange(ql, device=DEV)[None]          # last own key that each token sees
    seen = at[None, None] <= last[..., None]
    q = s["q"].float().view(batch, ql, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv, group * ql, dim)
    scores = torch.matmul(q, own_k.transpose(-1, -2)).mul_(dim ** -0.5)
    seen = seen[:, None, None].expand(batch, kv, group, ql, longest).reshape(batch, kv, group * ql, longest)
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if prefix:
        pk, pv = (s[x][s["prefix"].long()].float().permute(1, 0, 2, 3).reshape(kv, -1, dim)[:, :prefix]
                  for x in ("k_cache", "v_cache"))
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
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    return o.view(batch, kv, group, ql, dim).permute(0, 3, 1, 2, 4).reshape(batch, ql, heads, dim).to(torch.bfloat16)


def _plain(s):
    op = s["case"]["op"]
    if op == "rope":
        return {"q": _norm_rotate(s["q"], s["q_gamma"], s), "k": _norm_rotate(s["k"], s["k_gamma"], s)}
    if op == "append":
        page = s["case"]["page"]
        pos, seq = s["pos"].long(), s["seq"].long()
        at, row = s["table"][seq, pos // page].long(), pos % page
        s["k_cache"][at, :, row] = _norm_rotate(s["k"], s["k_gamma"], s)
        s["v_cache"][at, :, row] = s["v"].to(torch.bfloat16)
        return {"q": _norm_rotate(s["q"], s["q_gamma"], s), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return _plain_prompt(s) if op == "prompt" else _plain_paged(s)


# ------------------------------------------------------------------ the package
def _own(s):
    dsk, case = _package(), s["case"]
    if case["op"] == "rope":
        q, k = dsk.qk_norm_rope(s["q"], s["k"], s["pos"], s["freq"], interleaved=case["interleaved"],
                                q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=EPS)
        return {"q": q, "k": k}
    if case["op"] == "append":
        q = dsk.kv_append(s["q"], s["k"], s["v"], s["pos"], s["seq"], s["table"], s["k_cache"], s["v_cache"], s["freq"],
                          interleaved=case["interleaved"], q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=EPS)
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["op"] == "prompt":
        return dsk.prompt_attention(s["q"], s["k"], s["v"], s["cu"], s["cu_k"] if case["before"] else None, out=s["out"])
    if case["prefix"]:
        return dsk.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], prefix=s["prefix"],
                                   prefix_len=case["prefix"])
    return dsk.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ work and definition
def work(case):
    dim, heads, kv = case["dim"], case["heads"], case["kv_heads"]
    if case["op"] in ("rope", "append"):
        t = case["tokens"]
        rows = t * (heads + (kv if case["op"] == "rope" else 2 * kv)) * dim
        return {"bytes": rows * ((2 if case["dtype"] == "bf16" else 4) + 2), "flops": 10 * rows}
    lens = _lens_of(case)
    if case["op"] == "prompt":
        b = case["before"]
        pairs = sum(n * (n + 1) // 2 + n * b for n in lens)
        return {"bytes": 2 * dim * (2 * heads * sum(lens) + 2 * kv * sum(n + b for n in lens)),
                "flops": 4 * dim * heads * pairs}
    ql, prefix = case["q_len"], case["prefix"]
    pairs = sum(max(0, n - ql + 1 + i) for n in lens for i in range(ql)) + case["batch"] * ql * prefix
    return {"bytes": 2 * dim * (2 * heads * case["batch"] * ql + 2 * kv * (sum(lens) + prefix)),
            "flops": 4 * dim * heads * pairs}


def _exact_rotate(x, gamma, pos, freq, rot, interleaved):
    x = x.double()
    y = x / torch.sqrt(torch.mean(x ** 2, dim=-1, keepdim=True) + EPS) * gamma.double()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), pos.double()[:, None, None] * freq)
    i = torch.arange(rot // 2, device=DEV)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_attention(q, k, v, last):
    """q [rows, heads, dim], k and v [keys, kv heads, dim], last [rows]: the last key that each row sees."""
    heads, kv, dim = q.shape[1], k.shape[1], q.shape[2]
    o = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    if not len(k):
        return o
    hidden = torch.arange(len(k), device=DEV)[None] > last[:, None]
    for h in range(heads):
        kh, vh = (x[:, h * kv // heads].double() for x in (k, v))
        w = torch.softmax((q[:, h].double() @ kh.T / math.sqrt(dim)).masked_fill(hidden, -math.inf), -1)
        o[:, h] = w.masked_fill(hidden, 0.0) @ vh
    return o


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rope", "append"):
        q, k = (_exact_rotate(s[x], s[x + "_gamma"], s["pos"], s["freq"], case["rot"], case["interleaved"]) for x in "qk")
        if case["op"] == "rope":
            return {"q": q, "k": k}
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        slot = s["table"][s["seq"].long(), torch.div(s["pos"], case["page"], rounding_mode="floor").long()].long()
        for h in range(case["kv_heads"]):
            kc[slot, h, (s["pos"] % case["page"]).long()] = k[:, h]
            vc[slot, h, (s["pos"] % case["page"]).long()] = s["v"][:, h].double()
        return {"q": q, "k_cache": kc, "v_cache": vc}
    if case["op"] == "prompt":
        out, cu, ck = s["out"].double(), s["cu"].tolist(), s["cu_k"].tolist()
        for b in range(case["seqs"]):
            n = cu[b + 1] - cu[b]
            out[cu[b]:cu[b + 1]] = _exact_attention(s["q"][cu[b]:cu[b + 1]], s["k"][ck[b]:ck[b + 1]], s["v"][ck[b]:ck[b + 1]],
                                                    torch.arange(n, device=DEV) + ck[b + 1] - ck[b] - n)
        return out
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lens, ql = s["lens"].tolist(), case["q_len"]
    flat = lambda x, ids: s[x][ids.long()].transpose(1, 2).flatten(0, 1)  # noqa: E731
    for b, n in enumerate(lens):
        k, v = (torch.cat([flat(x, s["prefix"])[:case["prefix"]], flat(x, s["table"][b])[:n]]) for x in ("k_cache", "v_cache"))
        last = torch.arange(ql, device=DEV) + case["prefix"] + n - ql
        out[b] = _exact_attention(s["q"][b], k, v, last.clamp(min=case["prefix"] - 1))
    return out
