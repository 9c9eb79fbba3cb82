"""The attention half of a decoder layer: per-head norms and rotation, a paged
key / value cache, attention over packed prompts and over the cache.

Functions on torch tensors of one HIP device (any device, on its current
stream); outputs are bf16 and are allocated unless given.  Queries, keys and
values are [tokens, heads, head_dim] with any token and head strides that keep
16-byte pieces (so views of one fused projection do); a head's elements are
contiguous.  Outputs must not overlap inputs, except where said.

    freq, mscale = rope_frequencies(128, base=10000.0, device="cuda")
    q = kv_append(q, k, v, positions, seq, table, k_cache, v_cache, freq, q_gamma=gq, k_gamma=gk)
    o = paged_attention(q, k_cache, v_cache, table, lens)

``Attention`` is a whole sublayer (projections, norms, rotation, cache,
attention, output projection); ``MoEStack(layers, attention=[...])`` runs one
before every MoE layer, on a ``PromptStep`` or a ``DecodeStep``.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass, replace

import numpy as np
import torch

from . import _lib

_F32, _BF16, _I32, _F64 = torch.float32, torch.bfloat16, torch.int32, torch.float64


def rope_frequencies(rot_dim: int, base: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                     original_len: int = 4096, turns: tuple[float, float] = (1.0, 32.0),
                     device: torch.device | str = "cuda") -> tuple[torch.Tensor, float]:
    """(freq, mscale): radians per position of the rot_dim / 2 pairs (float64) and the
    factor on the rotated elements.

    ``scaling`` for contexts longer than the ``original_len`` that a model was trained on, by ``factor``:
    "linear" turns every pair ``factor`` times slower; "base" raises the base so that the slowest pair does and
    the quickest keeps its frequency; "ramp" keeps the pairs that make ``turns[1]`` turns or more over
    ``original_len``, slows those that make ``turns[0]`` or less, blends between, and sets
    mscale = 0.1 ln(factor) + 1."""
    if rot_dim < 16 or rot_dim % 16:
        raise ValueError(f"rot_dim must be a positive multiple of 16, got {rot_dim}")
    if not (base > 0 and math.isfinite(base)):
        raise ValueError(f"base must be positive and finite, got {base}")
    if not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError(f"factor must be at least 1 and finite, got {factor}")
    mscale = 1.0
    if scaling == "base":
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freq = base ** (-torch.arange(0, rot_dim, 2, dtype=_F64) / rot_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "ramp":
        lo, hi = turns
        if not 0 < lo < hi or original_len < 1:
            raise ValueError("ramp scaling needs 0 < turns[0] < turns[1] and original_len >= 1")
        keep = ((original_len * freq / (2.0 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / factor)
        mscale = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "base"):
        raise ValueError(f"scaling must be 'linear', 'base', 'ramp' or None, got {scaling!r}")
    return freq.to(device), mscale


# ------------------------------------------------------------------ checks
def _rows(t: torch.Tensor, what: str, dtypes: tuple, dev: torch.device) -> None:
    if t.device != dev:
        raise ValueError(f"{what} is on {t.device}, not on {dev}")
    if t.dim() != 3:
        raise ValueError(f"{what} must be [tokens, heads, head_dim], got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{what} must be {' or '.join(str(d)[6:] for d in dtypes)}, got {str(t.dtype)[6:]}")
    if t.stride(2) != 1:
        raise ValueError(f"the elements of a head of {what} must be contiguous")


def _vector(t: torch.Tensor, what: str, dtype: torch.dtype, n: int, dev: torch.device) -> None:
    if t.device != dev or t.dtype != dtype or t.dim() != 1 or t.shape[0] < n or t.stride(0) != 1:
        raise ValueError(f"{what} must be a contiguous {str(dtype)[6:]} vector of {n} elements on {dev}, "
                         f"got {str(t.dtype)[6:]} {tuple(t.shape)} on {t.device}")


def _exact(t: torch.Tensor, what: str, dtype: torch.dtype, n: int, dev: torch.device) -> None:
    _vector(t, what, dtype, n, dev)
    if t.shape[0] != n:
        raise ValueError(f"{what} must have {n} elements, got {t.shape[0]}")


def _hip(t: torch.Tensor) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"dsk_moe needs HIP device tensors, got a {t.device} tensor")
    return t.device


def _out_strides(out: torch.Tensor | None, shape: tuple, dev: torch.device, what: str) -> tuple[int, int]:
    """Token and head stride of a checked output, or of the one that will be allocated."""
    if out is None:
        return shape[1] * shape[2], shape[2]
    _rows(out, what, (_BF16,), dev)
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"{what} must be {tuple(shape)}, got {tuple(out.shape)}")
    return out.stride()[:2]


# A call's checks depend on its tensors' sizes, strides, types and devices and on its numbers alone, so what they
# found -- a plan: the device, the entry point and its descriptors; no tensor, no address -- serves later calls of the
# same kind.  A number given as something else (a tensor, say, which may change) is read at every call.  A decode step's
# host work is then a third of that of checking each time (18 us a call).
_plans: dict[str, dict[tuple, tuple]] = {"qk": {}, "append": {}, "prompt": {}, "paged": {}}
_MOST_PLANS = 1024
_CONTIGUOUS = torch.contiguous_format


def _sig(t: torch.Tensor | None):
    return (t.shape, t.stride(), t.dtype, t.get_device()) if t is not None else None


def _plan(kind: str, key: tuple, make, *args) -> tuple:
    plan = make(*args)
    if len(_plans[kind]) >= _MOST_PLANS:
        _plans[kind].clear()
    _plans[kind][key] = plan
    return plan


def _call(name: str, fn, dev: torch.device, *args) -> None:
    """The entry point on ``dev``'s current stream, with ``dev`` current."""
    index = dev.index
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(name, rc)


def _p(t: torch.Tensor | None):
    return t.data_ptr() if t is not None else None


def _check_cache(k_cache, v_cache, table, kv_heads: int, dim: int, dev: torch.device) -> None:
    for t, what in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if t.device != dev or t.dtype != _BF16 or t.dim() != 4 or not t.is_contiguous():
            raise ValueError(f"{what} must be contiguous bf16 [pages, kv_heads, page_size, head_dim] on {dev}")
    if k_cache.shape != v_cache.shape or k_cache.shape[1] != kv_heads or k_cache.shape[3] != dim:
        raise ValueError(f"caches {tuple(k_cache.shape)} and {tuple(v_cache.shape)} do not fit {kv_heads} key heads of {dim}")
    if table.device != dev or table.dtype != _I32 or table.dim() != 2 or table.stride(1) != 1:
        raise ValueError(f"table must be int32 [sequences, pages] on {dev} with contiguous rows")


def _cache(k_cache: torch.Tensor, table: torch.Tensor) -> _lib.KVCache:
    return _lib.KVCache(table.stride(0), k_cache.shape[0], k_cache.shape[2], table.shape[0], table.shape[1])


# ------------------------------------------------------------------ norms, rotation, append
def _qk_plan(q, k, v, positions, freq, q_gamma, k_gamma, q_out, k_out, seq, table, k_cache, v_cache, interleaved,
             rot_first, mscale, norm, eps, prefix_len):
    """(entry point, device, descriptor, cache) of a checked call; the outputs have q's and k's shapes."""
    dev = _hip(k)
    _rows(k, "k", (_BF16, _F32), dev)
    tokens, kv_heads, dim = k.shape
    if tokens < 1:
        raise ValueError("k has no tokens")
    heads, qs = 0, (0, 0, 0)
    if q is not None:
        _rows(q, "q", (k.dtype,), dev)
        heads, qs = q.shape[1], q.stride()
        if q.shape[0] != tokens or q.shape[2] != dim:
            raise ValueError(f"q {tuple(q.shape)} does not fit k {tuple(k.shape)}")
    elif q_out is not None or q_gamma is not None:
        raise ValueError("q_out and q_gamma need q")
    _exact(positions, "positions", _I32, tokens, dev)
    rot = 0
    if freq is not None:
        rot = 2 * freq.numel()
        _exact(freq, "freq", _F64, rot // 2, dev)
    for g, what in ((q_gamma, "q_gamma"), (k_gamma, "k_gamma")):
        if g is not None:
            _exact(g, what, _F32, dim, dev)
    vs = (0, 0, 0)
    if v is not None:
        _rows(v, "v", (k.dtype,), dev)
        if v.shape != k.shape:
            raise ValueError(f"v {tuple(v.shape)} does not fit k {tuple(k.shape)}")
        vs = v.stride()
        _exact(seq, "seq", _I32, tokens, dev)
        _check_cache(k_cache, v_cache, table, kv_heads, dim, dev)
    qo, ko = ((0, 0), (0, 0)) if q is None else (_out_strides(q_out, q.shape, dev, "q_out"), (0, 0))
    if k_out is not None or v is None:
        ko = _out_strides(k_out, k.shape, dev, "k_out")
    ks = k.stride()
    desc = _lib.QkDesc(tokens, heads, kv_heads, dim, _lib.DTYPE_BF16 if k.dtype == _BF16 else _lib.DTYPE_F32,
                            1 if norm else 0, rot, rot_first, 1 if interleaved else 0, prefix_len, eps,
                            mscale, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], *qo, *ko)
    lib = _lib.load()
    if v is None:
        return lib.dsk_qk_norm_rope, dev, ctypes.byref(desc), None
    return lib.dsk_kv_append, dev, ctypes.byref(desc), ctypes.byref(_cache(k_cache, table))


def qk_norm_rope(q: torch.Tensor | None, k: torch.Tensor, positions: torch.Tensor, freq: torch.Tensor | None = None, *,
                 interleaved: bool = False, rot_first: int = 0, mscale: float = 1.0,
                 q_gamma: torch.Tensor | None = None, k_gamma: torch.Tensor | None = None, norm: bool = True,
                 eps: float = 1e-6, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None) -> tuple[torch.Tensor | None, torch.Tensor]:
    """``dsk_qk_norm_rope``: RMS norm of every head of q and k (``norm``; gammas [head_dim] float32) and the rotation of
    elements rot_first .. rot_first + 2 len(freq) by positions[t] * freq (``interleaved``: pairs (2i, 2i+1), otherwise (i,
    i + len(freq))), in one pass.  q and k bf16 or float32; the results bf16.  Tokens at negative positions are left out
    (their output rows are not written).  q_out / k_out may be q / k themselves."""
    if not (type(mscale) is type(eps) is float and type(interleaved) is type(norm) is bool and type(rot_first) is int):
        interleaved, rot_first, mscale, norm, eps = bool(interleaved), int(rot_first), float(mscale), bool(norm), float(eps)
    key = (_sig(q), _sig(k), _sig(positions), _sig(freq), _sig(q_gamma), _sig(k_gamma), _sig(q_out), _sig(k_out),
           interleaved, rot_first, mscale, norm, eps)
    plan = _plans["qk"].get(key)
    if plan is None:
        plan = _plan("qk", key, _qk_plan, q, k, None, positions, freq, q_gamma, k_gamma, q_out, k_out, None, None, None, None,
                     interleaved, rot_first, mscale, norm, eps, 0)
    fn, dev, desc, _ = plan
    if q_out is None and q is not None:
        q_out = torch.empty_like(q, dtype=_BF16, memory_format=_CONTIGUOUS)
    if k_out is None:
        k_out = torch.empty_like(k, dtype=_BF16, memory_format=_CONTIGUOUS)
    _call("dsk_qk_norm_rope", fn, dev, desc, _p(q), k.data_ptr(), positions.data_ptr(), _p(freq), _p(q_gamma),
          _p(k_gamma), _p(q_out), k_out.data_ptr())
    return q_out, k_out


def kv_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, seq: torch.Tensor,
              table: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, freq: torch.Tensor | None = None, *,
              prefix_len: int = 0, interleaved: bool = False, rot_first: int = 0, mscale: float = 1.0,
              q_gamma: torch.Tensor | None = None, k_gamma: torch.Tensor | None = None, norm: bool = True,
              eps: float = 1e-6, q_out: torch.Tensor | None = None,
              k_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """``dsk_kv_append``: ``qk_norm_rope`` whose keys, with the values, go to the paged cache: token t to row
    positions[t] - prefix_len of sequence seq[t] (int32), whose pages are table[seq[t]].  Returns q's result; the keys
    are also written to ``k_out`` if given.  Tokens outside the table or with a page outside the cache are not kept; two
    tokens of one call must not share a row."""
    if not (type(mscale) is type(eps) is float and type(interleaved) is type(norm) is bool and type(rot_first) is int):
        interleaved, rot_first, mscale, norm, eps = bool(interleaved), int(rot_first), float(mscale), bool(norm), float(eps)
    if type(prefix_len) is not int:
        prefix_len = int(prefix_len)
    key = (_sig(q), _sig(k), _sig(v), _sig(positions), _sig(freq), _sig(q_gamma), _sig(k_gamma), _sig(q_out), _sig(k_out),
           _sig(seq), _sig(table), _sig(k_cache), _sig(v_cache), interleaved, rot_first, mscale, norm, eps, prefix_len)
    plan = _plans["append"].get(key)
    if plan is None:
        plan = _plan("append", key, _qk_plan, q, k, v, positions, freq, q_gamma, k_gamma, q_out, k_out, seq, table, k_cache, v_cache,
                     interleaved, rot_first, mscale, norm, eps, prefix_len)
    fn, dev, desc, cache = plan
    if q_out is None and q is not None:
        q_out = torch.empty_like(q, dtype=_BF16, memory_format=_CONTIGUOUS)
    _call("dsk_kv_append", fn, dev, desc, cache, _p(q), k.data_ptr(), v.data_ptr(), positions.data_ptr(), seq.data_ptr(),
          _p(freq), _p(q_gamma), _p(k_gamma), k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), _p(q_out), _p(k_out))
    return q_out


# ------------------------------------------------------------------ attention
def _prompt_plan(q, k, v, cu_q, cu_k, out, causal, scale):
    dev = _hip(q)
    for t, what in ((q, "q"), (k, "k"), (v, "v")):
        _rows(t, what, (_BF16,), dev)
    tokens, heads, dim = q.shape
    if v.shape != k.shape or k.shape[2] != dim:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)}")
    n = cu_q.numel()
    _exact(cu_q, "cu_q", _I32, n, dev)
    _exact(cu_k, "cu_k", _I32, n, dev)
    desc = _lib.PromptDesc(tokens, k.shape[0], n - 1, heads, k.shape[1], dim, 1 if causal else 0,
                           scale if scale is not None else dim ** -0.5,
                           *q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *_out_strides(out, q.shape, dev, "out"))
    return _lib.load().dsk_prompt_attention, dev, ctypes.byref(desc)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
                     cu_k: torch.Tensor | None = None, *, causal: bool = True, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """``dsk_prompt_attention`` over packed sequences: queries cu_q[s] .. cu_q[s+1] with keys cu_k[s] .. cu_k[s+1] (int32;
    cu_k: cu_q).  Causal: query i of Lq sees the keys j <= i + Lk - Lq; one that sees no key gives zeros.  scale:
    head_dim ** -0.5.  Rows of ``out`` behind the last sequence are left as they were."""
    if cu_k is None:
        cu_k = cu_q
    if type(causal) is not bool or not (scale is None or type(scale) is float):
        causal, scale = bool(causal), float(scale) if scale is not None else None
    key = (_sig(q), _sig(k), _sig(v), _sig(cu_q), _sig(cu_k), _sig(out), causal, scale)
    plan = _plans["prompt"].get(key)
    if plan is None:
        plan = _plan("prompt", key, _prompt_plan, q, k, v, cu_q, cu_k, out, causal, scale)
    fn, dev, desc = plan
    if out is None:
        out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    _call("dsk_prompt_attention", fn, dev, desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(),
          out.data_ptr())
    return out


def _token_rows(t: torch.Tensor, q_len: int, what: str) -> torch.Tensor:
    """[batch, q_len, heads, dim] as [batch * q_len, heads, dim], a view."""
    if t.dim() != 4 or t.shape[1] != q_len:
        raise ValueError(f"{what} must be [batch, {q_len}, heads, head_dim], got {tuple(t.shape)}")
    if q_len > 1 and t.shape[0] > 1 and t.stride(0) != q_len * t.stride(1):
        raise ValueError(f"the tokens of {what} must be evenly spaced")
    return t.flatten(0, 1)


def _paged_plan(q, k_cache, v_cache, table, lens, prefix, out, prefix_len, scale):
    """(entry point, device, descriptor, cache, bytes of workspace)."""
    dev = _hip(q)
    q_len = q.shape[1] if q.dim() == 4 else 1
    if q_len < 1:
        raise ValueError("q has no tokens")
    rows = _token_rows(q, q_len, "q") if q.dim() == 4 else q
    _rows(rows, "q", (_BF16,), dev)
    tokens, heads, dim = rows.shape
    kv_heads = k_cache.shape[1] if k_cache.dim() == 4 else 0
    _check_cache(k_cache, v_cache, table, kv_heads, dim, dev)
    batch = table.shape[0]
    if batch < 1 or tokens != batch * q_len:
        raise ValueError(f"q {tuple(q.shape)} does not fit a table of {batch} sequences")
    _exact(lens, "lens", _I32, batch, dev)
    if prefix_len < 0 or (prefix_len > 0) != (prefix is not None):
        raise ValueError("prefix and a positive prefix_len go together")
    if prefix is not None:
        _vector(prefix, "prefix", _I32, -(-prefix_len // k_cache.shape[2]), dev)
    if out is not None and q.dim() == 4:
        out = _token_rows(out, q_len, "out")
    desc = _lib.PagedDesc(batch, q_len, heads, kv_heads, dim, prefix_len,
                          scale if scale is not None else dim ** -0.5, *rows.stride()[:2],
                          *_out_strides(out, rows.shape, dev, "out"))
    cache = ctypes.byref(_cache(k_cache, table))
    n = ctypes.c_size_t(0)
    _lib.call("dsk_paged_attention_workspace_size", ctypes.byref(desc), cache, ctypes.byref(n))
    return _lib.load().dsk_paged_attention, dev, ctypes.byref(desc), cache, n.value


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor,
                    lens: torch.Tensor, *, prefix: torch.Tensor | None = None, prefix_len: int = 0,
                    scale: float | None = None, out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``dsk_paged_attention``: q [batch, heads, head_dim] (one token of each sequence) or [batch, q_len, heads, head_dim]
    over lens[s] (int32) keys of sequence s in the cache, the new tokens' among them (negative: an unused slot, zeros).  ``prefix`` (int32 page ids) with
    ``prefix_len`` keys that all sequences see first, read once for the batch.  The result has q's shape.  ``workspace``:
    uint8, 256-byte aligned, as large as ``dsk_paged_attention_workspace_size`` says, for one call at a time; otherwise
    allocated (inside a graph capture, in the graph's pool)."""
    if type(prefix_len) is not int or not (scale is None or type(scale) is float):
        prefix_len, scale = int(prefix_len), float(scale) if scale is not None else None
    key = (_sig(q), _sig(k_cache), _sig(v_cache), _sig(table), _sig(lens), _sig(prefix), _sig(out), prefix_len, scale)
    plan = _plans["paged"].get(key)
    if plan is None:
        plan = _plan("paged", key, _paged_plan, q, k_cache, v_cache, table, lens, prefix, out, prefix_len, scale)
    fn, dev, desc, cache, nbytes = plan
    if out is None:
        out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    if workspace is None:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    else:
        nbytes = workspace.numel()
        if workspace.device != dev or workspace.dtype != torch.uint8 or not workspace.is_contiguous():
            raise ValueError(f"workspace must be contiguous uint8 on {dev}")
    _call("dsk_paged_attention", fn, dev, desc, cache, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
          table.data_ptr(), lens.data_ptr(), _p(prefix), out.data_ptr(), workspace.data_ptr(), nbytes)
    return out


# ------------------------------------------------------------------ a sublayer
@dataclass
class PromptStep:
    """Whole prompts, packed: prompt i has the rows cu[i] .. cu[i+1]; token t is at positions[t] of sequence seq[t], whose
    pages are table[seq[t]] (all int32 on the device).  A prompt's tokens attend over its own keys alone, so its
    positions are 0, 1, ..; rows of no prompt have position -1.  A step with other positions (a prompt's later part,
    which would not see the keys kept before, or a prompt behind a shared prefix) is refused when it is made, by
    one look at the device's values (40 us, 65 for 8192 tokens); inside a graph capture, and of values written
    later, nothing is looked at."""

    positions: torch.Tensor
    seq: torch.Tensor
    table: torch.Tensor
    cu: torch.Tensor

    def __post_init__(self):
        if self.positions.is_cuda and torch.cuda.is_current_stream_capturing():
            return
        t = self.positions.numel()
        if t < 1 or self.cu.numel() < 2:
            return                       # the calls refuse these themselves
        at, cu = self.positions.cpu().numpy(), self.cu.cpu().numpy().astype(np.int64)
        n = np.diff(cu)
        whole = cu[0] >= 0 and cu[-1] <= t and (n >= 0).all()
        if not (whole and (at[:cu[0]] < 0).all() and (at[cu[-1]:] < 0).all()
                and (at[cu[0]:cu[-1]] == np.arange(cu[0], cu[-1]) - np.repeat(cu[:-1], n)).all()):
            raise ValueError("a PromptStep takes whole prompts: positions 0, 1, .. in the rows cu[i] .. cu[i+1], and -1 in others")

    def idle(self) -> PromptStep:
        """A step of the same sizes that has no sequences and keeps nothing."""
        return replace(self, positions=torch.full_like(self.positions, -1), cu=torch.zeros_like(self.cu))


@dataclass
class DecodeStep:
    """``q_len`` new tokens of every sequence, token t of sequence seq[t] = t // q_len at positions[t]; lens[s] keys of its
    own with them, behind ``prefix_len`` keys of the pages ``prefix`` that all sequences share.  An unused slot: positions
    and length -1."""

    positions: torch.Tensor
    seq: torch.Tensor
    table: torch.Tensor
    lens: torch.Tensor
    q_len: int = 1
    prefix: torch.Tensor | None = None
    prefix_len: int = 0

    def idle(self) -> DecodeStep:
        """A step of the same sizes whose slots are all unused: it keeps nothing."""
        return replace(self, positions=torch.full_like(self.positions, -1), lens=torch.full_like(self.lens, -1))


class Attention:
    """One attention sublayer over bf16 rows y [T, hidden]: y w_qkv^T, norms and rotation, the cache, attention, and the
    output projection w_o.

    w_qkv [(heads + 2 kv_heads) head_dim, hidden]: queries, keys, values; w_o [hidden, heads head_dim] (bf16).  The
    layer owns its cache: ``k_cache`` and ``v_cache`` [pages, kv_heads, page_size, head_dim], which ``new_cache``
    allocates; the steps' tables hold its page ids."""

    def __init__(self, w_qkv: torch.Tensor, w_o: torch.Tensor, heads: int, kv_heads: int, *,
                 freq: torch.Tensor | None = None, mscale: float = 1.0, interleaved: bool = False, rot_first: int = 0,
                 q_gamma: torch.Tensor | None = None, k_gamma: torch.Tensor | None = None, norm: bool = True,
                 eps: float = 1e-6, scale: float | None = None):
        if w_qkv.dim() != 2 or w_o.dim() != 2 or w_qkv.dtype != _BF16 or w_o.dtype != _BF16:
            raise ValueError("w_qkv and w_o must be 2-D bfloat16")
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"heads={heads} must be a multiple of kv_heads={kv_heads}")
        dim, rest = divmod(w_qkv.shape[0], heads + 2 * kv_heads)
        if rest or w_o.shape != (w_qkv.shape[1], heads * dim):
            raise ValueError(f"w_qkv {tuple(w_qkv.shape)} and w_o {tuple(w_o.shape)} do not fit {heads} + 2 x {kv_heads} heads")
        self.w_qkv, self.w_o, self.heads, self.kv_heads, self.head_dim = w_qkv, w_o, heads, kv_heads, dim
        self.scale = scale
        self._rotate = dict(freq=freq, mscale=mscale, interleaved=interleaved, rot_first=rot_first, q_gamma=q_gamma,
                            k_gamma=k_gamma, norm=norm, eps=eps)
        self.k_cache = self.v_cache = None

    def new_cache(self, n_pages: int, page_size: int = 64) -> None:
        """Allocate the layer's pages (zeros)."""
        shape = (n_pages, self.kv_heads, page_size, self.head_dim)
        self.k_cache, self.v_cache = (torch.zeros(shape, dtype=_BF16, device=self.w_qkv.device) for _ in range(2))

    def __call__(self, y: torch.Tensor, step: PromptStep | DecodeStep, out: torch.Tensor | None = None) -> torch.Tensor:
        """The sublayer's output [T, hidden] for y [T, hidden]; its new keys and values are in the cache afterwards.  Rows
        of a ``PromptStep`` behind the last sequence come out as zeros."""
        if self.k_cache is None:
            raise RuntimeError("new_cache() the attention layer first")
        if y.dim() != 2 or y.dtype != _BF16 or y.shape[1] != self.w_qkv.shape[1]:
            raise ValueError(f"y must be bfloat16 [tokens, {self.w_qkv.shape[1]}], got {str(y.dtype)[6:]} {tuple(y.shape)}")
        t, h, kv, d = y.shape[0], self.heads, self.kv_heads, self.head_dim
        qkv = torch.mm(y, self.w_qkv.t())
        q, k, v = (p.view(t, -1, d) for p in qkv.split([h * d, kv * d, kv * d], 1))
        if isinstance(step, PromptStep):
            kr = torch.empty((t, kv, d), dtype=_BF16, device=y.device)
            q = kv_append(q, k, v, step.positions, step.seq, step.table, self.k_cache, self.v_cache, k_out=kr, **self._rotate)
            o = prompt_attention(q, kr, v, step.cu, scale=self.scale, out=torch.zeros_like(q))
        else:
            q = kv_append(q, k, v, step.positions, step.seq, step.table, self.k_cache, self.v_cache,
                          prefix_len=step.prefix_len, **self._rotate)
            o = paged_attention(q.view(-1, step.q_len, h, d), self.k_cache, self.v_cache, step.table, step.lens,
                                prefix=step.prefix, prefix_len=step.prefix_len, scale=self.scale)
        return torch.mm(o.view(t, h * d), self.w_o.t(), out=out) if out is not None else torch.mm(o.view(t, h * d), self.w_o.t())
