"""CPU checks of the attention entry points: what they refuse (before any
launch, so no GPU is needed), the rotation's frequencies, and the float64
restatement that the GPU tests compare with."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import dsk_moe
from dsk_moe import _lib
from dsk_moe import attention as A
from oracle import attention as O

P = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 8)


def qk_desc(**kw):
    base = dict(tokens=4, heads=8, kv_heads=2, head_dim=128, dtype=0, norm=1, rot_dim=64, rot_first=0, interleaved=0,
                prefix_len=0, eps=1e-6, mscale=1.0, q_token=1024, q_head=128, k_token=256, k_head=128, v_token=256,
                v_head=128, qo_token=1024, qo_head=128, ko_token=256, ko_head=128)
    return _lib.QkDesc(**{**base, **kw})


def cache(**kw):
    base = dict(table_stride=8, n_pages=40, page_size=64, n_seqs=4, max_pages=8)
    return _lib.KVCache(**{**base, **kw})


def prompt_desc(**kw):
    base = dict(tokens=10, kv_tokens=10, n_seqs=2, heads=8, kv_heads=2, head_dim=64, causal=1, scale=0.1, q_token=512,
                q_head=64, k_token=128, k_head=64, v_token=128, v_head=64, o_token=512, o_head=64)
    return _lib.PromptDesc(**{**base, **kw})


def paged_desc(**kw):
    base = dict(batch=4, q_len=1, heads=8, kv_heads=2, head_dim=128, prefix_len=0, scale=0.1, q_token=1024, q_head=128,
                o_token=1024, o_head=128)
    return _lib.PagedDesc(**{**base, **kw})


def code(name, *args):
    with pytest.raises(_lib.DskError) as e:
        _lib.call(name, *args)
    return e.value.code


def rope_code(desc, q=P, k=P, pos=P, freq=P, gq=P, gk=P, qo=P, ko=P):
    return code("dsk_qk_norm_rope", ctypes.byref(desc), q, k, pos, freq, gq, gk, qo, ko, None)


@pytest.mark.parametrize("kw,want", [
    (dict(tokens=0), -1), (dict(head_dim=96), -3), (dict(heads=-1), -1), (dict(heads=1025), -1), (dict(kv_heads=0), -1),
    (dict(dtype=2), -1), (dict(rot_dim=24), -1), (dict(rot_dim=144), -1), (dict(rot_first=4), -1),
    (dict(rot_first=72), -1), (dict(rot_dim=-16), -1), (dict(eps=-1.0), -1), (dict(eps=math.nan), -1),
    (dict(mscale=math.inf), -1), (dict(norm=0), -1), (dict(q_token=1025), -2), (dict(k_head=-8), -1),
    (dict(dtype=1, q_token=1026), -2), (dict(qo_head=64), -1), (dict(ko_token=0), -1), (dict(qo_token=1020), -1),
    (dict(tokens=(1 << 23) + 1), -3)])
def test_norm_rope_refuses(kw, want):
    assert rope_code(qk_desc(**kw)) == want


def test_norm_rope_refuses_pointers():
    assert rope_code(qk_desc(), q=None) == -1 and rope_code(qk_desc(), ko=None) == -1
    assert rope_code(qk_desc(), freq=None) == -1 and rope_code(qk_desc(heads=0)) == -1
    assert rope_code(qk_desc(), q=ODD) == -2 and rope_code(qk_desc(), ko=ODD) == -2
    assert rope_code(qk_desc(), pos=ctypes.c_void_p(5)) == -2
    assert code("dsk_qk_norm_rope", None, P, P, P, P, P, P, P, P, None) == -1


@pytest.mark.parametrize("kw,want", [(dict(page_size=48), -1),
                                     (dict(page_size=512), -1), (dict(n_pages=0), -1), (dict(n_seqs=0), -1),
                                     (dict(max_pages=0), -1), (dict(table_stride=7), -1),
                                     (dict(max_pages=1 << 24, table_stride=1 << 24), -3)])
def test_cache_refuses(kw, want):
    c = cache(**kw)
    assert code("dsk_kv_append", ctypes.byref(qk_desc()), ctypes.byref(c), *[P] * 13, None) == want
    size = ctypes.c_size_t()
    assert code("dsk_paged_attention_workspace_size", ctypes.byref(paged_desc()), ctypes.byref(c), ctypes.byref(size)) == want


def test_append_refuses():
    call = lambda d, v=P, seq=P, c=cache(), ko=None, kc=P, vc=P, table=P: code(  # noqa: E731
        "dsk_kv_append", ctypes.byref(d), ctypes.byref(c) if c else None, P, P, v, P, seq, P, P, P, kc, vc, table, P, ko, None)
    assert call(qk_desc(), kc=None) == -1 and call(qk_desc(), vc=None) == -1 and call(qk_desc(), table=None) == -1
    assert call(qk_desc(), kc=ODD) == -2 and call(qk_desc(), vc=ODD) == -2
    assert call(qk_desc(), v=None) == -1 and call(qk_desc(), seq=None) == -1 and call(qk_desc(), c=None) == -1
    assert call(qk_desc(prefix_len=-1)) == -1 and call(qk_desc(v_token=250)) == -2 and call(qk_desc(), v=ODD) == -2
    assert call(qk_desc(ko_token=0), ko=P) == -1


@pytest.mark.parametrize("kw,want", [
    (dict(tokens=0), -1), (dict(kv_tokens=0), -1), (dict(n_seqs=0), -1), (dict(n_seqs=65536), -1), (dict(head_dim=80), -3),
    (dict(heads=9), -1), (dict(heads=0), -1), (dict(heads=130, kv_heads=2), -1), (dict(scale=0.0), -1),
    (dict(scale=math.nan), -1), (dict(tokens=1 << 28), -3), (dict(kv_tokens=1 << 30), -3), (dict(k_token=130), -2),
    (dict(o_token=256), -1), (dict(v_token=1 << 26), -3), (dict(n_seqs=65535, heads=1024, kv_heads=1024), -3)])
def test_prompt_refuses(kw, want):
    assert code("dsk_prompt_attention", ctypes.byref(prompt_desc(**kw)), P, P, P, P, P, P, None) == want


def test_prompt_refuses_pointers():
    for i in range(6):
        args = [P] * 6
        args[i] = None
        assert code("dsk_prompt_attention", ctypes.byref(prompt_desc()), *args, None) == -1
        args[i] = ctypes.c_void_p((1 << 20) + 2)
        assert code("dsk_prompt_attention", ctypes.byref(prompt_desc()), *args, None) == -2


@pytest.mark.parametrize("kw,want", [(dict(batch=0), -1), (dict(batch=3), -1), (dict(q_len=0), -3), (dict(q_len=17), -3),
                                     (dict(q_len=9, heads=16), -3), (dict(prefix_len=-1), -1), (dict(prefix_len=1 << 30), -1),
                                     (dict(scale=-1.0), -1), (dict(q_head=60), -2), (dict(o_head=0), -1),
                                     (dict(head_dim=256), -3)])
def test_paged_refuses(kw, want):
    size = ctypes.c_size_t()
    assert code("dsk_paged_attention_workspace_size", ctypes.byref(paged_desc(**kw)), ctypes.byref(cache()),
                ctypes.byref(size)) == want
    assert code("dsk_paged_attention", ctypes.byref(paged_desc(**kw)), ctypes.byref(cache()), *[P] * 8, 1 << 40, None) == want


def test_paged_refuses_pointers_and_space():
    call = lambda d, q=P, lens=P, prefix=None, out=P, ws=P, n=1 << 40, kc=P, table=P: code(  # noqa: E731
        "dsk_paged_attention", ctypes.byref(d), ctypes.byref(cache()), q, kc, P, table, lens, prefix, out, ws, n, None)
    assert call(paged_desc(), kc=None) == -1 and call(paged_desc(), table=None) == -1 and call(paged_desc(), kc=ODD) == -2
    assert call(paged_desc(), q=None) == -1 and call(paged_desc(), lens=None) == -1 and call(paged_desc(), ws=None) == -1
    assert call(paged_desc(prefix_len=5)) == -1
    assert call(paged_desc(), out=ODD) == -2 and call(paged_desc(), ws=ctypes.c_void_p((1 << 20) + 128)) == -2
    assert call(paged_desc(), n=128) == -5


def test_paged_refuses_more_work_than_it_counts():
    """Units of 128 keys are counted in 31 bits, over the batch and the key heads."""
    size = ctypes.c_size_t()
    wide = cache(n_seqs=65535, page_size=256, max_pages=1 << 20, table_stride=1 << 20)
    assert code("dsk_paged_attention_workspace_size", ctypes.byref(paged_desc(batch=65535, kv_heads=8)), ctypes.byref(wide),
                ctypes.byref(size)) == -3
    for heads, pages in ((8, 1 << 11), (1, 1 << 14)):                  # just below 2^31
        c = cache(n_seqs=65535, page_size=256, max_pages=pages - 1, table_stride=pages)
        _lib.call("dsk_paged_attention_workspace_size", ctypes.byref(paged_desc(batch=65535, heads=heads, kv_heads=heads)), ctypes.byref(c),
                  ctypes.byref(size))


def test_paged_workspace_grows_with_the_batch():
    size = lambda **kw: (lambda n: (_lib.call(  # noqa: E731
        "dsk_paged_attention_workspace_size", ctypes.byref(paged_desc(**kw)), ctypes.byref(cache(n_seqs=kw.get("batch", 4), max_pages=32, table_stride=32)),
        ctypes.byref(n)), n.value)[1])(ctypes.c_size_t())
    assert 0 < size() < size(batch=8) and size() < size(prefix_len=1) and size() % 256 == 0


def test_paged_items_for_more_threads_than_a_launch_counts():
    """2^23 items in short tables: not one workgroup of 512 threads for each, but shares, which need partial rows."""
    size = ctypes.c_size_t()
    for batch, shares in ((8191, False), (8192, True)):
        d = paged_desc(batch=batch, heads=1024, kv_heads=1024, head_dim=64, q_token=65536, q_head=64, o_token=65536, o_head=64)
        c = cache(n_seqs=batch, page_size=16, max_pages=4, table_stride=4)
        _lib.call("dsk_paged_attention_workspace_size", ctypes.byref(d), ctypes.byref(c), ctypes.byref(size))
        assert (size.value > 256) == shares


def test_functions_refuse_cpu_tensors():
    q = torch.zeros(4, 8, 128, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        dsk_moe.qk_norm_rope(q, q, i)
    with pytest.raises(ValueError, match="HIP device"):
        dsk_moe.prompt_attention(q, q, q, i)
    with pytest.raises(ValueError, match="HIP device"):
        dsk_moe.paged_attention(q, q, q, i, i)


def test_frequencies():
    f, m = dsk_moe.rope_frequencies(64, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and m == 1.0
    assert f[0] == 1.0 and math.isclose(float(f[31]), 10000.0 ** (-62 / 64), rel_tol=1e-14)
    g, m = dsk_moe.rope_frequencies(64, scaling="linear", factor=4.0, device="cpu")
    assert m == 1.0 and torch.allclose(g, f / 4, rtol=1e-14)
    g, _ = dsk_moe.rope_frequencies(64, scaling="base", factor=4.0, device="cpu")
    assert g[0] == 1.0 and math.isclose(float(g[31]), float(f[31]) / 4, rel_tol=1e-12)
    g, m = dsk_moe.rope_frequencies(64, scaling="ramp", factor=4.0, original_len=4096, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert math.isclose(m, 0.1 * math.log(4.0) + 1.0)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.allclose(g[turns <= 1], f[turns <= 1] / 4, rtol=1e-14)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and bool(((g < f) & (g > f / 4))[mid].all())
    for kw in (dict(rot_dim=24), dict(rot_dim=0), dict(rot_dim=32, base=-1.0), dict(rot_dim=32, scaling="other"),
               dict(rot_dim=32, scaling="linear", factor=0.5), dict(rot_dim=32, scaling="ramp", factor=2.0, turns=(4.0, 4.0))):
        with pytest.raises(ValueError):
            dsk_moe.rope_frequencies(**{"device": "cpu", **kw})


# ------------------------------------------------------------------ the restatement itself
def test_oracle_rotation_is_a_complex_turn():
    x = torch.randn(3, 2, 32, dtype=torch.float64)
    pos, f = torch.tensor([0, 5, 1 << 20]), torch.tensor([1.0, 0.1, 0.01, 0.001] * 2, dtype=torch.float64)
    y, _ = O.norm_rope(x, pos, f, interleaved=True, rot_first=8, norm=False)
    z = torch.view_as_complex(x[..., 8:24].reshape(3, 2, 8, 2).contiguous())
    z = z * torch.polar(torch.ones(8, dtype=torch.float64), pos.double()[:, None] * f)[:, None]
    assert torch.allclose(torch.view_as_real(z).flatten(-2), y[..., 8:24], atol=1e-12)
    assert torch.equal(y[..., :8], x[..., :8]) and torch.equal(y[..., 24:], x[..., 24:])


def test_oracle_attention_against_torch():
    q, k, v = (torch.randn(n, 4, 16, dtype=torch.float64) for n in (5, 9, 9))
    o, _ = O.attention(q, k, v, torch.arange(5) + 4, 0.25)
    mask = torch.arange(9)[None] <= torch.arange(5)[:, None] + 4
    want = torch.nn.functional.scaled_dot_product_attention(*(t.transpose(0, 1) for t in (q, k, v)), attn_mask=mask, scale=0.25)
    assert torch.allclose(o, want.transpose(0, 1), atol=1e-12)
    o, _ = O.attention(q, k, v, torch.tensor([-2, -1, 0, 1, 2]), 0.25)
    assert not o[:2].any() and torch.allclose(o[2], v[0])


def test_prompt_steps_are_whole_prompts():
    ints = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    step = lambda pos, cu: dsk_moe.PromptStep(ints(pos), ints([0] * len(pos)), ints([[0]]), ints(cu))  # noqa: E731
    for pos, cu in (([0, 1, 2, 0, -1], [0, 3, 4]), ([0], [0, 1]), ([0, 1, 0], [0, 0, 2, 2, 3]), ([-1, -1], [0, 0])):
        idle = step(pos, cu).idle()
        assert idle.positions.tolist() == [-1] * len(pos) and idle.cu.tolist() == [0] * len(cu)
    for pos, cu in (([4, 5], [0, 2]), ([0, 1, 3, 4], [0, 2, 4]), ([0, 1, 2], [0, 2]), ([0, -1], [0, 2]), ([0, 1], [0, 3]), ([0, 1], [0, 2, 1])):
        with pytest.raises(ValueError, match="whole prompts"):
            step(pos, cu)


def overlaps(token, head, tokens, heads, dim):
    at = sorted(t * token + h * head for t in range(tokens) for h in range(heads))
    return any(b - a < dim for a, b in zip(at, at[1:]))


@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 4), (2, 1), (2, 2), (3, 4), (10, 2), (12, 8)])
def test_outputs_whose_rows_overlap_are_refused(tokens, heads):
    """Every output, over strides from none to far apart, against all rows' places (a NULL input, which is looked for before or
    behind the strides, ends the others)."""
    d, refused = 64, 0
    n = ctypes.c_size_t()
    strides = [0, 8, 56, 64, 72, 96, 128, 192, 256, 264, 384, 512, 576, 640, 704, 768, 1024, 1280, 2048]
    for token in strides:
        for head in strides:
            want = overlaps(token, head, tokens, heads, d)
            refused += want
            p = prompt_desc(tokens=tokens, heads=heads, kv_heads=heads, o_token=token, o_head=head, k_token=1 << 26)
            with pytest.raises(_lib.DskError) as e:
                _lib.call("dsk_prompt_attention", ctypes.byref(p), P, P, P, P, P, P, None)
            assert ("rows of out overlap" in str(e.value)) == want, (token, head)
            for q_len in ({1, tokens} if tokens < 10 else {1, 2}):
                if tokens % q_len:
                    continue
                batch = tokens // q_len
                g = paged_desc(batch=batch, q_len=q_len, heads=heads, kv_heads=heads, head_dim=d, o_token=token, o_head=head)
                c = cache(n_seqs=batch)
                if want:
                    assert code("dsk_paged_attention_workspace_size", ctypes.byref(g), ctypes.byref(c), ctypes.byref(n)) == -1
                else:
                    _lib.call("dsk_paged_attention_workspace_size", ctypes.byref(g), ctypes.byref(c), ctypes.byref(n))
            r = qk_desc(tokens=tokens, heads=heads, kv_heads=heads, head_dim=d, rot_dim=32, qo_token=token, qo_head=head)
            with pytest.raises(_lib.DskError) as e:
                _lib.call("dsk_qk_norm_rope", ctypes.byref(r), P, P, P, P, P, P, P, None, None)
            assert ("rows of q_out overlap" in str(e.value)) == want, (token, head)
            if want:
                r = qk_desc(tokens=tokens, heads=heads, kv_heads=heads, head_dim=d, rot_dim=32, qo_token=heads * d, qo_head=d, ko_token=token,
                            ko_head=head)
                assert rope_code(r) == -1
                assert code("dsk_kv_append", ctypes.byref(r), ctypes.byref(cache()), *[P] * 13, None) == -1
    assert refused or tokens * heads == 1
