"""CPU checks of the cache in 8 bits, the keys' weights, eviction and several rotary axes: what the entry
points refuse before any launch, the frequencies and axes, and the restatement that the GPU tests
compare with."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

import dsk_moe
from dsk_moe import _lib
from dsk_moe import attention as A
from oracle import attention as O

P = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 2)


def qk_desc(**kw):
    base = dict(tokens=4, heads=8, kv_heads=2, head_dim=128, dtype=0, norm=1, rot_dim=64, rot_first=0, interleaved=0,
                prefix_len=0, eps=1e-6, mscale=1.0, q_token=1024, q_head=128, k_token=256, k_head=128, v_token=256,
                v_head=128, qo_token=1024, qo_head=128, ko_token=256, ko_head=128)
    return _lib.QkDesc(**{**base, **kw})


def cache(**kw):
    base = dict(table_stride=8, n_pages=40, page_size=64, n_seqs=4, max_pages=8)
    return _lib.KVCache(**{**base, **kw})


def paged_desc(**kw):
    base = dict(batch=4, q_len=1, heads=8, kv_heads=2, head_dim=128, prefix_len=0, scale=0.1, q_token=1024, q_head=128,
                o_token=1024, o_head=128)
    return _lib.PagedDesc(**{**base, **kw})


def evict_desc(**kw):
    return _lib.EvictDesc(**{**dict(kv_heads=2, head_dim=128, keep=100, first=4, recent=30), **kw})


def axes(**kw):
    return ctypes.byref(_lib.RopeAxes(**{**dict(axis_stride=4, n_axes=3, axis=P), **kw}))


def extra(**kw):
    return ctypes.byref(_lib.KVExtra(**{**dict(k_scale=P, v_scale=P, key_weights=P), **kw}))


def code(name, *args):
    with pytest.raises(_lib.DskError) as e:
        _lib.call(name, *args)
    return e.value.code


# ------------------------------------------------------------------ refusals
def test_structs_have_the_header_s_sizes():
    assert ctypes.sizeof(_lib.RopeAxes) == 24 and ctypes.sizeof(_lib.KVExtra) == 24 and ctypes.sizeof(_lib.EvictDesc) == 20


@pytest.mark.parametrize("kw,want", [(dict(n_axes=0), -1), (dict(n_axes=9), -1), (dict(axis=None), -1), (dict(axis=ODD), -2),
                                     (dict(axis_stride=-4), -1), (dict(axis_stride=(1 << 40) + 1), -1)])
def test_axes_refused(kw, want):
    assert code("dsk_qk_norm_rope_axes", ctypes.byref(qk_desc()), axes(**kw), *[P] * 8, None) == want
    assert code("dsk_kv_append_extra", ctypes.byref(qk_desc()), ctypes.byref(cache()), axes(**kw), extra(), *[P] * 14, None) == want


def test_axes_need_a_rotation():
    d = qk_desc(rot_dim=0)
    assert code("dsk_qk_norm_rope_axes", ctypes.byref(d), axes(), *[P] * 8, None) == -1
    assert code("dsk_qk_norm_rope_axes", ctypes.byref(qk_desc()), None, *[P] * 8, None) == -1
    assert code("dsk_qk_norm_rope_axes", ctypes.byref(qk_desc(tokens=0)), axes(), *[P] * 8, None) == -1


def test_append_refused():
    call = lambda d=qk_desc(), x=extra(), c=cache(), rows=P, v=P, kc=P: code(  # noqa: E731
        "dsk_kv_append_extra", ctypes.byref(d), ctypes.byref(c), axes(), x, P, P, v, P, P, rows, P, P, P, kc, P, P, P, None, None)
    assert call(x=extra(k_scale=None)) == -1 and call(x=extra(v_scale=None)) == -1
    assert call(x=extra(key_weights=ODD)) == -2 and call(rows=ODD) == -2
    assert call(d=qk_desc(prefix_len=5)) == -1                     # rows are rows: no prefix to take off
    assert call(c=cache(page_size=48)) == -1 and call(v=None) == -1 and call(kc=None) == -1 and call(kc=ODD) == -2


def test_paged_refused():
    n = ctypes.c_size_t()
    size = lambda d, x, c=cache(): code(  # noqa: E731
        "dsk_paged_attention_extra_workspace_size", ctypes.byref(d), ctypes.byref(c), x, ctypes.byref(n))
    assert size(paged_desc(), None) == -1 and size(paged_desc(), extra(k_scale=None)) == -1
    assert size(paged_desc(q_len=17), extra()) == -3 and size(paged_desc(), extra(), cache(n_pages=0)) == -1
    call = lambda d=paged_desc(), x=extra(), q=P, ws=P, nbytes=1 << 40: code(  # noqa: E731
        "dsk_paged_attention_extra", ctypes.byref(d), ctypes.byref(cache()), x, q, P, P, P, P, None, P, ws, nbytes, None)
    assert call(x=None) == -1 and call(x=extra(v_scale=None)) == -1 and call(x=extra(key_weights=ODD)) == -2
    assert call(q=None) == -1 and call(ws=ctypes.c_void_p((1 << 20) + 128)) == -2 and call(nbytes=64) == -5
    assert call(d=paged_desc(prefix_len=70)) == -1


def test_workspaces_hold_what_is_asked_for():
    def size(x, **kw):
        n = ctypes.c_size_t()
        _lib.call("dsk_paged_attention_extra_workspace_size", ctypes.byref(paged_desc(**kw)), ctypes.byref(cache(max_pages=32, table_stride=32)),
                  x, ctypes.byref(n))
        return n.value
    plain, codes, weights = extra(k_scale=None, v_scale=None, key_weights=None), extra(key_weights=None), extra(k_scale=None, v_scale=None)
    n = ctypes.c_size_t()
    _lib.call("dsk_paged_attention_workspace_size", ctypes.byref(paged_desc()), ctypes.byref(cache(max_pages=32, table_stride=32)), ctypes.byref(n))
    assert size(plain) == n.value
    # a float32 for each of 4 x 2 items, 4 rows and 2048 places
    assert size(weights) >= size(plain) + 4 * 2 * 4 * 2048 * 4
    # the prefix's partial rows: a float32 row, a maximum and a sum for each of 4 x 8 query rows
    assert size(codes, prefix_len=100) >= size(codes) + 4 * 8 * (128 + 2) * 4


@pytest.mark.parametrize("kw,want", [(dict(kv_heads=0), -1), (dict(kv_heads=1025), -1), (dict(head_dim=80), -3), (dict(keep=0), -1),
                                     (dict(first=-1), -1), (dict(recent=-1), -1), (dict(first=71), -1),
                                     (dict(first=(1 << 31) - 1, recent=(1 << 31) - 1), -1)])
def test_evict_refused(kw, want):
    n = ctypes.c_size_t()
    d = evict_desc(**kw)
    assert code("dsk_kv_evict_workspace_size", ctypes.byref(d), ctypes.byref(cache()), extra(), ctypes.byref(n)) == want
    assert code("dsk_kv_evict", ctypes.byref(d), ctypes.byref(cache()), extra(), *[P] * 6, 1 << 40, None) == want


def test_evict_refuses_pointers_space_and_sizes():
    q = ctypes.c_void_p(1 << 21)
    call = lambda x=extra(), c=cache(), kc=P, table=P, lens=P, out=q, ws=P, n=1 << 40: code(  # noqa: E731
        "dsk_kv_evict", ctypes.byref(evict_desc()), ctypes.byref(c), x, kc, P, table, lens, out, ws, n, None)
    assert call(x=None) == -1 and call(x=extra(key_weights=None)) == -1 and call(x=extra(k_scale=None)) == -1
    assert call(kc=None) == -1 and call(kc=ODD) == -2 and call(table=None) == -1 and call(lens=None) == -1 and call(out=None) == -1
    assert call(ws=None) == -1 and call(ws=ctypes.c_void_p((1 << 20) + 128)) == -2 and call(n=64) == -5
    assert call(out=ctypes.c_void_p((1 << 20) + 8)) == -1          # neither lens nor apart from it
    assert call(lens=ODD) == -2
    size = ctypes.c_size_t()
    many = cache(n_seqs=1 << 21)
    assert code("dsk_kv_evict_workspace_size", ctypes.byref(evict_desc()), ctypes.byref(many), extra(), ctypes.byref(size)) == -3


def test_functions_refuse_cpu_tensors_and_other_caches():
    b, i = torch.zeros(4, 2, 64, 128, dtype=torch.bfloat16), torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        dsk_moe.kv_evict(b, b, torch.zeros(4, 2, 64), i, i[0, :1], 2)
    # numbers that 32 bits would make others of
    for bad in (dict(keep=(1 << 32) + 2), dict(keep=1 << 31), dict(keep=8, first=1 << 32), dict(keep=8, recent=-(1 << 32))):
        with pytest.raises(ValueError, match="keep"):
            dsk_moe.kv_evict(b, b, torch.zeros(4, 2, 64), i, i[0, :1], **bad)
    check = lambda k=b.to(torch.float8_e4m3fn), s=torch.zeros(4, 2, 4, dtype=torch.uint8), v=None, w=None: A._check_cache(  # noqa: E731
        k, k, i, 2, 128, torch.device("cpu"), s, s if v is None else v, w)
    check()
    check(w=torch.zeros(4, 2, 64))
    for kw, text in ((dict(k=b), "float8_e4m3fn"), (dict(s=None), "go together|float8"), (dict(s=torch.zeros(4, 2, 64, dtype=torch.uint8)), "k_scale"),
                     (dict(v=torch.zeros(4, 2, 4)), "v_scale"), (dict(w=torch.zeros(4, 2, 4)), "key_weights"),
                     (dict(w=torch.zeros(4, 2, 64).bfloat16()), "key_weights")):
        with pytest.raises(ValueError, match=text):
            check(**kw)
    with pytest.raises(ValueError, match="go together"):
        A._check_cache(b, b, i, 2, 128, torch.device("cpu"), torch.zeros(4, 2, 4, dtype=torch.uint8), None)


def test_steps_on_several_axes_name_their_rows():
    ints = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    pos = ints([[0, 1, 2, 2], [0, 1, 2, 2], [0, 1, 2, 3]])
    with pytest.raises(ValueError, match="give rows"):
        dsk_moe.PromptStep(pos, ints([0] * 4), ints([[0]]), ints([0, 4]))
    step = dsk_moe.PromptStep(pos, ints([0] * 4), ints([[0]]), ints([0, 4]), rows=ints([0, 1, 2, 3]))
    assert step.idle().positions.shape == pos.shape and (step.idle().positions == -1).all()
    for rows in ([0, 1, 3, 2], [4, 5, 6, 7], [0, 1, 2, -1]):
        with pytest.raises(ValueError, match="whole prompts"):
            dsk_moe.PromptStep(pos, ints([0] * 4), ints([[0]]), ints([0, 4]), rows=ints(rows))


@pytest.mark.parametrize("axes", [None, 1, 3])
def test_prompt_steps_with_rows_refuse_tokens_that_would_be_left_out(axes):
    """A negative position of a prompt's token on any axis: its key would not be written, and its prompt would read it."""
    ints = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    rows, cu = ints([-1, 0, 1, 2, 0, 1, -1]), ints([1, 4, 4, 6])

    def step(pos):
        return dsk_moe.PromptStep(pos, ints([0, 0, 0, 0, 1, 1, 0]), ints([[0], [1]]), cu, rows=rows)

    good = torch.where(rows >= 0, 5 + rows, -1)
    good = good if axes is None else good.repeat(axes, 1)
    step(good)
    step(torch.full_like(good, 9))                                  # tokens of no prompt are not kept wherever they are
    for t in (1, 2, 5):
        bad = good.clone()
        bad[(-1, t) if axes else t] = -1
        with pytest.raises(ValueError, match="not negative"):
            step(bad)
    with pytest.raises(ValueError, match="7 tokens"):
        step(good[..., :6])


def test_decode_steps_on_several_axes_name_their_rows():
    ints = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="give rows"):
        dsk_moe.DecodeStep(ints([[5], [6]]), ints([0]), ints([[0]]), ints([6]))
    step = dsk_moe.DecodeStep(ints([[5], [6]]), ints([0]), ints([[0]]), ints([6]), rows=ints([5]))
    assert (step.idle().positions == -1).all() and step.idle().lens.tolist() == [-1]


def test_caches_and_stacks_refuse_what_they_cannot_keep():
    w = torch.zeros((8 + 4) * 64, 256, dtype=torch.bfloat16)
    att = dsk_moe.Attention(w, torch.zeros(256, 512, dtype=torch.bfloat16), 8, 2)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        att.new_cache(4, dtype=torch.float16)
    with pytest.raises(ValueError, match="weigh"):
        att.new_cache(4, weigh=17)
    att.new_cache(4, 32, dtype=torch.float8_e4m3fn, weigh=16)
    assert [tuple(t.shape) for t in att.cache_tensors()] == [(4, 2, 32, 64)] * 2 + [(4, 2, 2)] * 2 + [(4, 2, 32)]
    att.new_cache(4)
    assert att.cache_tensors()[2:] == (None, None, None)
    with pytest.raises(RuntimeError, match="weigh"):
        att.evict(None, None, 4)


class FakeAttention:
    """What ``MoEStack.evict`` asks of an attention sublayer: every sequence is cut down to 4 keys."""

    key_weights = torch.zeros(1)

    def evict(self, table, lens, keep, *, first, recent):
        return lens.clamp(max=keep)


def test_stack_evict_refuses_rows_and_lengths_that_are_other_tensors_too():
    """Before the first eviction positions and rows count the same, but rows are taken back and positions are not."""
    ints = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    stack = dsk_moe.MoEStack([object()], attention=[FakeAttention()])
    pos, seq, table = ints([9, 3]), ints([0, 1]), ints([[0], [1]])
    step = dsk_moe.DecodeStep(pos, seq, table, pos + 1, rows=pos.clone())
    stack.evict(step, 4)
    assert step.lens.tolist() == [4, 4] and step.rows.tolist() == [3, 3] and pos.tolist() == [9, 3]
    three, buffer = pos.repeat(3, 1), ints([9, 3, 10, 4])
    for bad in (dict(positions=pos, rows=pos), dict(positions=three, rows=three[2]), dict(positions=pos, rows=pos.view(2)),
                dict(positions=pos.clone(), rows=buffer[:2], lens=buffer[1:3]), dict(positions=buffer[2:], rows=pos, lens=buffer[2:])):
        held = [t.clone() for t in bad.values()]
        with pytest.raises(ValueError, match="shares memory"):
            stack.evict(dsk_moe.DecodeStep(**{**dict(seq=seq, table=table, lens=ints([10, 4])), **bad}), 4)
        assert all(torch.equal(t, h) for t, h in zip(bad.values(), held))
    stack.evict(dsk_moe.DecodeStep(pos, seq, table, buffer[2:], rows=buffer[:2]), 4)     # next to each other
    assert buffer.tolist() == [3, 3, 4, 4]


# ------------------------------------------------------------------ plans
class Records:
    """Stands in for torch's record of tensors' properties, and counts."""

    def __init__(self, fault=None):
        self.fault, self.made, self.asked = fault, 0, 0

    def __call__(self, *tensors, **kw):
        self.made += 1
        if self.fault == "raises":
            raise TypeError("other arguments")
        kinds = [(t.shape, t.dtype) for t in tensors]
        records = self

        class Record:
            def check(self, *given):
                records.asked += 1
                return records.fault is None and [(t.shape, t.dtype) for t in given] == kinds
        return Record()


def find(plans, *tensors):
    return plans.find((1, 0.5), tensors, tensors)


def test_plans_of_a_kind_are_made_once():
    made = []
    plans = A._Plans(lambda *tensors: made.append(tensors) or tuple(t.shape for t in tensors))
    a, b = torch.zeros(3, 4), torch.zeros(5)
    for _ in range(4):
        assert find(plans, a, b) == (a.shape, b.shape) and find(plans, b, a) == (b.shape, a.shape)
    assert find(plans, a.double(), b) == (a.shape, b.shape)         # another kind
    assert find(plans, torch.zeros(4, 3).t(), b) == (a.shape, b.shape)
    assert len(made) == 4


@pytest.mark.parametrize("real", [False, True])
def test_plans_record_no_call_that_a_record_cannot_find(monkeypatch, real):
    """A tensor given twice is never found by torch's record: such calls ask the dictionary alone, and leave the records of others in place."""
    if real and A._Properties is None:
        pytest.skip("this torch has no record of tensors' properties")
    records = Records()
    if not real:
        monkeypatch.setattr(A, "_Properties", records)
    plans = A._Plans(lambda *tensors: object())
    one, two = torch.zeros(3, 4), torch.zeros(3, 4)
    apart = find(plans, one, two)
    assert find(plans, one, two) is apart and len(plans._recent) == 1
    for _ in range(600):
        assert find(plans, one, one) is apart                       # (of the same kind: what is checked is the same)
    assert len(plans._recent) == 1
    plans = A._Plans(lambda *tensors: object())
    both = find(plans, one, one)
    for _ in range(600):
        assert find(plans, one, one) is both
    assert not plans._recent


def test_plans_record_no_kind_that_comes_once(monkeypatch):
    """Prompts of ever new lengths: a record of each would cost more than it finds."""
    records = Records()
    monkeypatch.setattr(A, "_Properties", records)
    plans = A._Plans(lambda *tensors: object())
    for n in range(1, 50):
        find(plans, torch.zeros(n), torch.zeros(n, 1))
    assert not plans._recent and records.made == 0
    find(plans, torch.zeros(7), torch.zeros(7, 1))
    assert len(plans._recent) == 1


@pytest.mark.parametrize("fault", ["raises", "never finds"])
def test_plans_do_without_a_record_that_does_not_work(monkeypatch, fault):
    records = Records(fault)
    monkeypatch.setattr(A, "_Properties", records)
    plans = A._Plans(lambda *tensors: object())
    a, b = torch.zeros(3, 4), torch.zeros(5)
    plan = find(plans, a, b)
    for _ in range(100):
        assert find(plans, a, b) is plan
    assert not plans._recent and 0 < records.made < 10
    monkeypatch.setattr(A, "_Properties", None)
    assert find(plans, a, b) is plan


# ------------------------------------------------------------------ axes
def test_rope_axes():
    f, a = dsk_moe.rope_axes([16, 24, 24], device="cpu")
    assert a.tolist() == [0] * 16 + [1] * 24 + [2] * 24 and f.dtype == torch.float64 and a.dtype == torch.int32
    assert torch.allclose(f, dsk_moe.rope_frequencies(128, device="cpu")[0], rtol=1e-14)
    f, a = dsk_moe.rope_axes([2, 4, 2], in_turn=True, device="cpu")
    assert a.tolist() == [0, 1, 2, 0, 1, 2, 1, 1]
    f, a = dsk_moe.rope_axes([8, 8], each=True, base=100.0, device="cpu")
    assert torch.equal(f[:8], f[8:]) and math.isclose(float(f[1]), 100.0 ** (-1 / 8))
    f, a = dsk_moe.rope_axes([0, 8], each=True, device="cpu")
    assert a.tolist() == [1] * 8
    for kw in (dict(sections=[]), dict(sections=[4]), dict(sections=[-8, 16]), dict(sections=[0, 0]), dict(sections=[1] * 9),
               dict(sections=[8], base=0.0)):
        with pytest.raises(ValueError):
            dsk_moe.rope_axes(**{"device": "cpu", **kw})


# ------------------------------------------------------------------ the restatement itself
def test_oracle_codes_are_e4m3():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double()
    one = torch.tensor(127)
    assert torch.equal(O._CODES.nan_to_num(999.0), want.nan_to_num(999.0))
    real = ~want.isnan()
    assert torch.equal(O.to_codes(want[real], one), codes[real])
    x = torch.cat([torch.randn(4000, dtype=torch.float64) * 10.0 ** e for e in (-3, -2, -1, 0, 1, 2)]).float()
    x = torch.cat([x, (want[real][1:] + want[real][:-1]).float() / 2]).clamp(-448, 448)       # and the middles
    assert torch.equal(O.to_codes(x.double(), one).view(torch.float8_e4m3fn).double(), x.to(torch.float8_e4m3fn).double())
    assert O.to_codes(torch.tensor([math.inf, -math.inf, math.nan, 1e9], dtype=torch.float64), one).tolist() == [127, 127, 127, 126]


def test_oracle_scale_is_the_least_that_holds():
    for top in (1.0, 448.0, 448.0000001, 1.75, 1.7500001, 3e-5, 1e20, 6.0):
        b = O.scale_byte(top)
        assert top <= 448.0 * 2.0 ** (b - 127) and top > 448.0 * 2.0 ** (b - 128)
    assert O.scale_byte(0.0) == O.LEAST and O.scale_byte(3e38) == O.MOST and O.scale_byte(1e-45) == O.LEAST


def test_oracle_rows_move_to_a_larger_scale():
    c = torch.arange(256, dtype=torch.uint8)
    two = O.rescale(c, 100, 101)
    want = O._CODES / 2
    exact = want.abs() >= 2.0 ** -6                     # normal codes: their exponents alone
    assert torch.equal(O._CODES[two.long()][exact], want[exact])
    assert (O._CODES[two.long()] - want).abs().nan_to_num(0.0).max() <= 2.0 ** -10
    assert torch.equal(two[127:128], c[127:128]) and O.rescale(c, 27, 246).long().bitwise_and(127)[:127].max() == 0


def test_oracle_weights_are_the_softmax():
    q, k = torch.randn(3, 4, 16, dtype=torch.float64), torch.randn(9, 2, 16, dtype=torch.float64)
    last = torch.tensor([6, 7, 8])
    w, _ = O.key_weights(q, k, last, 0.25)
    s = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(2, 1)) * 0.25
    s = s.masked_fill(torch.arange(9)[None] > last[:, None], -math.inf)
    want = torch.softmax(s, -1).sum(1).view(2, 2, 9).sum(1).t()
    assert torch.allclose(w, want, atol=1e-12) and math.isclose(float(w.sum()), 12.0)


def test_oracle_rows_of_a_head_at_once():
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(n, h, 16, generator=g) for n, h in ((3, 6), (11, 2), (11, 2)))
    for last in ([8, 9, 10], [-2, 0, 10], [10, 10, 12]):
        for got, want in zip(O.attention_of_many(q, k, v, torch.tensor(last), 0.3), O.attention(q, k, v, torch.tensor(last), 0.3)):
            assert torch.allclose(got, want, rtol=1e-11, atol=1e-14)


def test_oracle_eviction_by_hand():
    """Eight keys, five kept, one first and two recent: of the middle five those of weight 9 and 5."""
    page = 16
    rows = torch.arange(8, dtype=torch.float64)
    k = torch.zeros(1, 1, page, 1, dtype=torch.float64)
    k[0, 0, :8, 0] = rows
    w = torch.zeros(1, 1, page)
    w[0, 0, :8] = torch.tensor([0.0, 1.0, 5.0, 3.0, 9.0, 5.0, 0.0, 0.0])
    new = O.evict([(k, None)], w, torch.tensor([[0]]), [8], 5, 1, 2, page)
    # row 0; holes 1 and (2 stays): row 4 comes to 1; the last two follow
    assert new == [5] and k[0, 0, :8, 0].tolist() == [0, 4, 2, 6, 7, 5, 6, 7]
    assert w[0, 0, :5].tolist() == [0.0, 9.0, 5.0, 0.0, 0.0]
    assert O.evict([(k, None)], w, torch.tensor([[0]]), [5], 5, 1, 2, page) == [5]


def test_oracle_norm_rope_takes_a_position_for_each_pair():
    x = torch.randn(3, 2, 32)
    pos, f = torch.tensor([[1, 2, 3], [5, 6, 7]]), torch.rand(16, dtype=torch.float64)
    axis = torch.tensor([0, 1] * 8)
    y, _ = O.norm_rope(x, pos[axis].t(), f)
    for a in range(2):
        z, _ = O.norm_rope(x, pos[a], f)
        assert np.array_equal(y[..., a:16:2], z[..., a:16:2]) and np.array_equal(y[..., 16 + a::2], z[..., 16 + a::2])
