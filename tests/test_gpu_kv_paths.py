"""GPU parity of the cache in 8 bits and the keys' weights where only certain sizes and values lead: sums of a prefix
whose weights all round alike."""

from __future__ import annotations

import math

import pytest
import torch

import dsk_moe
from oracle import attention as O
from test_gpu_attention import assert_within, gen, ints, normal
from test_gpu_kv_extra import BF16, DEV, U8, paged8_setup, run_paged8, weights_want

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
