"""The log-sum-exp that attention over the quantised caches returns from its tiles of 128
columns, against the definition in float64, and the key weights that are formed from it.

The tiles round probabilities to 16 bits for the product with V; the log-sum-exp is that of
the probabilities before.  Bound: scores are fp32 sums of exact products (|ds| <= 2^-22
sum |q k| scale, the sum below 100: 2.4e-5), a probability adds its exponent's rounding (fma
of numbers below 64: 2^-19 of log2 units, 1.3e-6) and 2^-23 of exp2; the sum of a block of 64
keys is at most 20 additions, that of a sequence of 2100 at most 40 more with the parts'
merge (60 2^-24 = 3.6e-6); the soft-cap adds 2^-21 of its bound (5: 2.4e-6), ALiBi two roundings of
terms below 64 (7.6e-6) and the result one of 2^-24.  1e-4 + 2e-6 |lse| covers them; a sum of
rounded probabilities is off by up to 2^-8 (bf16) or 2^-11 (fp16).
"""
from __future__ import annotations

import pytest
import torch

import kv8_util
import mtlflashattn_amd as mfa
import test_gpu_kv4_attend as kv4
from kv8_util import DEV, attend64, cu_of

pytestmark = pytest.mark.gpu

FIXED = {4: mfa.flash_attn_kv4_func, 8: mfa.flash_attn_kv8_func}
VARLEN = {4: mfa.flash_attn_varlen_kv4_func, 8: mfa.flash_attn_varlen_kv8_func}


def make(bits, *args):
    """(q, K, V, lengths, table) and the reference of a call's options."""
    if bits == 4:
        x = kv4.make(*args)
        return x, lambda lens, lq, *opts: kv4.oracle(x[0], x[1], x[2], lens, x[4], lq, *opts)[1]
    x = kv8_util.make(*args)
    return x, lambda lens, lq, *opts: attend64(x[0], x[1], x[2], lens, x[4], lq, *opts)[1]


def check(lse, ref):
    finite = ref.isfinite()
    assert torch.equal(lse.cpu().isfinite(), finite)
    err = (lse.cpu().double() - ref).abs()[finite]
    assert bool((err <= 1e-4 + 2e-6 * ref[finite].abs()).all()), f"max err {float(err.max()):.3e}"


def run(bits, lens, lq, Hq, Hkv, D, dtype, slopes=None, **kw):
    (q, kc, vc, lens_t, table), oracle = make(bits, lens, 64, Hq, Hkv, D, dtype, lq)
    ref = oracle(lens, lq, kw.get("causal", False), kw.get("window_size", (-1, -1)), kw.get("softcap", 0.0), slopes)
    if slopes is not None:
        kw["alibi_slopes"] = slopes.to(DEV)
    if len(set(lq)) == 1:
        fixed = q.view(len(lq), lq[0], Hq, D)
        out, lse = FIXED[bits](fixed, kc, vc, lens_t, table, return_softmax_lse=True, **kw)
        check(lse.transpose(0, 1).reshape(Hq, -1), ref)
        assert torch.equal(out, FIXED[bits](fixed, kc, vc, lens_t, table, **kw))  # (the result is the same without)
    out, lse = VARLEN[bits](q, kc, vc, cu_of(lq), lens_t, table, return_softmax_lse=True, **kw)
    check(lse, ref)
    assert torch.equal(out, VARLEN[bits](q, kc, vc, cu_of(lq), lens_t, table, **kw))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_tiles(D, dtype, bits):
    """A unit's keys in one walk (sequences of one chunk) and in parts of several."""
    run(bits, [40, 41, 128, 100], [40] * 4, 4, 2, D, dtype, causal=True)
    run(bits, [2100], [70], 4, 2, D, dtype, causal=True)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kw", [
    dict(window_size=(20, 5)), dict(causal=True, window_size=(0, 0)), dict(causal=True, softcap=5.0),
    dict(causal=True, slopes=torch.tensor([0.02, 0.01, 0.03, 0.0])),
])
def test_masks_and_biases(kw, bits):
    """Rows of few keys, where a rounded weight shows most."""
    run(bits, [50, 777, 30], [50] * 3, 4, 2, 64, torch.bfloat16, **kw)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_mixed_steps(dtype, bits):
    """Chunks beside single rows: parts of both kernels in one merge; rows without keys."""
    run(bits, [500, 1000, 64, 2000, 130, 5], [1, 90, 1, 3, 130, 40], 8, 2, 128, dtype, causal=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,lq", [([150], [150]), ([400, 129], [60, 129]), ([2000, 33], [50, 33])])
def test_key_weights_of_a_prompt(lens, lq, dtype):
    """With the attention call's log-sum-exps every probability is within 1e-4 (theirs) + 8e-5 (the
    key weights' own: scores 2.4e-5, their scaling and difference 1.2e-5, exp2) of itself: the weights
    of a prompt's rows add up to 1 each, and the first key of the first row has the weight it should."""
    Hq, Hkv, D = 8, 2, 64
    q, kc, vc, lens_t, table = kv8_util.make(lens, 64, Hq, Hkv, D, dtype, lq)
    _, lse = mfa.flash_attn_varlen_kv8_func(q, kc, vc, cu_of(lq), lens_t, table, causal=True, return_softmax_lse=True)
    w = torch.zeros(kc[0].shape[:3], device=DEV)
    mfa.kv8_key_weights(q, kc, lse, w, lens_t, table, cu_of(lq), causal=True)
    rows = sum(lq) * Hq
    assert abs(float(w.double().sum()) - rows) <= 2e-4 * rows
    _, _, sums = attend64(q, kc, vc, lens, table, lq, causal=True)
    for b, L in enumerate(lens):
        have = w[table[b, :-(-L // 64)].long()].flatten(0, 1)[:L].T.cpu().double()
        # (sums of lq rows and 4 heads: one rounding each at most)
        assert bool(((have - sums[b]).abs() <= sums[b] * (1.8e-4 + lq[b] * 4 * 2.0 ** -24)).all())
