"""Magnitudes over the 8-bit cache: queries and keys that only differ by powers of two have
the same scores, so the same bits."""
from __future__ import annotations

import pytest
import torch

import mtlflashattn_amd as mfa
from kv8_util import DEV, make, rows64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e", [-90, -30, 30, 50, 70, 90])
@pytest.mark.parametrize("D,Hq,lq", [(64, 4, 1), (64, 6, 7), (64, 4, 40), (128, 2, 1), (96, 4, 100)])
@pytest.mark.parametrize("kw", [dict(), dict(softcap=3.0), dict(window_size=(70, 0))])
def test_large_queries_and_small_keys(D, Hq, lq, e, kw):
    """q 2^e over keys 2^-e of what they were, blocks that nobody wrote among them."""
    lens = [300, 129]
    q, kc, vc, lens_t, table = make(lens, 64, Hq, 2, D, torch.bfloat16, [lq] * 2)
    kc[0].view(torch.uint8)[table[0, 1].item()] = 0
    kc[1][table[0, 1].item()] = 0
    q = q.view(2, lq, Hq, D)
    moved = kc[0], torch.where(kc[1] == 0, 0, kc[1].int() - e).to(torch.uint8)
    assert int(moved[1].min()) == 0 and bool((moved[1][kc[1] > 0] >= 1).all())
    got = []
    for x, c in ((q, kc), (q * 2.0 ** e, moved)):
        o, lse = mfa.flash_attn_kv8_func(x, c, vc, lens_t, table, causal=True, return_softmax_lse=True, **kw)
        w = torch.ones(kc[0].shape[:3], device=DEV)
        mfa.kv8_key_weights(x, c, lse, w, lens_t, table, causal=True, **kw)
        got.append((o, lse, w))
    for a, b in zip(*got):
        assert bool(a.isfinite().all()) and torch.equal(a, b)


@pytest.mark.parametrize("scale", [1e-3, 1.01 * 2.0 ** -24, 2.0 ** -24, 2.0 ** -60])
@pytest.mark.parametrize("lq", [1, 7, 40])
def test_smallest_scales_beside_masked_keys(lq, scale):
    """Bytes 0 and 1 under small softmax scales: factors of scores that are hardly above 0.  Every
    score is 0 to fp32, so a row's result is the mean of what it sees: within half a step of bf16, and
    2^-7 of the largest value where probabilities are rounded once."""
    L = 200
    q, kc, vc, lens, table = make([L], 64, 4, 2, 64, torch.bfloat16, [lq])
    kc[1].fill_(1)
    kc[1][table[0, 3].item()] = 0
    out, lse = mfa.flash_attn_kv8_func(q.view(1, lq, 4, 64), kc, vc, lens, table, softmax_scale=scale, causal=True,
                                       window_size=(30, 0), return_softmax_lse=True)
    v = rows64(vc)[table[0, :4].cpu().long()].flatten(0, 1)
    for i in range(lq):
        ref = v[L - lq + i - 30:L - lq + i + 1].mean(0).repeat_interleave(2, 0)
        err = (out[0, i].cpu().double() - ref).abs()
        assert bool((err <= 2.0 ** -8 * ref.abs() + 2.0 ** -7 * 1.02 * float(v.abs().max())).all())
    assert torch.allclose(lse.cpu(), torch.full_like(lse, 31.0).log().cpu(), rtol=0, atol=1e-5)
