"""Varlen attention over the 8-bit cache where sequences have 17 to 32 columns on average: those of
up to 32 run on the kernel of 32 columns, whose probabilities are two bf16 terms.

Bounds of that kernel: half a step of the output's type, and 3e-4 vmax for what is left of the
probabilities (2^-16) and the scores' rounding (sum |q k| scale < 100: 100 * 2^-22 = 2.4e-5); 1e-4 +
2e-6 |lse| for the log-sum-exp.  A single 16-bit term would be off by up to 2^-8 vmax (bf16) in rows
of few keys, of which there are some here; of longer sequences on the tiles of 128 columns one is
(eps vmax, and 2 % for the second order)."""
from __future__ import annotations

import pytest
import torch

import mtlflashattn_amd as mfa
from kv8_util import DEV, attend64, cu_of, make, rows64

pytestmark = pytest.mark.gpu


def check(lq, lens, Hq, Hkv, D, dtype, few, **kw):
    """few: columns up to which a sequence is held to the bounds of two terms."""
    R = Hq // Hkv
    q, kc, vc, lens_t, table = make(lens, 64, Hq, Hkv, D, dtype, lq)
    ref, ref_lse, _ = attend64(q, kc, vc, lens, table, lq, True, kw.get("window_size", (-1, -1)), kw.get("softcap", 0.0))
    out, lse = mfa.flash_attn_varlen_kv8_func(q, kc, vc, cu_of(lq), lens_t, table, causal=True, return_softmax_lse=True, **kw)
    vmax, eps = float(rows64(vc).abs().max()), torch.finfo(dtype).eps
    tiles = torch.tensor([n * R > few for n in lq for _ in range(n)], dtype=torch.float64)[:, None, None]
    err = (out.cpu().double() - ref).abs()
    tol = eps / 2 * ref.abs() + 3e-4 * vmax + tiles * (1.02 * eps * vmax)
    assert bool((err <= tol).all()), f"max err {float(err.max()):.3e}, bound there {float(tol.flatten()[err.argmax()]):.3e}"
    seen = ref_lse.isfinite()
    assert torch.equal(lse.cpu().isfinite(), seen)
    assert bool(((lse.cpu().double() - ref_lse).abs() <= 1e-4 + 2e-6 * ref_lse.abs())[seen].all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("lq", [[5] * 6, [5, 8, 0, 1, 9, 12, 5], [8, 8, 8], [1, 15], [5, 5, 5, 5, 1, 20]])
def test_17_to_32_columns_on_average(lq, D, dtype):
    assert 16 < sum(lq) * 4 / len(lq) <= 32
    # (some rows see a handful of keys, some hundreds)
    check(lq, [max(n, 1) + 333 * (i % 3) for i, n in enumerate(lq)], 8, 2, D, dtype, 32)


@pytest.mark.parametrize("lq,few", [([4, 4, 4, 4], 16), ([4] * 9 + [3], 16), ([5, 5, 5], 32), ([16, 8, 7, 1], 32),
                                    ([17, 8, 7, 1], 16), ([9, 9, 9], 16)])
def test_the_means_at_the_edges(lq, few):
    """16 columns on average and less: the kernel of 16; more than 32: that of 16 and the tiles.
    ((16 + 8 + 7 + 1) 4 = 128 columns are 32 for each of four sequences, (17 + 8 + 7 + 1) 4 = 132 are
    33: there the sequences of 17, 8 and 7 rows are on the tiles, with their bound.)"""
    check(lq, [n + 211 * (i % 2) for i, n in enumerate(lq)], 8, 2, 64, torch.bfloat16, few)


@pytest.mark.parametrize("kw", [dict(window_size=(3, -1)), dict(window_size=(100, 0)), dict(softcap=4.0)])
def test_masks(kw):
    check([5, 8, 0, 7, 8, 6], [5, 700, 30, 64, 8, 133], 8, 2, 64, torch.bfloat16, 32, **kw)
