"""Sequences of almost 2^31 rows over the 8-bit cache: block tables of few real pages (the
others are outside the pool: their rows read as zeros with weight 0)."""
from __future__ import annotations

import pytest
import torch

import mtlflashattn_amd as mfa
from kv8_util import DEV, i32

pytestmark = pytest.mark.gpu

PAGE, COLS = 64 * 1801, 31 * 601  # 2^31 - 64 rows


def long_table(places):
    """[1, COLS] with page `id` at column `col` of the pairs, all others outside the pool."""
    table = torch.full((1, COLS), -1, dtype=torch.int32)
    for col, page in places:
        table[0, col] = page
    return table.to(DEV)


@pytest.mark.parametrize("n", [(1 << 31) - 64, (1 << 31) - 300, (1 << 31) - 4096 + 200])
def test_evict(n):
    """The heaviest rows of the first, a middle and the last page; rows of weight 0 stay behind."""
    g = torch.Generator().manual_seed(n % 1000)
    budget, recent = 300, 70
    kc, vc = mfa.kv8_cache(4, PAGE, 1, 32), mfa.kv8_cache(4, PAGE, 1, 32)
    for c in (kc, vc):  # (one scale, 448 in every row: rows move as they are)
        codes = torch.randint(0, 127, c[0].shape, generator=g, dtype=torch.uint8)
        codes[..., 0] = 0x7E
        c[0].view(torch.uint8).copy_(codes)
        c[1].fill_(120)
    last = (n - 1) // PAGE
    at = {0: 2, 9999: 0, last: 3}
    w = torch.zeros(4, PAGE, 1)
    heavy = [(0, 17), (0, 40), (0, 5000), (9999, 0), (9999, 77), (9999, PAGE - 1), (last, 3)]
    heavy += [(9999, int(r)) for r in torch.randperm(PAGE - 200, generator=g)[:budget - recent - len(heavy)] + 100]
    for col, row in heavy:
        w[at[col], row] = 0.5 + float(torch.rand(1, generator=g))
    w[:, 1::2][w[:, 1::2] == 0] = -1.0
    w[1] = 7.0  # (no sequence's)
    rows = sorted(col * PAGE + row for col, row in heavy) + list(range(n - recent, n))
    src = [(at[j // PAGE], j % PAGE) for j in rows]
    assert len(set(src)) == budget and all(j // PAGE in at for j in rows)
    p, r = (torch.tensor(x) for x in zip(*src))
    want = [(c[0].view(torch.uint8).cpu()[p, r], w[p, r]) for c in (kc, vc)]
    wd = w.to(DEV)
    assert mfa.kv8_evict(kc, vc, wd, i32(n), long_table(at.items()), budget, recent).tolist() == [budget]
    for c, (codes, weights) in zip((kc, vc), want):
        assert torch.equal(c[0].view(torch.uint8)[2, :budget].cpu(), codes)
        assert bool((c[1] == 120).all())
        assert torch.equal(wd[2, :budget].cpu(), weights)
    keep = wd.cpu()
    keep[2, :budget] = w[2, :budget]
    assert torch.equal(keep, w)


@pytest.mark.parametrize("lq,left", [(1, -1), (40, -1), (40, 1000), (300, 1000)])
@pytest.mark.parametrize("n", [(1 << 31) - 300, (1 << 31) - 700])
def test_key_weights(n, lq, left):
    """Keys of zeros and log-sum-exps of 0: a key gains the number of rows that see it, exactly."""
    kc = mfa.kv8_cache(3, PAGE, 1, 32)
    last = (n - 1) // PAGE
    table = long_table({0: 2, last: 1}.items())
    q = torch.randn(1, lq, 1, 32, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(3, PAGE, 1, device=DEV)
    mfa.kv8_key_weights(q, kc, torch.zeros(1, 1, lq, device=DEV), w, i32(n), table, causal=True, window_size=(left, -1))
    want = torch.ones(3, PAGE)
    for page, col in ((2, 0), (1, last)):
        j = col * PAGE + torch.arange(PAGE)
        i = n - lq + torch.arange(lq)[:, None]
        seen = (j <= i) & ((j >= i - left) | (left < 0))
        want[page] = torch.where(j < n, torch.where(j < n - lq, 1.0, 0.0) + seen.sum(0), 1.0)
    assert torch.equal(w[..., 0].cpu(), want)
