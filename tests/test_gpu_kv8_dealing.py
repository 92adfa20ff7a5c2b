"""How the key weights' work is dealt over workgroups, told by the time of calls that have the
same work."""
from __future__ import annotations

import pytest
import torch

import mtlflashattn_amd as mfa
from kv8_util import DEV, cu_of, i32

pytestmark = pytest.mark.gpu


def time_of(call):
    """Least time of five runs of three calls, ms."""
    call()
    times = []
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(3):
            call()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


def step(lens, lq, Hq, Hkv, D, varlen=False, page=256, **kw):
    """A key-weight call over caches of zeros: (call, weights)."""
    pages = max(-(-n // page) for n in lens)
    kc = mfa.kv8_cache(len(lens) * pages, page, Hkv, D)
    table = torch.arange(len(lens) * pages, dtype=torch.int32, device=DEV).view(len(lens), pages)
    q = torch.randn(len(lens), lq, Hq, D, device=DEV, dtype=torch.bfloat16)
    lse = torch.zeros(len(lens), Hq, lq, device=DEV)
    w = torch.zeros(len(lens) * pages, Hkv, page, device=DEV).transpose(1, 2)
    lens_t = i32(*lens)
    if varlen:
        q, lse, cu = q.flatten(0, 1), lse.transpose(0, 1).reshape(Hq, -1), cu_of([lq] * len(lens))
        return lambda: mfa.kv8_key_weights(q, kc, lse, w, lens_t, table, cu, causal=True, **kw), w
    return lambda: mfa.kv8_key_weights(q, kc, lse, w, lens_t, table, causal=True, **kw), w


@pytest.mark.parametrize("batch,lq,left,n", [(1, 2048, 4096, 131072), (8, 64, 4096, 65536), (2, 40, 8192, 262144)])
def test_a_window_over_a_long_cache(batch, lq, left, n):
    """It takes the time of the same window over a cache that is hardly longer: all workgroups
    have a share of the keys that are seen.  (Dealt by all keys it took 5 to 13 times as long.)"""
    times = []
    for L in (n, left + lq):
        call, w = step([L] * batch, lq, 32, 8, 128, window_size=(left, -1))
        call()
        # scores of 0 and log-sum-exps of 0: a key has the number of columns that see it
        assert float(w.double().sum()) == batch * 32 * sum(min(i + L - lq, left) + 1 for i in range(lq))
        times.append(time_of(call))
    assert times[0] <= 2 * times[1]


@pytest.mark.parametrize("batch,n", [(1024, 512), (2048, 256)])
def test_single_rows_of_a_varlen_call(batch, n):
    """The launch for sequences of more columns, of which there are none, costs little beside the
    work: a fifth, and half (it was 1.4 and 4 times the work)."""
    times, sums = [], []
    for varlen in (False, True):
        call, w = step([n] * batch, 1, 32, 8, 128, varlen=varlen)
        call()
        sums.append(w)
        assert bool((w == 4).all())
        times.append(time_of(call))
    assert torch.equal(*sums)
    assert times[1] <= (1.6 if batch == 1024 else 2.2) * times[0]


@pytest.mark.parametrize("lq", [[17] + [0] * 70 + [18, 1, 40], [1] * 130 + [17], [5] * 64 + [9, 17, 33], [300], [33] * 9])
def test_few_sequences_with_many_columns(lq):
    """All of them are found where rows leave room for no more."""
    lens = [n + 200 for n in lq]
    Hkv, D, page = 2, 32, 64
    for R in (1, 4):
        kc = mfa.kv8_cache(sum(-(-n // page) for n in lens), page, Hkv, D)
        table, at = torch.full((len(lens), 8), -1, dtype=torch.int32), 0
        for b, n in enumerate(lens):
            for i in range(-(-n // page)):
                table[b, i] = at
                at += 1
        q = torch.randn(sum(lq), R * Hkv, D, device=DEV, dtype=torch.bfloat16)
        w = torch.ones(at, page, Hkv, device=DEV)
        mfa.kv8_key_weights(q, kc, torch.zeros(R * Hkv, sum(lq), device=DEV), w, i32(*lens), table.to(DEV), cu_of(lq))
        for b, (n, L) in enumerate(zip(lq, lens)):
            got = w[table[b, :-(-L // page)].long()].flatten(0, 1)[:L].cpu()
            want = torch.where(torch.arange(L) < L - n, 1.0, 0.0) + R * n
            assert torch.equal(got, want[:, None].expand(-1, Hkv)), (R, b)
