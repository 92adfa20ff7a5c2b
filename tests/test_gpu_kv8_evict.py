"""Eviction from the paged 8-bit cache, and a server's steps with it.  What stays, where it
goes and every code, scale and weight is defined exactly: compared for equality."""
from __future__ import annotations

import math

import pytest
import torch

import mtlflashattn_amd as mfa
from kv8_util import DEV, append64, attend64, bits, cu_of, evict64, filled_cache, i32, rows64, table_of

pytestmark = pytest.mark.gpu


def state(lens, page, H, D, seed=0, extra=3, layout="heads", kind="random"):
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-n // page) for n in lens) + extra
    kc, vc = (filled_cache(g, pages, page, H, D, 1.0, layout) for _ in range(2))
    w = torch.exp(2 * torch.randn(pages, H, page, generator=g))
    if kind == "ties":
        w = torch.randint(0, 4, w.shape, generator=g).float()
    elif kind == "equal":
        w = torch.ones_like(w)
    elif kind == "odd":  # signs, zeros of both signs, infinities, NaN of both signs, subnormals
        values = torch.tensor([0.0, -0.0, 1.0, -1.0, math.inf, -math.inf, math.nan, -math.nan, 1e-42, -1e-42, 3e38])
        w = values[torch.randint(0, len(values), w.shape, generator=g)]
    elif kind == "falling":
        w = torch.arange(w.numel(), 0, -1).float().view(w.shape)
    w = w.to(DEV)
    w = w.transpose(1, 2) if layout == "heads" else w.transpose(1, 2).contiguous()
    return kc, vc, w, i32(*lens), table_of(lens, page, pages, seed, extra=1)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=7e33), torch.nan_to_num(b, nan=7e33))


def check(kc, vc, w, lens, table, budget, recent, max_k=None):
    want, want_w, want_n = evict64(kc, vc, w, lens.tolist(), table.cpu(), budget, recent)
    before = lens.clone()
    n = mfa.kv8_evict(kc, vc, w, lens, table, budget, recent, max_seqlen_k=max_k)
    assert n.dtype == torch.int32 and n.tolist() == want_n and torch.equal(lens, before)
    for c, ref in zip((kc, vc), want):
        for a, b in zip(bits(c), ref):
            assert torch.equal(a, b)
    assert same(w.cpu(), want_w)
    return n


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("budget,recent", [(0, 0), (1, 0), (1, 1), (63, 5), (64, 0), (65, 64), (100, 100), (128, 500), (200, 20),
                                           (299, 1), (300, 0)])
def test_evict(budget, recent, D):
    check(*state([300, 1, 0, 64, 65, 129, 200], 64, 2, D), budget, recent)


@pytest.mark.parametrize("kind", ["ties", "equal", "odd", "falling"])
@pytest.mark.parametrize("budget,recent", [(1, 0), (70, 10), (192, 0), (250, 33)])
def test_weights(kind, budget, recent):
    """Ties go to the lower row, NaN stands above everything, -0 is 0; rows that already
    are the first ones stay."""
    check(*state([300, 260, 251], 128, 2, 32, kind=kind), budget, recent)


@pytest.mark.parametrize("n,max_k", [(4000, None), (4096, 4096), (4160, None), (16000, 16384), (20000, None), (70000, None),
                                     (140000, 140000)])
def test_long_sequences(n, max_k):
    """Keys in registers at three sizes, and read again where they do not fit."""
    kc, vc, w, lens, table = state([n, 500], 256, 1, 32)
    check(kc, vc, w, lens, table, n // 3, 100, max_k)


@pytest.mark.parametrize("page", [64, 192, 256])
@pytest.mark.parametrize("layout", ["heads", "rows"])
def test_layouts_and_pages(layout, page):
    check(*state([700, 1, 513, 320], page, 3, 64, layout=layout), 300, 64)


def test_many_sequences():
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 200, (150,), generator=g).tolist()
    check(*state(lens, 64, 2, 32), 77, 13)


def test_max_seqlen_k_and_lengths_outside():
    """It cuts a sequence, as the table does; lengths below 0 count as 0."""
    kc, vc, w, lens, table = state([300, 200], 64, 2, 64)
    want, want_w, _ = evict64(kc, vc, w, [150, 150], table.cpu(), 100, 10)
    assert mfa.kv8_evict(kc, vc, w, lens, table, 100, 10, max_seqlen_k=150).tolist() == [100, 100]
    for c, ref in zip((kc, vc), want):
        assert torch.equal(bits(c)[0], ref[0]) and torch.equal(bits(c)[1], ref[1])
    assert same(w.cpu(), want_w)
    kc, vc, w, lens, table = state([64, 200], 64, 2, 64)
    n = mfa.kv8_evict(kc, vc, w, i32(-5, 1 << 30), table[:, :1].contiguous(), 40, 10)
    assert n.tolist() == [0, 40]
    assert mfa.kv8_evict(kc, vc, w, i32(3, 9), table, 1 << 40, 1 << 40).tolist() == [3, 9]


def test_page_ids_outside_the_pool():
    """Their rows read as zeros with weight 0 and drop what is written."""
    kc, vc, w, lens, table = state([300, 300, 300], 64, 2, 64)
    table[0, 1], table[1, 0], table[2, 4] = -1, 1 << 30, kc[0].shape[0]
    check(kc, vc, w, lens, table, 150, 50)


def test_nan_codes_move():
    kc, vc, w, lens, table = state([200], 64, 1, 32)
    for c in (kc, vc):
        c[0].view(torch.uint8)[:, ::7, :, ::5] = 0xFF
        c[0].view(torch.uint8)[table[0, 2].item()] = 0x7F
    check(kc, vc, w, lens, table, 130, 40)


def test_zeros_of_large_scales():
    """Rows of zeros from blocks of any scale make a block of the smallest scale: zeros still."""
    kc, vc, w, lens, table = state([400, 130], 64, 2, 64)
    for c in (kc, vc):
        codes = c[0].view(torch.uint8)
        codes &= 0x80
        codes[:, ::9] = 0x70
        c[1].copy_(torch.tensor([1, 100, 129, 200, 247], dtype=torch.uint8, device=DEV).repeat(99)[: c[1].shape[0]].view(-1, 1, 1))
    w[:, ::9] = 0
    check(kc, vc, w, lens, table, 128, 0)


@pytest.mark.parametrize("batch", [16, 24])
@pytest.mark.parametrize("D,page", [(32, 192), (64, 64), (96, 128), (128, 256)])
def test_batches(batch, D, page):
    """Many heads with much to move: ragged, some untouched, an odd budget, missing pages, odd weights."""
    g = torch.Generator().manual_seed(batch + D)
    lens = torch.randint(0, 1500, (batch,), generator=g).tolist()
    for layout, kind in (("heads", "odd"), ("rows", "random")):
        kc, vc, w, n, table = state(lens, page, 8, D, layout=layout, kind=kind)
        table[1, :2], table[2, 1] = -1, 1 << 30
        check(kc, vc, w, n, table, 611, 40)


@pytest.mark.parametrize("kind", ["random", "ties", "falling"])
@pytest.mark.parametrize("budget,recent", [(0, 0), (1, 1), (63, 5), (64, 0), (65, 64), (100, 100), (257, 20), (299, 1), (300, 0)])
def test_budgets_of_batches(budget, recent, kind):
    lens = [300, 1, 0, 64, 65, 129, 200, 299, 301, 270] * 4
    check(*state(lens, 64, 2, 32, kind=kind), budget, recent)


def test_again_on_a_stream_and_captured():
    """An eviction of what an eviction left; the same bits on another stream and in a graph."""
    args = state([900, 64, 500], 64, 2, 64, seed=3)
    n = check(*args, 400, 50)
    kc, vc, w, _, table = args
    check(kc, vc, w, n, table, 129, 50)
    runs = []
    for how in ("eager", "stream", "graph"):
        kc, vc, w, lens, table = state([900, 64, 500], 64, 2, 64, seed=4)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        if how == "graph":
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                n = mfa.kv8_evict(kc, vc, w, lens, table, 400, 50)
        for turn in range(4):
            if how == "graph":
                graph.replay()
            else:
                with torch.cuda.stream(s if how == "stream" else torch.cuda.current_stream()):
                    n = mfa.kv8_evict(kc, vc, w, lens, table, 400, 50)
            torch.cuda.synchronize()
            runs.append((turn, [*bits(kc), *bits(vc), w.cpu(), n.tolist()]))
            lens.sub_(70)
    for turn, got in runs[4:]:
        ref = runs[turn][1]
        assert all(torch.equal(a, b) for a, b in zip(got[:5], ref[:5])) and got[5] == ref[5]


def test_a_server_that_keeps_a_budget():
    """Prompt, steps, evictions: append, attention, key weights and eviction together, against the
    definitions over the rows that the cache was given."""
    Hq, Hkv, D, page, budget, recent, B = 8, 2, 64, 64, 160, 32, 2
    g = torch.Generator().manual_seed(11)
    kc, vc = mfa.kv8_cache(12, page, Hkv, D), mfa.kv8_cache(12, page, Hkv, D)
    w = torch.full((12, page, Hkv), math.nan, device=DEV)  # (needs no clearing)
    table = i32(7, 3, 0, 9, 1, 5, 2, 8).view(2, 4)
    lens = i32(0, 0)
    prompt = [150, 90]

    def step(new, check):
        nonlocal lens
        q = torch.randn(sum(new), Hq, D, generator=g).to(DEV, torch.bfloat16)
        k, v = (torch.randn(sum(new), Hkv, D, generator=g).to(DEV, torch.bfloat16) for _ in range(2))
        cu = cu_of(new)
        want = [append64(c, x, cu.tolist(), lens.tolist(), table.cpu(), page)[0] for c, x in zip((kc, vc), (k, v))] if check else None
        mfa.kv8_append(k, v, kc, vc, cu, lens, table)
        lens = lens + i32(*new)
        before = w.cpu().double()
        out, lse = mfa.flash_attn_varlen_kv8_func(q, kc, vc, cu, lens, table, causal=True, return_softmax_lse=True)
        mfa.kv8_key_weights(q, kc, lse, w, lens, table, cu, causal=True)
        if check:
            for c, ref in zip((kc, vc), want):
                assert torch.equal(bits(c)[0], ref[0]) and torch.equal(bits(c)[1], ref[1])
            ref, ref_lse, sums = attend64(q, kc, vc, lens.tolist(), table, new, causal=True)
            # (half a step of bf16 and, on the 128-column tiles, a step of the largest value)
            tol = 2.0 ** -8 * ref.abs() + (3e-4 + 2.0 ** -7 * 1.02) * float(rows64(vc).abs().max())
            assert bool(((out.cpu().double() - ref).abs() <= tol).all())
            # (the lse of the tiles is off by up to 1.01 * 2^-8: so are the weights)
            for b, n in enumerate(new):
                for j in range(int(lens[b])):
                    at = (int(table[b, j // page]), j % page)
                    have = sums[b][:, j] + (before[at] if j < int(lens[b]) - n else 0.0)
                    assert bool(((w[at].cpu().double() - have).abs() <= 4.2e-3 * sums[b][:, j] + 2.0 ** -22 * have).all())

    step(prompt, True)
    for i in range(60):
        step([1, 1], i in (0, 59))
        if i % 20 == 19:
            want, want_w, want_n = evict64(kc, vc, w, lens.tolist(), table.cpu(), budget, recent)
            lens = mfa.kv8_evict(kc, vc, w, lens, table, budget, recent, max_seqlen_k=256)
            assert lens.tolist() == want_n
            for c, ref in zip((kc, vc), want):
                assert torch.equal(bits(c)[0], ref[0]) and torch.equal(bits(c)[1], ref[1])
            assert same(w.cpu(), want_w)
    assert lens.tolist() == [160, 150]
