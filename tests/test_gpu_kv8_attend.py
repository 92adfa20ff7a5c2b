"""Attention over the paged 8-bit cache against the definition in float64.

The oracle reads the same codes and scales, so the quantisation plays no part.  Bounds
as for the 4-bit cache: the output is rounded to its type (half a step, finfo.eps / 2
relative); at most 32 columns of a sequence carry probabilities of two bf16 terms (2^-16
relative) and fp32 sums, which 3e-4 * vmax covers with the scores' own rounding (sum |q k|
scale < 100: 100 * 2^-22 = 2.4e-5); more columns (in a varlen call more than 16, unless
the whole call has at most 32) run on tiles of 128, whose probabilities are rounded once
to the queries' type, an error of at most finfo.eps * vmax, and of the log-sum-exp of at
most 1.01 * finfo.eps / 2.  V of these tests is exact in fp16.
"""
from __future__ import annotations

import math

import pytest
import torch

import mtlflashattn_amd as mfa
from kv8_util import DEV, attend64, cu_of, filled_cache, i32, make, rows64

pytestmark = pytest.mark.gpu


def on_tiles(lq, R, varlen):
    """Per query row: whether its sequence runs on 128-column tiles."""
    few = sum(lq) * R <= 32 if varlen else lq[0] * R <= 32
    return torch.tensor([not few and n * R > (16 if varlen else 32) for n in lq for _ in range(n)], dtype=torch.float64)


def check(out, ref, vmax, dtype, tiles):
    err = (out.cpu().double() - ref).abs()
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + 3e-4 * vmax + tiles[:, None, None] * (1.02 * torch.finfo(dtype).eps * vmax)
    assert not out.isnan().any()
    assert bool((err <= tol).all()), f"max err {float(err.max()):.3e}, bound there {float(tol.flatten()[err.argmax()]):.3e}"


def run_and_check(lens, lq, page, Hq, Hkv, D, dtype, seed=0, layout="heads", max_k=None, slopes=None, **kw):
    q, kc, vc, lens_t, table = make(lens, page, Hq, Hkv, D, dtype, lq, seed, layout)
    ref, ref_lse, _ = attend64(q, kc, vc, lens, table, lq, kw.get("causal", False), kw.get("window_size", (-1, -1)),
                               kw.get("softcap", 0.0), slopes)
    sl = None if slopes is None else slopes.to(DEV)
    vmax = float(rows64(vc).abs().max())
    got = []
    if len(set(lq)) == 1:
        o, lse = mfa.flash_attn_kv8_func(q.view(len(lq), lq[0], Hq, D), kc, vc, lens_t, table, max_seqlen_k=max_k,
                                         alibi_slopes=sl, return_softmax_lse=True, **kw)
        assert o.shape == (len(lq), lq[0], Hq, D) and lse.shape == (len(lq), Hq, lq[0])
        got.append((o.reshape(-1, Hq, D), lse.transpose(0, 1).reshape(Hq, -1), on_tiles(lq, Hq // Hkv, False)))
    o, lse = mfa.flash_attn_varlen_kv8_func(q, kc, vc, cu_of(lq), lens_t, table, max_seqlen_k=max_k, alibi_slopes=sl,
                                            return_softmax_lse=True, **kw)
    got.append((o, lse, on_tiles(lq, Hq // Hkv, True)))
    for o, lse, tiles in got:
        assert o.dtype == dtype and lse.dtype == torch.float32
        check(o, ref, vmax, dtype, tiles)
        fin = torch.isfinite(ref_lse)
        assert torch.equal(torch.isfinite(lse.cpu()), fin)
        tol = 1e-4 + 2e-6 * ref_lse.abs() + tiles * (1.01 * torch.finfo(dtype).eps / 2)
        assert bool(((lse.cpu().double() - ref_lse).abs() <= tol)[fin].all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (5, 1), (20, 1)])
def test_single_rows(D, Hq, Hkv, dtype):
    run_and_check([1, 33, 64, 129, 700, 0, 255], [1] * 7, 64, Hq, Hkv, D, dtype, causal=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("lq", [2, 5, 9, 40])
def test_drafted_tokens(D, lq, dtype):
    run_and_check([lq, 300, 41, 1000], [lq] * 4, 128, 6, 2, D, dtype, causal=True)


@pytest.mark.parametrize("D,dtype", [(32, torch.float16), (64, torch.bfloat16), (96, torch.float16), (128, torch.bfloat16)])
def test_drafts_in_a_varlen_call(D, dtype):
    """17 to 32 columns per sequence on average: the kernel of 32 columns, with the bits of the fixed
    call; longer sequences among them run on tiles of 128."""
    lq, R = 5, 4
    lens = [5, 300, 41, 1000, 2000, 64]
    q, kc, vc, lens_t, table = make(lens, 64, 8, 2, D, dtype, [lq] * 6)
    fixed = mfa.flash_attn_kv8_func(q.view(6, lq, 8, D), kc, vc, lens_t, table, causal=True)
    packed = mfa.flash_attn_varlen_kv8_func(q, kc, vc, cu_of([lq] * 6), lens_t, table, causal=True)
    assert torch.equal(fixed.flatten(0, 1), packed)
    for mixed in ([5, 8, 0, 1, 9, 12, 5], [8, 8, 8], [1, 15], [5, 5, 5, 5, 1, 20]):
        assert 16 < sum(mixed) * R / len(mixed) <= 32
        run_and_check([max(n, 1) + 333 * (i % 3) for i, n in enumerate(mixed)], mixed, 64, 8, 2, D, dtype, causal=True)


@pytest.mark.parametrize("kw", [
    dict(), dict(causal=True), dict(causal=True, window_size=(100, -1)), dict(window_size=(30, 20)),
    dict(window_size=(0, 0)), dict(window_size=(-1, 3)), dict(causal=True, softcap=2.0),
    dict(causal=True, window_size=(300, 0), softcap=5.0),
])
@pytest.mark.parametrize("lq", [1, 7, 70])
def test_masks(kw, lq):
    run_and_check([lq, 900, 513], [lq] * 3, 64, 4, 2, 64, torch.bfloat16, **kw)


@pytest.mark.parametrize("per_batch", [False, True])
@pytest.mark.parametrize("lq", [1, 6, 40])
def test_alibi(lq, per_batch):
    slopes = torch.tensor([0.5, 0.01, 0.3, 0.0])
    if per_batch:
        slopes = torch.stack((slopes, slopes.flip(0)))
    run_and_check([400, 77], [lq] * 2, 64, 4, 2, 128, torch.float16, causal=True, slopes=slopes)


@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_more_queries_than_keys(D):
    """Rows before the first key see nothing: 0 and -inf."""
    run_and_check([3, 0, 20], [8, 8, 8], 64, 4, 2, D, torch.bfloat16, causal=True)
    run_and_check([3, 0, 20], [30, 30, 30], 64, 4, 2, D, torch.float16, causal=True)


@pytest.mark.parametrize("layout", ["heads", "rows"])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_mixed_lengths(layout, D):
    """Single rows, drafted tokens, chunks and sequences without a query in one call."""
    lq = [1, 0, 5, 1, 77, 1, 4, 0, 17, 130]
    lens = [500, 200, 64, 1, 300, 129, 4, 0, 1000, 130]
    run_and_check(lens, lq, 64, 8, 2, D, torch.bfloat16, layout=layout, causal=True)


@pytest.mark.parametrize("nseq", [1, 63, 64, 65, 200])
def test_many_sequences(nseq):
    g = torch.Generator().manual_seed(nseq)
    lens = torch.randint(0, 400, (nseq,), generator=g).tolist()
    run_and_check(lens, [1] * nseq, 64, 2, 2, 32, torch.bfloat16, causal=True)


@pytest.mark.parametrize("lq", [1, 3])
def test_long_sequence_beside_short_ones(lq):
    run_and_check([20000, 3, 150], [lq] * 3, 256, 4, 1, 64, torch.bfloat16, causal=True)


@pytest.mark.parametrize("page", [64, 128, 192, 256, 320])
@pytest.mark.parametrize("lq", [[1, 3, 1], [40, 1, 70]])
def test_page_sizes(page, lq):
    """Pages that end inside a chunk, hold several, or begin between two."""
    run_and_check([777, 1000, 320], lq, page, 8, 2, 64, torch.bfloat16, causal=True)
    run_and_check([777, 1000, 320], lq, page, 8, 2, 128, torch.float16, window_size=(200, 30))


@pytest.mark.parametrize("Hq,Hkv", [(16, 1), (17, 1), (32, 1), (40, 1), (128, 1), (130, 1)])
def test_heads_that_fill_the_tiles(Hq, Hkv):
    run_and_check([257, 64, 1], [1, 1, 1], 64, Hq, Hkv, 64, torch.bfloat16, causal=True)


def test_max_seqlen_k():
    """It cuts a sequence; a bound above what the table names is no bound."""
    q, kc, vc, lens, table = make([500, 90], 64, 4, 2, 64, torch.bfloat16, [1, 1])
    args = (q.view(2, 1, 4, 64), kc, vc)
    cut = mfa.flash_attn_kv8_func(*args, lens, table, causal=True, max_seqlen_k=100)
    assert torch.equal(cut, mfa.flash_attn_kv8_func(*args, lens.clamp(max=100), table, causal=True))
    full = mfa.flash_attn_kv8_func(*args, lens, table, causal=True)
    assert torch.equal(mfa.flash_attn_kv8_func(*args, lens, table, causal=True, max_seqlen_k=1 << 30), full)
    assert not mfa.flash_attn_kv8_func(*args, lens, table, max_seqlen_k=0).any()


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
@pytest.mark.parametrize("lq", [2, 50])
def test_scales(scale, lq):
    """A scale of 0 (uniform weights), a negative one, and one that makes weights of a few keys."""
    q, kc, vc, lens, table = make([300], 64, 4, 2, 64, torch.bfloat16, [lq])
    ref, _, _ = attend64(q, kc, vc, [300], table, [lq], True, scale=scale)
    out = mfa.flash_attn_kv8_func(q.view(1, lq, 4, 64), kc, vc, lens, table, softmax_scale=scale, causal=True)
    check(out[0], ref, float(rows64(vc).abs().max()), torch.bfloat16, on_tiles([lq], 2, False))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lq", [1, 40])
def test_blocks_of_very_different_scales(dtype, lq):
    """Blocks of K and V that are 2^20 and 2^-20 times others, zero blocks between them.  (The
    bounds are those of the largest value; sum |q k| scale stays below 100.)"""
    L, H, D = 640, 2, 64
    q, kc, vc, lens, table = make([L], 64, H, H, D, dtype, [lq], spread=0.0)
    for i, e in enumerate((0, -20, 0, 8, -8, 0, -100, 0, -1, 1)):
        p = table[0, i].item()
        vc[1][p] = (vc[1][p].int() + e).clamp(1, 247).to(torch.uint8) if i != 2 else 0
        kc[1][p] = (kc[1][p].int() + min(e, 1)).clamp(1, 247).to(torch.uint8) if i != 5 else 0
    ref, _, _ = attend64(q, kc, vc, [L], table, [lq], True)
    out = mfa.flash_attn_kv8_func(q.view(1, lq, H, D), kc, vc, lens, table, causal=True)
    check(out[0], ref, float(rows64(vc).abs().max()), dtype, on_tiles([lq], 1, False))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lq", [1, 40])
def test_large_values(dtype, lq):
    """Blocks of V whose largest codes pass fp16's range saturate there on the tiles of fp16
    queries and reach no row that masks them."""
    L, D = 200, 64
    q, kc, vc, lens, table = make([L], 64, 2, 2, D, dtype, [lq], spread=0.0)
    first = table[0, 0].item()
    vc[0].view(torch.uint8)[first] = 0
    vc[0].view(torch.uint8)[first, 7] = 0x7E  # 448
    vc[1][first] = 127 + 8                    # times 256: 114688
    window = (139, 0)                         # (rows see keys from 21 or 60 on: of this block only zeros)
    out = mfa.flash_attn_kv8_func(q.view(1, lq, 2, D), kc, vc, lens, table, window_size=window)
    ref, _, _ = attend64(q, kc, vc, [L], table, [lq], window=window)
    small = rows64(vc)[table[0, 1:4].cpu().long()].abs().max()
    check(out[0], ref, float(small), dtype, on_tiles([lq], 1, False))
    seen = mfa.flash_attn_kv8_func(q.view(1, lq, 2, D), kc, vc, lens, table)
    assert bool(seen.isfinite().all())


def test_garbage_behind_the_rows():
    """Rows behind a sequence's last one, and pages of others, may hold NaN."""
    lens = [37, 130, 64]
    q, kc, vc, lens_t, table = make(lens, 64, 4, 2, 128, torch.bfloat16, [1, 1, 1])
    call = lambda: mfa.flash_attn_kv8_func(q.view(3, 1, 4, 128), kc, vc, lens_t, table, causal=True)  # noqa: E731
    before = call()
    live = torch.zeros(kc[0].shape[0], 64, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(n):
            live[table[b, j // 64].item(), j % 64] = True
    for c in (kc, vc):
        c[0].view(torch.uint8)[~live.to(DEV)] = 0xFF
    assert torch.equal(call(), before)
    # a NaN of V that a row sees shows in its element, one of K in the whole row
    vc[0].view(torch.uint8)[table[0, 0].item(), 5, 1, 66] = 0x7F
    out = call()
    assert out[0, 0, 2:, 66].isnan().all() and int(out.isnan().sum()) == 2
    kc[0].view(torch.uint8)[table[1, 1].item(), 5, 0, 3] = 0xFF
    out = call()
    assert out[1, 0, :2].isnan().all() and int(out.isnan().sum()) == 2 + 2 * 128


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("lq,Hq,window", [(1, 4, (40, 0)), (5, 4, (-1, 0)), (9, 6, (33, 0)), (70, 4, (-1, 0)), (70, 4, (50, 3)),
                                          (150, 2, (-1, -1))])
def test_nan_reaches_only_the_rows_that_see_it(D, lq, Hq, window, dtype):
    """NaN elements of V: NaN in that element of the rows whose mask holds their key, and in
    everything else the bits that it has without them."""
    L = 333
    q, kc, vc, lens, table = make([L], 64, Hq, 2, D, dtype, [lq])
    q = q.view(1, lq, Hq, D)
    call = lambda: mfa.flash_attn_kv8_func(q, kc, vc, lens, table, window_size=window)[0]  # noqa: E731
    clean = call()
    i = torch.arange(lq)[:, None] + L - lq
    j = torch.arange(L)[None]
    seen = torch.ones(lq, L, dtype=torch.bool)
    if window[0] >= 0:
        seen &= j >= i - window[0]
    if window[1] >= 0:
        seen &= j <= i + window[1]
    spots = [(L - 1, 0, 0), (L - 1, 0, 17), (L - lq // 2 - 1, 1, D - 1), (L - lq, 0, D // 2 + 5), (max(L - lq - 36, 0), 1, 9),
             (258, 0, 30), (L - 2, 1, 12), (L - 3, 1, 20)]
    want = torch.zeros(lq, Hq, D, dtype=torch.bool)
    for n, (key, h, d) in enumerate(spots):
        vc[0].view(torch.uint8)[table[0, key // 64].item(), key % 64, h, d] = 0x7F if n % 2 else 0xFF
        want[:, h * Hq // 2:(h + 1) * Hq // 2, d] |= seen[:, key][:, None]
    out = call()
    assert torch.equal(out.isnan().cpu(), want)
    assert torch.equal(out.cpu()[~want], clean.cpu()[~want])


def test_page_ids_outside_the_pool():
    """They read as zero keys and values, without a fault."""
    q, kc, vc, lens, table = make([100, 100], 64, 4, 2, 64, torch.bfloat16, [1, 1])
    table[0, 0], table[1, 1] = -7, 1 << 30
    assert torch.isfinite(mfa.flash_attn_kv8_func(q.view(2, 1, 4, 64), kc, vc, lens, table, causal=True)).all()


@pytest.mark.parametrize("scale", [None, 1e-30])
@pytest.mark.parametrize("lq", [1, 40])
def test_scale_bytes_of_0(lq, scale):
    """Blocks that nobody wrote stand for zeros, beside masked keys too."""
    L = 100
    q, kc, vc, lens, table = make([L], 64, 4, 2, 64, torch.bfloat16, [lq])
    for c in (kc, vc):
        c[0].view(torch.uint8)[table[0, 1].item()] = 0
        c[1][table[0, 1].item()] = 0
    ref, _, _ = attend64(q, kc, vc, [L], table, [lq], True, (30, 0), scale=scale)
    out = mfa.flash_attn_kv8_func(q.view(1, lq, 4, 64), kc, vc, lens, table, softmax_scale=scale, causal=True, window_size=(30, 0))
    check(out[0], ref, float(rows64(vc).abs().max()), torch.bfloat16, on_tiles([lq], 2, False))


def test_query_views_and_rows_of_no_sequence():
    q, kc, vc, lens, table = make([200, 90], 64, 4, 2, 64, torch.bfloat16, [3, 3])
    ref = mfa.flash_attn_kv8_func(q.view(2, 3, 4, 64), kc, vc, lens, table, causal=True)
    packed = torch.randn(2, 3, 8, 64, device=DEV, dtype=torch.bfloat16)
    packed[:, :, 2:6] = q.view(2, 3, 4, 64)
    assert torch.equal(mfa.flash_attn_kv8_func(packed[:, :, 2:6], kc, vc, lens, table, causal=True), ref)
    odd = torch.empty(q.numel() + 1, device=DEV, dtype=torch.bfloat16)[1:].view(2, 3, 4, 64)
    odd.copy_(q.view(2, 3, 4, 64))
    assert torch.equal(mfa.flash_attn_kv8_func(odd, kc, vc, lens, table, causal=True), ref)
    padded = torch.cat((torch.full_like(q[:2], math.nan), q, torch.full_like(q[:1], math.nan)))
    out, lse = mfa.flash_attn_varlen_kv8_func(padded, kc, vc, i32(2, 5, 8), lens, table, causal=True, return_softmax_lse=True)
    assert torch.equal(out[2:8], ref.view(6, 4, 64)) and not out[:2].any() and not out[8:].any()
    assert bool((lse[:, [0, 1, 8]] == -math.inf).all())


def test_same_bits_every_time_and_captured():
    """On another stream, and replayed as the sequences grow, with eager work in between."""
    q, kc, vc, lens, table = make([3200, 270, 700, 201], 64, 8, 2, 128, torch.bfloat16, [2] * 4)
    q, cu = q.view(4, 2, 8, 128), cu_of([2] * 4)
    run = lambda: (mfa.flash_attn_kv8_func(q, kc, vc, lens, table, causal=True),  # noqa: E731
                   mfa.flash_attn_varlen_kv8_func(q.flatten(0, 1), kc, vc, cu, lens, table, causal=True))
    ref = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        outs = [run() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    for o in outs:
        assert torch.equal(o[0], ref[0]) and torch.equal(o[1], ref[1])
    lens.sub_(160)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for _ in range(4):
        lens.add_(37)
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        ref = run()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], ref[0]) and torch.equal(outs[1], ref[1])


@pytest.mark.parametrize("lq", [1, 40])
@pytest.mark.parametrize("pages,cols", [(0, 0), (0, 2), (3, 0)])
def test_empty_pools_and_tables(lq, pages, cols):
    q = torch.randn(2, lq, 4, 64, device=DEV, dtype=torch.bfloat16)
    kc, vc = (mfa.kv8_cache(pages, 64, 2, 64) for _ in range(2))
    lens, table = i32(70, 5), torch.zeros(2, cols, dtype=torch.int32, device=DEV)
    out, lse = mfa.flash_attn_kv8_func(q, kc, vc, lens, table, return_softmax_lse=True)
    want = torch.full((2, 4, lq), -math.inf)
    if cols:
        want[:] = torch.tensor([70.0, 5.0]).log()[:, None, None]
    assert not out.any() and torch.allclose(lse.cpu(), want, rtol=1e-5, atol=1e-5)
    k = torch.randn(7, 2, 64, device=DEV, dtype=torch.bfloat16)
    mfa.kv8_append(k, k, kc, vc, i32(0, 3, 7), torch.zeros_like(lens), table)
    w = torch.zeros(pages, 64, 2, device=DEV)
    mfa.kv8_key_weights(q, kc, lse, w, lens, table)
    assert mfa.kv8_evict(kc, vc, w, lens, table, 3, 1).tolist() == ([3, 3] if cols else [0, 0])
    assert not any(x.view(torch.uint8).any() for c in (kc, vc) for x in c) and not w.any()
    assert mfa.flash_attn_varlen_kv8_func(q[:0, 0], kc, vc, i32(0, 0, 0), lens, table).shape == (0, 4, 64)
    assert not mfa.flash_attn_varlen_kv8_func(q[:, 0], kc, vc, i32(0, 0, 0), lens, table).any()


def test_offsets_past_32_bits():
    page, H, D = 256, 8, 128
    pages = (1 << 32) // (page * H * D) + 8
    g = torch.Generator().manual_seed(1)
    small = [filled_cache(g, 4, page, H, D) for _ in range(2)]
    big = []
    for c in small:
        x = mfa.kv8_cache(pages, page, H, D)
        x[0][-4:].view(torch.uint8).copy_(c[0].view(torch.uint8))
        x[1][-4:] = c[1]
        big.append(x)
    for lq in (2, 40):
        q = torch.randn(1, lq, 16, D, device=DEV, dtype=torch.bfloat16)
        table = i32(0, 1, 2, 3)[None]
        ref, lse = mfa.flash_attn_kv8_func(q, *small, i32(1000), table, causal=True, return_softmax_lse=True)
        out = mfa.flash_attn_kv8_func(q, *big, i32(1000), table + (pages - 4), causal=True)
        assert torch.equal(out, ref)
        w = [torch.ones(n, H, page, device=DEV).transpose(1, 2) for n in (4, pages)]
        mfa.kv8_key_weights(q, small[0], lse, w[0], i32(1000), table, causal=True)
        mfa.kv8_key_weights(q, big[0], lse, w[1], i32(1000), table + (pages - 4), causal=True)
        assert torch.equal(w[0], w[1][-4:]) and bool((w[1][:-4] == 1).all())
    before = [c[0].view(torch.uint8).clone() for c in small]
    mfa.kv8_evict(*small, w[0], i32(1000), table, 300, 20)
    mfa.kv8_evict(*big, w[1], i32(1000), table + (pages - 4), 300, 20)
    for a, b, c in zip(small, big, before):
        assert torch.equal(a[0].view(torch.uint8), b[0][-4:].view(torch.uint8)) and torch.equal(a[1], b[1][-4:])
        assert not torch.equal(a[0].view(torch.uint8), c)
    assert torch.equal(w[0], w[1][-4:])
