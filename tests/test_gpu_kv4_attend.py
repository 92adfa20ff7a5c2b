"""Attention over the paged 4-bit cache against the definition in float64.

The oracle reads the same codes and scales, so the quantisation plays no part: what
is tested is the attention.  Bounds: the output is rounded to its type (half a step,
finfo.eps / 2 relative), and before that carries fp32 sums and probabilities of two
bf16 terms; a probability is off by at most 2^-16 relative (the second term's
rounding, 2^-8 of 2^-8), its sum by fp32 rounding.  With |v| <= vmax that is
2^-16 vmax, scores add |ds| <= 2^-22 * sum |q k| scale through exp.  3e-4 * vmax
covers both for the sizes here (sum |q k| scale < 100: 100 * 2^-22 = 2.4e-5).

Sequences of more than 32 columns (query rows times query heads per K/V head; in a
varlen call more than 16, unless the whole call has at most 32) run on tiles of 128
columns, whose probabilities are rounded once to the queries' type, p (1 + d) with |d|
<= u = finfo.eps / 2, and whose row sum adds the rounded values.  Then
  |sum p (1 + d) v / sum p (1 + d) - o| = |sum p d (v - o)| / sum p (1 + d) <= 2 u vmax / (1 - u)
and the log-sum-exp is off by at most -ln(1 - u) <= 1.01 u.
"""
from __future__ import annotations

import math

import pytest
import torch

import mtlflashattn_amd as mfa

pytestmark = pytest.mark.gpu
DEV = "cuda"
LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def rows64(codes, scales):
    """float64 rows of (codes, scales), on the CPU."""
    codes, scales = codes.cpu().long(), scales.cpu().double()
    x = torch.stack((LEVELS[codes & 15], LEVELS[codes >> 4]), -1).flatten(-2)
    s = torch.where(scales == 255, torch.full_like(scales, math.nan), torch.pow(2.0, scales - 127))
    return x * s.repeat_interleave(32, -1)


def random_cache(g, pages, page, H, D, layout="heads"):
    """Random codes with scales near 2^-1; layout: heads-second or rows-first memory."""
    out = []
    for n, top in ((D // 2, 256), (D // 32, 4)):
        t = torch.randint(0, top, (pages, H, page, n), generator=g, dtype=torch.uint8)
        if top == 4:
            t = t + 123
        t = t.to(DEV)
        out.append(t.transpose(1, 2) if layout == "heads" else t.transpose(1, 2).contiguous())
    return tuple(out)


def make(lens, page, Hq, Hkv, D, dtype, lq, seed=0, layout="heads", extra_cols=1):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    kc, vc = random_cache(g, pages, page, Hkv, D, layout), random_cache(g, pages, page, Hkv, D, layout)
    ids = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), max(need + [0]) + extra_cols), 1 << 20, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = ids.pop()
    rows = sum(lq)
    q = torch.randn(rows, Hq, D, generator=g).to(DEV, dtype)
    return q, kc, vc, torch.tensor(lens, dtype=torch.int32, device=DEV), table.to(DEV)


def oracle(q, kc, vc, lens, table, lq, causal=False, window=(-1, -1), softcap=0.0, slopes=None, scale=None):
    """float64 (out [rows, Hq, D], lse [Hq, rows]) of packed q."""
    q = q.cpu().double()
    rows, Hq, D = q.shape
    Hkv, page = kc[0].shape[2], kc[0].shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out, lse = torch.zeros(rows, Hq, D, dtype=torch.float64), torch.full((Hq, rows), -math.inf, dtype=torch.float64)
    k64, v64 = rows64(*kc), rows64(*vc)
    start = 0
    for b, n in enumerate(lq):
        L = int(lens[b])
        ids = table[b, :-(-L // page)].cpu().long()
        K, V = (x[ids].flatten(0, 1)[:L] for x in (k64, v64))
        i = torch.arange(n)[:, None] + L - n
        j = torch.arange(L)[None]
        ok = torch.ones(n, L, dtype=torch.bool)
        if causal:
            ok &= j <= i
        if window[0] >= 0:
            ok &= j >= i - window[0]
        if window[1] >= 0:
            ok &= j <= i + window[1]
        for h in range(Hq):
            s = q[start:start + n, h] @ K[:, h * Hkv // Hq].T * scale
            if softcap > 0:
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                s = s - float(slopes[b, h] if slopes.dim() == 2 else slopes[h]) * (i - j).abs()
            s = s.masked_fill(~ok, -math.inf)
            p = torch.softmax(s, -1) if L else torch.zeros(n, 0, dtype=torch.float64)
            p = torch.where(ok.any(-1, keepdim=True), p, 0.0)
            out[start:start + n, h] = torch.where(p[:, :, None] > 0, p[:, :, None] * V[:, h * Hkv // Hq], 0.0).sum(1)
            lse[h, start:start + n] = torch.logsumexp(s, -1)
        start += n
    return out, lse


def on_tiles(lq, R, varlen):
    """Per query row: whether its sequence runs on 128-column tiles."""
    few = sum(lq) * R <= 32 if varlen else lq[0] * R <= 32
    return torch.tensor([not few and n * R > (16 if varlen else 32) for n in lq for _ in range(n)], dtype=torch.float64)


def check(out, ref, vmax, dtype, tiles=None):
    err = (out.cpu().double() - ref).abs()
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + 3e-4 * vmax
    if tiles is not None:
        tol = tol + tiles[:, None, None] * (1.02 * torch.finfo(dtype).eps * vmax)
    assert not out.isnan().any()
    assert bool((err <= tol).all()), f"max err {float(err.max()):.3e}, bound there {float(tol.flatten()[err.argmax()]):.3e}"


def run_and_check(lens, lq, page, Hq, Hkv, D, dtype, seed=0, layout="heads", max_k=None, slopes=None, **kw):
    q, kc, vc, lens_t, table = make(lens, page, Hq, Hkv, D, dtype, lq, seed, layout)
    ref, ref_lse = oracle(q, kc, vc, lens, table, lq, kw.get("causal", False), kw.get("window_size", (-1, -1)),
                          kw.get("softcap", 0.0), slopes)
    sl = None if slopes is None else slopes.to(DEV)
    vmax = float(rows64(*vc).abs().max())
    got = []
    if len(set(lq)) == 1:
        o, lse = mfa.flash_attn_kv4_func(q.view(len(lq), lq[0], Hq, D), kc, vc, lens_t, table, max_seqlen_k=max_k,
                                         alibi_slopes=sl, return_softmax_lse=True, **kw)
        assert o.shape == (len(lq), lq[0], Hq, D) and lse.shape == (len(lq), Hq, lq[0])
        got.append((o.reshape(-1, Hq, D), lse.transpose(0, 1).reshape(Hq, -1), on_tiles(lq, Hq // Hkv, False)))
    cu = torch.tensor([0] + lq, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV)
    o, lse = mfa.flash_attn_varlen_kv4_func(q, kc, vc, cu, lens_t, table, max_seqlen_k=max_k, alibi_slopes=sl,
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


@pytest.mark.parametrize("kw", [
    dict(), dict(causal=True), dict(causal=True, window_size=(100, -1)), dict(window_size=(30, 20)),
    dict(window_size=(0, 0)), dict(window_size=(-1, 3)), dict(causal=True, softcap=2.0),
    dict(causal=True, window_size=(300, 0), softcap=5.0),
])
@pytest.mark.parametrize("lq", [1, 7, 70])
def test_masks(kw, lq):
    run_and_check([lq, 900, 513], [lq] * 3, 64, 4, 2, 64, torch.bfloat16, **kw)


@pytest.mark.parametrize("per_batch", [False, True])
@pytest.mark.parametrize("lq", [1, 6])
def test_alibi(lq, per_batch):
    slopes = torch.tensor([0.5, 0.01, 0.3, 0.0])
    if per_batch:
        slopes = torch.stack((slopes, slopes.flip(0)))
    run_and_check([400, 77], [lq] * 2, 64, 4, 2, 128, torch.float16, causal=True, slopes=slopes)


def test_more_queries_than_keys():
    """Rows before the first key see nothing: 0 and -inf."""
    run_and_check([3, 0, 20], [8, 8, 8], 64, 4, 2, 64, torch.bfloat16, causal=True)
    run_and_check([3, 0, 20], [30, 30, 30], 64, 4, 2, 64, torch.float16, causal=True)


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


def test_lengths_bounded_by_max_seqlen_k():
    """max_seqlen_k cuts a sequence; a bound above what the table names is no bound."""
    lens, lq = [500, 90], [1, 1]
    q, kc, vc, lens_t, table = make(lens, 64, 4, 2, 64, torch.bfloat16, lq)
    args = (q.view(2, 1, 4, 64), kc, vc)
    cut = mfa.flash_attn_kv4_func(*args, lens_t, table, causal=True, max_seqlen_k=100)
    ref = mfa.flash_attn_kv4_func(*args, lens_t.clamp(max=100), table, causal=True)
    assert torch.equal(cut, ref)
    full = mfa.flash_attn_kv4_func(*args, lens_t, table, causal=True)
    assert torch.equal(mfa.flash_attn_kv4_func(*args, lens_t, table, causal=True, max_seqlen_k=1 << 30), full)
    assert not mfa.flash_attn_kv4_func(*args, lens_t, table, max_seqlen_k=0).any()


def test_garbage_behind_the_rows():
    """Rows behind a sequence's last one, and pages of others, may hold NaN."""
    lens, lq = [37, 130, 64], [1, 1, 1]
    q, kc, vc, lens_t, table = make(lens, 64, 4, 2, 128, torch.bfloat16, lq)
    before = mfa.flash_attn_kv4_func(q.view(3, 1, 4, 128), kc, vc, lens_t, table, causal=True)
    live = torch.zeros(kc[0].shape[0], 64, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(n):
            live[table[b, j // 64].item(), j % 64] = True
    for c in (kc, vc):
        c[1][~live.to(DEV)] = 255
    after = mfa.flash_attn_kv4_func(q.view(3, 1, 4, 128), kc, vc, lens_t, table, causal=True)
    assert torch.equal(before, after) and not after.isnan().any()
    # a NaN that a row does see shows
    vc[1][table[0, 0].item(), 5, 1, 2] = 255
    out = mfa.flash_attn_kv4_func(q.view(3, 1, 4, 128), kc, vc, lens_t, table, causal=True)
    assert out[0, 0, 2:, 64:96].isnan().all() and not out[1:].isnan().any()


def test_page_ids_outside_the_pool():
    """They read as zero keys and values, without a fault."""
    lens, lq = [100, 100], [1, 1]
    q, kc, vc, lens_t, table = make(lens, 64, 4, 2, 64, torch.bfloat16, lq)
    table[0, 0], table[1, 1] = -7, 1 << 30
    out = mfa.flash_attn_kv4_func(q.view(2, 1, 4, 64), kc, vc, lens_t, table, causal=True)
    assert torch.isfinite(out).all()


def test_query_views():
    """Queries read in place from a packed projection, and an unaligned one."""
    lens = [200, 90]
    q, kc, vc, lens_t, table = make(lens, 64, 4, 2, 64, torch.bfloat16, [3, 3])
    ref = mfa.flash_attn_kv4_func(q.view(2, 3, 4, 64), kc, vc, lens_t, table, causal=True)
    packed = torch.randn(2, 3, 8, 64, device=DEV, dtype=torch.bfloat16)
    packed[:, :, 2:6] = q.view(2, 3, 4, 64)
    assert torch.equal(mfa.flash_attn_kv4_func(packed[:, :, 2:6], kc, vc, lens_t, table, causal=True), ref)
    odd = torch.empty(q.numel() + 1, device=DEV, dtype=torch.bfloat16)[1:].view(2, 3, 4, 64)
    odd.copy_(q.view(2, 3, 4, 64))
    assert torch.equal(mfa.flash_attn_kv4_func(odd, kc, vc, lens_t, table, causal=True), ref)
    t = q.view(2, 3, 4, 64).transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(mfa.flash_attn_kv4_func(t, kc, vc, lens_t, table, causal=True), ref)


def test_same_bits_every_time_and_on_a_stream():
    lens = [3000, 70, 500, 1]
    q, kc, vc, lens_t, table = make(lens, 64, 8, 2, 128, torch.bfloat16, [2] * 4)
    call = lambda: mfa.flash_attn_kv4_func(q.view(4, 2, 8, 128), kc, vc, lens_t, table, causal=True)  # noqa: E731
    ref = call()
    for _ in range(5):
        assert torch.equal(call(), ref)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = call()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, ref)


def test_captured_call_follows_the_lengths():
    """A captured step replayed as the sequences grow, with eager work in between."""
    lens, Hq, Hkv, D = [60, 300], 4, 2, 64
    q, kc, vc, lens_t, table = make([l + 200 for l in lens], 64, Hq, Hkv, D, torch.bfloat16, [1, 1])
    lens_t.copy_(torch.tensor(lens, dtype=torch.int32))
    q4, cu = q.view(2, 1, Hq, D).clone(), torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    run = lambda: (mfa.flash_attn_kv4_func(q4, kc, vc, lens_t, table, causal=True),  # noqa: E731
                   mfa.flash_attn_varlen_kv4_func(q4[:, 0], kc, vc, cu, lens_t, table, causal=True))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for step in range(4):
        lens_t.add_(37)
        q4.normal_()
        graph.replay()
        torch.cuda.synchronize()
        ref = run()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], ref[0]) and torch.equal(outs[1], ref[1])


def test_rows_of_no_sequence():
    lens = [90, 200]
    q, kc, vc, lens_t, table = make(lens, 64, 4, 2, 64, torch.bfloat16, [1, 9])
    cu = torch.tensor([0, 1, 8], dtype=torch.int32, device=DEV)
    out, lse = mfa.flash_attn_varlen_kv4_func(q, kc, vc, cu, lens_t, table, causal=True, return_softmax_lse=True)
    assert not out[8:].any() and bool((lse[:, 8:] == -math.inf).all())
    ref = mfa.flash_attn_varlen_kv4_func(q[:8], kc, vc, cu, lens_t, table, causal=True)
    assert torch.equal(out[:8], ref)


def test_row_offsets_past_32_bits():
    """A pool of more than 4 GiB of codes: the last pages are the ones in use."""
    page, H, D = 256, 8, 128
    pages = (1 << 32) // (page * H * D // 2) + 64
    g = torch.Generator().manual_seed(1)
    small_k, small_v = random_cache(g, 4, page, H, D), random_cache(g, 4, page, H, D)
    big = []
    for small in (small_k, small_v):
        pair = []
        for t in small:
            x = torch.empty(pages, H, page, t.shape[-1], dtype=torch.uint8, device=DEV).transpose(1, 2)
            x[-4:] = t
            pair.append(x)
        big.append(tuple(pair))
    q = torch.randn(1, 2, 16, D, device=DEV, dtype=torch.bfloat16)
    lens = torch.tensor([1000], dtype=torch.int32, device=DEV)
    table = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    ref = mfa.flash_attn_kv4_func(q, small_k, small_v, lens, table, causal=True)
    out = mfa.flash_attn_kv4_func(q, *big, lens, table + (pages - 4), causal=True)
    assert torch.equal(out, ref)


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("lq,Hq,window", [(1, 4, (40, 0)), (5, 4, (-1, 0)), (9, 6, (33, 0)), (70, 4, (-1, 0)), (70, 4, (50, 3)),
                                          (150, 2, (-1, -1))])
def test_nan_values_reach_only_the_rows_that_see_them(D, lq, Hq, window):
    """Groups of V that are NaN: NaN in the rows whose mask holds their key, and in
    every other row the bits that it has without them."""
    L = 333
    q, kc, vc, lens_t, table = make([L], 64, Hq, 2, D, torch.bfloat16, [lq])
    q = q.view(1, lq, Hq, D)
    call = lambda: mfa.flash_attn_kv4_func(q, kc, vc, lens_t, table, window_size=window)[0]  # noqa: E731
    clean = call()
    i = torch.arange(lq)[:, None] + L - lq
    j = torch.arange(L)[None]
    seen = torch.ones(lq, L, dtype=torch.bool)
    if window[0] >= 0:
        seen &= j >= i - window[0]
    if window[1] >= 0:
        seen &= j <= i + window[1]
    spots = [(L - 1, 0, 0), (L - lq // 2 - 1, 1, D // 32 - 1), (L - lq, 0, D // 64), (max(L - lq - 36, 0), 1, 0), (258, 0, 0)]
    want = torch.zeros(lq, Hq, D, dtype=torch.bool)
    for key, h, grp in spots:
        vc[1][table[0, key // 64].item(), key % 64, h, grp] = 255
        want[:, h * Hq // 2:(h + 1) * Hq // 2, 32 * grp:32 * grp + 32] |= seen[:, key][:, None, None]
    out = call()
    assert torch.equal(out.isnan().cpu(), want)
    assert torch.equal(out.cpu()[~want], clean.cpu()[~want])


@pytest.mark.parametrize("page", [64, 128, 192, 256, 320])
@pytest.mark.parametrize("lq", [[1, 3, 1], [40, 1, 70]])
def test_page_sizes(page, lq):
    """Pages that end inside a chunk, hold several, or begin between two."""
    run_and_check([777, 1000, 320], lq, page, 8, 2, 64, torch.bfloat16, causal=True)
    run_and_check([777, 1000, 320], lq, page, 8, 2, 128, torch.float16, window_size=(200, 30))


@pytest.mark.parametrize("Hq,Hkv", [(16, 1), (17, 1), (32, 1), (40, 1), (128, 1), (130, 1)])
def test_heads_that_fill_the_tiles(Hq, Hkv):
    """Single rows whose heads alone are 16, 32, 128 columns and one or two more."""
    run_and_check([257, 64, 1], [1, 1, 1], 64, Hq, Hkv, 64, torch.bfloat16, causal=True)


def test_many_sequences_of_many_rows():
    g = torch.Generator().manual_seed(5)
    lq = torch.randint(0, 45, (100,), generator=g).tolist()
    lens = [n + int(x) for n, x in zip(lq, torch.randint(0, 200, (100,), generator=g))]
    run_and_check(lens, lq, 64, 4, 1, 32, torch.bfloat16, causal=True)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
@pytest.mark.parametrize("lq", [2, 50])
def test_scales(scale, lq):
    """A scale of 0 (uniform weights), a negative one, and one that makes weights of a single key."""
    q, kc, vc, lens, table = make([300], 64, 4, 2, 64, torch.bfloat16, [lq])
    kc[1].copy_(torch.full_like(kc[1], 122))
    ref, _ = oracle(q, kc, vc, lens.cpu(), table, [lq], True, scale=scale)
    out = mfa.flash_attn_kv4_func(q.view(1, lq, 4, 64), kc, vc, lens, table, softmax_scale=scale, causal=True)
    check(out[0], ref, float(rows64(*vc).abs().max()), torch.bfloat16, on_tiles([lq], 2, False))


@pytest.mark.parametrize("lq", [1, 40])
@pytest.mark.parametrize("pages,cols", [(0, 0), (0, 2), (3, 0)])
def test_empty_pools_and_tables(lq, pages, cols):
    """No page, or none named: no key where the table is empty, zero keys and values
    where its ids name nothing; what is appended is dropped."""
    q = torch.randn(2, lq, 4, 64, device=DEV, dtype=torch.bfloat16)
    kc, vc = (mfa.kv4_cache(pages, 64, 2, 64) for _ in range(2))
    lens = torch.tensor([70, 5], dtype=torch.int32, device=DEV)
    table = torch.zeros(2, cols, dtype=torch.int32, device=DEV)
    out, lse = mfa.flash_attn_kv4_func(q, kc, vc, lens, table, return_softmax_lse=True)
    want = torch.full((2, 4, lq), -math.inf)
    if cols:
        want[:] = torch.tensor([70.0, 5.0]).log()[:, None, None]
    assert not out.any() and torch.allclose(lse.cpu(), want, rtol=1e-5, atol=1e-5)
    k = torch.randn(7, 2, 64, device=DEV, dtype=torch.bfloat16)
    mfa.kv4_append(k, k, kc, vc, torch.tensor([0, 3, 7], dtype=torch.int32, device=DEV), torch.zeros_like(lens), table)
    assert not any(x.any() for c in (kc, vc) for x in c)
    cu = torch.tensor([0, 0, 0], dtype=torch.int32, device=DEV)
    assert mfa.flash_attn_varlen_kv4_func(q[:0, 0], kc, vc, cu, lens, table).shape == (0, 4, 64)
    assert not mfa.flash_attn_varlen_kv4_func(q[:, 0], kc, vc, cu, lens, table).any()
