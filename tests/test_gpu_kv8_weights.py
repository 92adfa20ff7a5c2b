"""The attention weight that each cached key received, against the definition in float64.

Bounds: a probability exp(s - lse) is off by its exponent's error, and the sums by theirs.
Scores are fp32 sums of exact products (|ds| <= 2^-22 sum |q k| scale, the sum below 100:
2.4e-5); lse in log2 units, the score's scaling and their difference round three numbers
below 64 to 2^-24 each (1.2e-5 together); the soft-cap adds 2^-21 of its bound (at most
8: 4e-6) and ALiBi two roundings of terms below 256 (3.1e-5); exp2 is within 2^-23.  That is less than
8e-5 of every probability, hence of their sum; adding n of them in fp32 costs at most n
2^-24 of it, the old weight one more rounding.
"""
from __future__ import annotations

import math

import pytest
import torch

import mtlflashattn_amd as mfa
from kv8_util import DEV, attend64, cu_of, i32, make

pytestmark = pytest.mark.gpu


def pool_like(kc, g):
    """A weight pool with what earlier steps left, each head's rows of a page side by side."""
    pages, page, H = kc[0].shape[:3]
    return torch.rand(pages, H, page, generator=g).to(DEV).transpose(1, 2)


def expected(before, weights, lens, lq, table, page):
    """(the pool after the step, its bound) on the CPU, from the sums of each sequence."""
    want, tol = before.cpu().double().clone(), torch.zeros(before.shape, dtype=torch.float64)
    for b, (L, n) in enumerate(zip(lens, lq)):
        if n == 0:
            continue
        for j in range(L):
            p = int(table[b, j // page])
            at = (p, j % page)
            new = weights[b][:, j]
            old = want[at] if j < L - n else torch.zeros_like(new)
            want[at] = old + new
            tol[at] = want[at] * 2.0 ** -23 + new * 8e-5
    return want, tol


def run_and_check(lens, lq, page, Hq, Hkv, D, dtype, seed=0, layout="heads", max_k=None, slopes=None, scale=None, **kw):
    q, kc, vc, lens_t, table = make(lens, page, Hq, Hkv, D, dtype, lq, seed, layout)
    _, ref_lse, sums = attend64(q, kc, vc, lens, table, lq, kw.get("causal", False), kw.get("window_size", (-1, -1)),
                                kw.get("softcap", 0.0), slopes, scale)
    sl = None if slopes is None else slopes.to(DEV)
    w0 = pool_like(kc, torch.Generator().manual_seed(seed))
    want, tol = expected(w0, sums, lens, lq, table.cpu(), page)
    tol = tol + want * max(lq) * (Hq // Hkv) * 2.0 ** -24
    lse = ref_lse.float().to(DEV)
    got = []
    args = dict(alibi_slopes=sl, max_seqlen_k=max_k, softmax_scale=scale, **kw)
    if len(set(lq)) == 1:
        w = w0.clone()
        dense = lse.view(Hq, len(lq), lq[0]).transpose(0, 1)  # (not contiguous: taken as it is)
        mfa.kv8_key_weights(q.view(len(lq), lq[0], Hq, D), kc, dense, w, lens_t, table, **args)
        got.append(w)
    w = w0.clone()
    mfa.kv8_key_weights(q, kc, lse, w, lens_t, table, cu_of(lq), **args)
    got.append(w)
    for w in got:
        err = (w.cpu().double() - want).abs()
        assert bool((err <= tol).all()), f"max err {float(err.max()):.3e}, bound there {float(tol.flatten()[err.argmax()]):.3e}"
    return w0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (5, 1), (20, 1)])
def test_single_rows(D, Hq, Hkv, dtype):
    run_and_check([1, 33, 64, 129, 700, 0, 255], [1] * 7, 64, Hq, Hkv, D, dtype, causal=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("lq", [2, 5, 9, 40, 130])
def test_several_rows(D, lq, dtype):
    run_and_check([lq, 300, 141, 1000], [lq] * 4, 128, 6, 2, D, dtype, causal=True)


@pytest.mark.parametrize("kw", [
    dict(), dict(causal=True), dict(causal=True, window_size=(100, -1)), dict(window_size=(30, 20)),
    dict(window_size=(0, 0)), dict(window_size=(-1, 3)), dict(causal=True, softcap=2.0),
    dict(causal=True, window_size=(300, 0), softcap=8.0),
])
@pytest.mark.parametrize("lq", [1, 7, 70, 200])
def test_masks(kw, lq):
    run_and_check([lq, 900, 513], [lq] * 3, 64, 4, 2, 64, torch.bfloat16, **kw)


@pytest.mark.parametrize("per_batch", [False, True])
@pytest.mark.parametrize("lq", [1, 6, 40])
def test_alibi(lq, per_batch):
    slopes = torch.tensor([0.5, 0.01, 0.3, 0.0])
    if per_batch:
        slopes = torch.stack((slopes, slopes.flip(0)))
    run_and_check([400, 77], [lq] * 2, 64, 4, 2, 128, torch.float16, causal=True, slopes=slopes)


@pytest.mark.parametrize("kw", [
    dict(causal=True), dict(causal=True, window_size=(100, -1)), dict(window_size=(30, 20)), dict(causal=True, softcap=2.0),
    dict(causal=True, slopes=torch.tensor([0.5, 0.01, 0.3, 0.0, 0.1, 0.2])),
])
@pytest.mark.parametrize("D,dtype", [(32, torch.float16), (64, torch.bfloat16), (96, torch.bfloat16), (128, torch.float16)])
def test_two_tiles_of_columns(D, dtype, kw):
    run_and_check([7, 900, 513], [7] * 3, 64, 6, 2, D, dtype, **kw)
    run_and_check([10, 900, 513, 64, 33, 300], [10, 11, 1, 0, 33, 8], 64, 6, 2, D, dtype, **kw)


@pytest.mark.parametrize("scale", [0.0, -0.2, 0.3])
@pytest.mark.parametrize("lq", [2, 50])
def test_scales(scale, lq):
    run_and_check([300], [lq], 64, 4, 2, 64, torch.bfloat16, causal=True, scale=scale)


@pytest.mark.parametrize("D", [32, 128])
def test_more_queries_than_keys(D):
    """Rows before the first key add nothing; every key is the queries' own and starts from 0."""
    run_and_check([3, 0, 20], [8, 8, 8], 64, 4, 2, D, torch.bfloat16, causal=True)
    run_and_check([3, 0, 20], [30, 30, 30], 64, 4, 2, D, torch.float16, causal=True)


@pytest.mark.parametrize("layout", ["heads", "rows"])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_mixed_lengths(layout, D):
    lq = [1, 0, 5, 1, 77, 1, 4, 0, 17, 130]
    lens = [500, 200, 64, 1, 300, 129, 4, 0, 1000, 130]
    run_and_check(lens, lq, 64, 8, 2, D, torch.bfloat16, layout=layout, causal=True)


@pytest.mark.parametrize("nseq", [1, 63, 65, 200])
def test_many_sequences(nseq):
    g = torch.Generator().manual_seed(nseq)
    lq = torch.randint(0, 12, (nseq,), generator=g).tolist()
    lens = [n + int(x) for n, x in zip(lq, torch.randint(0, 300, (nseq,), generator=g))]
    run_and_check(lens, lq, 64, 4, 2, 32, torch.bfloat16, causal=True)


@pytest.mark.parametrize("page", [64, 192, 320])
@pytest.mark.parametrize("lq", [[1, 3, 1], [40, 1, 70]])
def test_page_sizes(page, lq):
    run_and_check([777, 1000, 320], lq, page, 8, 2, 64, torch.bfloat16, causal=True)


@pytest.mark.parametrize("Hq,Hkv", [(16, 1), (17, 1), (32, 1), (33, 1), (64, 1), (65, 1), (130, 1)])
def test_heads_that_fill_the_tiles(Hq, Hkv):
    run_and_check([257, 64, 1], [1, 1, 1], 64, Hq, Hkv, 64, torch.bfloat16, causal=True)


def test_a_step_gives_each_query_a_weight_of_one():
    """With the attention call's own log-sum-exps: what a row gives to all keys adds up to 1 (each
    of the L probabilities within 1e-4 of itself, single rows' lse within 1e-5)."""
    L, Hq, Hkv = 3001, 8, 2
    q, kc, vc, lens, table = make([L, 200], 256, Hq, Hkv, 128, torch.bfloat16, [1, 1])
    q = q.view(2, 1, Hq, 128)
    _, lse = mfa.flash_attn_kv8_func(q, kc, vc, lens, table, causal=True, return_softmax_lse=True)
    w = torch.zeros(kc[0].shape[:3], device=DEV)
    mfa.kv8_key_weights(q, kc, lse, w, lens, table, causal=True)
    assert abs(float(w.double().sum()) - 2 * Hq) <= 2 * Hq * 2e-4
    mfa.kv8_key_weights(q, kc, lse, w, lens, table, causal=True)  # (the last rows start from 0 again)
    last = [(table[b, (n - 1) // 256].item(), (n - 1) % 256) for b, n in enumerate((L, 200))]
    own = sum(float(w[at].double().sum()) for at in last)
    assert abs(float(w.double().sum()) - (4 * Hq - own)) <= 4 * Hq * 2e-4


@pytest.mark.parametrize("lq", [1, 40])
def test_nan_and_infinities(lq):
    """A NaN key makes its own weight NaN where a row sees it, and no other; rows whose lse is -inf
    add nothing; weights of keys behind the rows and of other pages stay."""
    L, Hq, Hkv, D = 300, 4, 2, 64
    q, kc, vc, lens, table = make([L], 64, Hq, Hkv, D, torch.bfloat16, [lq])
    lse = attend64(q, kc, vc, [L], table, [lq], window=(50, 0))[1].float().to(DEV)
    w0 = pool_like(kc, torch.Generator().manual_seed(0))
    call = lambda lse: mfa.kv8_key_weights(q.view(1, lq, Hq, D), kc, lse[None], w, lens, table, window_size=(50, 0))  # noqa: E731
    w = w0.clone()
    call(lse)
    clean = w
    seen, hidden, behind = L - lq - 3, L - lq - 53, L + 2
    for j in (seen, hidden, behind):
        kc[0].view(torch.uint8)[table[0, j // 64].item(), j % 64, 1, 7] = 0x7F
    w = w0.clone()
    call(lse)
    at = (table[0, seen // 64].item(), seen % 64, 1)
    assert w[at].isnan() and int(w.isnan().sum()) == 1
    w[at] = clean[at]
    assert torch.equal(w, clean)
    p = table[0, 4].item()
    assert torch.equal(w[p, L % 64:], w0[p, L % 64:])
    w = w0.clone()
    call(torch.full_like(lse, -math.inf))
    want = w0.clone()
    for j in range(L - lq, L):
        want[table[0, j // 64].item(), j % 64] = 0
    keep = torch.ones_like(want, dtype=torch.bool)
    keep[at] = keep[(table[0, hidden // 64].item(), hidden % 64, 1)] = False
    assert torch.equal(w[keep], want[keep])


def test_layouts_streams_and_graphs():
    """Pools in any order, the same bits every time, on another stream and replayed."""
    lens, lq = [900, 70, 300], [1, 40, 3]
    q, kc, vc, lens_t, table = make(lens, 64, 8, 2, 64, torch.bfloat16, lq)
    cu = cu_of(lq)
    lse = attend64(q, kc, vc, lens, table, lq, causal=True)[1].float().to(DEV)
    w0 = pool_like(kc, torch.Generator().manual_seed(0))
    ref = w0.clone()
    mfa.kv8_key_weights(q, kc, lse, ref, lens_t, table, cu, causal=True)
    flat = w0.contiguous()
    wide = torch.zeros(w0.shape[0], 65, 5, device=DEV)[:, 1:, 1:4:2]
    wide.copy_(w0)
    qkv = torch.randn(q.shape[0], 12, 64, device=DEV, dtype=torch.bfloat16)
    qkv[:, 2:10] = q
    for w, x in ((flat, q), (wide, qkv[:, 2:10])):
        mfa.kv8_key_weights(x, kc, lse, w, lens_t.long(), table, cu.long(), causal=True)
        assert torch.equal(w, ref)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        w = w0.clone()
        mfa.kv8_key_weights(q, kc, lse, w, lens_t, table, cu, causal=True)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(w, ref)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mfa.kv8_key_weights(q, kc, lse, w, lens_t, table, cu, causal=True)
    eager = ref.clone()
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        mfa.kv8_key_weights(q, kc, lse, eager, lens_t, table, cu, causal=True)
        torch.cuda.synchronize()
        assert torch.equal(w, eager)


def test_page_ids_outside_the_pool():
    q, kc, vc, lens, table = make([100, 100], 64, 4, 2, 64, torch.bfloat16, [1, 1])
    table[0, 0], table[1, 1] = -7, 1 << 30
    w = torch.ones(kc[0].shape[:3], device=DEV)
    mfa.kv8_key_weights(q.view(2, 1, 4, 64), kc, torch.zeros(2, 4, 1, device=DEV), w, lens, table, causal=True)
    assert bool(w.isfinite().all())
    used = torch.zeros(w.shape[:2], dtype=torch.bool, device=DEV)
    used[table[0, 1], :36] = True
    used[table[1, 0]] = True
    assert bool((w[~used] == 1).all()) and bool((w[used] != 1).any())


@pytest.mark.parametrize("kw", [dict(), dict(softcap=4.0), dict(window_size=(2500, -1))])
@pytest.mark.parametrize("D", [32, 96])
def test_many_chunks_of_many_heads(D, kw):
    """More chunks than workgroups: several per workgroup, several blocks of keys per wavefront, the
    sums of some chunks after those of others; beside a sequence of few columns."""
    run_and_check([6400, 3001], [40, 24], 64, 48, 48, D, torch.bfloat16, causal=True, **kw)
    run_and_check([6400, 3001], [40, 3], 64, 48, 48, D, torch.bfloat16, causal=True, **kw)


@pytest.mark.parametrize("lq", [1, 6, 70])
def test_max_seqlen_k(lq):
    """It cuts a sequence as its length would; 0 leaves every weight as it was."""
    q, kc, _, lens_t, table = make([900, 500], 64, 8, 2, 64, torch.bfloat16, [lq] * 2)
    q = q.view(2, lq, 8, 64)
    lse = torch.randn(2, 8, lq, device=DEV) + 6
    w0 = pool_like(kc, torch.Generator().manual_seed(1))
    cut, short, none = w0.clone(), w0.clone(), w0.clone()
    mfa.kv8_key_weights(q, kc, lse, cut, lens_t, table, causal=True, max_seqlen_k=450)
    mfa.kv8_key_weights(q, kc, lse, short, i32(450, 450), table, causal=True)
    mfa.kv8_key_weights(q, kc, lse, none, lens_t, table, causal=True, max_seqlen_k=0)
    assert torch.equal(cut, short) and not torch.equal(cut, w0) and torch.equal(none, w0)
    mfa.kv8_key_weights(q, kc, lse, none, i32(0, -3), table, causal=True)
    mfa.kv8_key_weights(q[:0], kc, lse[:0], none, lens_t[:0], table[:0], causal=True)
    mfa.kv8_key_weights(q[:, :0], kc, lse[:, :, :0], none, lens_t, table, causal=True)
    assert torch.equal(none, w0)


@pytest.mark.parametrize("heads", [2, 40])
def test_weights_past_32_bits(heads):
    """Pages 4 GiB apart: the weights of a step, and an eviction that moves them."""
    lens, lq, page = [170, 120], [1, 40], 64
    q, kc, vc, lens_t, table = make(lens, page, 4 * heads, heads, 32, torch.bfloat16, lq)
    pages = kc[0].shape[0]
    near = pool_like(kc, torch.Generator().manual_seed(2))
    far = torch.empty(((pages - 1) << 30) + heads * page, device=DEV).as_strided((pages, page, heads), (1 << 30, 1, page))
    far.copy_(near)
    vc2, kc2 = (tuple(x.clone() for x in c) for c in (vc, kc))
    lse = torch.randn(4 * heads, sum(lq), device=DEV) + 5
    for w in (near, far):
        mfa.kv8_key_weights(q, kc, lse, w, lens_t, table, cu_of(lq), causal=True)
    assert torch.equal(near, far)
    n = [mfa.kv8_evict(k, v, w, lens_t, table, 100, 10) for k, v, w in ((kc, vc, near), (kc2, vc2, far))]
    assert n[0].tolist() == n[1].tolist() == [100, 100] and torch.equal(near, far)
    for a, b in zip((*kc, *vc), (*kc2, *vc2)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
