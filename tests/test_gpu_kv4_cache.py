"""Writing the paged 4-bit cache and copying its pages: every code, scale and byte is
defined exactly, so everything here is compared for equality."""
from __future__ import annotations

import math

import pytest
import torch

import mtlflashattn_amd as mfa

pytestmark = pytest.mark.gpu
DEV = "cuda"
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantize(x):
    """(codes 0..15 [..., D], scale bytes [..., D / 32]) from the definition, in float64."""
    g = x.double().cpu().unflatten(-1, (-1, 32))
    amax = g.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    scale = torch.zeros_like(amax, dtype=torch.long)
    ok = torch.zeros_like(bad)
    for byte in range(254, -1, -1):  # the smallest scale that holds the group within 7
        ok = amax <= 7 * 2.0 ** (byte - 127)
        scale = torch.where(ok, byte, scale)
    v = g / torch.pow(2.0, scale.double() - 127)[..., None]
    best, code = torch.full_like(v, math.inf), torch.zeros_like(v, dtype=torch.long)
    for c in (0, 2, 4, 6, 1, 3, 5, 7):  # ties to the even code
        d = (v.abs() - LEVELS[c]).abs()
        code = torch.where(d < best, c, code)
        best = torch.minimum(d, best)
    code = code + 8 * torch.signbit(g)
    code = torch.where(bad[..., None], 0, code)
    return code.flatten(-2), torch.where(bad, 255, scale)


def values(code, scale):
    lv = torch.tensor(LEVELS + tuple(-x for x in LEVELS), dtype=torch.float64)[code].unflatten(-1, (-1, 32))
    s = torch.where(scale == 255, math.nan, torch.pow(2.0, scale.double() - 127))
    return (lv * s[..., None]).flatten(-2)


def table_of(lens, page, pages, seed=0):
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    need = [-(-n // page) for n in lens]
    t = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            t[b, i] = ids.pop()
    return t.to(DEV)


def cu_of(lens):
    return torch.tensor([0] + list(lens), dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV)


def expect(pools, k, v, cu, old, table, page):
    """The pools (CPU copies) after the rows are written, by a loop."""
    out = [tuple(t.cpu().clone() for t in c) for c in pools]
    for x, (codes, scales) in zip((k, v), out):
        c, s = quantize(x)
        packed = (c[..., 0::2] + 16 * c[..., 1::2]).to(torch.uint8)
        for b in range(len(cu) - 1):
            for t in range(cu[b], cu[b + 1]):
                at = int(old[b]) + t - cu[b]
                if at < 0 or at // page >= table.shape[1]:
                    continue
                p = int(table[b, at // page])
                if 0 <= p < codes.shape[0]:
                    codes[p, at % page], scales[p, at % page] = packed[t], s[t].to(torch.uint8)
    return out


def check_pools(pools, want):
    for got, ref in zip(pools, want):
        for a, b in zip(got, ref):
            assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("page", [64, 192])
def test_append(page, D, dtype):
    new, old = [3, 0, 70, 1, 130], [0, 5, 60, 63, 100]
    g = torch.Generator().manual_seed(D)
    k, v = (torch.randn(sum(new), 3, D, generator=g).mul(torch.exp(2 * torch.randn(3, D, generator=g))).to(DEV, dtype)
            for _ in range(2))
    table = table_of([a + b for a, b in zip(new, old)], page, 16)
    pools = [mfa.kv4_cache(16, page, 3, D), mfa.kv4_cache(16, page, 3, D)]
    for c in pools:
        c[0].fill_(0x5A)
        c[1].fill_(0x33)
    cu = cu_of(new)
    want = expect(pools, k, v, cu.tolist(), old, table.cpu(), page)
    kv = mfa.kv4_append(k, v, *pools, cu, torch.tensor(old, dtype=torch.int32, device=DEV), table, return_values=True)
    check_pools(pools, want)
    for x, got in zip((k, v), kv):
        assert got.dtype == dtype and torch.equal(got.double().cpu(), values(*quantize(x)))
    assert mfa.kv4_append(k, v, *pools, cu, torch.tensor(old, dtype=torch.int32, device=DEV), table) is None
    check_pools(pools, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_borders_and_extremes(dtype):
    """Ties, the edges of the scale's choice, zeros, subnormals, the largest values, NaN and infinities."""
    fi = torch.finfo(dtype)
    rows = []
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 0.0, -0.0]
    for e in (-14, -3, 0, 7):
        for top in (7.0, 4.0, 3.5):
            r = torch.tensor((ties + [-t for t in ties] + [0.1] * 10)[:32], dtype=torch.float64)
            r = r.clamp(-top, top)
            r[31] = top
            rows.append(r * 2.0 ** e)
    for top in (7.0, 7.0 * (1 + fi.eps), 7.0 * (1 - fi.eps / 2), 8.0 * (1 - fi.eps / 2), 4.0):
        r = torch.linspace(-1, 1, 32, dtype=torch.float64) * 0.3
        r[3] = top
        rows.append(r)
    rows += [torch.zeros(32, dtype=torch.float64), torch.full((32,), fi.max, dtype=torch.float64),
             torch.linspace(-fi.max, fi.max, 32, dtype=torch.float64), torch.full((32,), fi.tiny, dtype=torch.float64),
             torch.full((32,), fi.smallest_normal * fi.eps, dtype=torch.float64)]
    for bad in (math.nan, math.inf, -math.inf):
        r = torch.ones(32, dtype=torch.float64)
        r[17] = bad
        rows.append(r)
    x = torch.stack(rows).to(dtype).view(-1, 1, 32).to(DEV)
    n = x.shape[0]
    pools = [mfa.kv4_cache(2, 64, 1, 32), mfa.kv4_cache(2, 64, 1, 32)]
    table, old = torch.tensor([[1]], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    want = expect(pools, x, x.flip(0), [0, n], [0], table.cpu(), 64)
    kv = mfa.kv4_append(x, x.flip(0), *pools, cu_of([n]), old, table, return_values=True)
    check_pools(pools, want)
    ref = values(*quantize(x))
    if dtype == torch.float16:
        ref = ref.clamp(-65504, 65504)  # (saturates)
    assert torch.equal(torch.nan_to_num(kv[0].double().cpu(), nan=-1.0), torch.nan_to_num(ref.to(dtype).double(), nan=-1.0))


def test_half_a_step():
    """No element is off by more than half a step of its place: 1 scale at most, 1/4 scale below 2 scales."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(200, 4, 128, generator=g).to(DEV)
    pools = [mfa.kv4_cache(8, 64, 4, 128), mfa.kv4_cache(8, 64, 4, 128)]
    table = table_of([200], 64, 8)
    kv = mfa.kv4_append(x, x, *pools, cu_of([200]), torch.zeros(1, dtype=torch.int32, device=DEV), table, return_values=True)
    _, s = quantize(x)
    scale = torch.pow(2.0, s.double() - 127).repeat_interleave(32, -1)
    err, mag = (kv[0].double().cpu() - x.double().cpu()).abs() / scale, x.double().cpu().abs() / scale
    bound = torch.where(mag < 2, 0.25, torch.where(mag < 4, 0.5, 1.0))
    assert bool((err <= bound).all())


def test_rows_that_have_no_place():
    """Dropped: behind the table, bad page ids, negative positions, tokens of no sequence."""
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(90, 2, 64, generator=g).to(DEV) for _ in range(2))
    pools = [mfa.kv4_cache(4, 64, 2, 64), mfa.kv4_cache(4, 64, 2, 64)]
    for c in pools:
        c[0].fill_(0x11)
        c[1].fill_(0x7F)
    table = torch.tensor([[0, 99], [2, -1], [3, 1]], dtype=torch.int32, device=DEV)
    cu, old = [0, 30, 50, 80], [50, 60, 120]
    want = expect(pools, k, v, cu, old, table.cpu(), 64)
    kv = mfa.kv4_append(k, v, *pools, torch.tensor(cu, dtype=torch.int32, device=DEV),
                        torch.tensor(old, dtype=torch.int32, device=DEV), table, return_values=True)
    check_pools(pools, want)
    assert torch.equal(kv[1].double().cpu(), values(*quantize(v)))
    old[0] = -10
    want = expect(pools, k, v, cu, old, table.cpu(), 64)
    mfa.kv4_append(k, v, *pools, torch.tensor(cu, device=DEV), torch.tensor(old, device=DEV), table)  # (int64)
    check_pools(pools, want)


@pytest.mark.parametrize("nseq", [1, 1000, 1024, 1025, 3000])
def test_many_sequences(nseq):
    """Up to 1024 prefix sums are searched in LDS, more in memory."""
    g = torch.Generator().manual_seed(nseq)
    new = torch.randint(0, 3, (nseq,), generator=g).tolist()
    old = torch.randint(0, 20, (nseq,), generator=g).tolist()
    k, v = (torch.randn(sum(new), 1, 32, generator=g).to(DEV, torch.bfloat16) for _ in range(2))
    pools = [mfa.kv4_cache(nseq, 64, 1, 32), mfa.kv4_cache(nseq, 64, 1, 32)]
    table = table_of([64] * nseq, 64, nseq)
    want = expect(pools, k, v, cu_of(new).tolist(), old, table.cpu(), 64)
    mfa.kv4_append(k, v, *pools, cu_of(new), torch.tensor(old, dtype=torch.int32, device=DEV), table)
    check_pools(pools, want)


def test_input_and_cache_layouts():
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(50, 8, 64, generator=g).to(DEV, torch.bfloat16)
    k, v = qkv[:, 4:6], qkv[:, 6:8]
    table, cu, old = table_of([50], 64, 4), cu_of([50]), torch.zeros(1, dtype=torch.int32, device=DEV)
    pools = [mfa.kv4_cache(4, 64, 2, 64), mfa.kv4_cache(4, 64, 2, 64)]
    mfa.kv4_append(k, v, *pools, cu, old, table)
    want = [tuple(t.cpu() for t in c) for c in pools]
    rows_first = [tuple(torch.zeros_like(t, memory_format=torch.contiguous_format) for t in c) for c in pools]
    mfa.kv4_append(k.contiguous(), v.contiguous(), *rows_first, cu, old, table)
    check_pools(rows_first, want)
    odd = torch.empty(50 * 2 * 64 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(50, 2, 64)
    odd.copy_(k)
    again = [mfa.kv4_cache(4, 64, 2, 64), mfa.kv4_cache(4, 64, 2, 64)]
    mfa.kv4_append(odd, v, *again, cu, old, table)
    check_pools(again, want)


def test_append_on_a_stream_and_captured():
    k, v = (torch.randn(4, 2, 64, device=DEV) for _ in range(2))
    pools = [mfa.kv4_cache(8, 64, 2, 64), mfa.kv4_cache(8, 64, 2, 64)]
    table, cu = table_of([128] * 4, 64, 8), cu_of([1] * 4)
    old = torch.tensor([0, 5, 63, 100], dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mfa.kv4_append(k, v, *pools, cu, old, table)
    for _ in range(4):
        k.normal_()
        want = expect(pools, k, v, cu.tolist(), old.tolist(), table.cpu(), 64)
        graph.replay()
        torch.cuda.synchronize()
        check_pools(pools, want)
        old.add_(1)


def test_step_by_step_as_a_server_runs():
    """Prompt, fork, two diverging sequences: norm and rotation, cache, attention,
    page copies together, against attention over the rows the cache was given."""
    Hq, Hkv, D, page = 8, 2, 64, 64
    g = torch.Generator().manual_seed(9)
    kc, vc = mfa.kv4_cache(12, page, Hkv, D), mfa.kv4_cache(12, page, Hkv, D)
    w = torch.ones(D, device=DEV, dtype=torch.bfloat16)
    ang = torch.arange(512, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(32, device=DEV) / 32)
    cos, sin = ang.cos().float(), ang.sin().float()

    def rows(n):
        return (torch.randn(n, Hq, D, generator=g).to(DEV, torch.bfloat16), *(
            torch.randn(n, Hkv, D, generator=g).to(DEV, torch.bfloat16) for _ in range(2)))

    q, k, v = rows(100)
    q, k = mfa.qk_norm_rope(q, k, w, w, cos, sin)
    table = torch.tensor([[7, 3, 0], [7, 5, 1]], dtype=torch.int32, device=DEV)
    k1, v1 = mfa.kv4_append(k, v, kc, vc, cu_of([100]), torch.zeros(1, dtype=torch.int32, device=DEV), table[:1],
                            return_values=True)
    out = mfa.flash_attn_varlen_kv4_func(q, kc, vc, cu_of([100]), torch.tensor([100], dtype=torch.int32, device=DEV),
                                         table[:1], causal=True)
    ref = mfa.flash_attn_func(q[None], k1[None], v1[None], causal=True)[0]
    assert float((out.float() - ref.float()).abs().max()) <= 2.0 ** -7 * float(v1.abs().max())
    # the second sequence shares page 7; its own copy of the half-filled page 3 is page 5
    mfa.copy_cache_pages([*kc, *vc], torch.tensor([3], dtype=torch.int32, device=DEV),
                         torch.tensor([5], dtype=torch.int32, device=DEV))
    held = [(k1, v1), (k1, v1)]
    lens = torch.tensor([100, 100], dtype=torch.int32, device=DEV)
    for step in range(70):  # (past the end of a page)
        q, k, v = rows(2)
        q, k = mfa.qk_norm_rope(q, k, w, w, cos, sin, lens)
        kn, vn = mfa.kv4_append(k, v, kc, vc, cu_of([1, 1]), lens, table, return_values=True)
        lens = lens + 1
        held = [(torch.cat((a, kn[i:i + 1])), torch.cat((b, vn[i:i + 1]))) for i, (a, b) in enumerate(held)]
        out = mfa.flash_attn_kv4_func(q[:, None], kc, vc, lens, table, causal=True)
        if step % 23 == 0 or step == 69:
            for i, (a, b) in enumerate(held):
                ref = mfa.flash_attn_func(q[i][None, None], a[None], b[None], causal=True)[0, 0]
                assert float((out[i, 0].float() - ref.float()).abs().max()) <= 2.0 ** -7 * float(b.abs().max())


# --------------------------------------------------------------------------
# page copies


def ids(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("shape,dtype", [
    ((10, 64, 2, 64), torch.bfloat16), ((10, 256, 8, 128), torch.float16), ((10, 3, 5), torch.float32),
    ((10, 7), torch.uint8), ((10, 1), torch.uint8), ((10,), torch.float32), ((10, 33, 2, 3), torch.int16),
    ((10, 0, 4), torch.float32), ((10, 64, 3, 50), torch.float64),
])
@pytest.mark.parametrize("views", ["whole", "heads", "padded", "unaligned"])
def test_copy(shape, dtype, views):
    g = torch.Generator().manual_seed(0)
    size = torch.Size(shape).numel()
    raw = torch.randint(0, 256, (size * torch.tensor([], dtype=dtype).element_size(),), generator=g, dtype=torch.uint8)
    full = raw.view(dtype).view(shape)
    if views == "heads" and len(shape) == 4:
        pool = full.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    elif views == "padded" and len(shape) > 1:
        pool = torch.zeros(10, full[0].numel() + 3, dtype=dtype, device=DEV)[:, :full[0].numel()].unflatten(1, shape[1:])
        pool.copy_(full)
    elif views == "unaligned":
        pool = torch.zeros(size + 1, dtype=dtype, device=DEV)[1:].view(shape)
        pool.copy_(full)
    else:
        pool = full.to(DEV)
    bits = lambda t: t.contiguous().view(torch.uint8) if t.dim() > 1 or t.numel() else t  # noqa: E731
    want = pool.clone()
    for a, b in ((0, 9), (4, 2), (4, 3)):
        want[b] = want[a]
    mfa.copy_cache_pages([pool], ids(0, 4, 4, -1, 5, 10, 6), ids(9, 2, 3, 1, -1, 1, 6))
    if size:
        assert torch.equal(bits(pool), bits(want))


@pytest.mark.parametrize("pools", [1, 3, 64, 65, 130])
def test_copy_many_pools(pools):
    ts = [torch.randn(6, 64, 2, 32 + 32 * (i % 3), device=DEV).to(torch.bfloat16) for i in range(pools)]
    want = [t.clone() for t in ts]
    for t in want:
        t[1], t[2] = t[5], t[0]
    mfa.copy_cache_pages(ts, ids(5, 0), ids(1, 2))
    assert all(torch.equal(a, b) for a, b in zip(ts, want))


def test_copy_none():
    t = torch.randn(4, 64, device=DEV)
    want = t.clone()
    mfa.copy_cache_pages([t], ids(), ids())
    mfa.copy_cache_pages([], ids(1), ids(2))
    mfa.copy_cache_pages([t[:0]], ids(0), ids(1))
    assert torch.equal(t, want)


def test_copy_many_pairs_and_large_pools():
    """Offsets past 32 bits, and enough work for several rounds per segment."""
    t = torch.zeros(5000, 1 << 20, dtype=torch.uint8, device=DEV)
    src, dst = torch.arange(0, 1000), torch.arange(4000, 5000)
    t[:1000] = torch.randint(0, 256, (1000, 1), device=DEV, dtype=torch.uint8)
    t[:1000, 17] = 3
    mfa.copy_cache_pages([t], src.to(DEV, torch.int32), dst.to(DEV, torch.int32))
    assert torch.equal(t[4000:], t[:1000]) and not t[1000:4000].any()


def test_copy_checks_pairs_on_request(monkeypatch):
    t = torch.randn(6, 64, device=DEV)
    monkeypatch.setenv("MTLFLASHATTN_CHECK_PAGES", "1")
    mfa.copy_cache_pages([t], ids(0, 0, -1), ids(1, 2, 1))
    for src, dst in ((ids(0, 1), ids(2, 2)), (ids(0, 1), ids(1, 2))):
        with pytest.raises(ValueError):
            mfa.copy_cache_pages([t], src, dst)


def test_page_checks_on_request(monkeypatch):
    monkeypatch.setenv("MTLFLASHATTN_CHECK_PAGES", "1")
    pools = [mfa.kv4_cache(3, 64, 2, 64), mfa.kv4_cache(3, 64, 2, 64)]
    q = torch.randn(1, 1, 2, 64, device=DEV, dtype=torch.bfloat16)
    k = torch.randn(3, 2, 64, device=DEV)
    good, bad = ids(2, 9)[None], ids(5, 1)[None]
    mfa.flash_attn_kv4_func(q, *pools, ids(60), good)
    mfa.kv4_append(k, k, *pools, ids(0, 3), ids(61), good)
    for call in (lambda: mfa.flash_attn_kv4_func(q, *pools, ids(65), good),
                 lambda: mfa.flash_attn_kv4_func(q, *pools, ids(5), bad),
                 lambda: mfa.kv4_append(k, k, *pools, ids(0, 3), ids(62), good),
                 lambda: mfa.kv4_append(k, k, *pools, ids(0, 3), ids(126), good)):
        with pytest.raises(ValueError):
            call()


def _serving_state(seed, D, dtype):
    """Tensors of one server's step: a prompt chunk and decoding sequences."""
    g = torch.Generator().manual_seed(seed)
    Hq, Hkv, page, lens, new = 8, 2, 64, [0, 130, 700, 63], [100, 1, 1, 1]
    pages = sum(-(-(a + b) // page) for a, b in zip(lens, new)) + 2
    kc, vc = mfa.kv4_cache(pages, page, Hkv, D), mfa.kv4_cache(pages, page, Hkv, D)
    for c in (kc, vc):
        c[0].copy_(torch.randint(0, 256, c[0].shape, generator=g, dtype=torch.uint8))
        c[1].copy_(torch.randint(122, 126, c[1].shape, generator=g, dtype=torch.uint8))
    ids, table = torch.randperm(pages, generator=g).tolist(), torch.full((4, 12), -1, dtype=torch.int32)
    for b, n in enumerate(zip(lens, new)):
        for i in range(-(-sum(n) // page)):
            table[b, i] = ids.pop()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    rows = lambda H: torch.randn(cu[-1], H, D, generator=g).to(DEV, dtype)  # noqa: E731
    angle = torch.randn(900, D // 2, generator=g).to(DEV)
    pos = torch.cat([torch.arange(a, a + b) for a, b in zip(lens, new)]).to(DEV, torch.int32)
    return dict(q=rows(Hq), k=rows(Hkv), v=rows(Hkv), qw=torch.randn(D, generator=g).to(DEV, dtype), cos=angle.cos(), sin=angle.sin(),
                pos=pos, kc=kc, vc=vc, cu=ints(cu), old=ints(lens), total=ints([a + b for a, b in zip(lens, new)]), table=table.to(DEV))


def _serving_step(s):
    q, k = mfa.qk_norm_rope(s["q"], s["k"], s["qw"], None, s["cos"], s["sin"], s["pos"])
    mfa.kv4_append(k, s["v"], s["kc"], s["vc"], s["cu"], s["old"], s["table"])
    out, lse = mfa.flash_attn_varlen_kv4_func(q, s["kc"], s["vc"], s["cu"], s["total"], s["table"], causal=True,
                                              return_softmax_lse=True)
    return q, k, *(x.clone() for c in (s["kc"], s["vc"]) for x in c), out, lse


CASES = [(1, 128, torch.bfloat16), (2, 64, torch.float16), (3, 96, torch.bfloat16), (4, 32, torch.float16)]


def test_steps_on_two_streams_at_once():
    refs = [_serving_step(_serving_state(*c)) for c in CASES]
    states = [_serving_state(*c) for c in CASES]
    streams = [torch.cuda.Stream() for _ in CASES]
    torch.cuda.synchronize()
    outs = [[] for _ in CASES]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(_serving_step(states[i]))
    torch.cuda.synchronize()
    for ref, runs in zip(refs, outs):
        for got in runs:
            assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_steps_in_two_threads_at_once():
    import threading

    refs = [_serving_step(_serving_state(*c)) for c in CASES]
    states = [_serving_state(*c) for c in CASES]
    torch.cuda.synchronize()
    outs, errors = [[] for _ in CASES], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    outs[i].append(_serving_step(states[i]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # (shown by the main thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(CASES))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for ref, runs in zip(refs, outs):
        assert len(runs) == 5
        for got in runs:
            assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_two_captured_steps_replayed_in_turn():
    """Two graphs, each with its own workspace, with eager steps between the replays."""
    states = [_serving_state(*c) for c in CASES[:2]]
    graphs, outs = [], []
    for s in states:
        _serving_step(s)
    torch.cuda.synchronize()
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_serving_step(s))
        graphs.append(graph)
    for turn in range(4):
        for s in states:
            for name in ("q", "k", "v"):
                s[name].normal_()
        graphs[turn % 2].replay()
        graphs[1 - turn % 2].replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        for s, g in zip(states, got):
            ref = _serving_step(s)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(g, ref)), turn


def test_the_same_pair_of_pages_twice_and_a_page_onto_itself():
    pool = torch.randint(0, 256, (9, 5000), dtype=torch.uint8, device=DEV)
    want = pool.clone()
    want[4] = want[2]
    ids = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    mfa.copy_cache_pages([pool, pool], ids(2, 2, 7, -1), ids(4, 4, 7, 4))
    assert torch.equal(pool, want)
