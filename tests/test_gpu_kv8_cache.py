"""Writing the paged 8-bit cache: every code, scale and value is defined exactly, so
everything here is compared for equality."""
from __future__ import annotations

import math

import pytest
import torch

import mtlflashattn_amd as mfa
from kv8_util import DEV, append64, bits, byte_of, cu_of, filled_cache, i32, power, table_of

pytestmark = pytest.mark.gpu


def same(pool, want):
    for a, b in zip(bits(pool), want):
        assert torch.equal(a, b)


def check(pools, k, v, cu, old, table, **kw):
    """An append against the definition; returns the values."""
    page = pools[0][0].shape[1]
    want = [append64(c, x, cu.tolist(), old.tolist(), table.cpu(), page) for c, x in zip(pools, (k, v))]
    got = mfa.kv8_append(k, v, *pools, cu, old, table, return_values=True, **kw)
    for c, x, y, (ref, val) in zip(pools, (k, v), got, want):
        same(c, ref)
        assert y.dtype == x.dtype and y.shape == x.shape
        if x.dtype == torch.float16:
            val = val.clamp(-65504, 65504)  # (saturates; NaN stays)
        assert torch.equal(torch.nan_to_num(y.double().cpu(), nan=-1.0), torch.nan_to_num(val.to(x.dtype).double(), nan=-1.0))
    # the same rows again: the same cache
    assert mfa.kv8_append(k, v, *pools, cu, old, table) is None
    for c, (ref, _) in zip(pools, want):
        same(c, ref)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("page", [64, 192])
def test_append(page, D, dtype):
    """Empty and half-filled blocks, one row and several blocks, a sequence without rows."""
    new, old = [3, 0, 70, 1, 130, 1, 2], [0, 5, 60, 63, 100, 64, 62]
    g = torch.Generator().manual_seed(D)
    k, v = (torch.randn(sum(new), 3, D, generator=g).mul(torch.exp(2 * torch.randn(sum(new), 3, 1, generator=g))).to(DEV, dtype)
            for _ in range(2))
    pools = [filled_cache(g, 24, page, 3, D) for _ in range(2)]
    table = table_of([a + b for a, b in zip(new, old)], page, 24)
    check(pools, k, v, cu_of(new), i32(*old), table)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_borders_and_extremes(dtype):
    """Ties, both sides of the scale's choice, zeros, subnormals, the largest values, NaN and
    infinities: a block each, as the sequences of one call."""
    fi = torch.finfo(dtype)
    ties = [0.0, -0.0, 2.0 ** -10, 3 * 2.0 ** -10, 5 * 2.0 ** -10, 17 / 16, 19 / 16, 31 / 16, 33.0, 35.0, 200.0, 216.0, 432.0]
    rows = []
    for top in (448.0, 448.0 * (1 + fi.eps), 448.0 * (1 - fi.eps / 2), 256.0, 512.0 * (1 - fi.eps / 2)):
        for e in (0, -6, 3):
            r = torch.tensor((ties + [-x for x in ties])[:26] + [0.1] * 6, dtype=torch.float64).clamp(-top, top)
            r[31] = top
            rows.append(r * 2.0 ** e)
    rows += [torch.zeros(32), torch.full((32,), fi.max), torch.linspace(-1, 1, 32) * fi.max / 2, torch.full((32,), fi.tiny),
             torch.full((32,), fi.smallest_normal * fi.eps)]
    for bad in (math.nan, math.inf, -math.inf):
        r = torch.linspace(-3, 3, 32)
        r[17] = bad
        rows.append(r)
        rows.append(torch.full((32,), bad))
    x = torch.stack([r.double() for r in rows]).to(dtype).view(-1, 1, 32).to(DEV)
    n = x.shape[0]
    g = torch.Generator().manual_seed(0)
    pools = [filled_cache(g, n, 64, 1, 32) for _ in range(2)]
    table = torch.randperm(n, generator=g).to(torch.int32)[:, None].to(DEV)
    check(pools, x, x.flip(0), cu_of([1] * n), i32(*[0] * n), table)


def test_no_element_is_off_by_more_than_half_a_step():
    """A step is 2^-3 of an element's power of two, at least 2^-9 of the scale."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(200, 4, 128, generator=g).mul(torch.exp(3 * torch.randn(200, 4, 1, generator=g))).to(DEV)
    pools = [mfa.kv8_cache(8, 64, 4, 128) for _ in range(2)]
    kv = mfa.kv8_append(x, x, *pools, cu_of([200]), i32(0), table_of([200], 64, 8), return_values=True)
    a = x.double().cpu()
    for b in range(0, 200, 64):
        for h in range(4):
            rows = a[b:b + 64, h]
            scale = float(power(torch.tensor(byte_of(float(rows.abs().max())))))
            step = torch.maximum(torch.exp2(torch.floor(torch.log2(rows.abs().clamp(min=1e-300)))) / 8,
                                 torch.tensor(scale * 2.0 ** -9, dtype=torch.float64))
            assert bool(((kv[0].double().cpu()[b:b + 64, h] - rows).abs() <= step / 2).all())


def test_rows_that_raise_a_scale():
    """One row at a time into one block, each larger than all before: the held codes follow
    every time, down to subnormals and to 0, and a NaN stays one."""
    g = torch.Generator().manual_seed(1)
    pools = [mfa.kv8_cache(3, 64, 2, 64) for _ in range(2)]
    table = i32(2)[None]
    for n in range(64):
        x = torch.randn(1, 2, 64, generator=g) * 2.0 ** (n * 0.7 - 20)
        if n == 3:
            x[0, 1, 5] = math.nan
        x = x.to(DEV, torch.bfloat16)
        check(pools, x, -x, cu_of([1]), i32(n), table)
    # a fresh block takes no notice of what stood there
    x = torch.full((1, 2, 64), 2.0 ** -30, device=DEV, dtype=torch.bfloat16)
    check(pools, x, x, cu_of([1]), i32(0), table)
    assert bool((pools[0][1][2, 0] == byte_of(2.0 ** -30)).all())


def test_scales_at_both_ends():
    """The smallest byte (1) under the largest rows and the other way round."""
    big, small = 3.3e38, 2.0 ** -126
    pools = [mfa.kv8_cache(1, 64, 1, 32) for _ in range(2)]
    table = i32(0)[None]
    for n, top in enumerate((small, 0.0, big, small, big)):
        x = torch.linspace(-1, 1, 32).mul(top).view(1, 1, 32).to(DEV)
        got = check(pools, x, x, cu_of([1]), i32(n), table)
        assert bool(got[0].isfinite().all())


def test_rows_that_have_no_place():
    """Dropped: behind the table and on bad page ids; tokens of no sequence have values of 0; a
    negative length counts as 0; prefix sums outside the tensor read nothing."""
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(90, 2, 64, generator=g).to(DEV) for _ in range(2))
    pools = [filled_cache(g, 4, 64, 2, 64) for _ in range(2)]
    table = i32(0, 99, 2, -1, 3, 1).view(3, 2)
    cu, old = i32(5, 30, 50, 80), i32(50, 60, 120)
    kv = check(pools, k, v, cu, old, table)
    assert not kv[0][:5].any() and not kv[1][80:].any()
    check(pools, k, v, cu.long(), i32(-10, 60, 120).long(), table)  # (int64 too)
    before = [bits(c) for c in pools]
    kv = mfa.kv8_append(k, v, *pools, i32(200, 300, 400, 1 << 30), old, table, return_values=True)
    assert not kv[0].any() and not kv[1].any()
    mfa.kv8_append(k, v, *pools, i32(-9, -5, -5, -1), old, table)
    for c, b in zip(pools, before):
        same(c, b)


@pytest.mark.parametrize("nseq", [1, 63, 64, 65, 1000, 3000])
def test_many_sequences(nseq):
    g = torch.Generator().manual_seed(nseq)
    new = torch.randint(0, 3, (nseq,), generator=g).tolist()
    old = torch.randint(0, 70, (nseq,), generator=g).tolist()
    k, v = (torch.randn(sum(new), 1, 32, generator=g).to(DEV, torch.bfloat16) for _ in range(2))
    pools = [mfa.kv8_cache(nseq * 2, 64, 1, 32) for _ in range(2)]
    table = table_of([128] * nseq, 64, nseq * 2, nseq)
    if sum(new):
        check(pools, k, v, cu_of(new), i32(*old), table)
    mfa.kv8_append(k[:0], v[:0], *pools, cu_of([0] * nseq), i32(*old), table)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("H", [28, 30])
def test_steps_of_many_heads(H, D, dtype):
    """A block is a wavefront's from 2048 heads of sequences on: full blocks, few rows, rows that
    raise the scale of those held, tokens of no sequence, missing pages, empty sequences."""
    g = torch.Generator().manual_seed(D + H)
    new = [3, 0, 70, 1, 130, 1, 2, 200, 17, 33] + [1, 0, 2, 1, 5, 1] * 10
    old = torch.randint(0, 130, (len(new),), generator=g).tolist()
    k, v = (torch.randn(sum(new) + 9, H, D, generator=g).mul(torch.exp(2 * torch.randn(sum(new) + 9, H, 1, generator=g))).to(DEV, dtype)
            for _ in range(2))
    pools = [filled_cache(g, 240, 64, H, D) for _ in range(2)]
    table = table_of([a + b for a, b in zip(new, old)], 64, 240)
    table[2, 0], table[4, 1], table[20, 0] = -1, 1 << 30, 240
    cu = cu_of(new)
    cu = cu + 4  # (rows in front and behind)
    kv = check(pools, k, v, cu, i32(*old), table)
    assert not kv[0][:4].any() and not kv[1][-5:].any()


def test_input_and_cache_layouts():
    """Views of a packed projection, unaligned rows, expanded heads; caches with rows or pages in any order."""
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(150, 8, 64, generator=g).to(DEV, torch.bfloat16)
    k, v = qkv[:, 4:6], qkv[:, 6:8]
    table, cu, old = table_of([150], 64, 4, extra=2), cu_of([150]), i32(0)
    pools = [mfa.kv8_cache(4, 64, 2, 64) for _ in range(2)]
    check(pools, k, v, cu, old, table)
    want = [bits(c) for c in pools]
    rows_first = [tuple(t.contiguous().zero_() for t in (c[0].view(torch.uint8), c[1])) for c in pools]
    rows_first = [(c.view(torch.float8_e4m3fn), s) for c, s in rows_first]
    mfa.kv8_append(k.contiguous(), v.contiguous(), *rows_first, cu, old, table[:, :3])
    odd = torch.empty(150 * 2 * 64 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(150, 2, 64)
    odd.copy_(k)
    padded = []
    for _ in range(2):
        c = torch.zeros(4, 65, 3, 96, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)[:, :64, 1:, 32:]
        padded.append((c, torch.zeros(4, 2, 5, dtype=torch.uint8, device=DEV)[:, 1:, ::2][:, :, 1:]))
    mfa.kv8_append(odd, v, *padded, cu, old, table)
    for c, p, w in zip(rows_first, padded, want):
        same(c, w)
        same(p, w)
    one = qkv[:, 4:5].expand(150, 2, 64)
    again = [mfa.kv8_cache(4, 64, 2, 64) for _ in range(2)]
    check(again, one, one, cu, old, table)


def test_append_captured():
    k, v = (torch.randn(4, 2, 64, device=DEV) for _ in range(2))
    pools = [mfa.kv8_cache(8, 64, 2, 64) for _ in range(2)]
    table, cu = table_of([128] * 4, 64, 8), cu_of([1] * 4)
    old = i32(0, 5, 62, 100)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv = mfa.kv8_append(k, v, *pools, cu, old, table, return_values=True)
    for _ in range(5):
        k.normal_().mul_(float(torch.randn(()).exp()))
        want = [append64(c, x, cu.tolist(), old.tolist(), table.cpu(), 64) for c, x in zip(pools, (k, v))]
        graph.replay()
        torch.cuda.synchronize()
        for c, y, (ref, val) in zip(pools, kv, want):
            same(c, ref)
            assert torch.equal(y.double().cpu(), val)
        old.add_(1)


def test_offsets_past_32_bits():
    """A pool of more than 4 GiB of codes: the last pages are the ones in use."""
    page, H, D = 256, 8, 128
    pages = (1 << 32) // (page * H * D) + 8
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(600, H, D, generator=g).to(DEV, torch.bfloat16) for _ in range(2))
    small, big = ([mfa.kv8_cache(n, page, H, D) for _ in range(2)] for n in (4, pages))
    table = i32(3, 0, 2)[None]
    mfa.kv8_append(k, v, *small, cu_of([600]), i32(70), table)
    mfa.kv8_append(k, v, *big, cu_of([600]), i32(70), table + (pages - 4))
    for a, b in zip(small, big):
        assert torch.equal(a[0].view(torch.uint8), b[0][-4:].view(torch.uint8)) and torch.equal(a[1], b[1][-4:])
        assert not b[0][:4].view(torch.uint8).any()
