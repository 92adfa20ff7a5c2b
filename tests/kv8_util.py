"""The 8-bit K/V cache from its definitions, in float64 on the CPU."""
from __future__ import annotations

import math

import torch

import mtlflashattn_amd as mfa

DEV = "cuda"
F8 = torch.float8_e4m3fn
BLOCK = 64


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cu_of(lens):
    return torch.tensor([0] + list(lens), dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV)


def code_values():
    """float64 values of the 256 codes."""
    out = []
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v = math.nan if c & 127 == 127 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(-v if c & 128 else v)
    return torch.tensor(out, dtype=torch.float64)


VALUES = code_values()
_ORDER = torch.tensor(sorted(range(127), key=lambda c: VALUES[c].item()))  # magnitudes, ascending: codes 0..126


def round8(x):
    """Codes of the nearest values of float64 x (|x| <= 448, or NaN), of two equally near the even code."""
    mag, a = VALUES[_ORDER], x.abs().contiguous()
    hi = torch.searchsorted(mag, torch.nan_to_num(a)).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = mag[hi] - a, a - mag[lo]
    take_hi = (up < down) | ((up == down) & (hi % 2 == 0))
    c = torch.where(take_hi, hi, lo)
    c = torch.where(a.isnan(), 127, c)
    return c + 128 * (torch.signbit(x) & ~a.isnan())


def power(byte):
    return torch.where(byte == 0, 0.0, torch.ldexp(torch.tensor(1.0, dtype=torch.float64), byte.long() - 127))


def byte_of(amax):
    """The smallest byte from 1 on that holds a magnitude (a float)."""
    return next(b for b in range(1, 255) if amax <= 448 * 2.0 ** (b - 127))


def bits(pool):
    """(codes, scales) as uint8 copies on the CPU, codes of NaN as 127."""
    c = pool[0].contiguous().view(torch.uint8).cpu().clone()
    c[c & 127 == 127] = 127
    return c, pool[1].cpu().clone()


def rows64(pool):
    """float64 rows [pages, page, H, D] of a pool."""
    c, s = bits(pool)
    return VALUES[c.long()] * power(s).repeat_interleave(BLOCK, 1)[..., None]


def append64(pool, x, cu, old, table, page):
    """((codes, scales) of a pool after rows x [total, H, D] are written, their values)."""
    codes, scales = bits(pool)
    H = codes.shape[2]
    x = x.double().cpu()
    values = torch.zeros_like(x)
    for b in range(len(cu) - 1):
        lo, end = max(int(old[b]), 0), max(int(old[b]), 0) + cu[b + 1] - cu[b]
        t = cu[b]
        while lo < end:
            base = lo // BLOCK * BLOCK
            hi = min(end, base + BLOCK)
            rows, n = x[t:t + hi - lo], hi - lo
            finite = torch.where(rows.isfinite(), rows.abs(), 0.0).amax((0, 2))
            byte = torch.tensor([byte_of(float(m)) for m in finite])
            p = int(table[b, base // page]) if base // page < table.shape[1] else -1
            placed = 0 <= p < codes.shape[0]
            r = base % page
            if placed and lo > base:
                was = scales[p, r // BLOCK].long()
                byte = torch.maximum(byte, was)
                held = VALUES[codes[p, r:r + lo - base].long()] * (power(was) / power(byte))[:, None]
                raised = (byte > was)[None, :, None]
                codes[p, r:r + lo - base] = torch.where(raised, round8(held).to(torch.uint8), codes[p, r:r + lo - base])
            top = torch.where(byte == 247, 240.0, 448.0)[:, None]  # (256 * 2^120 would be infinite)
            c = round8((torch.where(rows.isfinite(), rows, math.nan) / power(byte)[:, None]).clamp(-top, top))
            values[t:t + n] = VALUES[c] * power(byte)[:, None]
            if placed:
                codes[p, r + lo - base:r + hi - base] = c.to(torch.uint8)
                scales[p, r // BLOCK] = byte.to(torch.uint8)
            lo, t = hi, t + n
    assert H == x.shape[1]
    return (codes, scales), values


def evict64(kc, vc, weights, lens, table, budget, recent):
    """((codes, scales) of K, of V, weights, new lengths) after an eviction."""
    page, H = kc[0].shape[1:3]
    pools = [bits(kc), bits(vc)]
    values = [rows64(kc), rows64(vc)]
    old = weights.cpu().clone()
    out = old.clone()
    table = table.tolist()
    for b, n in enumerate(int(x) for x in lens):
        if n <= budget:
            continue

        def place(j):
            p = table[b][j // page]
            return (p, j % page) if 0 <= p < kc[0].shape[0] else None

        at = [place(j) for j in range(n)]
        for h in range(H):
            head = old[:, :, h].tolist()
            w = [head[p[0]][p[1]] if p else 0.0 for p in at]
            tail = min(recent, budget)
            key = lambda j: (-math.inf if math.isnan(w[j]) else -w[j], not math.isnan(w[j]), j)  # noqa: E731
            kept = sorted(sorted(range(n - tail), key=key)[:budget - tail]) + list(range(n - tail, n))
            for first in range(0, budget, BLOCK):
                rows = range(first, min(first + BLOCK, budget))
                if all(kept[i] == i for i in rows):
                    continue
                to = place(first)
                for (codes, scales), v in zip(pools, values):
                    x = torch.stack([v[at[kept[i]]][h] if at[kept[i]] else torch.zeros(v.shape[-1], dtype=torch.float64)
                                     for i in rows])
                    byte = byte_of(float(torch.where(x.isfinite(), x.abs(), 0.0).max()))
                    if to:
                        codes[to[0], to[1]:to[1] + len(rows), h] = round8(x / power(torch.tensor(byte))).to(torch.uint8)
                        scales[to[0], to[1] // BLOCK, h] = byte
                if to:
                    for i in rows:
                        out[to[0], to[1] + i - first, h] = w[kept[i]]
    return pools, out, [min(int(n), budget) for n in lens]


def filled_cache(g, pages, page, H, D, spread=1.0, layout="heads"):
    """A pool of rows ~ N(0, 1), each block times exp(spread N(0, 1)); layout: of the memory."""
    x = torch.randn(pages, page, H, D, generator=g, dtype=torch.float64)
    gain = torch.exp(spread * torch.randn(pages, page // BLOCK, H, generator=g, dtype=torch.float64))
    x = x * gain.repeat_interleave(BLOCK, 1)[..., None]
    amax = x.abs().unflatten(1, (-1, BLOCK)).amax((2, 4))
    byte = torch.tensor([byte_of(float(m)) for m in amax.flatten()]).view(amax.shape)
    codes = round8(x / power(byte).repeat_interleave(BLOCK, 1)[..., None]).to(torch.uint8)
    scales = byte.to(torch.uint8)
    if layout == "heads":
        pool = mfa.kv8_cache(pages, page, H, D)
        pool[0].view(torch.uint8).copy_(codes)
        pool[1].copy_(scales)
        return pool
    return codes.to(DEV).view(F8), scales.to(DEV)


def table_of(lens, page, pages, seed=0, fill=1 << 20, extra=0):
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    need = [-(-n // page) for n in lens]
    t = torch.full((len(lens), max(need + [1]) + extra), fill, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            t[b, i] = ids.pop()
    return t.to(DEV)


def scores64(q, K, n, L, causal, window, softcap, slope, scale):
    """Masked scores [n, L] of one head's rows q over keys K, and the mask."""
    i = torch.arange(n)[:, None] + L - n
    j = torch.arange(L)[None]
    ok = torch.ones(n, L, dtype=torch.bool)
    if causal:
        ok &= j <= i
    if window[0] >= 0:
        ok &= j >= i - window[0]
    if window[1] >= 0:
        ok &= j <= i + window[1]
    s = q @ K.T * scale
    if softcap > 0:
        s = softcap * torch.tanh(s / softcap)
    if slope is not None:
        s = s - float(slope) * (i - j).abs()
    return s.masked_fill(~ok, -math.inf), ok


def attend64(q, kc, vc, lens, table, lq, causal=False, window=(-1, -1), softcap=0.0, slopes=None, scale=None):
    """float64 (out [rows, Hq, D], lse [Hq, rows], per-sequence key weights [Hkv, keys]) of packed q."""
    q = q.cpu().double()
    rows, Hq, D = q.shape
    page, Hkv = kc[0].shape[1:3]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out, lse = torch.zeros(rows, Hq, D, dtype=torch.float64), torch.full((Hq, rows), -math.inf, dtype=torch.float64)
    k64, v64 = rows64(kc), rows64(vc)
    weights, start = [], 0
    for b, n in enumerate(lq):
        L = int(lens[b])
        ids = table[b, :-(-L // page)].cpu().long()
        K, V = (x[ids].flatten(0, 1)[:L] for x in (k64, v64))
        w = torch.zeros(Hkv, L, dtype=torch.float64)
        for h in range(Hq):
            hk = h * Hkv // Hq
            slope = None if slopes is None else slopes[b, h] if slopes.dim() == 2 else slopes[h]
            s, ok = scores64(q[start:start + n, h], K[:, hk], n, L, causal, window, softcap, slope, scale)
            p = torch.softmax(s, -1) if L else torch.zeros(n, 0, dtype=torch.float64)
            p = torch.where(ok.any(-1, keepdim=True), p, 0.0)
            out[start:start + n, h] = torch.where(p[:, :, None] > 0, p[:, :, None] * V[:, hk], 0.0).sum(1)
            lse[h, start:start + n] = torch.logsumexp(s, -1)
            w[hk] += p.sum(0)
        weights.append(w)
        start += n
    return out, lse, weights


def make(lens, page, Hq, Hkv, D, dtype, lq, seed=0, layout="heads", extra=1, spread=0.3):
    """(q [rows, Hq, D], K and V pools, lengths, table) with pages in random order."""
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-n // page) for n in lens) + 3
    kc, vc = (filled_cache(g, pages, page, Hkv, D, spread, layout) for _ in range(2))
    q = torch.randn(sum(lq), Hq, D, generator=g).to(DEV, dtype)
    return q, kc, vc, i32(*lens), table_of(lens, page, pages, seed, extra=extra)
