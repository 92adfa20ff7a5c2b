"""The operators of the 8-bit K/V cache that this package is timed on.

A case is one pass through an operator, described by plain values.  `listed()`
holds the fixed ones, `draw(rng)` makes more of the same ranges, `prepare`
builds what a program holds before the call, `run` is one pass -- the plain
form in elementary torch operations, or with `own` the package's calls --,
`work` what the pass cannot do without and `exact` the result in 64 bits.

The kinds, and what each stands for:

  append   new K/V rows written into a paged cache held in 8 bits (kv8_append):
           one row per sequence in a decoding step, whole prompts otherwise.
  attend   attention of equal query counts over such a cache
           (flash_attn_kv8_func): one row per sequence, a few drafted tokens, or
           a long chunk of a prompt.
  mixed    a serving step that mixes decoding sequences and a prompt chunk
           (flash_attn_varlen_kv8_func).
  weights  the attention weight that each cached key received from the queries
           of a step, added to what it had (kv8_key_weights).
  evict    of every head the recent and the heaviest rows stay and move together
           (kv8_evict).

8-bit caches hold e4m3 floats (three mantissa bits, largest 448); the 64 rows of a
block (rows 64 i .. 64 i + 63 of a page) and a head share one power of two
2^(s - 127), a byte s, the smallest from 1 on with every element within 448 times
it; elements round to the nearest value, ties to the even code.  New rows in a
block that holds rows already never lower its byte; where they raise it, the codes
of the held rows are rounded again.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_DEV = "cuda"
_BLOCK = 64  # rows that share a scale
_F8 = torch.float8_e4m3fn


# --------------------------------------------------------------------------
# the cases


def listed():
    return [
        # One new row for each of 24 sequences: the smallest append.
        dict(name="append_step", kind="append", dtype="bf16", nseq=24, new_min=1, new_max=1, old_min=128, old_max=4096,
             len_seed=24, page=256, Hkv=8, D=128),
        # Eight ragged prompts into an empty cache.
        dict(name="append_prompts", kind="append", dtype="fp16", nseq=8, new_min=256, new_max=4096, old_min=0, old_max=0,
             len_seed=3, page=256, Hkv=8, D=128),
        # One user's next token over a short and odd context: latency and idle
        # compute units decide it.
        dict(name="attend_one_d128", kind="attend", dtype="bf16", nseq=1, Lq=1, len_min=3001, len_max=3001, len_seed=1,
             page=256, Hq=32, Hkv=8, D=128, causal=True, left=-1, softcap=0.0),
        # A serving batch of 64 ragged contexts: the stream of the cache.
        dict(name="attend_batch_d128", kind="attend", dtype="bf16", nseq=64, Lq=1, len_min=512, len_max=16384, len_seed=64,
             page=256, Hq=32, Hkv=8, D=128, causal=True, left=-1, softcap=0.0),
        # Five drafted tokens per sequence, head dim 64, sliding window and
        # soft-cap, small pages.
        dict(name="attend_draft_d64_fp16", kind="attend", dtype="fp16", nseq=6, Lq=5, len_min=700, len_max=5000, len_seed=6,
             page=64, Hq=16, Hkv=16, D=64, causal=True, left=1024, softcap=30.0),
        # A chunk of a long prompt: compute decides it.  The largest case.
        dict(name="attend_chunk_d128", kind="attend", dtype="bf16", nseq=1, Lq=1024, len_min=16384, len_max=16384,
             len_seed=1, page=256, Hq=32, Hkv=8, D=128, causal=True, left=-1, softcap=0.0),
        # 31 decoding sequences beside a 512-token prompt chunk.
        dict(name="mixed_step", kind="mixed", dtype="bf16", nseq=31, Lq=512, len_min=256, len_max=4096, len_seed=31,
             page=256, Hq=32, Hkv=8, D=128, causal=True, left=-1, softcap=0.0),
        # The weights of one decoding step of a ragged batch.
        dict(name="weights_step", kind="weights", dtype="bf16", nseq=32, Lq=1, len_min=512, len_max=8192, len_seed=32,
             page=256, Hq=32, Hkv=8, D=128, causal=True, left=-1, softcap=0.0),
        # What the last 64 rows of two long prompts look at.
        dict(name="weights_observe", kind="weights", dtype="bf16", nseq=2, Lq=64, len_min=12000, len_max=16384, len_seed=2,
             page=256, Hq=32, Hkv=8, D=128, causal=True, left=-1, softcap=0.0),
        # All rows of a prompt chunk, head dim 64, plain heads.
        dict(name="weights_chunk_fp16", kind="weights", dtype="fp16", nseq=1, Lq=512, len_min=4096, len_max=4096, len_seed=1,
             page=128, Hq=16, Hkv=16, D=64, causal=True, left=-1, softcap=0.0),
        # One sequence has grown 128 rows past its budget.
        dict(name="evict_one", kind="evict", dtype="bf16", nseq=1, len_min=2176, len_max=2176, budget=2048, recent=256,
             len_seed=1, page=256, Hkv=8, D=128),
        # A batch of ragged prompts comes down to one odd budget.
        dict(name="evict_batch", kind="evict", dtype="bf16", nseq=16, len_min=4096, len_max=16384, budget=4001, recent=512,
             len_seed=16, page=256, Hkv=8, D=128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    """Rough seconds of a pass, to bound what is drawn."""
    w = work(case)
    return w["flops"] / 4e14 + w["bytes"] / 3e12


def draw(rng):
    bound = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= bound and _size(case) <= 1 << 30:
            return case


def _size(case):
    """Elements of the cache that a pass holds, to bound what is drawn."""
    if case["kind"] == "append":
        return case["nseq"] * (case["old_max"] + case["new_max"]) * case["Hkv"] * case["D"]
    return case["nseq"] * case["len_max"] * case["Hkv"] * case["D"]


def _draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "mixed", "weights", "weights", "evict", "evict"])
    half = rng.choice(["bf16", "bf16", "fp16"])
    hq, hkv = rng.choice([(32, 8), (16, 16), (64, 8), (32, 4), (12, 12), (16, 8)])
    seed = rng.randrange(1 << 20)
    d = rng.choice([64, 128, 128, 96, 32])
    page = rng.choice([64, 128, 256, 256])
    base = dict(kind=kind, dtype=half, len_seed=seed, page=page, Hkv=hkv, D=d)
    if kind == "append":
        top = rng.randrange(1, 6) if rng.random() < 0.5 else _log_int(rng, 16, 8192)
        return dict(base, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), nseq=_log_int(rng, 1, 64), new_min=1,
                    new_max=top, old_min=0, old_max=_log_int(rng, 1, 4096))
    if kind == "evict":
        top = _log_int(rng, 100, 32768)
        budget = rng.randrange(1, top)
        return dict(base, nseq=_log_int(rng, 1, 32), len_min=max(1, top // 4), len_max=top, budget=budget,
                    recent=rng.randrange(0, budget // 2 + 1))
    base.update(Hq=hq, causal=rng.random() < 0.8, left=_log_int(rng, 32, 4096) if rng.random() < 0.25 else -1,
                softcap=rng.choice([0.0, 0.0, 0.0, 30.0]))
    if kind == "mixed":
        chunk = _log_int(rng, 32, 1024)
        top = _log_int(rng, max(chunk, 256), 8192)
        return dict(base, nseq=_log_int(rng, 1, 48), Lq=chunk, len_min=max(1, top // 16), len_max=top)
    form = rng.choice(["one", "one", "draft", "chunk"])
    if form == "one":
        nseq, lq, top = _log_int(rng, 1, 64), 1, _log_int(rng, 200, 16384)
    elif form == "draft":
        nseq, lq, top = _log_int(rng, 1, 32), rng.randrange(2, 17), _log_int(rng, 200, 16384)
    else:
        nseq, lq = _log_int(rng, 1, 6), _log_int(rng, 17, 2048)
        top = _log_int(rng, max(lq, 300), 16384)
    return dict(base, nseq=nseq, Lq=lq, len_min=min(top, max(lq, top // 16)), len_max=top)


# --------------------------------------------------------------------------
# inputs


def _lens(case, lo="len_min", hi="len_max", salt=0):
    """Ragged lengths, uniform between the bounds, the same for every input seed."""
    g = torch.Generator().manual_seed(case["len_seed"] + salt)
    return torch.randint(case[lo], case[hi] + 1, (case["nseq"],), generator=g).tolist()


def _cu(lens):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(device=_DEV, dtype=torch.int32)


def _randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device=_DEV).to(dtype)


def _table(lens, page, seed):
    """(block table with the pages of every sequence in random order, pages of the pool)."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 4  # (a pool holds pages that no sequence uses)
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.zeros(len(lens), max(1, max(need)), dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    return table.to(_DEV), pages


def _filled_cache(g, gain, pages, page, heads, d):
    """An 8-bit pool (codes, scales) of rows ~ N(0, gain^2), each head's rows of a page side by side."""
    codes = torch.empty(pages, heads, page, d, dtype=_F8, device=_DEV)
    scales = torch.empty(pages, heads, page // _BLOCK, dtype=torch.uint8, device=_DEV)
    step = max(1, (1 << 26) // (page * heads * d))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = torch.randn(n, heads, page // _BLOCK, _BLOCK, d, generator=g, device=_DEV) * gain[:, None, None]
        s = _byte_of(x.abs().amax((-1, -2)))
        codes[p:p + n] = (x * _inverse(s)[..., None, None]).to(_F8).flatten(2, 3)
        scales[p:p + n] = s.to(torch.uint8)
    return codes.transpose(1, 2), scales.transpose(1, 2)


def _row_lens(case):
    """(query rows, cached keys) of each sequence; a mixed step's chunk comes last."""
    lens = _lens(case)
    if case["kind"] == "mixed":
        return [1] * len(lens) + [case["Lq"]], lens + [max(case["Lq"], case["len_max"])]
    return [case["Lq"]] * len(lens), lens


def prepare(case, seed):
    """Inputs from the seed alone, on the GPU."""
    g = torch.Generator(device=_DEV).manual_seed(seed)
    dt, kind, page, Hkv, D = _DTYPES[case["dtype"]], case["kind"], case["page"], case["Hkv"], case["D"]
    s = dict(case=case)
    # a few larger channels, for the cached and the new rows alike
    gains = [torch.exp(0.5 * torch.randn(Hkv, D, generator=g, device=_DEV)) for _ in range(2)]
    if kind == "append":
        new, old = _lens(case, "new_min", "new_max"), _lens(case, "old_min", "old_max", 1)
        held = [a + b for a, b in zip(new, old)]
        s["k"], s["v"] = ((torch.randn(sum(new), Hkv, D, generator=g, device=_DEV) * x).to(dt) for x in gains)
        s["cu"], s["old"] = _cu(new), torch.tensor(old, dtype=torch.int32, device=_DEV)
        s["total"] = sum(new)
        s["touched"] = sum((b - 1) // _BLOCK - a // _BLOCK + 1 for a, b in zip(old, held))
    else:
        lq, held = ([], _lens(case)) if kind == "evict" else _row_lens(case)
        s["lens"] = torch.tensor(held, dtype=torch.int32, device=_DEV)
        s["keys"], s["max_k"] = sum(held), max(held)
        s["over"] = torch.tensor([b for b, n in enumerate(held) if n > case.get("budget", n)], dtype=torch.int64, device=_DEV)
    s["table"], pages = _table(held, page, seed)
    s["kc"], s["vc"] = (_filled_cache(g, x, pages, page, Hkv, D) for x in gains)
    if kind in ("attend", "weights"):
        s["q"] = _randn(g, len(lq), case["Lq"], case["Hq"], D, dtype=dt)
    elif kind == "mixed":
        s["q"], s["cu_q"] = _randn(g, sum(lq), case["Hq"], D, dtype=dt), _cu(lq)
    if kind in ("weights", "evict"):
        # what earlier steps left: a few heavy keys, some that nobody looked at
        w = torch.exp(2 * torch.randn(pages, Hkv, page, generator=g, device=_DEV))
        w = w * (torch.rand(pages, Hkv, page, generator=g, device=_DEV) > 0.05)
        s["weights"] = w.transpose(1, 2)
    if kind == "weights":  # the attention call of this step has returned the log-sum-exps
        s["lse"] = _scores(s["q"], s["kc"], s["table"], s["lens"], case).logsumexp(-1).flatten(1, 2)
    return s


# --------------------------------------------------------------------------
# one pass


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import mtlflashattn_amd as mfa

    case = s["case"]
    kind = case["kind"]
    if kind == "append":
        k, v = mfa.kv8_append(s["k"], s["v"], s["kc"], s["vc"], s["cu"], s["old"], s["table"], return_values=True)
        return k, v, *s["kc"], *s["vc"]
    if kind == "evict":
        lens = mfa.kv8_evict(s["kc"], s["vc"], s["weights"], s["lens"], s["table"], case["budget"], case["recent"],
                             max_seqlen_k=s["max_k"])
        return lens, s["weights"], *s["kc"], *s["vc"]
    opts = dict(causal=case["causal"], window_size=(case["left"], -1), softcap=case["softcap"], max_seqlen_k=s["max_k"])
    with torch.no_grad():
        if kind == "attend":
            return mfa.flash_attn_kv8_func(s["q"], s["kc"], s["vc"], s["lens"], s["table"], **opts)
        if kind == "mixed":
            return mfa.flash_attn_varlen_kv8_func(s["q"], s["kc"], s["vc"], s["cu_q"], s["lens"], s["table"], **opts)
        mfa.kv8_key_weights(s["q"], s["kc"], s["lse"], s["weights"], s["lens"], s["table"], **opts)
        return s["weights"]


# The plain forms: elementary operations in 32 bits.


def _byte_of(amax):
    """The smallest scale bytes (int32, from 1 on) that hold magnitudes up to amax."""
    m, e = torch.frexp(amax)
    return torch.where(amax == 0, 1, e + 118 + (m > 0.875)).clamp(min=1).to(torch.int32)


def _power(byte):
    return (byte.int() << 23).view(torch.float32)


def _inverse(byte):
    return ((254 - byte.int()) << 23).view(torch.float32)


def _gather(t, table):
    """Pages of a pool, [B, max_pages * rows, ...] (8-bit floats are moved as bytes)."""
    if t.dtype == _F8:
        return t.view(torch.uint8)[table.long()].view(_F8).flatten(1, 2)
    return t[table.long()].flatten(1, 2)


def _dequantize(codes, scales, table):
    """fp32 rows [B, keys, Hkv, D] of the sequences."""
    s = _power(_gather(scales, table)).repeat_interleave(_BLOCK, 1)
    return _gather(codes, table).float() * s[..., None]


def _masked(s, lens, lq, case):
    """Scores [B, Hkv, heads, Lq, keys], what a row does not see at -inf."""
    j = torch.arange(s.shape[-1], device=s.device)
    center = torch.arange(lq, device=s.device) + (lens.long()[:, None] - lq)  # [B, Lq]
    ok = (j < lens.long()[:, None])[:, None, :]
    if case["causal"]:
        ok = ok & (j <= center[..., None])
    if case["left"] >= 0:
        ok = ok & (j >= center[..., None] - case["left"])
    return s.masked_fill(~ok[:, None, None], -math.inf)


def _scores(q, kc, table, lens, case):
    """The masked scores of q [B, Lq, Hq, D], [B, Hkv, heads, Lq, keys]."""
    k = _dequantize(*kc, table).permute(0, 2, 3, 1).contiguous()  # [B, Hkv, D, keys]
    lq = q.shape[1]
    qf = q.float().unflatten(2, (case["Hkv"], -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, Hkv, heads * Lq, D]
    s = torch.matmul(qf, k) / math.sqrt(q.shape[-1])
    if case["softcap"] > 0:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    return _masked(s.unflatten(2, (-1, lq)), lens, lq, case)


def _attend_plain(q, kc, vc, table, lens, case):
    """q [B, Lq, Hq, D] over the cached keys of each sequence."""
    lq = q.shape[1]
    s = _scores(q, kc, table, lens, case)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    v = _dequantize(*vc, table).transpose(1, 2).contiguous()  # [B, Hkv, keys, D]
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (-1, lq)) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3).to(q.dtype)


def _put(pool, page, row, rows):
    """rows into pool[page, row] (8-bit floats are moved as bytes)."""
    if pool.dtype == _F8:
        pool, rows = pool.view(torch.uint8), rows.view(torch.uint8)
    pool[page, row] = rows


def _append_plain(x, pool, s):
    """New rows into one pool; returns their values."""
    codes, scales = pool
    case = s["case"]
    n, page = case["nseq"], case["page"]
    old, new = s["old"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n, device=_DEV), new, output_size=s["total"])
    at = old[seq] + torch.arange(s["total"], device=_DEV) - s["cu"].long()[seq]
    # the blocks that the rows fall into, sequence after sequence
    first, count = old // _BLOCK, (old + new - 1) // _BLOCK - old // _BLOCK + 1
    start = count.cumsum(0) - count
    block = start[seq] + at // _BLOCK - first[seq]
    xf = x.float()
    amax = torch.zeros(s["touched"], case["Hkv"], device=_DEV).scatter_reduce_(
        0, block[:, None].expand(-1, case["Hkv"]), xf.abs().amax(-1), "amax")
    byte = _byte_of(amax)
    # rows that the first blocks hold already: the byte stays or rises, their codes follow
    held = old % _BLOCK
    page0, row0 = s["table"].long()[torch.arange(n, device=_DEV), old // page], old % page // _BLOCK
    before = scales[page0, row0].int()
    byte[start] = torch.where(held[:, None] > 0, torch.maximum(byte[start], before), byte[start])
    rows = (row0 * _BLOCK)[:, None] + torch.arange(_BLOCK, device=_DEV)
    c = codes.view(torch.uint8)[page0[:, None], rows].view(_F8)  # [B, 64, Hkv, D]
    moved = (c.float() * (_power(before) * _inverse(byte[start]))[:, None, :, None]).to(_F8)
    keep = (torch.arange(_BLOCK, device=_DEV) < held[:, None])[..., None, None]
    _put(codes, page0[:, None], rows, torch.where(keep, moved.view(torch.uint8), c.view(torch.uint8)).view(_F8))
    page_of = s["table"][seq, at // page].long()
    scales[page_of, at % page // _BLOCK] = byte[block].to(torch.uint8)
    fresh = (xf * _inverse(byte[block])[..., None]).to(_F8)
    _put(codes, page_of, at % page, fresh)
    return (fresh.float() * _power(byte[block])[..., None]).to(x.dtype)


def _evict_plain(s):
    case = s["case"]
    page, budget, H, n = case["page"], case["budget"], case["Hkv"], s["over"].numel()
    lens = torch.minimum(s["lens"], torch.full_like(s["lens"], budget))
    if n == 0:
        return lens
    held, table = s["lens"][s["over"]].long()[:, None], s["table"][s["over"]].long()  # the sequences past their budget
    j = torch.arange(table.shape[1] * page, device=_DEV)
    w = _gather(s["weights"], table).transpose(1, 2)  # [n, H, keys]
    w = w.masked_fill((j >= held - case["recent"])[:, None], math.inf).masked_fill((j >= held)[:, None], -math.inf)
    kept = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :budget].sort(dim=-1).values
    # blocks whose rows all stay where they are do not change
    to = torch.arange(budget, device=_DEV)
    blocks = -(-budget // _BLOCK)
    pad = blocks * _BLOCK - budget
    change = ~torch.nn.functional.pad(kept == to, (0, pad), value=True).unflatten(-1, (blocks, _BLOCK)).all(-1)
    rows = change.repeat_interleave(_BLOCK, -1)[..., :budget]
    b, h = torch.arange(n, device=_DEV)[:, None, None], torch.arange(H, device=_DEV)[:, None]
    src, dst = (table[b, kept // page], kept % page, h), (table[b, to // page], to % page, h)
    s["weights"][dst] = torch.where(rows, s["weights"][src], s["weights"][dst])
    first = torch.arange(blocks, device=_DEV) * _BLOCK
    place = (table[b, first // page], first % page // _BLOCK, h)
    for codes, scales in (s["kc"], s["vc"]):
        c = codes.view(torch.uint8)
        x = c[src].view(_F8).float() * _power(scales[src[0], src[1] // _BLOCK, h])[..., None]
        x = torch.nn.functional.pad(x, (0, 0, 0, pad)).unflatten(2, (blocks, _BLOCK))
        byte = _byte_of(x.abs().amax((-1, -2)))
        fresh = (x * _inverse(byte)[..., None, None]).to(_F8).view(torch.uint8).flatten(2, 3)[:, :, :budget]
        c[dst] = torch.where(rows[..., None], fresh, c[dst])
        scales[place] = torch.where(change, byte.to(torch.uint8), scales[place])
    return lens


@torch.no_grad()
def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "append":
        return _append_plain(s["k"], s["kc"], s), _append_plain(s["v"], s["vc"], s), *s["kc"], *s["vc"]
    if kind == "evict":
        return _evict_plain(s), s["weights"], *s["kc"], *s["vc"]
    if kind == "attend":
        return _attend_plain(s["q"], s["kc"], s["vc"], s["table"], s["lens"], case)
    if kind == "mixed":
        n = case["nseq"]
        one = _attend_plain(s["q"][:n, None], s["kc"], s["vc"], s["table"][:n], s["lens"][:n], case)
        chunk = _attend_plain(s["q"][None, n:], s["kc"], s["vc"], s["table"][n:], s["lens"][n:], case)
        return torch.cat((one[:, 0], chunk[0]))
    lse = s["lse"].unflatten(1, (case["Hkv"], -1))[..., None]
    p = torch.exp(_scores(s["q"], s["kc"], s["table"], s["lens"], case) - torch.where(lse == -math.inf, 0.0, lse))
    p = p.sum((2, 3)).transpose(1, 2)  # [B, keys, Hkv]
    seq = torch.repeat_interleave(torch.arange(case["nseq"], device=_DEV), s["lens"].long(), output_size=s["keys"])
    at = torch.arange(s["keys"], device=_DEV) - (s["lens"].long().cumsum(0) - s["lens"].long())[seq]
    place = (s["table"][seq, at // case["page"]].long(), at % case["page"])
    # the rows of the queries themselves had no weight before
    before = torch.where((at < s["lens"].long()[seq] - case["Lq"])[:, None], s["weights"][place], 0.0)
    s["weights"][place] = before + p[seq, at]
    return s["weights"]


# --------------------------------------------------------------------------
# what a pass cannot do without


def _pairs(lq, lk, causal, left):
    """Valid (query, key) pairs of one head (bottom-right aligned masks)."""
    i = torch.arange(lq, dtype=torch.int64) + lk - lq
    lo = (i - left).clamp(min=0) if left >= 0 else torch.zeros_like(i)
    hi = torch.minimum(i, torch.tensor(lk - 1)) if causal else torch.full_like(i, lk - 1)
    return int((hi - lo + 1).clamp(min=0).sum())


def _read(lq, lk, left):
    """Keys that some row of the sequence sees."""
    return lk if left < 0 else min(lk, lq + left)


def work(case):
    """Each input read once, each output written once."""
    kind, D, Hkv = case["kind"], case["D"], case["Hkv"]
    es = 4 if case["dtype"] == "fp32" else 2
    if kind == "append":
        # the rows in, their codes and values out, a scale per block
        n = sum(_lens(case, "new_min", "new_max")) * Hkv * 2
        return {"bytes": n * (2 * D * es + D) + n / _BLOCK, "flops": 3 * n * D}
    if kind == "evict":
        # the weights of long sequences in, the kept rows and weights in and out
        over = [n for n in _lens(case) if n > case["budget"]]
        rows = Hkv * case["budget"] * len(over)
        return {"bytes": 4 * Hkv * sum(over) + rows * (4 * D + 4) + 8 * case["nseq"], "flops": 0}
    lq, lk = _row_lens(case)
    pairs = sum(_pairs(a, b, case["causal"], case["left"]) for a, b in zip(lq, lk))
    keys = sum(_read(a, b, case["left"]) for a, b in zip(lq, lk))
    if kind == "weights":
        return {"bytes": keys * Hkv * (D + 8 + 1 / _BLOCK) + sum(lq) * case["Hq"] * (D * es + 4),
                "flops": 2 * D * case["Hq"] * pairs}
    return {"bytes": 2 * keys * Hkv * (D + 1 / _BLOCK) + 2 * sum(lq) * case["Hq"] * D * es,
            "flops": 4 * D * case["Hq"] * pairs}


# --------------------------------------------------------------------------
# the result in 64 bits, from the definitions


def _pow2(n):
    """2^n of whole n, exactly (a power function may be a last bit off, which breaks ties)."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _round8(x):
    """The nearest e4m3 values of float64 x with |x| <= 448, of two equally near the even one."""
    _, e = torch.frexp(x.abs())
    step = _pow2((e - 4).clamp(min=-9))
    return torch.round(x / step) * step


def _scale8(amax):
    """The smallest bytes from 1 on with amax <= 448 * 2^(byte - 127), by search."""
    byte = torch.ones_like(amax, dtype=torch.int64)
    for bit in (128, 64, 32, 16, 8, 4, 2, 1):
        short = amax > 448 * _pow2(byte + bit - 1 - 127)
        byte = torch.where(short, byte + bit, byte)
    return byte


def _rows64(codes, scales):
    """float64 rows of [page rows, D] codes and their [page rows / 64] scales, one head."""
    return codes.double() * _pow2(scales.long() - 127).repeat_interleave(_BLOCK)[:, None]


def _sequence64(pool, ids, h):
    """float64 rows of one head of a sequence's pages."""
    codes, scales = pool
    return _rows64(codes.view(torch.uint8)[ids][:, :, h].view(_F8).flatten(0, 1), scales[ids][:, :, h].flatten())


def _probabilities64(q, k, case, lse=None):
    """softmax of one head's rows q [Lq, D] over k [Lk, D], or exp(score - lse)."""
    lq, lk = q.shape[0], k.shape[0]
    s = (q @ k.t()) / math.sqrt(q.shape[1])
    if case["softcap"] > 0:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    d = torch.arange(lk, device=q.device)[None, :] - (torch.arange(lq, device=q.device) + lk - lq)[:, None]
    hidden = torch.zeros_like(d, dtype=torch.bool)
    if case["causal"]:
        hidden |= d > 0
    if case["left"] >= 0:
        hidden |= d < -case["left"]
    s = s.masked_fill(hidden, -math.inf)
    p = torch.softmax(s, -1) if lse is None else torch.exp(s - lse[:, None])
    return p.masked_fill(hidden.all(-1, keepdim=True), 0.0)


def _append64(s):
    case = s["case"]
    page, cu, old = case["page"], s["cu"].tolist(), s["old"].tolist()
    outs, pools = [], []
    for x, (codes, _) in (("k", s["kc"]), ("v", s["vc"])):
        scales = s[x + "c"][1].clone()
        held = codes.double()
        values = torch.empty(s[x].shape, dtype=torch.float64, device=_DEV)
        for b in range(case["nseq"]):
            lo, end = old[b], old[b] + cu[b + 1] - cu[b]
            while lo < end:  # block by block
                base = lo // _BLOCK * _BLOCK
                hi = min(end, base + _BLOCK)
                rows = s[x][cu[b] + lo - old[b]:cu[b] + hi - old[b]].double()
                p, r = int(s["table"][b, base // page]), base % page
                byte = _scale8(rows.abs().amax((0, 2)))
                if lo > base:
                    was = scales[p, r // _BLOCK].long()
                    byte = torch.maximum(byte, was)
                    part = held[p, r:r + lo - base]
                    part.copy_(_round8(part * _pow2(was - byte)[:, None]))
                c = _round8(rows * _pow2(127 - byte)[:, None])
                held[p, r + lo - base:r + hi - base] = c
                scales[p, r // _BLOCK] = byte.to(torch.uint8)
                values[cu[b] + lo - old[b]:cu[b] + hi - old[b]] = c * _pow2(byte - 127)[:, None]
                lo = hi
        outs.append(values)
        pools += [held, None]
    return (*outs, *pools)


def _evict64(s):
    case = s["case"]
    page, budget, recent = case["page"], case["budget"], case["recent"]
    held = [s["kc"][0].double(), s["vc"][0].double()]
    weights = s["weights"].double()
    for b, n in enumerate(s["lens"].tolist()):
        if n <= budget:
            continue
        ids = s["table"][b, :-(-n // page)].long()
        for h in range(case["Hkv"]):
            w = s["weights"][ids][:, :, h].flatten()[:n]
            tail = min(recent, budget)
            order = torch.argsort(-w[:n - tail].double(), stable=True)[:budget - tail]
            kept = torch.cat((order.sort().values, torch.arange(n - tail, n, device=_DEV)))
            to = torch.arange(budget, device=_DEV)
            moved = (kept != to).nonzero().flatten()
            if moved.numel() == 0:
                continue
            start = int(moved[0]) // _BLOCK * _BLOCK  # (rows only move down: all blocks behind the first change)
            place = (ids[to[start:] // page], to[start:] % page, h)
            weights[place] = w[kept[start:]].double()
            for pool, out in ((s["kc"], held[0]), (s["vc"], held[1])):
                x = _sequence64(pool, ids, h)[kept[start:]]
                x = torch.nn.functional.pad(x, (0, 0, 0, -x.shape[0] % _BLOCK)).unflatten(0, (-1, _BLOCK))
                byte = _scale8(x.abs().amax((1, 2)))
                out[place] = _round8(x * _pow2(127 - byte)[:, None, None]).flatten(0, 1)[:budget - start]
    return None, weights, held[0], None, held[1], None


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "append":
        return _append64(s)
    if kind == "evict":
        return _evict64(s)
    lq, lk = _row_lens(case)
    r = case["Hq"] // case["Hkv"]
    rows = s["q"] if kind == "mixed" else s["q"].flatten(0, 1)
    out = torch.empty(rows.shape, dtype=torch.float64, device=rows.device)
    weights = s["weights"].double() if kind == "weights" else None
    start = 0
    for b, (n, keys) in enumerate(zip(lq, lk)):
        ids = s["table"][b, :-(-keys // case["page"])].long()
        q = rows[start:start + n].double()
        for h in range(case["Hkv"]):
            k = _sequence64(s["kc"], ids, h)[:keys]
            heads = range(h * r, h * r + r)
            if kind == "weights":
                w = weights[ids][:, :, h].flatten()[:keys]
                w[keys - n:] = 0
                for i in heads:
                    w += _probabilities64(q[:, i].contiguous(), k, case, s["lse"][b, i].double()).sum(0)
                at = torch.arange(keys, device=w.device)
                weights[ids[at // case["page"]], at % case["page"], h] = w
            else:
                v = _sequence64(s["vc"], ids, h)[:keys]
                for i in heads:
                    out[start:start + n, i] = _probabilities64(q[:, i].contiguous(), k, case) @ v
        start += n
    return weights if kind == "weights" else out.view(s["q"].shape)
