"""The operators around the attention call that this package is timed on.

A case is one pass through an operator, described by plain values.  `listed()`
holds the fixed ones, `draw(rng)` makes more of the same ranges, `prepare`
builds what a program holds before the call, `run` is one pass -- the plain
form in elementary torch operations, or with `own` the package's calls --,
`work` what the pass cannot do without and `exact` the result in 64 bits.

The kinds, and what each stands for:

  qknr        qk_norm_rope, forward: the RMS norm of every query and key head
              and the rotation of its position in one pass, on the views that
              a packed projection leaves.
  qknr_train  the same, forward and backward: both outputs and the gradients of
              the queries, the keys and the two norm weights.
  kv4_append  new K/V rows written into a paged cache held in 4 bits
              (kv4_append): one row per sequence in a decoding step, whole
              prompts otherwise.
  kv4_attend  attention of equal query counts over such a cache
              (flash_attn_kv4_func): one row per sequence, a few drafted
              tokens, or a long chunk of a prompt.
  kv4_mixed   a serving step that mixes decoding sequences and a prompt chunk
              (flash_attn_varlen_kv4_func).
  copy        pages copied inside the pools of a cache (copy_cache_pages):
              forked sequences, compaction.

4-bit caches hold, per 32 consecutive elements of a head, one power-of-two scale
2^(s - 127) (a byte s) and 32 four-bit floats (sign, two exponent bits, one
mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), element 2i in the low half of byte i.
The scale is the smallest that leaves every element within 7 of it, so no element
is off by more than half a step; elements round to the nearest value, ties to the
even code.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_DEV = "cuda"


# --------------------------------------------------------------------------
# the cases


def listed():
    return [
        # The next token of 24 users: the smallest norm-and-rotate call.
        dict(name="qknr_step_bf16", kind="qknr", dtype="bf16", B=0, L=24, Hq=32, Hkv=8, D=128, rotary=128,
             interleaved=False, top=8192),
        # Training on long rows, plain heads, head dim 128.
        dict(name="qknr_train_bf16", kind="qknr_train", dtype="bf16", B=1, L=8192, Hq=16, Hkv=16, D=128, rotary=128,
             interleaved=False, top=8192),
        # Training on a ragged packed batch, head dim 64, half of each head
        # rotated in adjacent pairs.
        dict(name="qknr_train_part_fp16", kind="qknr_train", dtype="fp16", B=0, L=11037, Hq=12, Hkv=12, D=64, rotary=32,
             interleaved=True, top=2048),
        # One new row for each of 24 sequences.
        dict(name="kv4_append_step", kind="kv4_append", dtype="bf16", nseq=24, new_min=1, new_max=1, old_min=128,
             old_max=4096, len_seed=24, page=256, Hkv=8, D=128),
        # Eight ragged prompts into an empty cache.
        dict(name="kv4_append_prompts", kind="kv4_append", dtype="fp16", nseq=8, new_min=256, new_max=4096, old_min=0,
             old_max=0, len_seed=3, page=256, Hkv=8, D=128),
        # One user's next token over a short and odd context: latency and idle
        # compute units decide it.
        dict(name="kv4_one_d128", kind="kv4_attend", dtype="bf16", nseq=1, Lq=1, len_min=3001, len_max=3001, len_seed=1,
             page=256, Hq=32, Hkv=8, D=128, causal=True, left=-1, softcap=0.0),
        # A serving batch of 64 ragged contexts: the stream of the cache.
        dict(name="kv4_batch_d128", kind="kv4_attend", dtype="bf16", nseq=64, Lq=1, len_min=512, len_max=16384,
             len_seed=64, page=256, Hq=32, Hkv=8, D=128, causal=True, left=-1, softcap=0.0),
        # Five drafted tokens per sequence, head dim 64, sliding window and
        # soft-cap, small pages.
        dict(name="kv4_draft_d64_fp16", kind="kv4_attend", dtype="fp16", nseq=6, Lq=5, len_min=700, len_max=5000,
             len_seed=6, page=64, Hq=16, Hkv=16, D=64, causal=True, left=1024, softcap=30.0),
        # A chunk of a long prompt: compute decides it.  The largest case.
        dict(name="kv4_chunk_d128", kind="kv4_attend", dtype="bf16", nseq=1, Lq=1024, len_min=16384, len_max=16384,
             len_seed=1, page=256, Hq=32, Hkv=8, D=128, causal=True, left=-1, softcap=0.0),
        # 31 decoding sequences beside a 512-token prompt chunk.
        dict(name="kv4_mixed_step", kind="kv4_mixed", dtype="bf16", nseq=31, Lq=512, len_min=256, len_max=4096,
             len_seed=31, page=256, Hq=32, Hkv=8, D=128, causal=True, left=-1, softcap=0.0),
        # Two forked sequences: the last, half-filled page of each is copied in
        # the K and the V pool.
        dict(name="copy_fork", kind="copy", dtype="bf16", pairs=2, pages=64, pools=2, page=256, Hkv=8, D=128),
        # Compaction: 300 pages move down, in K and V pools of 512 KB pages.
        dict(name="copy_compact", kind="copy", dtype="fp16", pairs=300, pages=1024, pools=2, page=256, Hkv=8, D=128),
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
    """Elements of the cache or the pools that a pass holds, to bound what is drawn."""
    if case["kind"] == "copy":
        return case["pages"] * case["pools"] * case["page"] * case["Hkv"] * case["D"]
    if case["kind"] in ("kv4_attend", "kv4_mixed"):
        return case["nseq"] * case["len_max"] * case["Hkv"] * case["D"]
    return 0


def _draw(rng):
    kind = rng.choice(["qknr", "qknr_train", "kv4_append", "kv4_attend", "kv4_attend", "kv4_attend", "kv4_mixed",
                       "copy"])
    half = rng.choice(["bf16", "bf16", "fp16"])
    hq, hkv = rng.choice([(32, 8), (16, 16), (64, 8), (32, 4), (12, 12), (16, 8)])
    seed = rng.randrange(1 << 20)
    if kind in ("qknr", "qknr_train"):
        d = rng.choice([64, 128, 128, 96, 80, 36])
        length = _log_int(rng, 1, 16384)
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), B=rng.choice([0, 0, 1, 3]), L=length,
                    Hq=hq, Hkv=hkv, D=d, rotary=rng.choice([d, d, d // 2, d // 4 * 2 - 2]),
                    interleaved=rng.random() < 0.3, top=_log_int(rng, max(64, length), 65536))
    d = rng.choice([64, 128, 128, 96, 32])
    page = rng.choice([64, 128, 256, 256])
    if kind == "kv4_append":
        if rng.random() < 0.5:
            new = (1, rng.randrange(1, 6))
        else:
            new = (1, _log_int(rng, 16, 8192))
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), nseq=_log_int(rng, 1, 64),
                    new_min=new[0], new_max=new[1], old_min=0, old_max=_log_int(rng, 1, 4096), len_seed=seed, page=page,
                    Hkv=hkv, D=d)
    if kind == "copy":
        pages = _log_int(rng, 16, 1024)
        return dict(kind=kind, dtype=rng.choice(["bf16", "fp16", "fp32"]), pairs=_log_int(rng, 1, pages // 2), pages=pages,
                    pools=rng.choice([1, 2, 2, 8]), page=page, Hkv=hkv, D=rng.choice([64, 128, 72]))
    opts = dict(causal=rng.random() < 0.8, left=_log_int(rng, 32, 4096) if rng.random() < 0.25 else -1,
                softcap=rng.choice([0.0, 0.0, 0.0, 30.0]))
    if kind == "kv4_mixed":
        chunk = _log_int(rng, 32, 1024)
        top = _log_int(rng, max(chunk, 256), 8192)
        return dict(kind=kind, dtype=half, nseq=_log_int(rng, 1, 48), Lq=chunk, len_min=max(1, top // 16), len_max=top,
                    len_seed=seed, page=page, Hq=hq, Hkv=hkv, D=d, **opts)
    form = rng.choice(["one", "one", "draft", "chunk"])
    if form == "one":
        nseq, lq, top = _log_int(rng, 1, 64), 1, _log_int(rng, 200, 16384)
    elif form == "draft":
        nseq, lq, top = _log_int(rng, 1, 32), rng.randrange(2, 17), _log_int(rng, 200, 16384)
    else:
        nseq, lq = _log_int(rng, 1, 6), _log_int(rng, 17, 2048)
        top = _log_int(rng, max(lq, 300), 16384)
    return dict(kind=kind, dtype=half, nseq=nseq, Lq=lq, len_min=min(top, max(lq, top // 16)), len_max=top, len_seed=seed,
                page=page, Hq=hq, Hkv=hkv, D=d, **opts)


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


def _empty_cache(pages, page, heads, d):
    """A 4-bit pool (codes, scales), each head's rows of a page side by side in memory."""
    return tuple(torch.zeros(pages, heads, page, n, dtype=torch.uint8, device=_DEV).transpose(1, 2)
                 for n in (d // 2, d // 32))


def _filled_cache(g, pages, page, heads, d):
    """The same, of rows ~ N(0, 1) with a few larger channels."""
    codes, scales = _empty_cache(pages, page, heads, d)
    gain = torch.exp(0.5 * torch.randn(heads, d, generator=g, device=_DEV))
    step = max(1, (1 << 26) // (page * heads * d))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        c, s = _quantize(torch.randn(n, page, heads, d, generator=g, device=_DEV) * gain)
        codes[p:p + n], scales[p:p + n] = c, s
    return codes, scales


def _attend_lens(case):
    """(query rows, cached keys) of each sequence; a mixed step's chunk comes last."""
    lens = _lens(case)
    if case["kind"] == "kv4_mixed":
        return [1] * len(lens) + [case["Lq"]], lens + [max(case["Lq"], case["len_max"])]
    return [case["Lq"]] * len(lens), lens


def prepare(case, seed):
    """Inputs from the seed alone, on the GPU."""
    g = torch.Generator(device=_DEV).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    kind = case["kind"]
    s = dict(case=case)
    if kind in ("qknr", "qknr_train"):
        B, L, Hq, Hkv, D = (case[x] for x in ("B", "L", "Hq", "Hkv", "D"))
        lead = (B, L) if B else (L,)
        if kind == "qknr":  # views of a packed projection
            qkv = _randn(g, *lead, Hq + 2 * Hkv, D, dtype=dt)
            s["q"], s["k"] = qkv[..., :Hq, :], qkv[..., Hq:Hq + Hkv, :]
        else:
            s["q"], s["k"] = _randn(g, *lead, Hq, D, dtype=dt), _randn(g, *lead, Hkv, D, dtype=dt)
            s["dq"], s["dk"] = _randn(g, *lead, Hq, D, dtype=dt), _randn(g, *lead, Hkv, D, dtype=dt)
        for x in ("qw", "kw"):
            s[x] = (1 + 0.2 * torch.randn(D, generator=g, device=_DEV)).to(dt)
        if kind == "qknr_train":
            for x in ("q", "k", "qw", "kw"):
                s[x].requires_grad_()
        # angles in 64 bits, as a model makes its tables once
        half = case["rotary"] // 2
        freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=_DEV) / max(half, 1))
        angle = torch.arange(case["top"], dtype=torch.float64, device=_DEV)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["pos"] = torch.randint(0, case["top"], lead, generator=g, device=_DEV, dtype=torch.int32)
    elif kind == "kv4_append":
        new, old = _lens(case, "new_min", "new_max"), _lens(case, "old_min", "old_max", 1)
        s["k"], s["v"] = (_randn(g, sum(new), case["Hkv"], case["D"], dtype=dt) for _ in range(2))
        s["table"], pages = _table([a + b for a, b in zip(new, old)], case["page"], seed)
        s["kc"], s["vc"] = (_empty_cache(pages, case["page"], case["Hkv"], case["D"]) for _ in range(2))
        s["cu"], s["old"] = _cu(new), torch.tensor(old, dtype=torch.int32, device=_DEV)
        s["new"] = torch.tensor(new, device=_DEV)
        s["total"] = sum(new)
    elif kind in ("kv4_attend", "kv4_mixed"):
        lq, lk = _attend_lens(case)
        s["table"], pages = _table(lk, case["page"], seed)
        s["kc"], s["vc"] = (_filled_cache(g, pages, case["page"], case["Hkv"], case["D"]) for _ in range(2))
        s["lens"], s["lq"], s["max_k"] = torch.tensor(lk, dtype=torch.int32, device=_DEV), lq, max(lk)
        if kind == "kv4_attend":
            s["q"] = _randn(g, len(lk), case["Lq"], case["Hq"], case["D"], dtype=dt)
        else:
            s["q"] = _randn(g, sum(lq), case["Hq"], case["D"], dtype=dt)
            s["cu_q"] = _cu(lq)
    else:  # copy
        shape = (case["pages"], case["page"], case["Hkv"], case["D"])
        s["pools"] = [torch.empty(shape, dtype=dt, device=_DEV).normal_(generator=g) for _ in range(case["pools"])]
        ids = torch.randperm(case["pages"], generator=torch.Generator().manual_seed(seed)).to(_DEV, torch.int32)
        s["src"], s["dst"] = ids[:case["pairs"]].contiguous(), ids[case["pairs"]:2 * case["pairs"]].contiguous()
    return s


# --------------------------------------------------------------------------
# one pass


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import mtlflashattn_amd as mfa

    case = s["case"]
    kind = case["kind"]
    if kind == "qknr":
        with torch.no_grad():
            return mfa.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], s["pos"],
                                    interleaved=case["interleaved"])
    if kind == "qknr_train":
        q, k = mfa.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], s["pos"],
                                interleaved=case["interleaved"])
        return (q.detach(), k.detach(),
                *torch.autograd.grad((q, k), (s["q"], s["k"], s["qw"], s["kw"]), (s["dq"], s["dk"])))
    if kind == "kv4_append":
        k, v = mfa.kv4_append(s["k"], s["v"], s["kc"], s["vc"], s["cu"], s["old"], s["table"], return_values=True)
        return k, v, *s["kc"], *s["vc"]
    opts = {} if kind == "copy" else dict(causal=case["causal"], window_size=(case["left"], -1), softcap=case["softcap"])
    if kind == "kv4_attend":
        with torch.no_grad():
            return mfa.flash_attn_kv4_func(s["q"], s["kc"], s["vc"], s["lens"], s["table"], max_seqlen_k=s["max_k"],
                                           **opts)
    if kind == "kv4_mixed":
        with torch.no_grad():
            return mfa.flash_attn_varlen_kv4_func(s["q"], s["kc"], s["vc"], s["cu_q"], s["lens"], s["table"],
                                                  max_seqlen_k=s["max_k"], **opts)
    mfa.copy_cache_pages(s["pools"], s["src"], s["dst"])
    return s["pools"]


# The plain forms: elementary operations in 32 bits.


def _quantize(x):
    """(codes, scales) of [..., D] rows."""
    g = x.float().unflatten(-1, (-1, 32))
    amax = g.abs().amax(-1)
    m, e = torch.frexp(amax)
    e = torch.where(amax == 0, -127, e - 3 + (m > 0.875)).clamp(-127, 126).to(torch.int32)
    bad = ~torch.isfinite(amax)
    v = g * ((127 - e) << 23).view(torch.float32)[..., None]
    a = v.abs()
    code = (a > 0.25).to(torch.uint8)
    for border, above in ((0.75, False), (1.25, True), (1.75, False), (2.5, True), (3.5, False), (5.0, True)):
        code += (a > border) if above else (a >= border)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).masked_fill(bad[..., None], 0).flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), torch.where(bad, 255, e + 127).to(torch.uint8)


def _dequantize(codes, scales):
    """fp32 rows of (codes, scales)."""
    levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    x = torch.where(c > 7, -levels[c & 7], levels[c & 7]).unflatten(-1, (-1, 32))
    return (x * (scales.int() << 23).view(torch.float32)[..., None]).flatten(-2)


def _rotate(x, cos, sin, rotary, interleaved, back=False):
    """The first `rotary` elements of each row turned by their angles (or back)."""
    if back:
        sin = -sin
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., rotary:]), -1)


def _attend_plain(q, kc, vc, table, lens, case):
    """q [B, Lq, Hq, D] over the cached keys of each sequence."""
    B, Lq, Hq, D = q.shape
    Hkv = case["Hkv"]
    k, v = (_dequantize(codes[table.long()], scales[table.long()]).flatten(1, 2).transpose(1, 2).contiguous()
            for codes, scales in (kc, vc))  # [B, Hkv, keys, D]
    qf = q.float().unflatten(2, (Hkv, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, Hkv, heads * Lq, D]
    s = torch.matmul(qf, k.transpose(2, 3)) / math.sqrt(D)
    if case["softcap"] > 0:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    j = torch.arange(k.shape[2], device=q.device)
    center = torch.arange(Lq, device=q.device) + (lens.long()[:, None] - Lq)  # [B, Lq]
    ok = (j < lens.long()[:, None])[:, None, :]
    if case["causal"]:
        ok = ok & (j <= center[..., None])
    if case["left"] >= 0:
        ok = ok & (j >= center[..., None] - case["left"])
    ok = ok.expand(B, Lq, j.shape[0])[:, None, None]
    s = s.unflatten(2, (-1, Lq)).masked_fill(~ok, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (-1, Lq)) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3).to(q.dtype)


@torch.no_grad()
def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind in ("qknr", "qknr_train"):
        rot, inter = case["rotary"], case["interleaved"]
        cos, sin = s["cos"][s["pos"].long()][..., None, :], s["sin"][s["pos"].long()][..., None, :]
        outs, grads, wgrads = [], [], []
        for x, w, d in (("q", "qw", "dq"), ("k", "kw", "dk")):
            xf, wf = s[x].float(), s[w].float()
            r = torch.rsqrt(xf.square().mean(-1, keepdim=True) + 1e-6)
            n = xf * r
            outs.append(_rotate(n * wf, cos, sin, rot, inter).to(s[x].dtype))
            if kind == "qknr_train":
                gy = _rotate(s[d].float(), cos, sin, rot, inter, back=True)
                h = gy * wf
                grads.append((r * (h - n * (h * n).mean(-1, keepdim=True))).to(s[x].dtype))
                wgrads.append((gy * n).flatten(0, -2).sum(0).to(s[w].dtype))
        return (*outs, *grads, *wgrads)
    if kind == "kv4_append":
        seq = torch.repeat_interleave(torch.arange(case["nseq"], device=_DEV), s["new"], output_size=s["total"])
        at = s["old"].long()[seq] + torch.arange(s["total"], device=_DEV) - s["cu"].long()[seq]
        page = s["table"][seq, at // case["page"]].long()
        values = []
        for x, (codes, scales) in (("k", s["kc"]), ("v", s["vc"])):
            c, e = _quantize(s[x])
            codes[page, at % case["page"]] = c
            scales[page, at % case["page"]] = e
            values.append(_dequantize(c, e).to(s[x].dtype))
        return *values, *s["kc"], *s["vc"]
    if kind == "kv4_attend":
        return _attend_plain(s["q"], s["kc"], s["vc"], s["table"], s["lens"], case)
    if kind == "kv4_mixed":
        n = case["nseq"]
        one = _attend_plain(s["q"][:n, None], s["kc"], s["vc"], s["table"][:n], s["lens"][:n], case)
        chunk = _attend_plain(s["q"][None, n:], s["kc"], s["vc"], s["table"][n:], s["lens"][n:], case)
        return torch.cat((one[:, 0], chunk[0]))
    for pool in s["pools"]:
        pool[s["dst"].long()] = pool[s["src"].long()]
    return s["pools"]


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
    kind = case["kind"]
    es = 4 if case["dtype"] == "fp32" else 2
    if kind in ("qknr", "qknr_train"):
        tokens = max(case["B"], 1) * case["L"]
        n = tokens * (case["Hq"] + case["Hkv"]) * case["D"]
        tables = min(tokens, case["top"]) * case["rotary"] * 4 + 4 * tokens
        if kind == "qknr":
            return {"bytes": 2 * n * es + tables, "flops": 8 * n}
        return {"bytes": 5 * n * es + 2 * tables, "flops": 26 * n}
    D, Hkv = case["D"], case["Hkv"]
    row4 = D // 2 + D // 32  # bytes of a cached row of one head
    if kind == "kv4_append":
        # the rows in, their codes and scales out, their values out
        n = sum(_lens(case, "new_min", "new_max")) * Hkv * 2
        return {"bytes": n * (2 * D * es + row4), "flops": 6 * n * D}
    if kind == "copy":
        return {"bytes": 2 * case["pairs"] * case["pools"] * case["page"] * Hkv * D * es, "flops": 0}
    lq, lk = _attend_lens(case)
    pairs = sum(_pairs(a, b, case["causal"], case["left"]) for a, b in zip(lq, lk))
    keys = sum(_read(a, b, case["left"]) for a, b in zip(lq, lk))
    return {"bytes": 2 * keys * Hkv * row4 + 2 * sum(lq) * case["Hq"] * D * es, "flops": 4 * D * case["Hq"] * pairs}


# --------------------------------------------------------------------------
# the result in 64 bits, from the definitions


_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pow2(n):
    return torch.pow(2.0, n.double())


def _codes64(x):
    """(four-bit codes, scale bytes, values) of finite [..., D] rows by search: the
    smallest scale within 7, the nearest level, of two equally near the even one."""
    g = x.double().unflatten(-1, (-1, 32))
    amax = g.abs().amax(-1)
    scale = torch.zeros_like(amax, dtype=torch.int64)
    for bit in (128, 64, 32, 16, 8, 4, 2, 1):  # the smallest byte whose scale holds the group
        low = scale + (bit - 1)
        scale = torch.where(amax * _pow2(127 - low) <= 7, scale, scale + bit)
    v = g * _pow2(127 - scale)[..., None]
    order = (0, 2, 4, 6, 1, 3, 5, 7)  # even codes first: argmin takes the first of equals
    best = torch.full_like(v, math.inf)
    code = torch.zeros_like(v, dtype=torch.int64)
    for c in order:
        dist = (v.abs() - _LEVELS[c]).abs()
        code = torch.where(dist < best, c, code)
        best = torch.minimum(dist, best)
    level = torch.tensor(_LEVELS, dtype=torch.float64, device=x.device)[code]
    value = torch.copysign(level, g) * _pow2(scale - 127)[..., None]
    code = (code + 8 * torch.signbit(g)).flatten(-2)
    return code, scale, value.flatten(-2)


def _rows64(codes, scales):
    """float64 rows [n, D] of one head's cached rows."""
    signed = torch.tensor(_LEVELS + tuple(-x for x in _LEVELS), dtype=torch.float64, device=codes.device)
    x = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device=codes.device)
    x[:, 0::2], x[:, 1::2] = signed[(codes % 16).long()], signed[(codes // 16).long()]
    return x * _pow2(scales.double() - 127).repeat_interleave(32, 1)


def _attend64(q, k, v, case):
    """One head: q [Lq, D] over k, v [Lk, D] in float64."""
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
    p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
    return p.masked_fill(hidden.all(-1, keepdim=True), 0.0) @ v


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("qknr", "qknr_train"):
        train, rot = kind == "qknr_train", case["rotary"]
        angle = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()].unsqueeze(-2)
        outs, leaves, ups = [], [], []
        for x, w, d in (("q", "qw", "dq"), ("k", "kw", "dk")):
            xx, ww = (s[i].detach().double().requires_grad_(train) for i in (x, w))
            y = xx / torch.sqrt((xx * xx).sum(-1, keepdim=True) / case["D"] + 1e-6) * ww
            head = y[..., :rot]
            pair = head.unflatten(-1, (-1, 2)) if case["interleaved"] else head.unflatten(-1, (2, -1)).transpose(-1, -2)
            z = torch.view_as_real(torch.complex(pair[..., 0], pair[..., 1]) * angle)
            z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
            outs.append(torch.cat((z, y[..., rot:]), -1))
            leaves.append((xx, ww))
            ups.append(s[d].double() if train else None)
        if not train:
            return tuple(outs)
        (q, qw), (k, kw) = leaves
        grads = torch.autograd.grad(outs, (q, k, qw, kw), ups)
        return (*(o.detach() for o in outs), *grads)
    if kind == "kv4_append":
        outs, pools = [], []
        cu, old, page = s["cu"].tolist(), s["old"].tolist(), case["page"]
        for x, (codes, scales) in (("k", s["kc"]), ("v", s["vc"])):
            c, e, value = _codes64(s[x])
            outs.append(value)
            codes, scales = codes.clone(), scales.clone()
            for b in range(case["nseq"]):
                for t in range(cu[b], cu[b + 1]):
                    stop = min(cu[b + 1], t + page)
                    at = old[b] + t - cu[b]
                    if at % page and t > cu[b]:
                        continue  # (rows of this page are already written)
                    stop = min(stop, t + page - at % page)
                    p, r = int(s["table"][b, at // page]), at % page
                    codes[p, r:r + stop - t] = (c[t:stop, :, 0::2] + 16 * c[t:stop, :, 1::2]).to(torch.uint8)
                    scales[p, r:r + stop - t] = e[t:stop].to(torch.uint8)
            pools += [codes, scales]
        return (*outs, *pools)
    if kind == "copy":
        pairs = list(zip(s["src"].tolist(), s["dst"].tolist()))
        for pool in s["pools"]:
            for a, b in pairs:
                pool[b].copy_(pool[a])
        return s["pools"]
    lq, lk = _attend_lens(case)
    r = case["Hq"] // case["Hkv"]
    rows = s["q"].flatten(0, 1) if kind == "kv4_attend" else s["q"]
    out = torch.empty(rows.shape, dtype=torch.float64, device=rows.device)
    start = 0
    for b, (n, keys) in enumerate(zip(lq, lk)):
        ids = s["table"][b, :-(-keys // case["page"])].long()
        q = rows[start:start + n].double()
        parts = [tuple(t[ids].flatten(0, 1)[:keys] for t in pool) for pool in (s["kc"], s["vc"])]
        for h in range(case["Hkv"]):
            k, v = (_rows64(c[:, h], e[:, h]) for c, e in parts)
            for i in range(h * r, h * r + r):
                out[start:start + n, i] = _attend64(q[:, i].contiguous(), k, v, case)
        start += n
    return out.view(s["q"].shape)
