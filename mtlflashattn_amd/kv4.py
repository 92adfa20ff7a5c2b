"""A paged K/V cache held in 4 bits: writing it, attention over it, and copies of
its pages.  The reference has no cache (block_table raises,
metal_flash_attn/__init__.py:130-131); here 16-bit pages are read by
flash_attn_varlen_func and 4-bit pages, 17/64 of their size, by the functions of
this module.

Format (include/mfa.h): 32 consecutive elements of a head share one power-of-two
scale byte and are 4-bit floats (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives).
A cache of K or V is a pair (codes, scales) of uint8 tensors [num_pages,
page_block_size, Hkv, D / 2] and [..., D / 32], as kv4_cache makes it.
"""
from __future__ import annotations

import math

import torch

from . import _hip, _kernel
from ._kernel import MAX_HEAD_DIM

_ATTEND_DTYPES = (torch.float16, torch.bfloat16)

# prepared parameters (everything but the data pointers) of a call's signature
_plans = {}


def _remember(key, plan):
    if len(_plans) >= _kernel._PLANS_MAX:
        _plans.clear()
    _plans[key] = plan
    return plan


def _not_tensors(k_cache, v_cache):
    """The error for arguments of which no signature can be formed."""
    for what, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not isinstance(c, (tuple, list)) or len(c) != 2 or not (torch.is_tensor(c[0]) and torch.is_tensor(c[1])):
            return ValueError(f"mtlflashattn_amd: {what} must be a pair (codes, scales), as kv4_cache makes it")
    return ValueError("mtlflashattn_amd: tensors expected")


def kv4_cache(num_pages, page_block_size, num_heads_kv, head_dim, device="cuda"):
    """An empty 4-bit cache of K or of V: (codes, scales).

    codes: uint8 [num_pages, page_block_size, num_heads_kv, head_dim / 2], scales:
    uint8 [..., head_dim / 32], zeroed (rows read as 0).  In memory each head's
    rows of a page lie side by side (the heads-third shape is a view), which the
    kernels read fastest; they take any other order too.  page_block_size: a
    multiple of 64; head_dim: 32, 64, 96 or 128.
    """
    if page_block_size <= 0 or page_block_size % 64:
        raise ValueError(f"mtlflashattn_amd: page_block_size {page_block_size} must be a positive multiple of 64")
    if head_dim <= 0 or head_dim % 32 or head_dim > MAX_HEAD_DIM:
        raise NotImplementedError(f"mtlflashattn_amd: head_dim {head_dim} of a 4-bit cache must be 32, 64, 96 or 128")
    return tuple(torch.zeros(num_pages, num_heads_kv, page_block_size, n, dtype=torch.uint8, device=device).transpose(1, 2)
                 for n in (head_dim // 2, head_dim // 32))


def _check_cache(cache, D, Hkv, device, what):
    codes, scales = cache
    if codes.dim() != 4 or scales.dim() != 4 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError(f"mtlflashattn_amd: {what}: codes and scales must be 4-D uint8 tensors")
    page = codes.shape[1]
    if page == 0 or page % 64:
        raise ValueError(f"mtlflashattn_amd: page_block_size {page} must be a positive multiple of 64")
    if tuple(codes.shape[2:]) != (Hkv, D // 2) or tuple(scales.shape) != (*codes.shape[:3], D // 32):
        raise ValueError(f"mtlflashattn_amd: {what}: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not "
                         f"hold {Hkv} heads of {D} elements")
    for t, unit in ((codes, 16), (scales, 1)):
        if t.device != device:
            raise ValueError(f"mtlflashattn_amd: tensors on different devices ({device} vs {t.device})")
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"mtlflashattn_amd: {what}: the last dimension must be contiguous")
        if any(s % unit for s, n in zip(t.stride()[:3], t.shape[:3]) if n > 1):
            raise ValueError(f"mtlflashattn_amd: {what}: code strides must be multiples of 16 bytes")


def _check_table(block_table, batch, device):
    if not torch.is_tensor(block_table) or block_table.dim() != 2 or block_table.dtype != torch.int32:
        raise ValueError("mtlflashattn_amd: block_table must be an int32 [batch, max_pages] tensor")
    if block_table.shape[0] != batch:
        raise ValueError(f"mtlflashattn_amd: block_table has {block_table.shape[0]} rows for {batch} sequences")
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise ValueError("mtlflashattn_amd: block_table must have contiguous rows")
    if block_table.device != device:
        raise ValueError(f"mtlflashattn_amd: tensors on different devices ({device} vs {block_table.device})")


def _check_ints(t, n, device, what):
    if not torch.is_tensor(t) or t.dtype not in (torch.int32, torch.int64) or tuple(t.shape) != (n,):
        raise ValueError(f"mtlflashattn_amd: {what} must be an int32 tensor of {n} elements")
    if t.device != device:
        raise ValueError(f"mtlflashattn_amd: tensors on different devices ({device} vs {t.device})")


def _cache_struct(c, k_cache, v_cache, block_table):
    """The strides and sizes of a cache."""
    for pool, (codes, scales) in ((c.k, k_cache), (c.v, v_cache)):
        pool.code_page_stride, pool.code_row_stride, pool.code_head_stride = (
            s if n > 1 else 0 for s, n in zip(codes.stride()[:3], codes.shape[:3]))
        pool.scale_page_stride, pool.scale_row_stride, pool.scale_head_stride = (
            s if n > 1 else 0 for s, n in zip(scales.stride()[:3], scales.shape[:3]))
    c.num_pages, c.page_block_size = pages, page = k_cache[0].shape[:2]
    _kernel._check_sizes(pages, block_table.shape[1] * page)  # (rows that a sequence's table names)
    c.max_pages = block_table.shape[1]
    c.block_table_batch_stride = block_table.stride(0) if block_table.shape[0] > 1 else 0


def _cache_pointers(c, kc, ks, vc, vs, block_table):
    pool = c.k
    pool.codes, pool.scales = kc.data_ptr(), ks.data_ptr()
    pool = c.v
    pool.codes, pool.scales = vc.data_ptr(), vs.data_ptr()
    c.block_table = block_table.data_ptr()


# (tensors written in place: a graph that saved one raises the usual error in its backward)
_written = torch.autograd.graph.increment_version


def _i32(t):
    return t if t.dtype is torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _check_pages(block_table, lens, page, num_pages):
    """The page ids that `lens` rows use, on the host (MTLFLASHATTN_CHECK_PAGES=1)."""
    lens = lens.clamp(min=0).cpu().long()
    used = torch.arange(block_table.shape[1]).unsqueeze(0) < ((lens + page - 1) // page).unsqueeze(1)
    if lens.numel() and int(lens.max()) > block_table.shape[1] * page:
        raise ValueError(f"mtlflashattn_amd: block_table has {block_table.shape[1]} pages per sequence, "
                         f"too few for {int(lens.max())} rows")
    ids = block_table.cpu()[used]
    if ids.numel() and (int(ids.min()) < 0 or int(ids.max()) >= num_pages):
        raise ValueError(f"mtlflashattn_amd: block_table holds page ids outside [0, {num_pages})")


def kv4_append(k, v, k_cache, v_cache, cu_seqlens, cache_seqlens, block_table, return_values=False):
    """Write new rows into a paged 4-bit cache, in one launch.

    k, v: [total, Hkv, D] fp16 / bf16 / fp32 rows packed without padding (views are
    read in place); cu_seqlens: int32 [B + 1], sequence b owning tokens
    [cu_seqlens[b], cu_seqlens[b + 1]); cache_seqlens: int32 [B], the rows each
    sequence holds already.  Token t of sequence b becomes row cache_seqlens[b] + t -
    cu_seqlens[b], which is row j % page_block_size of page block_table[b, j //
    page_block_size].  cache_seqlens is not changed.  All of them are read on the
    device (no synchronisation): a row behind the last column of the table or on a
    page id outside the pool is dropped, as are tokens of no sequence.  No two
    tokens may land on one row: a page that forked sequences share is copied
    (copy_cache_pages) before one of them writes to it.

    Each 32 elements take the smallest power-of-two scale that leaves them within 7
    times it; elements are rounded to the nearest 4-bit value, ties to the even
    code.  A group with an infinity or a NaN is held as NaN.

    return_values=True returns (k', v') [total, Hkv, D] in k.dtype: the rows as the
    cache now holds them (or would, where a row is dropped), for attention over a prompt that later steps will read
    back from the cache (flash_attn_varlen_func(q, k', v', ...)).  Not
    differentiable: inputs that require grad raise.
    """
    try:
        (kc, ks), (vc, vs) = k_cache, v_cache
        key = ("append", k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device,
               kc.shape, kc.stride(), kc.dtype, kc.device, ks.shape, ks.stride(), ks.dtype, ks.device,
               vc.shape, vc.stride(), vc.dtype, vc.device, vs.shape, vs.stride(), vs.dtype, vs.device,
               cu_seqlens.shape, cu_seqlens.stride(), cu_seqlens.dtype, cu_seqlens.device,
               cache_seqlens.shape, cache_seqlens.stride(), cache_seqlens.dtype, cache_seqlens.device,
               block_table.shape, block_table.stride(), block_table.dtype, block_table.device)
    except (AttributeError, TypeError, ValueError):
        raise _not_tensors(k_cache, v_cache) from None
    _kernel._check_no_tangent(k, v)
    if _kernel._needs_grad(k, v):
        raise NotImplementedError("mtlflashattn_amd: kv4_append is not differentiable; run it under torch.no_grad() or on "
                                  "detached rows")
    plan = _plans.get(key) or _remember(key, _append_plan(k, v, k_cache, v_cache, cu_seqlens, cache_seqlens, block_table))
    template, direct = plan
    p = _hip.MfaKv4AppendParams.from_buffer_copy(template)
    kp, vp = k.data_ptr(), v.data_ptr()
    if not direct or (kp | vp) & 15:
        k_, v_, cu_seqlens, cache_seqlens = (_kernel._abi_operand(k), _kernel._abi_operand(v), _i32(cu_seqlens),
                                             _i32(cache_seqlens))
        kp, vp = k_.data_ptr(), v_.data_ptr()
        p.k_token_stride, p.k_head_stride = _token_strides(k_)
        p.v_token_stride, p.v_head_stride = _token_strides(v_)
    if _kernel._check_pages_enabled():
        _check_pages(block_table, cache_seqlens + (cu_seqlens[1:] - cu_seqlens[:-1]), kc.shape[1], kc.shape[0])
    p.k, p.v, p.cu_seqlens, p.cache_seqlens = kp, vp, cu_seqlens.data_ptr(), cache_seqlens.data_ptr()
    _cache_pointers(p.cache, kc, ks, vc, vs, block_table)
    values = None
    if return_values:
        values = tuple(torch.empty_like(t, memory_format=torch.contiguous_format) for t in (k, v))
        p.k_values, p.v_values = values[0].data_ptr(), values[1].data_ptr()
    _kernel._launch_on(k.device, _hip.kv4_append, p)
    _written((kc, ks, vc, vs))
    return values


def _token_strides(x):
    return tuple(s if n > 1 else 0 for s, n in zip(x.stride()[:2], x.shape[:2]))


def _append_plan(k, v, k_cache, v_cache, cu_seqlens, cache_seqlens, block_table):
    """(parameters without data pointers, whether the tensors are used in place) of a kv4_append call."""
    if k.dim() != 3 or v.dim() != 3 or k.shape != v.shape:
        raise ValueError(f"mtlflashattn_amd: expected k and v [total,H,D], got {tuple(k.shape)} and {tuple(v.shape)}")
    _kernel._check_device(k, v)
    if k.dtype not in _kernel._SUPPORTED_DTYPES or v.dtype != k.dtype:
        raise NotImplementedError(f"mtlflashattn_amd: dtype {k.dtype} (k/v must match, fp16/bf16/fp32)")
    total, Hkv, D = k.shape
    if D == 0 or D % 32 or D > MAX_HEAD_DIM:
        raise NotImplementedError(f"mtlflashattn_amd: head_dim {D} of a 4-bit cache must be 32, 64, 96 or 128")
    _check_cache(k_cache, D, Hkv, k.device, "k_cache")
    _check_cache(v_cache, D, Hkv, k.device, "v_cache")
    if k_cache[0].shape != v_cache[0].shape:
        raise ValueError("mtlflashattn_amd: k_cache and v_cache differ in pages")
    batch = cache_seqlens.shape[0] if cache_seqlens.dim() == 1 else 0
    _check_ints(cache_seqlens, batch, k.device, "cache_seqlens")
    _check_ints(cu_seqlens, batch + 1, k.device, "cu_seqlens")
    _check_table(block_table, batch, k.device)
    for c in (*k_cache, *v_cache):
        if any(s == 0 for s, n in zip(c.stride()[:3], c.shape[:3]) if n > 1):
            raise ValueError("mtlflashattn_amd: an expanded cache (rows that share memory) cannot be written")
    _kernel._check_sizes(total, Hkv, batch)
    p = _hip.MfaKv4AppendParams()
    _cache_struct(p.cache, k_cache, v_cache, block_table)
    p.k_token_stride, p.k_head_stride = _token_strides(k)
    p.v_token_stride, p.v_head_stride = _token_strides(v)
    p.batch, p.total, p.heads_kv, p.head_dim = batch, total, Hkv, D
    p.dtype = _hip.DTYPE_CODES[k.dtype]
    return p, (_kernel._fits_strides(k) and _kernel._fits_strides(v) and _i32(cu_seqlens) is cu_seqlens
               and _i32(cache_seqlens) is cache_seqlens)


def flash_attn_kv4_func(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale=None, causal=False,
                        window_size=(-1, -1), softcap=0.0, alibi_slopes=None, max_seqlen_k=None,
                        return_softmax_lse=False):
    """Attention of [B, Lq, Hq, D] queries over a paged 4-bit cache.

    q: fp16 or bf16, the last Lq positions of each sequence (Lq = 1: a decoding
    step; a few: drafted tokens; many: a chunk of a prompt whose rows kv4_append has
    written).  k_cache, v_cache: (codes, scales) pairs; cache_seqlens: int32 [B], the
    rows of each sequence in the cache, the queries' own included; block_table: int32
    [B, max_pages].  Masks, soft-cap, ALiBi, grouped-query heads as in
    flash_attn_func; rows with no valid key give 0, and keys that a row's mask leaves
    out do not reach it, NaN groups included.  Returns [B, Lq, Hq, D] in q.dtype,
    with return_softmax_lse=True also the log-sum-exp [B, Hq, Lq] fp32.

    Lengths and page ids are read on the device (no synchronisation: a call can be
    captured into a graph and replayed as the sequences grow).  A sequence has at
    most max_seqlen_k keys (None: as many as the table names); a tight bound keeps
    the workspace and the grid small.  Sequences of more than 32 columns (query
    positions times heads per K/V head) run on tiles of 128 columns, whose
    probabilities are rounded once to q.dtype (bf16: an error of 1.4 times the output's
    rounding alone) and which, for fp16 queries, round K and V to fp16 (beyond 65504
    they saturate); fewer columns keep two terms and exact K and V.  A page id outside the pool reads as zeros and
    its keys are not masked; MTLFLASHATTN_CHECK_PAGES=1 checks the ids on the host.
    Forward only: a query that requires grad raises.
    """
    if torch.is_tensor(q) and q.dim() != 4:
        raise ValueError(f"mtlflashattn_amd: expected q [B,Lq,H,D], got {q.dim()}-D")
    return _attend(q, k_cache, v_cache, None, cache_seqlens, block_table, softmax_scale, causal, window_size, softcap,
                   alibi_slopes, max_seqlen_k, return_softmax_lse)


def flash_attn_varlen_kv4_func(q, k_cache, v_cache, cu_seqlens_q, cache_seqlens, block_table, softmax_scale=None,
                               causal=False, window_size=(-1, -1), softcap=0.0, alibi_slopes=None, max_seqlen_k=None,
                               return_softmax_lse=False):
    """flash_attn_kv4_func for sequences of different query counts (a serving step
    that mixes prompt chunks and decoding sequences).

    q: [total, Hq, D] packed without padding, sequence b owning rows
    [cu_seqlens_q[b], cu_seqlens_q[b + 1]) (int32 [B + 1], read on the device; it must
    be non-decreasing).  Rows of no sequence come back as 0 (one workgroup clears them:
    8128 rows of 32 x 128 take 1 ms, so a captured step is padded little).  In a call
    of more than 32 columns in total sequences of more than 16 run on the tiles of 128.
    Returns [total, Hq, D]
    and, if asked, the log-sum-exp [Hq, total].
    """
    if torch.is_tensor(q) and q.dim() != 3:
        raise ValueError(f"mtlflashattn_amd: expected q [total,H,D], got {q.dim()}-D")
    return _attend(q, k_cache, v_cache, cu_seqlens_q, cache_seqlens, block_table, softmax_scale, causal, window_size,
                   softcap, alibi_slopes, max_seqlen_k, return_softmax_lse)


def _attend(q, k_cache, v_cache, cu_q, cache_seqlens, block_table, softmax_scale, causal, window_size, softcap, alibi_slopes,
            max_seqlen_k, return_lse):
    _kernel._check_options(window_size, softcap, alibi_slopes)
    # (numbers, so that the signature holds a value whatever type it came in)
    softmax_scale = None if softmax_scale is None else float(softmax_scale)
    # (a window as wide as a 32-bit number is as good as none)
    most = _kernel._INT32_MAX
    softcap, window_size = float(softcap), (min(int(window_size[0]), most), min(int(window_size[1]), most))
    max_seqlen_k = None if max_seqlen_k is None else int(max_seqlen_k)
    try:
        (kc, ks), (vc, vs) = k_cache, v_cache
        varlen = q.dim() == 3
        key = (q.shape, q.stride(), q.dtype, q.device, kc.shape, kc.stride(), kc.dtype, kc.device,
               ks.shape, ks.stride(), ks.dtype, ks.device, vc.shape, vc.stride(), vc.dtype, vc.device,
               vs.shape, vs.stride(), vs.dtype, vs.device,
               cache_seqlens.shape, cache_seqlens.stride(), cache_seqlens.dtype, cache_seqlens.device,
               block_table.shape, block_table.stride(), block_table.dtype, block_table.device,
               varlen and (cu_q.shape, cu_q.stride(), cu_q.dtype, cu_q.device),
               alibi_slopes is not None and (alibi_slopes.shape, alibi_slopes.device),
               softmax_scale, bool(causal), window_size, softcap, max_seqlen_k)
    except (AttributeError, TypeError, ValueError):
        raise _not_tensors(k_cache, v_cache) from None
    _kernel._check_no_tangent(q)
    if q.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("mtlflashattn_amd: attention over a 4-bit cache is forward-only; run it under "
                                  "torch.no_grad() or without inputs that require grad")
    plan = _plans.get(key) or _remember(key, _attend_plan(
        q, k_cache, v_cache, cu_q, cache_seqlens, block_table, softmax_scale, causal, window_size, softcap, alibi_slopes,
        max_seqlen_k))
    template, nbytes, direct = plan
    if _kernel._trace_enabled():
        _kernel._record_trace(q.dtype, q.shape[-1], q.shape[0 if varlen else 1], template.max_seqlen_k, causal, "hip-kv4")
    p = _hip.MfaKv4FwdParams.from_buffer_copy(template)
    device, qp = q.device, q.data_ptr()
    if not direct or qp & 15:
        q_, cache_seqlens = _kernel._abi_operand(q), _i32(cache_seqlens)
        qp = q_.data_ptr()
        strides = [s if n > 1 else 0 for s, n in zip(q_.stride(), q_.shape)]
        p.q_batch_stride, p.q_seq_stride, p.q_head_stride = (0, *strides[:2]) if varlen else strides[:3]
        if varlen:
            cu_q = _i32(cu_q)
    if _kernel._check_pages_enabled():
        _check_pages(block_table, cache_seqlens.clamp(max=template.max_seqlen_k), kc.shape[1], kc.shape[0])
    out, lse = torch.empty_like(q, memory_format=torch.contiguous_format), None
    if return_lse:
        shape = (q.shape[1], q.shape[0]) if varlen else (q.shape[0], q.shape[2], q.shape[1])
        lse = torch.empty(shape, dtype=torch.float32, device=device)
        p.softmax_lse = lse.data_ptr()
    if varlen:
        p.cu_seqlens_q = cu_q.data_ptr()
    if alibi_slopes is not None:
        slopes, p.alibi_batch_stride = _kernel._alibi_arg(alibi_slopes, p.batch, p.heads_q, device)
        p.alibi_slopes = slopes.data_ptr()
    p.q, p.o, p.cache_seqlens = qp, out.data_ptr(), cache_seqlens.data_ptr()
    _cache_pointers(p.cache, kc, ks, vc, vs, block_table)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _kernel._launch_on(device, _hip.kv4_fwd, p, None if ws is None else ws.data_ptr(), nbytes)
    return (out, lse) if return_lse else out


def _attend_plan(q, k_cache, v_cache, cu_q, cache_seqlens, block_table, softmax_scale, causal, window_size, softcap,
                 alibi_slopes, max_seqlen_k):
    """(parameters without data pointers, workspace bytes, whether the tensors are used in place) of a call."""
    varlen = q.dim() == 3
    _kernel._check_device(q)
    if q.dtype not in _ATTEND_DTYPES:
        raise NotImplementedError(f"mtlflashattn_amd: dtype {q.dtype} (queries over a 4-bit cache are fp16 or bf16)")
    Hq, D = q.shape[-2:]
    if D not in (32, 64, 96, 128):
        raise NotImplementedError(f"mtlflashattn_amd: head_dim {D} of a 4-bit cache must be 32, 64, 96 or 128")
    Hkv = k_cache[0].shape[2] if k_cache[0].dim() == 4 else 0
    _check_cache(k_cache, D, Hkv, q.device, "k_cache")
    _check_cache(v_cache, D, Hkv, q.device, "v_cache")
    if k_cache[0].shape != v_cache[0].shape:
        raise ValueError("mtlflashattn_amd: k_cache and v_cache differ in pages or heads")
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"mtlflashattn_amd: num_heads_kv ({Hkv}) must divide num_heads_q ({Hq})")
    if varlen:
        batch = cache_seqlens.shape[0] if cache_seqlens.dim() == 1 else 0
        _check_ints(cu_q, batch + 1, q.device, "cu_seqlens_q")
    else:
        batch = q.shape[0]
    _check_ints(cache_seqlens, batch, q.device, "cache_seqlens")
    _check_table(block_table, batch, q.device)
    if max_seqlen_k is not None and max_seqlen_k < 0:
        raise ValueError("mtlflashattn_amd: max_seqlen_k must be >= 0")
    _kernel._alibi_arg(alibi_slopes, batch, Hq, q.device)
    _kernel._check_sizes(*q.shape, batch)
    p = _hip.MfaKv4FwdParams()
    _cache_struct(p.cache, k_cache, v_cache, block_table)
    p.batch, p.heads_q, p.heads_kv, p.head_dim = batch, Hq, Hkv, D
    strides = [s if n > 1 else 0 for s, n in zip(q.stride(), q.shape)]
    if varlen:
        p.total_q = q.shape[0]
        p.q_seq_stride, p.q_head_stride = strides[:2]
        p.o_seq_stride, p.o_head_stride = Hq * D, D
        p.lse_head_stride = q.shape[0]
    else:
        p.seqlen_q = q.shape[1]
        p.q_batch_stride, p.q_seq_stride, p.q_head_stride = strides[:3]
        p.o_batch_stride, p.o_seq_stride, p.o_head_stride = q.shape[1] * Hq * D, Hq * D, D
        p.lse_batch_stride, p.lse_head_stride = Hq * q.shape[1], q.shape[1]
    cap = block_table.shape[1] * k_cache[0].shape[1]
    p.max_seqlen_k = cap if max_seqlen_k is None else min(max_seqlen_k, cap)
    if p.max_seqlen_k == 0:  # (0 means no bound to the library)
        p.cache.max_pages = 0
    p.scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D)
    p.softcap = softcap
    p.window_left, p.window_right = window_size
    p.causal = int(bool(causal))
    p.dtype = _hip.DTYPE_CODES[q.dtype]
    # placeholders: sizing the workspace reads no tensor
    sized = _hip.MfaKv4FwdParams.from_buffer_copy(p)
    sized.q = sized.o = sized.cache_seqlens = sized.cache.block_table = 256
    sized.cache.k.codes = sized.cache.k.scales = sized.cache.v.codes = sized.cache.v.scales = 256
    sized.cu_seqlens_q = 256 if varlen else None
    sized.q_batch_stride = sized.q_seq_stride = sized.q_head_stride = 0
    with _kernel._on(q.device):
        nbytes = _hip.kv4_fwd_workspace_bytes(sized)
    return p, nbytes, (_kernel._fits_strides(q) and _i32(cache_seqlens) is cache_seqlens
                       and (not varlen or _i32(cu_q) is cu_q))


def copy_cache_pages(pools, src, dst):
    """Copy page src[i] to page dst[i] in every pool, in one launch per 64 pools.

    pools: tensors [num_pages, ...] of any dtype that hold one page after another:
    16-bit K and V pools, (codes, scales) of 4-bit caches, of one layer or many; each
    page dense in memory (any order of its dimensions).  src, dst: int32 [n] page ids,
    read on the device (no synchronisation); a pair with an id outside the pools is
    skipped, so -1 pads a list.  This is what forked sequences (the shared last page is
    copied before one of them writes to it) and compaction (pages move into free ones)
    need.  The destinations have to differ from each other and from every source; pairs
    are copied in no order.  MTLFLASHATTN_CHECK_PAGES=1 checks that on the host and raises
    ValueError.  The pools count as modified in place.
    """
    pools = list(pools)
    if not pools:
        return
    try:
        key = ("copy", src.shape, src.stride(), src.dtype, src.device, dst.shape, dst.stride(), dst.dtype, dst.device,
               *[x for t in pools for x in (t.shape, t.stride(), t.dtype, t.device)])
    except AttributeError:
        raise ValueError("mtlflashattn_amd: pools, src and dst must be tensors") from None
    if torch.is_grad_enabled() and any([t.requires_grad for t in pools]):
        raise NotImplementedError("mtlflashattn_amd: copy_cache_pages is not differentiable")
    plan = _plans.get(key) or _remember(key, _copy_plan(pools, src, dst))
    templates, direct = plan
    device = pools[0].device
    if not direct:
        src, dst = _i32(src), _i32(dst)
    if _kernel._check_pages_enabled():
        num_pages = pools[0].shape[0]
        pairs = [(a, b) for a, b in zip(src.tolist(), dst.tolist()) if 0 <= a < num_pages and 0 <= b < num_pages and a != b]
        to = [b for _, b in pairs]
        if len(set(to)) != len(to) or set(to) & {a for a, _ in pairs}:
            raise ValueError("mtlflashattn_amd: copy_cache_pages: a destination is given twice or is a source too")
    first = 0
    for template in templates:
        p = _hip.MfaCopyPagesParams.from_buffer_copy(template)
        pool = p.pool
        for i in range(p.pools):
            pool[i].base = pools[first + i].data_ptr()
        first += p.pools
        p.src, p.dst = src.data_ptr(), dst.data_ptr()
        _kernel._launch_on(device, _hip.copy_pages, p)
    _written(pools)


def _copy_plan(pools, src, dst):
    """(parameters without data pointers of each launch, whether the ids are used in place)."""
    _kernel._check_device(*pools)
    if any(t.dim() < 1 for t in pools) or src.dim() != 1:
        raise ValueError("mtlflashattn_amd: pools must be [num_pages, ...] tensors, src and dst int32 [n] page ids")
    device, num_pages = pools[0].device, pools[0].shape[0]
    _check_ints(src, src.shape[0], device, "src")
    _check_ints(dst, src.shape[0], device, "dst")
    _kernel._check_sizes(num_pages, src.shape[0])
    templates = []
    for first in range(0, len(pools), _hip.MFA_COPY_MAX_POOLS):
        p = _hip.MfaCopyPagesParams()
        part = pools[first:first + _hip.MFA_COPY_MAX_POOLS]
        for i, t in enumerate(part):
            if t.shape[0] != num_pages:
                raise ValueError(f"mtlflashattn_amd: pools of {num_pages} and {t.shape[0]} pages")
            n = 1
            for size, stride in sorted(zip(t.shape[1:], t.stride()[1:]), key=lambda x: x[1]):
                if size > 1 and stride != n:
                    raise ValueError("mtlflashattn_amd: the pages of a pool must be dense in memory")
                n *= size
            if num_pages > 1 and n and t.stride(0) < n:
                raise ValueError("mtlflashattn_amd: the pages of a pool must not overlap")
            p.pool[i] = (None, t.stride(0) * t.element_size() if num_pages > 1 else 0, n * t.element_size())
        p.pools, p.pairs, p.num_pages = len(part), src.shape[0], num_pages
        templates.append(p)
    return templates, _i32(src) is src and _i32(dst) is dst
