"""A paged K/V cache held in 8 bits: writing it, attention over it, the weight that
each cached key received, and eviction by that weight.  The reference has no cache
(block_table raises, metal_flash_attn/__init__.py:130-131); kv4.py holds one in 4 bits.

Format (include/mfa.h): elements are e4m3 floats, and the 64 rows of a block (rows 64 i
.. 64 i + 63 of a page) and a head share one power of two 2^(s - 127), a byte s.  A
cache of K or V is a pair (codes, scales): float8_e4m3fn [num_pages, page_block_size,
Hkv, D] and uint8 [num_pages, page_block_size / 64, Hkv], as kv8_cache makes it.
"""
from __future__ import annotations

import torch

from . import _hip, _kernel, kv4
from ._kernel import _launch_on
from .kv4 import _i32, _plans, _remember

BLOCK = _hip.MFA_KV8_BLOCK

_KV8 = kv4._Format(8, torch.float8_e4m3fn, lambda D: D, lambda pages, page, heads, D: (pages, page // BLOCK, heads))


def kv8_cache(num_pages, page_block_size, num_heads_kv, head_dim, device="cuda"):
    """An empty 8-bit cache of K or of V: (codes, scales).

    codes: float8_e4m3fn [num_pages, page_block_size, num_heads_kv, head_dim], scales:
    uint8 [num_pages, page_block_size / 64, num_heads_kv], zeroed (rows read as 0).  In
    memory each head's rows of a page lie side by side (the heads-third shape is a view),
    which the kernels read fastest; they take any other order too.  page_block_size: a
    multiple of 64; head_dim: 32, 64, 96 or 128.
    """
    kv4._check_page_and_head(page_block_size, head_dim, _KV8)
    codes = torch.zeros(num_pages, num_heads_kv, page_block_size, head_dim, dtype=torch.uint8, device=device)
    scales = torch.zeros(num_pages, num_heads_kv, page_block_size // BLOCK, dtype=torch.uint8, device=device)
    return codes.view(torch.float8_e4m3fn).transpose(1, 2), scales.transpose(1, 2)


def kv8_append(k, v, k_cache, v_cache, cu_seqlens, cache_seqlens, block_table, return_values=False):
    """Write new rows into a paged 8-bit cache, in one launch.

    Arguments as in kv4_append: k, v [total, Hkv, D] fp16 / bf16 / fp32 rows packed
    without padding; token t of sequence b becomes row cache_seqlens[b] + t -
    cu_seqlens[b] of the sequence; lengths and page ids are read on the device (no
    synchronisation); rows behind the last column of the table or on a page id outside
    the pool are dropped, and a negative length counts as 0.  No two sequences may write
    into one block of 64 rows: a page that forked sequences share is copied
    (copy_cache_pages) before one of them writes to it.

    A block takes the smallest power of two from 2^-126 on that leaves the largest
    finite magnitude of its rows within 448 times it; elements are rounded to the
    nearest e4m3 value, ties to the even code (beyond 240 * 2^120 to that: the next would
    be infinite in bf16 and fp32); infinities and NaN become NaN.  Rows that
    a block holds already never lower its scale; where new ones raise it, the codes of
    the held rows are rounded again (exact but for the smallest ones).

    return_values=True returns (k', v') [total, Hkv, D] in k.dtype: the rows as the
    cache now holds them (of a dropped row: as a block of the call's rows alone would;
    of a token of no sequence: 0; in fp16 saturated at 65504), for attention over a
    prompt that later steps will read back from the cache.  A later append into the same
    block may round them once more.  Not differentiable: inputs that require grad raise.
    """
    return kv4._append(_KV8, k, v, k_cache, v_cache, cu_seqlens, cache_seqlens, block_table, return_values)


def flash_attn_kv8_func(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale=None, causal=False,
                        window_size=(-1, -1), softcap=0.0, alibi_slopes=None, max_seqlen_k=None,
                        return_softmax_lse=False):
    """Attention of [B, Lq, Hq, D] queries over a paged 8-bit cache: flash_attn_kv4_func
    over another format, with its arguments, masks, limits and results.

    K is exact; so is V, except on the tiles of 128 columns (sequences of more than 32
    columns; in a varlen call of more than 32 in total, of more than 16, but not where its
    sequences have 17 to 32 on average) with fp16 queries, where it is rounded to fp16 (beyond 65504 it saturates;
    scales below 2^-15 may lose bits).  The log-sum-exps are those of the probabilities before
    they are rounded.  NaN elements reach only the rows whose mask holds their key.
    """
    if torch.is_tensor(q) and q.dim() != 4:
        raise ValueError(f"mtlflashattn_amd: expected q [B,Lq,H,D], got {q.dim()}-D")
    return kv4._attend(_KV8, q, k_cache, v_cache, None, cache_seqlens, block_table, softmax_scale, causal, window_size,
                       softcap, alibi_slopes, max_seqlen_k, return_softmax_lse)


def flash_attn_varlen_kv8_func(q, k_cache, v_cache, cu_seqlens_q, cache_seqlens, block_table, softmax_scale=None,
                               causal=False, window_size=(-1, -1), softcap=0.0, alibi_slopes=None, max_seqlen_k=None,
                               return_softmax_lse=False):
    """flash_attn_kv8_func for sequences of different query counts: as
    flash_attn_varlen_kv4_func, q [total, Hq, D] packed without padding, sequence b owning
    rows [cu_seqlens_q[b], cu_seqlens_q[b + 1]); rows of no sequence come back as 0.
    Returns [total, Hq, D] and, if asked, the log-sum-exp [Hq, total].
    """
    if torch.is_tensor(q) and q.dim() != 3:
        raise ValueError(f"mtlflashattn_amd: expected q [total,H,D], got {q.dim()}-D")
    return kv4._attend(_KV8, q, k_cache, v_cache, cu_seqlens_q, cache_seqlens, block_table, softmax_scale, causal,
                       window_size, softcap, alibi_slopes, max_seqlen_k, return_softmax_lse)


def _check_weights(weights, codes, device):
    if not torch.is_tensor(weights) or weights.dtype != torch.float32 or tuple(weights.shape) != tuple(codes.shape[:3]):
        raise ValueError("mtlflashattn_amd: weights must be an fp32 [num_pages, page_block_size, Hkv] tensor of the cache's "
                         "pages and heads")
    if weights.device != device:
        raise ValueError(f"mtlflashattn_amd: tensors on different devices ({device} vs {weights.device})")
    kv4._check_written(weights)


def _weight_strides(p, weights):
    p.weight_page_stride, p.weight_row_stride, p.weight_head_stride = (
        s if n > 1 else 0 for s, n in zip(weights.stride(), weights.shape))


def kv8_key_weights(q, k_cache, softmax_lse, weights, cache_seqlens, block_table, cu_seqlens_q=None, softmax_scale=None,
                    causal=False, window_size=(-1, -1), softcap=0.0, alibi_slopes=None, max_seqlen_k=None):
    """Add the attention weight that each cached key received from the queries of a step.

    q, cache_seqlens, block_table and the options are those of the step's attention call
    (flash_attn_kv8_func, or flash_attn_varlen_kv8_func with cu_seqlens_q), softmax_lse
    the log-sum-exps it returned, fp32 [B, Hq, Lq] ([Hq, total]).  weights: fp32
    [num_pages, page_block_size, Hkv], a pool that is addressed with the cache's block
    table and written in place: of key j of sequence b and K/V head h
      weights = (j < Lk - Lq ? weights : 0) + sum of softmax(...)[i, j] over the sequence's
                query rows i and the query heads of h,
    so keys before the queries' own rows add to what they had and the queries' own, new
    in this step, start from 0: where every row of a sequence has been a query of some call
    the pool needs no clearing.  What a row's mask leaves out adds nothing, and sequences
    without queries keep their weights.  Sequences with queries must not share pages (a
    fork's weights need pages of their own).  The weights that the last rows of a prompt
    alone give come from a call with those rows and their log-sum-exps: then only those
    rows' own keys start from 0, and the others add to what their pages held, from other
    sequences too, so clear the pages of such a prompt first (weights[pages] = 0).

    A weight is as exact as the log-sum-exps are (those of the attention calls: 1e-4).
    Sums in fp32, every key by one owner in an order that sizes and lengths alone
    decide; no synchronisation.  Any strides; each head's rows of a page side by side are
    read fastest.  Not differentiable: tensors that require grad raise.
    """
    softmax_scale, window_size, softcap, max_seqlen_k = kv4._numbers(softmax_scale, window_size, softcap, alibi_slopes,
                                                                     max_seqlen_k)
    try:
        kc, ks = k_cache
        varlen = cu_seqlens_q is not None
        key = ("weights", q.shape, q.stride(), q.dtype, q.device, kc.shape, kc.stride(), kc.dtype, kc.device,
               ks.shape, ks.stride(), ks.dtype, ks.device, softmax_lse.shape, softmax_lse.dtype, softmax_lse.device,
               weights.shape, weights.stride(), weights.dtype, weights.device,
               cache_seqlens.shape, cache_seqlens.stride(), cache_seqlens.dtype, cache_seqlens.device,
               block_table.shape, block_table.stride(), block_table.dtype, block_table.device,
               varlen and (cu_seqlens_q.shape, cu_seqlens_q.stride(), cu_seqlens_q.dtype, cu_seqlens_q.device),
               alibi_slopes is not None and (alibi_slopes.shape, alibi_slopes.device),
               softmax_scale, bool(causal), window_size, softcap, max_seqlen_k)
    except (AttributeError, TypeError, ValueError):
        raise kv4._not_tensors(k_cache, k_cache, _KV8) from None
    _kernel._check_no_tangent(q, softmax_lse, weights)
    if _kernel._needs_grad(q, softmax_lse, weights):
        raise NotImplementedError("mtlflashattn_amd: kv8_key_weights is not differentiable; run it under torch.no_grad() or "
                                  "on detached tensors")
    template, direct = _plans.get(key) or _remember(key, _weights_plan(
        q, k_cache, softmax_lse, weights, cu_seqlens_q, cache_seqlens, block_table, softmax_scale, causal, window_size,
        softcap, alibi_slopes, max_seqlen_k))
    p = _hip.MfaKv8WeightsParams.from_buffer_copy(template)
    f = p.fwd
    qp = q.data_ptr()
    if not direct or qp & 15:
        q, cache_seqlens = _kernel._abi_operand(q), _i32(cache_seqlens)
        qp = q.data_ptr()
        strides = [s if n > 1 else 0 for s, n in zip(q.stride(), q.shape)]
        f.q_batch_stride, f.q_seq_stride, f.q_head_stride = (0, *strides[:2]) if varlen else strides[:3]
        if varlen:
            cu_seqlens_q = _i32(cu_seqlens_q)
    if _kernel._check_pages_enabled():
        kv4._check_pages(block_table, cache_seqlens.clamp(max=f.max_seqlen_k), kc.shape[1], kc.shape[0])
    softmax_lse = softmax_lse.contiguous()
    if varlen:
        f.cu_seqlens_q = cu_seqlens_q.data_ptr()
    if alibi_slopes is not None:
        slopes, f.alibi_batch_stride = _kernel._alibi_arg(alibi_slopes, f.batch, f.heads_q, q.device)
        f.alibi_slopes = slopes.data_ptr()
    f.q, f.softmax_lse, f.cache_seqlens = qp, softmax_lse.data_ptr(), cache_seqlens.data_ptr()
    kv4._cache_pointers(f.cache, kc, ks, kc, ks, block_table)
    p.weights = weights.data_ptr()
    _launch_on(q.device, _hip.kv8_weights, p)
    kv4._written((weights,))


def _weights_plan(q, k_cache, softmax_lse, weights, cu_q, cache_seqlens, block_table, softmax_scale, causal, window_size,
                  softcap, alibi_slopes, max_seqlen_k):
    """(parameters without data pointers, whether the tensors are used in place) of a call."""
    if q.dim() != (4 if cu_q is None else 3):
        raise ValueError(f"mtlflashattn_amd: expected q {'[B,Lq,H,D]' if cu_q is None else '[total,H,D]'}, got {q.dim()}-D")
    p = _hip.MfaKv8WeightsParams()
    p.fwd = kv4._attend_params(_KV8, q, k_cache, k_cache, cu_q, cache_seqlens, block_table, softmax_scale, causal,
                               window_size, softcap, alibi_slopes, max_seqlen_k)
    p.fwd.o_batch_stride = p.fwd.o_seq_stride = p.fwd.o_head_stride = 0
    shape = (q.shape[1], q.shape[0]) if cu_q is not None else (q.shape[0], q.shape[2], q.shape[1])
    if softmax_lse.dtype != torch.float32 or tuple(softmax_lse.shape) != shape:
        raise ValueError(f"mtlflashattn_amd: softmax_lse must be the fp32 log-sum-exps {shape} of the attention call")
    if softmax_lse.device != q.device:
        raise ValueError(f"mtlflashattn_amd: tensors on different devices ({q.device} vs {softmax_lse.device})")
    _check_weights(weights, k_cache[0], q.device)
    _weight_strides(p, weights)
    return p, kv4._attend_direct(q, cu_q, cache_seqlens)


def kv8_evict(k_cache, v_cache, weights, cache_seqlens, block_table, budget, recent, max_seqlen_k=None):
    """Bring the sequences of a paged 8-bit cache down to `budget` rows, by weight.

    Of every K/V head of a sequence with more than `budget` rows (cache_seqlens, int32
    [B]), the last min(recent, budget) rows and the heaviest of the others stay (weights
    as kv8_key_weights accumulates them; ties go to the lower row, NaN stands above
    everything), `budget` in all.  They become rows 0 .. budget - 1 of the sequence in
    their order, their weights with them; heads keep different rows.  A block of 64 rows
    whose rows all stay where they are is left as it is; any other takes a new scale by
    kv8_append's rule for a block without rows, from the values its rows have.  Rows from
    `budget` on keep their codes and weights: their pages can be given back.  Shorter
    sequences do not change.  Returns the new lengths, int32 [B]: min(rows, budget).

    Row numbers are what masks, windows and ALiBi count from here on: keys keep the
    rotation they were written with, and the last `recent` rows stay the last.

    Lengths and page ids are read on the device (no synchronisation: a call can be
    captured into a graph).  A sequence has at most max_seqlen_k rows (None: as many as
    the table names); a tight bound keeps the selection short and, where the budget is
    not below it, the workspace empty.  A row on a page id outside the pool reads as
    zeros with weight 0.  The pool has less than 2^31 rows.  No two sequences may share a page that
    changes; k_cache and v_cache are two caches.
    """
    budget, recent = int(budget), int(recent)
    max_seqlen_k = None if max_seqlen_k is None else int(max_seqlen_k)
    try:
        (kc, ks), (vc, vs) = k_cache, v_cache
        key = ("evict", kc.shape, kc.stride(), kc.dtype, kc.device, ks.shape, ks.stride(), ks.dtype, ks.device,
               vc.shape, vc.stride(), vc.dtype, vc.device, vs.shape, vs.stride(), vs.dtype, vs.device,
               weights.shape, weights.stride(), weights.dtype, weights.device,
               cache_seqlens.shape, cache_seqlens.stride(), cache_seqlens.dtype, cache_seqlens.device,
               block_table.shape, block_table.stride(), block_table.dtype, block_table.device,
               budget, recent, max_seqlen_k)
    except (AttributeError, TypeError, ValueError):
        raise kv4._not_tensors(k_cache, v_cache, _KV8) from None
    _kernel._check_no_tangent(weights)
    if _kernel._needs_grad(weights):
        raise NotImplementedError("mtlflashattn_amd: kv8_evict is not differentiable; run it under torch.no_grad() or on "
                                  "detached weights")
    template, nbytes = _plans.get(key) or _remember(key, _evict_plan(k_cache, v_cache, weights, cache_seqlens, block_table,
                                                                     budget, recent, max_seqlen_k))
    cache_seqlens = _i32(cache_seqlens)
    if _kernel._check_pages_enabled():
        kv4._check_pages(block_table, cache_seqlens.clamp(max=template.max_seqlen_k), kc.shape[1], kc.shape[0])
    p = _hip.MfaKv8EvictParams.from_buffer_copy(template)
    device = kc.device
    new_seqlens = torch.empty_like(cache_seqlens)
    p.cache_seqlens, p.new_seqlens, p.weights = cache_seqlens.data_ptr(), new_seqlens.data_ptr(), weights.data_ptr()
    kv4._cache_pointers(p.cache, kc, ks, vc, vs, block_table)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _launch_on(device, _hip.kv8_evict, p, None if ws is None else ws.data_ptr(), nbytes)
    kv4._written((kc, ks, vc, vs, weights))
    return new_seqlens


def _evict_plan(k_cache, v_cache, weights, cache_seqlens, block_table, budget, recent, max_seqlen_k):
    """(parameters without data pointers, workspace bytes) of a call."""
    codes = k_cache[0]
    _kernel._check_device(codes)
    if codes.dim() != 4:
        raise ValueError("mtlflashattn_amd: k_cache: codes must be 4-D")
    Hkv, D = codes.shape[2:]
    if D not in (32, 64, 96, 128):
        raise NotImplementedError(f"mtlflashattn_amd: head_dim {D} of an 8-bit cache must be 32, 64, 96 or 128")
    kv4._check_cache(k_cache, D, Hkv, codes.device, "k_cache", _KV8)
    kv4._check_cache(v_cache, D, Hkv, codes.device, "v_cache", _KV8)
    if k_cache[0].shape != v_cache[0].shape:
        raise ValueError("mtlflashattn_amd: k_cache and v_cache differ in pages")
    if Hkv == 0:
        raise ValueError("mtlflashattn_amd: a cache without heads")
    kv4._check_written(*k_cache, *v_cache)
    _check_weights(weights, codes, codes.device)
    batch = cache_seqlens.shape[0] if cache_seqlens.dim() == 1 else 0
    kv4._check_ints(cache_seqlens, batch, codes.device, "cache_seqlens")
    kv4._check_table(block_table, batch, codes.device)
    if budget < 0 or recent < 0 or (max_seqlen_k is not None and max_seqlen_k < 0):
        raise ValueError("mtlflashattn_amd: budget, recent and max_seqlen_k must be >= 0")
    p = _hip.MfaKv8EvictParams()
    kv4._cache_struct(p.cache, k_cache, v_cache, block_table)
    _kernel._check_sizes(batch, Hkv)
    _weight_strides(p, weights)
    p.batch, p.heads_kv, p.head_dim = batch, Hkv, D
    cap = block_table.shape[1] * codes.shape[1]
    p.max_seqlen_k = cap if max_seqlen_k is None else min(max_seqlen_k, cap)
    if p.max_seqlen_k == 0:  # (0 means no bound to the library)
        p.cache.max_pages = 0
    # (no more than the longest sequence: ctypes would cut larger numbers off)
    p.budget, p.recent = min(budget, _kernel._INT32_MAX), min(recent, _kernel._INT32_MAX)
    # placeholders: sizing the workspace reads no tensor
    sized = _hip.MfaKv8EvictParams.from_buffer_copy(p)
    sized.weights = sized.cache_seqlens = sized.new_seqlens = sized.cache.block_table = 256
    sized.cache.k.codes = sized.cache.k.scales = sized.cache.v.codes = sized.cache.v.scales = 256
    return p, _hip.kv8_evict_workspace_bytes(sized)
