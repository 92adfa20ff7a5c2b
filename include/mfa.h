/*
 * mfa.h -- C ABI of the MI355X (gfx950) flash-attention library
 * (libmtlfa_hip.so, built from the sources in mtlflashattn_amd/csrc).
 *
 * This is the drop-in boundary that replaces the reference's per-tier Metal
 * launch calls.  In the reference the Python launcher binds a JIT-compiled
 * Metal library and calls one kernel per tier with device buffers Q, K, V, O
 * plus three small parameter tensors:
 *   SH  int32 shape vector   [B, Hq, Hkv, Lq, Lk, causal(, Lkp)]
 *   PR  fp32 parameter vector [scale, softcap, win_left, win_right, alibi_on]
 *   AL  fp32 [B*Hq] ALiBi slopes (or a 1-element dummy)
 * (metal_flash_attn/_kernel.py:1309-1312 `lib.flash_attn_fwd_v2r_dtype(...)`,
 *  :1333-1337, :1368-1373, :1397-1401, :1416-1419; SH/PR/AL semantics at
 *  :1221-1272).  Here the same information travels in one POD struct, passed
 * by pointer and copied by value into the kernel arguments, so no per-call
 * device parameter tensors exist at all.
 *
 * Contract:
 *  - Every entry point is stateless and re-entrant.  mfa_fwd only enqueues
 *    work on `stream` (a hipStream_t, e.g. torch.cuda.current_stream()
 *    .cuda_stream); it never synchronizes and never allocates.
 *  - Return value 0 = success, negative = error; the message is available
 *    from mfa_last_error() on the same thread.
 *  - All pointers are device pointers.  The head dimension must be
 *    contiguous (element stride 1) in q, k, v and o; every other stride is an
 *    element stride and may describe any layout (views, packed qkv,
 *    heads-second or heads-third), as long as q, k, v and o start at 16-byte
 *    aligned addresses and each of their strides is a multiple of 16 bytes
 *    (8 elements of 16 bits, 4 of fp32); other layouts return
 *    MFA_ERR_INVALID.
 */
#ifndef MTLFA_MFA_H
#define MTLFA_MFA_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MFA_ABI_VERSION 7

/* element types (dtype_in / dtype_out) */
#define MFA_DTYPE_F16 0
#define MFA_DTYPE_BF16 1
#define MFA_DTYPE_F32 2

/* error codes */
#define MFA_OK 0
#define MFA_ERR_INVALID -1     /* bad argument (shape, stride, alignment, dtype) */
#define MFA_ERR_UNSUPPORTED -2 /* valid request this build does not implement */
#define MFA_ERR_LAUNCH -3      /* the HIP runtime refused the launch */

#define MFA_MAX_HEAD_DIM 128

/* tile_hint values (bf16/fp16 only; fp32 has two kernels of the same bits, the
 * library's choice).  Sequences of one
 * query row always run the single-row kernel, which computes the query heads
 * of a K/V head together and whose probabilities carry two 16-bit terms; the
 * hint applies to the rest. */
#define MFA_TILE_AUTO 0     /* library's choice */
#define MFA_TILE_256 1      /* 256-row tiles, 4 wavefronts */
#define MFA_TILE_PINGPONG 2 /* ping-pong tiles, 8 wavefronts: 512 rows at head_dim <= 64,
                               256 rows at head_dim 97..128 (not 65..96) */
#define MFA_TILE_PINGPONG256 3 /* 256-row ping-pong tiles, 8 wavefronts (head_dim <= 64 or
                                  97..128); the library's choice at head_dim <= 64 for causal
                                  calls whose 512-row tiles would leave CUs idle while the
                                  heaviest tiles finish */

/*
 * Forward parameters.  Replaces the SH/PR/AL buffers of the reference
 * (metal_flash_attn/_kernel.py:1221-1272) and the heads-second tensor
 * arguments of flash_attn_forward (metal_flash_attn/_kernel.py:1052-1053).
 *
 * Dense mode (cu_seqlens_q == NULL):
 *   q [batch, seqlen_q, heads_q, head_dim] addressed through the q_*_stride
 *   fields, likewise k/v [batch, seqlen_k, heads_kv, head_dim] and
 *   o [batch, seqlen_q, heads_q, head_dim].
 * Varlen mode (cu_seqlens_q != NULL, metal_flash_attn/__init__.py:102-183):
 *   q [total_q, heads_q, head_dim], k/v [total_k, heads_kv, head_dim],
 *   o [total_q, heads_q, head_dim]; sequence i owns tokens
 *   [cu_seqlens_q[i], cu_seqlens_q[i+1]) of q/o and
 *   [cu_seqlens_k[i], cu_seqlens_k[i+1]) of k/v.  `batch` is the number of
 *   sequences, the *_batch_stride fields are ignored, and seqlen_q/seqlen_k
 *   must hold max_seqlen_q/max_seqlen_k (upper bounds of every sequence).
 *   The kernel and tile choice is made from these bounds (e.g. seqlen_k <= 32
 *   under many query rows selects a kernel that holds one 32-key block per
 *   sequence), so a bound below a sequence's real length gives wrong
 *   results for that sequence; it is not detected on the device.
 *
 * Masking/bias (metal_flash_attn/_kernel.py:32-87): for query row i of a
 * sequence with Lq queries and Lk keys, center = i + (Lk - Lq); key j is
 * valid iff j <= center (causal), j >= center - window_left (window_left >= 0)
 * and j <= center + window_right (window_right >= 0).  Scores are
 * s = scale * q.k; s = softcap * tanh(s / softcap) when softcap > 0;
 * s -= slope * |center - j| when alibi_slopes != NULL, with
 * slope = alibi_slopes[b * alibi_batch_stride + h] (alibi_batch_stride 0 for
 * per-head [Hq] slopes, Hq for [B, Hq]).  Rows with no valid key produce 0.
 */
typedef struct mfa_fwd_params {
    const void* q;
    const void* k;
    const void* v;
    void* o;

    int64_t q_batch_stride, q_seq_stride, q_head_stride;
    int64_t k_batch_stride, k_seq_stride, k_head_stride;
    int64_t v_batch_stride, v_seq_stride, v_head_stride;
    int64_t o_batch_stride, o_seq_stride, o_head_stride;

    int32_t batch;
    int32_t heads_q;
    int32_t heads_kv;
    int32_t seqlen_q;
    int32_t seqlen_k;
    int32_t head_dim;

    const int32_t* cu_seqlens_q; /* NULL = dense */
    const int32_t* cu_seqlens_k; /* NULL = dense */

    float scale;
    float softcap;        /* 0 = off; must be >= 0 */
    int32_t window_left;  /* -1 = unbounded */
    int32_t window_right; /* -1 = unbounded */
    int32_t causal;       /* 0/1, bottom-right aligned */

    const float* alibi_slopes; /* NULL = off; fp32 */
    int32_t alibi_batch_stride;

    int32_t dtype_in;  /* MFA_DTYPE_* of q, k and v */
    int32_t dtype_out; /* == dtype_in, or MFA_DTYPE_F32 (full-precision output) */
    int32_t tile_hint; /* MFA_TILE_AUTO (0); the others force a bf16/fp16 kernel
                          (tests and tuning; results meet the same bars either
                          way) for every sequence of more than one query row */

    /* Softmax log-sum-exp output (optional; the reference raises for it,
     * metal_flash_attn/__init__.py:49-50).  lse = ln(sum_j exp(s_j)) over the
     * row's valid keys, s the transformed score above (natural-log units, as
     * CUDA flash-attn's softmax_lse), -inf for a row with no valid key.  fp32,
     * query rows contiguous: dense lse[b * lse_batch_stride + h *
     * lse_head_stride + i]; varlen lse[h * lse_head_stride + cu_seqlens_q[b]
     * + i] (lse_batch_stride ignored; [heads_q, total_q] when
     * lse_head_stride = total_q). */
    float* softmax_lse; /* NULL = not written */
    int64_t lse_batch_stride;
    int64_t lse_head_stride;

    /* Paged K/V (optional; the reference raises for block_table,
     * metal_flash_attn/__init__.py:130-131).  k and v are
     * [num_pages, page_block_size, heads_kv, head_dim] addressed through
     * k_batch_stride/v_batch_stride (page stride), *_seq_stride and
     * *_head_stride; key j of sequence b is row j % page_block_size of page
     * block_table[b * block_table_batch_stride + j / page_block_size].  The
     * key count of sequence b is seqlen_k (dense) or cu_seqlens_k[b+1] -
     * cu_seqlens_k[b] (varlen; the start offsets are not used for k/v).
     * page_block_size is a positive multiple of 256; a page id outside
     * [0, num_pages) reads as zeros, never out of bounds, but its keys are
     * not masked: they score 0 and take weight in the softmax, so the rows
     * that see them come out wrong (callers validate their tables).  Paged
     * calls run on the 256-row and fp32 kernels: MFA_TILE_PINGPONG with a
     * block_table is MFA_ERR_UNSUPPORTED. */
    const int32_t* block_table; /* NULL = contiguous k/v */
    int64_t block_table_batch_stride;
    int32_t page_block_size;
    int32_t num_pages;

    /* Varlen calls, optional (0 = unknown; ABI 7): 1 when the caller knows
     * that no sequence has exactly one query row.  A varlen call otherwise
     * adds a launch of the single-row kernel for such sequences (the main
     * launch leaves them to it); 1 skips that launch, so a sequence of one
     * query row would keep its o rows (and lse) unwritten.  Ignored by dense
     * calls.  No counterpart in the reference. */
    int32_t varlen_no_single_rows;
} mfa_fwd_params;

/* Launch geometry of one mfa_fwd call (for profiling/roofline reports). */
typedef struct mfa_launch_info {
    int32_t grid_x;          /* workgroups launched */
    int32_t block_x;         /* threads per workgroup */
    int32_t rows_per_block;  /* query rows per workgroup tile */
    int32_t keys_per_block;  /* keys per K/V block */
    int32_t lds_bytes;       /* LDS bytes per workgroup */
    char kernel_name[96];    /* short name of the kernel instantiation */
} mfa_launch_info;

/* ABI version of the loaded library (MFA_ABI_VERSION).  No counterpart in
 * the reference (its kernels are JIT-compiled from source strings). */
int mfa_abi_version(void);

/* Message of the last failed call on this thread ("" if none).  Replaces
 * the RuntimeError strings of the reference's forced-tier checks
 * (metal_flash_attn/_kernel.py:1083-1140). */
const char* mfa_last_error(void);

/* 1 if mfa_fwd implements (dtype_in, head_dim) on this build, else 0.
 * Replaces the eligibility probes _v1_eligible/_v2_dtype_eligible
 * (metal_flash_attn/_kernel.py:928-936, :896-912). */
int mfa_supported(int32_t dtype_in, int32_t head_dim);

/* Enqueue the attention forward on `stream` (hipStream_t; NULL = default
 * stream).  Replaces the tier launchers _flash_v2r_dtype / _flash_v2_dtype /
 * _flash_v2 / _flash_v1 / _flash_v0 (metal_flash_attn/_kernel.py:1288-1420)
 * and their kernel calls. */
int mfa_fwd(const mfa_fwd_params* params, void* stream);

/* Fill *info with the geometry mfa_fwd would launch for `params`; enqueues
 * nothing.  No counterpart in the reference. */
int mfa_fwd_launch_info(const mfa_fwd_params* params, mfa_launch_info* info);

/* sizeof(mfa_fwd_params) as compiled into the library, so FFI bindings can
 * check their struct mirror.  No counterpart in the reference. */
int mfa_params_size(void);

/* Split-KV forward for decode-like shapes (few query rows, long key ranges):
 * the key range of every sequence is cut into chunks of `split_keys` keys,
 * workgroups compute the chunks in parallel into a caller-provided
 * workspace, and a second kernel merges them (log-sum-exp weighting).  No
 * counterpart in the reference, whose Metal kernels run one threadgroup per
 * query tile over all keys; these calls are the build's addition for
 * HBM-bound shapes.  bf16/fp16 only; results meet the same bars as mfa_fwd.
 *
 * mfa_fwd_split_request: the split_keys with which mfa_fwd_splitkv (and a
 * workspace of mfa_fwd_workspace_bytes) launches `params` fastest, 0 = use
 * mfa_fwd.  It is mfa_fwd_split_keys, except for sequences of one query row
 * (seqlen_q = 1): there it is non-zero exactly where a workspace is used (also
 * at 2048 keys and below, where mfa_fwd_split_keys is 0).  For a varlen call
 * that may mix such sequences with longer ones (varlen_no_single_rows 0) and
 * whose longer ones are not split, it is a chunk of seqlen_k keys or more
 * wherever the single rows would use a workspace: the longer ones then run as
 * in mfa_fwd.
 * mfa_fwd_split_keys: the chunk of sequences of several query rows, 0 = none.
 * It is 2048 (above 2M keys the next multiple of 256 that makes at most 1024
 * chunks) when seqlen_q (the longest query for varlen) is at most 256 and
 * seqlen_k exceeds 2048, else 0 (fp32 and forced ping-pong tiles: 0); a
 * dense call with batch > 1 and batch * heads_q >= 512 gets 0 too (the
 * single pass already fills the chip).  For varlen and batch = 1 calls the
 * choice depends on the lengths only, so a sequence is chunked alike alone or
 * inside a varlen batch (bit-identical rows either way).
 * mfa_fwd_workspace_bytes: device bytes mfa_fwd_splitkv needs for this call
 * and chunk size (0 for split_keys 0 or an empty problem; < 0 on error).
 * mfa_fwd_splitkv: enqueue both kernels on `stream`; `workspace` is a
 * 256-byte aligned device buffer of at least that many bytes, owned by the
 * caller and reused only after the call's kernels ran (stream order).
 * split_keys must be 0 (same as mfa_fwd) or a positive multiple of 64 (of
 * 256 with a block_table).  Sequences of one query row are chunked by the
 * library, from their own key count, in every entry point alike: there
 * split_keys != 0 only offers the workspace (0 bytes where a workgroup per
 * sequence and K/V head walking all chunks is faster), and the results of
 * mfa_fwd and mfa_fwd_splitkv are the same bits.  In a call that mixes them with
 * longer sequences their partials follow the longer ones' in the workspace; a
 * workspace of the longer ones' size (as reported with varlen_no_single_rows 1)
 * is taken too, the single rows are then not split.  softmax_lse and block_table work as in mfa_fwd. */
int32_t mfa_fwd_split_request(const mfa_fwd_params* params);
int32_t mfa_fwd_split_keys(const mfa_fwd_params* params);
int64_t mfa_fwd_workspace_bytes(const mfa_fwd_params* params, int32_t split_keys);
int mfa_fwd_splitkv(const mfa_fwd_params* params, int32_t split_keys, void* workspace, int64_t workspace_bytes,
                    void* stream);

/* Size of the static scratch array behind mfa_fwd_splitkv_static (64 MiB per
 * GPU, held from the library's first use on that GPU until the process
 * ends). */
#define MFA_STATIC_SCRATCH_BYTES (64LL << 20)

/* mfa_fwd_splitkv without a caller workspace, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  No counterpart in the reference.  The
 * split-KV partials go to a file-scope device array of
 * MFA_STATIC_SCRATCH_BYTES bytes (one per GPU).  Which calls are taken depends
 * on the request alone: partials of ceil(seqlen_k / split_keys) * batch *
 * heads_q * seqlen_q rows of head_dim (padded to 32, 64, 96 or 128) floats, and
 * a float per row rounded up to 256 bytes, have to fit, else MFA_ERR_INVALID
 * with a message -- also for single rows, whose own chunks count differently
 * and which are walked, not refused, where theirs do not fit.  Allocates nothing (no hipMalloc, hipFree or allocating library
 * call); the first call on a GPU looks up the array's device address once.
 * Same kernels, chunks and results as mfa_fwd_splitkv (bit for bit);
 * split_keys 0 behaves as mfa_fwd.  Every call on one GPU shares that GPU's
 * array: calls that overlap on one GPU (different streams, or host threads
 * without ordering between them) race and must be serialised by the caller;
 * calls in one stream are ordered and safe.  The array keeps the last call's
 * partials; nothing needs clearing (each call writes every partial it reads). */
int mfa_fwd_splitkv_static(const mfa_fwd_params* params, int32_t split_keys, void* stream);

/*
 * Backward pass (gradients of q, k, v).  No counterpart in the reference,
 * which is forward-only (metal_flash_attn/__init__.py:3-4, README.md:159-161;
 * training callers fall back to other attention).  Same masking and bias
 * semantics as the forward; the forward's O and softmax_lse are inputs:
 *   P = exp(s - lse), dV = P^T dO, dP = dO V^T, Dsum = rowsum(dO * O),
 *   dS = P * (dP - Dsum) [* (1 - tanh^2) under softcap], dQ = scale dS K,
 *   dK = scale dS^T Q.
 * With grouped-query heads, dK/dV of a K/V head sum over its query heads.
 * Deterministic (no atomics): one kernel owns each dK/dV block and loops over
 * every query of its K/V head; another owns each dQ block.
 * fp32 (dtype_in = MFA_DTYPE_F32: q, k, v, o, dout and the gradients fp32)
 * runs fp32 kernels on the fp32 matrix cores with the fp32 forward's score
 * transform (strides then multiples of 4 elements; the workspace holds the row
 * sums only).
 */
typedef struct mfa_bwd_params {
    /* q, k, v, o (the forward output), shapes, strides, masks and biases as
     * in the forward; fwd.softmax_lse (+ strides) is the forward's lse and
     * required; fwd.block_table must be NULL; fwd.tile_hint is ignored;
     * fwd.dtype_out is o's dtype and must equal dtype_in. */
    mfa_fwd_params fwd;
    const void* dout; /* dL/dO, laid out like o (its own strides), o's dtype */
    int64_t do_batch_stride, do_seq_stride, do_head_stride;
    void* dq;         /* laid out like q */
    int64_t dq_batch_stride, dq_seq_stride, dq_head_stride;
    void* dk;         /* laid out like k */
    int64_t dk_batch_stride, dk_seq_stride, dk_head_stride;
    void* dv;         /* laid out like v */
    int64_t dv_batch_stride, dv_seq_stride, dv_head_stride;
    int32_t dtype_grad; /* dtype of dq/dk/dv: dtype_in or MFA_DTYPE_F32 */
    int32_t reserved;
    /* Optional gradient of the loss with respect to softmax_lse (fp32, same
     * layout and strides as fwd.softmax_lse; NULL = zero).  Since
     * d lse_i / d s_ij = P_ij, it enters as Dsum_i - dlse_i. */
    const float* dlse;
} mfa_bwd_params;

/* 1 if mfa_bwd implements (dtype_in, head_dim): bf16/fp16/fp32, head_dim a
 * multiple of 8 up to MFA_MAX_HEAD_DIM. */
int mfa_bwd_supported(int32_t dtype_in, int32_t head_dim);
/* Device workspace mfa_bwd needs, 0 for an empty problem, < 0 on error: the
 * fp32 row sums Dsum, and with grouped-query heads (heads_q > heads_kv) the
 * fp32 dK/dV partials of each query head (2 * heads_q * batch * seqlen_k *
 * padded head_dim * 4 bytes) when they fit in 2 GiB -- the query heads of a
 * K/V head then run in parallel workgroups and are summed in head order. */
int64_t mfa_bwd_workspace_bytes(const mfa_bwd_params* params);
/* Enqueue the backward kernels on `stream`; `workspace`: 256-byte aligned
 * device buffer of at least mfa_bwd_workspace_bytes bytes, owned by the
 * caller.  Never synchronizes, never allocates. */
int mfa_bwd(const mfa_bwd_params* params, void* workspace, int64_t workspace_bytes, void* stream);
int mfa_bwd_params_size(void);

/*
 * Merge of attention partials of the same queries over disjoint key sets
 * (context-parallel shards, cache + new tokens).  No counterpart in the
 * reference.  Part i holds o [batch, seqlen, heads, head_dim] (16-byte
 * aligned, head dim contiguous, element strides in multiples of 16 bytes) and
 * its log-sum-exp lse [batch, heads, seqlen] (fp32, any element strides).
 *   lse_out = ln(sum_i exp(lse_i)), out = sum_i exp(lse_i - lse_out) o_i,
 * both contiguous ([batch, seqlen, heads, head_dim] in `dtype`, the parts'
 * element type, and [batch, heads, seqlen] fp32); a row whose merged lse is
 * infinite (no key in any part) gets weights of 0.  Sums in fp32, in part
 * order.  head_dim is a multiple of 16 bytes.  Enqueues one kernel on
 * `stream`; never synchronizes, never allocates.
 */
#define MFA_MERGE_MAX_PARTS 16
typedef struct mfa_merge_part {
    const void* o;
    const float* lse;
    int64_t o_batch_stride, o_seq_stride, o_head_stride;
    int64_t lse_batch_stride, lse_head_stride, lse_seq_stride;
} mfa_merge_part;
typedef struct mfa_merge_params {
    mfa_merge_part part[MFA_MERGE_MAX_PARTS];
    void* out;
    float* lse_out;
    int32_t parts;
    int32_t dtype; /* MFA_DTYPE_* */
    int32_t batch, seqlen, heads, head_dim;
} mfa_merge_params;
int mfa_merge(const mfa_merge_params* params, void* stream);
int mfa_merge_params_size(void);

/*
 * Paged 4-bit K/V cache.  No counterpart in the reference.
 *
 * K and V are pools of pages, [num_pages, page_block_size, heads_kv, ...], held
 * as code and scale bytes: a row of one head has head_dim / 2 code bytes and
 * head_dim / 32 scale bytes, both contiguous.  32 consecutive elements share the
 * power of two 2^(s - 127) of their scale byte s (255: all NaN); element 2i is
 * the low half and element 2i + 1 the high half of code byte i, each a 4-bit
 * float with a sign bit, two exponent bits and one mantissa bit (magnitudes 0,
 * 0.5, 1, 1.5, 2, 3, 4, 6).  Page, row and head strides are in bytes, any order,
 * row and head strides >= 0 (each head's rows of a page side by side read
 * fastest); codes start at 16-byte aligned addresses with strides that are
 * multiples of 16 bytes, scales have none to keep.
 * Row j of sequence b is row j % page_block_size of page
 * block_table[b * block_table_batch_stride + j / page_block_size];
 * page_block_size is a multiple of 64, and max_pages the columns of the table.
 * Page ids are read on the device: an id outside [0, num_pages) reads as zeros
 * and drops what is written, never out of bounds.
 */
typedef struct mfa_kv4_pool {
    uint8_t* codes;
    uint8_t* scales;
    int64_t code_page_stride, code_row_stride, code_head_stride;
    int64_t scale_page_stride, scale_row_stride, scale_head_stride;
} mfa_kv4_pool;
typedef struct mfa_kv4_cache {
    mfa_kv4_pool k, v;
    const int32_t* block_table;
    int64_t block_table_batch_stride;
    int32_t max_pages, page_block_size, num_pages;
    int32_t reserved;
} mfa_kv4_cache;

/*
 * New rows into the cache.  k and v are [total, heads_kv, head_dim] of `dtype`
 * (16-byte aligned, strides multiples of 16 bytes, head dim contiguous); token t
 * of sequence b, cu_seqlens[b] <= t < cu_seqlens[b + 1], becomes row
 * cache_seqlens[b] + t - cu_seqlens[b].  A row outside the table, or whose page
 * id is outside the pool, is dropped, as are tokens of no sequence; two tokens
 * must not share a row.  The scale of 32 elements is the smallest power of two
 * (2^-127 at least) that leaves them within 7 times it, so that none is off by
 * more than half a step; elements are rounded to the nearest value, ties to the
 * even code, and a group that holds an infinity or NaN becomes NaN.
 * k_values / v_values (optional, both or none): what the cache now holds for
 * every token (what it would, for one that is dropped), contiguous [total,
 * heads_kv, head_dim] of `dtype`.
 * head_dim: a multiple of 32 up to MFA_MAX_HEAD_DIM.  One kernel; never
 * synchronizes, never allocates.
 */
typedef struct mfa_kv4_append_params {
    mfa_kv4_cache cache;
    const void* k;
    const void* v;
    int64_t k_token_stride, k_head_stride, v_token_stride, v_head_stride; /* elements */
    void* k_values;
    void* v_values;
    const int32_t* cu_seqlens;    /* [batch + 1] */
    const int32_t* cache_seqlens; /* [batch], rows already held */
    int32_t batch, total, heads_kv, head_dim;
    int32_t dtype; /* MFA_DTYPE_* of k, v and the values */
} mfa_kv4_append_params;
int mfa_kv4_append(const mfa_kv4_append_params* params, void* stream);
int mfa_kv4_append_params_size(void);

/*
 * Attention over the cache: the forward of mfa_fwd (masks, soft-cap, ALiBi,
 * grouped-query heads and softmax_lse as there) with K and V from the cache.
 * Sequence b has min(cache_seqlens[b], max_seqlen_k, what the table can name, 2^31 -
 * 256) keys, read on the device; max_seqlen_k 0 leaves the bound out.  Queries: q
 * [batch, seqlen_q, heads_q, head_dim], or with cu_seqlens_q q [total_q, heads_q,
 * head_dim], sequence b owning tokens [cu_seqlens_q[b], cu_seqlens_q[b + 1])
 * (tokens of no sequence get 0, lse -inf).  The query rows are the last
 * positions of their sequence.  q and o: fp16 or bf16, 16-byte aligned, strides
 * multiples of 8 elements.  head_dim: 32, 64, 96 or 128.  A NaN of V reaches only
 * the rows whose mask holds its key; elements of V of 2^128 and more (scale bytes
 * 253 and 254) count as 1.5 * 2^127, so that they reach no other row either.
 * The columns of a sequence are its query positions times the query heads per K/V
 * head.  Sequences of more than 32 columns, and in a varlen call of more than 32
 * columns in total those of more than 16, run on tiles of 128 columns: there a
 * probability is rounded to one 16-bit term (elsewhere to two bf16 terms; softmax_lse is
 * that of the probabilities before, on either), and with
 * fp16 queries K and V are rounded to fp16, so that elements beyond +/-65504 saturate
 * and those of groups with scales below 2^-23 lose bits (elsewhere both are exact).
 * Enqueues up to three kernels; never synchronizes, never allocates.  The results
 * do not depend on the workspace's address or content; they may differ in the
 * last bit with the batch a sequence stands in (its keys are dealt over
 * workgroups with the others').
 */
typedef struct mfa_kv4_fwd_params {
    mfa_kv4_cache cache;
    const void* q;
    void* o;
    int64_t q_batch_stride, q_seq_stride, q_head_stride;
    int64_t o_batch_stride, o_seq_stride, o_head_stride;
    float* softmax_lse; /* NULL = not written; layout as in mfa_fwd_params */
    int64_t lse_batch_stride, lse_head_stride;
    const int32_t* cu_seqlens_q; /* NULL = seqlen_q rows per sequence */
    const int32_t* cache_seqlens;
    const float* alibi_slopes;
    int32_t alibi_batch_stride;
    int32_t batch, seqlen_q, total_q, heads_q, heads_kv, head_dim, max_seqlen_k;
    float scale, softcap;
    int32_t window_left, window_right, causal;
    int32_t dtype;
} mfa_kv4_fwd_params;
int64_t mfa_kv4_fwd_workspace_bytes(const mfa_kv4_fwd_params* params);
int mfa_kv4_fwd(const mfa_kv4_fwd_params* params, void* workspace, int64_t workspace_bytes, void* stream);
int mfa_kv4_fwd_params_size(void);

/*
 * Paged 8-bit K/V cache.  No counterpart in the reference.
 *
 * The structures, tables and rules of the 4-bit cache with another format: a row of
 * one head has head_dim code bytes, contiguous, each an e4m3 float (sign, four
 * exponent bits with bias 7, three mantissa bits; largest 448, 0x7f and 0xff NaN);
 * the 64 rows of a block (rows 64 i to 64 i + 63 of a page) and a head share the power
 * of two 2^(s - 127) of one scale byte s (0 stands for 0).  scale_row_stride is the
 * bytes between the scales of neighbouring blocks: scales are [num_pages,
 * page_block_size / 64, heads_kv].
 */
#define MFA_KV8_BLOCK 64
typedef mfa_kv4_pool mfa_kv8_pool;
typedef mfa_kv4_cache mfa_kv8_cache;

/*
 * New rows into the cache: the parameters of mfa_kv4_append.  The byte of a block is
 * the smallest from 1 on with 448 * 2^(s - 127) at least the largest finite magnitude
 * of the rows that are written into it; where the block holds rows of the sequence
 * already (cache_seqlens is no multiple of 64), at least the byte that it had, and if
 * the byte rises the codes of those rows are rounded again.  Elements are rounded to
 * the nearest code, ties to the even one (elements beyond 240 * 2^120, which would round
 * to 2^128, to that); infinities and NaN become NaN.  What stands
 * in a block behind the last row may change its value with the byte.  No two sequences
 * may write into one block.  A negative length counts as 0.  Values of tokens of no
 * sequence are 0; values of rows that are dropped are those of a block that holds
 * the call's rows alone; fp16 values saturate at +/-65504.  head_dim: 32, 64, 96 or
 * 128.  One kernel; never synchronizes, never allocates.
 */
typedef mfa_kv4_append_params mfa_kv8_append_params;
int mfa_kv8_append(const mfa_kv8_append_params* params, void* stream);
int mfa_kv8_append_params_size(void);

/*
 * Attention over the cache: the parameters and rules of mfa_kv4_fwd; a varlen call whose
 * sequences have 17 to 32 columns on average takes those of up to 32 as a fixed call
 * does, so with two terms of the probabilities.  A NaN element of
 * V reaches only the rows whose mask holds its key.  K is exact; V is exact with bf16
 * queries and for at most 32 columns; on the tiles of 128 columns fp16 queries take V
 * rounded to fp16 (elements beyond +/-65504 saturate, those of scales below 2^-15 may
 * lose bits).  Codes above 240 with scale bytes from 247 on, which mfa_kv8_append never writes, may
 * stand for values that are not finite.
 */
typedef mfa_kv4_fwd_params mfa_kv8_fwd_params;
int64_t mfa_kv8_fwd_workspace_bytes(const mfa_kv8_fwd_params* params);
int mfa_kv8_fwd(const mfa_kv8_fwd_params* params, void* workspace, int64_t workspace_bytes, void* stream);
int mfa_kv8_fwd_params_size(void);

/*
 * The attention weight that each cached key received: with the forward's parameters
 * (cache.v, o and their strides unused; softmax_lse an input, what mfa_kv8_fwd wrote)
 *   weight[j, hkv] = (j < Lk - Lq ? weight[j, hkv] : 0)
 *                  + sum over query rows i and query heads h of hkv of exp(score_ihj - lse_ih)
 * for the keys j < Lk of every sequence with queries, Lq of them: keys before the
 * queries' own rows add to what they had, the queries' own start from 0.  (So a pool needs
 * no clearing where every row passes through a call as a query's own; rows that do not, as
 * those of a prompt whose last rows alone are given, keep what their page held, from
 * another sequence too, and the caller clears them first.)  What a row's mask leaves out, and rows whose lse is -inf, add nothing.  Sequences with queries must
 * not share pages.  weights: fp32
 * [num_pages, page_block_size, heads_kv] by element strides (row and head strides >= 0),
 * addressed with the cache's block table; a page id outside the pool drops what is
 * written.  Sums in fp32, in an order that sizes and lengths alone decide; every key has
 * one owner.  The soft-cap is off by up to softcap 2^-21.  One or two kernels; never synchronizes, never allocates.
 */
typedef struct mfa_kv8_weights_params {
    mfa_kv8_fwd_params fwd;
    float* weights;
    int64_t weight_page_stride, weight_row_stride, weight_head_stride;
} mfa_kv8_weights_params;
int mfa_kv8_weights(const mfa_kv8_weights_params* params, void* stream);
int mfa_kv8_weights_params_size(void);

/*
 * Eviction: of every head of a sequence with n > budget rows, the last min(recent,
 * budget) rows and the heaviest of the others (by weights, ties to the lower row, NaN
 * above everything), budget in all, move together in their order: they become rows 0 ..
 * budget - 1, weights with them.  A block of 64 rows of a head whose rows all stay where
 * they are is left as it is; any other gets a new scale byte by the rule of
 * mfa_kv8_append for a block without rows, from the values that its rows have, and
 * their codes are rounded by it (NaN stays NaN).  Rows from budget on keep their codes
 * and weights.  n = min(cache_seqlens, max_seqlen_k, what the table can name), max_seqlen_k
 * 0 leaving that bound out; new_seqlens [batch] (may be cache_seqlens itself) receives
 * min(n, budget).  A row on a page id outside the pool reads as zeros with weight 0 and
 * drops what is written.  budget and recent >= 0; the pool has less than 2^31 rows.
 * K and V do not share memory.  `workspace`: 256-byte aligned, at least
 * mfa_kv8_evict_workspace_bytes bytes (0, where no row can move: may be NULL).  One to
 * three kernels; never synchronizes, never allocates.
 */
typedef struct mfa_kv8_evict_params {
    mfa_kv8_cache cache;
    float* weights;
    int64_t weight_page_stride, weight_row_stride, weight_head_stride;
    const int32_t* cache_seqlens;
    int32_t* new_seqlens;
    int32_t batch, heads_kv, head_dim, max_seqlen_k, budget, recent;
} mfa_kv8_evict_params;
int64_t mfa_kv8_evict_workspace_bytes(const mfa_kv8_evict_params* params);
int mfa_kv8_evict(const mfa_kv8_evict_params* params, void* workspace, int64_t workspace_bytes, void* stream);
int mfa_kv8_evict_params_size(void);

/*
 * Pages copied inside pools: page src[i] to page dst[i] of every pool, i < pairs
 * (a forked sequence's last page, compaction).  No counterpart in the reference.
 * A pool is `page_bytes` contiguous bytes per page, `page_stride` bytes apart.
 * Pairs with an id outside [0, num_pages) are skipped.  The destinations have to
 * differ from each other and from every source: pairs are copied in no order.
 * One kernel; never synchronizes, never allocates.
 */
#define MFA_COPY_MAX_POOLS 64
typedef struct mfa_copy_pool {
    void* base;
    int64_t page_stride, page_bytes;
} mfa_copy_pool;
typedef struct mfa_copy_pages_params {
    mfa_copy_pool pool[MFA_COPY_MAX_POOLS];
    const int32_t* src;
    const int32_t* dst;
    int32_t pools, pairs, num_pages;
    int32_t reserved;
} mfa_copy_pages_params;
int mfa_copy_pages(const mfa_copy_pages_params* params, void* stream);
int mfa_copy_pages_params_size(void);

/*
 * RMS norm of every query and key head and the rotation of its position, in one
 * pass.  No counterpart in the reference.  For a row x of head_dim elements at
 * position pos:
 *   n = x / sqrt(mean(x^2) + eps), y = n * weight (q_weight / k_weight, NULL: 1),
 *   out_a = y_a cos - y_b sin, out_b = y_b cos + y_a sin
 * for each pair i < rotary_dim / 2 with cos[pos][i], sin[pos][i]: elements (a, b)
 * = (i, i + rotary_dim / 2), or (2i, 2i + 1) with `interleaved`; elements from
 * rotary_dim on are y.  fp32 arithmetic, one rounding.  A position outside
 * [0, table_rows) gives NaN in the rotated elements, never a read out of bounds.
 * q [batch, seqlen, heads_q, head_dim], k [batch, seqlen, heads_kv, head_dim] by
 * element strides (head dim contiguous); outputs and gradients are contiguous.
 * positions: [batch, seqlen] int32 or int64 (positions_64) with
 * positions_batch_stride (0: one row for the batch) and unit stride inside, NULL:
 * 0, 1, 2, ...  cos / sin: [table_rows, rotary_dim / 2], rows table_stride
 * elements apart.  head_dim up to MFA_MAX_HEAD_DIM, rotary_dim even, 0 <=
 * rotary_dim <= head_dim.  One kernel; never synchronizes, never allocates.
 */
typedef struct mfa_norm_rope_params {
    const void* q;
    const void* k;
    void* q_out;
    void* k_out;
    int64_t q_batch_stride, q_seq_stride, q_head_stride;
    int64_t k_batch_stride, k_seq_stride, k_head_stride;
    const void* q_weight;
    const void* k_weight;
    const void* cos;
    const void* sin;
    int64_t table_stride;
    const void* positions;
    int64_t positions_batch_stride;
    int32_t batch, seqlen, heads_q, heads_kv, head_dim, rotary_dim, table_rows;
    int32_t positions_64, interleaved;
    int32_t dtype;        /* of q, k and the outputs */
    int32_t dtype_weight; /* of the weights and their gradients */
    int32_t dtype_table;  /* of cos and sin: dtype or MFA_DTYPE_F32 */
    float eps;
} mfa_norm_rope_params;
int mfa_norm_rope(const mfa_norm_rope_params* params, void* stream);
int mfa_norm_rope_params_size(void);

/*
 * Backward of mfa_norm_rope (fwd.q_out / k_out unused): with g the rotation of
 * dq_out turned back, h = g * weight,
 *   dq = (h - n mean(h n)) / sqrt(mean(x^2) + eps),  dq_weight = sum over rows g n
 * and the same for k.  dq / dk are contiguous.  Weight gradients (dtype_weight)
 * where the weight is set and the pointer is not NULL: summed in fp32, in an
 * order that sizes, strides and alignment decide.  `workspace`: 256-byte aligned, at least
 * mfa_norm_rope_bwd_workspace_bytes bytes.  One or two kernels; never
 * synchronizes, never allocates.
 */
typedef struct mfa_norm_rope_bwd_params {
    mfa_norm_rope_params fwd;
    const void* dq_out;
    const void* dk_out;
    int64_t dqo_batch_stride, dqo_seq_stride, dqo_head_stride;
    int64_t dko_batch_stride, dko_seq_stride, dko_head_stride;
    void* dq;
    void* dk;
    void* dq_weight;
    void* dk_weight;
} mfa_norm_rope_bwd_params;
int64_t mfa_norm_rope_bwd_workspace_bytes(const mfa_norm_rope_bwd_params* params);
int mfa_norm_rope_bwd(const mfa_norm_rope_bwd_params* params, void* workspace, int64_t workspace_bytes, void* stream);
int mfa_norm_rope_bwd_params_size(void);

#ifdef __cplusplus
}
#endif

#endif /* MTLFA_MFA_H */
