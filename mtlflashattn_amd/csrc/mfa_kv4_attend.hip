// mfa_kv4_attend.hip -- attention over a paged 4-bit K/V cache
// (mfa_kv4_fwd in include/mfa.h): the 4-bit format of the kernel for sequences of
// at most 32 columns (mfa_kv_rows.h), and, for every format, the merge of parts and
// the host's plan.
//
// Bound by the stream of the cache (68 bytes per key and head at head dim 128)
// where batches are large, by latency where they are small.  Lane group g of a
// key's row takes elements g D/4 .. (g+1) D/4 - 1, at D = 128 one 16-byte load that
// holds one whole scale group; v_cvt_scalef32_pk_bf16_fp4 turns codes into bf16.
//
// Work is dealt by length: every sequence's keys are cut into chunks of 128, the
// chunks of all (sequence, head, column tile) units are laid end to end, and
// workgroup w of G takes chunks [w C / G, (w+1) C / G) of the C there are, so
// ragged batches end together and the lengths are read on the device only.  A
// unit that one workgroup walks alone is stored by it; the parts of any other go
// to the workspace (at most two per workgroup, its first and its last unit) and
// mfa_kv_merge_kernel adds them in order.
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>

#include "mfa_kv_rows.h"

namespace {

// The codes of a 32-key block: K, DP/8 bytes of each of two 16-key tiles per lane
// and their scale bytes (two where a lane's elements cross a scale group: DP =
// 96); V, 32-element groups.
// Non-temporal buffer loads: a unit holds all columns of its K/V head, so a byte
// of the cache is read once a call (64 sequences of 512 to 16384 keys, Hq=32
// Hkv=8 D=128 bf16: 104.6 us, 108.9 with ordinary loads; 31 of 256 to 4096, which the
// last-level cache holds from call to call: 22.9 and 22.4 us).
template <int DP>
struct Block4 {
    static constexpr int D = DP;
    // codes (even x) and scales of a row
    static constexpr int bytes(int x) { return x & 1 ? DP / 32 : DP / 2; }
    static constexpr int rows_per(int) { return 1; }
    static constexpr int KW = DP / 32;         // dwords per lane and tile
    static constexpr int GPR = DP / 32;        // scale groups per row
    static constexpr int VG = (DP + 63) / 64;  // V groups per lane
    uint32_t k[2][KW];
    // (scales stay bytes until they are used: widening them would wait for the loads)
    uint8_t ks[2][DP == 96 ? 2 : 1];
    u32x4_t v[VG];
    uint8_t vs[VG];

    struct Offsets {
        uint32_t koff[2], ksoff[2][2], voff[VG], vsoff[VG];
        int vrow[VG], vgrp[VG];
        __device__ __forceinline__ void init(K4Const& a, int lane) {
            const int l16 = lane & 15, grp = lane >> 4;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const int row = 16 * kk + l16;
                koff[kk] = (uint32_t)(row * (int)a.k.cr + grp * (DP / 8));
                ksoff[kk][0] = (uint32_t)(row * (int)a.k.sr + (DP == 96 ? (24 * grp) >> 5 : grp * (DP / 4) / 32));
                ksoff[kk][1] = (uint32_t)(row * (int)a.k.sr + ((24 * grp + 16) >> 5));
            }
#pragma unroll
            for (int i = 0; i < VG; ++i) {
                const int cc = 64 * i + lane;
                vrow[i] = cc / GPR;
                vgrp[i] = cc - vrow[i] * GPR;
                const bool in = cc < 32 * GPR;
                voff[i] = in ? (uint32_t)(vrow[i] * (int)a.v.cr + vgrp[i] * 16) : 0x80000000u;
                vsoff[i] = in ? (uint32_t)(vrow[i] * (int)a.v.sr + vgrp[i]) : 0x80000000u;
            }
        }
    };
    __device__ __forceinline__ void load(const __amdgpu_buffer_rsrc_t (&rs)[4], const Offsets& off, uint32_t kr, uint32_t ksr,
                                         uint32_t vr, uint32_t vsr) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            if constexpr (DP == 128) {
                const u32x4_t y = __builtin_amdgcn_raw_buffer_load_b128(rs[0], off.koff[kk] + kr, 0, kOnce4);
#pragma unroll
                for (int i = 0; i < 4; ++i) k[kk][i] = y[i];
            } else if constexpr (DP == 96) {
                const auto y = __builtin_amdgcn_raw_buffer_load_b96(rs[0], off.koff[kk] + kr, 0, kOnce4);
#pragma unroll
                for (int i = 0; i < 3; ++i) k[kk][i] = y[i];
            } else if constexpr (DP == 64) {
                const auto y = __builtin_amdgcn_raw_buffer_load_b64(rs[0], off.koff[kk] + kr, 0, kOnce4);
                k[kk][0] = y[0];
                k[kk][1] = y[1];
            } else {
                k[kk][0] = __builtin_amdgcn_raw_buffer_load_b32(rs[0], off.koff[kk] + kr, 0, kOnce4);
            }
            ks[kk][0] = __builtin_amdgcn_raw_buffer_load_b8(rs[1], off.ksoff[kk][0] + ksr, 0, kOnce4);
            if constexpr (DP == 96) ks[kk][1] = __builtin_amdgcn_raw_buffer_load_b8(rs[1], off.ksoff[kk][1] + ksr, 0, kOnce4);
        }
#pragma unroll
        for (int i = 0; i < VG; ++i) {
            v[i] = __builtin_amdgcn_raw_buffer_load_b128(rs[2], off.voff[i] + vr, 0, kOnce4);
            vs[i] = __builtin_amdgcn_raw_buffer_load_b8(rs[3], off.vsoff[i] + vsr, 0, kOnce4);
        }
    }

    // step s of lane group grp: eight elements from here on
    static __device__ __forceinline__ int element(int grp, int s) { return grp * (DP / 4) + 8 * s; }
    __device__ __forceinline__ bf16x8_t k_operand(int kk, int s, int grp) const {
        uint8_t sb = ks[kk][0];
        if constexpr (DP == 96) {  // elements 24 grp + 8 s .. lie in the first or the second of the lane's groups
            if (s == 2 || (s == 1 && grp == 1)) sb = ks[kk][1];
        }
        return __builtin_bit_cast(bf16x8_t, kv4_bf16x8(k[kk][s], kv4_scale(sb)));
    }
    // what the scores of the block are still to be multiplied by
    __device__ __forceinline__ float k_scale() const { return 1.f; }

    struct Nans {
        uint64_t lanes[VG];  // lanes that hold a NaN group
        template <int NT>
        __device__ __forceinline__ void add(f32x4_t (&o)[NT][DP / 16], int j, const int (&lo)[NT], const int (&hi)[NT], int) const {
#pragma unroll
            for (int i = 0; i < VG; ++i) {
                for (uint64_t x = lanes[i]; x; x &= x - 1) {
                    const int cc = 64 * i + __builtin_ctzll(x), row = cc / GPR;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const bool sees = j + row >= lo[t] && j + row <= hi[t];
#pragma unroll
                        for (int g = 0; g < GPR; ++g) {
                            float y = sees && g == cc - row * GPR ? __builtin_nanf("") : 0.f;
                            pin(y);  // (no indexing of o by the group)
                            o[t][2 * g] += y;
                            o[t][2 * g + 1] += y;
                        }
                    }
                }
            }
        }
    };
    template <class Swz>
    __device__ __forceinline__ void stage_v(uint16_t* vt, Swz&& vswz, const Offsets& off, bool masked, int lane, Nans& nans) const {
#pragma unroll
        for (int i = 0; i < VG; ++i) {
            const bool nan = masked && vs[i] == 255;
            nans.lanes[i] = __ballot(nan);
            if (32 * GPR % 64 == 0 || 64 * i + lane < 32 * GPR) {
                const float s = nan ? 0.f : kv4_scale(vs[i]);
                u32x4_t codes = v[i];
                if (__builtin_expect(kv4_beyond(vs[i]), 0)) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) codes[e] = kv4_saturate8(codes[e], vs[i]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *reinterpret_cast<u32x4_t*>(vt + off.vrow[i] * DP + (((4 * off.vgrp[i] + e) ^ vswz(off.vrow[i])) << 3)) =
                        kv4_bf16x8(codes[e], s);
            }
        }
    }
};

// The parts of a unit that several workgroups walked, added in the order of its
// keys: block (w, z) takes merge_cols columns of the unit whose walk workgroup w is
// the first to go on with.  Up to two launches' units in one (blocks of the first,
// then of the second); a thread holds four elements of a column, and where there
// are few of them (one or a few columns) groups of threads take every P-th part.
// Bound by the latency of its loads: a part's reference, sum and elements are
// loaded at once (no pass for the largest reference first), N parts at a time (4,
// not 8, for columns that fill the block: 13.6 us instead of 16.5 after a launch of
// 512 rows over 4096 keys beside 31 decoding sequences).
// Blocks of T threads: 512 where all units have few columns, more threads per column
// (5 rows of 6 sequences at head dim 64: 3.9 us, 5.9 with 256, 6.4 with 1024); 256
// where some have many (13.6 us for the step above, 18.8 with 512).
constexpr int kMergeFew = 512, kMergeMany = 256;
constexpr int merge_cols(int threads) { return threads / (MFA_MAX_HEAD_DIM / 4); }
// LE: some parts have a sum for the log-sum-exp of their own (ws_le).
template <int DP, bool IS_BF16, int T, bool LE>
__global__ void __launch_bounds__(T) mfa_kv_merge_kernel(K4Args, K4Args) {
    constexpr int kMergeCols = merge_cols(T);
    __shared__ f32x4_t o_s[T];
    __shared__ float2 ml_s[T];
    __shared__ float le_s[LE ? T : 1];
    const int tid = threadIdx.x;
    const int first = args4(0).ws_merge ? args4(0).G * (args4(0).cols / kMergeCols) : 0;
    const int which = __builtin_amdgcn_readfirstlane((int)blockIdx.x >= first);
    K4Const& a = args4(which);
    const int cols = a.cols, blk = blockIdx.x - (which ? first : 0), w = blk / (cols / kMergeCols);
    const int cbeg = (blk - w * (cols / kMergeCols)) * kMergeCols;  // first of this block's columns
    const Merge4 g4 = a.ws_merge[w];
    const int w0 = w - 1, w1 = g4.w1, ncol = min(kMergeCols, g4.ncol - cbeg), items = ncol * (DP / 4);
    if (w1 < 0 || ncol <= 0) return;
    // the part of workgroup v: its first unit, unless it began before this one
    auto at = [&](int v) { return ((int64_t)v * 2 + (v == w0 ? g4.slot0 : 0)) * cols + cbeg; };
    const int P = items <= T / 8 ? 8 : items <= T / 4 ? 4 : items <= T / 2 ? 2 : 1, S = T / P;
    const int g = tid / S, it = tid - g * S;  // (a round holds every item)
    const bool in = it < items;
    const int r = in ? it / (DP / 4) : 0, d = in ? 4 * (it - r * (DP / 4)) : 0;
    const float* ws_o = a.ws_o;
    const float* ws_ml = a.ws_ml;
    const float* ws_le = a.ws_le ? a.ws_le : ws_ml + 1;  // (by le_step)
    const int le_step = a.ws_le ? 1 : 2;
    float m = -INFINITY, l = 0.f, le = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](float mw, float lw, float lew, const f32x4_t& y) {
        const float mn = fmax_nn(m, mw), e0 = pow2_diff(m, mn), e1 = pow2_diff(mw, mn);
        l = fmaf(lw, e1, l * e0);
        if constexpr (LE) le = fmaf(lew, e1, le * e0);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = fmaf(y[k], e1, acc[k] * e0);
        m = mn;
    };
    auto walk = [&](auto ahead, int P) {
        constexpr int N = decltype(ahead)::value;
        for (int v0 = w0 + g; v0 <= w1; v0 += P * N) {
            float2 ml[N];
            float lw[N];
            f32x4_t y[N];
#pragma unroll
            for (int z = 0; z < N; ++z) {
                const int64_t row = at(min(v0 + P * z, w1)) + r;
                ml[z] = *reinterpret_cast<const float2*>(ws_ml + 2 * row);
                lw[z] = LE ? ws_le[le_step * row] : 0.f;
                y[z] = *reinterpret_cast<const f32x4_t*>(ws_o + row * DP + d);
            }
#pragma unroll
            for (int z = 0; z < N; ++z)
                if (v0 + P * z <= w1) add(ml[z].x, ml[z].y, lw[z], y[z]);
        }
    };
    if (w1 - w0 + 1 <= 2 * P)
        walk(std::integral_constant<int, 2>{}, P);
    else if (P > 1)
        walk(std::integral_constant<int, 8>{}, P);
    else
        walk(std::integral_constant<int, 4>{}, 1);
    if (P > 1) {
        o_s[tid] = acc;
        ml_s[tid] = make_float2(m, l);
        if constexpr (LE) le_s[tid] = le;
        __syncthreads();
        if (g > 0) return;
        for (int z = 1; z < P; ++z) add(ml_s[tid + z * S].x, ml_s[tid + z * S].y, LE ? le_s[tid + z * S] : 0.f, o_s[tid + z * S]);
    }
    if (in) {
        const int col = g4.col0 + cbeg + r, i = (int)div4(col, a.by_r), h = g4.hkv * a.R + col - i * a.R;
        store_row4<IS_BF16>(a.o + row_off4(a.cu_q != nullptr, g4.b, g4.q0, i, h, a.ob, a.os, a.oh) * 2, d, acc, l);
        if (d == 0) store_lse4(a, g4.b, g4.q0, i, h, m, LE ? le : l);
    }
}
static_assert(16 % merge_cols(kMergeFew) == 0 && kTileCols4 % merge_cols(kMergeMany) == 0, "whole blocks per unit");

typedef void (*k4_fn)(K4Args);
typedef void (*k4_merge_fn)(K4Args, K4Args);
// threads: of the merge's blocks
template <int DP, bool IS_BF16>
k4_merge_fn merge4(int threads, bool le) {
    return threads == kMergeFew ? mfa_kv_merge_kernel<DP, IS_BF16, kMergeFew, false>  // (no tiles of 128 columns)
           : le                 ? mfa_kv_merge_kernel<DP, IS_BF16, kMergeMany, true>
                                : mfa_kv_merge_kernel<DP, IS_BF16, kMergeMany, false>;
}
template <bool IS_BF16>
k4_merge_fn merge4(int dp, int threads, bool le) {
    switch (dp) {
        case 32: return merge4<32, IS_BF16>(threads, le);
        case 64: return merge4<64, IS_BF16>(threads, le);
        case 96: return merge4<96, IS_BF16>(threads, le);
        default: return merge4<128, IS_BF16>(threads, le);
    }
}

int k4err(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(mfa_error_buffer(), 512, fmt, ap);
    va_end(ap);
    return code;
}

// Columns of a unit for sequences of at most `cols` columns: the smallest tile that
// takes them all, so that the cache is read once.  (36 columns, D = 128 bf16: as two
// tiles of 32, 158 us for 32 sequences over 8192 keys and 23 for 4 over 1024; as
// one of 128, 166 and 21.  80 columns: 228 and 25, against 163 and 24.)
int unit_cols(int64_t cols) { return cols <= 16 ? 16 : cols <= 32 ? 32 : kTileCols4; }

// A launch: the sequences of min_cols to max_cols columns.
struct K4Launch {
    K4Args a;
    int64_t parts;  // rows of its partial results, 0: no merge
};
// workspace of a launch: parts, their references and sums (of 128 columns one more, for the
// log-sum-exp, whether it is asked for or not), what is merged
int64_t part_bytes(const K4Launch& l, int D) {
    const int64_t row = D * 4 + (l.a.cols == kTileCols4 ? 12 : 8);
    return l.parts ? (l.parts * row + (int64_t)l.a.G * sizeof(Merge4) + 255) / 256 * 256 : 0;
}
struct K4Plan {
    K4Launch l[2];
    int n = 0;
    int64_t ws_bytes = 0;
};

}  // namespace

int mfa_kv_args(const mfa_kv4_fwd_params* p, const char* who, void* args) {
    if (!p) return k4err(MFA_ERR_INVALID, "%s: params is NULL", who);
    if (p->dtype != MFA_DTYPE_F16 && p->dtype != MFA_DTYPE_BF16)
        return k4err(MFA_ERR_UNSUPPORTED, "%s: dtype %d (fp16 and bf16 queries)", who, p->dtype);
    const int D = p->head_dim;
    if (D != 32 && D != 64 && D != 96 && D != 128)
        return k4err(MFA_ERR_UNSUPPORTED, "%s: head_dim %d (32, 64, 96 or 128)", who, D);
    if (p->batch < 0 || p->seqlen_q < 0 || p->total_q < 0 || p->max_seqlen_k < 0)
        return k4err(MFA_ERR_INVALID, "%s: negative size", who);
    if (p->heads_q <= 0 || p->heads_kv <= 0 || p->heads_q % p->heads_kv)
        return k4err(MFA_ERR_INVALID, "%s: num_heads_kv (%d) must divide num_heads_q (%d)", who, p->heads_kv, p->heads_q);
    if (!(p->softcap >= 0.f)) return k4err(MFA_ERR_INVALID, "%s: softcap must be >= 0", who);
    if (p->window_left < -1 || p->window_right < -1)
        return k4err(MFA_ERR_INVALID, "%s: window bounds must be >= -1", who);
    const int rc = mfa_kv4_check_cache(&p->cache, p->batch, D, who);
    if (rc != MFA_OK) return rc;
    const bool varlen = p->cu_seqlens_q != nullptr;
    const int64_t rows = varlen ? p->total_q : (int64_t)p->batch * p->seqlen_q;
    K4Args& a = *static_cast<K4Args*>(args);
    memset(&a, 0, sizeof(a));
    if (rows == 0) return MFA_OK;
    auto bad = [](const void* x, uintptr_t al) { return !x || (reinterpret_cast<uintptr_t>(x) & (al - 1)); };
    if (bad(p->q, 16) || bad(p->o, 16)) return k4err(MFA_ERR_INVALID, "%s: q and o must be 16-byte aligned", who);
    if (p->batch > 0 && bad(p->cache_seqlens, 4)) return k4err(MFA_ERR_INVALID, "%s: cache_seqlens is required", who);
    const int64_t st[] = {p->q_batch_stride, p->q_seq_stride, p->q_head_stride, p->o_batch_stride, p->o_seq_stride, p->o_head_stride};
    for (int64_t s : st)
        if (s % 8) return k4err(MFA_ERR_INVALID, "%s: q and o strides must be multiples of 8 elements", who);
    if (p->alibi_slopes && p->alibi_batch_stride != 0 && p->alibi_batch_stride != p->heads_q)
        return k4err(MFA_ERR_INVALID, "%s: alibi_batch_stride must be 0 or heads_q", who);

    a.q = static_cast<const char*>(p->q);
    a.o = static_cast<char*>(p->o);
    a.lse = p->softmax_lse;
    a.qb = p->q_batch_stride; a.qs = p->q_seq_stride; a.qh = p->q_head_stride;
    a.ob = p->o_batch_stride; a.os = p->o_seq_stride; a.oh = p->o_head_stride;
    a.lse_b = p->lse_batch_stride; a.lse_h = p->lse_head_stride;
    a.k = kv4_pool(p->cache.k);
    a.v = kv4_pool(p->cache.v);
    a.bt = p->cache.block_table;
    a.bt_b = p->cache.block_table_batch_stride;
    a.lens = p->cache_seqlens;
    a.cu_q = p->cu_seqlens_q;
    a.alibi = p->alibi_slopes;
    a.alibi_bstride = p->alibi_batch_stride;
    a.B = p->batch; a.Hq = p->heads_q; a.Hkv = p->heads_kv;
    a.R = p->heads_q / p->heads_kv;
    a.Lq = p->seqlen_q;
    a.rows_q = (int32_t)rows;
    // (a sequence holds at most what its table can name)
    const int64_t cap = (int64_t)p->cache.max_pages * p->cache.page_block_size;
    a.max_k = (int32_t)std::min<int64_t>(p->max_seqlen_k ? p->max_seqlen_k : cap, std::min<int64_t>(cap, 0x7fffff00));
    a.page = p->cache.page_block_size;
    a.npages = p->cache.num_pages;
    a.by_page = fast_div(a.page);
    a.by_r = fast_div(a.R);
    a.scale = p->scale;
    a.scale_log2 = p->scale * kLog2e;
    a.softcap = p->softcap;
    a.softcap_sk = p->softcap > 0.f ? p->scale * (2.f * kLog2e / p->softcap) : 0.f;
    a.bias = p->softcap > 0.f || p->alibi_slopes || !(p->scale > 0.f);
    // (a window that holds every key of every row is none)
    a.wl = p->window_left >= a.max_k ? -1 : p->window_left;
    a.wr = p->window_right >= rows + a.max_k ? -1 : p->window_right;
    a.causal = p->causal ? 1 : 0;
    if (rows > 0x3fffffff || rows * a.Hq > 0x3fffffff) return k4err(MFA_ERR_INVALID, "%s: problem too large", who);
    return MFA_OK;
}

namespace {

int k4_plan(const mfa_kv4_fwd_params* p, const MfaKvFormat& f, K4Plan* plan, int cus) {
    K4Args a;
    const int rc = mfa_kv_args(p, f.who, &a);
    if (rc != MFA_OK || a.rows_q == 0) return rc;
    const bool varlen = p->cu_seqlens_q != nullptr;
    const int64_t rows = a.rows_q;
    const int D = p->head_dim;
    a.bias |= !(p->scale > f.least_scale);

    // Columns per workgroup: a sequence's, at most 128.  The sequences of a
    // varlen call are known on the device only: one launch takes those of at most
    // 16 columns (32 by the mean, where the format says so), another the longer ones.
    // (no sequences: the launch only clears the rows)
    const int64_t cols = p->batch == 0 ? 1 : (varlen ? rows : p->seqlen_q) * (int64_t)a.R;
    plan->n = varlen && cols > 16 ? 2 : 1;
    const int few = f.varlen32 && cols > 16 * (int64_t)p->batch && cols <= 32 * (int64_t)p->batch ? 32 : 16;
    const int64_t chunks = p->batch == 0 ? 1 : std::max<int64_t>(1, ((int64_t)a.max_k + kChunk4 - 1) / kChunk4);
    for (int i = 0; i < plan->n; ++i) {
        K4Launch& l = plan->l[i];
        l.a = a;
        l.a.cols = unit_cols(plan->n == 2 && i == 0 ? few : cols);
        l.a.min_cols = i == 0 ? 1 : few + 1;
        l.a.max_cols = plan->n == 2 && i == 0 ? few : 0x7fffffff;
        // (a bound on the items, which are counted on the device in int32)
        const int64_t tiles = !varlen       ? p->batch * ((cols + l.a.cols - 1) / l.a.cols)
                              : l.a.max_cols == few ? std::min<int64_t>(p->batch, rows)
                                                   : (cols + l.a.cols - 1) / l.a.cols + std::min<int64_t>(p->batch, rows);
        const int64_t units = tiles * a.Hkv;
        if (units > 0x3fffffff || units * chunks > 0x7fffffffLL) return k4err(MFA_ERR_INVALID, "%s: problem too large", f.who);
        l.a.G = (int32_t)std::min<int64_t>(units * chunks, (int64_t)cus * (l.a.cols == kTileCols4 ? f.tile_wgs : f.rows_wgs[l.a.cols / 16 - 1]));
        // (neighbouring tiles of a K/V head share its rows in their XCD's L2)
        l.a.xcds = l.a.cols == kTileCols4 && l.a.G % 8 == 0 ? 8 : 1;
        l.parts = chunks > 1 ? (int64_t)l.a.G * 2 * l.a.cols : 0;
        plan->ws_bytes += part_bytes(l, D);
    }
    return MFA_OK;
}

// Kernels of the 4-bit format.  Workgroups per CU at NT column tiles: as many as the
// registers hold (the batch above: 98.6 us with three, 107 with two, 118 with four,
// which spill; at D = 64 three and four measure the same); a third of the 128-column
// ones is dealt work but not resident (335 us become 369).
template <int DP>
void* rows4(int cols, bool bf16) {
    return cols == 16 ? (void*)(bf16 ? (k4_fn)mfa_kv_rows_kernel<Block4<DP>, 1, true> : (k4_fn)mfa_kv_rows_kernel<Block4<DP>, 1, false>)
                      : (void*)(bf16 ? (k4_fn)mfa_kv_rows_kernel<Block4<DP>, 2, true> : (k4_fn)mfa_kv_rows_kernel<Block4<DP>, 2, false>);
}
void* rows_kernel4(int dp, int cols, bool bf16) {
    switch (dp) {
        case 32: return rows4<32>(cols, bf16);
        case 64: return rows4<64>(cols, bf16);
        case 96: return rows4<96>(cols, bf16);
        default: return rows4<128>(cols, bf16);
    }
}
const MfaKvFormat kFormat4 = {"mfa_kv4_fwd", {wgs4(1), wgs4(2)}, 2, 0.f, false, rows_kernel4, mfa_kv4_tile_kernel_of};

}  // namespace

int64_t mfa_kv_fwd_workspace_bytes(const mfa_kv4_fwd_params* p, const MfaKvFormat& f) {
    mfa_error_buffer()[0] = 0;
    K4Plan plan;
    const int rc = k4_plan(p, f, &plan, mfa_chip_cus(nullptr));
    return rc != MFA_OK ? rc : plan.ws_bytes;
}

int mfa_kv_fwd(const mfa_kv4_fwd_params* p, const MfaKvFormat& f, void* workspace, int64_t workspace_bytes, void* stream) {
    mfa_error_buffer()[0] = 0;
    K4Plan plan;
    const int rc = k4_plan(p, f, &plan, mfa_chip_cus(stream));
    if (rc != MFA_OK || plan.n == 0) return rc;
    if (plan.ws_bytes) {
        if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u))
            return k4err(MFA_ERR_INVALID, "%s: workspace must be a 256-byte aligned device pointer", f.who);
        if (workspace_bytes < plan.ws_bytes)
            return k4err(MFA_ERR_INVALID, "%s: workspace of %lld bytes, %lld needed", f.who, (long long)workspace_bytes,
                         (long long)plan.ws_bytes);
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    const bool bf16 = p->dtype == MFA_DTYPE_BF16;
    int merge = 0;
    const int threads = plan.l[plan.n - 1].a.cols == kTileCols4 ? kMergeMany : kMergeFew;
    for (int i = 0; i < plan.n; ++i) {
        K4Launch& l = plan.l[i];
        const k4_fn attend = (k4_fn)(l.a.cols == kTileCols4 ? f.tile_kernel(p->head_dim, bf16, l.a.bias != 0, l.a.lse != nullptr)
                                                            : f.rows_kernel(p->head_dim, l.a.cols, bf16));
        if (l.parts) {
            l.a.ws_o = reinterpret_cast<float*>(ws);
            l.a.ws_ml = l.a.ws_o + l.parts * p->head_dim;
            l.a.ws_merge = reinterpret_cast<Merge4*>(l.a.ws_ml + l.parts * 2);
            if (l.a.cols == kTileCols4 && l.a.lse) l.a.ws_le = reinterpret_cast<float*>(l.a.ws_merge + l.a.G);
            ws += part_bytes(l, p->head_dim);
            merge += l.a.G * (l.a.cols / merge_cols(threads));
        }
        hipLaunchKernelGGL(attend, dim3(l.a.G), dim3(kThreads4), 0, st, l.a);
    }
    if (merge) {
        const bool le = plan.l[plan.n - 1].a.ws_le != nullptr;
        const k4_merge_fn fn = bf16 ? merge4<true>(p->head_dim, threads, le) : merge4<false>(p->head_dim, threads, le);
        hipLaunchKernelGGL(fn, dim3(merge), dim3(threads), 0, st, plan.l[0].a, plan.l[plan.n - 1].a);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return k4err(MFA_ERR_LAUNCH, "%s: launch failed: %s", f.who, hipGetErrorString(e));
    return MFA_OK;
}

extern "C" {

int mfa_kv4_fwd_params_size(void) { return (int)sizeof(mfa_kv4_fwd_params); }

int64_t mfa_kv4_fwd_workspace_bytes(const mfa_kv4_fwd_params* p) { return mfa_kv_fwd_workspace_bytes(p, kFormat4); }

int mfa_kv4_fwd(const mfa_kv4_fwd_params* p, void* workspace, int64_t workspace_bytes, void* stream) {
    return mfa_kv_fwd(p, kFormat4, workspace, workspace_bytes, stream);
}

}  // extern "C"
