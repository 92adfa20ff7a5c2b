// mfa_kv8_weights.hip -- the attention weight that each cached key received
// (mfa_kv8_weights in include/mfa.h): w_j += sum over the rows i and heads of its K/V
// head of exp(score_ij - lse_i).
//
// The log-sum-exps are known, so keys do not depend on each other: every key has one
// owner, which forms its scores with all columns ((query position, query head) pairs)
// of its K/V head and adds them up in registers: no atomics, no second pass.  The
// products are S = Q K^T with the queries as the A operand, so that a lane owns a key
// and its registers are columns: the sum over columns is mostly a sum over registers.
// K's codes are exact in the queries' type; the block's scale multiplies the scores.
//
// Two kernels, by the columns of a sequence, over chunks of 128 keys that are dealt as
// in the attention (mfa_kv4_attend.hip):
//  * at most 16: bound by the stream of K and the weights (136 bytes per key and head
//    at head dim 128).  A wavefront takes every fourth 32-key block, the next one on
//    its way into registers;
//  * more: bound by the exponentials (24 cycles of a SIMD per 64 scores, against 16 of
//    the products at head dim 128).  A wavefront holds 64 keys as operands and goes
//    over the columns, 32 at a time; two wavefronts share the keys and two the columns,
//    64 of which stand in LDS while the next 64 are loaded.
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>

#include "mfa_kv8_block.h"

namespace {

// The way through the pages: K's codes and scales, and the weights in V's place.
template <int DP>
struct WFormat {
    static constexpr int D = DP;
    static constexpr int bytes(int x) { return x == 0 ? DP : x == 1 ? 1 : x == 2 ? 4 : 0; }
    static constexpr int rows_per(int x) { return x & 1 ? kKv8Block : 1; }
};

template <bool IS_BF16>
using op_of = typename std::conditional<IS_BF16, bf16x8_t, f16x8_t>::type;

// -lse in log2 units of a row; -inf (weight 0) for rows without keys and for no row
__device__ __forceinline__ float neg_lse2(K4Const& a, bool in, int b, int q0, int i, int h) {
    if (!in) return -INFINITY;
    const float l = a.lse[(a.cu_q ? (int64_t)(q0 + i) : b * a.lse_b + i) + h * a.lse_h];
    return l == -INFINITY ? -INFINITY : -l * kLog2e;
}

// Scores to log2 units less the log-sum-exp, from the products s of one column.
struct ScoreOf {
    float scale, scale_log2, softcap;
    bool bias, alibi;
    __device__ __forceinline__ float operator()(float s, float sk, float nlse, float slope, int dist) const {
        if (!bias) return fmaf(s, scale_log2 * sk, nlse);
        float x = s * (scale * sk);
        // (tanh to the last bits: the sums are fp32 results)
        if (softcap > 0.f) x = softcap * precise_tanh(x / softcap);
        if (alibi) x = fmaf(-slope, fabsf((float)dist), x);
        return fmaf(x, kLog2e, nlse);
    }
};
__device__ __forceinline__ ScoreOf score_of(K4Const& a) {
    return ScoreOf{a.scale, a.scale_log2, a.softcap, a.bias != 0, a.alibi != nullptr};
}

constexpr int kFewWgs = 4;
template <int DP, bool IS_BF16>
__global__ void __launch_bounds__(kThreads4) __attribute__((amdgpu_waves_per_eu(kFewWgs)))
mfa_kv8_weights_few_kernel(K4Args) {
    typedef op_of<IS_BF16> op_t;
    typedef KeyBlock8<DP> Blk;
    constexpr int KS = DP / 32;
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Walk4 wk;
    if (!wk.start()) return;
    typename Blk::Offsets off;
    off.init(args4(), lane);
    while (true) {
        K4Const& a = args4();
        if (!wk.next(a)) return;
        const int Lk = wk.sq.Lk, dq = Lk - wk.sq.Lq;
        const ScoreOf score = score_of(a);
        const int i_last = (int)div4(wk.ncol - 1, a.by_r);
        // the keys of any column, and of every column
        const int t_lo = lo4(a.wl, dq), t_hi = hi4(a.causal, a.wr, i_last + dq, Lk);
        const int f_lo = lo4(a.wl, i_last + dq), f_hi = hi4(a.causal, a.wr, dq, Lk);
        const int key0 = chunks4(t_lo, t_hi, wk.c0, wk.nch).beg * kChunk4 + 32 * wave;
        const int n1 = t_hi < key0 ? 0 : min(wk.nch, (t_hi - key0) / kChunk4 + 1);  // this wavefront's blocks

        Pages4<WFormat<DP>> pg;
        pg.start(a, wk.b, wk.hkv, Lk, key0, kChunk4);
        struct {
            Blk k;
            float w;
            uint32_t at;
            __amdgpu_buffer_rsrc_t rs;
        } blk;
        auto load = [&](int n) {
            const int row = pg.row_of(key0 + max(min(n, n1 - 1), 0) * kChunk4);
            const bool on = n < n1;
            blk.k.load(pg.rs, off, on ? row * pg.rstride[0] : 0x80000000u, on ? row / kKv8Block * pg.rstride[1] : 0x80000000u);
            // (lanes 0..31 hold the block's weights)
            blk.at = on && lane < 32 ? (uint32_t)((row + lane) * pg.rstride[2]) : 0x80000000u;
            blk.w = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(pg.rs[2], blk.at, 0, 0));
            blk.rs = pg.rs[2];
        };
        // queries: lane (column l16, group grp) holds elements Blk::element(grp, s) .. + 7;
        // the products' registers are columns 4 grp + e
        op_t qf[KS];
        float nlse[4], slope[4];
        int lo[4], hi[4], center[4];
        {
            const int i = (int)div4(l16, a.by_r), h = wk.hkv * a.R + l16 - i * a.R;
            const bool in = l16 < wk.ncol;
            const char* q = a.q + row_off4(a.cu_q != nullptr, wk.b, wk.sq.q0, in ? i : 0, in ? h : 0, a.qb, a.qs, a.qh) * 2;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                u32x4_t w = {0, 0, 0, 0};
                if (in) w = *reinterpret_cast<const u32x4_t*>(q + Blk::element(grp, s) * 2);
                qf[s] = __builtin_bit_cast(op_t, w);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int col = 4 * grp + e, i = (int)div4(col, a.by_r), h = wk.hkv * a.R + col - i * a.R;
            const bool in = col < wk.ncol;
            center[e] = i + dq;
            lo[e] = lo4(a.wl, center[e]);
            hi[e] = in ? hi4(a.causal, a.wr, center[e], Lk) : -1;
            nlse[e] = neg_lse2(a, in, wk.b, wk.sq.q0, i, h);
            slope[e] = score.alibi && in ? a.alibi[wk.b * a.alibi_bstride + h] : 0.f;
        }
        load(0);
        // (waited for here: a wait inside the loop would drain the codes' loads too)
#pragma unroll
        for (int s = 0; s < KS; ++s) pin(qf[s]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            pin(nlse[e]);
            pin(slope[e]);
        }
        for (int n = 0; n < n1; ++n) {
            const int j = key0 + n * kChunk4;
            f32x4_t st[2];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                st[kk] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const op_t kf = blk.k.template k_operand<op_t>(kk, s, grp);
                    if constexpr (IS_BF16) st[kk] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qf[s], kf, st[kk], 0, 0, 0);
                    else st[kk] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qf[s], kf, st[kk], 0, 0, 0);
                }
            }
            const float sk = blk.k.k_scale(), old = j + lane < dq ? blk.w : 0.f;
            const uint32_t at = blk.at;
            const __amdgpu_buffer_rsrc_t rs = blk.rs;
            load(n + 1);
            const bool masked = j < f_lo || j + 31 > f_hi;
            float sum[2];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const int key = j + 16 * kk + l16;
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = fast_exp2(score(st[kk][e], sk, nlse[e], slope[e], center[e] - key));
                    if (masked) p[e] = ((key >= lo[e]) & (key <= hi[e])) ? p[e] : 0.f;
                }
                sum[kk] = sum_groups4((p[0] + p[1]) + (p[2] + p[3]));
            }
            // lane 16 kk + l16 has the sum of its own key
            const float w = old + (grp & 1 ? sum[1] : sum[0]);
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(w), rs, at, 0, 0);
        }
    }
}

constexpr int kWCols = 64;     // columns in LDS
constexpr int kManyWgs = 2;
template <int DP, bool IS_BF16, bool BIAS>
__global__ void __launch_bounds__(kThreads4) __attribute__((amdgpu_waves_per_eu(kManyWgs)))
mfa_kv8_weights_many_kernel(K4Args) {
    typedef op_of<IS_BF16> op_t;
    constexpr int DS = DP / 16, CPR = DP / 8, QST = DP + 8, NQ = kWCols * CPR / kThreads4;
    static_assert(kWCols * CPR % kThreads4 == 0, "whole rounds of loads");
    __shared__ __attribute__((aligned(16))) uint16_t q_s[2][kWCols * QST];
    __shared__ __attribute__((aligned(16))) float nlse_s[2][kWCols], slope_s[2][BIAS ? kWCols : 1];
    __shared__ __attribute__((aligned(16))) int center_s[2][kWCols];
    __shared__ float sum_s[2][64];
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave & 1, cg = wave >> 1;
    Walk4 wk;
    if (!wk.start()) return;
    while (true) {
        if (!wk.next(args4())) return;
        K4Const& a = args4();
        const int Lk = wk.sq.Lk, dq = Lk - wk.sq.Lq;
        ScoreOf score = score_of(a);
        score.bias = BIAS;
        const int i_last = (int)div4(wk.ncol - 1, a.by_r);
        const int t_lo = lo4(a.wl, dq), t_hi = hi4(a.causal, a.wr, i_last + dq, Lk);
        const Chunks4 ch = chunks4(t_lo, t_hi, wk.c0, wk.nch);
        Pages4<WFormat<DP>> pg;
        pg.start(a, wk.b, wk.hkv, Lk, ch.beg * kChunk4 + 64 * kg, kChunk4);
        for (int c = ch.beg; c < ch.end; ++c) {
            const int j0 = c * kChunk4, j = j0 + 64 * kg;
            // ---- this wavefront's 64 keys: lane (key l32, half) of tile kt holds elements
            // 32 p + 16 half + 0..15, steps 2 p and 2 p + 1 of the product
            op_t kf[2][DS];
            const int row = pg.row_of(j);
            const uint32_t at = (uint32_t)((row + lane) * pg.rstride[2]);
            const float before = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(pg.rs[2], at, 0, 0));
            const uint8_t ks = __builtin_amdgcn_raw_buffer_load_b8(pg.rs[1], (uint32_t)(row / kKv8Block * pg.rstride[1]), 0, 0);
            {
                u32x4_t raw[2][DP / 32];
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int p = 0; p < DP / 32; ++p)
                        raw[kt][p] = __builtin_amdgcn_raw_buffer_load_b128(
                            pg.rs[0], (uint32_t)((row + 32 * kt + l32) * pg.rstride[0] + 32 * p + 16 * half), 0, 0);
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int p = 0; p < DP / 32; ++p) {
                        kf[kt][2 * p] = kv8_operand<op_t>(raw[kt][p][0], raw[kt][p][1]);
                        kf[kt][2 * p + 1] = kv8_operand<op_t>(raw[kt][p][2], raw[kt][p][3]);
                    }
            }
            const float sk = kv8_scale(ks);
            // ---- the columns that see any key of the chunk, 64 at a time
            K4Const& b = args4();
            const int jl = min(j0 + kChunk4 - 1, Lk - 1);
            int i0 = 0, i1 = wk.sq.Lq;
            if (b.causal) i0 = max(i0, j0 - dq);
            if (b.wr >= 0) i0 = max(i0, (int)max((int64_t)j0 - b.wr - dq, (int64_t)0));
            if (b.wl >= 0) i1 = (int)min((int64_t)i1, (int64_t)jl + b.wl - dq + 1);
            const int cbeg = i0 < i1 ? i0 * b.R / kWCols * kWCols : 0, cend = i0 < i1 ? i1 * b.R : 0;
            u32x4_t qr[NQ];
            float nl = 0.f, sl = 0.f;
            auto qload = [&](int col0) {
                K4Const& e = args4();
#pragma unroll
                for (int x = 0; x < NQ; ++x) {
                    const int u = tid + kThreads4 * x, col = col0 + u / CPR, d = 8 * (u % CPR);
                    const int i = (int)div4(col, e.by_r), h = wk.hkv * e.R + col - i * e.R;
                    qr[x] = u32x4_t{0, 0, 0, 0};
                    if (col < wk.ncol)
                        qr[x] = *reinterpret_cast<const u32x4_t*>(
                            e.q + (row_off4(e.cu_q != nullptr, wk.b, wk.sq.q0, i, h, e.qb, e.qs, e.qh) + d) * 2);
                }
                if (tid < kWCols) {
                    const int col = col0 + tid, i = (int)div4(col, e.by_r), h = wk.hkv * e.R + col - i * e.R;
                    nl = neg_lse2(e, col < wk.ncol, wk.b, wk.sq.q0, i, h);
                    if (BIAS && score.alibi) sl = col < wk.ncol ? e.alibi[wk.b * e.alibi_bstride + h] : 0.f;
                }
            };
            auto qstore = [&](int to, int col0) {
#pragma unroll
                for (int x = 0; x < NQ; ++x) {
                    const int u = tid + kThreads4 * x;
                    *reinterpret_cast<u32x4_t*>(q_s[to] + u / CPR * QST + 8 * (u % CPR)) = qr[x];
                }
                if (tid < kWCols) {
                    nlse_s[to][tid] = nl;
                    if constexpr (BIAS) slope_s[to][tid] = sl;
                    center_s[to][tid] = (int)div4(col0 + tid, args4().by_r) + dq;
                }
            };
            float acc[2] = {0.f, 0.f};
            if (cbeg < cend) qload(cbeg);
            __syncthreads();  // (the last chunk's tiles and sums are read)
            if (cbeg < cend) qstore(0, cbeg);
            __syncthreads();
            for (int col0 = cbeg, buf = 0; col0 < cend; col0 += kWCols, buf ^= 1) {
                const bool more = col0 + kWCols < cend;
                if (more) qload(col0 + kWCols);
                const int cw = col0 + 32 * cg;  // this wavefront's columns
                if (cw < wk.ncol) {
                    f32x16_t s[2];
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[kt][r] = 0.f;
#pragma unroll
                    for (int t = 0; t < DS; ++t) {
                        const op_t qf = *reinterpret_cast<const op_t*>(q_s[buf] + (32 * cg + l32) * QST + 32 * (t >> 1) + 16 * half + 8 * (t & 1));
#pragma unroll
                        for (int kt = 0; kt < 2; ++kt) {
                            if constexpr (IS_BF16) s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf, kf[kt][t], s[kt], 0, 0, 0);
                            else s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(qf, kf[kt][t], s[kt], 0, 0, 0);
                        }
                    }
                    // register r is column cw + 8 (r / 4) + 4 half + r % 4
                    K4Const& e = args4();
                    const int ca = (int)div4(cw, e.by_r) + dq, cb = (int)div4(min(cw + 31, wk.ncol - 1), e.by_r) + dq;
                    const bool masked = j < lo4(e.wl, cb) || j + 63 > hi4(e.causal, e.wr, ca, Lk);
                    const int causal = e.causal, wl = e.wl, wr = e.wr;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int at0 = 32 * cg + 8 * g + 4 * half;
                        const f32x4_t nls = *reinterpret_cast<const f32x4_t*>(nlse_s[buf] + at0);
                        f32x4_t sls = {0.f, 0.f, 0.f, 0.f};
                        if (BIAS) sls = *reinterpret_cast<const f32x4_t*>(slope_s[buf] + at0);
                        int cen[4] = {0, 0, 0, 0};
                        if (BIAS || masked) {
#pragma unroll
                            for (int r = 0; r < 4; ++r) cen[r] = center_s[buf][at0 + r];
                        }
#pragma unroll
                        for (int kt = 0; kt < 2; ++kt) {
                            const int key = j + 32 * kt + l32;
                            float p[4];
#pragma unroll
                            for (int r = 0; r < 4; ++r) p[r] = fast_exp2(score(s[kt][4 * g + r], sk, nls[r], sls[r], cen[r] - key));
                            if (masked) {
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    const bool sees = (key >= lo4(wl, cen[r])) & (key <= hi4(causal, wr, cen[r], Lk)) &
                                                      (nls[r] != -INFINITY);
                                    p[r] = sees ? p[r] : 0.f;
                                }
                            }
                            acc[kt] += (p[0] + p[1]) + (p[2] + p[3]);
                        }
                    }
                }
                if (more) qstore(buf ^ 1, col0 + kWCols);
                __syncthreads();
            }
            // lane 32 kt + l32 has the sum of its own key
            const float s0 = sum_halves(acc[0]), s1 = sum_halves(acc[1]);
            const float sum = half ? s1 : s0;
            if (cg == 1) sum_s[kg][lane] = sum;
            __syncthreads();
            if (cg == 0) {
                const float w = (j + lane < dq ? before : 0.f) + (sum + sum_s[kg][lane]);
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(w), pg.rs[2], at, 0, 0);
            }
        }
    }
}

typedef void (*w8_fn)(K4Args);
template <int DP>
w8_fn weights_of(bool few, bool bf16, bool bias) {
    if (few) return bf16 ? (w8_fn)mfa_kv8_weights_few_kernel<DP, true> : (w8_fn)mfa_kv8_weights_few_kernel<DP, false>;
    if (bias) return bf16 ? (w8_fn)mfa_kv8_weights_many_kernel<DP, true, true> : (w8_fn)mfa_kv8_weights_many_kernel<DP, false, true>;
    return bf16 ? (w8_fn)mfa_kv8_weights_many_kernel<DP, true, false> : (w8_fn)mfa_kv8_weights_many_kernel<DP, false, false>;
}
w8_fn weights_of(int dp, bool few, bool bf16, bool bias) {
    switch (dp) {
        case 32: return weights_of<32>(few, bf16, bias);
        case 64: return weights_of<64>(few, bf16, bias);
        case 96: return weights_of<96>(few, bf16, bias);
        default: return weights_of<128>(few, bf16, bias);
    }
}

int w8err(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(mfa_error_buffer(), 512, fmt, ap);
    va_end(ap);
    return code;
}

}  // namespace

extern "C" {

int mfa_kv8_weights_params_size(void) { return (int)sizeof(mfa_kv8_weights_params); }

int mfa_kv8_weights(const mfa_kv8_weights_params* p, void* stream) {
    static const char who[] = "mfa_kv8_weights";
    mfa_error_buffer()[0] = 0;
    if (!p) return w8err(MFA_ERR_INVALID, "%s: params is NULL", who);
    mfa_kv8_fwd_params f = p->fwd;
    f.cache.v = f.cache.k;  // (neither V nor an output here)
    f.o = const_cast<void*>(f.q);
    f.o_batch_stride = f.o_seq_stride = f.o_head_stride = 0;
    K4Args a;
    const int rc = mfa_kv_args(&f, who, &a);
    if (rc != MFA_OK || a.rows_q == 0 || f.batch == 0) return rc;
    auto bad = [](const void* x) { return !x || (reinterpret_cast<uintptr_t>(x) & 3); };
    if (bad(f.softmax_lse)) return w8err(MFA_ERR_INVALID, "%s: softmax_lse is required", who);
    if (f.cache.num_pages > 0 && bad(p->weights)) return w8err(MFA_ERR_INVALID, "%s: weights are required", who);
    if (p->weight_row_stride < 0 || p->weight_head_stride < 0)
        return w8err(MFA_ERR_INVALID, "%s: row and head strides must be >= 0", who);
    if (f.cache.page_block_size * p->weight_row_stride >= (1LL << 29))
        return w8err(MFA_ERR_INVALID, "%s: the rows of a page must span less than 2 GiB", who);
    a.v = Kv4Pool{reinterpret_cast<uint8_t*>(p->weights), nullptr, p->weight_page_stride * 4, p->weight_row_stride * 4,
                  p->weight_head_stride * 4, 0, 0, 0};
    // Sequences of at most 16 columns, then those of more (a varlen call's are known on
    // the device only: both)
    const bool varlen = f.cu_seqlens_q != nullptr;
    const int64_t cols = (varlen ? (int64_t)a.rows_q : f.seqlen_q) * (int64_t)a.R;
    const int64_t chunks = std::max<int64_t>(1, ((int64_t)a.max_k + kChunk4 - 1) / kChunk4);
    const int64_t units = (varlen ? std::min<int64_t>(f.batch, a.rows_q) : f.batch) * (int64_t)a.Hkv;
    if (cols > 0x3fffffff || units > 0x3fffffff || units * chunks > 0x7fffffffLL)
        return w8err(MFA_ERR_INVALID, "%s: problem too large", who);
    const int cus = mfa_chip_cus(stream);
    for (int few = 1; few >= 0; --few) {
        if (few ? !varlen && cols > 16 : cols <= 16) continue;
        a.cols = few ? 16 : 0x3fffffff;  // (one unit per sequence and K/V head)
        a.min_cols = few ? 1 : 17;
        a.max_cols = few ? 16 : 0x7fffffff;
        a.G = (int32_t)std::min<int64_t>(units * chunks, (int64_t)cus * (few ? kFewWgs : kManyWgs));
        a.xcds = !few && a.G % 8 == 0 ? 8 : 1;  // (neighbouring chunks of a K/V head share its queries in their XCD's L2)
        const w8_fn fn = weights_of(f.head_dim, few != 0, f.dtype == MFA_DTYPE_BF16, a.bias != 0);
        hipLaunchKernelGGL(fn, dim3(a.G), dim3(kThreads4), 0, static_cast<hipStream_t>(stream), a);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return w8err(MFA_ERR_LAUNCH, "%s: launch failed: %s", who, hipGetErrorString(e));
    return MFA_OK;
}

}  // extern "C"
