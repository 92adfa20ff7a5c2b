// mfa_norm_rope.hip -- RMS norm of every query and key head and the rotation of
// its position, forward and backward (mfa_norm_rope, mfa_norm_rope_bwd in
// include/mfa.h).
//
// Bound by memory: a row (one head of one token) is held in the registers of LPR
// neighbouring lanes, 8 elements each, so it is read once and written once; its
// sum of squares takes log2(LPR) cross-lane steps.  A lane holds four elements
// of the first and four of the second half of the rotated part (or 8 adjacent
// ones, interleaved), so both elements of a pair are in one lane.  Shapes that
// do not divide into such pieces, and unaligned tensors, take single elements
// (MODE kAny).
// Backward reads x and g once and writes dx; the statistics are formed again
// from x.  A lane keeps the weight gradient of its 8 elements over all rows that
// it walks; a workgroup adds its lanes' and stores one partial sum, and a second
// kernel adds the workgroups' in order (no atomics).
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>

#include "mfa_kv4.h"

namespace {

constexpr int kNThreads = 256;
// Workgroups per tensor: a row per lane group up to here, then walks.  Few, as a
// workgroup's start (weights, first positions, first angles) is a chain of loads:
// 8192 tokens of 16 + 16 heads of 128 in bf16 took 28.4 us forward with 768 (3 per
// CU; 35.0 with 4096, 30.2 with 512) and 42.6 us backward with 640 (47.8 with 1024,
// 44.9 with 512, 53 with 256); two rows of a lane group in flight at once measured
// 27.5 and 44.3.  With non-temporal stores 27.7 and 39.4 us (4.9 and 5.1 TB/s read
// and written, a large library copy reaches 5.15).
constexpr int kNFwdPerCu = 3;
constexpr int kNMaxBlocks = 640;  // (backward: each leaves a partial sum of the weight gradients)
enum { kHalf = 0, kInterleaved = 1, kAny = 2 };

struct NTensor {
    const char* x;
    const char* g;
    char* out;  // forward: result, backward: gradient; contiguous
    const char* w;
    int64_t xb, xs, xh, gb, gs, gh;  // element strides
    int32_t H;
    FastDiv by_h;
    int64_t rows;
};
struct NArgs {
    NTensor t[2];  // q, k
    const char* cos;
    const char* sin;
    int64_t table_stride;
    const uint32_t* pos;  // 32-bit words
    int64_t pos_b;        // elements
    int32_t pos64, table_rows;
    int32_t L, D, rot;
    FastDiv by_l;
    int32_t interleaved, wdt, tdt;
    float eps, inv_d;
    int32_t blocks[2];  // workgroups of q, k
    float* ws;          // [blocks[0] + blocks[1]][D] partial weight sums
    char* dw[2];
};

template <int DT>
__device__ __forceinline__ float load1(const char* p) {
    if constexpr (DT == MFA_DTYPE_F32) return *reinterpret_cast<const float*>(p);
    else if constexpr (DT == MFA_DTYPE_BF16) return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16);
    else return (float)*reinterpret_cast<const _Float16*>(p);
}
__device__ __forceinline__ float load1(const char* p, int64_t i, int dt) {
    return dt == MFA_DTYPE_F32 ? load1<MFA_DTYPE_F32>(p + 4 * i) : dt == MFA_DTYPE_BF16 ? load1<MFA_DTYPE_BF16>(p + 2 * i) : load1<MFA_DTYPE_F16>(p + 2 * i);
}
template <int DT>
__device__ __forceinline__ void store1(char* p, float x) {
    if constexpr (DT == MFA_DTYPE_F32) *reinterpret_cast<float*>(p) = x;
    else if constexpr (DT == MFA_DTYPE_BF16) *reinterpret_cast<__bf16*>(p) = (__bf16)x;
    else *reinterpret_cast<_Float16*>(p) = (_Float16)x;
}
// four consecutive elements
template <int DT>
__device__ __forceinline__ void load4(const char* p, float* x) {
    if constexpr (DT == MFA_DTYPE_F32) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
        const u32x2_t v = *reinterpret_cast<const u32x2_t*>(p);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (DT == MFA_DTYPE_BF16) {
                x[2 * i] = __uint_as_float(v[i] << 16);
                x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
            } else {
                const k4_f16x2_t h = __builtin_bit_cast(k4_f16x2_t, (uint32_t)v[i]);
                x[2 * i] = (float)h[0];
                x[2 * i + 1] = (float)h[1];
            }
        }
    }
}
template <int DT>
__device__ __forceinline__ void store4(char* p, const float* x) {
    if constexpr (DT == MFA_DTYPE_F32) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        u32x2_t v;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (DT == MFA_DTYPE_BF16) v[i] = __builtin_bit_cast(uint32_t, k4_bf16x2_t{(__bf16)x[2 * i], (__bf16)x[2 * i + 1]});
            else v[i] = __builtin_bit_cast(uint32_t, k4_f16x2_t{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
        }
        store_stream(reinterpret_cast<u32x2_t*>(p), v);
    }
}

// what is loaded in place of a position or a table row that is not there (at most
// four floats from its start)
alignas(16) __device__ const uint32_t kZeros[64] = {0};

// Token and head of a row, and the table row of the token's position.
struct Where {
    int b, i, h;
    int64_t row;
    bool ok;  // the position is in the table
};
__device__ __forceinline__ Where where_of(const NArgs& a, const NTensor& t, int64_t r) {
    Where w;
    const uint32_t tok = quotient((uint32_t)r, t.by_h);
    w.h = (int)((uint32_t)r - tok * (uint32_t)t.H);
    w.b = (int)quotient(tok, a.by_l);
    w.i = (int)(tok - (uint32_t)w.b * (uint32_t)a.L);
    // (low and high word of an int64, the word twice of an int32; without positions
    // a zero is loaded, and the token's place counts)
    const uint32_t* p = a.pos ? a.pos : kZeros;
    const int64_t at = a.pos ? (w.b * a.pos_b + w.i) << a.pos64 : 0;
    const uint32_t lo = p[at], hi = p[at + a.pos64];
    const uint32_t pos = a.pos ? lo : (uint32_t)w.i;
    w.ok = pos < (uint32_t)a.table_rows && (!a.pos64 || hi == 0);
    w.row = w.ok ? pos : 0;
    return w;
}

// A lane's elements: pair i of its four is (x[i], x[4 + i]).
template <int MODE, int LPR>
struct Lane {
    int d0, d1;     // (not kAny) first element of each four
    int p0;         // first pair of the rotation, or >= rot / 2
    bool in, turn;  // lane holds elements / they are rotated
    int sub;

    __device__ __forceinline__ Lane(const NArgs& a) {
        sub = threadIdx.x & (LPR - 1);
        const int nr = a.rot / 8;  // lanes of the rotated part
        turn = sub < nr;
        in = MODE == kAny || sub < a.D / 8;
        p0 = turn ? 4 * sub : 0;
        if (MODE == kHalf && turn) {
            d0 = 4 * sub;
            d1 = a.rot / 2 + 4 * sub;
        } else {
            d0 = in ? 8 * sub : 0;
            d1 = d0 + 4;
        }
    }
    // (kAny) element index of slot i (0..7), or -1: pair p = sub + 16 i
    __device__ __forceinline__ static int element(const NArgs& a, int sub, int i) {
        const int p = sub + LPR * (i & 3), second = i >> 2, half = a.rot / 2;
        const int d = p < half ? (a.interleaved ? 2 * p + second : p + second * half) : a.rot + 2 * (p - half) + second;
        return d < a.D ? d : -1;
    }
    template <int DT>
    __device__ __forceinline__ void load(const NArgs& a, const char* row, float (&x)[8]) const {
        constexpr int ES = DT == MFA_DTYPE_F32 ? 4 : 2;
        if constexpr (MODE == kAny) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = element(a, sub, i);
                x[i] = d >= 0 ? load1<DT>(row + d * ES) : 0.f;
            }
        } else {
            // (a lane without elements loads the row's first ones and drops them)
            float u[8];
            load4<DT>(row + d0 * ES, u);
            load4<DT>(row + d1 * ES, u + 4);
            // (interleaved: adjacent elements are the pairs)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[MODE == kInterleaved ? 4 * (i & 1) + (i >> 1) : i] = in ? u[i] : 0.f;
        }
    }
    template <int DT>
    __device__ __forceinline__ void store(const NArgs& a, char* row, const float (&x)[8]) const {
        constexpr int ES = DT == MFA_DTYPE_F32 ? 4 : 2;
        if constexpr (MODE == kAny) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = element(a, sub, i);
                if (d >= 0) store1<DT>(row + d * ES, x[i]);
            }
        } else if (in) {
            float u[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = x[MODE == kInterleaved ? 4 * (i & 1) + (i >> 1) : i];
            store4<DT>(row + d0 * ES, u);
            store4<DT>(row + d1 * ES, u + 4);
        }
    }
    // element of slot i in x
    __device__ __forceinline__ int slot_element(const NArgs& a, int i) const {
        if constexpr (MODE == kAny) return element(a, sub, i);
        if (!in) return -1;
        if (MODE == kInterleaved) return d0 + 2 * (i & 3) + (i >> 2);
        return i < 4 ? d0 + i : d1 + i - 4;
    }
    __device__ __forceinline__ void weights(const NArgs& a, const char* w, float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = slot_element(a, i);
            x[i] = d < 0 ? 0.f : w ? load1(w, d, a.wdt) : 1.f;
        }
    }
    // cosine and sine of the lane's pairs (1 and 0 where not rotated, NaN at a
    // position outside the table); TDT: the tables' type
    template <int TDT>
    __device__ __forceinline__ void angles(const NArgs& a, const Where& w, float (&c)[4], float (&s)[4]) const {
        constexpr int TS = TDT == MFA_DTYPE_F32 ? 4 : 2;
        const float off = w.ok ? 0.f : __builtin_nanf("");
        if constexpr (MODE != kAny) {
            // (without branches: these loads run beside the elements';
            // zeros stand for a table that has no rows or columns)
            const bool some = a.table_rows > 0 && a.rot > 0;
            const char* cos = some ? a.cos : reinterpret_cast<const char*>(kZeros);
            const char* sin = some ? a.sin : reinterpret_cast<const char*>(kZeros);
            load4<TDT>(cos + (w.row * a.table_stride + p0) * TS, c);
            load4<TDT>(sin + (w.row * a.table_stride + p0) * TS, s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[i] = turn ? c[i] + off : 1.f;
                s[i] = turn ? s[i] + off : 0.f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int p = sub + LPR * i;
                c[i] = 1.f;
                s[i] = 0.f;
                if (p >= a.rot / 2) continue;
                c[i] = w.ok ? load1<TDT>(a.cos + (w.row * a.table_stride + p) * TS) : off;
                s[i] = w.ok ? load1<TDT>(a.sin + (w.row * a.table_stride + p) * TS) : off;
            }
        }
    }
};

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
__device__ __forceinline__ float sum8(const float (&x)[8]) {
    return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
}

template <int DT, int TDT, int MODE, int LPR>
__global__ void __launch_bounds__(kNThreads) mfa_norm_rope_kernel(NArgs a) {
    constexpr int ES = DT == MFA_DTYPE_F32 ? 4 : 2;
    constexpr int RPB = kNThreads / LPR;
    const Lane<MODE, LPR> ln(a);
    const int which = blockIdx.x >= (unsigned)a.blocks[0];
    const NTensor& t = a.t[which];
    const int64_t blk = blockIdx.x - (which ? a.blocks[0] : 0);
    float w[8];
    ln.weights(a, t.w, w);
    for (int64_t r = blk * RPB + threadIdx.x / LPR; r < t.rows; r += (int64_t)a.blocks[which] * RPB) {
        const Where at = where_of(a, t, r);
        float x[8], c[4], s[4], sq[8], y[8];
        ln.template load<DT>(a, t.x + (at.b * t.xb + at.i * t.xs + at.h * t.xh) * ES, x);
        ln.template angles<TDT>(a, at, c, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) sq[i] = x[i] * x[i];
        const float rs = rsqrtf(fmaf(row_sum<LPR>(sum8(sq)), a.inv_d, a.eps));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float u = x[i] * rs * w[i], v = x[4 + i] * rs * w[4 + i];
            y[i] = u * c[i] - v * s[i];
            y[4 + i] = v * c[i] + u * s[i];
        }
        ln.template store<DT>(a, t.out + r * a.D * ES, y);
    }
}

template <int DT, int TDT, int MODE, int LPR>
__global__ void __launch_bounds__(kNThreads) mfa_norm_rope_bwd_kernel(NArgs a) {
    constexpr int ES = DT == MFA_DTYPE_F32 ? 4 : 2;
    constexpr int RPB = kNThreads / LPR;
    __shared__ float sh[4][128];
    const Lane<MODE, LPR> ln(a);
    const int which = blockIdx.x >= (unsigned)a.blocks[0];
    const NTensor& t = a.t[which];
    const int64_t blk = blockIdx.x - (which ? a.blocks[0] : 0);
    float w[8], dw[8];
    ln.weights(a, t.w, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[i] = 0.f;
    for (int64_t r = blk * RPB + threadIdx.x / LPR; r < t.rows; r += (int64_t)a.blocks[which] * RPB) {
        const Where at = where_of(a, t, r);
        float x[8], g[8], c[4], s[4], sq[8], hn[8];
        ln.template load<DT>(a, t.x + (at.b * t.xb + at.i * t.xs + at.h * t.xh) * ES, x);
        ln.template load<DT>(a, t.g + (at.b * t.gb + at.i * t.gs + at.h * t.gh) * ES, g);
        ln.template angles<TDT>(a, at, c, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) sq[i] = x[i] * x[i];
        const float rs = rsqrtf(fmaf(row_sum<LPR>(sum8(sq)), a.inv_d, a.eps));
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // g turned back, then g w n
            const float u = g[i] * c[i] + g[4 + i] * s[i], v = g[4 + i] * c[i] - g[i] * s[i];
            g[i] = u;
            g[4 + i] = v;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] *= rs;
            dw[i] = fmaf(g[i], x[i], dw[i]);
            g[i] *= w[i];
            hn[i] = g[i] * x[i];
        }
        const float mean = row_sum<LPR>(sum8(hn)) * a.inv_d;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = rs * fmaf(-x[i], mean, g[i]);
        ln.template store<DT>(a, t.out + r * a.D * ES, x);
    }
    if (!a.dw[which]) return;
    // the workgroup's sums: over the rows of a wavefront, then over wavefronts
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[i] += __shfl_xor(dw[i], o);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) < LPR) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = ln.slot_element(a, i);
            if (d >= 0) sh[wave][d] = dw[i];
        }
    }
    __syncthreads();
    if (threadIdx.x < (unsigned)a.D)
        a.ws[(int64_t)blockIdx.x * a.D + threadIdx.x] =
            (sh[0][threadIdx.x] + sh[1][threadIdx.x]) + (sh[2][threadIdx.x] + sh[3][threadIdx.x]);
}

// Weight gradients: 8 columns of one tensor per workgroup, 32 partial sums of
// each at a time.
constexpr int kRCols = 8;
__global__ void __launch_bounds__(kNThreads) mfa_norm_rope_dw_kernel(NArgs a) {
    __shared__ float sh[kNThreads];
    const int tiles = (a.D + kRCols - 1) / kRCols;
    const int which = blockIdx.x / tiles, d = (blockIdx.x - which * tiles) * kRCols + threadIdx.x % kRCols;
    if (!a.dw[which]) return;
    const float* ws = a.ws + (which ? (int64_t)a.blocks[0] * a.D : 0);
    float sum = 0.f;
    if (d < a.D) {
#pragma unroll 8
        for (int r = threadIdx.x / kRCols; r < a.blocks[which]; r += kNThreads / kRCols) sum += ws[(int64_t)r * a.D + d];
    }
    sh[threadIdx.x] = sum;
    __syncthreads();
    for (int n = kNThreads / 2; n >= kRCols; n >>= 1) {
        if (threadIdx.x < (unsigned)n) sh[threadIdx.x] += sh[threadIdx.x + n];
        __syncthreads();
    }
    if (threadIdx.x < kRCols && d < a.D) {
        const float x = sh[threadIdx.x];
        if (a.wdt == MFA_DTYPE_F32) store1<MFA_DTYPE_F32>(a.dw[which] + 4 * d, x);
        else if (a.wdt == MFA_DTYPE_BF16) store1<MFA_DTYPE_BF16>(a.dw[which] + 2 * d, x);
        else store1<MFA_DTYPE_F16>(a.dw[which] + 2 * d, x);
    }
}

typedef void (*n_fn)(NArgs);
template <int DT, int TDT, int MODE>
n_fn pick(bool bwd, int lpr) {
    switch (lpr) {
        case 4: return bwd ? mfa_norm_rope_bwd_kernel<DT, TDT, MODE, 4> : mfa_norm_rope_kernel<DT, TDT, MODE, 4>;
        case 8: return bwd ? mfa_norm_rope_bwd_kernel<DT, TDT, MODE, 8> : mfa_norm_rope_kernel<DT, TDT, MODE, 8>;
        default: return bwd ? mfa_norm_rope_bwd_kernel<DT, TDT, MODE, 16> : mfa_norm_rope_kernel<DT, TDT, MODE, 16>;
    }
}
template <int DT, int TDT>
n_fn pick(bool bwd, int mode, int lpr) {
    if (mode == kHalf) return pick<DT, TDT, kHalf>(bwd, lpr);
    if (mode == kInterleaved) return pick<DT, TDT, kInterleaved>(bwd, lpr);
    return bwd ? mfa_norm_rope_bwd_kernel<DT, TDT, kAny, 16> : mfa_norm_rope_kernel<DT, TDT, kAny, 16>;
}
// tables in fp32 or in the tensors' type
template <int DT>
n_fn pick_tables(bool bwd, int tdt, int mode, int lpr) {
    return tdt == MFA_DTYPE_F32 ? pick<DT, MFA_DTYPE_F32>(bwd, mode, lpr) : pick<DT, DT>(bwd, mode, lpr);
}

int nerr(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(mfa_error_buffer(), 512, fmt, ap);
    va_end(ap);
    return code;
}
bool known(int dt) { return dt == MFA_DTYPE_F16 || dt == MFA_DTYPE_BF16 || dt == MFA_DTYPE_F32; }

struct NPlan {
    NArgs a;
    int mode = kAny, lpr = 16;
    bool empty = false;
};

// b: NULL forward
int n_plan(const mfa_norm_rope_params* p, const mfa_norm_rope_bwd_params* b, NPlan* plan, const char* who, int cus) {
    if (!known(p->dtype) || !known(p->dtype_weight) || (p->dtype_table != p->dtype && p->dtype_table != MFA_DTYPE_F32))
        return nerr(MFA_ERR_INVALID, "%s: unknown dtype (%d, weight %d, table %d)", who, p->dtype, p->dtype_weight, p->dtype_table);
    if (p->batch < 0 || p->seqlen < 0 || p->heads_q < 0 || p->heads_kv < 0 || p->table_rows < 0)
        return nerr(MFA_ERR_INVALID, "%s: negative size", who);
    if (p->head_dim <= 0 || p->head_dim > MFA_MAX_HEAD_DIM)
        return nerr(MFA_ERR_UNSUPPORTED, "%s: head_dim %d outside [1, %d]", who, p->head_dim, MFA_MAX_HEAD_DIM);
    if (p->rotary_dim < 0 || p->rotary_dim % 2 || p->rotary_dim > p->head_dim)
        return nerr(MFA_ERR_INVALID, "%s: rotary_dim %d must be even and in [0, head_dim]", who, p->rotary_dim);
    NArgs& a = plan->a;
    memset(&a, 0, sizeof(a));
    const int es = p->dtype == MFA_DTYPE_F32 ? 4 : 2;
    const int64_t tokens = (int64_t)p->batch * p->seqlen;
    if (tokens > 0x7fffffffLL || tokens * p->heads_q > 0x7fffffffLL || tokens * p->heads_kv > 0x7fffffffLL)
        return nerr(MFA_ERR_INVALID, "%s: problem too large", who);
    plan->empty = tokens == 0 || p->heads_q + p->heads_kv == 0;
    const void* x[2] = {p->q, p->k};
    const void* g[2] = {b ? b->dq_out : nullptr, b ? b->dk_out : nullptr};
    void* out[2] = {b ? b->dq : p->q_out, b ? b->dk : p->k_out};
    const void* w[2] = {p->q_weight, p->k_weight};
    const int64_t xs[2][3] = {{p->q_batch_stride, p->q_seq_stride, p->q_head_stride}, {p->k_batch_stride, p->k_seq_stride, p->k_head_stride}};
    int64_t gs[2][3] = {{0, 0, 0}, {0, 0, 0}};
    if (b) {
        gs[0][0] = b->dqo_batch_stride; gs[0][1] = b->dqo_seq_stride; gs[0][2] = b->dqo_head_stride;
        gs[1][0] = b->dko_batch_stride; gs[1][1] = b->dko_seq_stride; gs[1][2] = b->dko_head_stride;
    }
    const int H[2] = {p->heads_q, p->heads_kv};
    // everything 16-byte aligned, in pieces of 8 elements
    bool whole = p->head_dim % 8 == 0 && p->rotary_dim % 8 == 0;
    auto off = [](const void* q, uintptr_t al) { return (reinterpret_cast<uintptr_t>(q) & (al - 1)) != 0; };
    for (int i = 0; i < 2; ++i) {
        NTensor& t = a.t[i];
        t.x = static_cast<const char*>(x[i]);
        t.g = static_cast<const char*>(g[i]);
        t.out = static_cast<char*>(out[i]);
        t.w = static_cast<const char*>(w[i]);
        t.xb = xs[i][0]; t.xs = xs[i][1]; t.xh = xs[i][2];
        t.gb = gs[i][0]; t.gs = gs[i][1]; t.gh = gs[i][2];
        t.H = H[i];
        t.by_h = fast_div(std::max(H[i], 1));
        t.rows = tokens * H[i];
        if (t.rows == 0) continue;
        if (!t.x || !t.out || (b && !t.g)) return nerr(MFA_ERR_INVALID, "%s: NULL tensor pointer", who);
        if (off(t.x, es) || off(t.out, es) || off(t.g, es)) return nerr(MFA_ERR_INVALID, "%s: a tensor is not aligned to its elements", who);
        whole = whole && !off(t.x, 16) && !off(t.out, 16) && !off(t.g, 16);
        for (int j = 0; j < 3; ++j) whole = whole && xs[i][j] % 8 == 0 && gs[i][j] % 8 == 0;
    }
    if (p->rotary_dim > 0 && !plan->empty) {
        if (p->table_rows > 0 && (!p->cos || !p->sin)) return nerr(MFA_ERR_INVALID, "%s: cos and sin are required", who);
        if (p->table_stride < 0) return nerr(MFA_ERR_INVALID, "%s: table_stride must be >= 0", who);
        const int ts = p->dtype_table == MFA_DTYPE_F32 ? 4 : 2;
        if (off(p->cos, ts) || off(p->sin, ts)) return nerr(MFA_ERR_INVALID, "%s: cos or sin is not aligned to its elements", who);
        whole = whole && !off(p->cos, 4 * ts) && !off(p->sin, 4 * ts) && p->table_stride % 4 == 0;
    }
    if (off(p->positions, p->positions_64 ? 8 : 4) || p->positions_batch_stride < 0)
        return nerr(MFA_ERR_INVALID, "%s: positions are not aligned or have a negative stride", who);
    a.cos = static_cast<const char*>(p->cos);
    a.sin = static_cast<const char*>(p->sin);
    // (a table without columns has one row: kZeros stands for it, whatever the position)
    a.table_stride = p->rotary_dim > 0 ? p->table_stride : 0;
    a.pos = static_cast<const uint32_t*>(p->positions);
    a.pos_b = p->positions_batch_stride;
    a.pos64 = p->positions_64 != 0;
    a.table_rows = p->table_rows;
    a.L = p->seqlen;
    a.D = p->head_dim;
    a.rot = p->rotary_dim;
    a.by_l = fast_div(std::max(p->seqlen, 1));
    a.interleaved = p->interleaved != 0;
    a.wdt = p->dtype_weight;
    a.tdt = p->dtype_table;
    a.eps = p->eps;
    a.inv_d = 1.f / p->head_dim;
    plan->mode = !whole ? kAny : p->interleaved ? kInterleaved : kHalf;
    plan->lpr = plan->mode == kAny ? 16 : p->head_dim <= 32 ? 4 : p->head_dim <= 64 ? 8 : 16;
    const int ws = p->dtype_weight == MFA_DTYPE_F32 ? 4 : 2;
    if (off(p->q_weight, ws) || off(p->k_weight, ws) || (b && (off(b->dq_weight, ws) || off(b->dk_weight, ws))))
        return nerr(MFA_ERR_INVALID, "%s: a weight is not aligned to its elements", who);
    const int64_t rpb = kNThreads / plan->lpr, most = b ? kNMaxBlocks : (int64_t)cus * kNFwdPerCu;
    for (int i = 0; i < 2; ++i) a.blocks[i] = (int32_t)std::min<int64_t>((a.t[i].rows + rpb - 1) / rpb, most);
    if (b) {
        a.dw[0] = p->q_weight ? static_cast<char*>(b->dq_weight) : nullptr;
        a.dw[1] = p->k_weight ? static_cast<char*>(b->dk_weight) : nullptr;
    }
    return MFA_OK;
}

// (by the sizes alone, also where alignment decides the lanes per row)
int64_t n_ws_bytes(const NPlan& plan) {
    const NArgs& a = plan.a;
    if (!a.dw[0] && !a.dw[1]) return 0;
    int64_t blocks = 0;
    for (const NTensor& t : a.t) blocks += std::min<int64_t>((t.rows + kNThreads / 16 - 1) / (kNThreads / 16), kNMaxBlocks);
    return blocks * a.D * 4;
}

void n_launch(const NPlan& plan, bool bwd, int dtype, hipStream_t st) {
    const int tdt = plan.a.tdt;
    const n_fn fn = dtype == MFA_DTYPE_F32    ? pick_tables<MFA_DTYPE_F32>(bwd, tdt, plan.mode, plan.lpr)
                    : dtype == MFA_DTYPE_BF16 ? pick_tables<MFA_DTYPE_BF16>(bwd, tdt, plan.mode, plan.lpr)
                                              : pick_tables<MFA_DTYPE_F16>(bwd, tdt, plan.mode, plan.lpr);
    hipLaunchKernelGGL(fn, dim3(plan.a.blocks[0] + plan.a.blocks[1]), dim3(kNThreads), 0, st, plan.a);
}

}  // namespace

extern "C" {

int mfa_norm_rope_params_size(void) { return (int)sizeof(mfa_norm_rope_params); }
int mfa_norm_rope_bwd_params_size(void) { return (int)sizeof(mfa_norm_rope_bwd_params); }

int mfa_norm_rope(const mfa_norm_rope_params* p, void* stream) {
    mfa_error_buffer()[0] = 0;
    if (!p) return nerr(MFA_ERR_INVALID, "mfa_norm_rope: params is NULL");
    NPlan plan;
    const int rc = n_plan(p, nullptr, &plan, "mfa_norm_rope", mfa_chip_cus(stream));
    if (rc != MFA_OK || plan.empty) return rc;
    n_launch(plan, false, p->dtype, static_cast<hipStream_t>(stream));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return nerr(MFA_ERR_LAUNCH, "mfa_norm_rope: launch failed: %s", hipGetErrorString(e));
    return MFA_OK;
}

int64_t mfa_norm_rope_bwd_workspace_bytes(const mfa_norm_rope_bwd_params* p) {
    mfa_error_buffer()[0] = 0;
    if (!p) return nerr(MFA_ERR_INVALID, "mfa_norm_rope_bwd: params is NULL");
    NPlan plan;
    const int rc = n_plan(&p->fwd, p, &plan, "mfa_norm_rope_bwd", mfa_chip_cus(nullptr));
    if (rc != MFA_OK) return rc;
    return plan.empty ? 0 : n_ws_bytes(plan);
}

int mfa_norm_rope_bwd(const mfa_norm_rope_bwd_params* p, void* workspace, int64_t workspace_bytes, void* stream) {
    mfa_error_buffer()[0] = 0;
    if (!p) return nerr(MFA_ERR_INVALID, "mfa_norm_rope_bwd: params is NULL");
    NPlan plan;
    const int rc = n_plan(&p->fwd, p, &plan, "mfa_norm_rope_bwd", mfa_chip_cus(stream));
    if (rc != MFA_OK) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t need = n_ws_bytes(plan);
    if (need && !plan.empty) {
        if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u))
            return nerr(MFA_ERR_INVALID, "mfa_norm_rope_bwd: workspace must be a 256-byte aligned device pointer");
        if (workspace_bytes < need)
            return nerr(MFA_ERR_INVALID, "mfa_norm_rope_bwd: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
        plan.a.ws = static_cast<float*>(workspace);
    }
    if (!plan.empty) n_launch(plan, true, p->fwd.dtype, st);
    // (no rows: the sums are zero)
    if (plan.a.dw[0] || plan.a.dw[1])
        hipLaunchKernelGGL(mfa_norm_rope_dw_kernel, dim3(2 * ((plan.a.D + kRCols - 1) / kRCols)), dim3(kNThreads), 0, st, plan.a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return nerr(MFA_ERR_LAUNCH, "mfa_norm_rope_bwd: launch failed: %s", hipGetErrorString(e));
    return MFA_OK;
}

}  // extern "C"
