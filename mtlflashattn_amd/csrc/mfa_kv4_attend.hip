// mfa_kv4_attend.hip -- attention over a paged 4-bit K/V cache
// (mfa_kv4_fwd in include/mfa.h).
//
// A column is one (query position, query head) pair of a K/V head; a workgroup
// takes NT tiles of 16 columns and walks keys, its four wavefronts every fourth
// 32-key block, each with a softmax state of its own; the four are added at the
// end of the walk.  Per 32-key block a wavefront
//  * loads K straight into the A operand's registers: the order in which the
//    products of a score are added is free, so lane group g of a key's row takes
//    elements g D/4 .. (g+1) D/4 - 1, at D = 128 one 16-byte load that holds one
//    whole scale group, and the queries' operand takes the same order;
//  * turns the codes into bf16 (exact) with v_cvt_scalef32_pk_bf16_fp4 and forms
//    S^T = K Q^T with v_mfma_f32_16x16x32_bf16: lane = column, registers = keys;
//  * turns V into bf16 rows in LDS, whose transposed operand is read with
//    ds_read_b64_tr_b16, and adds O^T += V^T P^T.
// fp16 queries are two bf16 terms (exact), and probabilities are two bf16 terms,
// hi = round(p) and lo = round(p - hi): a row over thousands of near-equal
// weights averages V, and one 16-bit rounding of every weight would be visible
// against its small result.  Sums and statistics are fp32.
//
// Work is dealt by length: every sequence's keys are cut into chunks of 128, the
// chunks of all (sequence, head, column tile) units are laid end to end, and
// workgroup w of G takes chunks [w C / G, (w+1) C / G) of the C there are, so
// ragged batches end together and the lengths are read on the device only.  A
// unit that one workgroup walks alone is stored by it; the parts of any other go
// to the workspace (at most two per workgroup, its first and its last unit) and
// mfa_kv4_merge_kernel adds them in order.
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>

#include "mfa_kv4.h"

namespace {

typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4_t;

constexpr int kThreads4 = 256;
constexpr int kChunk4 = 128;  // keys per chunk: one 32-key block per wavefront
constexpr float kLn2f = 0.6931471805599453f;

struct K4Args {
    const char* q;
    char* o;
    float* lse;
    int64_t qb, qs, qh, ob, os, oh, lse_b, lse_h;
    Kv4Pool k, v;
    const int32_t* bt;
    int64_t bt_b;
    const int32_t* lens;
    const int32_t* cu_q;  // NULL: Lq rows per sequence
    const float* alibi;
    int32_t alibi_bstride;
    int32_t B, Hq, Hkv, R, Lq, max_k;
    int32_t page, npages;
    FastDiv by_page, by_r;
    float scale, scale_log2, softcap, softcap_sk;
    int32_t wl, wr, causal, bias;
    int32_t G;         // workgroups
    int32_t cols;      // columns per unit, 16 NT
    int32_t rows_q;    // rows of q (varlen: all of them)
    int32_t min_cols, max_cols;  // a sequence with fewer or more columns is another launch's
    float* ws_o;       // [G][2][cols][D]
    float* ws_ml;      // [G][2][cols][2] exponent reference, sum of p
};

__device__ __forceinline__ float max_groups4(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
    return max_halves(fmax_nn(__int_as_float(a[0]), __int_as_float(a[1])));
}
__device__ __forceinline__ float sum_groups4(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
    return sum_halves(__int_as_float(a[0]) + __int_as_float(a[1]));
}

__device__ __forceinline__ int lo4(const K4Args& a, int c) { return a.wl >= 0 ? max(c - a.wl, 0) : 0; }
__device__ __forceinline__ int hi4(const K4Args& a, int c, int Lk) {
    int hi = Lk - 1;
    if (a.causal) hi = min(hi, c);
    if (a.wr >= 0) hi = min(hi, c + a.wr);
    return hi;
}

// The work of a sequence: its rows, keys, column tiles and chunks per unit.
struct Seq4 {
    int q0, Lq, Lk, tiles, chunks;
    __device__ __forceinline__ int items(int Hkv) const { return tiles * Hkv * chunks; }
};
__device__ __forceinline__ Seq4 seq4(const K4Args& a, int b) {
    Seq4 s;
    s.q0 = 0;
    s.Lq = a.Lq;
    if (a.cu_q) {
        // (bounded by the tensor whatever the prefix sums hold)
        s.q0 = min(max(a.cu_q[b], 0), a.rows_q);
        s.Lq = min(max(a.cu_q[b + 1], s.q0), a.rows_q) - s.q0;
    }
    s.Lk = min(max(a.lens[b], 0), a.max_k);
    const int cols = s.Lq * a.R;
    s.tiles = cols >= a.min_cols && cols <= a.max_cols ? (cols + a.cols - 1) / a.cols : 0;
    // chunks that hold the widest key range of a tile's rows (at least one: a
    // row without keys is stored too)
    int n = (s.Lk + kChunk4 - 1) / kChunk4;
    if (a.wl >= 0 && (a.causal || a.wr >= 0)) {
        const int64_t span = (int64_t)a.wl + (a.causal ? 0 : a.wr) + (a.cols - 1) / a.R + 1;
        n = (int)min((int64_t)n, (span + kChunk4 - 1) / kChunk4 + 1);
    }
    s.chunks = max(n, 1);
    return s;
}

// Items before sequence b0 + lane + 1 of the 64 sequences from b0 on (inclusive
// prefix sums over the wavefront).
__device__ __forceinline__ int scan64(int x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    return x;
}
__device__ __forceinline__ int items_of(const K4Args& a, int b) { return b < a.B ? seq4(a, b).items(a.Hkv) : 0; }

// all items of the call
__device__ __forceinline__ int total_items(const K4Args& a) {
    const int lane = threadIdx.x & 63;
    int sum = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) sum += items_of(a, b0 + lane);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    return __builtin_amdgcn_readfirstlane(sum);
}
// the sequence of item x, and the items before it
__device__ __forceinline__ int find_item(const K4Args& a, int x, int& before) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int n = items_of(a, b0 + lane), inc = scan64(n) + base;
        const uint64_t past = __ballot(inc > x);
        if (past) {
            const int l = __builtin_ctzll(past);
            before = __builtin_amdgcn_readlane(inc - n, l);
            return b0 + l;
        }
        base = __builtin_amdgcn_readlane(inc, 63);
    }
    before = base;
    return a.B;
}
// items before sequence b
__device__ __forceinline__ int items_before(const K4Args& a, int b) {
    const int lane = threadIdx.x & 63;
    int sum = 0;
    for (int b0 = 0; b0 < b; b0 += 64) sum += b0 + lane < b ? items_of(a, b0 + lane) : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    return __builtin_amdgcn_readfirstlane(sum);
}
__device__ __forceinline__ int first_item(int w, int C, int G) { return (int)((int64_t)w * C / G); }
__device__ __forceinline__ int wg_of_item(int x, int C, int G) { return (int)((((int64_t)x + 1) * G - 1) / C); }

__device__ __forceinline__ void split_bf16(float x, float y, uint32_t& hi, uint32_t& lo) {
    const k4_bf16x2_t h = {(__bf16)x, (__bf16)y};
    hi = __builtin_bit_cast(uint32_t, h);
    const k4_bf16x2_t l = {(__bf16)(x - __uint_as_float(hi << 16)), (__bf16)(y - __uint_as_float(hi & 0xffff0000u))};
    lo = __builtin_bit_cast(uint32_t, l);
}

// four elements of a result row (o = sum of p v, l = sum of p)
template <bool IS_BF16>
__device__ __forceinline__ void store_row4(char* row, int d, const f32x4_t& o, float l) {
    f32x4_t x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = l > 0.f ? o[i] / l : o[i];  // (l = 0: no key, o = 0; NaN stays NaN)
    if constexpr (IS_BF16) {
        typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 v4;
        store_stream(reinterpret_cast<v4*>(reinterpret_cast<__bf16*>(row) + d),
                     v4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]});
    } else {
        typedef __attribute__((__vector_size__(4 * sizeof(_Float16)))) _Float16 v4;
        store_stream(reinterpret_cast<v4*>(reinterpret_cast<_Float16*>(row) + d),
                     v4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]});
    }
}
__device__ __forceinline__ int64_t row_off4(const K4Args& a, int b, int q0, int i, int h, int64_t sb, int64_t ss, int64_t sh) {
    return (a.cu_q ? (int64_t)(q0 + i) * ss : b * sb + i * ss) + h * sh;
}
__device__ __forceinline__ void store_lse4(const K4Args& a, int b, int q0, int i, int h, float m, float l) {
    if (!a.lse) return;
    a.lse[(a.cu_q ? (int64_t)(q0 + i) : b * a.lse_b + i) + h * a.lse_h] =
        m == -INFINITY ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2f;
}

// K registers of a 32-key block: DP/8 bytes of each of two 16-key tiles per
// lane, and their scale bytes (two where a lane's elements cross a scale group:
// DP = 96); V: 32-element groups.
template <int DP>
struct Block4 {
    static constexpr int KW = DP / 32;                // dwords per lane and tile
    static constexpr int VG = (DP + 63) / 64;         // V groups per lane
    uint32_t k[2][KW];
    uint32_t ks[2][DP == 96 ? 2 : 1];
    u32x4_t v[VG];
    uint32_t vs[VG];
};

template <int DP, int NT, bool IS_BF16>
__global__ void __launch_bounds__(kThreads4) __attribute__((amdgpu_waves_per_eu(NT == 1 ? 3 : NT == 2 ? 2 : 1)))
mfa_kv4_kernel(K4Args a) {
    typedef Block4<DP> Blk;
    constexpr int NQ = IS_BF16 ? 1 : 2;  // bf16 terms of a query
    constexpr int KS = DP / 32;          // k-steps of QK^T
    constexpr int DT = DP / 16;          // 16-row tiles of O^T
    constexpr int CPR = DP / 8;          // 16-byte chunks of a bf16 row
    constexpr int GPR = DP / 32;         // scale groups per row
    constexpr int TILE = 32 * DP;        // elements of a V tile
    constexpr int ITEMS = 16 * (DP / 4) / kThreads4 > 0 ? (16 * (DP / 4) + kThreads4 - 1) / kThreads4 : 1;
    constexpr bool QLDS = NT * NQ > 2;   // queries' operands kept in LDS, not in registers
    static_assert(16 * DP * 4 <= TILE * 2, "a V tile holds a wavefront's sums of 16 columns");
    __shared__ __attribute__((aligned(16))) uint16_t vsm[4][TILE];
    __shared__ __attribute__((aligned(16))) uint16_t qsm[QLDS ? NT * NQ * 16 * DP : 8];
    __shared__ float m_s[4][16], l_s[4][16];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, grp = lane >> 4;

    const int C = total_items(a);
    const int G = min(a.G, C);  // (every workgroup below G has an item: the merge reads them all)
    if ((int)blockIdx.x >= G) return;
    int x = first_item(blockIdx.x, C, G);
    const int xend = first_item(blockIdx.x + 1, C, G);
    const int xbeg = x;
    int before;
    int b = __builtin_amdgcn_readfirstlane(find_item(a, x, before));
    if (b >= a.B) return;

    uint16_t* const vt = vsm[wave];
    // 16-byte chunk c of row r of a V tile is in slot c ^ vswz(r): the
    // transposing reads' 16 lanes (four rows) and the stores spread over the banks
    auto vswz = [](int r) { return CPR == 16 ? 2 * (r & 7) : CPR == 8 ? 2 * ((r >> 1) & 3) : CPR == 4 ? 2 * ((r >> 2) & 1) : 0; };
    auto qswz = [](int r) { return CPR == 16 ? r & 15 : CPR == 8 ? (r >> 1) & 7 : (r >> 2) & 3; };
    const float c = a.bias ? kLog2e : a.scale_log2;

    // per-lane byte offsets inside a 32-key block
    int koff[2], ksoff[2][2], voff[Blk::VG], vsoff[Blk::VG], vrow[Blk::VG], vgrp[Blk::VG];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
        const int row = 16 * kk + l16;
        koff[kk] = row * (int)a.k.cr + grp * (DP / 8);
        ksoff[kk][0] = row * (int)a.k.sr + (DP == 96 ? (24 * grp) >> 5 : grp * (DP / 4) / 32);
        ksoff[kk][1] = row * (int)a.k.sr + ((24 * grp + 16) >> 5);
    }
#pragma unroll
    for (int i = 0; i < Blk::VG; ++i) {
        const int cc = 64 * i + lane;
        vrow[i] = cc / GPR;
        vgrp[i] = cc - vrow[i] * GPR;
        const bool in = cc < 32 * GPR;
        voff[i] = in ? vrow[i] * (int)a.v.cr + vgrp[i] * 16 : 0x7fffffff;
        vsoff[i] = in ? vrow[i] * (int)a.v.sr + vgrp[i] : 0x7fffffff;
    }

    Seq4 sq = seq4(a, b);
    while (x < xend) {
        // ---- the unit of item x: (sequence b, K/V head, column tile)
        int off = x - before;
        if (off >= sq.items(a.Hkv)) {  // (the next sequence with rows)
            if (b + 1 >= a.B) return;
            before += sq.items(a.Hkv);
            sq = seq4(a, ++b);
            continue;
        }
        const int unit = off / sq.chunks, c0 = off - unit * sq.chunks;
        const int nch = min(sq.chunks - c0, xend - x);
        const bool whole = nch == sq.chunks;
        const int slot = x == xbeg ? 0 : 1;
        x += nch;
        const int hkv = unit / sq.tiles, col0 = (unit - hkv * sq.tiles) * (16 * NT);
        const int ncol = min(16 * NT, sq.Lq * a.R - col0);
        const int Lk = sq.Lk, dq = Lk - sq.Lq;
        const int i_first = (int)quotient(col0, a.by_r), i_last = (int)quotient(col0 + ncol - 1, a.by_r);
        const int t_lo = lo4(a, i_first + dq), t_hi = hi4(a, i_last + dq, Lk);       // the tile's keys
        const int f_lo = lo4(a, i_last + dq), f_hi = hi4(a, i_first + dq, Lk);       // keys of every row
        const int key0 = (t_lo / kChunk4 + c0) * kChunk4 + 32 * wave;

        // ---- page ids, 64 at a time, one per lane
        const int32_t* bt = a.bt + b * a.bt_b;
        const int last_page = (int)quotient(max(Lk - 1, 0), a.by_page);
        int ids0 = -1, ids = 0;
        auto page_of = [&](int j, int& row) {
            const int idx = (int)quotient(j, a.by_page);
            row = j - idx * a.page;
            if (ids0 < 0 || idx - ids0 >= 64) {
                ids0 = idx;
                ids = bt[min(idx + lane, last_page)];
            }
            return __builtin_amdgcn_readlane(ids, idx - ids0);
        };
        auto live = [&](int n) {
            const int j = key0 + n * kChunk4;
            return n < nch && j <= t_hi && j + 31 >= t_lo;
        };
        auto load = [&](int n, Blk& w) {
            const int j = key0 + n * kChunk4;
            int row;
            const int id = page_of(j, row);
            const bool ok = (uint32_t)id < (uint32_t)a.npages;
            const int64_t pg = ok ? id : 0;
            const int rm1 = min(Lk - j, 32) - 1, on = ok ? -1 : 0;
            auto rsrc = [&](const uint8_t* base, int64_t sp, int64_t sr, int64_t sh, int bytes) {
                const uint8_t* p = base + pg * sp + row * sr + hkv * sh;
                return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0,
                                                         __builtin_amdgcn_readfirstlane((int)(rm1 * sr + bytes) & on),
                                                         kBufferDword3);
            };
            const __amdgpu_buffer_rsrc_t kr = rsrc(a.k.codes, a.k.cp, a.k.cr, a.k.ch, DP / 2);
            const __amdgpu_buffer_rsrc_t ksr = rsrc(a.k.scales, a.k.sp, a.k.sr, a.k.sh, GPR);
            const __amdgpu_buffer_rsrc_t vr = rsrc(a.v.codes, a.v.cp, a.v.cr, a.v.ch, DP / 2);
            const __amdgpu_buffer_rsrc_t vsr = rsrc(a.v.scales, a.v.sp, a.v.sr, a.v.sh, GPR);
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                if constexpr (DP == 128) {
                    const u32x4_t y = __builtin_amdgcn_raw_buffer_load_b128(kr, koff[kk], 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) w.k[kk][i] = y[i];
                } else if constexpr (DP == 96) {
                    const auto y = __builtin_amdgcn_raw_buffer_load_b96(kr, koff[kk], 0, 0);
#pragma unroll
                    for (int i = 0; i < 3; ++i) w.k[kk][i] = y[i];
                } else if constexpr (DP == 64) {
                    const auto y = __builtin_amdgcn_raw_buffer_load_b64(kr, koff[kk], 0, 0);
                    w.k[kk][0] = y[0];
                    w.k[kk][1] = y[1];
                } else {
                    w.k[kk][0] = __builtin_amdgcn_raw_buffer_load_b32(kr, koff[kk], 0, 0);
                }
                w.ks[kk][0] = __builtin_amdgcn_raw_buffer_load_b8(ksr, ksoff[kk][0], 0, 0);
                if constexpr (DP == 96) w.ks[kk][1] = __builtin_amdgcn_raw_buffer_load_b8(ksr, ksoff[kk][1], 0, 0);
            }
#pragma unroll
            for (int i = 0; i < Blk::VG; ++i) {
                w.v[i] = __builtin_amdgcn_raw_buffer_load_b128(vr, voff[i], 0, 0);
                w.vs[i] = __builtin_amdgcn_raw_buffer_load_b8(vsr, vsoff[i], 0, 0);
            }
        };
        Blk cur, nxt;
        bool now = live(0);
        if (now) load(0, cur);

        // ---- queries: lane (column l16, group grp) holds elements
        // grp DP/4 + 8 s .. + 7 of its row as the operand of step s
        bf16x8_t qf[QLDS ? 1 : NT][QLDS ? 1 : NQ][KS];
        int lo[NT], hi[NT], center[NT];
        float slope[NT];
        if constexpr (QLDS) __syncthreads();  // (the last unit's readers are done)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int col = col0 + 16 * t + l16;
            const int i = (int)quotient(col, a.by_r), h = hkv * a.R + col - i * a.R;
            const bool in = 16 * t + l16 < ncol;
            center[t] = i + dq;
            lo[t] = lo4(a, center[t]);
            hi[t] = in ? hi4(a, center[t], Lk) : -1;
            slope[t] = a.alibi && in ? a.alibi[b * a.alibi_bstride + h] : 0.f;
            if (!QLDS || t % 4 == wave) {
                const char* q = a.q + row_off4(a, b, sq.q0, in ? i : 0, in ? h : 0, a.qb, a.qs, a.qh) * 2;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    u32x4_t w = {0, 0, 0, 0};
                    if (in) w = *reinterpret_cast<const u32x4_t*>(q + (grp * (DP / 4) + 8 * s) * 2);
                    u32x4_t term[2] = {w, w};
                    if constexpr (!IS_BF16) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const k4_f16x2_t y = __builtin_bit_cast(k4_f16x2_t, (uint32_t)w[e]);
                            uint32_t h0, l0;
                            split_bf16((float)y[0], (float)y[1], h0, l0);
                            term[0][e] = h0;
                            term[1][e] = l0;
                        }
                    }
#pragma unroll
                    for (int z = 0; z < NQ; ++z) {
                        if constexpr (QLDS)
                            *reinterpret_cast<u32x4_t*>(qsm + ((t * NQ + z) * 16 + l16) * DP +
                                                        (((KS * grp + s) ^ qswz(l16)) << 3)) = term[z];
                        else
                            qf[t][z][s] = __builtin_bit_cast(bf16x8_t, term[z]);
                    }
                }
            }
        }
        if constexpr (QLDS) __syncthreads();
        auto query = [&](int t, int z, int s) -> bf16x8_t {
            if constexpr (QLDS)
                return *reinterpret_cast<const bf16x8_t*>(qsm + ((t * NQ + z) * 16 + l16) * DP +
                                                          (((KS * grp + s) ^ qswz(l16)) << 3));
            else
                return qf[t][z][s];
        };

        float m[NT], l[NT];
        f32x4_t o[NT][DT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[t][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }

        auto compute = [&](int j, const Blk& w) {
            // V to LDS as bf16 rows
#pragma unroll
            for (int i = 0; i < Blk::VG; ++i) {
                if (32 * GPR % 64 == 0 || 64 * i + lane < 32 * GPR) {
                    const float s = kv4_scale(w.vs[i]);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<u32x4_t*>(vt + vrow[i] * DP + (((4 * vgrp[i] + e) ^ vswz(vrow[i])) << 3)) =
                            kv4_bf16x8(w.v[i][e], s);
                }
            }
            // S^T = K Q^T: two 16-key tiles, lane = column, registers = keys
            // j + 16 kk + 4 grp + 0..3
            f32x4_t st[NT][2];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                bf16x8_t kf[KS];
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    uint32_t sb = w.ks[kk][0];
                    if constexpr (DP == 96) {  // elements 24 grp + 8 s .. lie in the first or the second of the lane's groups
                        if (s == 2 || (s == 1 && grp == 1)) sb = w.ks[kk][1];
                    }
                    kf[s] = __builtin_bit_cast(bf16x8_t, kv4_bf16x8(w.k[kk][s], kv4_scale(sb)));
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    st[t][kk] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int z = 0; z < NQ; ++z)
#pragma unroll
                        for (int s = 0; s < KS; ++s)
                            st[t][kk] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[s], query(t, z, s), st[t][kk], 0, 0, 0);
                }
            }
            u32x4_t ph[NT], pl[NT];
            const bool masked = j < f_lo || j + 31 > f_hi;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                f32x4_t(&s)[2] = st[t];
                if (a.bias) {
                    // natural-log units: x = scale*s, soft-cap c tanh(x/c) =
                    // c - 2c / (exp(2x/c) + 1), ALiBi
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float y = s[e >> 2][e & 3];
                        if (a.softcap > 0.f)
                            y = fmaf(-2.f * a.softcap, __builtin_amdgcn_rcpf(fast_exp2(y * a.softcap_sk) + 1.f), a.softcap);
                        else
                            y *= a.scale;
                        if (a.alibi)
                            y = fmaf(-slope[t], fabsf((float)(center[t] - (j + 16 * (e >> 2) + 4 * grp + (e & 3)))), y);
                        s[e >> 2][e & 3] = y;
                    }
                }
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int key = j + 16 * (e >> 2) + 4 * grp + (e & 3);
                        s[e >> 2][e & 3] = ((key >= lo[t]) & (key <= hi[t])) ? s[e >> 2][e & 3] : -INFINITY;
                    }
                }
                float mx = s[0][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) mx = fmax_nn(mx, s[e >> 2][e & 3]);
                // (an integer reference: rescaling is a multiplication by a power of two)
                const float mn = fmax_nn(m[t], __builtin_ceilf(max_groups4(mx) * c));
                if (__any(mn != m[t])) {
                    const float alpha = pow2_diff(m[t], mn);
                    l[t] *= alpha;
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[t][d] *= alpha;
                    m[t] = mn;
                }
                const float mu = m[t] == -INFINITY ? 0.f : m[t];
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = fast_exp2(fmaf(s[e >> 2][e & 3], c, -mu));
                l[t] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t h0, l0;
                    split_bf16(p[2 * e], p[2 * e + 1], h0, l0);
                    ph[t][e] = h0;
                    pl[t][e] = l0;
                }
            }
            // O^T += V^T P^T: k-slots 0..3 / 4..7 of a group are keys 4 grp +
            // 0..3 of the first / second 16
            const int r0 = 4 * grp + (l16 >> 2);
            typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 v4;
            typedef __attribute__((address_space(3))) v4* lp;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const int cb = 2 * d + ((l16 >> 1) & 1);
                const uint16_t* p0 = vt + r0 * DP + ((cb ^ vswz(r0)) << 3) + 4 * (l16 & 1);
                // (the swizzle of row r0 + 16 is row r0's)
                const bf16x8_t va = __builtin_shufflevector(__builtin_amdgcn_ds_read_tr16_b64_v4bf16((lp)(p0)),
                                                            __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lp)(p0 + 16 * DP)),
                                                            0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(bf16x8_t, ph[t]), o[t][d], 0, 0, 0);
                    o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(bf16x8_t, pl[t]), o[t][d], 0, 0, 0);
                }
            }
        };

        for (int n = 0; n < nch; ++n) {
            const bool next = live(n + 1);
            if (next) load(n + 1, nxt);
            if (now) compute(key0 + n * kChunk4, cur);
            cur = nxt;
            now = next;
        }

        // ---- the four wavefronts' sums, 16 columns at a time through their V
        // tiles: elements 4 c .. of column r at 4 (c ^ (r mod 8))
        float* const os = reinterpret_cast<float*>(vt);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (16 * t >= ncol) break;
            const float lt = sum_groups4(l[t]);
#pragma unroll
            for (int d = 0; d < DT; ++d)
                *reinterpret_cast<f32x4_t*>(os + l16 * DP + 4 * ((4 * d + grp) ^ (l16 & 7))) = o[t][d];
            if (grp == 0) {
                m_s[wave][l16] = m[t];
                l_s[wave][l16] = lt;
            }
            __syncthreads();
            const int items = min(16, ncol - 16 * t) * (DP / 4);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int it = tid + kThreads4 * i;
                if (it < items) {
                    const int r = it / (DP / 4), d = 4 * (it - r * (DP / 4));
                    float mc = m_s[0][r];
#pragma unroll
                    for (int z = 1; z < 4; ++z) mc = fmax_nn(mc, m_s[z][r]);
                    f32x4_t oc = {0.f, 0.f, 0.f, 0.f};
                    float lc = 0.f;
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const float e = pow2_diff(m_s[z][r], mc);
                        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(vsm[z]) +
                                                                            r * DP + (d ^ (4 * (r & 7))));
#pragma unroll
                        for (int k = 0; k < 4; ++k) oc[k] = fmaf(y[k], e, oc[k]);
                        lc = fmaf(l_s[z][r], e, lc);
                    }
                    if (whole) {
                        const int col = col0 + 16 * t + r;
                        const int qi = (int)quotient(col, a.by_r), h = hkv * a.R + col - qi * a.R;
                        store_row4<IS_BF16>(a.o + row_off4(a, b, sq.q0, qi, h, a.ob, a.os, a.oh) * 2, d, oc, lc);
                        if (d == 0) store_lse4(a, b, sq.q0, qi, h, mc, lc);
                    } else {
                        const int64_t row = ((int64_t)blockIdx.x * 2 + slot) * (16 * NT) + 16 * t + r;
                        *reinterpret_cast<f32x4_t*>(a.ws_o + row * DP + d) = oc;
                        if (d == 0) *reinterpret_cast<float2*>(a.ws_ml + 2 * row) = make_float2(mc, lc);
                    }
                }
            }
            __syncthreads();
        }
    }
}

// Sum of a row's parts in the order of its keys, one wavefront per (row, query
// head): 32 lanes hold four elements each, and the halves take every other part.
template <int DP, bool IS_BF16>
__global__ void __launch_bounds__(64) mfa_kv4_merge_kernel(K4Args a) {
    const int lane = threadIdx.x, half = lane >> 5, d = 4 * (lane & 31);
    const int row = blockIdx.x / a.Hq, h = blockIdx.x - row * a.Hq;
    const int hkv = h / a.R;
    int b, i;
    if (a.cu_q) {
        // the sequence of this row: the last whose rows begin at or before it
        b = -1;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            const uint64_t at = __ballot(b0 + lane < a.B && a.cu_q[min(b0 + lane, a.B - 1)] <= row);
            if (!at) break;
            b = b0 + 63 - __builtin_clzll(at);
        }
        b = __builtin_amdgcn_readfirstlane(b);
        if (b < 0) return;
        i = row - a.cu_q[b];
    } else {
        b = row / a.Lq;
        i = row - b * a.Lq;
    }
    const Seq4 sq = seq4(a, b);
    if (i < 0 || i >= sq.Lq || sq.tiles == 0) return;  // (rows of no sequence, or of another launch's)
    const int C = total_items(a), G = min(a.G, C);
    const int col = i * a.R + h - hkv * a.R, tile = col / a.cols;
    const int x0 = items_before(a, b) + (hkv * sq.tiles + tile) * sq.chunks;
    const int w0 = wg_of_item(x0, C, G), w1 = wg_of_item(x0 + sq.chunks - 1, C, G);
    if (w0 == w1) return;  // (stored by the workgroup that walked it)
    const int cc = col - tile * a.cols;
    // part w: the workgroup's first unit, unless it began before this one
    auto at = [&](int w) {
        const int slot = first_item(w, C, G) >= x0 ? 0 : 1;
        return ((int64_t)w * 2 + slot) * a.cols + cc;
    };
    float m = -INFINITY;
    for (int w = w0 + lane; w <= w1; w += 64) m = fmax_nn(m, a.ws_ml[2 * at(w)]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmax_nn(m, __shfl_xor(m, o));
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    const bool in = d < DP;
#pragma unroll 4
    for (int w = w0 + half; w <= w1; w += 2) {
        const int64_t r = at(w);
        const float2 ml = *reinterpret_cast<const float2*>(a.ws_ml + 2 * r);
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(a.ws_o + r * DP + (in ? d : 0));
        const float e = pow2_diff(ml.x, m);
        l = fmaf(ml.y, e, l);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = fmaf(y[k], e, acc[k]);
    }
    l = sum_halves(l);
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = sum_halves(acc[k]);
    if (in && half == 0) store_row4<IS_BF16>(a.o + row_off4(a, b, sq.q0, i, h, a.ob, a.os, a.oh) * 2, d, acc, l);
    if (lane == 0) store_lse4(a, b, sq.q0, i, h, m, l);
}

typedef void (*k4_fn)(K4Args);
struct K4Kernels {
    k4_fn attend, merge;
};
template <int DP, bool IS_BF16>
K4Kernels kernels4(int nt) {
    const k4_fn merge = mfa_kv4_merge_kernel<DP, IS_BF16>;
    switch (nt) {
        case 1: return {mfa_kv4_kernel<DP, 1, IS_BF16>, merge};
        case 2: return {mfa_kv4_kernel<DP, 2, IS_BF16>, merge};
        default: return {mfa_kv4_kernel<DP, 4, IS_BF16>, merge};
    }
}
template <bool IS_BF16>
K4Kernels kernels4(int dp, int nt) {
    switch (dp) {
        case 32: return kernels4<32, IS_BF16>(nt);
        case 64: return kernels4<64, IS_BF16>(nt);
        case 96: return kernels4<96, IS_BF16>(nt);
        default: return kernels4<128, IS_BF16>(nt);
    }
}

int k4err(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(mfa_error_buffer(), 512, fmt, ap);
    va_end(ap);
    return code;
}

// Column tiles of 16 per workgroup for sequences of at most `cols` columns.
int tiles_for(int64_t cols) { return cols <= 16 ? 1 : cols <= 32 ? 2 : 4; }

// A launch: the sequences of min_cols to max_cols columns.
struct K4Launch {
    K4Args a;
    int nt;
    int64_t parts;  // rows of its partial results, 0: no merge
};
struct K4Plan {
    K4Launch l[2];
    int n = 0;
    int64_t rows = 0, ws_bytes = 0;
};

int k4_plan(const mfa_kv4_fwd_params* p, K4Plan* plan, int cus) {
    if (!p) return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: params is NULL");
    if (p->dtype != MFA_DTYPE_F16 && p->dtype != MFA_DTYPE_BF16)
        return k4err(MFA_ERR_UNSUPPORTED, "mfa_kv4_fwd: dtype %d (fp16 and bf16 queries)", p->dtype);
    const int D = p->head_dim;
    if (D != 32 && D != 64 && D != 96 && D != 128)
        return k4err(MFA_ERR_UNSUPPORTED, "mfa_kv4_fwd: head_dim %d (32, 64, 96 or 128)", D);
    if (p->batch < 0 || p->seqlen_q < 0 || p->total_q < 0 || p->max_seqlen_k < 0)
        return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: negative size");
    if (p->heads_q <= 0 || p->heads_kv <= 0 || p->heads_q % p->heads_kv)
        return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: num_heads_kv (%d) must divide num_heads_q (%d)", p->heads_kv, p->heads_q);
    if (!(p->softcap >= 0.f)) return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: softcap must be >= 0");
    if (p->window_left < -1 || p->window_right < -1)
        return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: window bounds must be >= -1");
    const int rc = mfa_kv4_check_cache(&p->cache, D, "mfa_kv4_fwd");
    if (rc != MFA_OK) return rc;
    const bool varlen = p->cu_seqlens_q != nullptr;
    const int64_t rows = varlen ? p->total_q : (int64_t)p->batch * p->seqlen_q;
    if (p->batch == 0 || rows == 0) return MFA_OK;
    auto bad = [](const void* x, uintptr_t al) { return !x || (reinterpret_cast<uintptr_t>(x) & (al - 1)); };
    if (bad(p->q, 16) || bad(p->o, 16)) return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: q and o must be 16-byte aligned");
    if (bad(p->cache_seqlens, 4)) return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: cache_seqlens is required");
    const int64_t st[] = {p->q_batch_stride, p->q_seq_stride, p->q_head_stride, p->o_batch_stride, p->o_seq_stride, p->o_head_stride};
    for (int64_t s : st)
        if (s % 8) return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: q and o strides must be multiples of 8 elements");
    if (p->alibi_slopes && p->alibi_batch_stride != 0 && p->alibi_batch_stride != p->heads_q)
        return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: alibi_batch_stride must be 0 or heads_q");

    K4Args a;
    memset(&a, 0, sizeof(a));
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
    const int64_t cap = p->cache.num_pages ? (int64_t)p->cache.max_pages * p->cache.page_block_size : 0;
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
    // clamp windows so center +/- window cannot overflow int32
    const int64_t wmax = std::min<int64_t>(rows + (int64_t)a.max_k + 1, 0x3fffffff);
    a.wl = p->window_left < 0 ? -1 : (int32_t)std::min<int64_t>(p->window_left, wmax);
    a.wr = p->window_right < 0 ? -1 : (int32_t)std::min<int64_t>(p->window_right, wmax);
    a.causal = p->causal ? 1 : 0;
    if (rows > 0x3fffffff || rows * a.Hq > 0x3fffffff) return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: problem too large");

    // Columns per workgroup: a sequence's, at most 64.  The sequences of a
    // varlen call are known on the device only: one launch takes those of at most
    // 16 columns, another the longer ones.
    const int64_t cols = (varlen ? rows : p->seqlen_q) * (int64_t)a.R;
    plan->n = varlen && cols > 16 ? 2 : 1;
    plan->rows = rows;
    const int64_t chunks = std::max<int64_t>(1, ((int64_t)a.max_k + kChunk4 - 1) / kChunk4);
    for (int i = 0; i < plan->n; ++i) {
        K4Launch& l = plan->l[i];
        l.a = a;
        l.nt = tiles_for(plan->n == 2 && i == 0 ? 16 : cols);
        l.a.cols = 16 * l.nt;
        l.a.min_cols = i == 0 ? 1 : 17;
        l.a.max_cols = plan->n == 2 && i == 0 ? 16 : 0x7fffffff;
        // (a bound on the items, which are counted on the device in int32)
        const int64_t tiles = !varlen       ? p->batch * ((cols + l.a.cols - 1) / l.a.cols)
                              : l.a.max_cols == 16 ? std::min<int64_t>(p->batch, rows)
                                                   : (cols + l.a.cols - 1) / l.a.cols + std::min<int64_t>(p->batch, rows);
        const int64_t units = tiles * a.Hkv;
        if (units > 0x3fffffff || units * chunks > 0x7fffffffLL) return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: problem too large");
        l.a.G = (int32_t)std::min<int64_t>(units * chunks, (int64_t)cus * (l.nt == 1 ? 4 : 2));
        l.parts = chunks > 1 ? (int64_t)l.a.G * 2 * l.a.cols : 0;
        plan->ws_bytes += (l.parts * (D * 4 + 8) + 255) / 256 * 256;
    }
    return MFA_OK;
}

}  // namespace

extern "C" {

int mfa_kv4_fwd_params_size(void) { return (int)sizeof(mfa_kv4_fwd_params); }

int64_t mfa_kv4_fwd_workspace_bytes(const mfa_kv4_fwd_params* p) {
    mfa_error_buffer()[0] = 0;
    K4Plan plan;
    const int rc = k4_plan(p, &plan, mfa_chip_cus(nullptr));
    return rc != MFA_OK ? rc : plan.ws_bytes;
}

int mfa_kv4_fwd(const mfa_kv4_fwd_params* p, void* workspace, int64_t workspace_bytes, void* stream) {
    mfa_error_buffer()[0] = 0;
    K4Plan plan;
    const int rc = k4_plan(p, &plan, mfa_chip_cus(stream));
    if (rc != MFA_OK || plan.n == 0) return rc;
    if (plan.ws_bytes) {
        if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u))
            return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: workspace must be a 256-byte aligned device pointer");
        if (workspace_bytes < plan.ws_bytes)
            return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                         (long long)plan.ws_bytes);
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    for (int i = 0; i < plan.n; ++i) {
        K4Launch& l = plan.l[i];
        const K4Kernels k = p->dtype == MFA_DTYPE_BF16 ? kernels4<true>(p->head_dim, l.nt) : kernels4<false>(p->head_dim, l.nt);
        l.a.ws_o = reinterpret_cast<float*>(ws);
        l.a.ws_ml = l.a.ws_o + l.parts * p->head_dim;
        ws += (l.parts * (p->head_dim * 4 + 8) + 255) / 256 * 256;
        hipLaunchKernelGGL(k.attend, dim3(l.a.G), dim3(kThreads4), 0, st, l.a);
        if (l.parts) hipLaunchKernelGGL(k.merge, dim3((unsigned)(plan.rows * l.a.Hq)), dim3(64), 0, st, l.a);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return k4err(MFA_ERR_LAUNCH, "mfa_kv4_fwd: launch failed: %s", hipGetErrorString(e));
    return MFA_OK;
}

}  // extern "C"
