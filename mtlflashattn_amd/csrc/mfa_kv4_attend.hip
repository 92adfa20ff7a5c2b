// mfa_kv4_attend.hip -- attention over a paged 4-bit K/V cache
// (mfa_kv4_fwd in include/mfa.h): sequences of at most 32 columns, the merge of
// parts, and the C entry point.
//
// A column is one (query position, query head) pair of a K/V head; a workgroup
// takes NT tiles of 16 columns and walks keys, its four wavefronts every fourth
// 32-key block, each with a softmax state of its own; the four are added at the
// end of the walk.  Bound by the stream of the cache (68 bytes per key and head at
// head dim 128) where batches are large, by latency where they are small.  Per
// 32-key block a wavefront
//  * loads K straight into the A operand's registers: the order in which the
//    products of a score are added is free, so lane group g of a key's row takes
//    elements g D/4 .. (g+1) D/4 - 1, at D = 128 one 16-byte load that holds one
//    whole scale group, and the queries' operand takes the same order;
//  * turns the codes into bf16 (exact) with v_cvt_scalef32_pk_bf16_fp4 and forms
//    S^T = K Q^T with v_mfma_f32_16x16x32_bf16: lane = column, registers = keys;
//  * turns V into bf16 rows in LDS, whose transposed operand is read with
//    ds_read_b64_tr_b16, and adds O^T += V^T P^T.
// The codes of the next block are on their way into registers from the moment the
// current one's are consumed (two blocks ahead took the registers of the third
// workgroup of a CU: below).
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

#include "mfa_kv4_attend.h"

namespace {

// max / sum over the four 16-lane groups (each lane of a group is one column)
__device__ __forceinline__ float max_groups4(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
    return max_halves(fmax_nn(__int_as_float(a[0]), __int_as_float(a[1])));
}
__device__ __forceinline__ float sum_groups4(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
    return sum_halves(__int_as_float(a[0]) + __int_as_float(a[1]));
}

__device__ __forceinline__ void split_bf16(float x, float y, uint32_t& hi, uint32_t& lo) {
    const k4_bf16x2_t h = {(__bf16)x, (__bf16)y};
    hi = __builtin_bit_cast(uint32_t, h);
    const k4_bf16x2_t l = {(__bf16)(x - __uint_as_float(hi << 16)), (__bf16)(y - __uint_as_float(hi & 0xffff0000u))};
    lo = __builtin_bit_cast(uint32_t, l);
}

// The codes of a 32-key block: K, DP/8 bytes of each of two 16-key tiles per lane
// and their scale bytes (two where a lane's elements cross a scale group: DP =
// 96); V, 32-element groups.
template <int DP>
struct Block4 {
    static constexpr int KW = DP / 32;         // dwords per lane and tile
    static constexpr int VG = (DP + 63) / 64;  // V groups per lane
    uint32_t k[2][KW];
    // (scales stay bytes until they are used: widening them would wait for the loads)
    uint8_t ks[2][DP == 96 ? 2 : 1];
    u32x4_t v[VG];
    uint8_t vs[VG];
};

// Non-temporal buffer loads: a unit holds all columns of its K/V head, so a byte
// of the cache is read once a call (64 sequences of 512 to 16384 keys, Hq=32
// Hkv=8 D=128 bf16: 104.6 us, 108.9 with ordinary loads; 31 of 256 to 4096, which the
// last-level cache holds from call to call: 22.9 and 22.4 us).
constexpr int kOnce4 = 2;
template <int DP>
__device__ __forceinline__ void load_block4(Block4<DP>& w, const __amdgpu_buffer_rsrc_t (&rs)[4], const uint32_t (&koff)[2],
                                            const uint32_t (&ksoff)[2][2], const uint32_t* voff, const uint32_t* vsoff,
                                            uint32_t kr, uint32_t ksr, uint32_t vr, uint32_t vsr) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
        if constexpr (DP == 128) {
            const u32x4_t y = __builtin_amdgcn_raw_buffer_load_b128(rs[0], koff[kk] + kr, 0, kOnce4);
#pragma unroll
            for (int i = 0; i < 4; ++i) w.k[kk][i] = y[i];
        } else if constexpr (DP == 96) {
            const auto y = __builtin_amdgcn_raw_buffer_load_b96(rs[0], koff[kk] + kr, 0, kOnce4);
#pragma unroll
            for (int i = 0; i < 3; ++i) w.k[kk][i] = y[i];
        } else if constexpr (DP == 64) {
            const auto y = __builtin_amdgcn_raw_buffer_load_b64(rs[0], koff[kk] + kr, 0, kOnce4);
            w.k[kk][0] = y[0];
            w.k[kk][1] = y[1];
        } else {
            w.k[kk][0] = __builtin_amdgcn_raw_buffer_load_b32(rs[0], koff[kk] + kr, 0, kOnce4);
        }
        w.ks[kk][0] = __builtin_amdgcn_raw_buffer_load_b8(rs[1], ksoff[kk][0] + ksr, 0, kOnce4);
        if constexpr (DP == 96) w.ks[kk][1] = __builtin_amdgcn_raw_buffer_load_b8(rs[1], ksoff[kk][1] + ksr, 0, kOnce4);
    }
#pragma unroll
    for (int i = 0; i < Block4<DP>::VG; ++i) {
        w.v[i] = __builtin_amdgcn_raw_buffer_load_b128(rs[2], voff[i] + vr, 0, kOnce4);
        w.vs[i] = __builtin_amdgcn_raw_buffer_load_b8(rs[3], vsoff[i] + vsr, 0, kOnce4);
    }
}

// Query rows of no sequence (varlen): 0 and -inf.
template <int DP>
__device__ __forceinline__ void clear_rest() {
    K4Const& a = args4();
    if (!a.cu_q) return;
    const int rows = a.rows_q, first = min(max(a.cu_q[0], 0), rows), end = min(max(a.cu_q[a.B], 0), rows);
    for (int r = 0; r < rows; ++r) {
        if (r >= first && r < end) {
            r = end - 1;
            continue;
        }
        for (int x = threadIdx.x; x < a.Hq * (DP / 8); x += kThreads4) {
            const int h = x / (DP / 8), d = 8 * (x - h * (DP / 8));
            *reinterpret_cast<u32x4_t*>(a.o + (r * a.os + h * a.oh + d) * 2) = u32x4_t{0, 0, 0, 0};
        }
        if (a.lse)
            for (int h = threadIdx.x; h < a.Hq; h += kThreads4) a.lse[r + h * a.lse_h] = -INFINITY;
    }
}

// Workgroups per CU, at NT column tiles: as many as the registers hold (the batch
// above: 98.6 us with three, 107 with two, 118 with four, which spill; at D = 64
// three and four measure the same).
constexpr int wgs4(int nt) { return nt == 1 ? 3 : 2; }
constexpr int kTileWgs4 = 2;  // of 128 columns (a third is dealt work but not resident: 335 us become 369)

template <int DP, int NT, bool IS_BF16>
__global__ void __launch_bounds__(kThreads4) __attribute__((amdgpu_waves_per_eu(wgs4(NT))))
mfa_kv4_kernel(K4Args) {
    typedef Block4<DP> Blk;
    constexpr int NQ = IS_BF16 ? 1 : 2;  // bf16 terms of a query
    constexpr int KS = DP / 32;          // k-steps of QK^T
    constexpr int DT = DP / 16;          // 16-row tiles of O^T
    constexpr int CPR = DP / 8;          // 16-byte chunks of a bf16 row
    constexpr int GPR = DP / 32;         // scale groups per row
    constexpr int TILE = 32 * DP;        // elements of a V tile
    constexpr int ITEMS = (16 * (DP / 4) + kThreads4 - 1) / kThreads4;
    constexpr bool QLDS = NT * NQ > 2;   // queries' operands kept in LDS, not in registers
    static_assert(16 * DP * 4 <= TILE * 2, "a V tile holds a wavefront's sums of 16 columns");
    __shared__ __attribute__((aligned(16))) uint16_t vsm[4][TILE];
    __shared__ __attribute__((aligned(16))) uint16_t qsm[QLDS ? NT * NQ * 16 * DP : 8];
    __shared__ float m_s[4][16], l_s[4][16];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, grp = lane >> 4;
    if (blockIdx.x == gridDim.x - 1) clear_rest<DP>();
    Walk4 wk;
    if (!wk.start()) return;

    uint16_t* const vt = vsm[wave];
    // 16-byte chunk c of row r of a V tile is in slot c ^ vswz(r): the
    // transposing reads' 16 lanes (four rows) and the stores spread over the banks
    auto vswz = [](int r) { return CPR == 16 ? 2 * (r & 7) : CPR == 8 ? 2 * ((r >> 1) & 3) : CPR == 4 ? 2 * ((r >> 2) & 1) : 0; };
    auto qswz = [](int r) { return CPR == 16 ? r & 15 : CPR == 8 ? (r >> 1) & 7 : (r >> 2) & 3; };

    // per-lane byte offsets inside a 32-key block
    uint32_t koff[2], ksoff[2][2], voff[Blk::VG], vsoff[Blk::VG];
    int vrow[Blk::VG], vgrp[Blk::VG];
    {
        K4Const& a = args4();
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int row = 16 * kk + l16;
            koff[kk] = (uint32_t)(row * (int)a.k.cr + grp * (DP / 8));
            ksoff[kk][0] = (uint32_t)(row * (int)a.k.sr + (DP == 96 ? (24 * grp) >> 5 : grp * (DP / 4) / 32));
            ksoff[kk][1] = (uint32_t)(row * (int)a.k.sr + ((24 * grp + 16) >> 5));
        }
#pragma unroll
        for (int i = 0; i < Blk::VG; ++i) {
            const int cc = 64 * i + lane;
            vrow[i] = cc / GPR;
            vgrp[i] = cc - vrow[i] * GPR;
            const bool in = cc < 32 * GPR;
            voff[i] = in ? (uint32_t)(vrow[i] * (int)a.v.cr + vgrp[i] * 16) : 0x80000000u;
            vsoff[i] = in ? (uint32_t)(vrow[i] * (int)a.v.sr + vgrp[i]) : 0x80000000u;
        }
    }

    while (true) {
        K4Const& a = args4();
        if (!wk.next(a)) return;
        const int Lk = wk.sq.Lk, dq = Lk - wk.sq.Lq;
        const bool bias = a.bias != 0, alibi = a.alibi != nullptr;
        const float c = bias ? kLog2e : a.scale_log2;
        const float scale = a.scale, softcap = a.softcap, softcap_sk = a.softcap_sk;
        const int i_first = (int)div4(wk.col0, a.by_r), i_last = (int)div4(wk.col0 + wk.ncol - 1, a.by_r);
        // the keys of any column, and of every column, of the tile
        const int t_lo = lo4(a.wl, i_first + dq), t_hi = hi4(a.causal, a.wr, i_last + dq, Lk);
        const int f_lo = lo4(a.wl, i_last + dq), f_hi = hi4(a.causal, a.wr, i_first + dq, Lk);
        const int key0 = chunks4(t_lo, t_hi, wk.c0, wk.nch).beg * kChunk4 + 32 * wave;
        // this wavefront's blocks with keys: n0 .. n1 - 1
        const int n0 = t_lo - key0 > 31 ? 1 : 0;  // (only the first chunk may begin outside)
        const int n1 = t_hi < key0 ? 0 : min(wk.nch, (t_hi - key0) / kChunk4 + 1);

        Pages4<DP> pg;
        pg.start(a, wk.b, wk.hkv, Lk, key0 + n0 * kChunk4, kChunk4);
        // (always issued, with offsets past the resource behind the last block: on a
        // path without them the wait for a block would be one for all)
        auto load = [&](int n, Blk& w) {
            const int row = pg.row_of(key0 + max(min(n, n1 - 1), 0) * kChunk4);
            const bool on = n < n1;
            const uint32_t kr = on ? row * pg.rstride[0] : 0x80000000u, ksr = on ? row * pg.rstride[1] : 0x80000000u;
            const uint32_t vr = on ? row * pg.rstride[2] : 0x80000000u, vsr = on ? row * pg.rstride[3] : 0x80000000u;
            load_block4<DP>(w, pg.rs, koff, ksoff, voff, vsoff, kr, ksr, vr, vsr);
        };
        // ---- queries: lane (column l16, group grp) holds elements
        // grp DP/4 + 8 s .. + 7 of its row as the operand of step s
        constexpr int NL = QLDS ? 1 : NT;  // column tiles a wavefront loads (QLDS: tile `wave`)
        u32x4_t qw[NL][KS];
        int lo[NT], hi[NT], center[NT];
        float slope[NT];
        {
            K4Const& b = args4();
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int col = wk.col0 + 16 * t + l16;
                const int i = (int)div4(col, b.by_r), h = wk.hkv * b.R + col - i * b.R;
                const bool in = 16 * t + l16 < wk.ncol;
                center[t] = i + dq;
                lo[t] = lo4(b.wl, center[t]);
                hi[t] = in ? hi4(b.causal, b.wr, center[t], Lk) : -1;
                slope[t] = alibi && in ? b.alibi[wk.b * b.alibi_bstride + h] : 0.f;
                if (!QLDS || t == wave) {
                    const char* q = b.q + row_off4(b.cu_q != nullptr, wk.b, wk.sq.q0, in ? i : 0, in ? h : 0, b.qb, b.qs, b.qh) * 2;
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        qw[QLDS ? 0 : t][s] = u32x4_t{0, 0, 0, 0};
                        if (in) qw[QLDS ? 0 : t][s] = *reinterpret_cast<const u32x4_t*>(q + (grp * (DP / 4) + 8 * s) * 2);
                    }
                }
            }
        }
        Blk blk;
        load(n0, blk);
        // (waited for here: a wait inside the loop would drain the codes' loads too)
#pragma unroll
        for (int t = 0; t < NT; ++t) pin(slope[t]);
        bf16x8_t qf[QLDS ? 1 : NT][QLDS ? 1 : NQ][KS];
        if constexpr (QLDS) __syncthreads();  // (the last unit's readers are done)
#pragma unroll
        for (int t = 0; t < NL; ++t) {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                u32x4_t w = qw[t][s];
                pin(w);
                u32x4_t term[2] = {w, w};
                if constexpr (!IS_BF16) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t x = w[e];
                        const k4_f16x2_t y = __builtin_bit_cast(k4_f16x2_t, x);
                        uint32_t h0, l0;
                        split_bf16((float)y[0], (float)y[1], h0, l0);
                        term[0][e] = h0;
                        term[1][e] = l0;
                    }
                }
#pragma unroll
                for (int z = 0; z < NQ; ++z) {
                    if constexpr (QLDS) {
                        if (wave < NT)
                            *reinterpret_cast<u32x4_t*>(qsm + ((wave * NQ + z) * 16 + l16) * DP +
                                                        (((KS * grp + s) ^ qswz(l16)) << 3)) = term[z];
                    } else {
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

        // `refill` is called once the block's registers are consumed
        auto compute = [&](int j, const Blk& w, auto&& refill) {
            // S^T = K Q^T: two 16-key tiles, lane = column, registers = keys
            // j + 16 kk + 4 grp + 0..3
            f32x4_t st[NT][2];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
                for (int t = 0; t < NT; ++t) st[t][kk] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    uint8_t sb = w.ks[kk][0];
                    if constexpr (DP == 96) {  // elements 24 grp + 8 s .. lie in the first or the second of the lane's groups
                        if (s == 2 || (s == 1 && grp == 1)) sb = w.ks[kk][1];
                    }
                    const bf16x8_t kf = __builtin_bit_cast(bf16x8_t, kv4_bf16x8(w.k[kk][s], kv4_scale(sb)));
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int z = 0; z < NQ; ++z)
                            st[t][kk] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, query(t, z, s), st[t][kk], 0, 0, 0);
                }
            }
            // V to LDS as bf16 rows; NaN groups of a block that some column does not
            // see whole as zeros (below)
            const bool masked = j < f_lo || j + 31 > f_hi;
            uint64_t nans[Blk::VG];
#pragma unroll
            for (int i = 0; i < Blk::VG; ++i) {
                const bool nan = masked && w.vs[i] == 255;
                nans[i] = __ballot(nan);
                if (32 * GPR % 64 == 0 || 64 * i + lane < 32 * GPR) {
                    const float s = nan ? 0.f : kv4_scale(w.vs[i]);
                    u32x4_t codes = w.v[i];
                    if (__builtin_expect(kv4_beyond(w.vs[i]), 0)) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) codes[e] = kv4_saturate8(codes[e], w.vs[i]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<u32x4_t*>(vt + vrow[i] * DP + (((4 * vgrp[i] + e) ^ vswz(vrow[i])) << 3)) =
                            kv4_bf16x8(codes[e], s);
                }
            }
            refill();
            u32x4_t ph[NT], pl[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                f32x4_t(&s)[2] = st[t];
                if (bias) {
                    // natural-log units: x = scale*s, soft-cap c tanh(x/c) =
                    // c - 2c / (exp(2x/c) + 1), ALiBi
                    if (softcap > 0.f) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            s[e >> 2][e & 3] = fmaf(-2.f * softcap,
                                                    __builtin_amdgcn_rcpf(fast_exp2(s[e >> 2][e & 3] * softcap_sk) + 1.f), softcap);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) s[e >> 2][e & 3] *= scale;
                    }
                    if (alibi) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            s[e >> 2][e & 3] = fmaf(-slope[t], fabsf((float)(center[t] - (j + 16 * (e >> 2) + 4 * grp + (e & 3)))),
                                                    s[e >> 2][e & 3]);
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
                    float alpha = pow2_diff(m[t], mn);
                    asm volatile("" : "+v"(alpha));  // (keeps the products inside the branch)
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
            // NaN groups for the columns that see their keys (a product with the zero
            // weight of a masked key would reach the others too)
#pragma unroll
            for (int i = 0; i < Blk::VG; ++i) {
                for (uint64_t x = nans[i]; x; x &= x - 1) {
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
        };

        for (int n = n0; n < n1; ++n) compute(key0 + n * kChunk4, blk, [&]() { load(n + 1, blk); });

        // ---- the four wavefronts' sums, 16 columns at a time through their V
        // tiles: elements 4 c .. of column r at 4 (c ^ (r mod 8))
        K4Const& e4 = args4();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float* const os = reinterpret_cast<float*>(vt);
            if (16 * t >= wk.ncol) break;
            const float lt = sum_groups4(l[t]);
#pragma unroll
            for (int d = 0; d < DT; ++d)
                *reinterpret_cast<f32x4_t*>(os + l16 * DP + 4 * ((4 * d + grp) ^ (l16 & 7))) = o[t][d];
            if (grp == 0) {
                m_s[wave][l16] = m[t];
                l_s[wave][l16] = lt;
            }
            __syncthreads();
            const int items = min(16, wk.ncol - 16 * t) * (DP / 4);
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
                    if (wk.whole) {
                        const int col = wk.col0 + 16 * t + r;
                        const int qi = (int)div4(col, e4.by_r), h = wk.hkv * e4.R + col - qi * e4.R;
                        store_row4<IS_BF16>(e4.o + row_off4(e4.cu_q != nullptr, wk.b, wk.sq.q0, qi, h, e4.ob, e4.os, e4.oh) * 2, d, oc, lc);
                        if (d == 0) store_lse4(e4, wk.b, wk.sq.q0, qi, h, mc, lc);
                    } else {
                        const int64_t row = wk.part_row(16 * NT) + 16 * t + r;
                        *reinterpret_cast<f32x4_t*>(e4.ws_o + row * DP + d) = oc;
                        if (d == 0) *reinterpret_cast<float2*>(e4.ws_ml + 2 * row) = make_float2(mc, lc);
                    }
                }
            }
            __syncthreads();
        }
    }
}

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
template <int DP, bool IS_BF16, int T>
__global__ void __launch_bounds__(T) mfa_kv4_merge_kernel(K4Args, K4Args) {
    constexpr int kMergeCols = merge_cols(T);
    __shared__ f32x4_t o_s[T];
    __shared__ float2 ml_s[T];
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
    float m = -INFINITY, l = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](float mw, float lw, const f32x4_t& y) {
        const float mn = fmax_nn(m, mw), e0 = pow2_diff(m, mn), e1 = pow2_diff(mw, mn);
        l = fmaf(lw, e1, l * e0);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = fmaf(y[k], e1, acc[k] * e0);
        m = mn;
    };
    auto walk = [&](auto ahead, int P) {
        constexpr int N = decltype(ahead)::value;
        for (int v0 = w0 + g; v0 <= w1; v0 += P * N) {
            float2 ml[N];
            f32x4_t y[N];
#pragma unroll
            for (int z = 0; z < N; ++z) {
                const int64_t row = at(min(v0 + P * z, w1)) + r;
                ml[z] = *reinterpret_cast<const float2*>(ws_ml + 2 * row);
                y[z] = *reinterpret_cast<const f32x4_t*>(ws_o + row * DP + d);
            }
#pragma unroll
            for (int z = 0; z < N; ++z)
                if (v0 + P * z <= w1) add(ml[z].x, ml[z].y, y[z]);
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
        __syncthreads();
        if (g > 0) return;
        for (int z = 1; z < P; ++z) add(ml_s[tid + z * S].x, ml_s[tid + z * S].y, o_s[tid + z * S]);
    }
    if (in) {
        const int col = g4.col0 + cbeg + r, i = (int)div4(col, a.by_r), h = g4.hkv * a.R + col - i * a.R;
        store_row4<IS_BF16>(a.o + row_off4(a.cu_q != nullptr, g4.b, g4.q0, i, h, a.ob, a.os, a.oh) * 2, d, acc, l);
        if (d == 0) store_lse4(a, g4.b, g4.q0, i, h, m, l);
    }
}
static_assert(16 % merge_cols(kMergeFew) == 0 && kTileCols4 % merge_cols(kMergeMany) == 0, "whole blocks per unit");

typedef void (*k4_fn)(K4Args);
typedef void (*k4_merge_fn)(K4Args, K4Args);
struct K4Kernels {
    k4_fn attend;
    k4_merge_fn merge;
};
// cols: columns of a unit, 16, 32 or kTileCols4; threads: of the merge's blocks
template <int DP, bool IS_BF16>
K4Kernels kernels4(int cols, bool bias, int threads) {
    const k4_merge_fn merge = threads == kMergeFew ? mfa_kv4_merge_kernel<DP, IS_BF16, kMergeFew> : mfa_kv4_merge_kernel<DP, IS_BF16, kMergeMany>;
    if (cols == 16) return {mfa_kv4_kernel<DP, 1, IS_BF16>, merge};
    if (cols == 32) return {mfa_kv4_kernel<DP, 2, IS_BF16>, merge};
    return {(k4_fn)mfa_kv4_tile_kernel_of(DP, IS_BF16, bias), merge};
}
template <bool IS_BF16>
K4Kernels kernels4(int dp, int cols, bool bias, int threads) {
    switch (dp) {
        case 32: return kernels4<32, IS_BF16>(cols, bias, threads);
        case 64: return kernels4<64, IS_BF16>(cols, bias, threads);
        case 96: return kernels4<96, IS_BF16>(cols, bias, threads);
        default: return kernels4<128, IS_BF16>(cols, bias, threads);
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
// workspace of a launch: parts, their references and sums, what is merged
int64_t part_bytes(const K4Launch& l, int D) {
    return l.parts ? (l.parts * (D * 4 + 8) + (int64_t)l.a.G * sizeof(Merge4) + 255) / 256 * 256 : 0;
}
struct K4Plan {
    K4Launch l[2];
    int n = 0;
    int64_t ws_bytes = 0;
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
    const int rc = mfa_kv4_check_cache(&p->cache, p->batch, D, "mfa_kv4_fwd");
    if (rc != MFA_OK) return rc;
    const bool varlen = p->cu_seqlens_q != nullptr;
    const int64_t rows = varlen ? p->total_q : (int64_t)p->batch * p->seqlen_q;
    if (rows == 0) return MFA_OK;
    auto bad = [](const void* x, uintptr_t al) { return !x || (reinterpret_cast<uintptr_t>(x) & (al - 1)); };
    if (bad(p->q, 16) || bad(p->o, 16)) return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: q and o must be 16-byte aligned");
    if (p->batch > 0 && bad(p->cache_seqlens, 4)) return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: cache_seqlens is required");
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
    if (rows > 0x3fffffff || rows * a.Hq > 0x3fffffff) return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: problem too large");

    // Columns per workgroup: a sequence's, at most 128.  The sequences of a
    // varlen call are known on the device only: one launch takes those of at most
    // 16 columns, another the longer ones.
    // (no sequences: the launch only clears the rows)
    const int64_t cols = p->batch == 0 ? 1 : (varlen ? rows : p->seqlen_q) * (int64_t)a.R;
    plan->n = varlen && cols > 16 ? 2 : 1;
    const int64_t chunks = p->batch == 0 ? 1 : std::max<int64_t>(1, ((int64_t)a.max_k + kChunk4 - 1) / kChunk4);
    for (int i = 0; i < plan->n; ++i) {
        K4Launch& l = plan->l[i];
        l.a = a;
        l.a.cols = unit_cols(plan->n == 2 && i == 0 ? 16 : cols);
        l.a.min_cols = i == 0 ? 1 : 17;
        l.a.max_cols = plan->n == 2 && i == 0 ? 16 : 0x7fffffff;
        // (a bound on the items, which are counted on the device in int32)
        const int64_t tiles = !varlen       ? p->batch * ((cols + l.a.cols - 1) / l.a.cols)
                              : l.a.max_cols == 16 ? std::min<int64_t>(p->batch, rows)
                                                   : (cols + l.a.cols - 1) / l.a.cols + std::min<int64_t>(p->batch, rows);
        const int64_t units = tiles * a.Hkv;
        if (units > 0x3fffffff || units * chunks > 0x7fffffffLL) return k4err(MFA_ERR_INVALID, "mfa_kv4_fwd: problem too large");
        l.a.G = (int32_t)std::min<int64_t>(units * chunks, (int64_t)cus * (l.a.cols == kTileCols4 ? kTileWgs4 : wgs4(l.a.cols / 16)));
        // (neighbouring tiles of a K/V head share its rows in their XCD's L2)
        l.a.xcds = l.a.cols == kTileCols4 && l.a.G % 8 == 0 ? 8 : 1;
        l.parts = chunks > 1 ? (int64_t)l.a.G * 2 * l.a.cols : 0;
        plan->ws_bytes += part_bytes(l, D);
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
    K4Kernels k{};
    int merge = 0;
    const int threads = plan.l[plan.n - 1].a.cols == kTileCols4 ? kMergeMany : kMergeFew;
    for (int i = 0; i < plan.n; ++i) {
        K4Launch& l = plan.l[i];
        const bool bias = l.a.bias != 0;
        k = p->dtype == MFA_DTYPE_BF16 ? kernels4<true>(p->head_dim, l.a.cols, bias, threads)
                                          : kernels4<false>(p->head_dim, l.a.cols, bias, threads);
        if (l.parts) {
            l.a.ws_o = reinterpret_cast<float*>(ws);
            l.a.ws_ml = l.a.ws_o + l.parts * p->head_dim;
            l.a.ws_merge = reinterpret_cast<Merge4*>(l.a.ws_ml + l.parts * 2);
            ws += part_bytes(l, p->head_dim);
            merge += l.a.G * (l.a.cols / merge_cols(threads));
        }
        hipLaunchKernelGGL(k.attend, dim3(l.a.G), dim3(kThreads4), 0, st, l.a);
    }
    if (merge) hipLaunchKernelGGL(k.merge, dim3(merge), dim3(threads), 0, st, plan.l[0].a, plan.l[plan.n - 1].a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return k4err(MFA_ERR_LAUNCH, "mfa_kv4_fwd: launch failed: %s", hipGetErrorString(e));
    return MFA_OK;
}

}  // extern "C"
