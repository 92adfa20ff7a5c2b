// mfa_kv_rows.h -- attention over a paged cache of quantised K/V, sequences of at
// most 32 columns (mfa_kv4_attend.hip, mfa_kv8_attend.hip).
//
// A column is one (query position, query head) pair of a K/V head; a workgroup
// takes NT tiles of 16 columns and walks keys, its four wavefronts every fourth
// 32-key block, each with a softmax state of its own; the four are added at the
// end of the walk.  Per 32-key block a wavefront
//  * loads K straight into the A operand's registers: the order in which the
//    products of a score are added is free, so lane group g of a key's row takes
//    the elements that wide loads bring it, and the queries' operand takes the same
//    order;
//  * turns the codes into bf16 (exact) and forms S^T = K Q^T with
//    v_mfma_f32_16x16x32_bf16: lane = column, registers = keys;
//  * turns V into bf16 rows in LDS, whose transposed operand is read with
//    ds_read_b64_tr_b16, and adds O^T += V^T P^T.
// The codes of the next block are on their way into registers from the moment the
// current one's are consumed.
// fp16 queries are two bf16 terms (exact), and probabilities are two bf16 terms,
// hi = round(p) and lo = round(p - hi): a row over thousands of near-equal
// weights averages V, and one 16-bit rounding of every weight would be visible
// against its small result.  Sums and statistics are fp32.
//
// A format is a block type Blk: the registers of a 32-key block's codes and scales,
// how they are loaded, and how K becomes an operand and V rows in LDS.
#pragma once

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

constexpr int kOnce4 = 2;  // non-temporal buffer loads
// Workgroups per CU, at NT column tiles
constexpr int wgs4(int nt) { return nt == 1 ? 3 : 2; }

template <class Blk, int NT, bool IS_BF16>
__global__ void __launch_bounds__(kThreads4) __attribute__((amdgpu_waves_per_eu(wgs4(NT))))
mfa_kv_rows_kernel(K4Args) {
    constexpr int DP = Blk::D;
    constexpr int NQ = IS_BF16 ? 1 : 2;  // bf16 terms of a query
    constexpr int KS = DP / 32;          // k-steps of QK^T
    constexpr int DT = DP / 16;          // 16-row tiles of O^T
    constexpr int CPR = DP / 8;          // 16-byte chunks of a bf16 row
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

    typename Blk::Offsets off;  // per-lane byte offsets inside a 32-key block
    off.init(args4(), lane);

    while (true) {
        K4Const& a = args4();
        if (!wk.next(a)) return;
        const int Lk = wk.sq.Lk, dq = Lk - wk.sq.Lq;
        const bool bias = a.bias != 0, alibi = a.alibi != nullptr;
        const float scale = a.scale, scale_log2 = a.scale_log2, softcap = a.softcap, softcap_sk = a.softcap_sk;
        const int i_first = (int)div4(wk.col0, a.by_r), i_last = (int)div4(wk.col0 + wk.ncol - 1, a.by_r);
        // the keys of any column, and of every column, of the tile
        const int t_lo = lo4(a.wl, i_first + dq), t_hi = hi4(a.causal, a.wr, i_last + dq, Lk);
        const int f_lo = lo4(a.wl, i_last + dq), f_hi = hi4(a.causal, a.wr, i_first + dq, Lk);
        const int key0 = chunks4(t_lo, t_hi, wk.c0, wk.nch).beg * kChunk4 + 32 * wave;
        // this wavefront's blocks with keys: n0 .. n1 - 1
        const int n0 = t_lo - key0 > 31 ? 1 : 0;  // (only the first chunk may begin outside)
        const int n1 = t_hi < key0 ? 0 : min(wk.nch, (t_hi - key0) / kChunk4 + 1);

        Pages4<Blk> pg;
        pg.start(a, wk.b, wk.hkv, Lk, key0 + n0 * kChunk4, kChunk4);
        // (always issued, with offsets past the resource behind the last block: on a
        // path without them the wait for a block would be one for all)
        auto load = [&](int n, Blk& w) {
            const int row = pg.row_of(key0 + max(min(n, n1 - 1), 0) * kChunk4);
            const bool on = n < n1;
            const int srow = row / Blk::rows_per(1);
            const uint32_t kr = on ? row * pg.rstride[0] : 0x80000000u, ksr = on ? srow * pg.rstride[1] : 0x80000000u;
            const uint32_t vr = on ? row * pg.rstride[2] : 0x80000000u, vsr = on ? srow * pg.rstride[3] : 0x80000000u;
            w.load(pg.rs, off, kr, ksr, vr, vsr);
        };
        // ---- queries: lane (column l16, group grp) holds elements
        // Blk::element(grp, s) .. + 7 of its row as the operand of step s
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
                        if (in) qw[QLDS ? 0 : t][s] = *reinterpret_cast<const u32x4_t*>(q + Blk::element(grp, s) * 2);
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
        auto compute = [&](int j, Blk& w, auto&& refill) {
            // S^T = K Q^T: two 16-key tiles, lane = column, registers = keys
            // j + 16 kk + 4 grp + 0..3
            f32x4_t st[NT][2];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
                for (int t = 0; t < NT; ++t) st[t][kk] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const bf16x8_t kf = w.k_operand(kk, s, grp);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int z = 0; z < NQ; ++z)
                            st[t][kk] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, query(t, z, s), st[t][kk], 0, 0, 0);
                }
            }
            // V to LDS as bf16 rows; NaN in a block that some column does not see whole
            // as zeros (below)
            const bool masked = j < f_lo || j + 31 > f_hi;
            const float sk = w.k_scale();
            typename Blk::Nans nans;
            w.stage_v(vt, vswz, off, masked, lane, nans);
            refill();
            const float c = bias ? kLog2e : scale_log2 * sk;
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
                                                    __builtin_amdgcn_rcpf(fast_exp2(s[e >> 2][e & 3] * (softcap_sk * sk)) + 1.f), softcap);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) s[e >> 2][e & 3] *= scale * sk;
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
            // NaN for the columns that see their keys (a product with the zero weight of a
            // masked key would reach the others too)
            nans.template add<NT>(o, j, lo, hi, grp);
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

}  // namespace
