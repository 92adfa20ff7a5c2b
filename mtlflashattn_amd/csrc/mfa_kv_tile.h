// mfa_kv_tile.h -- attention over a paged cache of quantised K/V for many columns (a
// chunk of a prompt): tiles of 128 columns, a column being one (query position,
// query head) pair of a K/V head (mfa_kv4_tile.hip, mfa_kv8_tile.hip).
//
// Each of the four wavefronts owns 32 columns; 64 keys at a time, the workgroup
// turns the codes of K and V into 16-bit rows in LDS once for all of them.  There
// are two tiles: the next 64 keys are converted between the products of the current
// ones, and the codes of the 64 after those are on their way into registers.
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16: a lane owns a column, its
// probabilities go from the accumulators into the second product as they are, and
// V is read transposed (ds_read_b64_tr_b16).  Exponent references are integers
// (ceil), so parts of a column's keys that other workgroups walked are added by
// the merge kernel without a rounding of their own.
//
// A format is a type Stage: a thread's codes of a block, how they are loaded, and
// how they become rows of the tiles.
#pragma once

#include "mfa_kv4_attend.h"

namespace {

constexpr int kTK = 64;  // keys per block

// A block's tiles in LDS: K's rows padded against bank conflicts, V's not.
template <int DP>
struct TileShape {
    static constexpr int KST = DP + 8, VST = DP;  // elements between rows
    static constexpr int K_ELEMS = kTK * KST, V_ELEMS = kTK * VST, T_ELEMS = K_ELEMS + V_ELEMS;
};

// A row of the V tile is not padded: 16-byte chunk c of row r is in slot c ^
// vswz4<DP>(r), which spreads the stores of 16 lanes and the transposing reads' four
// rows over the 16 slots of 256 bytes.
template <int DP>
__device__ __forceinline__ int vswz4(int r) {
    return DP == 128 ? 5 * (r & 3) : DP == 64 ? 4 * ((r >> 1) & 1) + ((r >> 1) & 3) : DP == 96 ? r & 3 : (r >> 2) & 3;
}

// LSE: the log-sum-exp is asked for.  Its sum is of the probabilities before they are
// rounded, beside that of the rounded ones, which the result is divided by: what the
// roundings of a row's weights have in common cancels there, but would leave the
// log-sum-exp off by up to 2^-8 in bf16 and 2^-11 in fp16.  (The 8-bit cache, 1024 rows over
// 16384 keys, Hq=32 Hkv=8 D=128: 326 us for 316, 348 for 331 in fp16.)
template <class Stage, bool BIAS, bool LSE>
__global__ void __launch_bounds__(kThreads4) __attribute__((amdgpu_waves_per_eu(2)))
mfa_kv_tile_kernel(K4Args) {
    constexpr int DP = Stage::D;
    constexpr bool IS_BF16 = Stage::kBf16;
    typedef typename std::conditional<IS_BF16, bf16x8_t, f16x8_t>::type op_t;
    typedef TileShape<DP> Shape;
    constexpr int DS = DP / 16, DB = DP / 32, CPR = DP / 8;
    constexpr int KST = Shape::KST, VST = Shape::VST, K_ELEMS = Shape::K_ELEMS, T_ELEMS = Shape::T_ELEMS;
    constexpr int R_ELEMS = 4 * 32 * KST;       // the wavefronts' result rows, in the tiles' place
    static_assert(R_ELEMS <= 2 * T_ELEMS, "the result rows fit the tiles' place");
    __shared__ __attribute__((aligned(16))) uint16_t smem[2 * T_ELEMS];
    __shared__ typename Stage::Nans nan_s[2];  // where a block's V is NaN

    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Walk4 wk;
    if (!wk.start()) return;

    Stage stage;  // this thread's part of a block's codes
    stage.init(args4(), tid);

    while (true) {
        K4Const& a = args4();
        if (!wk.next(a)) return;
        const int Lk = wk.sq.Lk, dq = Lk - wk.sq.Lq;
        const float scale = a.scale, scale_log2 = a.scale_log2, softcap = a.softcap, softcap_sk = a.softcap_sk;
        const bool alibi = BIAS && a.alibi != nullptr;
        // key ranges: of the tile, and those that all columns of the tile or of this wavefront see
        const int i_first = (int)div4(wk.col0, a.by_r), i_last = (int)div4(wk.col0 + wk.ncol - 1, a.by_r);
        const int t_lo = lo4(a.wl, i_first + dq), t_hi = hi4(a.causal, a.wr, i_last + dq, Lk);
        const Chunks4 ch = chunks4(t_lo, t_hi, wk.c0, wk.nch);
        const int jbeg = max(ch.beg * kChunk4, t_lo / kTK * kTK), jend = min(ch.end * kChunk4, t_hi + 1);
        const int wcol = wk.col0 + 32 * wave, wlast = min(wcol + 32, wk.col0 + wk.ncol) - 1;
        const bool live = wlast >= wcol;
        const int wi0 = (int)div4(wcol, a.by_r), wi1 = (int)div4(max(wlast, wcol), a.by_r);
        const int a_lo = lo4(a.wl, i_last + dq), a_hi = hi4(a.causal, a.wr, i_first + dq, Lk);  // of every column of the tile
        const int f_lo = lo4(a.wl, wi1 + dq), f_hi = hi4(a.causal, a.wr, wi0 + dq, Lk);    // of every column
        // (a lane behind the last column holds zero queries and stores nothing)
        int center;
        float slope = 0.f;

        // queries: lane (column l32, half) holds elements 16 s + 8 half .. as the
        // operand of step s
        op_t qf[DS];
        {
            const int col = wcol + l32, qi = (int)div4(col, a.by_r), h = wk.hkv * a.R + col - qi * a.R;
            const bool in = col <= wlast;
            center = qi + dq;
            if (alibi && in) slope = a.alibi[wk.b * a.alibi_bstride + h];
            const char* q = a.q + row_off4(a.cu_q != nullptr, wk.b, wk.sq.q0, in ? qi : 0, in ? h : 0, a.qb, a.qs, a.qh) * 2;
#pragma unroll
            for (int s = 0; s < DS; ++s) {
                u32x4_t w = {0, 0, 0, 0};
                if (in) w = *reinterpret_cast<const u32x4_t*>(q + (16 * s + 8 * half) * 2);
                qf[s] = __builtin_bit_cast(op_t, w);
            }
        }

        // the codes of the next block
        Pages4<Stage> pg;
        pg.start(a, wk.b, wk.hkv, Lk, jbeg, kTK);
        auto gload = [&](int j) { stage.load(pg, pg.row_of(j)); };
        // the codes into tile `to`, the even or odd (half_) of this thread's loads; part:
        // some column of the tile does not see the whole block (no divergent branches:
        // these run between the products of the other tile)
        auto swrite = [&](bool part, int to, int half_) { stage.write(smem + to * T_ELEMS, nan_s[to], part, half_, tid); };

        float m = -INFINITY, l = 0.f, l_exact = 0.f;  // (l_exact: with LSE)
        f32x16_t o[DB];
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[db][r] = 0.f;

        auto mfma = [](const op_t& x, const op_t& y, const f32x16_t& acc) {
            if constexpr (IS_BF16)
                return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, acc, 0, 0, 0);
            else
                return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, acc, 0, 0, 0);
        };
        const int tr_row = 4 * half + ((lane & 15) >> 2), tr_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        auto load_vf = [&](const uint16_t* vtile, int db, int kb, int st) -> op_t {
            // (rows 16 apart have the same swizzle)
            auto at = [&](int r) { return r * VST + (((4 * db + tr_chunk) ^ vswz4<DP>(r)) << 3) + 4 * (lane & 1); };
            const uint16_t* p0 = vtile + (32 * kb + 16 * st) * VST + at(tr_row);
            const uint16_t* p1 = vtile + (32 * kb + 16 * st) * VST + at(tr_row + 8);
            if constexpr (IS_BF16) {
                typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 v4;
                typedef __attribute__((address_space(3))) v4* lp;
                return __builtin_shufflevector(__builtin_amdgcn_ds_read_tr16_b64_v4bf16((lp)(p0)),
                                               __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lp)(p1)), 0, 1, 2, 3, 4, 5, 6, 7);
            } else {
                typedef __attribute__((__vector_size__(4 * sizeof(__fp16)))) __fp16 v4h;
                typedef __attribute__((__vector_size__(4 * sizeof(_Float16)))) _Float16 v4;
                typedef __attribute__((address_space(3))) v4h* lp;
                const v4 x = __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lp)(p0)));
                const v4 y = __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lp)(p1)));
                return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
            }
        };

        auto block = [&](bool masked, int j, int at, float sk, auto&& stage, auto&& fetch) {
            const float c = BIAS ? kLog2e : scale_log2 * sk;
            const uint16_t *ktile = smem + at * T_ELEMS, *vtile = ktile + K_ELEMS;
            // (the barriers to scheduling keep the LDS reads of 32 keys in flight ahead of
            // the products that take them; left alone, each is read and waited for: 2 %)
            f32x16_t s[2];
            op_t kf[DS], vf[DB][2];
            auto load_k = [&](int kb) {
#pragma unroll
                for (int t = 0; t < DS; ++t)
                    kf[t] = *reinterpret_cast<const op_t*>(ktile + (32 * kb + l32) * KST + 16 * t + 8 * half);
                __builtin_amdgcn_sched_barrier(0);
            };
            load_k(0);
            stage(0);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
                for (int t = 0; t < DS; ++t) s[kb] = mfma(kf[t], qf[t], s[kb]);
                if (kb == 0) {
                    load_k(1);
                    stage(1);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            fetch();
            auto load_v = [&](int kb) {
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int st = 0; st < 2; ++st) vf[db][st] = load_vf(vtile, db, kb, st);
                __builtin_amdgcn_sched_barrier(0);
            };
            load_v(0);
            // register r of s[kb] is key j + 32 kb + 4 half + acc_row(r)
            if constexpr (BIAS) {
                // natural-log units: x = scale*s, soft-cap c tanh(x/c) =
                // c - 2c / (exp(2x/c) + 1), ALiBi
                if (softcap > 0.f) {
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            s[kb][r] = fmaf(-2.f * softcap, __builtin_amdgcn_rcpf(fast_exp2(s[kb][r] * (softcap_sk * sk)) + 1.f), softcap);
                } else {
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) s[kb] *= scale * sk;
                }
                if (alibi) {
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) {
                        const float dist = (float)(center - (j + 32 * kb + 4 * half));
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[kb][r] = fmaf(-slope, fabsf(dist - (float)acc_row(r)), s[kb][r]);
                    }
                }
            }
            if (masked) {
                // (the pinned copy keeps the key indices out of the other blocks)
                int jm = j;
                asm volatile("" : "+v"(jm));
                K4Const& b = args4();
                const int lo = lo4(b.wl, center), hi = hi4(b.causal, b.wr, center, Lk);
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int key = jm + 32 * kb + 4 * half + acc_row(r);
                        s[kb][r] = ((key >= lo) & (key <= hi)) ? s[kb][r] : -INFINITY;
                    }
            }
            float m0 = s[0][0], m1 = s[0][1];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    if (kb == 0 && r == 0) continue;
                    m0 = fmax_nn(m0, s[kb][r]);
                    m1 = fmax_nn(m1, s[kb][r + 1]);
                }
            const float mn = fmax_nn(m, __builtin_ceilf(max_halves(fmax_nn(m0, m1)) * c));
            if (__any(mn != m)) {
                float alpha = pow2_diff(m, mn);
                asm volatile("" : "+v"(alpha));  // (keeps the products inside the branch)
                l *= alpha;
                if constexpr (LSE) l_exact *= alpha;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
                m = mn;
            }
            const float mu = m == -INFINITY ? 0.f : m;
            // probabilities rounded to 16 bits; l adds them as rounded.  (A second term
            // doubles the values' products: the chunk above takes 395 us, not 303, a mixed
            // step 97, not 87.  One term has an error of 1.4 times that of rounding the
            // result: 4.3e-5 rms against 3.1e-5 for results of 1.8e-2 over 8192 keys in
            // bf16, 5.4e-6 against 3.8e-6 in fp16; two have the latter.)  The second 32
            // keys' are formed while the first's products run.
            float acc[2] = {0.f, 0.f}, exact = 0.f;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                u32x4_t pw[2];
#pragma unroll
                for (int st = 0; st < 2; ++st)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const float p0 = fast_exp2(fmaf(s[kb][8 * st + 2 * w], c, -mu));
                        const float p1 = fast_exp2(fmaf(s[kb][8 * st + 2 * w + 1], c, -mu));
                        if constexpr (LSE) exact += p0 + p1;
                        if constexpr (IS_BF16) {
                            const k4_bf16x2_t pk = {(__bf16)p0, (__bf16)p1}, one = {(__bf16)1.f, (__bf16)1.f};
                            acc[w & 1] = __builtin_amdgcn_fdot2_f32_bf16(pk, one, acc[w & 1], false);
                            pw[st][w] = __builtin_bit_cast(uint32_t, pk);
                        } else {
                            const k4_f16x2_t pk = {(_Float16)p0, (_Float16)p1}, one = {(_Float16)1.f, (_Float16)1.f};
                            acc[w & 1] = __builtin_amdgcn_fdot2(pk, one, acc[w & 1], false);
                            pw[st][w] = __builtin_bit_cast(uint32_t, pk);
                        }
                    }
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int st = 0; st < 2; ++st)
                        o[db] = mfma(vf[db][st], __builtin_bit_cast(op_t, pw[st]), o[db]);
                __builtin_amdgcn_s_setprio(0);
                if (kb == 0) load_v(1);
            }
            l += acc[0] + acc[1];
            if constexpr (LSE) l_exact += exact;
        };

        if (jbeg < jend) gload(jbeg);
        // (waited for here: a wait inside the loop would drain the codes' loads too)
#pragma unroll
        for (int s = 0; s < DS; ++s) pin(qf[s]);
        pin(slope);
        float sk = 1.f;  // K's scale of the block at hand
        auto part = [&](int j) { return (j < a_lo) | (j + kTK - 1 > a_hi); };
        if (jbeg < jend) {
            swrite(part(jbeg), 0, 0);
            swrite(part(jbeg), 0, 1);
            sk = stage.k_scale();
            gload(jbeg + kTK);
        }
        __syncthreads();
        for (int j = jbeg, at = 0; j < jend; j += kTK, at ^= 1) {
            // (behind the last block the tile that is written is not read)
            float sk_next = 1.f;
            auto convert = [&](int half_) {
                swrite(part(j + kTK), at ^ 1, half_);
                sk_next = stage.k_scale();
            };
            auto fetch = [&]() { gload(j + 2 * kTK); };  // (behind the last key: zeros or rows that are not used)
            // (also where a wavefront's columns see nothing of it: a second path past the
            // products would copy the accumulators)
            block(j < f_lo || j + kTK - 1 > f_hi, j, at, sk, convert, fetch);
            sk = sk_next;
            // NaN for the columns that see their keys (a product with the zero weight of a
            // masked key would reach the others too)
            if (part(j)) {
                K4Const& b = args4();
                stage.add_nans(nan_s[at], o, j, lo4(b.wl, center), hi4(b.causal, b.wr, center, Lk), half);
            }
            __syncthreads();
        }

        // ---- results: lane (column, half) holds elements 32 db + 8 g + 4 half + 0..3
        K4Const& e = args4();
        const float lt = sum_halves(l);
        float le = lt;
        if constexpr (LSE) le = sum_halves(l_exact);
        const int col = wcol + l32, qi = (int)div4(col, e.by_r), h = wk.hkv * e.R + col - qi * e.R;
        const bool in = col <= wlast;
        if (live && wk.whole) {
            const float inv = lt > 0.f ? 1.f / lt : 1.f;  // (lt = 0: no key, o = 0; NaN stays NaN)
            uint16_t* rows = smem + wave * 32 * KST;      // (this wavefront's alone)
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    u32x2_t w;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float y0 = o[db][4 * g + 2 * x] * inv, y1 = o[db][4 * g + 2 * x + 1] * inv;
                        if constexpr (IS_BF16) w[x] = __builtin_bit_cast(uint32_t, k4_bf16x2_t{(__bf16)y0, (__bf16)y1});
                        else w[x] = __builtin_bit_cast(uint32_t, k4_f16x2_t{(_Float16)y0, (_Float16)y1});
                    }
                    *reinterpret_cast<u32x2_t*>(rows + l32 * KST + 32 * db + 8 * g + 4 * half) = w;
                }
            if (in && half == 0) store_lse4(e, wk.b, wk.sq.q0, qi, h, m, le);
            for (int x = lane; x < (wlast - wcol + 1) * CPR; x += 64) {
                const int r = x / CPR, d = 8 * (x - r * CPR);
                const int ri = (int)div4(wcol + r, e.by_r), rh = wk.hkv * e.R + wcol + r - ri * e.R;
                char* p = e.o + (row_off4(e.cu_q != nullptr, wk.b, wk.sq.q0, ri, rh, e.ob, e.os, e.oh) + d) * 2;
                store_stream(reinterpret_cast<u32x4_t*>(p), *reinterpret_cast<const u32x4_t*>(rows + r * KST + d));
            }
        } else if (live && in) {
            const int64_t row = wk.part_row(kTileCols4) + 32 * wave + l32;
            float* p = e.ws_o + row * DP;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<f32x4_t*>(p + 32 * db + 8 * g + 4 * half) =
                        f32x4_t{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
            if (half == 0) {
                *reinterpret_cast<float2*>(e.ws_ml + 2 * row) = make_float2(m, lt);
                if constexpr (LSE) e.ws_le[row] = le;
            }
        }
        __syncthreads();  // (the result rows are read before the next unit's tiles are written)
    }
}

}  // namespace
