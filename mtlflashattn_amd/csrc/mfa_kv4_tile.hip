// mfa_kv4_tile.hip -- attention over a paged 4-bit K/V cache for many columns (a
// chunk of a prompt): tiles of 128 columns, a column being one (query position,
// query head) pair of a K/V head.
//
// Each of the four wavefronts owns 32 columns; 64 keys at a time, the workgroup
// turns the codes of K and V into 16-bit rows in LDS once for all of them (a thread
// takes one 32-element scale group of each: 16 conversions, exact in bf16 and
// saturating in fp16).  There are two tiles: the next 64 keys are converted between
// the products of the current ones, and the codes of the 64 after those are on
// their way into registers.  1024 rows over 16384 keys, Hq=32 Hkv=8 D=128 bf16,
// take 298 to 304 us with the merge in a timed loop (876 to 893 TFLOP/s), the kernel
// alone 324 to 340 in short traces over machines (side by side on one: 316 to 324, and
// 329 to 334 with one tile, converted between two barriers); over 8192 keys 167 us,
// with soft-cap 212, with ALiBi 188.  Bound by no one unit: the matrix pipe is busy 40 % of the time, LDS bank conflicts take 10 % of it.
// In the form with one tile (332 us), with one part taken out at a time, the products
// of the scores were worth 64 us, those of the values 37, the softmax 43, the
// conversion 50 and most reads of K 17.
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16: a lane owns a column, its
// probabilities go from the accumulators into the second product as they are, and
// V is read transposed (ds_read_b64_tr_b16).  Exponent references are integers
// (ceil), so parts of a column's keys that other workgroups walked are added by
// the merge kernel without a rounding of their own.
#include <math.h>
#include <stdint.h>

#include "mfa_kv4_attend.h"

namespace {

constexpr int kTK = 64;  // keys per block

// A row of the V tile is not padded: 16-byte chunk c of row r is in slot c ^
// vswz<DP>(r), which spreads the stores of 16 lanes (a scale group each, the same
// chunk of it) and the transposing reads' four rows over the 16 slots of 256 bytes.
template <int DP>
__device__ __forceinline__ int vswz4(int r) {
    return DP == 128 ? 5 * (r & 3) : DP == 64 ? 4 * ((r >> 1) & 1) + ((r >> 1) & 3) : DP == 96 ? r & 3 : (r >> 2) & 3;
}

template <int DP, bool IS_BF16, bool BIAS>
__global__ void __launch_bounds__(kThreads4) __attribute__((amdgpu_waves_per_eu(2)))
mfa_kv4_tile_kernel(K4Args) {
    typedef typename std::conditional<IS_BF16, bf16x8_t, f16x8_t>::type op_t;
    constexpr int DS = DP / 16, DB = DP / 32, GPR = DP / 32, CPR = DP / 8;
    constexpr int KST = DP + 8, VST = DP;       // LDS rows (elements); K's padded against bank conflicts
    constexpr int K_ELEMS = kTK * KST, V_ELEMS = kTK * VST;
    constexpr int GROUPS = 2 * kTK * GPR;       // scale groups of a block, K's then V's
    constexpr int NG = (GROUPS + kThreads4 - 1) / kThreads4;
    constexpr int R_ELEMS = 4 * 32 * KST;       // the wavefronts' result rows, in the tiles' place
    constexpr int T_ELEMS = K_ELEMS + V_ELEMS;
    static_assert(R_ELEMS <= 2 * T_ELEMS, "the result rows fit the tiles' place");
    __shared__ __attribute__((aligned(16))) uint16_t smem[2 * T_ELEMS];
    __shared__ uint64_t nan_s[2][GPR + 1];  // NaN groups of a block's V, a bit each (and a place for what nobody reads)

    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Walk4 wk;
    if (!wk.start()) return;

    // this thread's groups of a block: wavefront-uniform choice of K or V
    bool gv[NG];
    int glds[NG], gsw[NG];
    uint32_t goff[NG], gsoff[NG];
    {
        K4Const& a = args4();
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int g = tid + kThreads4 * i;
            gv[i] = __builtin_amdgcn_readfirstlane(g) >= kTK * GPR;
            const int u = g - (gv[i] ? kTK * GPR : 0);
            const int row = u / GPR, grp = u - row * GPR;
            const bool in = g < GROUPS;
            goff[i] = in ? (uint32_t)(row * (int)(gv[i] ? a.v.cr : a.k.cr) + grp * 16) : 0x80000000u;
            gsoff[i] = in ? (uint32_t)(row * (int)(gv[i] ? a.v.sr : a.k.sr) + grp) : 0x80000000u;
            // (chunk e of the group: + 8 (e ^ gsw))
            glds[i] = gv[i] ? K_ELEMS + row * VST + ((32 * grp) ^ ((vswz4<DP>(row) & ~3) << 3)) : row * KST + 32 * grp;
            gsw[i] = gv[i] ? vswz4<DP>(row) & 3 : 0;
        }
    }

    while (true) {
        K4Const& a = args4();
        if (!wk.next(a)) return;
        const int Lk = wk.sq.Lk, dq = Lk - wk.sq.Lq;
        const float c = BIAS ? kLog2e : a.scale_log2;
        const float scale = a.scale, softcap = a.softcap, softcap_sk = a.softcap_sk;
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
        u32x4_t gc[NG];
        uint8_t gs[NG];  // (bytes until they are used: widening them here would wait for the loads)
        Pages4<DP> pg;
        pg.start(a, wk.b, wk.hkv, Lk, jbeg, kTK);
        auto gload = [&](int j) {
            const int row = pg.row_of(j);
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const int x = gv[i] ? 2 : 0;
                gc[i] = __builtin_amdgcn_raw_buffer_load_b128(gv[i] ? pg.rs[2] : pg.rs[0], goff[i] + (uint32_t)row * (uint32_t)pg.rstride[x], 0, 0);
                gs[i] = __builtin_amdgcn_raw_buffer_load_b8(gv[i] ? pg.rs[3] : pg.rs[1], gsoff[i] + (uint32_t)row * (uint32_t)pg.rstride[x + 1], 0, 0);
            }
        };
        // the codes into tile `to`, the even or odd (half_) of this thread's groups; part:
        // some column of the tile does not see the whole block (no branches: these run
        // between the products of the other tile)
        auto swrite = [&](bool part, int to, int half_) {
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                if (i % 2 != half_) continue;
                if (GROUPS % kThreads4 == 0 || tid + kThreads4 * i < GROUPS) {
                    uint16_t* p = smem + to * T_ELEMS + glds[i];
                    const bool nan = part & gv[i] & (gs[i] == 255);
                    nan_s[to][gv[i] && lane == 0 ? (tid + kThreads4 * i - kTK * GPR) >> 6 : GPR] = __ballot(nan);
                    const float s = nan ? 0.f : kv4_scale(gs[i]);
                    if constexpr (IS_BF16) {  // (fp16 saturates below; the test costs 1 % of the chunk above)
                        if (__builtin_expect(gv[i] && kv4_beyond(gs[i]), 0)) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) gc[i][e] = kv4_saturate8(gc[i][e], gs[i]);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<u32x4_t*>(p + 8 * (e ^ gsw[i])) = IS_BF16 ? kv4_bf16x8(gc[i][e], s) : kv4_f16x8(gc[i][e], s);
                }
            }
        };

        float m = -INFINITY, l = 0.f;
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

        auto block = [&](bool masked, int j, int at, auto&& stage, auto&& fetch) {
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
                            s[kb][r] = fmaf(-2.f * softcap, __builtin_amdgcn_rcpf(fast_exp2(s[kb][r] * softcap_sk) + 1.f), softcap);
                } else {
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) s[kb] *= scale;
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
            float acc[2] = {0.f, 0.f};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                u32x4_t pw[2];
#pragma unroll
                for (int st = 0; st < 2; ++st)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const float p0 = fast_exp2(fmaf(s[kb][8 * st + 2 * w], c, -mu));
                        const float p1 = fast_exp2(fmaf(s[kb][8 * st + 2 * w + 1], c, -mu));
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
        };

        // NaN groups for the columns that see their keys (a product with the zero weight
        // of a masked key would reach the others too)
        auto nan_groups = [&](int j, int at) {
#pragma unroll
            for (int i = 0; i < GPR; ++i) {
                for (uint64_t x = nan_s[at][i]; x; x &= x - 1) {
                    const int u = __builtin_amdgcn_readfirstlane(64 * i + __builtin_ctzll(x)), row = u / GPR;
                    K4Const& b = args4();
                    const int lo = lo4(b.wl, center), hi = hi4(b.causal, b.wr, center, Lk);
                    const bool sees = j + row >= lo && j + row <= hi;
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        float y = sees && db == u - row * GPR ? __builtin_nanf("") : 0.f;
                        pin(y);  // (no indexing of o by the group)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[db][r] += y;
                    }
                }
            }
        };

        if (jbeg < jend) gload(jbeg);
        // (waited for here: a wait inside the loop would drain the codes' loads too)
#pragma unroll
        for (int s = 0; s < DS; ++s) pin(qf[s]);
        pin(slope);
        auto part = [&](int j) { return (j < a_lo) | (j + kTK - 1 > a_hi); };
        if (jbeg < jend) {
            swrite(part(jbeg), 0, 0);
            swrite(part(jbeg), 0, 1);
            gload(jbeg + kTK);
        }
        __syncthreads();
        for (int j = jbeg, at = 0; j < jend; j += kTK, at ^= 1) {
            // (behind the last block the tile that is written is not read)
            auto stage = [&](int half_) { swrite(part(j + kTK), at ^ 1, half_); };
            auto fetch = [&]() { gload(j + 2 * kTK); };  // (behind the last key: zeros or rows that are not used)
            // (also where a wavefront's columns see nothing of it: a second path past the
            // products would copy the accumulators)
            block(j < f_lo || j + kTK - 1 > f_hi, j, at, stage, fetch);
            if (part(j)) nan_groups(j, at);
            __syncthreads();
        }

        // ---- results: lane (column, half) holds elements 32 db + 8 g + 4 half + 0..3
        K4Const& e = args4();
        const float lt = sum_halves(l);
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
            if (in && half == 0) store_lse4(e, wk.b, wk.sq.q0, qi, h, m, lt);
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
            if (half == 0) *reinterpret_cast<float2*>(e.ws_ml + 2 * row) = make_float2(m, lt);
        }
        __syncthreads();  // (the result rows are read before the next unit's tiles are written)
    }
}

template <int DP>
void* tile_of(bool bf16, bool bias) {
    typedef void (*fn)(K4Args);
    return bf16 ? (void*)(bias ? (fn)mfa_kv4_tile_kernel<DP, true, true> : (fn)mfa_kv4_tile_kernel<DP, true, false>)
                : (void*)(bias ? (fn)mfa_kv4_tile_kernel<DP, false, true> : (fn)mfa_kv4_tile_kernel<DP, false, false>);
}

}  // namespace

void* mfa_kv4_tile_kernel_of(int dp, bool bf16, bool bias) {
    switch (dp) {
        case 32: return tile_of<32>(bf16, bias);
        case 64: return tile_of<64>(bf16, bias);
        case 96: return tile_of<96>(bf16, bias);
        default: return tile_of<128>(bf16, bias);
    }
}
