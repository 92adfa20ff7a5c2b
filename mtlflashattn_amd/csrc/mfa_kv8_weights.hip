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
//  * at most 32: bound by the stream of K and the weights (136 bytes per key and head
//    at head dim 128).  A wavefront takes every fourth 32-key block, the next one on
//    its way into registers, and multiplies one or two tiles of 16 columns;
//  * more: bound by vector instructions, nine per 64 scores beside the product's one, of
//    which the exponential takes four slots (1024 rows over 8192 keys, D=128, 120 us: vector
//    units active 69 % of the cycles, matrix pipe 25 %).  A wavefront holds 32 keys as
//    operands and goes over
//    the columns, 128 of which stand in LDS while the next are loaded straight into it;
//    eight wavefronts share them.  64 rows over two prompts of 12000 to 16384 keys, Hq=32
//    Hkv=8 D=128: 32 us, of which about 10 pass before the first product (the dealing,
//    the page, the first queries and keys); 46 us with the pieces of two XCDs on the other
//    six, 54 with eight-way unrolled loads (their code costs more to fetch than to run).
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
    float scale, scale_log2, softcap, softcap_sk;
    bool bias, alibi;
    __device__ __forceinline__ float operator()(float s, float sk, float nlse, float slope, int dist) const {
        if (!bias) return fmaf(s, scale_log2 * sk, nlse);
        // (the soft-cap as the attention forms it, off by up to softcap 2^-21; tanh to the last
        // bits made a chunk of 1024 rows over 8192 keys take 306 us instead of 199)
        float x = s * (scale * sk);
        if (softcap > 0.f) x = fmaf(-2.f * softcap, __builtin_amdgcn_rcpf(fast_exp2(s * (softcap_sk * sk)) + 1.f), softcap);
        if (alibi) x = fmaf(-slope, fabsf((float)dist), x);
        return fmaf(x, kLog2e, nlse);
    }
};
__device__ __forceinline__ ScoreOf score_of(K4Const& a) {
    return ScoreOf{a.scale, a.scale_log2, a.softcap, a.softcap_sk, a.bias != 0, a.alibi != nullptr};
}

// (32 sequences of 512 to 8192 keys, Hq=32 Hkv=8 D=128 bf16: 34.9 us with three
// workgroups per CU, 37.4 with two, 35.5 with five; two blocks ahead instead of one: 35.7.
// Of that about 11 us pass before the stream runs and after it ends.  64 sequences of 5 rows
// over 8192: two tiles of columns 122 us, 133 with three workgroups, 198 by the kernel for
// more columns.)
constexpr int few_wgs(int nt) { return nt == 1 ? 3 : 2; }
template <int DP, bool IS_BF16, int NT>
__global__ void __launch_bounds__(kThreads4) __attribute__((amdgpu_waves_per_eu(few_wgs(NT))))
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
        // queries: lane (column 16 t + l16, group grp) holds elements Blk::element(grp, s) .. + 7;
        // the products' registers are columns 16 t + 4 grp + e
        op_t qf[NT][KS];
        float nlse[NT][4], slope[NT][4];
        int lo[NT][4], hi[NT][4], center[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int mine = 16 * t + l16, i = (int)div4(mine, a.by_r), h = wk.hkv * a.R + mine - i * a.R;
            const bool in = mine < wk.ncol;
            const char* q = a.q + row_off4(a.cu_q != nullptr, wk.b, wk.sq.q0, in ? i : 0, in ? h : 0, a.qb, a.qs, a.qh) * 2;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                u32x4_t w = {0, 0, 0, 0};
                if (in) w = *reinterpret_cast<const u32x4_t*>(q + Blk::element(grp, s) * 2);
                qf[t][s] = __builtin_bit_cast(op_t, w);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = 16 * t + 4 * grp + e, ie = (int)div4(col, a.by_r), he = wk.hkv * a.R + col - ie * a.R;
                const bool some = col < wk.ncol;
                center[t][e] = ie + dq;
                lo[t][e] = lo4(a.wl, center[t][e]);
                hi[t][e] = some ? hi4(a.causal, a.wr, center[t][e], Lk) : -1;
                nlse[t][e] = neg_lse2(a, some, wk.b, wk.sq.q0, ie, he);
                slope[t][e] = score.alibi && some ? a.alibi[wk.b * a.alibi_bstride + he] : 0.f;
            }
        }
        load(0);
        // (waited for here: a wait inside the loop would drain the codes' loads too)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int s = 0; s < KS; ++s) pin(qf[t][s]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pin(nlse[t][e]);
                pin(slope[t][e]);
            }
        }
        for (int n = 0; n < n1; ++n) {
            const int j = key0 + n * kChunk4;
            f32x4_t st[NT][2];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
                for (int t = 0; t < NT; ++t) st[t][kk] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const op_t kf = blk.k.template k_operand<op_t>(kk, s, grp);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        if constexpr (IS_BF16) st[t][kk] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qf[t][s], kf, st[t][kk], 0, 0, 0);
                        else st[t][kk] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qf[t][s], kf, st[t][kk], 0, 0, 0);
                    }
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
                float all = 0.f;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p[e] = fast_exp2(score(st[t][kk][e], sk, nlse[t][e], slope[t][e], center[t][e] - key));
                        if (masked) p[e] = ((key >= lo[t][e]) & (key <= hi[t][e])) ? p[e] : 0.f;
                    }
                    all += (p[0] + p[1]) + (p[2] + p[3]);
                }
                sum[kk] = sum_groups4(all);
            }
            // lane 16 kk + l16 has the sum of its own key
            const float w = old + (grp & 1 ? sum[1] : sum[0]);
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(w), rs, at, 0, 0);
        }
    }
}

constexpr int kManyWgs = 2, kManyThreads = 512;  // (workgroups per CU: what their LDS leaves room for)

// A workgroup's piece of the work: consecutive chunks of one unit (a sequence and K/V
// head).  The units' chunks are cut into pieces of at most ceil(chunks of all units /
// G), the same for all of a unit to one chunk, so that no workgroup pays the latency
// of a second unit's queries and pages.  Where all chunks leave half of the workgroups
// without one, pieces of sequences with many columns are halves of a chunk (a prompt of
// 2048 rows over themselves, Hq=32 Hkv=8 D=128: 158 us by chunks, 118 by halves, now 108,
// and 120 by quarters; 4 sequences of 9 rows over 1000: 8.1 by chunks, 10.6 by halves).
constexpr int kHalfCols = 256;
struct Piece4 {
    int b, hkv, c0, nch, part, parts;  // part: of `parts` of one chunk
    Seq4 sq;
    // pieces of at most `most` chunks of a sequence, a chunk in `parts`
    static __device__ __forceinline__ int pieces(const Seq4& s, int most) { return (s.chunks + most - 1) / most; }
    static __device__ __forceinline__ int parts_of(const Seq4& s, int R, bool half) { return half && s.Lq * R >= kHalfCols ? 2 : 1; }
    __device__ __forceinline__ bool find(K4Const& a) {
        const int lane = threadIdx.x & 63, B = a.B, H = a.Hkv;
        auto seq = [&](int b0) { return b0 + lane < B ? seq4(a, b0 + lane) : Seq4{0, 0, 0, 0, 1}; };
        Seq4 s = seq(0);
        int all = __builtin_amdgcn_readlane(scan64(s.items(H)), 63);
        for (int b0 = 64; b0 < B; b0 += 64) all += __builtin_amdgcn_readlane(scan64(seq(b0).items(H)), 63);
        if (all == 0) return false;
        const int most = (all + a.G - 1) / a.G;
        const bool half = all <= a.G / 2;
        auto of = [&](const Seq4& y) { return y.tiles * H * pieces(y, most) * parts_of(y, a.R, half); };
        int n = of(s), inc = scan64(n), total = __builtin_amdgcn_readlane(inc, 63);
        for (int b0 = 64; b0 < B; b0 += 64) {
            total += __builtin_amdgcn_readlane(scan64(of(seq(b0))), 63);
        }
        // neighbouring pieces, which share their queries, on one XCD
        const int per = (total + 7) / 8, w = blockIdx.x % 8 * per + blockIdx.x / 8;
        if ((int)blockIdx.x / 8 >= per || w >= total) return false;
        for (int b0 = 0, base = 0;;) {
            const uint64_t past = __ballot(inc + base > w);
            if (past) {
                const int l = __builtin_ctzll(past);
                b = b0 + l;
                sq = lane_seq4(s, l);
                parts = parts_of(sq, a.R, half);
                const int at = w - base - __builtin_amdgcn_readlane(inc - n, l), np = pieces(sq, most), nx = np * parts;
                hkv = at / nx;
                const int kx = at - hkv * nx, k = kx / parts;
                part = kx - k * parts;
                c0 = first_item(k, sq.chunks, np);
                nch = first_item(k + 1, sq.chunks, np) - c0;
                return true;
            }
            base += __builtin_amdgcn_readlane(inc, 63);
            b0 += 64;
            if (b0 >= B) return false;
            s = seq(b0);
            n = of(s);
            inc = scan64(n);
        }
    }
};

template <int DP, bool IS_BF16, bool BIAS>
__global__ void __launch_bounds__(kManyThreads) __attribute__((amdgpu_waves_per_eu(2 * kManyWgs)))
mfa_kv8_weights_many_kernel(K4Args) {
    typedef op_of<IS_BF16> op_t;
    typedef KeyBlock8<DP> Blk;
    constexpr int KS = DP / 32, CPR = DP / 8;
    constexpr int kWCols = 128;             // columns of a tile in LDS
    constexpr int kWChunks = BIAS ? 2 : 4;  // chunks whose sums are kept in LDS
    constexpr int NQ = kWCols * CPR / kManyThreads;
    constexpr int kBlocks = kWChunks * kChunk4 / 32, kWaves = kManyThreads / 64;
    static_assert(kWCols * CPR % kManyThreads == 0, "whole rounds of loads");
    // two tiles of queries: 16-byte chunk c of row r is in slot c ^ swz(r) (the loads
    // straight into LDS leave no room for padding; a read takes a chunk of 16 rows)
    __shared__ __attribute__((aligned(16))) uint16_t q_s[2][kWCols * DP];
    auto swz = [](int r) { return DP == 128 ? r & 15 : DP == 64 ? r >> 1 & 7 : r >> 2 & 3; };
    // of the columns of three tiles: the query's address, the log-sum-exp, the keys that they
    // see, and for the biases
    __shared__ const char* row_s[3][kWCols];
    __shared__ __attribute__((aligned(16))) float nlse_s[3][kWCols], slope_s[3][BIAS ? kWCols : 4];
    __shared__ __attribute__((aligned(16))) int lo_s[3][kWCols], hi_s[3][kWCols], center_s[3][BIAS ? kWCols : 4];
    __shared__ float sum_s[4][kBlocks][32];
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    K4Const& a = args4();
    Piece4 wk;
    if (!wk.find(a)) return;
    const int Lk = wk.sq.Lk, dq = Lk - wk.sq.Lq, causal = a.causal, wl = a.wl, wr = a.wr;
    ScoreOf score = score_of(a);
    score.bias = BIAS;
    const FastDiv by_r = {a.by_r.d, a.by_r.m, a.by_r.s};
    // (what columns are looked up with: read from the arguments in the loop, each is a latency)
    const int R = a.R;
    const char* const q_0 = a.q + row_off4(a.cu_q != nullptr, wk.b, wk.sq.q0, 0, wk.hkv * R, a.qb, a.qs, a.qh) * 2;
    const int64_t q_i = a.qs * 2, q_h = a.qh * 2, lse_h = a.lse_h;
    const float* const lse_0 = a.lse + (a.cu_q ? (int64_t)wk.sq.q0 : wk.b * a.lse_b) + wk.hkv * R * lse_h;
    const float* const alibi_0 = BIAS && a.alibi ? a.alibi + wk.b * a.alibi_bstride + wk.hkv * R : nullptr;
    const int i_last = wk.sq.Lq - 1;
    const int t_lo = lo4(wl, dq), t_hi = hi4(causal, wr, i_last + dq, Lk);
    const Chunks4 ch = chunks4(t_lo, t_hi, wk.c0, wk.nch);
    for (int c0 = ch.beg; c0 < ch.end; c0 += kWChunks) {
        // ---- some chunks: blocks of 32 keys, dealt over the wavefronts; where there are
        // fewer than wavefronts, two or four share one and take every second or fourth 32
        // columns
        const int keys = wk.parts > 1 ? kChunk4 / 2 : kWChunks * kChunk4;
        // (as differences: j0 + keys may pass 31 bits)
        const int j0 = c0 * kChunk4 + wk.part * keys, jend = j0 + min(min(ch.end * kChunk4, Lk) - j0, keys);
        if (j0 >= jend) break;
        const int nb = (jend - j0 + 31) / 32, cw = nb <= kWaves / 4 ? 4 : nb <= kWaves / 2 ? 2 : 1, kw = kWaves / cw;
        const int cg = wave / kw, b0 = wave - cg * kw;
        typename Blk::Offsets off;
        off.init(args4(), lane);
        Pages4<WFormat<DP>> pg;
        pg.start(a, wk.b, wk.hkv, Lk, j0 + 32 * b0, 32 * kw);
        Blk raw;
        auto kload = [&](int blk) {
            const int row = pg.row_of(j0 + 32 * min(blk, nb - 1));
            raw.load(pg.rs, off, (uint32_t)(row * pg.rstride[0]), (uint32_t)(row / kKv8Block * pg.rstride[1]));
        };
        kload(b0);
        auto place = [&](int blk) { return (uint32_t)((pg.row_of(j0 + 32 * blk) + (lane & 31)) * pg.rstride[2]); };
        // (the first block's weights: where there is no other, nothing waits for them at the end)
        const float before = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(pg.rs[2], place(min(b0, nb - 1)), 0, 0));
        for (int blk = b0; blk < nb; blk += kw) sum_s[cg][blk][lane & 31] = 0.f;
        // the columns that see any of these keys
        int i0 = 0, i1 = wk.sq.Lq;
        if (causal) i0 = max(i0, j0 - dq);
        if (wr >= 0) i0 = (int)max((int64_t)i0, (int64_t)j0 - wr - dq);
        if (wl >= 0) i1 = (int)min((int64_t)i1, (int64_t)jend + wl - dq);
        const int cbeg = i0 < i1 ? i0 * R / 32 * 32 : 0, cend = i0 < i1 ? i1 * R : 0;
        const int n = (cend - cbeg + kWCols - 1) / kWCols;  // tiles of columns
        // Step k brings tile k in, works on tile k - 1 and looks up the columns of tile k + 1.
        // (Every part stands here once: what is run once costs the fetch of its code.)
        for (int k = -1; k <= n; ++k) {
            __syncthreads();
            if (k >= 0 && k < n) {
#pragma unroll 2
                for (int x = 0; x < NQ; ++x) {
                    const int first = (kWaves * x + wave) * 64, u = first + lane, r = u / CPR, c = (u - r * CPR) ^ swz(r);
                    lds_load16(row_s[k % 3][r] + 16 * c, q_s[k & 1] + 8 * first);
                }
            }
            const int at = (k - 1) & 1, col0 = cbeg + (k - 1) * kWCols, as = (k + 2) % 3;
            const int tiles = k < 1 ? 0 : min((cend - col0 + 31) / 32, kWCols / 32);
            for (int blk = b0; blk < nb && tiles > 0; blk += kw) {
                const int j = j0 + 32 * blk;
                op_t kf[2][KS];  // keys 16 kk + l16
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                    for (int s = 0; s < KS; ++s) kf[kk][s] = raw.template k_operand<op_t>(kk, s, grp);
                const float sk = raw.k_scale();
                // (the next block, or the first one again for the next columns)
                if (nb > kw) kload(blk + kw < nb ? blk + kw : b0);
                float acc[2] = {0.f, 0.f};
                // 32 columns; masked: some column does not see some key
                auto tile = [&](int t, auto masked) {
#pragma unroll
                    for (int ct = 0; ct < 2; ++ct) {
                        const int row = 32 * t + 16 * ct + l16, at0 = 32 * t + 16 * ct + 4 * grp;
                        f32x4_t s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                        for (int d = 0; d < KS; ++d) {
                            const op_t qf = *reinterpret_cast<const op_t*>(q_s[at] + row * DP + 8 * ((Blk::element(grp, d) / 8) ^ swz(row)));
#pragma unroll
                            for (int kk = 0; kk < 2; ++kk) {
                                if constexpr (IS_BF16) s[kk] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qf, kf[kk][d], s[kk], 0, 0, 0);
                                else s[kk] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qf, kf[kk][d], s[kk], 0, 0, 0);
                            }
                        }
                        // register r is column 32 t + 16 ct + 4 grp + r
                        const f32x4_t nls = *reinterpret_cast<const f32x4_t*>(nlse_s[as] + at0);
#pragma unroll
                        for (int kk = 0; kk < 2; ++kk) {
                            const int key = j + 16 * kk + l16;
                            float p[4];
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                p[r] = fast_exp2(score(s[kk][r], sk, nls[r], BIAS ? slope_s[as][at0 + r] : 0.f,
                                                       BIAS ? center_s[as][at0 + r] - key : 0));
                            if constexpr (masked.value) {
#pragma unroll
                                for (int r = 0; r < 4; ++r)
                                    p[r] = ((key >= lo_s[as][at0 + r]) & (key <= hi_s[as][at0 + r])) ? p[r] : 0.f;
                            }
                            acc[kk] += (p[0] + p[1]) + (p[2] + p[3]);
                        }
                    }
                };
                for (int t = cg; t < tiles; t += cw) {
                    const int cw0 = col0 + 32 * t;
                    const int ca = (int)quotient(cw0, by_r) + dq, cb = (int)quotient(min(cw0 + 31, cend - 1), by_r) + dq;
                    if (hi4(causal, wr, cb, Lk) < j || lo4(wl, ca) > j + 31) continue;  // (no column sees a key)
                    if (j < lo4(wl, cb) || j + 31 > hi4(causal, wr, ca, Lk)) tile(t, std::true_type{});
                    else tile(t, std::false_type{});
                }
                // lane 16 kk + l16 has the sum of its own key
                const float s0 = sum_groups4(acc[0]), s1 = sum_groups4(acc[1]);
                if (lane < 32) sum_s[cg][blk][lane] += grp ? s1 : s0;
            }
            if (k + 1 < n && tid < kWCols) {
                // (columns behind the last repeat it, with a log-sum-exp that leaves them out)
                const int to = (k + 1) % 3, mine = cbeg + (k + 1) * kWCols + tid, col = min(mine, cend - 1);
                const int i = (int)quotient(col, by_r), h = col - i * R, c = i + dq;
                const float l = lse_0[i + h * lse_h];
                row_s[to][tid] = q_0 + (i * q_i + h * q_h);
                lo_s[to][tid] = lo4(wl, c);
                if constexpr (BIAS) {
                    center_s[to][tid] = c;
                    slope_s[to][tid] = score.alibi ? alibi_0[h] : 0.f;
                }
                const bool sees = mine < cend && l != -INFINITY;
                nlse_s[to][tid] = sees ? -l * kLog2e : -INFINITY;
                hi_s[to][tid] = sees ? hi4(causal, wr, c, Lk) : -1;
            }
            wait_vm<0>();
        }
        if (cw > 1) __syncthreads();
        if (cg == 0) {
            for (int blk = b0; blk < nb; blk += kw) {
                // (outside of the condition: a page looked up by some lanes would no longer be uniform)
                const uint32_t all = place(blk), at = lane < 32 ? all : 0x80000000u;
                float w = blk == b0 ? before : __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(pg.rs[2], at, 0, 0));
                w = j0 + 32 * blk + lane < dq ? w : 0.f;
                float sum = sum_s[0][blk][lane & 31];
                for (int z = 1; z < cw; ++z) sum += sum_s[z][blk][lane & 31];
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(w + sum), pg.rs[2], at, 0, 0);
            }
        }
        if (cw > 1) __syncthreads();  // (the sums are read)
    }
}

typedef void (*w8_fn)(K4Args);
// few: 16-column tiles of the kernel for few columns, 0: the other
template <int DP, bool IS_BF16>
w8_fn weights_of(int few, bool bias) {
    return few == 1 ? mfa_kv8_weights_few_kernel<DP, IS_BF16, 1> : few == 2 ? mfa_kv8_weights_few_kernel<DP, IS_BF16, 2>
           : bias   ? mfa_kv8_weights_many_kernel<DP, IS_BF16, true> : mfa_kv8_weights_many_kernel<DP, IS_BF16, false>;
}
template <bool IS_BF16>
w8_fn weights_of(int dp, int few, bool bias) {
    switch (dp) {
        case 32: return weights_of<32, IS_BF16>(few, bias);
        case 64: return weights_of<64, IS_BF16>(few, bias);
        case 96: return weights_of<96, IS_BF16>(few, bias);
        default: return weights_of<128, IS_BF16>(few, bias);
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
    // Sequences of few columns, then those of more (a varlen call's are known on the device
    // only: both)
    const bool varlen = f.cu_seqlens_q != nullptr;
    const int64_t cols = (varlen ? (int64_t)a.rows_q : f.seqlen_q) * (int64_t)a.R;
    const int64_t chunks = std::max<int64_t>(1, ((int64_t)a.max_k + kChunk4 - 1) / kChunk4);
    const int64_t units = (varlen ? std::min<int64_t>(f.batch, a.rows_q) : f.batch) * (int64_t)a.Hkv;
    if (cols > 0x3fffffff || units > 0x3fffffff || units * chunks > 0x7fffffffLL)
        return w8err(MFA_ERR_INVALID, "%s: problem too large", who);
    const int cus = mfa_chip_cus(stream);
    // (a varlen call's tiles by the mean of its sequences; beyond 32 columns they are single rows
    // beside chunks, as a rule)
    const int64_t mean = varlen ? (cols + f.batch - 1) / f.batch : cols;
    const int nt = mean > 16 && mean <= 32 ? 2 : 1;
    for (int few = nt; few >= 0; few -= nt) {
        if (few ? !varlen && cols > 16 * nt : cols <= 16 * nt) continue;
        a.cols = few ? 16 * few : kAllCols4;  // (one unit per sequence and K/V head)
        a.min_cols = few ? 1 : 16 * nt + 1;
        a.max_cols = few ? 16 * few : 0x7fffffff;
        // (of a varlen call's sequences no more than its rows allow have the columns for it)
        const int64_t mine = few || !varlen ? units : std::min<int64_t>(units, cols / a.min_cols * a.Hkv);
        const int64_t most = mine * chunks * (few ? 1 : 2);  // (halves of chunks)
        a.G = (int32_t)std::min<int64_t>(most, (int64_t)cus * (few ? few_wgs(few) : kManyWgs));
        // (pieces: at most one more of each unit than its share)
        int64_t grid = few ? a.G : std::min<int64_t>(most, a.G + mine);
        if (!few) grid = (grid + 7) / 8 * 8;
        a.xcds = 1;
        const bool bias = a.bias != 0;
        const w8_fn fn = f.dtype == MFA_DTYPE_BF16 ? weights_of<true>(f.head_dim, few, bias) : weights_of<false>(f.head_dim, few, bias);
        hipLaunchKernelGGL(fn, dim3((unsigned)grid), dim3(few ? kThreads4 : kManyThreads), 0, static_cast<hipStream_t>(stream), a);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return w8err(MFA_ERR_LAUNCH, "%s: launch failed: %s", who, hipGetErrorString(e));
    return MFA_OK;
}

}  // extern "C"
