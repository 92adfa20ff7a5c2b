// mfa_kv8_evict.hip -- eviction from a paged 8-bit K/V cache by accumulated weight
// (mfa_kv8_evict in include/mfa.h).
//
//  * select: one workgroup per (sequence, head) finds the weight of the last row that
//    stays and lists the rows that stay in order.  Weights become unsigned keys of the
//    same order; the threshold, the largest key that as many candidates reach as are
//    to stay, is found 11, 11 and 10 bits at a time from histograms in LDS (weights
//    crowd into few exponents: lanes of a wavefront that agree count once together).
//    Keys stay in LDS where a sequence fits (32768 rows), else they are read again.
// (Where the bound on the lengths or the budget says that no row moves, one kernel writes the
// lengths.)  Then, with many heads in the batch:
//  * walk: a workgroup per head, for K and for V, moves the rows block by block, in place.
// With few, a workgroup per block:
//  * save: rows only move down, and no block behind the one that holds row budget - 1
//    is written to; the rows that stay and lie in front are what another block's new
//    rows, or its new scale, may overwrite.  They go to the workspace as they are.
//  * gather: a workgroup per block of 64 new rows of a head, in K or in V, collects
//    its rows from the workspace and the cache, takes their largest magnitude, and
//    writes them with a new scale.
// One sequence (2048 of 2176 rows stay, 8 heads of 128) takes 19 us, of which select, save
// and gather have 8.6, 5.2 and 6.0: the latency of a few dependent passes each.  Sixteen
// sequences (4001 of 4096 to 16384 rows stay) take 81 us over data that the last-level cache
// holds, select 22 of them and the rest the bytes and the conversions of the walk, and 98 us
// over data outside of it (save and gather: 111).  Selecting by 32 passes
// over one bit took 41 us, and save and gather by 512 threads instead of 256 18 us more.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>

#include "mfa_kv4_attend.h"
#include "mfa_kv8.h"

namespace {

constexpr int kSThreads = 1024, kSWaves = kSThreads / 64;
constexpr int kEThreads = 256;
// Sequences times heads from which on one workgroup moves all rows of a head.  (64 heads of
// 128, 2067 of 2176 rows: 47 us against 53 by save and gather; 32 heads 41 against 37, 128
// heads 55 against 81, 8 heads 39 against 24.  128 heads, 4275 of 9500: 98 against 128.
// How many of them are over the budget is known on the device only: one sequence of 8 heads
// that keeps 4275 of 9500 rows takes 66 us beside 63 that stay as they are, 26 alone, and one
// of 2048 of 2176 33 and 16.)
constexpr int kWalk = 64;
constexpr int walk_threads(int d) { return d == 96 ? 768 : 1024; }  // (whole blocks per step)
constexpr int kStay = 0x7fffffff;

// What select leaves for the kernels behind it.
struct Head8 {
    int32_t first;  // first row that moves (kStay: none)
    int32_t n;      // rows of the sequence afterwards
    int32_t low;    // rows that stay and lie in front of `safe`
    int32_t pad;
};

struct E8Args {
    Kv4Pool pool[2];
    float* w;
    int64_t wp, wr, wh;  // elements
    const int32_t* bt;
    int64_t bt_b;
    const int32_t* lens;
    int32_t* new_lens;
    int32_t B, H, D, page, npages, max_k, budget, recent;
    int32_t rows;    // of the workspace per (sequence, head): the budget, or none where no row moves
    int32_t blocks;  // of 64 new rows per (sequence, head)
    int32_t safe;    // rows from here on are read where they are
    int32_t walk;    // one workgroup moves all rows of a head
    int32_t four;    // weights of four adjacent rows may be loaded at once
    FastDiv by_page, by_blocks;
    Head8* head;      // [B H]
    int32_t* idx;     // [B H rows] rows that stay, in order: their places in the pool (page page_block_size + row), or -1
    float* sw;        // [B H rows] saved weights
    uint8_t* codes;   // [2][B H rows][D] saved rows
    uint8_t* scales;  // [2][B H rows]
};

// Where row j of a sequence is: the page, and the row in it (id -1: outside the pool).
struct Place8 {
    int id, row;
};
__device__ __forceinline__ Place8 place8(const E8Args& a, const int32_t* bt, int j) {
    const int i = (int)quotient((uint32_t)j, a.by_page), id = bt[i];
    return Place8{(uint32_t)id < (uint32_t)a.npages ? id : -1, j - i * a.page};
}
__device__ __forceinline__ int packed8(const E8Args& a, const Place8& p) { return p.id < 0 ? -1 : p.id * a.page + p.row; }
__device__ __forceinline__ Place8 unpacked8(const E8Args& a, int x) {
    const int id = (int)quotient((uint32_t)x, a.by_page);
    return Place8{id, x - id * a.page};
}
__device__ __forceinline__ float* weight_at(const E8Args& a, const Place8& p, int h) {
    return a.w + p.id * a.wp + p.row * a.wr + h * a.wh;
}

// The unsigned order of a weight: NaN above everything, 0 for no row.
__device__ __forceinline__ uint32_t key_of(float w) {
    const uint32_t u = __float_as_uint(w);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    if ((u & 0x7fffffffu) == 0) return 0x80000000u;  // (-0 = 0)
    return u >> 31 ? ~u : u | 0x80000000u;
}

constexpr int kBins = 2048;
static_assert(kBins == 2 * kSThreads, "two bins per thread");

// KEYS: keys that LDS holds, 0: none
template <int KEYS>
__global__ void __launch_bounds__(kSThreads) mfa_kv8_select_kernel(E8Args a) {
    __shared__ __attribute__((aligned(16))) uint32_t key_s[KEYS > 0 ? KEYS : 4];
    __shared__ int count_s[kBins];
    __shared__ int sum_s[kSWaves], found_s[3];
    __shared__ int gt_s[kSWaves], eq_s[kSWaves];
    __shared__ int first_s, low_s;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int bh = blockIdx.x, b = bh / a.H, h = bh - b * a.H;
    const int n = min(max(a.lens[b], 0), a.max_k);
    if (n <= a.budget) {
        if (tid == 0) a.head[bh] = Head8{kStay, n, 0, 0};
        return;
    }
    const int tail = min(a.recent, a.budget), m = n - tail, need = a.budget - tail;  // need < m
    const int32_t* bt = a.bt + b * a.bt_b;
    int32_t* const idx = a.idx + (int64_t)bh * a.rows;
    if (tid == 0) {
        first_s = m;
        low_s = max(0, min(tail, a.safe - m));
    }

    // (rows are counted without a sign: whole rounds behind m may pass 2^31)
    const uint32_t rows = (uint32_t)m;
    // the keys of rows j .. j + 3 (j a multiple of 4), 0 for rows from m on
    auto read4 = [&](uint32_t j) {
        float w[4] = {0.f, 0.f, 0.f, 0.f};
        if (j < rows) {
            const Place8 p = place8(a, bt, (int)j);  // (of all four)
            if (p.id >= 0) {
                const float* at = weight_at(a, p, h);
                if (a.four) {
                    const float4 y = *reinterpret_cast<const float4*>(at);
                    w[0] = y.x; w[1] = y.y; w[2] = y.z; w[3] = y.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = at[i * a.wr];
                }
            }
        }
        u32x4_t k;
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = j + i < rows ? key_of(w[i]) : 0u;
        return k;
    };
    auto keys4 = [&](uint32_t j) {
        if constexpr (KEYS > 0) return *reinterpret_cast<const u32x4_t*>(key_s + j);
        else return read4(j);
    };
    const uint32_t end4 = (rows + 4 * kSThreads - 1) / (4 * kSThreads) * (4 * kSThreads);  // whole rounds of the workgroup
    if constexpr (KEYS > 0) {
        static_assert(KEYS % (4 * kSThreads) == 0, "whole rounds");
#pragma unroll 2
        for (uint32_t j = 4 * tid; j < end4; j += 4 * kSThreads) *reinterpret_cast<u32x4_t*>(key_s + j) = read4(j);
    }
    __syncthreads();

    // ---- the threshold t: candidates above it stay, and of those at it the first `spare`
    uint32_t t = 0;
    bool met = need == 0;  // (none but the tail stays)
    for (int pass = 0, left = need; pass < 3 && !met; ++pass) {  // left: to stay of those that begin with t's bits
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, known = pass == 0 ? 0 : pass == 1 ? 21 : 10;
        const uint32_t mask = pass < 2 ? kBins - 1 : kBins / 2 - 1;
        count_s[tid] = count_s[tid + kSThreads] = 0;
        __syncthreads();
        for (uint32_t j = 4 * tid; j < end4; j += 4 * kSThreads) {
            const u32x4_t k = keys4(j);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool on = j + i < rows && (pass == 0 || (k[i] ^ t) >> known == 0);
                const uint64_t any = __ballot(on);
                if (any == 0) continue;
                const int bin = (int)(k[i] >> shift & mask), one = __builtin_amdgcn_readlane(bin, __builtin_ctzll(any));
                if (__ballot(on && bin == one) == any) {  // (all the same)
                    if (lane == __builtin_ctzll(any)) atomicAdd(&count_s[one], __builtin_popcountll(any));
                } else if (on) {
                    atomicAdd(&count_s[bin], 1);
                }
            }
        }
        __syncthreads();
        // sums from the top: thread i holds the two bins of its place counted from above
        const int top = kBins - 1 - 2 * tid, c0 = count_s[top], c1 = count_s[top - 1];
        const int inc = scan64(c0 + c1);
        if (lane == 63) sum_s[wave] = inc;
        __syncthreads();
        int above = inc - c0 - c1;
#pragma unroll
        for (int w = 0; w < kSWaves; ++w) above += w < wave ? sum_s[w] : 0;
        if (above < left && left <= above + c0 + c1) {  // (one thread)
            const bool first = left <= above + c0;
            found_s[0] = first ? top : top - 1;
            found_s[1] = left - above - (first ? 0 : c0);  // to stay of this bin
            found_s[2] = first ? c0 : c1;                  // and what it holds
        }
        __syncthreads();
        t |= (uint32_t)found_s[0] << shift;
        left = found_s[1];
        met = found_s[2] == left;
    }
    // (met: all that reach t stay; with need = 0 none)
    if (met) t -= 1;

    // ---- the rows that stay, in order: those above t, and of those at t the first.  Each
    // wavefront takes consecutive rows.
    const uint32_t per = ((rows + kSWaves - 1) / kSWaves + 255) / 256 * 256, w0 = wave * per, w1 = min(w0 + per, rows);
    int gt = 0, eq = 0;
    for (uint32_t j = w0; j < w1; j += 256) {
        const u32x4_t k = j + 4 * lane < end4 ? keys4(j + 4 * lane) : u32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            gt += __builtin_popcountll(__ballot(k[i] > t));
            eq += __builtin_popcountll(__ballot(k[i] == t));
        }
    }
    if (lane == 0) {
        gt_s[wave] = gt;
        eq_s[wave] = eq;
    }
    __syncthreads();
    int all_gt = 0, base_gt = 0, base_eq = 0;
#pragma unroll
    for (int w = 0; w < kSWaves; ++w) {
        all_gt += gt_s[w];
        base_gt += w < wave ? gt_s[w] : 0;
        base_eq += w < wave ? eq_s[w] : 0;
    }
    const int spare = need - all_gt;  // (of those at t; none where all that reach it stay)
    uint32_t gone = rows;  // the first row that goes
    int low = 0;           // rows that stay in front of `safe`
    for (uint32_t j = w0; j < w1; j += 256) {
        const u32x4_t k = j + 4 * lane < end4 ? keys4(j + 4 * lane) : u32x4_t{0, 0, 0, 0};
        // a lane's four rows are adjacent: sums of the lanes below
        int g = 0, e = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            g += k[i] > t;
            e += k[i] == t;
        }
        const int both = g | e << 16, inc = scan64(both), last = __builtin_amdgcn_readlane(inc, 63);
        int at_g = base_gt + ((inc - both) & 0xffff), at_e = base_eq + ((inc - both) >> 16);
        const Place8 p = both ? place8(a, bt, (int)(j + 4 * lane)) : Place8{-1, 0};  // (of all four)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t row = j + 4 * lane + i;
            const bool is_gt = k[i] > t, is_eq = k[i] == t;
            if (is_gt || (is_eq && at_e < spare)) {
                idx[at_g + min(at_e, spare)] = packed8(a, Place8{p.id, p.row + i});
                low += row < (uint32_t)a.safe;
            } else {
                gone = min(gone, row);
            }
            at_g += is_gt;
            at_e += is_eq;
        }
        base_gt += last & 0xffff;
        base_eq += last >> 16;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        gone = min(gone, (uint32_t)__shfl_xor((int)gone, o));
        low += __shfl_xor(low, o);
    }
    if (lane == 0) {
        if (gone < rows) atomicMin(&first_s, (int)gone);
        atomicAdd(&low_s, low);
    }
    for (int r = tid; r < tail; r += kSThreads) idx[need + r] = packed8(a, place8(a, bt, m + r));
    __syncthreads();
    // (first_s = budget: the rows that stay are the first ones)
    if (tid == 0) a.head[bh] = Head8{first_s < a.budget ? first_s : kStay, a.budget, low_s, 0};
}

// Rows of changing blocks that stay and lie in front of `safe`, into the workspace: 64
// per workgroup, in K (blockIdx.y 0) or V.
template <int D>
__global__ void __launch_bounds__(kEThreads) mfa_kv8_save_kernel(E8Args a) {
    constexpr int CPR = D / 16, NI = (kKv8Block * CPR + kEThreads - 1) / kEThreads;
    const int bh = (int)quotient(blockIdx.x, a.by_blocks), h = bh % a.H, which = blockIdx.y;
    const int i0 = ((int)blockIdx.x - bh * a.blocks) * kKv8Block;
    const Head8 head = a.head[bh];
    // (a block that changes takes all of its rows)
    if (head.first == kStay || i0 + kKv8Block <= head.first || i0 >= head.low) return;
    const int32_t* idx = a.idx + (int64_t)bh * a.rows;
    const Kv4Pool& q = a.pool[which];
    const int64_t pools = (int64_t)a.B * a.H * a.rows, saved = (int64_t)bh * a.rows;
    const int rows = min(head.low - i0, kKv8Block);
    u32x4_t w[NI];
    uint8_t s[NI];
    float weight[NI];
    bool on[NI];
#pragma unroll
    for (int x = 0; x < NI; ++x) {
        const int u = (int)threadIdx.x + kEThreads * x, r = u / CPR, c = u - r * CPR;
        on[x] = false;
        if (r >= rows) continue;
        const int j = idx[i0 + r];
        on[x] = j >= 0;
        if (!on[x]) continue;
        const Place8 p = unpacked8(a, j);
        w[x] = *reinterpret_cast<const u32x4_t*>(q.codes + p.id * q.cp + p.row * q.cr + h * q.ch + 16 * c);
        if (c == 0) s[x] = q.scales[p.id * q.sp + p.row / kKv8Block * q.sr + h * q.sh];
        if (which == 0 && c == 0) weight[x] = *weight_at(a, p, h);
    }
#pragma unroll
    for (int x = 0; x < NI; ++x) {
        const int u = (int)threadIdx.x + kEThreads * x, r = u / CPR, c = u - r * CPR;
        if (!on[x]) continue;
        const int64_t at = saved + i0 + r;
        *reinterpret_cast<u32x4_t*>(a.codes + (which * pools + at) * D + 16 * c) = w[x];
        if (c == 0) a.scales[which * pools + at] = s[x];
        if (which == 0 && c == 0) a.sw[at] = weight[x];
    }
}

// The largest finite magnitude of 16 codes at scale s, as bits.  Magnitudes of codes have
// the order of their values: one more than each (NaN: 0) compares in halves of a dword.
__device__ __forceinline__ uint32_t largest8(const u32x4_t& w, float s) {
    if (s >= 0x1p120f) {  // (some codes stand for values that are not finite)
        uint32_t mx = 0;
#pragma unroll 1
        for (int e = 0; e < 16; ++e) {
            const uint32_t z = __float_as_uint(__builtin_amdgcn_cvt_f32_fp8((int)(w[e >> 2] >> 8 * (e & 3)), 0) * s) & 0x7fffffffu;
            mx = max(mx, z < 0x7f800000u ? z : 0u);
        }
        return mx;
    }
    typedef __attribute__((__vector_size__(2 * sizeof(uint16_t)))) uint16_t u16x2_t;
    u16x2_t m = {0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t y = ((w[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x7f7f7f7fu;
        m = __builtin_elementwise_max(m, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, y & 0x00ff00ffu),
                                                                   __builtin_bit_cast(u16x2_t, y >> 8 & 0x00ff00ffu)));
    }
    const uint32_t code = max(max((uint32_t)m[0], (uint32_t)m[1]), 1u) - 1;
    return __float_as_uint(__builtin_amdgcn_cvt_f32_fp8((int)code, 0) * s);
}
// 16 codes of scale s under a new byte.  Above 2^18 the factor only meets zeros and NaN (a
// code is at least 2^-9, a new one at most 448), and an infinite one would make them NaN.
__device__ __forceinline__ u32x4_t rounded8(const u32x4_t& w, float s, uint32_t byte) {
    const float f = fminf(s * kv8_inverse(byte), 0x1p18f);
    typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f2;
    u32x4_t z;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const f2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[e], f, false), y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[e], f, true);
        z[e] = kv8_round4(x[0], x[1], y[0], y[1]);
    }
    return z;
}

// 64 new rows of a head, in K (blockIdx.y 0) or V
template <int D>
__global__ void __launch_bounds__(kEThreads) mfa_kv8_gather_kernel(E8Args a) {
    constexpr int CPR = D / 16, NI = (kKv8Block * CPR + kEThreads - 1) / kEThreads;
    __shared__ uint32_t max_s[kEThreads / 64];
    const int bh = (int)quotient(blockIdx.x, a.by_blocks), b = bh / a.H, h = bh - b * a.H, which = blockIdx.y;
    const int i0 = ((int)blockIdx.x - bh * a.blocks) * kKv8Block;
    const int tid = threadIdx.x, lane = tid & 63;
    const Head8 head = a.head[bh];
    if (i0 == 0 && h == 0 && which == 0 && tid == 0) a.new_lens[b] = head.n;
    if (head.first == kStay || i0 + kKv8Block <= head.first || i0 >= a.budget) return;
    const int32_t* bt = a.bt + b * a.bt_b;
    const int32_t* idx = a.idx + (int64_t)bh * a.rows;
    const Kv4Pool& q = a.pool[which];
    const int64_t pools = (int64_t)a.B * a.H * a.rows, saved = (int64_t)bh * a.rows;
    u32x4_t w[NI];
    float s[NI], weight[NI];
    const int rows = min(a.budget - i0, kKv8Block);
#pragma unroll
    for (int x = 0; x < NI; ++x) {
        const int u = tid + kEThreads * x, r = u / CPR, c = u - r * CPR;
        w[x] = u32x4_t{0, 0, 0, 0};
        s[x] = weight[x] = 0.f;
        if (r >= rows) continue;
        const int j = idx[i0 + r];
        if (j < 0) continue;  // (zeros)
        const Place8 p = unpacked8(a, j);
        if (i0 + r < head.low) {
            const int64_t at = saved + i0 + r;
            w[x] = *reinterpret_cast<const u32x4_t*>(a.codes + (which * pools + at) * D + 16 * c);
            s[x] = kv8_scale(a.scales[which * pools + at]);
            if (which == 0 && c == 0) weight[x] = a.sw[at];
        } else {
            w[x] = *reinterpret_cast<const u32x4_t*>(q.codes + p.id * q.cp + p.row * q.cr + h * q.ch + 16 * c);
            s[x] = kv8_scale(q.scales[p.id * q.sp + p.row / kKv8Block * q.sr + h * q.sh]);
            if (which == 0 && c == 0) weight[x] = *weight_at(a, p, h);
        }
    }
    uint32_t mx = 0;
#pragma unroll
    for (int x = 0; x < NI; ++x) mx = max(mx, largest8(w[x], s[x]));
    mx = max64(mx);
    if (lane == 63) max_s[tid >> 6] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEThreads / 64; ++i) mx = max(mx, max_s[i]);
    const uint32_t byte = kv8_byte_of(mx);
    const Place8 to = place8(a, bt, i0);  // (64 rows lie in one page)
    if (to.id < 0) return;
    uint8_t* const dst = q.codes + to.id * q.cp + to.row * q.cr + h * q.ch;
    if (tid == 0) q.scales[to.id * q.sp + to.row / kKv8Block * q.sr + h * q.sh] = (uint8_t)byte;
#pragma unroll
    for (int x = 0; x < NI; ++x) {
        const int u = tid + kEThreads * x, r = u / CPR, c = u - r * CPR;
        if (r >= rows) continue;
        *reinterpret_cast<u32x4_t*>(dst + r * q.cr + 16 * c) = rounded8(w[x], s[x], byte);
        if (which == 0 && c == 0) a.w[to.id * a.wp + (to.row + r) * a.wr + h * a.wh] = weight[x];
    }
}

// All new rows of a head, in K or in V, by one workgroup, blocks in order: row i comes from
// a row >= i, so what a step writes lies in front of all that later steps read, and the
// rows of the next two steps are on their way while this one's are rounded.  Loads have no
// branches (a row that is none reads the pool's first), so that waits can be counted.
template <int D, bool IS_K>
__device__ __forceinline__ void walk8(const E8Args& a, const Head8& head, int b, int h) {
    constexpr int THREADS = walk_threads(D), CPR = D / 16, NI = 2;
    constexpr int UNITS = THREADS / 64 * NI;  // wavefront loads per step, CPR of them a block
    constexpr int ROWS = UNITS / CPR * kKv8Block;
    static_assert(UNITS % CPR == 0, "whole blocks");
    __shared__ uint32_t max_s[2][UNITS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int32_t* bt = a.bt + b * a.bt_b;
    const int32_t* idx = a.idx + (int64_t)(b * a.H + h) * a.rows;
    const Kv4Pool& q = a.pool[IS_K ? 0 : 1];
    int row[NI], col[NI];  // of a step
#pragma unroll
    for (int x = 0; x < NI; ++x) {
        const int u = tid + THREADS * x;
        row[x] = u / CPR;
        col[x] = u - row[x] * CPR;
    }
    struct Places {
        int from[NI], to[NI];  // place of a row, page id of its new one
    };
    struct Rows {
        u32x4_t w[NI];
        uint32_t s[NI];
        float weight[NI];
        bool on[NI];
        int to[NI];
    };
    auto places = [&](int base, Places& j) {
#pragma unroll
        for (int x = 0; x < NI; ++x) {
            const int i = min(base + row[x], a.budget - 1);
            j.from[x] = idx[i];
            j.to[x] = bt[quotient((uint32_t)i, a.by_page)];
        }
    };
    auto load = [&](int base, const Places& j, Rows& y) {
#pragma unroll
        for (int x = 0; x < NI; ++x) {
            y.on[x] = j.from[x] >= 0 && base + row[x] < a.budget;
            y.to[x] = j.to[x];
            const Place8 p = unpacked8(a, max(j.from[x], 0));
            y.w[x] = *reinterpret_cast<const u32x4_t*>(q.codes + p.id * q.cp + p.row * q.cr + h * q.ch + 16 * col[x]);
            y.s[x] = q.scales[p.id * q.sp + p.row / kKv8Block * q.sr + h * q.sh];
            if (IS_K) y.weight[x] = *weight_at(a, p, h);
        }
    };
    int base = head.first / kKv8Block * kKv8Block, turn = 0;
    // rows `now` are written; `last`, two steps on, are loaded from `j`, and the places
    // after them into `fill`
    auto step = [&](Rows& now, Rows& last, const Places& j, Places& fill) {
        places(base + 3 * ROWS, fill);
        load(base + 2 * ROWS, j, last);
        float s[NI];
#pragma unroll
        for (int x = 0; x < NI; ++x) {
            if (!now.on[x]) now.w[x] = u32x4_t{0, 0, 0, 0};
            s[x] = kv8_scale(now.s[x]);
            const uint32_t mx = max64(largest8(now.w[x], s[x]));
            if (lane == 63) max_s[turn][wave + THREADS / 64 * x] = mx;
        }
        __syncthreads();  // (and this step's rows are all read)
#pragma unroll
        for (int x = 0; x < NI; ++x) {
            const int block = (wave + THREADS / 64 * x) / CPR, i = base + row[x], id = now.to[x];
            if (i >= a.budget || (uint32_t)id >= (uint32_t)a.npages) continue;
            uint32_t mx = 0;
#pragma unroll
            for (int i = 0; i < CPR; ++i) mx = max(mx, max_s[turn][block * CPR + i]);
            const uint32_t byte = kv8_byte_of(mx);
            const int r = i - (int)quotient((uint32_t)i, a.by_page) * a.page;
            *reinterpret_cast<u32x4_t*>(q.codes + id * q.cp + r * q.cr + h * q.ch + 16 * col[x]) =
                rounded8(now.w[x], s[x], byte);
            if (col[x] != 0) continue;
            if (r % kKv8Block == 0) q.scales[id * q.sp + r / kKv8Block * q.sr + h * q.sh] = (uint8_t)byte;
            if (IS_K) a.w[id * a.wp + r * a.wr + h * a.wh] = now.on[x] ? now.weight[x] : 0.f;
        }
        base += ROWS;
        turn ^= 1;
        return base < a.budget;
    };
    Places j0, j1, j2;
    Rows r0, r1, r2;
    places(base, j0);
    places(base + ROWS, j1);
    load(base, j0, r0);
    places(base + 2 * ROWS, j2);
    load(base + ROWS, j1, r1);
    while (step(r0, r2, j2, j0) && step(r1, r0, j0, j1) && step(r2, r1, j1, j2)) {
    }
}

template <int D>
__global__ void __launch_bounds__(walk_threads(D)) mfa_kv8_walk_kernel(E8Args a) {
    const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H;
    const Head8 head = a.head[blockIdx.x];
    if (h == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.new_lens[b] = head.n;
    if (head.first == kStay || a.npages == 0) return;
    if (blockIdx.y == 0) walk8<D, true>(a, head, b, h);
    else walk8<D, false>(a, head, b, h);
}

// No row moves: no sequence is longer than its budget, or none keeps a row
__global__ void __launch_bounds__(kEThreads) mfa_kv8_lengths_kernel(E8Args a) {
    const int b = blockIdx.x * kEThreads + threadIdx.x;
    if (b < a.B) a.new_lens[b] = min(max(a.lens[b], 0), min(a.max_k, a.budget));
}

int e8err(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(mfa_error_buffer(), 512, fmt, ap);
    va_end(ap);
    return code;
}

// checks, arguments (without the workspace's addresses) and the workspace's bytes
int e8_plan(const mfa_kv8_evict_params* p, E8Args* out, int64_t* bytes) {
    static const char who[] = "mfa_kv8_evict";
    if (!p) return e8err(MFA_ERR_INVALID, "%s: params is NULL", who);
    if (p->head_dim != 32 && p->head_dim != 64 && p->head_dim != 96 && p->head_dim != 128)
        return e8err(MFA_ERR_UNSUPPORTED, "%s: head_dim %d (32, 64, 96 or 128)", who, p->head_dim);
    if (p->batch < 0 || p->heads_kv <= 0 || p->max_seqlen_k < 0 || p->budget < 0 || p->recent < 0)
        return e8err(MFA_ERR_INVALID, "%s: negative size, budget or recent, or no heads", who);
    const int rc = mfa_kv4_check_cache(&p->cache, p->batch, p->head_dim, who);
    if (rc != MFA_OK) return rc;
    E8Args& a = *out;
    memset(&a, 0, sizeof(a));
    *bytes = 0;
    if (p->batch == 0) return MFA_OK;
    auto bad = [](const void* x) { return !x || (reinterpret_cast<uintptr_t>(x) & 3); };
    if (bad(p->cache_seqlens) || bad(p->new_seqlens))
        return e8err(MFA_ERR_INVALID, "%s: cache_seqlens and new_seqlens are required", who);
    if (p->cache.num_pages > 0 && bad(p->weights)) return e8err(MFA_ERR_INVALID, "%s: weights are required", who);
    if (p->weight_row_stride < 0 || p->weight_head_stride < 0)
        return e8err(MFA_ERR_INVALID, "%s: row and head strides must be >= 0", who);
    const int64_t cap = (int64_t)p->cache.max_pages * p->cache.page_block_size;
    a.max_k = (int32_t)std::min<int64_t>(p->max_seqlen_k ? p->max_seqlen_k : cap, cap);  // (below 2^31: checked)
    a.pool[0] = kv4_pool(p->cache.k);
    a.pool[1] = kv4_pool(p->cache.v);
    a.w = p->weights;
    a.wp = p->weight_page_stride; a.wr = p->weight_row_stride; a.wh = p->weight_head_stride;
    a.four = a.wr == 1 && a.wp % 4 == 0 && a.wh % 4 == 0 && (reinterpret_cast<uintptr_t>(a.w) & 15) == 0;
    a.bt = p->cache.block_table;
    a.bt_b = p->cache.block_table_batch_stride;
    a.lens = p->cache_seqlens;
    a.new_lens = p->new_seqlens;
    a.B = p->batch; a.H = p->heads_kv; a.D = p->head_dim;
    a.page = p->cache.page_block_size; a.npages = p->cache.num_pages;
    if ((int64_t)a.page * a.npages > 0x7fffffffLL) return e8err(MFA_ERR_INVALID, "%s: a pool of more than 2^31 - 1 rows", who);
    a.budget = p->budget; a.recent = p->recent;
    a.by_page = fast_div(a.page);
    const int64_t units = (int64_t)a.B * a.H;
    // (none: no row moves)
    a.rows = a.budget < a.max_k ? a.budget : 0;
    const int64_t blocks = ((int64_t)a.rows + kKv8Block - 1) / kKv8Block;
    // (a launch has less than 2^32 threads)
    if (units > 0x3fffff || units * blocks > 0x7fffff) return e8err(MFA_ERR_INVALID, "%s: problem too large", who);
    a.blocks = (int32_t)blocks;
    a.safe = (int32_t)(blocks * kKv8Block);
    a.by_blocks = fast_div(a.blocks);
    a.walk = units >= kWalk;
    const int64_t rows = units * a.rows;
    *bytes = a.rows == 0 ? 0 : (units * (int64_t)sizeof(Head8) + 255) / 256 * 256 + rows * (a.walk ? 4 : 8 + 2 * a.D + 2) + 64;
    return MFA_OK;
}

}  // namespace

extern "C" {

int mfa_kv8_evict_params_size(void) { return (int)sizeof(mfa_kv8_evict_params); }

int64_t mfa_kv8_evict_workspace_bytes(const mfa_kv8_evict_params* p) {
    mfa_error_buffer()[0] = 0;
    E8Args a;
    int64_t bytes;
    const int rc = e8_plan(p, &a, &bytes);
    return rc != MFA_OK ? rc : bytes;
}

int mfa_kv8_evict(const mfa_kv8_evict_params* p, void* workspace, int64_t workspace_bytes, void* stream) {
    mfa_error_buffer()[0] = 0;
    E8Args a;
    int64_t bytes;
    const int rc = e8_plan(p, &a, &bytes);
    if (rc != MFA_OK || a.B == 0) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (a.rows == 0) {
        hipLaunchKernelGGL(mfa_kv8_lengths_kernel, dim3((unsigned)((a.B + kEThreads - 1) / kEThreads)), dim3(kEThreads), 0, st, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e8err(MFA_ERR_LAUNCH, "mfa_kv8_evict: launch failed: %s", hipGetErrorString(e));
        return MFA_OK;
    }
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u))
        return e8err(MFA_ERR_INVALID, "mfa_kv8_evict: workspace must be a 256-byte aligned device pointer");
    if (workspace_bytes < bytes)
        return e8err(MFA_ERR_INVALID, "mfa_kv8_evict: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                     (long long)bytes);
    if (a.npages > 0 && p->cache.k.codes == p->cache.v.codes)
        return e8err(MFA_ERR_INVALID, "mfa_kv8_evict: K and V are the same memory");
    const int64_t units = (int64_t)a.B * a.H, rows = units * a.rows;
    char* ws = static_cast<char*>(workspace);
    a.head = reinterpret_cast<Head8*>(ws);
    ws += (units * (int64_t)sizeof(Head8) + 255) / 256 * 256;
    if (!a.walk) {
        a.codes = reinterpret_cast<uint8_t*>(ws);  // (16-byte aligned: rows of 32, 64, 96 or 128 bytes)
        ws += 2 * rows * a.D;
        a.sw = reinterpret_cast<float*>(ws);
        ws += 4 * rows;
    }
    a.idx = reinterpret_cast<int32_t*>(ws);
    if (!a.walk) a.scales = reinterpret_cast<uint8_t*>(a.idx + rows);
    const auto select = a.max_k <= 4096    ? mfa_kv8_select_kernel<4096>
                        : a.max_k <= 32768 ? mfa_kv8_select_kernel<32768>
                                           : mfa_kv8_select_kernel<0>;
    hipLaunchKernelGGL(select, dim3((unsigned)units), dim3(kSThreads), 0, st, a);
    typedef void (*fn)(E8Args);
    const auto of = [&](auto pick) { return a.D == 32 ? pick(std::integral_constant<int, 32>{}) : a.D == 64 ? pick(std::integral_constant<int, 64>{})
                                          : a.D == 96 ? pick(std::integral_constant<int, 96>{}) : pick(std::integral_constant<int, 128>{}); };
    if (a.walk) {
        const fn walk = of([](auto d) { return (fn)mfa_kv8_walk_kernel<decltype(d)::value>; });
        hipLaunchKernelGGL(walk, dim3((unsigned)units, 2), dim3(walk_threads(a.D)), 0, st, a);
    } else {
        const dim3 grid((unsigned)(units * a.blocks), 2);
        const fn save = of([](auto d) { return (fn)mfa_kv8_save_kernel<decltype(d)::value>; });
        hipLaunchKernelGGL(save, grid, dim3(kEThreads), 0, st, a);
        const fn gather = of([](auto d) { return (fn)mfa_kv8_gather_kernel<decltype(d)::value>; });
        hipLaunchKernelGGL(gather, grid, dim3(kEThreads), 0, st, a);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e8err(MFA_ERR_LAUNCH, "mfa_kv8_evict: launch failed: %s", hipGetErrorString(e));
    return MFA_OK;
}

}  // extern "C"
