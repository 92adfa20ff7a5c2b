// mfa_kv8_evict.hip -- eviction from a paged 8-bit K/V cache by accumulated weight
// (mfa_kv8_evict in include/mfa.h).
//
// Three kernels:
//  * select: one workgroup per (sequence, head) finds the weight of the last row that
//    stays and lists the rows that stay in order.  Weights become unsigned keys of the
//    same order; the threshold, the largest key that as many candidates reach as are
//    to stay, is found two bits at a time by counting with ballots (no histogram:
//    weights crowd into a few exponents, where counters in LDS would collide).  Keys
//    stay in registers where a sequence fits (64 K rows), else they are read again.
//  * save: rows only move down, and no block behind the one that holds row budget - 1
//    is written to; the rows that stay and lie in front are what another block's new
//    rows, or its new scale, may overwrite.  They go to the workspace as they are.
//  * gather: a workgroup per block of 64 new rows of a head, in K or in V, collects
//    its rows from the workspace and the cache, takes their largest magnitude, and
//    writes them with a new scale.
// Bound by the latency of the selection for one sequence, by the bytes of save and
// gather for a batch.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>

#include "mfa_kv8.h"

namespace {

constexpr int kSThreads = 1024, kSWaves = kSThreads / 64;
constexpr int kSKeys = 64;  // keys of a thread in registers, at most
constexpr int kEThreads = 256;
constexpr int kStay = 0x7fffffff;

// What select leaves for the kernels behind it.
struct Head8 {
    int32_t first;  // first row that moves (kStay: none)
    int32_t n;      // rows of the sequence afterwards
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
    int32_t rows;    // of the workspace per (sequence, head): the budget, or none where no sequence is longer
    int32_t blocks;  // of 64 new rows per (sequence, head), at least 1
    int32_t safe;    // rows from here on are read where they are
    FastDiv by_page, by_blocks;
    Head8* head;      // [B H]
    int32_t* idx;     // [B H rows] rows that stay, ascending
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

// N: keys of a thread, row ((i kSWaves + wavefront) 64 + lane) of a segment of 1024 N
template <int N>
__global__ void __launch_bounds__(kSThreads) mfa_kv8_select_kernel(E8Args a) {
    constexpr int kSegment = kSThreads * N, kGroups = kSWaves * N;  // groups of 64 rows
    static_assert(kGroups <= kSThreads, "a thread per group");
    __shared__ int count_s[16][4];
    __shared__ int gt_s[kGroups], eq_s[kGroups];
    __shared__ int2 part_s[kSWaves];
    __shared__ int first_s;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int bh = blockIdx.x, b = bh / a.H, h = bh - b * a.H;
    const int n = min(max(a.lens[b], 0), a.max_k);
    if (n <= a.budget) {
        if (tid == 0) a.head[bh] = Head8{kStay, n};
        return;
    }
    const int tail = min(a.recent, a.budget), m = n - tail, need = a.budget - tail;  // need < m
    const int32_t* bt = a.bt + b * a.bt_b;
    int32_t* const idx = a.idx + (int64_t)bh * a.rows;
    if (tid < 64) count_s[tid >> 2][tid & 3] = 0;
    if (tid == 0) first_s = m;
    uint32_t key[N];
    auto load = [&](int seg) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            // (64 rows of a wavefront lie in one page)
            const int j0 = seg + (i * kSWaves + wave) * 64;
            float w = 0.f;
            if (j0 < m) {
                const Place8 p = place8(a, bt, j0);
                if (p.id >= 0 && j0 + lane < m) w = a.w[p.id * a.wp + (p.row + lane) * a.wr + h * a.wh];
            }
            key[i] = __float_as_uint(w);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) key[i] = seg + (i * kSWaves + wave) * 64 + lane < m ? key_of(__uint_as_float(key[i])) : 0u;
    };
    const bool once = m <= kSegment;
    if (once) load(0);
    __syncthreads();

    // ---- the largest key that `need` candidates reach (need = 0: none stays but the tail)
    uint32_t t = 0;
    if (need > 0) {
        for (int step = 0; step < 16; ++step) {
            const int shift = 30 - 2 * step;
            const uint32_t t1 = t | 1u << shift, t2 = t | 2u << shift, t3 = t | 3u << shift;
            int c1 = 0, c2 = 0, c3 = 0;
            for (int seg = 0; seg < m; seg += kSegment) {
                if (!once) load(seg);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    c1 += __builtin_popcountll(__ballot(key[i] >= t1));
                    c2 += __builtin_popcountll(__ballot(key[i] >= t2));
                    c3 += __builtin_popcountll(__ballot(key[i] >= t3));
                }
            }
            if (lane == 0) {
                atomicAdd(&count_s[step][0], c1);
                atomicAdd(&count_s[step][1], c2);
                atomicAdd(&count_s[step][2], c3);
            }
            __syncthreads();
            if (count_s[step][2] >= need) t = t3;
            else if (count_s[step][1] >= need) t = t2;
            else if (count_s[step][0] >= need) t = t1;
        }
    }

    // ---- the rows that stay, in order: those above t, and of those at t the first
    int base_gt = 0, base_eq = 0, spare = 0;
    if (need > 0) {
        // (how many at t: need less those above it, counted on the way below)
        int gt = 0;
        for (int seg = 0; seg < m; seg += kSegment) {
            if (!once) load(seg);
#pragma unroll
            for (int i = 0; i < N; ++i) gt += __builtin_popcountll(__ballot(key[i] > t));
        }
        if (lane == 0) atomicAdd(&count_s[0][3], gt);
        __syncthreads();
        spare = need - count_s[0][3];
        for (int seg = 0; seg < m; seg += kSegment) {
            if (!once) load(seg);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint64_t g = __ballot(key[i] > t), e = __ballot(key[i] == t);
                if (lane == 0) {
                    gt_s[i * kSWaves + wave] = __builtin_popcountll(g);
                    eq_s[i * kSWaves + wave] = __builtin_popcountll(e);
                }
            }
            __syncthreads();
            // exclusive prefix sums over the groups
            const int g0 = tid < kGroups ? gt_s[tid] : 0, e0 = tid < kGroups ? eq_s[tid] : 0;
            int g = g0, e = e0;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int yg = __shfl_up(g, o), ye = __shfl_up(e, o);
                if (lane >= o) {
                    g += yg;
                    e += ye;
                }
            }
            if (lane == 63) part_s[wave] = make_int2(g, e);
            __syncthreads();
            int all_g = 0, all_e = 0;
#pragma unroll
            for (int w = 0; w < kSWaves; ++w) {
                const int2 p = part_s[w];
                if (w < wave) {
                    g += p.x;
                    e += p.y;
                }
                all_g += p.x;
                all_e += p.y;
            }
            if (tid < kGroups) {
                gt_s[tid] = base_gt + g - g0;
                eq_s[tid] = base_eq + e - e0;
            }
            __syncthreads();
            int gone = m;  // the first row that goes
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int row = seg + (i * kSWaves + wave) * 64 + lane;
                const bool is_gt = key[i] > t, is_eq = key[i] == t;
                const uint64_t gb = __ballot(is_gt), eb = __ballot(is_eq), below = (1ull << lane) - 1;
                const int eq = eq_s[i * kSWaves + wave] + __builtin_popcountll(eb & below);
                const bool stays = is_gt || (is_eq && eq < spare);
                if (stays) idx[gt_s[i * kSWaves + wave] + __builtin_popcountll(gb & below) + min(eq, spare)] = row;
                else if (row < gone) gone = row;
            }
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) gone = min(gone, __shfl_xor(gone, o));
            if (lane == 0 && gone < m) atomicMin(&first_s, gone);
            base_gt += all_g;
            base_eq += all_e;
            __syncthreads();
        }
    } else {
        if (tid == 0) first_s = 0;
        __syncthreads();
    }
    for (int r = tid; r < tail; r += kSThreads) idx[need + r] = m + r;
    // (first_s = budget: the rows that stay are the first ones)
    if (tid == 0) a.head[bh] = Head8{first_s < a.budget ? first_s : kStay, a.budget};
}

// Rows of changing blocks that stay and lie in front of `safe`, into the workspace: 64
// per workgroup.
__global__ void __launch_bounds__(kEThreads) mfa_kv8_save_kernel(E8Args a) {
    const int bh = (int)quotient(blockIdx.x, a.by_blocks), b = bh / a.H, h = bh - b * a.H;
    const int i0 = ((int)blockIdx.x - bh * a.blocks) * kKv8Block;
    const int first = a.head[bh].first;
    const int from = first / kKv8Block * kKv8Block;  // (a block that changes takes all of its rows)
    if (first == kStay || i0 + kKv8Block <= from) return;
    const int32_t* bt = a.bt + b * a.bt_b;
    const int32_t* idx = a.idx + (int64_t)bh * a.rows;
    const int tid = threadIdx.x, cpr = a.D / 16;
    for (int u = tid; u < kKv8Block * cpr; u += kEThreads) {
        const int r = u / cpr, c = u - r * cpr, i = i0 + r;
        if (i >= a.budget) break;
        const int j = idx[i];
        if (j >= a.safe) break;  // (ascending)
        const Place8 p = place8(a, bt, j);
        if (p.id < 0) continue;
        const int64_t at = (int64_t)bh * a.rows + i, pools = (int64_t)a.B * a.H * a.rows;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const Kv4Pool& q = a.pool[x];
            *reinterpret_cast<u32x4_t*>(a.codes + (x * pools + at) * a.D + 16 * c) =
                *reinterpret_cast<const u32x4_t*>(q.codes + p.id * q.cp + p.row * q.cr + h * q.ch + 16 * c);
            if (c == 0) a.scales[x * pools + at] = q.scales[p.id * q.sp + p.row / kKv8Block * q.sr + h * q.sh];
        }
        if (c == 0) a.sw[at] = *weight_at(a, p, h);
    }
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
        const Place8 p = place8(a, bt, j);
        if (p.id < 0) continue;  // (zeros)
        if (j < a.safe) {
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
    // the largest finite magnitude
    uint32_t mx = 0;
#pragma unroll
    for (int x = 0; x < NI; ++x) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float y[4];
            kv8_values4(w[x][e], s[x], y);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t z = __float_as_uint(y[i]) & 0x7fffffffu;
                mx = max(mx, z < 0x7f800000u ? z : 0u);
            }
        }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o));
    if (lane == 0) max_s[tid >> 6] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEThreads / 64; ++i) mx = max(mx, max_s[i]);
    const uint32_t byte = kv8_byte_of(mx);
    const float inv = kv8_inverse(byte);
    const Place8 to = place8(a, bt, i0);  // (64 rows lie in one page)
    if (to.id < 0) return;
    uint8_t* const dst = q.codes + to.id * q.cp + to.row * q.cr + h * q.ch;
    if (tid == 0) q.scales[to.id * q.sp + to.row / kKv8Block * q.sr + h * q.sh] = (uint8_t)byte;
#pragma unroll
    for (int x = 0; x < NI; ++x) {
        const int u = tid + kEThreads * x, r = u / CPR, c = u - r * CPR;
        if (r >= rows) continue;
        u32x4_t z;
        const float f = s[x] * inv;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float y[4];
            kv8_values4(w[x][e], f, y);
            z[e] = kv8_round4(y[0], y[1], y[2], y[3]);
        }
        *reinterpret_cast<u32x4_t*>(dst + r * q.cr + 16 * c) = z;
        if (which == 0 && c == 0) a.w[to.id * a.wp + (to.row + r) * a.wr + h * a.wh] = weight[x];
    }
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
    a.max_k = (int32_t)std::min<int64_t>(p->max_seqlen_k ? p->max_seqlen_k : cap, std::min<int64_t>(cap, 0x7fffff00));
    a.pool[0] = kv4_pool(p->cache.k);
    a.pool[1] = kv4_pool(p->cache.v);
    a.w = p->weights;
    a.wp = p->weight_page_stride; a.wr = p->weight_row_stride; a.wh = p->weight_head_stride;
    a.bt = p->cache.block_table;
    a.bt_b = p->cache.block_table_batch_stride;
    a.lens = p->cache_seqlens;
    a.new_lens = p->new_seqlens;
    a.B = p->batch; a.H = p->heads_kv; a.D = p->head_dim;
    a.page = p->cache.page_block_size; a.npages = p->cache.num_pages;
    a.budget = p->budget; a.recent = p->recent;
    a.by_page = fast_div(a.page);
    const int64_t units = (int64_t)a.B * a.H;
    // (no sequence is longer than its budget: no rows to hold)
    a.rows = a.budget < a.max_k ? a.budget : 0;
    const int64_t blocks = std::max<int64_t>(((int64_t)a.rows + kKv8Block - 1) / kKv8Block, 1);
    // (a launch has less than 2^32 threads)
    if (units > 0x3fffff || units * blocks > 0x7fffff) return e8err(MFA_ERR_INVALID, "%s: problem too large", who);
    a.blocks = (int32_t)blocks;
    a.safe = a.rows > 0 ? (int32_t)(blocks * kKv8Block) : 0;
    a.by_blocks = fast_div(a.blocks);
    const int64_t rows = units * a.rows;
    *bytes = (units * (int64_t)sizeof(Head8) + 255) / 256 * 256 + rows * (8 + 2 * a.D + 2) + 64;
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
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u))
        return e8err(MFA_ERR_INVALID, "mfa_kv8_evict: workspace must be a 256-byte aligned device pointer");
    if (workspace_bytes < bytes)
        return e8err(MFA_ERR_INVALID, "mfa_kv8_evict: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                     (long long)bytes);
    const int64_t units = (int64_t)a.B * a.H, rows = units * a.rows;
    char* ws = static_cast<char*>(workspace);
    a.head = reinterpret_cast<Head8*>(ws);
    ws += (units * (int64_t)sizeof(Head8) + 255) / 256 * 256;
    a.codes = reinterpret_cast<uint8_t*>(ws);  // (16-byte aligned: rows of 32, 64, 96 or 128 bytes)
    ws += 2 * rows * a.D;
    a.idx = reinterpret_cast<int32_t*>(ws);
    a.sw = reinterpret_cast<float*>(a.idx + rows);
    a.scales = reinterpret_cast<uint8_t*>(a.sw + rows);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    // keys in registers: as few as hold the longest sequence
    const auto select = a.max_k <= 4 * kSThreads    ? mfa_kv8_select_kernel<4>
                        : a.max_k <= 16 * kSThreads ? mfa_kv8_select_kernel<16>
                                                    : mfa_kv8_select_kernel<kSKeys>;
    hipLaunchKernelGGL(select, dim3((unsigned)units), dim3(kSThreads), 0, st, a);
    const unsigned grid = (unsigned)(units * a.blocks);
    if (a.rows > 0) hipLaunchKernelGGL(mfa_kv8_save_kernel, dim3(grid), dim3(kEThreads), 0, st, a);
    const auto gather = a.D == 32 ? mfa_kv8_gather_kernel<32> : a.D == 64 ? mfa_kv8_gather_kernel<64>
                        : a.D == 96 ? mfa_kv8_gather_kernel<96> : mfa_kv8_gather_kernel<128>;
    hipLaunchKernelGGL(gather, dim3(grid, 2), dim3(kEThreads), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e8err(MFA_ERR_LAUNCH, "mfa_kv8_evict: launch failed: %s", hipGetErrorString(e));
    return MFA_OK;
}

}  // extern "C"
