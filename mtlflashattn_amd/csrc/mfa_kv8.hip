// mfa_kv8.hip -- writing a paged 8-bit K/V cache (mfa_kv8_append in include/mfa.h).
//
// Bound by memory for prompts (8 prompts of 256 to 4096 rows, 8 heads of 128, fp16: 39 us,
// the copy rate), by the latency of dependent loads (prefix sums, page id, old scale) for
// decoding steps (24 rows: 5 us, half of what the call takes on the host).  A workgroup
// owns one block of 64 cache rows of one head, in K or in V: it takes the largest
// magnitude of all of the call's rows that fall into the block (held in registers where
// they fit, else read twice) and writes codes, values and the scale; so no two workgroups
// share a scale.  Four wavefronts where blocks fill, one for the few rows of steps, whose
// blocks are mostly latency: four times as many are on their way at once.  Where the
// block holds rows already and the new ones raise its scale, their codes are rounded
// again, at most 64 rows.  The scale comes from the maximum's exponent and mantissa
// bits and the elements are multiplied by its inverse, a power of two, before the
// conversion: every step but the rounding is exact.
//
// The blocks of the sequences are laid end to end; a workgroup finds its own from the
// prefix sums and lengths on the device, 64 sequences per step.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>

#include "mfa_kv8.h"

namespace {

// A block is one wavefront's where a call has at most this many new rows per sequence on
// average, and at least this many heads of sequences.  Which sequence has many rows is known
// on the device only, and a full block takes a wavefront 12 us and a workgroup 5: calls of
// fewer heads, whose blocks all run at once, lose more by it where they are ragged than they
// gain where they are not.
// (us as wavefronts / as workgroups, bf16 heads of 128.  8 of them, 256 sequences of 1, 5,
// 16, 32 rows: 8.0 / 12.7, 9.4 / 15.9, 12.0 / 18.4, 20.4 / 24.0; 255 single rows beside 400:
// 16.7 / 15.8, beside 3000: 18.2 / 18.8.  64 sequences of 1, 5, 16, 32: 5.0 / 5.7, 5.8 / 6.1,
// 6.7 / 6.4, 10.3 / 7.7; 63 single rows beside 900: 12.7 / 7.2.  32 heads, 64 single rows:
// 6.5 / 10.6; 63 beside 900: 16.7 / 15.8.)
constexpr int kStepRows = 16, kStepHeads = 2048;

struct A8Args {
    const char* x[2];  // k, v
    int64_t ts[2], hs[2];
    char* val[2];
    Kv4Pool pool[2];
    const int32_t* bt;
    int64_t bt_b;
    const int32_t* cu;
    const int32_t* lens;
    int32_t B, T, H, max_pages, npages, page, blocks;
    FastDiv by_page, by_heads;
};

// A sequence's new rows: tokens t0 .. t0 + n - 1 become rows p0 ..
struct NewRows {
    int t0, n;
    int p0;
    __device__ __forceinline__ int blocks() const { return n > 0 ? (int)(((int64_t)p0 + n - 1) / kKv8Block - p0 / kKv8Block) + 1 : 0; }
};
__device__ __forceinline__ NewRows new_rows(const A8Args& a, int b) {
    // (bounded by the tensor whatever the prefix sums hold)
    const int q0 = min(max(a.cu[b], 0), a.T), end = min(max(a.cu[b + 1], q0), a.T);
    return NewRows{q0, end - q0, max(a.lens[b], 0)};
}

template <int DT>
struct Raw8 {  // eight elements as loaded
    u32x4_t w[DT == MFA_DTYPE_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const char* p) {
        w[0] = *reinterpret_cast<const u32x4_t*>(p);
        if constexpr (DT == MFA_DTYPE_F32) w[1] = *reinterpret_cast<const u32x4_t*>(p + 16);
    }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (DT == MFA_DTYPE_F32) return __uint_as_float(w[i >> 2][i & 3]);
        const uint32_t y = w[0][i >> 1];
        if constexpr (DT == MFA_DTYPE_BF16) return __uint_as_float(i & 1 ? y & 0xffff0000u : y << 16);
        return (float)__builtin_bit_cast(k4_f16x2_t, y)[i & 1];
    }
};
template <int DT>
__device__ __forceinline__ void store_values8(char* p, u32x2_t codes, float s) {
    float x[8];
    float a[4], b[4];
    kv8_values4(codes[0], s, a);
    kv8_values4(codes[1], s, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = a[i];
        x[4 + i] = b[i];
    }
    if constexpr (DT == MFA_DTYPE_F32) {
        float4* q = reinterpret_cast<float4*>(p);
        q[0] = make_float4(x[0], x[1], x[2], x[3]);
        q[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        u32x4_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == MFA_DTYPE_BF16) {
                w[i] = __builtin_bit_cast(uint32_t, k4_bf16x2_t{(__bf16)x[2 * i], (__bf16)x[2 * i + 1]});
            } else {
                // (65504 may be held as 65536, one step above fp16's range: saturated, NaN stays NaN)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    x[2 * i + e] = __builtin_elementwise_minimum(__builtin_elementwise_maximum(x[2 * i + e], -65504.f), 65504.f);
                w[i] = __builtin_bit_cast(uint32_t, k4_f16x2_t{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
            }
        }
        *reinterpret_cast<u32x4_t*>(p) = w;
    }
}

template <int DT, int D, int T>
__global__ void __launch_bounds__(T) mfa_kv8_append_kernel(A8Args a) {
    constexpr int ES = DT == MFA_DTYPE_F32 ? 4 : 2, CPR = D / 8;
    constexpr int ALL = kKv8Block * CPR / T, NI = ALL < 4 ? ALL : 4;  // loads of 64 rows, and of those held at once
    __shared__ uint32_t max_s[T / 64];
    const int tid = threadIdx.x, lane = tid & 63, which = blockIdx.y;
    const int blk = (int)quotient(blockIdx.x, a.by_heads), h = (int)blockIdx.x - blk * a.H;
    char* const val = a.val[which] ? a.val[which] + (int64_t)h * D * ES : nullptr;
    const int64_t row_bytes = (int64_t)a.H * D * ES;

    // tokens of no sequence: values of 0, dealt over the blocks' workgroups
    if (val) {
        const int first = a.B > 0 ? min(max(a.cu[0], 0), a.T) : 0, end = a.B > 0 ? max(min(max(a.cu[a.B], 0), a.T), first) : 0;
        for (int t = blk; t < first + (a.T - end); t += a.blocks) {
            char* p = val + (int64_t)(t < first ? t : t - first + end) * row_bytes;
            if (tid < CPR) {
                *reinterpret_cast<u32x4_t*>(p + tid * 8 * ES) = u32x4_t{0, 0, 0, 0};
                if constexpr (ES == 4) *reinterpret_cast<u32x4_t*>(p + tid * 8 * ES + 16) = u32x4_t{0, 0, 0, 0};
            }
        }
    }

    // the sequence of block `blk`
    int b = -1, off = 0;
    for (int b0 = 0, base = 0; b0 < a.B && b < 0; b0 += 64) {
        const int n = b0 + lane < a.B ? new_rows(a, b0 + lane).blocks() : 0, inc = scan64(n);
        const uint64_t past = __ballot(inc + base > blk);
        if (past) {
            const int l = __builtin_ctzll(past);
            b = b0 + l;
            off = blk - base - __builtin_amdgcn_readlane(inc - n, l);
        }
        base += __builtin_amdgcn_readlane(inc, 63);
    }
    if (b < 0) return;  // (workgroup-uniform)
    const NewRows s = new_rows(a, b);
    const int64_t base = ((int64_t)(s.p0 / kKv8Block) + off) * kKv8Block;  // the block's first row
    const int lo = (int)max((int64_t)s.p0 - base, (int64_t)0);            // rows that it holds already
    const int n = (int)min((int64_t)s.p0 + s.n - base, (int64_t)kKv8Block) - lo;
    const int t0 = s.t0 + (int)(base + lo - s.p0);

    Raw8<DT> x[NI];
    uint32_t mx = 0;
    const char* const src = a.x[which] + (t0 * a.ts[which] + h * a.hs[which]) * ES;
    auto load = [&](int first) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int u = first + tid + T * i, r = u / CPR, d = 8 * (u - r * CPR);
            if (r < n) x[i].load(src + (r * a.ts[which] + d) * ES);
        }
    };
    load(0);
    // the block's place (none: behind the table or on a page outside the pool)
    const Kv4Pool& p = a.pool[which];
    uint8_t *codes = nullptr, *scale = nullptr;
    uint32_t old = 0;
    if (base < (int64_t)a.max_pages * a.page) {
        const int idx = (int)quotient((uint32_t)base, a.by_page), row = (int)base - idx * a.page;
        const int id = a.bt[b * a.bt_b + idx];
        if ((uint32_t)id < (uint32_t)a.npages) {
            codes = p.codes + id * p.cp + row * p.cr + h * p.ch;
            scale = p.scales + id * p.sp + row / kKv8Block * p.sr + h * p.sh;
            if (lo > 0) old = min((uint32_t)*scale, 253u);
        }
    }
    // the largest finite magnitude
    for (int first = 0; first < n * CPR; first += T * NI) {
        if (first > 0) load(first);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            if ((first + tid + T * i) / CPR < n) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t y = __float_as_uint(x[i].at(e)) & 0x7fffffffu;
                    mx = max(mx, y < 0x7f800000u ? y : 0u);
                }
            }
        }
        if (NI == ALL) break;
    }
    mx = max64(mx);
    if (lane == 63) max_s[tid >> 6] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 64; ++w) mx = max(mx, max_s[w]);
    const uint32_t byte = max(kv8_byte_of(mx), old);
    const float inv = kv8_inverse(byte), sc = kv8_scale(byte), top = kv8_top(byte);

    for (int first = 0; first < n * CPR; first += T * NI) {
        if (n * CPR > T * NI) load(first);  // (else still held)
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int u = first + tid + T * i, r = u / CPR, d = 8 * (u - r * CPR);
            if (r >= n) continue;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float z = x[i].at(e);
                y[e] = (__float_as_uint(z) & 0x7fffffffu) < 0x7f800000u ? __builtin_amdgcn_fmed3f(z * inv, -top, top) : __builtin_nanf("");
            }
            const u32x2_t c = {kv8_round4(y[0], y[1], y[2], y[3]), kv8_round4(y[4], y[5], y[6], y[7])};
            if (codes) *reinterpret_cast<u32x2_t*>(codes + (int64_t)(lo + r) * p.cr + d) = c;
            if (val) store_values8<DT>(val + (t0 + r) * row_bytes + d * ES, c, sc);
        }
        if (NI == ALL) break;
    }
    if (!codes) return;
    if (tid == 0) *scale = (uint8_t)byte;
    if (lo > 0 && byte > old) {  // the rows that were there, by the new scale
        const float f = kv8_scale(old) * inv;
        for (int u = tid; u < lo * CPR; u += T) {
            const int r = u / CPR;
            u32x2_t* q = reinterpret_cast<u32x2_t*>(codes + (int64_t)r * p.cr + 8 * (u - r * CPR));
            const u32x2_t c = *q;
            float y[4], z[4];
            kv8_values4(c[0], f, y);
            kv8_values4(c[1], f, z);
            *q = u32x2_t{kv8_round4(y[0], y[1], y[2], y[3]), kv8_round4(z[0], z[1], z[2], z[3])};
        }
    }
}

int a8err(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(mfa_error_buffer(), 512, fmt, ap);
    va_end(ap);
    return code;
}

typedef void (*a8_fn)(A8Args);
template <int DT, int T>
a8_fn append_of(int d) {
    return d == 32 ? mfa_kv8_append_kernel<DT, 32, T> : d == 64 ? mfa_kv8_append_kernel<DT, 64, T>
           : d == 96 ? mfa_kv8_append_kernel<DT, 96, T> : mfa_kv8_append_kernel<DT, 128, T>;
}
template <int T>
a8_fn append_of(int dtype, int d) {
    return dtype == MFA_DTYPE_F32    ? append_of<MFA_DTYPE_F32, T>(d)
           : dtype == MFA_DTYPE_BF16 ? append_of<MFA_DTYPE_BF16, T>(d)
                                     : append_of<MFA_DTYPE_F16, T>(d);
}

}  // namespace

extern "C" {

int mfa_kv8_append_params_size(void) { return (int)sizeof(mfa_kv8_append_params); }

int mfa_kv8_append(const mfa_kv8_append_params* p, void* stream) {
    mfa_error_buffer()[0] = 0;
    if (!p) return a8err(MFA_ERR_INVALID, "mfa_kv8_append: params is NULL");
    if (p->dtype != MFA_DTYPE_F16 && p->dtype != MFA_DTYPE_BF16 && p->dtype != MFA_DTYPE_F32)
        return a8err(MFA_ERR_INVALID, "mfa_kv8_append: unknown dtype %d", p->dtype);
    if (p->batch < 0 || p->total < 0 || p->heads_kv < 0) return a8err(MFA_ERR_INVALID, "mfa_kv8_append: negative size");
    if (p->head_dim != 32 && p->head_dim != 64 && p->head_dim != 96 && p->head_dim != 128)
        return a8err(MFA_ERR_UNSUPPORTED, "mfa_kv8_append: head_dim %d (32, 64, 96 or 128)", p->head_dim);
    const int rc = mfa_kv4_check_cache(&p->cache, p->batch, p->head_dim, "mfa_kv8_append");
    if (rc != MFA_OK) return rc;
    // (tokens of no sequence have values too)
    if (p->total == 0 || p->heads_kv == 0 || (p->batch == 0 && !p->k_values && !p->v_values)) return MFA_OK;
    auto bad = [](const void* x, uintptr_t al) { return !x || (reinterpret_cast<uintptr_t>(x) & (al - 1)); };
    if (bad(p->k, 16) || bad(p->v, 16)) return a8err(MFA_ERR_INVALID, "mfa_kv8_append: k and v must be 16-byte aligned");
    const int al = p->dtype == MFA_DTYPE_F32 ? 4 : 8;
    if (p->k_token_stride % al || p->k_head_stride % al || p->v_token_stride % al || p->v_head_stride % al)
        return a8err(MFA_ERR_INVALID, "mfa_kv8_append: k and v strides must be multiples of %d elements", al);
    if ((p->k_values == nullptr) != (p->v_values == nullptr) || (p->k_values && (bad(p->k_values, 16) || bad(p->v_values, 16))))
        return a8err(MFA_ERR_INVALID, "mfa_kv8_append: k_values and v_values must both be NULL or 16-byte aligned");
    if (bad(p->cu_seqlens, 4) || (p->batch > 0 && bad(p->cache_seqlens, 4)))
        return a8err(MFA_ERR_INVALID, "mfa_kv8_append: cu_seqlens and cache_seqlens are required");
    A8Args a;
    memset(&a, 0, sizeof(a));
    a.x[0] = static_cast<const char*>(p->k);
    a.x[1] = static_cast<const char*>(p->v);
    a.ts[0] = p->k_token_stride; a.hs[0] = p->k_head_stride;
    a.ts[1] = p->v_token_stride; a.hs[1] = p->v_head_stride;
    a.val[0] = static_cast<char*>(p->k_values);
    a.val[1] = static_cast<char*>(p->v_values);
    a.pool[0] = kv4_pool(p->cache.k);
    a.pool[1] = kv4_pool(p->cache.v);
    a.bt = p->cache.block_table;
    a.bt_b = p->cache.block_table_batch_stride;
    a.cu = p->cu_seqlens;
    a.lens = p->cache_seqlens;
    a.B = p->batch; a.T = p->total; a.H = p->heads_kv;
    a.max_pages = p->cache.max_pages; a.npages = p->cache.num_pages; a.page = p->cache.page_block_size;
    a.by_page = fast_div(a.page);
    a.by_heads = fast_div(a.H);
    // a bound on the blocks: a sequence of n rows touches at most n / 64 + 2, and at most n
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(p->total, p->total / kKv8Block + 2 * (int64_t)p->batch));
    if (blocks * p->heads_kv > 0x7fffff) return a8err(MFA_ERR_INVALID, "mfa_kv8_append: problem too large");
    a.blocks = (int32_t)blocks;
    const bool step = p->total <= kStepRows * (int64_t)p->batch && (int64_t)p->batch * p->heads_kv >= kStepHeads;
    const int threads = step ? 64 : 256;
    const a8_fn fn = step ? append_of<64>(p->dtype, p->head_dim) : append_of<256>(p->dtype, p->head_dim);
    hipLaunchKernelGGL(fn, dim3((unsigned)(blocks * p->heads_kv), 2), dim3(threads), 0, static_cast<hipStream_t>(stream), a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return a8err(MFA_ERR_LAUNCH, "mfa_kv8_append: launch failed: %s", hipGetErrorString(e));
    return MFA_OK;
}

}  // extern "C"
