// mfa_kv4.hip -- writing a paged 4-bit K/V cache (mfa_kv4_append in
// include/mfa.h) and the argument checks that its users share.
//
// Bound by memory: a lane takes 8 elements (16 bytes of a 16-bit row), the four
// lanes of a 32-element group share its maximum by two cross-lane steps, and each
// stores 4 code bytes, so loads and stores of a wavefront are contiguous.  The
// scale comes from the maximum's exponent and mantissa bits and the elements are
// multiplied by its inverse, a power of two, before the conversion: every step
// but the rounding is exact.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include "mfa_kv4.h"

namespace {

constexpr int kAThreads = 256;
constexpr int kASeqs = 1024;  // prefix sums kept in LDS (above: read from memory)

struct AArgs {
    const char* x[2];  // k, v
    int64_t ts[2], hs[2];
    char* val[2];
    Kv4Pool pool[2];
    const int32_t* bt;
    int64_t bt_b;
    const int32_t* cu;
    const int32_t* lens;
    int32_t B, T, H, D, max_pages, npages, page;
    FastDiv by_page, by_row, by_head;  // elements: chunks of a token, chunks of a head
    int32_t chunks;                    // T * H * D / 8
};

// DT: MFA_DTYPE_*; eight elements as floats and back
template <int DT>
__device__ __forceinline__ void load8(const char* p, float (&x)[8]) {
    if constexpr (DT == MFA_DTYPE_F32) {
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(p), b = *reinterpret_cast<const u32x4_t*>(p + 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = __uint_as_float(a[i]);
            x[4 + i] = __uint_as_float(b[i]);
        }
    } else {
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == MFA_DTYPE_BF16) {
                x[2 * i] = __uint_as_float(a[i] << 16);
                x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
            } else {
                const k4_f16x2_t h = __builtin_bit_cast(k4_f16x2_t, (uint32_t)a[i]);
                x[2 * i] = (float)h[0];
                x[2 * i + 1] = (float)h[1];
            }
        }
    }
}
template <int DT>
__device__ __forceinline__ void store_values8(char* p, uint32_t codes, uint32_t scale) {
    const float s = kv4_scale(scale);
    if constexpr (DT == MFA_DTYPE_F32) {
        typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f2;
        const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 1);
        const f2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 3);
        float4* q = reinterpret_cast<float4*>(p);
        q[0] = make_float4(a[0], a[1], b[0], b[1]);
        q[1] = make_float4(c[0], c[1], d[0], d[1]);
    } else {
        *reinterpret_cast<u32x4_t*>(p) = DT == MFA_DTYPE_BF16 ? kv4_bf16x8(codes, s) : kv4_f16x8(codes, s);
    }
}

template <int DT>
__global__ void __launch_bounds__(kAThreads) mfa_kv4_append_kernel(AArgs a) {
    __shared__ int32_t cu_s[kASeqs + 1];
    const int tid = threadIdx.x;
    if (a.B <= kASeqs) {
        for (int i = tid; i <= a.B; i += kAThreads) cu_s[i] = a.cu[i];
        __syncthreads();
    }
    const int which = blockIdx.y;
    const int64_t at = (int64_t)blockIdx.x * kAThreads + tid;
    if (at >= a.chunks) return;  // (whole groups of four lanes: a row has a multiple of four chunks)
    const uint32_t cc = (uint32_t)at;
    const int t = (int)quotient(cc, a.by_row);
    const uint32_t rest = cc - t * a.by_row.d;
    const int h = (int)quotient(rest, a.by_head), d = 8 * (int)(rest - h * a.by_head.d);
    float x[8];
    constexpr int ES = DT == MFA_DTYPE_F32 ? 4 : 2;
    load8<DT>(a.x[which] + (t * a.ts[which] + h * a.hs[which] + d) * ES, x);

    // the group's largest magnitude (as bits: an infinity or NaN is the largest)
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = max(mx, __float_as_uint(x[i]) & 0x7fffffffu);
    mx = max(mx, (uint32_t)__shfl_xor((int)mx, 1));
    mx = max(mx, (uint32_t)__shfl_xor((int)mx, 2));
    const bool bad = mx >= 0x7f800000u;
    // 2^e <= max < 2^(e+1): scale 2^(e-2), or 2^(e-1) for a mantissa above 1.75
    // (bytes below 0 are 0: everything then rounds against 2^-127)
    const int byte = max((int)(mx >> 23) - 2 + ((mx & 0x7fffffu) > 0x600000u ? 1 : 0), 0);
    const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);
    uint32_t codes = 0;
    if (!bad) {
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0] * inv, x[1] * inv, 1.f, 0);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2] * inv, x[3] * inv, 1.f, 1);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4] * inv, x[5] * inv, 1.f, 2);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6] * inv, x[7] * inv, 1.f, 3);
    }
    const uint32_t scale = bad ? 255u : (uint32_t)byte;
    if (a.val[which]) store_values8<DT>(a.val[which] + ((int64_t)t * a.H * a.D + h * a.D + d) * ES, codes, scale);

    // the token's sequence: the last whose tokens begin at or before it
    const int32_t* cu = a.B <= kASeqs ? cu_s : a.cu;
    int lo = 0, hi = a.B;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    if (lo >= a.B || cu[lo] > t) return;  // (a token of no sequence)
    const int64_t pos = (int64_t)a.lens[lo] + t - cu[lo];
    if (pos < 0 || pos >= (int64_t)a.max_pages * a.page) return;
    const int idx = (int)quotient((uint32_t)pos, a.by_page), row = (int)pos - idx * a.page;
    const int id = a.bt[lo * a.bt_b + idx];
    if ((uint32_t)id >= (uint32_t)a.npages) return;
    const Kv4Pool& p = a.pool[which];
    *reinterpret_cast<uint32_t*>(p.codes + id * p.cp + row * p.cr + h * p.ch + d / 2) = codes;
    if ((d & 31) == 0) p.scales[id * p.sp + row * p.sr + h * p.sh + d / 32] = (uint8_t)scale;
}

int aerr(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(mfa_error_buffer(), 512, fmt, ap);
    va_end(ap);
    return code;
}

}  // namespace

int mfa_kv4_check_cache(const mfa_kv4_cache* c, int batch, int head_dim, const char* who) {
    if (c->page_block_size <= 0 || c->page_block_size % 64)
        return aerr(MFA_ERR_INVALID, "%s: page_block_size %d must be a positive multiple of 64", who, c->page_block_size);
    if (c->num_pages < 0 || c->max_pages < 0 || c->block_table_batch_stride < 0)
        return aerr(MFA_ERR_INVALID, "%s: negative num_pages, max_pages or block_table stride", who);
    if ((int64_t)c->max_pages * c->page_block_size > 0x7fffffffLL)
        return aerr(MFA_ERR_INVALID, "%s: a block table names at most 2^31 - 1 rows", who);
    // (no sequences: a table of no rows, which may have no memory)
    if (batch > 0 && c->max_pages > 0 && (!c->block_table || (reinterpret_cast<uintptr_t>(c->block_table) & 3)))
        return aerr(MFA_ERR_INVALID, "%s: block_table is required", who);
    const mfa_kv4_pool* pools[2] = {&c->k, &c->v};
    for (const mfa_kv4_pool* p : pools) {
        if (c->num_pages == 0) break;
        if (!p->codes || !p->scales || (reinterpret_cast<uintptr_t>(p->codes) & 15))
            return aerr(MFA_ERR_INVALID, "%s: codes (16-byte aligned) and scales are required", who);
        if (p->code_page_stride % 16 || p->code_row_stride % 16 || p->code_head_stride % 16)
            return aerr(MFA_ERR_INVALID, "%s: code strides must be multiples of 16 bytes", who);
        if (p->code_row_stride < 0 || p->code_head_stride < 0 || p->scale_row_stride < 0 || p->scale_head_stride < 0)
            return aerr(MFA_ERR_INVALID, "%s: row and head strides must be >= 0", who);
        // (a page's rows are addressed with 32-bit byte offsets)
        if (c->page_block_size * p->code_row_stride + head_dim >= (1LL << 31) ||
            c->page_block_size * p->scale_row_stride + head_dim >= (1LL << 31))
            return aerr(MFA_ERR_INVALID, "%s: the rows of a page must span less than 2 GiB", who);
    }
    return MFA_OK;
}

extern "C" {

int mfa_kv4_append_params_size(void) { return (int)sizeof(mfa_kv4_append_params); }

int mfa_kv4_append(const mfa_kv4_append_params* p, void* stream) {
    mfa_error_buffer()[0] = 0;
    if (!p) return aerr(MFA_ERR_INVALID, "mfa_kv4_append: params is NULL");
    if (p->dtype != MFA_DTYPE_F16 && p->dtype != MFA_DTYPE_BF16 && p->dtype != MFA_DTYPE_F32)
        return aerr(MFA_ERR_INVALID, "mfa_kv4_append: unknown dtype %d", p->dtype);
    if (p->batch < 0 || p->total < 0 || p->heads_kv < 0) return aerr(MFA_ERR_INVALID, "mfa_kv4_append: negative size");
    if (p->head_dim <= 0 || p->head_dim % kKv4Group || p->head_dim > MFA_MAX_HEAD_DIM)
        return aerr(MFA_ERR_UNSUPPORTED, "mfa_kv4_append: head_dim %d is not a multiple of %d up to %d", p->head_dim, kKv4Group,
                    MFA_MAX_HEAD_DIM);
    const int rc = mfa_kv4_check_cache(&p->cache, p->batch, p->head_dim, "mfa_kv4_append");
    if (rc != MFA_OK) return rc;
    // (tokens of no sequence have values too)
    if (p->total == 0 || p->heads_kv == 0 || (p->batch == 0 && !p->k_values && !p->v_values)) return MFA_OK;
    auto bad = [](const void* x, uintptr_t al) { return !x || (reinterpret_cast<uintptr_t>(x) & (al - 1)); };
    if (bad(p->k, 16) || bad(p->v, 16)) return aerr(MFA_ERR_INVALID, "mfa_kv4_append: k and v must be 16-byte aligned");
    const int al = p->dtype == MFA_DTYPE_F32 ? 4 : 8;
    if (p->k_token_stride % al || p->k_head_stride % al || p->v_token_stride % al || p->v_head_stride % al)
        return aerr(MFA_ERR_INVALID, "mfa_kv4_append: k and v strides must be multiples of %d elements", al);
    if ((p->k_values == nullptr) != (p->v_values == nullptr) || (p->k_values && (bad(p->k_values, 16) || bad(p->v_values, 16))))
        return aerr(MFA_ERR_INVALID, "mfa_kv4_append: k_values and v_values must both be NULL or 16-byte aligned");
    if (bad(p->cu_seqlens, 4) || (p->batch > 0 && bad(p->cache_seqlens, 4)))
        return aerr(MFA_ERR_INVALID, "mfa_kv4_append: cu_seqlens and cache_seqlens are required");
    const int64_t per_token = (int64_t)p->heads_kv * (p->head_dim / 8);
    if (per_token > 0x7fffffffLL || per_token * p->total > 0x7fffffffLL)
        return aerr(MFA_ERR_INVALID, "mfa_kv4_append: problem too large");
    AArgs a;
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
    a.B = p->batch; a.T = p->total; a.H = p->heads_kv; a.D = p->head_dim;
    a.max_pages = p->cache.max_pages; a.npages = p->cache.num_pages; a.page = p->cache.page_block_size;
    a.by_page = fast_div(a.page);
    a.by_row = fast_div((uint32_t)per_token);
    a.by_head = fast_div(p->head_dim / 8);
    a.chunks = (int32_t)(per_token * p->total);
    const auto fn = p->dtype == MFA_DTYPE_F32    ? mfa_kv4_append_kernel<MFA_DTYPE_F32>
                    : p->dtype == MFA_DTYPE_BF16 ? mfa_kv4_append_kernel<MFA_DTYPE_BF16>
                                                 : mfa_kv4_append_kernel<MFA_DTYPE_F16>;
    hipLaunchKernelGGL(fn, dim3((unsigned)((a.chunks + (int64_t)kAThreads - 1) / kAThreads), 2), dim3(kAThreads), 0,
                       static_cast<hipStream_t>(stream), a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return aerr(MFA_ERR_LAUNCH, "mfa_kv4_append: launch failed: %s", hipGetErrorString(e));
    return MFA_OK;
}

}  // extern "C"
