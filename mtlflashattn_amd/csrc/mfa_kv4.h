// mfa_kv4.h -- the 4-bit K/V cache as its kernels see it (mfa_kv4.hip,
// mfa_kv4_attend.hip): element format, pool addressing and argument checks.
//
// A cached row of one head is D/2 code bytes and D/32 scale bytes: 32
// consecutive elements share the power of two 2^(s - 127) of their scale byte s
// (255: NaN) and each is a 4-bit float, sign, two exponent bits and one mantissa
// bit (0, 0.5, 1, 1.5, 2, 3, 4, 6), element 2i in the low half of byte i.  The
// gfx950 conversions v_cvt_scalef32_pk_*_fp4 read and write this form, taking
// the scale from the exponent bits of a float, so the byte shifted to bits 23..30
// is the scale operand as it stands (0: 2^-127, 255: NaN).
#pragma once

#include "mfa.h"
#include "mfa_common.h"

// Checks of the pointers, strides and sizes of the cache of `batch` sequences:
// MFA_OK, or an error code with the message set (mfa_kv4.hip).
__attribute__((visibility("hidden"))) int mfa_kv4_check_cache(const mfa_kv4_cache* cache, int batch, int head_dim,
                                                              const char* who);

namespace {

constexpr int kKv4Group = 32;  // elements per scale

typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 k4_bf16x2_t;
typedef __attribute__((__vector_size__(2 * sizeof(_Float16)))) _Float16 k4_f16x2_t;

// One of K and V: [num_pages, page, heads, ...] code and scale bytes.
struct Kv4Pool {
    uint8_t* codes;
    uint8_t* scales;
    int64_t cp, cr, ch;  // bytes between pages, rows and heads of the codes
    int64_t sp, sr, sh;  // ... and of the scales
};

inline Kv4Pool kv4_pool(const mfa_kv4_pool& p) {
    return Kv4Pool{p.codes, p.scales, p.code_page_stride, p.code_row_stride, p.code_head_stride,
                   p.scale_page_stride, p.scale_row_stride, p.scale_head_stride};
}

__device__ __forceinline__ float kv4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight codes (a dword) as eight bf16: exact, a code has two significant bits.
__device__ __forceinline__ u32x4_t kv4_bf16x8(uint32_t w, float s) {
    u32x4_t r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
    return r;
}

// ... as eight fp16, the operand type of fp16 queries in the 128-column kernel (bf16
// operands, exact, would need the queries as two terms and twice the products):
// saturating, as 65504 may be held as 4 * 2^14, one step above fp16's range (IEEE
// minimum and maximum: NaN stays NaN), and rounded where 2^-24 is above half a unit of
// the scale, below 2^-23.
__device__ __forceinline__ u32x4_t kv4_f16x8(uint32_t w, float s) {
    const k4_f16x2_t top = {(_Float16)65504.f, (_Float16)65504.f};
    auto sat = [&](k4_f16x2_t x) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_minimum(__builtin_elementwise_maximum(x, -top), top));
    };
    u32x4_t r;
    r[0] = sat(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0));
    r[1] = sat(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1));
    r[2] = sat(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2));
    r[3] = sat(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3));
    return r;
}

// Eight codes of V of a group whose elements may pass the range of fp32 and bf16
// (scale bytes 253 and 254), saturated to 1.5 * 2^127: magnitudes above 3 * 2^126
// (code 5) or 1.5 * 2^127 (code 3) become those.  An infinite element would reach
// the rows that mask its key, as 0 * inf.
__device__ __forceinline__ bool kv4_beyond(uint32_t byte) { return byte == 253 || byte == 254; }
__device__ __forceinline__ uint32_t kv4_saturate8(uint32_t w, uint32_t byte) {
    const uint32_t top = byte == 253 ? 5 : 3;
    // (bit 3 of a half byte that holds magnitude + 7 - top: magnitude > top)
    const uint32_t over = ((w & 0x77777777u) + (7 - top) * 0x11111111u) >> 3 & 0x11111111u;
    return (w & ~(over * 7)) | over * top;
}

// j / d for 0 <= j < 2^31 as umulhi(j, m) >> s (round-up method: l = ceil(log2
// d), m = ceil(2^(31+l) / d) < 2^32, s = l - 1; d = 1 is m = 0, s = 0 and is
// taken by the caller's quotient()).
struct FastDiv {
    uint32_t d, m;
    int32_t s;
};
inline FastDiv fast_div(uint32_t d) {
    FastDiv f{d, 0, 0};
    if (d <= 1) return f;
    int l = 0;
    while ((1ull << l) < d) ++l;
    f.m = (uint32_t)((((unsigned __int128)1 << (31 + l)) + d - 1) / d);
    f.s = l - 1;
    return f;
}
__device__ __forceinline__ uint32_t quotient(uint32_t j, const FastDiv& f) {
    return f.d <= 1 ? j : __umulhi(j, f.m) >> f.s;
}

// inclusive prefix sum over the wavefront: shifts inside rows of 16 lanes, then the
// last lanes of rows and of halves to what is behind them
__device__ __forceinline__ int scan64(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 to rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 to rows 2 and 3
    return x;
}

}  // namespace
