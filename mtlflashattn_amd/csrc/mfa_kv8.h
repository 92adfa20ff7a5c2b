// mfa_kv8.h -- the 8-bit K/V cache as its kernels see it (mfa_kv8.hip,
// mfa_kv8_attend.hip, mfa_kv8_tile.hip, mfa_kv8_weights.hip, mfa_kv8_evict.hip):
// element format and conversions.
//
// A cached row of one head is D code bytes, e4m3 floats (sign, four exponent bits
// with bias 7, three mantissa bits; 0x7f and 0xff are NaN, the largest is 448, there
// are no infinities); the 64 rows of a block (rows 64 i .. 64 i + 63 of a page) and a
// head share the power of two 2^(s - 127) of one scale byte s.  The byte shifted to
// bits 23..30 is the scale as a float (0: 0).  Codes are exact in bf16 and fp16, and
// times the scale in bf16, so kernels multiply scores by K's scale (one number per
// 64 keys) and turn V into values with its scale in the conversion
// (v_cvt_scalef32_pk_*_fp8).
#pragma once

#include "mfa_kv4.h"

namespace {

constexpr int kKv8Block = MFA_KV8_BLOCK;  // rows per scale

__device__ __forceinline__ float kv8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// K's scale as a factor of scores in log2 units before their mask is applied: that of byte 1
// for byte 0 (which a page outside the pool reads as), as a factor of 0 times a masked
// score, -inf, would be NaN.  Softmax scales up to 2^-24, whose product with it is 0 in
// fp32, take the path that masks behind the scaling.
constexpr float kKv8LeastScale = 0x1p-24f;
__device__ __forceinline__ float kv8_k_scale(uint32_t byte) { return kv8_scale(max(byte, 1u)); }

// Eight codes (two dwords) as eight bf16: exact while code * s is a normal bf16.
__device__ __forceinline__ u32x4_t kv8_bf16x8(uint32_t w0, uint32_t w1, float s) {
    u32x4_t r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, true));
    return r;
}

// ... as eight fp16: exact while code * s keeps to fp16's range and steps.
__device__ __forceinline__ u32x4_t kv8_f16x8(uint32_t w0, uint32_t w1, float s) {
    u32x4_t r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, s, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, s, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, s, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, s, true));
    return r;
}
// Eight codes as they are, without their scale: exact in either type.
template <class Op>
__device__ __forceinline__ Op kv8_operand(uint32_t w0, uint32_t w1) {
    if constexpr (std::is_same<Op, f16x8_t>::value) return __builtin_bit_cast(Op, kv8_f16x8(w0, w1, 1.f));
    else return __builtin_bit_cast(Op, kv8_bf16x8(w0, w1, 1.f));
}
// Scales from 2^8 on, whose largest codes pass fp16's range (448 * 2^8 > 65504).
__device__ __forceinline__ bool kv8_beyond_f16(uint32_t byte) { return byte > 127 + 7; }
// Eight values saturated to +/-65504 (IEEE minimum and maximum: NaN stays NaN): an
// infinite element would reach the rows that mask its key, as 0 * inf.
__device__ __forceinline__ u32x4_t kv8_saturate_f16(u32x4_t x) {
    const k4_f16x2_t top = {(_Float16)65504.f, (_Float16)65504.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t y = x[i];
        x[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_minimum(
                                                __builtin_elementwise_maximum(__builtin_bit_cast(k4_f16x2_t, y), -top), top));
    }
    return x;
}

// The NaN codes of a dword: bit 7 of each such byte.
__device__ __forceinline__ uint32_t kv8_nans(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// ... as bits 0..3, and the dword with zeros in their place.
__device__ __forceinline__ uint32_t kv8_nan_bits(uint32_t n) { return (n >> 7 & 1) | (n >> 14 & 2) | (n >> 21 & 4) | (n >> 28 & 8); }
__device__ __forceinline__ uint32_t kv8_without(uint32_t w, uint32_t n) { return w & ~((n >> 7) * 255u); }

// The smallest byte from 1 on with max <= 448 * 2^(byte - 127), for the bits of a
// finite max >= 0: 2^e <= max < 2^(e+1) takes 2^(e-8), or 2^(e-7) for a mantissa
// above 1.75.
__device__ __forceinline__ uint32_t kv8_byte_of(uint32_t max_bits) {
    const int b = (int)(max_bits >> 23) - 8 + ((max_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)max(b, 1);
}
// The largest value to write under a byte: 448, or 240 under the largest byte there is
// (scale 2^120), where 256 would stand for 2^128.
__device__ __forceinline__ float kv8_top(uint32_t byte) { return byte < 247 ? 448.f : 240.f; }
// 2^(127 - byte), for bytes 1 .. 253
__device__ __forceinline__ float kv8_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Unsigned maximum of a wavefront, in lane 63
__device__ __forceinline__ uint32_t max64(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false));  // row_shr:1, 2, 4, 8
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false));  // row_bcast:15 to rows 1 and 3
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false));  // row_bcast:31 to rows 2 and 3
    return x;
}

// Four floats, at most 448 in magnitude or NaN, as four codes: the nearest values,
// ties to the even code.
__device__ __forceinline__ uint32_t kv8_round4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// Four codes times s, a power of two.
__device__ __forceinline__ void kv8_values4(uint32_t w, float s, float (&x)[4]) {
    typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f2;
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = a[0] * s;
    x[1] = a[1] * s;
    x[2] = b[0] * s;
    x[3] = b[1] * s;
}

}  // namespace
