// mfa_kv8_block.h -- a 32-key block of K of the 8-bit cache in registers, as the kernels
// for few columns take it (mfa_kv8_attend.hip, mfa_kv8_weights.hip).
#pragma once

#include "mfa_kv8.h"
#include "mfa_kv_rows.h"

namespace {

// The codes of two 16-key tiles, and their scale, which the whole block shares (32 keys
// from a multiple of 32 on lie in one block of 64 rows).  Loads are non-temporal: the kernels
// for few columns read a byte of the cache once a call.  (The key weights of many columns
// read a block again for every 128 of them where a workgroup has more blocks than
// wavefronts.)
//
// The four lanes of a key's row take 16 adjacent bytes each of 64, so that a load
// covers whole 64-byte pieces: piece p of a row gives lane group g elements 64 p + 16 g
// .. + 15, two steps of the product; the 32 elements left of a row of 32 or 96 give it
// 8, one step.
template <int DP>
struct KeyBlock8 {
    static constexpr int P = DP / 64;           // 16-byte pieces per lane and row
    static constexpr bool HALF = DP % 64 != 0;  // and one of 8
    u32x4_t k[2][P > 0 ? P : 1];
    u32x2_t kh[2];
    uint8_t ks;  // (a byte until it is used: widening it would wait for the load)

    struct Offsets {
        uint32_t koff[2], khoff[2];
        __device__ __forceinline__ void init(K4Const& a, int lane) {
            const int l16 = lane & 15, grp = lane >> 4;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const int row = (16 * kk + l16) * (int)a.k.cr;
                koff[kk] = (uint32_t)(row + 16 * grp);
                khoff[kk] = (uint32_t)(row + 64 * P + 8 * grp);
            }
        }
    };
    // kr, ksr: byte offsets of the block's first row and of its scale
    __device__ __forceinline__ void load(const __amdgpu_buffer_rsrc_t (&rs)[4], const Offsets& off, uint32_t kr, uint32_t ksr) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
            for (int p = 0; p < P; ++p) k[kk][p] = __builtin_amdgcn_raw_buffer_load_b128(rs[0], off.koff[kk] + 64 * p + kr, 0, kOnce4);
            if constexpr (HALF) kh[kk] = __builtin_amdgcn_raw_buffer_load_b64(rs[0], off.khoff[kk] + kr, 0, kOnce4);
        }
        ks = __builtin_amdgcn_raw_buffer_load_b8(rs[1], ksr, 0, 0);
    }

    // step s of lane group grp: eight elements from here on
    static __device__ __forceinline__ int element(int grp, int s) {
        return s < 2 * P ? 64 * (s >> 1) + 16 * grp + 8 * (s & 1) : 64 * P + 8 * grp;
    }
    template <class Op = bf16x8_t>
    __device__ __forceinline__ Op k_operand(int kk, int s, int) const {
        return s < 2 * P ? kv8_operand<Op>(k[kk][s >> 1][2 * (s & 1)], k[kk][s >> 1][2 * (s & 1) + 1]) : kv8_operand<Op>(kh[kk][0], kh[kk][1]);
    }
    // what the scores of the block are still to be multiplied by
    __device__ __forceinline__ float k_scale() const { return kv8_k_scale(ks); }
};

}  // namespace
