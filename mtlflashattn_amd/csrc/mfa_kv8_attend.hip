// mfa_kv8_attend.hip -- attention over a paged 8-bit K/V cache (mfa_kv8_fwd in
// include/mfa.h): the 8-bit format of the kernel for sequences of at most 32 columns
// (mfa_kv_rows.h) and the C entry point.  Dealing, merge and plan are those of the
// 4-bit cache (mfa_kv4_attend.hip).
//
// Bound by the stream of the cache (256 bytes per key and head at head dim 128) where
// batches are large, by latency where they are small.  64 sequences of 512 to 16384 keys,
// Hq=32 Hkv=8 D=128 bf16: 181 us with the merge, 6.1 TB/s; one sequence of 3001: 8.2 us and
// 4.2 of the merge.  At head dim 128 fp16 queries, two terms, do not fit the registers (15 of
// them spilled with 16 columns, 17 with 32): 64 single rows over 8192 keys 205 us, 179 in bf16.
#include <math.h>
#include <stdint.h>

#include "mfa_kv8_block.h"

namespace {

// A 32-key block: K (mfa_kv8_block.h), and V in 16-element chunks with its scale.
template <int DP>
struct Block8 : KeyBlock8<DP> {
    typedef KeyBlock8<DP> Keys;
    static constexpr int D = DP;
    static constexpr int bytes(int x) { return x & 1 ? 1 : DP; }
    static constexpr int rows_per(int x) { return x & 1 ? kKv8Block : 1; }
    static constexpr int VG = DP / 32;   // V chunks per lane
    static constexpr int CPR = DP / 16;  // V chunks per row
    u32x4_t v[VG];
    uint8_t vs;

    struct Offsets : Keys::Offsets {
        uint32_t voff[VG];
        int vrow[VG], vchunk[VG];
        __device__ __forceinline__ void init(K4Const& a, int lane) {
            Keys::Offsets::init(a, lane);
#pragma unroll
            for (int i = 0; i < VG; ++i) {
                const int cc = 64 * i + lane;
                vrow[i] = cc / CPR;
                vchunk[i] = cc - vrow[i] * CPR;
                voff[i] = (uint32_t)(vrow[i] * (int)a.v.cr + vchunk[i] * 16);
            }
        }
    };
    __device__ __forceinline__ void load(const __amdgpu_buffer_rsrc_t (&rs)[4], const Offsets& off, uint32_t kr, uint32_t ksr,
                                         uint32_t vr, uint32_t vsr) {
        Keys::load(rs, off, kr, ksr);
#pragma unroll
        for (int i = 0; i < VG; ++i) v[i] = __builtin_amdgcn_raw_buffer_load_b128(rs[2], off.voff[i] + vr, 0, kOnce4);
        vs = __builtin_amdgcn_raw_buffer_load_b8(rs[3], vsr, 0, 0);
    }

    // NaN elements of a block's V: bit e of half i % 2 of bits[i / 2] is element e of the
    // lane's chunk i
    struct Nans {
        uint32_t bits[(VG + 1) / 2];
        uint64_t lanes[VG];  // lanes that have any
        template <int NT>
        __device__ __forceinline__ void add(f32x4_t (&o)[NT][DP / 16], int j, const int (&lo)[NT], const int (&hi)[NT],
                                            int grp) const {
#pragma unroll
            for (int i = 0; i < VG; ++i) {
                for (uint64_t x = lanes[i]; x; x &= x - 1) {
                    const int l = __builtin_ctzll(x), cc = 64 * i + l, row = cc / CPR;
                    const uint32_t mine = (uint32_t)__builtin_amdgcn_readlane((int)bits[i / 2], l) >> (16 * (i % 2) + 4 * grp);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const bool sees = j + row >= lo[t] && j + row <= hi[t];
#pragma unroll
                        for (int d = 0; d < DP / 16; ++d) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float y = sees && d == cc - row * CPR && (mine >> e & 1) ? __builtin_nanf("") : 0.f;
                                pin(y);  // (no indexing of o by the chunk)
                                o[t][d][e] += y;
                            }
                        }
                    }
                }
            }
        }
    };
    template <class Swz>
    __device__ __forceinline__ void stage_v(uint16_t* vt, Swz&& vswz, const Offsets& off, bool masked, int, Nans& nans) {
#pragma unroll
        for (int i = 0; i < (VG + 1) / 2; ++i) nans.bits[i] = 0;
#pragma unroll
        for (int i = 0; i < VG; ++i) nans.lanes[i] = 0;
        if (masked) {  // (wavefront-uniform)
#pragma unroll
            for (int i = 0; i < VG; ++i) {
                uint32_t bits = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t n = kv8_nans(v[i][e]);
                    bits |= kv8_nan_bits(n) << (4 * e);
                    v[i][e] = kv8_without(v[i][e], n);
                }
                nans.bits[i / 2] |= bits << (16 * (i % 2));
                nans.lanes[i] = __ballot(bits != 0);
            }
        }
        const float s = kv8_scale(vs);
#pragma unroll
        for (int i = 0; i < VG; ++i) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
                *reinterpret_cast<u32x4_t*>(vt + off.vrow[i] * DP + (((2 * off.vchunk[i] + e) ^ vswz(off.vrow[i])) << 3)) =
                    kv8_bf16x8(v[i][2 * e], v[i][2 * e + 1], s);
        }
    }
};

typedef void (*k8_fn)(K4Args);
template <int DP>
void* rows8(int cols, bool bf16) {
    return cols == 16 ? (void*)(bf16 ? (k8_fn)mfa_kv_rows_kernel<Block8<DP>, 1, true> : (k8_fn)mfa_kv_rows_kernel<Block8<DP>, 1, false>)
                      : (void*)(bf16 ? (k8_fn)mfa_kv_rows_kernel<Block8<DP>, 2, true> : (k8_fn)mfa_kv_rows_kernel<Block8<DP>, 2, false>);
}
void* rows_kernel8(int dp, int cols, bool bf16) {
    switch (dp) {
        case 32: return rows8<32>(cols, bf16);
        case 64: return rows8<64>(cols, bf16);
        case 96: return rows8<96>(cols, bf16);
        default: return rows8<128>(cols, bf16);
    }
}
// (varlen calls of 17 to 32 columns per sequence: 64 sequences of 5 rows over 8192 keys, Hq=32
// Hkv=8 D=128 bf16: 311 us by the 128-column kernel, 209 by the kernel of 32)
const MfaKvFormat kFormat8 = {"mfa_kv8_fwd", {wgs4(1), wgs4(2)}, 2, kKv8LeastScale, true, rows_kernel8, mfa_kv8_tile_kernel_of};

}  // namespace

extern "C" {

int mfa_kv8_fwd_params_size(void) { return (int)sizeof(mfa_kv8_fwd_params); }

int64_t mfa_kv8_fwd_workspace_bytes(const mfa_kv8_fwd_params* p) { return mfa_kv_fwd_workspace_bytes(p, kFormat8); }

int mfa_kv8_fwd(const mfa_kv8_fwd_params* p, void* workspace, int64_t workspace_bytes, void* stream) {
    return mfa_kv_fwd(p, kFormat8, workspace, workspace_bytes, stream);
}

}  // extern "C"
