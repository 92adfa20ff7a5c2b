// mfa_kv8_tile.hip -- the 8-bit format of the 128-column kernel (mfa_kv_tile.h).
//
// A thread takes 16-element chunks of K and of V of a block, 16 conversions for every
// 32 elements as in the 4-bit format; K's codes stand in the tile without their scale,
// which multiplies the scores (exact for fp16 queries too).  1024 rows over 16384 keys,
// Hq=32 Hkv=8 D=128 bf16: 300 to 309 us with the merge, 860 to 890 TFLOP/s; bound by no one
// unit (matrix pipe 41 % busy), two wavefronts per SIMD waiting for each other's steps.  At
// head dim 128 it spills 20 to 24 bytes per lane, 116 to 132 with soft-cap or ALiBi.
#include <math.h>
#include <stdint.h>

#include "mfa_kv8.h"
#include "mfa_kv_tile.h"

namespace {

template <int DP, bool IS_BF16>
struct Stage8 {
    static constexpr int D = DP;
    static constexpr int bytes(int x) { return x & 1 ? 1 : DP; }
    static constexpr int rows_per(int x) { return x & 1 ? kKv8Block : 1; }
    static_assert(kTK == kKv8Block, "a block of keys has one scale");
    static constexpr bool kBf16 = IS_BF16;
    typedef TileShape<DP> Shape;
    static constexpr int CPR = DP / 16, CHUNKS = kTK * CPR;      // chunks of a row, and of K or of V
    static constexpr int NG = 2 * CHUNKS / kThreads4;            // this thread's, K's first
    static_assert(2 * CHUNKS % kThreads4 == 0 && CHUNKS % 64 == 0, "whole wavefronts of chunks");
    bool gv[NG];  // V (wavefront-uniform)
    int glds[NG], gsw[NG];
    uint32_t goff[NG];
    u32x4_t gc[NG];
    uint8_t ks, vs;  // the loaded block's scales (bytes until they are used: widening them at the load would wait for it)
    float sk;

    __device__ __forceinline__ void init(K4Const& a, int tid) {
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int g = tid + kThreads4 * i;
            gv[i] = __builtin_amdgcn_readfirstlane(g) >= CHUNKS;
            const int u = g - (gv[i] ? CHUNKS : 0);
            const int row = u / CPR, c = u - row * CPR;
            goff[i] = (uint32_t)(row * (int)(gv[i] ? a.v.cr : a.k.cr) + c * 16);
            // (16-byte half e of the chunk's values: + 8 (e ^ gsw))
            const int slot = (2 * c) ^ vswz4<DP>(row);
            glds[i] = gv[i] ? Shape::K_ELEMS + row * Shape::VST + 8 * (slot & ~1) : row * Shape::KST + 16 * c;
            gsw[i] = gv[i] ? slot & 1 : 0;
        }
        sk = 0.f;
    }
    __device__ __forceinline__ void load(const Pages4<Stage8>& pg, int row) {
#pragma unroll
        for (int i = 0; i < NG; ++i)
            gc[i] = __builtin_amdgcn_raw_buffer_load_b128(gv[i] ? pg.rs[2] : pg.rs[0], goff[i] + (uint32_t)row * (uint32_t)(gv[i] ? pg.rstride[2] : pg.rstride[0]), 0, 0);
        const int srow = row / kKv8Block;
        ks = __builtin_amdgcn_raw_buffer_load_b8(pg.rs[1], (uint32_t)(srow * pg.rstride[1]), 0, 0);
        vs = __builtin_amdgcn_raw_buffer_load_b8(pg.rs[3], (uint32_t)(srow * pg.rstride[3]), 0, 0);
    }

    // NaN elements of a block's V: a bit for each chunk that has any, and its elements
    struct Nans {
        uint64_t chunks[CHUNKS / 64];
        uint16_t bits[CHUNKS];
    };
    __device__ __forceinline__ void write(uint16_t* tile, Nans& nans, bool part, int half_, int tid) {
        if (half_ == 0) sk = kv8_k_scale(ks);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            if (i % 2 != half_) continue;
            if (__builtin_expect(part & gv[i], 0)) {  // (wavefront-uniform)
                uint32_t bits = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t n = kv8_nans(gc[i][e]);
                    bits |= kv8_nan_bits(n) << (4 * e);
                    gc[i][e] = kv8_without(gc[i][e], n);
                }
                const int u = tid + kThreads4 * i - CHUNKS;
                nans.bits[u] = (uint16_t)bits;
                nans.chunks[u >> 6] = __ballot(bits != 0);
            }
            uint16_t* p = tile + glds[i];
            const float s = gv[i] ? kv8_scale(vs) : 1.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                u32x4_t x = IS_BF16 ? kv8_bf16x8(gc[i][2 * e], gc[i][2 * e + 1], s) : kv8_f16x8(gc[i][2 * e], gc[i][2 * e + 1], s);
                if constexpr (!IS_BF16) {
                    if (__builtin_expect(gv[i] && kv8_beyond_f16(vs), 0)) x = kv8_saturate_f16(x);
                }
                *reinterpret_cast<u32x4_t*>(p + 8 * (e ^ gsw[i])) = x;
            }
        }
    }
    // what the scores of the block that was written last are still to be multiplied by
    __device__ __forceinline__ float k_scale() const { return sk; }

    // a lane holds elements 32 db + 8 g + 4 half + 0..3 (g < 4) of its column
    __device__ __forceinline__ void add_nans(const Nans& nans, f32x16_t (&o)[DP / 32], int j, int lo, int hi, int half) const {
        for (int i = 0; i < CHUNKS / 64; ++i) {
            for (uint64_t x = nans.chunks[i]; x; x &= x - 1) {
                const int u = __builtin_amdgcn_readfirstlane(64 * i + __builtin_ctzll(x)), row = u / CPR;
                const uint32_t bits = (uint32_t)nans.bits[u] >> (4 * half);
                const bool sees = j + row >= lo && j + row <= hi;
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const bool here = 2 * db + (r >> 3) == u - row * CPR;
                        float y = sees && here && (bits >> (8 * (r >> 2 & 1) + (r & 3)) & 1) ? __builtin_nanf("") : 0.f;
                        pin(y);  // (no indexing of o by the chunk)
                        o[db][r] += y;
                    }
            }
        }
    }
};

template <class Stage>
void* tile_of(bool bias, bool lse) {
    typedef void (*fn)(K4Args);
    return (void*)(bias ? (lse ? (fn)mfa_kv_tile_kernel<Stage, true, true> : (fn)mfa_kv_tile_kernel<Stage, true, false>)
                        : (lse ? (fn)mfa_kv_tile_kernel<Stage, false, true> : (fn)mfa_kv_tile_kernel<Stage, false, false>));
}
template <int DP>
void* tile_of(bool bf16, bool bias, bool lse) {
    return bf16 ? tile_of<Stage8<DP, true>>(bias, lse) : tile_of<Stage8<DP, false>>(bias, lse);
}

}  // namespace

void* mfa_kv8_tile_kernel_of(int dp, bool bf16, bool bias, bool lse) {
    switch (dp) {
        case 32: return tile_of<32>(bf16, bias, lse);
        case 64: return tile_of<64>(bf16, bias, lse);
        case 96: return tile_of<96>(bf16, bias, lse);
        default: return tile_of<128>(bf16, bias, lse);
    }
}
