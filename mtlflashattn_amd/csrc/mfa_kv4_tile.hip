// mfa_kv4_tile.hip -- the 4-bit format of the 128-column kernel (mfa_kv_tile.h).
//
// A thread takes one 32-element scale group of K and of V of a block: 16
// conversions, exact in bf16 and saturating in fp16.  1024 rows over 16384 keys,
// Hq=32 Hkv=8 D=128 bf16, take 298 to 304 us with the merge in a timed loop (876 to
// 893 TFLOP/s), the kernel alone 324 to 340 in short traces over machines (side by
// side on one: 316 to 324, and 329 to 334 with one tile, converted between two
// barriers); over 8192 keys 167 us, with soft-cap 212, with ALiBi 188.  Bound by no one
// unit: the matrix pipe is busy 40 % of the time, LDS bank conflicts take 10 % of it.
// In the form with one tile (332 us), with one part taken out at a time, the products
// of the scores were worth 64 us, those of the values 37, the softmax 43, the
// conversion 50 and most reads of K 17.
#include <math.h>
#include <stdint.h>

#include "mfa_kv_tile.h"

namespace {

template <int DP, bool IS_BF16>
struct Stage4 {
    static constexpr int D = DP;
    // codes (even x) and scales of a row
    static constexpr int bytes(int x) { return x & 1 ? DP / 32 : DP / 2; }
    static constexpr int rows_per(int) { return 1; }
    static constexpr bool kBf16 = IS_BF16;
    typedef TileShape<DP> Shape;
    static constexpr int GPR = DP / 32;
    static constexpr int GROUPS = 2 * kTK * GPR;  // scale groups of a block, K's then V's
    static constexpr int NG = (GROUPS + kThreads4 - 1) / kThreads4;
    // this thread's groups: wavefront-uniform choice of K or V
    bool gv[NG];
    int glds[NG], gsw[NG];
    uint32_t goff[NG], gsoff[NG];
    u32x4_t gc[NG];
    uint8_t gs[NG];  // (bytes until they are used: widening them at the load would wait for it)

    __device__ __forceinline__ void init(K4Const& a, int tid) {
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int g = tid + kThreads4 * i;
            gv[i] = __builtin_amdgcn_readfirstlane(g) >= kTK * GPR;
            const int u = g - (gv[i] ? kTK * GPR : 0);
            const int row = u / GPR, grp = u - row * GPR;
            const bool in = g < GROUPS;
            goff[i] = in ? (uint32_t)(row * (int)(gv[i] ? a.v.cr : a.k.cr) + grp * 16) : 0x80000000u;
            gsoff[i] = in ? (uint32_t)(row * (int)(gv[i] ? a.v.sr : a.k.sr) + grp) : 0x80000000u;
            // (chunk e of the group: + 8 (e ^ gsw))
            glds[i] = gv[i] ? Shape::K_ELEMS + row * Shape::VST + ((32 * grp) ^ ((vswz4<DP>(row) & ~3) << 3))
                            : row * Shape::KST + 32 * grp;
            gsw[i] = gv[i] ? vswz4<DP>(row) & 3 : 0;
        }
    }
    __device__ __forceinline__ void load(const Pages4<Stage4>& pg, int row) {
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int x = gv[i] ? 2 : 0;
            gc[i] = __builtin_amdgcn_raw_buffer_load_b128(gv[i] ? pg.rs[2] : pg.rs[0], goff[i] + (uint32_t)row * (uint32_t)pg.rstride[x], 0, 0);
            gs[i] = __builtin_amdgcn_raw_buffer_load_b8(gv[i] ? pg.rs[3] : pg.rs[1], gsoff[i] + (uint32_t)row * (uint32_t)pg.rstride[x + 1], 0, 0);
        }
    }

    // NaN groups of a block's V, a bit each (and a place for what nobody reads)
    struct Nans {
        uint64_t groups[GPR + 1];
    };
    __device__ __forceinline__ void write(uint16_t* tile, Nans& nans, bool part, int half_, int tid) {
        const int lane = tid & 63;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            if (i % 2 != half_) continue;
            if (GROUPS % kThreads4 == 0 || tid + kThreads4 * i < GROUPS) {
                uint16_t* p = tile + glds[i];
                const bool nan = part & gv[i] & (gs[i] == 255);
                nans.groups[gv[i] && lane == 0 ? (tid + kThreads4 * i - kTK * GPR) >> 6 : GPR] = __ballot(nan);
                const float s = nan ? 0.f : kv4_scale(gs[i]);
                if constexpr (IS_BF16) {  // (fp16 saturates below; the test costs 1 % of the chunk above)
                    if (__builtin_expect(gv[i] && kv4_beyond(gs[i]), 0)) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) gc[i][e] = kv4_saturate8(gc[i][e], gs[i]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *reinterpret_cast<u32x4_t*>(p + 8 * (e ^ gsw[i])) = IS_BF16 ? kv4_bf16x8(gc[i][e], s) : kv4_f16x8(gc[i][e], s);
            }
        }
    }
    // what the scores of the block that was written last are still to be multiplied by
    __device__ __forceinline__ float k_scale() const { return 1.f; }

    __device__ __forceinline__ void add_nans(const Nans& nans, f32x16_t (&o)[DP / 32], int j, int lo, int hi, int) const {
#pragma unroll
        for (int i = 0; i < GPR; ++i) {
            for (uint64_t x = nans.groups[i]; x; x &= x - 1) {
                const int u = __builtin_amdgcn_readfirstlane(64 * i + __builtin_ctzll(x)), row = u / GPR;
                const bool sees = j + row >= lo && j + row <= hi;
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) {
                    float y = sees && db == u - row * GPR ? __builtin_nanf("") : 0.f;
                    pin(y);  // (no indexing of o by the group)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[db][r] += y;
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
    return bf16 ? tile_of<Stage4<DP, true>>(bias, lse) : tile_of<Stage4<DP, false>>(bias, lse);
}

}  // namespace

void* mfa_kv4_tile_kernel_of(int dp, bool bf16, bool bias, bool lse) {
    switch (dp) {
        case 32: return tile_of<32>(bf16, bias, lse);
        case 64: return tile_of<64>(bf16, bias, lse);
        case 96: return tile_of<96>(bf16, bias, lse);
        default: return tile_of<128>(bf16, bias, lse);
    }
}
