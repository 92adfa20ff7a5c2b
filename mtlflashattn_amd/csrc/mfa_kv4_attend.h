// mfa_kv4_attend.h -- what the kernels of attention over the paged 4-bit cache
// (mfa_kv4_attend.hip, mfa_kv4_tile.hip) share: arguments, the dealing of work
// over workgroups, pages and result rows.
#pragma once

#include "mfa_kv4.h"

namespace {

typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4_t;

constexpr int kThreads4 = 256;
constexpr int kChunk4 = 128;  // keys per chunk, the unit of dealt work
constexpr float kLn2f = 0.6931471805599453f;

// What the merge kernel adds for workgroup w: the parts of workgroups w - 1 to w1
// (-1: nothing) of a unit, whose first part is in slot0.
struct Merge4 {
    int32_t w1, slot0, b, q0, hkv, col0, ncol, pad;
};

struct K4Args {
    const char* q;
    char* o;
    float* lse;
    int64_t qb, qs, qh, ob, os, oh, lse_b, lse_h;
    Kv4Pool k, v;
    const int32_t* bt;
    int64_t bt_b;
    const int32_t* lens;
    const int32_t* cu_q;  // NULL: Lq rows per sequence
    const float* alibi;
    int32_t alibi_bstride;
    int32_t B, Hq, Hkv, R, Lq, max_k;
    int32_t page, npages;
    FastDiv by_page, by_r;
    float scale, scale_log2, softcap, softcap_sk;
    int32_t wl, wr, causal, bias;
    int32_t G;       // workgroups
    int32_t xcds;    // of which every xcds-th runs on the same XCD (1: unknown, or G not a multiple)
    int32_t cols;    // columns per unit
    int32_t rows_q;  // rows of q (varlen: all of them)
    int32_t min_cols, max_cols;  // a sequence with fewer or more columns is another launch's
    float* ws_o;     // [G][2][cols][D]
    float* ws_ml;    // [G][2][cols][2] exponent reference, sum of p
    Merge4* ws_merge;  // [G], NULL: no unit is walked by more than one workgroup
};

// The kernels read their arguments where they need them, through a pointer that
// the compiler cannot see through: all of them in scalar registers at once are
// more than there are, and the spills land in the inner loop.
typedef const __attribute__((address_space(4))) K4Args K4Const;
__device__ __forceinline__ K4Const& args4(int which = 0) {
    K4Const* p = (K4Const*)__builtin_amdgcn_kernarg_segment_ptr() + which;
    asm volatile("" : "+s"(p));
    return *p;
}

__device__ __forceinline__ uint32_t div4(uint32_t j, const __attribute__((address_space(4))) FastDiv& f) {
    return f.d <= 1 ? j : __umulhi(j, f.m) >> f.s;
}

__device__ __forceinline__ int lo4(int wl, int c) { return wl >= 0 && c > wl ? c - wl : 0; }
__device__ __forceinline__ int hi4(int causal, int wr, int c, int Lk) {
    int hi = Lk - 1;
    if (causal) hi = min(hi, c);
    if (wr >= 0 && wr < hi - c) hi = c + wr;  // (c + wr may pass 31 bits)
    return hi;
}

// The chunks with keys among chunks c0 to c0 + nch - 1 of a unit with keys t_lo to
// t_hi, counted from the sequence's first key (none: beg = end, behind t_hi; the
// dealt ones behind it may begin past 31 bits).
struct Chunks4 {
    int beg, end;
};
__device__ __forceinline__ Chunks4 chunks4(int t_lo, int t_hi, int c0, int nch) {
    const int past = t_hi < 0 ? 0 : t_hi / kChunk4 + 1, beg = t_lo / kChunk4 + c0;
    return Chunks4{min(beg, past), min(beg + nch, past)};
}

// The work of a sequence: its rows, keys, column tiles and chunks per unit.
struct Seq4 {
    int q0, Lq, Lk, tiles, chunks;
    __device__ __forceinline__ int items(int Hkv) const { return tiles * Hkv * chunks; }
};
__device__ __forceinline__ Seq4 seq4(K4Const& a, int b) {
    Seq4 s;
    s.q0 = 0;
    s.Lq = a.Lq;
    if (a.cu_q) {
        // (bounded by the tensor whatever the prefix sums hold)
        s.q0 = min(max(a.cu_q[b], 0), a.rows_q);
        s.Lq = min(max(a.cu_q[b + 1], s.q0), a.rows_q) - s.q0;
    }
    s.Lk = min(max(a.lens[b], 0), a.max_k);
    const int cols = s.Lq * a.R;
    s.tiles = cols >= a.min_cols && cols <= a.max_cols ? (cols + a.cols - 1) / a.cols : 0;
    // chunks that hold the widest key range of a tile's rows (at least one: a
    // row without keys is stored too)
    int n = (s.Lk + kChunk4 - 1) / kChunk4;
    if (a.wl >= 0 && (a.causal || a.wr >= 0)) {
        const int64_t span = (int64_t)a.wl + (a.causal ? 0 : a.wr) + (a.cols - 1) / a.R + 1;
        n = (int)min((int64_t)n, (span + kChunk4 - 1) / kChunk4 + 1);
    }
    s.chunks = max(n, 1);
    return s;
}
__device__ __forceinline__ Seq4 lane_seq4(const Seq4& s, int l) {
    return Seq4{__builtin_amdgcn_readlane(s.q0, l), __builtin_amdgcn_readlane(s.Lq, l), __builtin_amdgcn_readlane(s.Lk, l),
                __builtin_amdgcn_readlane(s.tiles, l), __builtin_amdgcn_readlane(s.chunks, l)};
}

// inclusive prefix sum over the wavefront
__device__ __forceinline__ int scan64(int x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// The items of the call are laid end to end, sequence by sequence (a sequence's:
// K/V head by K/V head, tile by tile, chunk by chunk); of C items workgroup w
// takes w C / G to (w + 1) C / G.
__device__ __forceinline__ int first_item(int w, int C, int G) { return (int)((int64_t)w * C / G); }
__device__ __forceinline__ int wg_of_item(int x, int C, int G) { return (int)((((int64_t)x + 1) * G - 1) / C); }

// A workgroup's walk over its items.
struct Walk4 {
    int C, G, w;  // items, workgroups that have some, this one
    int x, xbeg, xend;
    int b, before;  // sequence of item x, items before that sequence
    Seq4 sq;

    // of this workgroup; false: no items
    __device__ __forceinline__ bool start() {
        K4Const& a = args4();
        w = blockIdx.x;
        if (a.xcds > 1) w = (w % a.xcds) * (a.G / a.xcds) + w / a.xcds;  // (neighbours share an XCD)
        const bool some = find(a);
        if (a.ws_merge && threadIdx.x == 0) {
            // the unit of the first item is merged here where it began in the
            // walk of the workgroup before
            Merge4 g{-1, 0, 0, 0, 0, 0, 0, 0};
            if (some && w > 0) {
                const int off = x - before, unit = off / sq.chunks, x0 = before + unit * sq.chunks;
                const int first = first_item(w - 1, C, G);
                if (x0 < x && wg_of_item(x0, C, G) == w - 1) {
                    g.w1 = wg_of_item(x0 + sq.chunks - 1, C, G);
                    g.slot0 = first >= x0 ? 0 : 1;
                    g.b = b;
                    g.q0 = sq.q0;
                    g.hkv = unit / sq.tiles;
                    g.col0 = (unit - g.hkv * sq.tiles) * a.cols;
                    g.ncol = min(a.cols, sq.Lq * a.R - g.col0);
                }
            }
            a.ws_merge[w] = g;
        }
        return some;
    }
    __device__ __forceinline__ bool find(K4Const& a) {
        const int lane = threadIdx.x & 63, B = a.B;
        // (one pass where the sequences fit a wavefront)
        Seq4 s{0, 0, 0, 0, 1};
        if (lane < B) s = seq4(a, lane);
        int n = s.items(a.Hkv), inc = scan64(n);
        C = __builtin_amdgcn_readlane(inc, 63);
        for (int b0 = 64; b0 < B; b0 += 64) {
            const int y = b0 + lane < B ? seq4(a, b0 + lane).items(a.Hkv) : 0;
            C += __builtin_amdgcn_readlane(scan64(y), 63);
        }
        G = min(a.G, C);  // (every workgroup below G has an item: the merge reads them all)
        if (w >= G) return false;
        xbeg = x = first_item(w, C, G);
        xend = first_item(w + 1, C, G);
        int base = 0;
        for (int b0 = 0;;) {
            const uint64_t past = __ballot(inc + base > x);
            if (past) {
                const int l = __builtin_ctzll(past);
                before = base + __builtin_amdgcn_readlane(inc - n, l);
                b = b0 + l;
                sq = lane_seq4(s, l);
                return true;
            }
            base += __builtin_amdgcn_readlane(inc, 63);
            b0 += 64;
            if (b0 >= B) return false;
            s = b0 + lane < B ? seq4(a, b0 + lane) : Seq4{0, 0, 0, 0, 1};
            n = s.items(a.Hkv);
            inc = scan64(n);
        }
    }

    // The unit of item x and the chunks of it that are this workgroup's.
    int hkv, col0, ncol, c0, nch, slot;
    bool whole;
    // false: the walk is over
    __device__ __forceinline__ bool next(K4Const& a) {
        if (x >= xend) return false;
        while (x - before >= sq.items(a.Hkv)) {  // (the next sequence with rows)
            if (b + 1 >= a.B) return false;
            before += sq.items(a.Hkv);
            sq = seq4(a, ++b);
        }
        const int off = x - before, unit = off / sq.chunks;
        c0 = off - unit * sq.chunks;
        nch = min(sq.chunks - c0, xend - x);
        whole = nch == sq.chunks;
        slot = x == xbeg ? 0 : 1;
        x += nch;
        hkv = unit / sq.tiles;
        col0 = (unit - hkv * sq.tiles) * a.cols;
        ncol = min(a.cols, sq.Lq * a.R - col0);
        return true;
    }
    __device__ __forceinline__ int64_t part_row(int cols) const { return ((int64_t)w * 2 + slot) * cols; }
};

// A wavefront's way through the pages of a unit: the buffer resources of the
// current page of K's codes and scales and V's, which end with the sequence
// (rows behind it, and any row of a page id outside the pool, read as zeros).
// The id of the page that is expected next is loaded ahead, by the scalar unit: a
// vector load of it would have to wait for all the codes on their way.
template <int DP>
struct Pages4 {
    typedef const __attribute__((address_space(4))) int32_t* ids_t;
    __amdgpu_buffer_rsrc_t rs[4];
    ids_t bt;
    FastDiv by_page;
    int Lk, npages, last, idx, row0, ahead, next_idx, next_id;
    uint64_t base[4];
    int64_t ps[4];
    int rstride[4];  // bytes between rows

    // step: keys between the blocks that are loaded one after the other
    __device__ __forceinline__ void start(K4Const& a, int b, int hkv, int Lk_, int key, int step) {
        bt = (ids_t)(uintptr_t)(a.bt + b * a.bt_b);
        by_page = FastDiv{a.by_page.d, a.by_page.m, a.by_page.s};
        Lk = Lk_;
        npages = a.npages;
        last = (int)quotient((uint32_t)max(Lk - 1, 0), by_page);
        idx = -1;
        row0 = 0;
        ahead = max(1, step / a.page);
        next_idx = min((int)quotient((uint32_t)key, by_page), last);
        next_id = Lk > 0 ? bt[next_idx] : 0;
        base[0] = (uint64_t)(a.k.codes + hkv * a.k.ch);
        base[1] = (uint64_t)(a.k.scales + hkv * a.k.sh);
        base[2] = (uint64_t)(a.v.codes + hkv * a.v.ch);
        base[3] = (uint64_t)(a.v.scales + hkv * a.v.sh);
        ps[0] = a.k.cp; ps[1] = a.k.sp; ps[2] = a.v.cp; ps[3] = a.v.sp;
        rstride[0] = (int)a.k.cr; rstride[1] = (int)a.k.sr; rstride[2] = (int)a.v.cr; rstride[3] = (int)a.v.sr;
    }
    // the row of key j in its page, which becomes the current one (behind the last
    // key: the last page stays; without keys: resources of no bytes)
    __device__ __forceinline__ int row_of(int j) {
        const int i = min((int)quotient((uint32_t)j, by_page), last);
        if (i != idx) {
            int id = next_id;
            if (i != next_idx) id = Lk > 0 ? bt[i] : 0;
            idx = i;
            next_idx = min(i + ahead, last);
            next_id = Lk > 0 ? bt[next_idx] : 0;
            row0 = i * (int)by_page.d;
            const int rows = min(Lk - row0, (int)by_page.d);
            const bool ok = (uint32_t)id < (uint32_t)npages && rows > 0;
#pragma unroll
            for (int x = 0; x < 4; ++x)
                rs[x] = __builtin_amdgcn_make_buffer_rsrc((void*)(base[x] + (ok ? id : 0) * ps[x]), (short)0,
                                                          ok ? (rows - 1) * rstride[x] + (x & 1 ? DP / 32 : DP / 2) : 0, kBufferDword3);
        }
        return j - row0;
    }
};

template <bool IS_BF16>
__device__ __forceinline__ void store_row4(char* row, int d, const f32x4_t& o, float l) {
    f32x4_t x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = l > 0.f ? o[i] / l : o[i];  // (l = 0: no key, o = 0; NaN stays NaN)
    if constexpr (IS_BF16) {
        typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 v4;
        store_stream(reinterpret_cast<v4*>(reinterpret_cast<__bf16*>(row) + d),
                     v4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]});
    } else {
        typedef __attribute__((__vector_size__(4 * sizeof(_Float16)))) _Float16 v4;
        store_stream(reinterpret_cast<v4*>(reinterpret_cast<_Float16*>(row) + d),
                     v4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]});
    }
}
__device__ __forceinline__ int64_t row_off4(bool varlen, int b, int q0, int i, int h, int64_t sb, int64_t ss, int64_t sh) {
    return (varlen ? (int64_t)(q0 + i) * ss : b * sb + i * ss) + h * sh;
}
__device__ __forceinline__ void store_lse4(K4Const& a, int b, int q0, int i, int h, float m, float l) {
    if (!a.lse) return;
    a.lse[(a.cu_q ? (int64_t)(q0 + i) : b * a.lse_b + i) + h * a.lse_h] =
        m == -INFINITY ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2f;
}

}  // namespace

// 128-column tiles (mfa_kv4_tile.hip): void(*)(K4Args)
__attribute__((visibility("hidden"))) void* mfa_kv4_tile_kernel_of(int dp, bool bf16, bool bias);
constexpr int kTileCols4 = 128;
