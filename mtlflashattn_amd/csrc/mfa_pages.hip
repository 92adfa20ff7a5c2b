// mfa_pages.hip -- pages copied inside the pools of a paged cache
// (mfa_copy_pages in include/mfa.h).
//
// Bound by memory: a workgroup copies one segment of one page of one pool, every
// load of a thread in flight before its first store.  Non-temporal stores keep the
// copies from pushing what is read next out of the L2: 300 pages of 512 KB in two
// pools take 113.5 us (5.54 TB/s read and written; a large library copy reaches
// 5.15), 135 with ordinary stores, 128 with loads non-temporal too.  One launch takes
// all pairs and up to 64 pools (the K and V pools, or codes and scales, of many
// layers).
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>

#include "mfa.h"
#include "mfa_common.h"

namespace {

constexpr int kCThreads = 256;
constexpr int kCLoads = 4;  // loads of a thread in flight (two: 118 us, eight: 130)

struct CArgs {
    char* base[MFA_COPY_MAX_POOLS];
    int64_t stride[MFA_COPY_MAX_POOLS], bytes[MFA_COPY_MAX_POOLS];
    int32_t seg0[MFA_COPY_MAX_POOLS];  // first segment of a pool's pages
    const int32_t* src;
    const int32_t* dst;
    int32_t pools, segs, npages;
    int32_t rounds;  // rounds of kCLoads loads per segment
};

// T: the widest type that every base, stride and size is a multiple of
template <class T>
__global__ void __launch_bounds__(kCThreads) mfa_copy_pages_kernel(CArgs a) {
    const int pair = blockIdx.x / a.segs, seg = blockIdx.x - pair * a.segs;
    const int src = a.src[pair], dst = a.dst[pair];
    if ((uint32_t)src >= (uint32_t)a.npages || (uint32_t)dst >= (uint32_t)a.npages || src == dst) return;
    int p = 0;
    while (p + 1 < a.pools && seg >= a.seg0[p + 1]) ++p;
    const int64_t per_round = (int64_t)kCThreads * kCLoads;
    int64_t at = (int64_t)(seg - a.seg0[p]) * a.rounds * per_round + threadIdx.x;
    const int64_t n = a.bytes[p] / (int64_t)sizeof(T);
    const T* s = reinterpret_cast<const T*>(a.base[p] + src * a.stride[p]);
    T* d = reinterpret_cast<T*>(a.base[p] + dst * a.stride[p]);
    for (int r = 0; r < a.rounds && at < n; ++r, at += per_round) {
        T x[kCLoads];
#pragma unroll
        for (int i = 0; i < kCLoads; ++i)
            if (at + i * kCThreads < n) x[i] = s[at + i * kCThreads];
#pragma unroll
        for (int i = 0; i < kCLoads; ++i)
            if (at + i * kCThreads < n) __builtin_nontemporal_store(x[i], d + at + i * kCThreads);
    }
}

int cerr_(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(mfa_error_buffer(), 512, fmt, ap);
    va_end(ap);
    return code;
}

}  // namespace

extern "C" {

int mfa_copy_pages_params_size(void) { return (int)sizeof(mfa_copy_pages_params); }

int mfa_copy_pages(const mfa_copy_pages_params* p, void* stream) {
    mfa_error_buffer()[0] = 0;
    if (!p) return cerr_(MFA_ERR_INVALID, "mfa_copy_pages: params is NULL");
    if (p->pools < 0 || p->pools > MFA_COPY_MAX_POOLS)
        return cerr_(MFA_ERR_INVALID, "mfa_copy_pages: %d pools outside [0, %d]", p->pools, MFA_COPY_MAX_POOLS);
    if (p->pairs < 0 || p->num_pages < 0) return cerr_(MFA_ERR_INVALID, "mfa_copy_pages: negative size");
    CArgs a;
    memset(&a, 0, sizeof(a));
    uint64_t all = 0;  // (its low bits: what everything is a multiple of)
    int64_t total = 0;
    for (int i = 0; i < p->pools; ++i) {
        const mfa_copy_pool& q = p->pool[i];
        if (q.page_bytes < 0 || (q.page_bytes > 0 && p->num_pages > 0 && !q.base))
            return cerr_(MFA_ERR_INVALID, "mfa_copy_pages: pool %d: base and page_bytes >= 0 are required", i);
        if (p->num_pages > 1 && q.page_stride < q.page_bytes)
            return cerr_(MFA_ERR_INVALID, "mfa_copy_pages: pool %d: pages overlap", i);
        a.base[i] = static_cast<char*>(q.base);
        a.stride[i] = q.page_stride;
        a.bytes[i] = q.page_bytes;
        all |= (uint64_t)reinterpret_cast<uintptr_t>(q.base) | (uint64_t)q.page_bytes | (p->num_pages > 1 ? (uint64_t)q.page_stride : 0);
        total += q.page_bytes;
    }
    if (p->pairs == 0 || p->num_pages == 0 || total == 0) return MFA_OK;
    auto bad = [](const void* x) { return !x || (reinterpret_cast<uintptr_t>(x) & 3); };
    if (bad(p->src) || bad(p->dst)) return cerr_(MFA_ERR_INVALID, "mfa_copy_pages: src and dst are required");
    const int width = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    // rounds per segment: as many, up to 16, as leave four workgroups per CU (the
    // pages above: 116.1 us with one, 118.3 with four, 113.5 with 16)
    const int64_t round = (int64_t)kCThreads * kCLoads * width;
    a.rounds = (int32_t)std::min<int64_t>(std::max<int64_t>(p->pairs * (total / round) / (4 * (int64_t)mfa_chip_cus(stream)), 1), 16);
    int64_t segs = 0;
    for (int i = 0; i < p->pools; ++i) {
        a.seg0[i] = (int32_t)segs;
        segs += (a.bytes[i] + round * a.rounds - 1) / (round * a.rounds);
        if (segs > 0x7fffffffLL) return cerr_(MFA_ERR_INVALID, "mfa_copy_pages: problem too large");
    }
    // (a launch has less than 2^32 threads)
    if (segs * p->pairs > 0xffffff) return cerr_(MFA_ERR_INVALID, "mfa_copy_pages: problem too large");
    a.src = p->src;
    a.dst = p->dst;
    a.pools = p->pools;
    a.segs = (int32_t)segs;
    a.npages = p->num_pages;
    const auto fn = width == 16 ? mfa_copy_pages_kernel<u32x4_t> : width == 4 ? mfa_copy_pages_kernel<uint32_t> : mfa_copy_pages_kernel<uint8_t>;
    hipLaunchKernelGGL(fn, dim3((unsigned)(segs * p->pairs)), dim3(kCThreads), 0, static_cast<hipStream_t>(stream), a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return cerr_(MFA_ERR_LAUNCH, "mfa_copy_pages: launch failed: %s", hipGetErrorString(e));
    return MFA_OK;
}

}  // extern "C"
