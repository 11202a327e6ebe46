// Copies of pages (ssq_copy_pages): every pool of a cache (codes, values, scales, passthrough rows) in one launch.
//
// A page of a pool is a run of bytes; the work is (pair, pool, piece of 4 KiB), one piece a wave at a time, 16 bytes a
// lane, four loads in flight.  Bound by bytes for many pages, by the launch for few: 16,384 pages
// (336 MB read and as many written) 139 us, 4.8 TB/s, where a large copy reaches 5.1 (147 us with stores that stay in the
// caches); 64 pages 6.4 us a call, 4.0 in the kernel.
#include "ssq_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kPiece = 4096;
constexpr int kInFlight = kPiece / (SSQ_WAVE * 16);

struct Pool {
    const uint8_t* src;
    uint8_t* dst;
    int64_t src_stride, dst_stride;  // bytes from page to page
    int64_t src_pages, dst_pages, bytes;
    int first, unit;                 // its first piece of a pair; bytes a lane moves at once
};
struct CopyParams {
    Pool pool[SSQ_COPY_POOLS];
    int n_pools, pieces;             // pieces of a pair
    const int64_t* from;
    const int64_t* to;
    int64_t n;
};

template <class T>
__device__ __forceinline__ void move(const uint8_t* src, uint8_t* dst, int lane, int64_t bytes) {
    const T* s = reinterpret_cast<const T*>(src);
    T* d = reinterpret_cast<T*>(dst);
    const int n = (int)(bytes / (int64_t)sizeof(T));
    for (int i = lane; i < n; i += SSQ_WAVE * kInFlight) {
        T x[kInFlight];
#pragma unroll
        for (int k = 0; k < kInFlight; ++k)
            if (i + SSQ_WAVE * k < n) x[k] = __builtin_nontemporal_load(s + i + SSQ_WAVE * k);
#pragma unroll
        for (int k = 0; k < kInFlight; ++k)
            if (i + SSQ_WAVE * k < n) __builtin_nontemporal_store(x[k], d + i + SSQ_WAVE * k);
    }
}

__global__ __launch_bounds__(kThreads) void k_copy_pages(const CopyParams p) {
    typedef unsigned int u4 __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x & (SSQ_WAVE - 1);
    const int64_t waves = (int64_t)gridDim.x * (kThreads / SSQ_WAVE), all = p.n * p.pieces;
    for (int64_t w = (int64_t)blockIdx.x * (kThreads / SSQ_WAVE) + __builtin_amdgcn_readfirstlane(threadIdx.x / SSQ_WAVE); w < all;
         w += waves) {
        const int64_t pair = w / p.pieces;
        const int piece = (int)(w - pair * p.pieces);
        int k = 0;
        while (k + 1 < p.n_pools && piece >= p.pool[k + 1].first) ++k;
        const Pool& c = p.pool[k];
        const int64_t from = p.from[pair], to = p.to[pair];
        if (from < 0 || to < 0 || from >= c.src_pages || to >= c.dst_pages) continue;
        const int64_t at = (int64_t)(piece - c.first) * kPiece, bytes = min((int64_t)kPiece, c.bytes - at);
        const uint8_t* src = c.src + from * c.src_stride + at;
        uint8_t* dst = c.dst + to * c.dst_stride + at;
        if (c.unit == 16) move<u4>(src, dst, lane, bytes);
        else if (c.unit == 4) move<uint32_t>(src, dst, lane, bytes);
        else move<uint8_t>(src, dst, lane, bytes);
    }
}

}  // namespace

extern "C" int ssq_copy_pages(const ssq_copy_args* a, void* stream) {
    if (!a) return ssq_fail(SSQ_ERR_INVALID, "args is NULL");
    if (a->struct_size != sizeof(ssq_copy_args))
        return ssq_fail(SSQ_ERR_ABI, "ssq_copy_args size %u != library's %zu", a->struct_size, sizeof(ssq_copy_args));
    SSQ_REQUIRE(a->n_pools >= 1 && a->n_pools <= SSQ_COPY_POOLS, "n_pools must be in [1, %d]", SSQ_COPY_POOLS);
    SSQ_REQUIRE(a->n_pairs >= 0 && a->n_pairs <= 0x7fffffff, "bad n_pairs");
    CopyParams p{};
    p.n_pools = a->n_pools;
    p.n = a->n_pairs;
    p.from = a->from;
    p.to = a->to;
    int64_t pieces = 0;
    for (int k = 0; k < a->n_pools; ++k) {
        const ssq_copy_pool& c = a->pool[k];
        SSQ_REQUIRE(c.bytes >= 0 && c.src_pages >= 0 && c.dst_pages >= 0, "bad pool %d", k);
        SSQ_UNSUPPORTED(c.bytes <= 1ll << 32, "pages are too large");
        SSQ_REQUIRE((c.src && c.dst) || c.bytes == 0 || c.src_pages == 0 || c.dst_pages == 0, "pool %d is NULL", k);
        const uint64_t at = (uint64_t)(uintptr_t)c.src | (uint64_t)(uintptr_t)c.dst | (uint64_t)c.src_stride | (uint64_t)c.dst_stride | (uint64_t)c.bytes;
        p.pool[k] = {reinterpret_cast<const uint8_t*>(c.src), reinterpret_cast<uint8_t*>(c.dst), c.src_stride, c.dst_stride,
                     c.src_pages, c.dst_pages, c.bytes, (int)pieces, at % 16 == 0 ? 16 : at % 4 == 0 ? 4 : 1};
        pieces += (c.bytes + kPiece - 1) / kPiece;
        SSQ_UNSUPPORTED(pieces <= 1 << 24, "pages are too large");
    }
    if (p.n == 0 || pieces == 0) return SSQ_OK;
    SSQ_REQUIRE(p.from && p.to, "from and to must be non-NULL");
    p.pieces = (int)pieces;
    const int64_t per = kThreads / SSQ_WAVE, need = (p.n * pieces + per - 1) / per, most = (int64_t)ssq_device_cus() * 8;
    hipLaunchKernelGGL(k_copy_pages, dim3((unsigned)(need < most ? need : most)), dim3(kThreads), 0, (hipStream_t)stream, p);
    return ssq_check_hip(hipGetLastError(), "k_copy_pages launch");
}
