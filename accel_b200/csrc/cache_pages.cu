// Copies of whole cache pages in every cache of a model at once: what a fork's copy on write and a
// compaction of the pool move.  No counterpart in the reference.
//
// caches[c][dst[i]] = caches[c][src[i]] for every cache c and pair i: 2 * caches * pairs * page bytes
// of traffic and no arithmetic, so HBM bounds a large call and the launch a small one.  The pairs are
// host numbers (the pool that chose them is host code) and travel with the cache pointers in the
// kernel's parameters: no copy to the device precedes the launch and nothing has to outlive it.
#include <algorithm>
#include <new>
#include <vector>

#include "common.cuh"

namespace ab {

namespace {

constexpr int kMaxCaches = 128;       // per launch: 1 KB of the parameters
constexpr int kThreads = 256;
constexpr uint32_t kChunk = 16384;    // bytes a CTA copies (537 MB in 16 caches: 81.6 us, 6.6 TB/s; 81.9 with 8 KB, 86.0 with 64 KB; one
                                      // page of 64 KB in 8 caches: 2.4, 2.0 and 4.8 us)

template <int P> struct CopyParams {
    void *cache[kMaxCaches];
    uint32_t src[P], dst[P];
    uint64_t page_bytes;
    uint32_t n_caches, n_pairs, chunks;
};

template <typename V, int P> __global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ CopyParams<P> p)
{
    pdl_wait();
    const uint32_t chunk = blockIdx.x % p.chunks, pair = blockIdx.x / p.chunks;
    char *cache = static_cast<char *>(p.cache[blockIdx.y]);
    const uint64_t at = (uint64_t)chunk * kChunk;
    const uint32_t n = (uint32_t)min((uint64_t)kChunk, p.page_bytes - at) / sizeof(V);
    const V *s = reinterpret_cast<const V *>(cache + (uint64_t)p.src[pair] * p.page_bytes + at);
    V *d = reinterpret_cast<V *>(cache + (uint64_t)p.dst[pair] * p.page_bytes + at);
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) d[i] = s[i];
}

template <typename V, int P>
int run_copy(cudaStream_t stream, void *const *caches, int n_caches, uint64_t page_bytes, const uint32_t *src,
             const uint32_t *dst, int n_pairs)
{
    CopyParams<P> p;
    p.page_bytes = page_bytes;
    p.chunks = (uint32_t)((page_bytes + kChunk - 1) / kChunk);
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const int per_launch = (int)std::min<uint64_t>(P, std::max<uint64_t>(1, 0x7fffffffull / p.chunks));
    for (int c0 = 0; c0 < n_caches; c0 += kMaxCaches)
        for (int i0 = 0; i0 < n_pairs; i0 += per_launch) {
            p.n_caches = (uint32_t)std::min(kMaxCaches, n_caches - c0);
            p.n_pairs = (uint32_t)std::min(per_launch, n_pairs - i0);
            memcpy(p.cache, caches + c0, p.n_caches * sizeof(void *));
            memcpy(p.src, src + i0, p.n_pairs * 4);
            memcpy(p.dst, dst + i0, p.n_pairs * 4);
            cfg.gridDim = dim3(p.chunks * p.n_pairs, p.n_caches);
            const cudaError_t e = cudaLaunchKernelEx(&cfg, copy_pages_kernel<V, P>, p);
            count_launch();
            const int rc = check_cuda(e, "ab_cache_copy_pages");
            if (rc) return rc;
        }
    return AB_OK;
}

// 2 KB of parameters for the few pairs of a fork, 29 KB of the 32 that a launch may have for a compaction's (one pair in 64
// caches: 2.6 us on the device with the small block, 2.8 with the large, and 29 KB less to write on the host)
template <typename V>
int run_copy(cudaStream_t stream, void *const *caches, int n_caches, uint64_t page_bytes, const uint32_t *src, const uint32_t *dst, int n_pairs)
{
    return n_pairs <= 96 ? run_copy<V, 96>(stream, caches, n_caches, page_bytes, src, dst, n_pairs)
                         : run_copy<V, 3500>(stream, caches, n_caches, page_bytes, src, dst, n_pairs);
}

}  // namespace
}  // namespace ab

using namespace ab;

extern "C" int ab_cache_copy_pages(void *stream, void *const *caches, int n_caches, size_t page_bytes, uint32_t pages,
                                   const uint32_t *src, const uint32_t *dst, int n_pairs)
{
    if (n_caches < 0 || n_pairs < 0 || (n_caches && !caches) || (n_pairs && (!src || !dst)) || page_bytes == 0)
        return fail(AB_ERR_INVALID, "ab_cache_copy_pages: bad argument");
    if ((page_bytes + kChunk - 1) / kChunk > 0x7fffffffull)
        return fail(AB_ERR_INVALID, "ab_cache_copy_pages: a page of %zu bytes", page_bytes);
    if (n_pairs == 0) return AB_OK;
    uintptr_t align = (uintptr_t)page_bytes;
    for (int c = 0; c < n_caches; c++) {
        if (!caches[c]) return fail(AB_ERR_INVALID, "ab_cache_copy_pages: cache %d is NULL", c);
        align |= reinterpret_cast<uintptr_t>(caches[c]);
    }
    // One pass in no particular order is a copy only if no page is written twice, or both written and read.  A bit per page
    // says what is written; it is laid out for the pages between the smallest and the largest destination
    uint32_t low = 0xffffffffu, high = 0;
    for (int i = 0; i < n_pairs; i++) {
        if (src[i] >= pages || dst[i] >= pages)
            return fail(AB_ERR_INVALID, "ab_cache_copy_pages: pair %d copies page %u to page %u of a cache of %u pages", i,
                        src[i], dst[i], pages);
        low = std::min(low, dst[i]);
        high = std::max(high, dst[i]);
    }
    std::vector<uint64_t> written;
    std::vector<uintptr_t> starts;
    try {
        written.assign((size_t)(high - low) / 64 + 1, 0);
        starts.resize((size_t)n_caches);
    } catch (const std::bad_alloc &) {
        return fail(AB_ERR_OOM, "ab_cache_copy_pages: host allocation failed");
    }
    for (int i = 0; i < n_pairs; i++) {
        uint64_t &w = written[(dst[i] - low) / 64];
        const uint64_t bit = 1ull << ((dst[i] - low) % 64);
        if (w & bit) return fail(AB_ERR_INVALID, "ab_cache_copy_pages: page %u is written twice", dst[i]);
        w |= bit;
    }
    for (int i = 0; i < n_pairs; i++)
        if (src[i] >= low && src[i] <= high && (written[(src[i] - low) / 64] >> ((src[i] - low) % 64) & 1))
            return fail(AB_ERR_INVALID, "ab_cache_copy_pages: page %u is both read and written", src[i]);
    if (n_caches == 0) return AB_OK;
    for (int c = 0; c < n_caches; c++) starts[c] = reinterpret_cast<uintptr_t>(caches[c]);
    std::sort(starts.begin(), starts.end());
    for (int c = 1; c < n_caches; c++)
        if ((starts[c] - starts[c - 1]) / page_bytes < pages)
            return fail(AB_ERR_INVALID, "ab_cache_copy_pages: two of the caches overlap; each is copied on its own");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (align % 16 == 0) return run_copy<uint4>(s, caches, n_caches, page_bytes, src, dst, n_pairs);
    if (align % 4 == 0) return run_copy<uint32_t>(s, caches, n_caches, page_bytes, src, dst, n_pairs);
    return run_copy<uint8_t>(s, caches, n_caches, page_bytes, src, dst, n_pairs);
}
