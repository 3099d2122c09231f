// Windowed attention: what its row kernel (window_attention.cu) and its tile kernel (window_prefill.cu) share.
#pragma once
#include "common.cuh"

namespace ab {

enum Form { kDecode = 0, kBatch = 1, kRaggedStep = 2, kPrefillRows = 3 };

struct WinParams {
    const float *q;
    const void *k, *v;
    const uint32_t *pages, *lengths, *offsets;     // pages NULL: a contiguous cache
    float *out;
    uint32_t rows, batch, q_heads, kv_heads, head_dim, block, max_pages;
    uint32_t window, sinks;
    uint32_t reach;                                // positions the page table (or the cache) addresses
    uint32_t capacity;                             // rows of the cache
    uint32_t base;
    const uint4 *left;                             // a ragged step some of whose rows went on tiles: {how many did not}, then their
                                                   // {row, sequence (0xffffffff: zeros), position + 1, length}; or NULL
    float scale_log2;                              // Scale * log2(e)
    int form;
};

#ifdef __CUDACC__
// the cache row of position j; 0xffffffff where its page lies outside the cache
__device__ __forceinline__ uint32_t win_cache_row(const WinParams &p, const uint32_t *pages, uint32_t j)
{
    uint64_t r = j;
    if (pages) {
        const uint32_t pg = j / p.block;
        r = (uint64_t)pages[pg] * p.block + (j - pg * p.block);
    }
    return r < p.capacity ? (uint32_t)r : 0xffffffffu;
}
__device__ __forceinline__ float ld_cluster(uint32_t smem, uint32_t rank)
{
    float v;
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.f32 %0, [r];\n\t}"
                 : "=f"(v) : "r"(smem), "r"(rank) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t smem, uint32_t rank)
{
    float4 v;
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [r];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(smem), "r"(rank) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
#endif

// query rows (tokens x heads of a KV head) of one sequence from which 128-row tiles take over
constexpr uint32_t kTileFrom = 64;
// a prefill, or the sequences of a ragged step that have that many rows (it then sets p.left), on 128-row tiles
// (window_prefill.cu); p.q_heads / p.kv_heads <= 128
int run_window_tiles(Launch &l, WinParams &p, bool f16, const char *name);
int window_error_flag();

}  // namespace ab
