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

// Whether `rows` query rows (tokens x heads of a KV head) of one sequence, each of which sees up to `seen` positions, go
// on 128-row tiles.  A tile call costs its two launches and the packing of the positions, whatever the rows; the row
// kernel's time grows with rows x seen x KV heads.  (Head dimension 128, contiguous; tiles / rows one by one, us:
//     rows x seen           f32, groups of 4      f16, groups of 4      f16, groups of 8
//                           8 KV heads            8 KV heads            4 KV heads
//       32 x   512          20.8 /  11.5          17.8 /  11.9          17.7 /  10.3
//       64 x   512          21.4 /  15.7          17.7 /  13.7          17.7 /  10.5
//      128 x   512          21.7 /  22.8          17.7 /  18.8          17.6 /  13.6
//      256 x   512          21.7 /  46.7          18.5 /  25.0          17.7 /  15.7
//       16 x  4096          35.0 /  24.9          29.0 /  28.8          24.0 /  15.7
//       32 x  4096          35.3 /  42.7          29.0 /  26.9          23.9 /  17.7
//       64 x  4096          35.7 /  85.6          29.3 /  44.1          24.2 /  31.1
//       16 x 32768         185.5 / 147.0         147.7 / 123.2         103.8 /  57.8
//       32 x 32768         185.4 / 319.5         147.9 / 144.7         103.4 /  67.8
//       64 x 32768         186.0 / 587.2         148.7 / 278.6         104.3 / 125.3
//  and with 32 KV heads of one query head each
//       32 x   512          23.9 /  57.8          19.7 /  40.4
//      128 x   512          24.0 / 143.7          19.7 / 132.5
//       64 x  2048          51.7 / 279.0          32.4 / 270.7
//  with one KV head of eight
//      128 x   512          21.0 /  15.8          16.7 /   9.6
//      128 x  2048          23.1 /  20.0          18.7 /  14.3
//       64 x  8192          33.2 /  36.3          26.2 /  21.9
//      256 x  2048          23.1 /  24.0          18.8 /  23.9
//  The rule knows neither the type nor the group, and an f16 group of eight is the cheapest row by row: there it takes up to 1.5
//  times the better side (103.4 against 67.8 us at 32 x 32768), elsewhere in this table 1.2 times at most.)
constexpr uint32_t kTileFrom = 32;
__host__ __device__ inline bool on_tiles(uint64_t rows, uint64_t seen, uint32_t kv_heads)
{
    return rows >= 256 || (rows >= kTileFrom && rows * seen >= (8u * 65536u + kv_heads - 1) / kv_heads);
}
// a prefill, or a ragged step: its sequences with that many rows, on 128-row tiles (window_prefill.cu); p.left says which rows
// are left, and `rows` launches the kernel for those.  p.q_heads / p.kv_heads <= 128
using WindowRows = int (*)(Launch &l, const WinParams &p, const char *name);
int run_window_tiles(Launch &l, WinParams &p, bool f16, WindowRows rows, const char *name);
int window_error_flag();

}  // namespace ab
