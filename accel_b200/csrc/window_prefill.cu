// Attention with a sliding window for many query rows of one sequence (a prompt, or a chunk of one), on
// the tensor cores of sm_100a: tcgen05 with the operands in shared and tensor memory.  What it
// computes is defined in window_attention.cu, whose row kernel does the same for few rows.
//
// Two kernels.  win_pack_kernel gathers the positions that any of the rows sees, through the page table, into
// tiles of 128 positions per KV head, as the MMAs read them (K-major 8 x 8 core matrices; V transposed),
// so that the tile kernel fetches an operand with one bulk copy, whatever the pages, strides or head
// dimension were.  win_tile_kernel takes 128 query rows (tokens x the query heads of one KV head, so the
// group shares every tile) over the tiles its rows see.
//
// Accuracy.  q, K and V have up to 24 bits and f16 holds 11, so an operand is two f16 parts, x = hi + lo,
// and a product three MMAs, lo.hi + hi.lo + hi.hi (2^-22 is dropped); an f16 cache is exact in one
// part and its products take two.  Powers of two keep the parts inside f16's range: one per query row
// and one per tile of an f32 cache; the softmax weights are carried times 2^14 (window_attention.cu).  Of an f32
// cache, a tile whose elements lie too far apart for that goes to the CUDA cores (kReach, kSpread).  With an f16 cache an element
// of a query is off by at most 2^-38 of the row's largest element, and a weight by 2^-38 of the row's largest weight.
// The accumulators of a tile start from zero, the small products first, and the sums over tiles are
// f32 additions in registers: an accumulator in the tensor core over thousands of positions would
// truncate at every step.
//
// Bound: the tensor pipe.  4 (f16 cache) or 6 (f32) MMAs of 128 x 128 x 128 for every 128 x 128 scores where
// 2 would be the floor.  A CTA of 384 threads per SM: two groups of four warps do the softmax of the even
// and the odd tiles, each with its own maximum, sum and output in registers, so that one group's
// exponentials run under the other's MMAs; one lane issues the MMAs in the order QK(0) QK(1) PV(0) QK(2)
// PV(1) ..., one lane the bulk copies, in the same order, into a ring of slots.  Tensor memory: 128 columns of
// scores and 128 of output for each group; the weights overwrite their scores.
//
// Measured, the tile kernel alone: 4096 tokens of 32 heads over windows of 2048, f16 cache, groups of 4, 225 us, which is
// 0.92 PFLOP/s of issued products (the MMAs and copies without the softmax: 196 us); 4096 tokens behind 4096 over windows of
// 4096, f32 cache, 32 heads, 695 us, 1.19 PFLOP/s issued (592 us: there the tiles from L2, 33 bytes a clock and SM).
#include <algorithm>
#include <math_constants.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "sm100.cuh"
#include "window.cuh"

namespace ab {

namespace {

constexpr int kKeys = 128;                  // positions of a tile
constexpr int kRows = 128;                  // query rows of a CTA
constexpr int kSoftWarps = 8;
constexpr int kTileThreads = kSoftWarps * 32 + 128;
constexpr int kSlots = 5;
constexpr float kBias = 14.f;               // the softmax weights are carried times 2^14

// What the pack kernel says about a tile.
struct TileHead {
    float k_scale, v_scale;                 // what the parts have to be multiplied by
    uint32_t flags;                         // kBad: a value is not finite (it is left out of the tile); kApart: see kSpread
    float k_sum;                            // an f32 cache: at least the sum of the magnitudes of any position's key
    uint32_t seen[4];                       // a bit per position: it exists
};
constexpr uint32_t kBad = 1, kApart = 2;
// An f32 tile's parts share one power of two, so an element below 2^-16 of the tile's largest is held to 2^-38 of that
// largest and not to 22 bits of its own.  Two conditions say where that is as good as f32; rows for which one fails have that
// tile's scores and values summed in f32 on the CUDA cores instead (exact_tile).
// Keys and queries: a score is off by at most 2^-38 (largest key * sum |q| + largest |q| * sum |key|) beside what 22 bits of
// every operand give; while that sum of products is below kReach the error is below 2^-22, in the exponent of a weight.
// Values: no position's and no dimension's largest magnitude (but for those that are all zero) lies more than kSpread binary
// places below the tile's largest.  What is lost is then at most 2^-24 of the largest element of the position and of the dimension.
constexpr float kReach = 65536.f;
constexpr uint32_t kSpread = 14;

// A sequence whose rows go on tiles, and the list of positions packed for it: sinks in front of the first row's window,
// then all from that on.
struct Segment {
    uint32_t row0, rows;                    // its query rows: tokens of the call
    uint32_t base, end;                     // the first row's position; the positions that may exist for any of them
    uint32_t seq;                           // its row of the page table
    uint32_t ns, lo;                        // the list: positions [0, ns) and [lo, end)
    uint32_t sink_tiles, tiles, tile0;      // tiles of 128 of them, and where they start among the call's
};
__host__ __device__ inline void segment_list(Segment &s, uint32_t window, uint32_t sinks)
{
    s.lo = (uint64_t)s.base + 1 > window ? s.base + 1 - window : 0;
    s.ns = sinks < s.lo ? sinks : s.lo;
    if (s.ns > s.end) s.ns = s.end;
    s.sink_tiles = (s.ns + kKeys - 1) / kKeys;
    s.tiles = s.sink_tiles + (s.end > s.lo ? (s.end - s.lo + kKeys - 1) / kKeys : 0);
}
// What a call's tiles are: one segment (a prefill), or those that win_plan_kernel found in a ragged step.
struct TilePlan {
    Segment one;
    const Segment *segments;                // NULL: one
    const uint4 *key_tiles;                 // {first position, end of the positions, sequence} of each
    const uint2 *row_tiles;                 // (segment, tile) of each
    const uint32_t *counts;                 // how many of either
    uint32_t max_key_tiles, max_row_tiles;
};
__device__ __forceinline__ uint32_t win_tile_start(const Segment &s, uint32_t tile)
{
    return tile < s.sink_tiles ? tile * kKeys : s.lo + (tile - s.sink_tiles) * kKeys;
}
// positions below it exist in the cache
__device__ __forceinline__ uint32_t win_end(const WinParams &p, const TilePlan &plan, const Segment &s)
{
    return plan.segments ? s.end : min(s.end, p.lengths[0]);
}

template <typename T> constexpr int kParts = sizeof(T) == 4 ? 2 : 1;
template <typename T, int DP> constexpr uint32_t kSlotBytes = kKeys * DP * 2;
template <typename T, int DP> constexpr uint32_t kTileBytes = 2 * kParts<T> * kSlotBytes<T, DP>;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

// the power of two that brings a largest magnitude into [2^13, 2^14), as an exponent
__device__ __forceinline__ int fit_exponent(float amax)
{
    const int e = amax > 0.f ? 13 - ((int)(__float_as_uint(amax) >> 23) - 127) : 0;
    return min(max(e, -126), 126);
}
__device__ __forceinline__ uint32_t pack_f16x2(float x, float y)
{
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// x = hi + lo in f16
__device__ __forceinline__ void split_f16x2(float x, float y, uint32_t &hi, uint32_t &lo)
{
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = pack_f16x2(x - f.x, y - f.y);
}
__device__ __forceinline__ void split8(const float (&x)[8], uint4 &hi, uint4 &lo)
{
    split_f16x2(x[0], x[1], hi.x, lo.x);
    split_f16x2(x[2], x[3], hi.y, lo.y);
    split_f16x2(x[4], x[5], hi.z, lo.z);
    split_f16x2(x[6], x[7], hi.w, lo.w);
}

// ------------------------------------------------------------------------------------------------
// grid (tiles, KV heads of this pass, 2): K or V of one tile.  An operand's element (r, c), c along the contraction, lies
// at (c / 8) * rows * 16 + r * 16 + (c % 8) * 2: 128 rows of positions for K, DP rows of dimensions for V.
// Every element is read once and written once per part: HBM (or L2) bounds it.
// Measured: 8192 f32 positions of 32 heads, 537 MB in 107 us (5.0 TB/s); 4096 f16 positions of 8 heads, 33.5 MB in 11.5 us,
// where the values of an f16 cache stay as they are, a copy in another order (16.3 us through f32 registers).
constexpr int kPackThreads = 512;

// Plan: a ragged step's tiles, which the CTAs take by turns; or one for each.
template <typename T, int DP, bool Plan>
__global__ void __launch_bounds__(kPackThreads, sizeof(T) == 2 ? 3 : 2)
win_pack_kernel(const WinParams p, const TilePlan plan, unsigned char *tiles, TileHead *heads, uint32_t kvh0)
{
    __shared__ uint32_t rows[kKeys], amax_bits, bad_any;
    // an f32 cache, V: the exponents of the largest magnitudes, by position (a byte for each, of every 32 dimensions) and by
    // dimension; 0 for zeros (and numbers below 2^-126)
    __shared__ uint32_t sum_bits, smallest, of_positions[kPackThreads / 32 * 8], of_dims[DP];
    if (!Plan) pdl_wait();
    pdl_trigger();                                       // the tile kernel may set itself up meanwhile
    const uint32_t kvh = kvh0 + blockIdx.y, t = threadIdx.x, D = p.head_dim, lane = t & 31;
    // elements of a thread; dimensions that it takes of V together (4 bytes of a position); groups of eight positions at a time
    constexpr int kEach = kKeys * DP / kPackThreads, kWide = sizeof(T) == 2 ? 2 : 1, kTogether = kPackThreads * kWide / DP;
    // K: eight dimensions of a position at a time; a warp takes eight positions x 32 dimensions, whole lines to read and to
    // write.  V: eight positions of kWide dimensions at a time, neighbouring threads neighbouring dimensions.
    const uint32_t dim = t % (DP / kWide) * kWide, group0 = t / (DP / kWide);
    const auto k_task = [&](int i, uint32_t &key, uint32_t &d) {
        const uint32_t task = (i / 8) * (kPackThreads / 32) + (t >> 5);            // of 16 x DP / 32
        key = task / (DP / 32) * 8 + (lane & 7);
        d = task % (DP / 32) * 32 + (lane >> 3) * 8;
    };
    const auto v_to = [&](int i) { return (i / (8 * kWide) * kTogether + group0) * (DP * 16) + (dim + i / 8 % kWide) * 16; };
    uint32_t tile = blockIdx.x;
    while (!Plan || tile < plan.counts[0]) {
        uint4 span;                                      // first position, end of the positions, sequence
        if (Plan) {
            span = plan.key_tiles[tile];
        } else {
            span.x = win_tile_start(plan.one, tile);
            span.y = min(tile < plan.one.sink_tiles ? min(plan.one.ns, plan.one.end) : plan.one.end, p.lengths[0]);
            span.z = 0;
        }
        const size_t at = (size_t)blockIdx.y * plan.max_key_tiles + tile;
        TileHead &head = heads[at];
        unsigned char *dst = tiles + at * kTileBytes<T, DP> + (blockIdx.z ? kParts<T> * kSlotBytes<T, DP> : 0);
        if (t == 0) { amax_bits = 0; bad_any = 0; }
        if constexpr (sizeof(T) == 4) {
            if (t == 0) { sum_bits = 0; smallest = 0xffffffffu; }
            if (t < DP) of_dims[t] = 0;
        }
        if (t < kKeys) {
            const uint64_t j = (uint64_t)span.x + t;
            uint32_t r = 0xffffffffu;
            if (j < span.y) r = win_cache_row(p, p.pages ? p.pages + (size_t)span.z * p.max_pages : nullptr, (uint32_t)j);
            rows[t] = r;
            const uint32_t seen = __ballot_sync(0xffffffffu, r != 0xffffffffu);
            if (blockIdx.z == 0 && (t & 31) == 0) head.seen[t >> 5] = seen;
        }
        __syncthreads();
        if constexpr (sizeof(T) == 2) {
            if (blockIdx.z == 0) {
                uint4 x[kEach / 8];
#pragma unroll
                for (int i = 0; i < kEach / 8; i++) {
                    uint32_t key, d;
                    k_task(i * 8, key, d);
                    const uint32_t r = rows[key];
                    x[i] = make_uint4(0, 0, 0, 0);
                    if (r != 0xffffffffu && d < D)
                        x[i] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.k) + ((uint64_t)r * p.kv_heads + kvh) * D + d);
                }
#pragma unroll
                for (int i = 0; i < kEach / 8; i++) {
                    uint32_t key, d;
                    k_task(i * 8, key, d);
                    *reinterpret_cast<uint4 *>(dst + d / 8 * (kKeys * 16) + key * 16) = x[i];
                }
            } else {
                const T *v = static_cast<const T *>(p.v) + (uint64_t)kvh * D + dim;
                uint32_t x[kEach / 2];
                bool bad = false;
#pragma unroll
                for (int i = 0; i < kEach / 2; i++) {
                    const uint32_t r = rows[(i / 8 * kTogether + group0) * 8 + (i & 7)];
                    x[i] = r != 0xffffffffu && dim < D ? *reinterpret_cast<const uint32_t *>(v + (uint64_t)r * p.kv_heads * D) : 0;
                }
#pragma unroll
                for (int i = 0; i < kEach / 2; i++) {    // (values that are not finite are left out: see the other case)
                    if ((x[i] & 0x7c00u) == 0x7c00u) { x[i] &= 0xffff0000u; bad = true; }
                    if ((x[i] & 0x7c000000u) == 0x7c000000u) { x[i] &= 0xffffu; bad = true; }
                }
#pragma unroll
                for (int i = 0; i < kEach / 2; i += 8) {
                    *reinterpret_cast<uint4 *>(dst + v_to(2 * i)) =
                        make_uint4(__byte_perm(x[i], x[i + 1], 0x5410), __byte_perm(x[i + 2], x[i + 3], 0x5410),
                                   __byte_perm(x[i + 4], x[i + 5], 0x5410), __byte_perm(x[i + 6], x[i + 7], 0x5410));
                    *reinterpret_cast<uint4 *>(dst + v_to(2 * i + 8)) =
                        make_uint4(__byte_perm(x[i], x[i + 1], 0x7632), __byte_perm(x[i + 2], x[i + 3], 0x7632),
                                   __byte_perm(x[i + 4], x[i + 5], 0x7632), __byte_perm(x[i + 6], x[i + 7], 0x7632));
                }
                if (__any_sync(0xffffffffu, bad) && lane == 0) bad_any = 1;
            }
            __syncthreads();
            if (t == 0) {
                if (blockIdx.z) { head.v_scale = 1.f; head.flags = bad_any ? kBad : 0; }
                else head.k_scale = 1.f;
            }
        } else {
            float x[kEach];
            if (blockIdx.z == 0) {
#pragma unroll
                for (int i = 0; i < kEach; i += 8) {
                    uint32_t key, d;
                    k_task(i, key, d);
                    const uint32_t r = rows[key];
#pragma unroll
                    for (int e = 0; e < 8; e++) x[i + e] = 0.f;
                    if (r != 0xffffffffu && d < D) {
                        const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const T *>(p.k) + ((uint64_t)r * p.kv_heads + kvh) * D + d);
                        uint4 raw[2];
                        raw[0] = src[0];
                        raw[1] = src[1];
#pragma unroll
                        for (int e = 0; e < 8; e++) x[i + e] = reinterpret_cast<const float *>(raw)[e];
                    }
                }
            } else {
                const T *v = static_cast<const T *>(p.v) + (uint64_t)kvh * D + dim;
#pragma unroll
                for (int i = 0; i < kEach; i++) {
                    const uint32_t r = rows[(i / 8 * kTogether + group0) * 8 + (i & 7)];
                    const T *src = v + (uint64_t)r * p.kv_heads * D;
                    const bool on = r != 0xffffffffu && dim < D;
                    x[i] = on ? to_f32(*src) : 0.f;
                }
            }
            // the largest magnitude, and what kReach and kSpread ask about.  Values that are not finite show in the first look (in a
            // sum; as an exponent of 255), and then a second one leaves them out
            const auto look = [&](auto finite) {
                float big = 0.f, all = 0.f;
                bool lost;
                if (blockIdx.z == 0) {
                    float sums = 0.f;
#pragma unroll
                    for (int i = 0; i < kEach; i += 8) {
                        float sum = 0.f;
#pragma unroll
                        for (int n = 0; n < 8; n++) {
                            float y = fabsf(x[i + n]);
                            if (decltype(finite)::value && !(y <= 3.402823466e38f)) y = 0.f;
                            sum += y;
                            big = fmaxf(big, y);
                        }
                        all += sum;
                        sum += __shfl_xor_sync(0xffffffffu, sum, 8);         // (a position's 32 dimensions: lanes 8 and 16 apart
                        sum += __shfl_xor_sync(0xffffffffu, sum, 16);        // have the rest)
                        sums = fmaxf(sums, sum);
                    }
                    const uint32_t c = __reduce_max_sync(0xffffffffu, __float_as_uint(sums));
                    if (lane == 0) atomicMax(&sum_bits, c);
                    lost = !(all <= 3.402823466e38f);
                } else {
                    constexpr int kWords = kEach / 4;
                    uint32_t exponents[kWords];                              // a byte a value
#pragma unroll
                    for (int i = 0; i < kEach; i += 4) {
                        uint32_t u[4];
#pragma unroll
                        for (int n = 0; n < 4; n++) {
                            big = fmaxf(big, fabsf(x[i + n]));
                            u[n] = __float_as_uint(x[i + n]) << 1;
                        }
                        exponents[i / 4] = __byte_perm(__byte_perm(u[0], u[1], 0x73), __byte_perm(u[2], u[3], 0x73), 0x5410);
                    }
                    atomicMax(&of_dims[dim], __float_as_uint(big) >> 23);
                    // the warp's 32 dimensions: lanes give away half of their words until each has one, then whole ones
                    uint32_t word = 0;                                       // which of them a lane ends with
#pragma unroll
                    for (int w = 16, n = kWords; w; w /= 2) {
                        if (n > 1) {
                            n /= 2;
                            const bool upper = (lane & w) != 0;
                            if (upper) word += n;
#pragma unroll
                            for (int j = 0; j < n; j++) {
                                const uint32_t give = upper ? exponents[j] : exponents[j + n], keep = upper ? exponents[j + n] : exponents[j];
                                exponents[j] = __vmaxu4(keep, __shfl_xor_sync(0xffffffffu, give, w));
                            }
                        } else {
                            exponents[0] = __vmaxu4(exponents[0], __shfl_xor_sync(0xffffffffu, exponents[0], w));
                        }
                    }
                    of_positions[t / 32 * 8 + word] = exponents[0];          // (the lanes that share a word write the same)
                    lost = __vcmpeq4(exponents[0], 0xffffffffu) != 0;
                }
                const uint32_t b = __reduce_max_sync(0xffffffffu, __float_as_uint(big));
                if (lane == 0) atomicMax(&amax_bits, b);
                if (__any_sync(0xffffffffu, lost) && lane == 0) bad_any = 1;
                __syncthreads();
            };
            look(std::false_type());
            if (bad_any) {
                // a value that is not finite would spoil rows that do not see it (0 * inf): it is left out here and added to
                // the rows that do by the tile kernel.  A score is masked after its product, so a key may stay
                if (blockIdx.z) {
#pragma unroll
                    for (int i = 0; i < kEach; i++)
                        if (!(fabsf(x[i]) <= 3.402823466e38f)) x[i] = 0.f;
                }
                __syncthreads();
                if (t == 0) amax_bits = sum_bits = 0;
                if (t < DP) of_dims[t] = 0;
                __syncthreads();
                look(std::true_type());
            }
            const int e = fit_exponent(__uint_as_float(amax_bits));
            if (blockIdx.z) {
                // (the DP / 32 warps that share a group's positions are neighbours)
                uint32_t m = 0;
                if (t < kKeys) {
                    const uint32_t per = kEach, from = t / per * (DP / 32), i = t % per;
#pragma unroll
                    for (int w = 0; w < DP / 32; w++) m = max(m, of_positions[(from + w) * 8 + i / 4] >> (i % 4 * 8) & 255u);
                } else if (t < kKeys + DP) {
                    m = of_dims[t - kKeys];
                }
                const uint32_t least = __reduce_min_sync(0xffffffffu, m ? m : 0xffffffffu);
                if (lane == 0 && least != 0xffffffffu) atomicMin(&smallest, least);
                __syncthreads();
            }
            if (t == 0) {
                if (blockIdx.z) {
                    // (the weights' 2^14 goes with it: the sums of an f32 cache are carried without)
                    head.v_scale = ab_pow2(-e) * (1.f / 16384.f);
                    const bool apart = smallest != 0xffffffffu && smallest + kSpread < amax_bits >> 23;
                    head.flags = (bad_any ? kBad : 0) | (apart ? kApart : 0);
                } else {
                    head.k_scale = ab_pow2(-e);
                    head.k_sum = __uint_as_float(sum_bits) * (DP / 32);
                }
            }
            const float f = ab_pow2(e);
#pragma unroll
            for (int i = 0; i < kEach; i += 8) {
                float y[8];
#pragma unroll
                for (int n = 0; n < 8; n++) y[n] = x[i + n] * f;
                uint4 hi, lo;
                split8(y, hi, lo);
                uint32_t to = v_to(i);
                if (blockIdx.z == 0) {
                    uint32_t key, d;
                    k_task(i, key, d);
                    to = d / 8 * (kKeys * 16) + key * 16;
                }
                *reinterpret_cast<uint4 *>(dst + to) = hi;
                *reinterpret_cast<uint4 *>(dst + kSlotBytes<T, DP> + to) = lo;
            }
        }
        if (!Plan) return;
        tile += gridDim.x;
        __syncthreads();
    }
    pdl_wait();                                          // beside a ragged step's rows (run_tiles): done when those are
}

// ------------------------------------------------------------------------------------------------
template <typename T, int DP> struct TileSmem {
    static constexpr uint32_t kQ = kRows * DP * 2;                  // one part of the query rows
    static constexpr uint32_t kRing = 2 * kQ;
    static constexpr uint32_t kBars = kRing + kSlots * kSlotBytes<T, DP>;
    static constexpr uint32_t kScale = kBars + 256;                 // of every query row: a power of two; its largest magnitude; the sum of all
    static constexpr uint32_t kBytes = kScale + 3 * kRows * 4;
};

// sx_bar_wait without its function call: the softmax threads hold more registers than survive one
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity)
{
    const uint32_t addr = sx_smem(bar);
    if (sx_bar_try(addr, parity)) return true;
    const long long t0 = clock64();
    while (!sx_bar_try(addr, parity))
        if (clock64() - t0 > kSxWaitCycles) {
            atomicExch(&g_sm100_error, 1);
            return false;
        }
    return true;
}
// D[tmem_d] (+)= A[smem] * B[smem]
__device__ __forceinline__ void mma_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float cut(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }
// bits [a, b) of a word, a and b clipped to it
__device__ __forceinline__ uint32_t bit_range(int a, int b)
{
    a = max(a, 0);
    b = min(b, 32);
    return a < b ? (0xffffffffu >> (32 - (b - a))) << a : 0u;
}

// scores whose bit is not set become -inf
__device__ __forceinline__ void hide(uint32_t (&s)[32], uint32_t bits)
{
#pragma unroll
    for (int e = 0; e < 32; e++) s[e] = (bits >> e) & 1 ? s[e] : 0xff800000u;
}

// The tiles that the rows at positions [pa, pb] see: [0, sinks_end) and [begin, end).
struct Range { uint32_t sinks_end, begin, end; };
__device__ __forceinline__ Range win_range(const WinParams &p, const Segment &k, uint64_t pa, uint64_t pb)
{
    const uint32_t lo = (uint32_t)(pa + 1 > p.window ? pa + 1 - p.window : 0), s = min(min(p.sinks, lo), k.end);
    Range r;
    r.sinks_end = s <= k.ns ? (s + kKeys - 1) / kKeys : k.sink_tiles + (s - k.lo + kKeys - 1) / kKeys;
    r.end = (uint32_t)min((uint64_t)k.tiles, k.sink_tiles + (pb + 1 - k.lo + kKeys - 1) / kKeys);
    r.sinks_end = min(r.sinks_end, r.end);
    r.begin = min(max(r.sinks_end, k.sink_tiles + (lo - k.lo) / kKeys), r.end);
    return r;
}

// A tile whose elements lie too far apart for two f16 parts (kReach, kSpread), in f32 on the CUDA cores: by the softmax warps,
// once the rows' outputs lie in shared memory.  The tile's keys and values are fetched as they are, behind those; a thread
// has a row, works out the scores of half of the positions (its partner in the other group the others; they meet in tensor
// memory), and then sums half of the dimensions.  2 x 128 x 128 multiply-adds a row, operands from shared memory, the same to all
// lanes.  Measured: 2048 tokens of 32 heads over windows of 2048, 8 f32 KV heads, every tile this way: 3580 us
// (231 us with ordinary numbers; one by one from global memory 44600).
template <int DP> struct ExactSmem {
    static constexpr uint32_t kRowOf = kRows * (DP + 4) * 4 + 8 * kRows * 4;          // the positions' cache rows
    static constexpr uint32_t kK = kRowOf + kKeys * 4, kV = kK + kKeys * DP * 4, kEnd = kV + kKeys * DP * 4;
};
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// all softmax threads, and what they wrote to tensor memory
__device__ __forceinline__ void soft_sync()
{
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    asm volatile("bar.sync 1, %0;" ::"n"(kSoftWarps * 32) : "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// the same barrier; does any thread say yes?
__device__ __forceinline__ bool soft_sync_or(bool x)
{
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(any) : "r"((uint32_t)x), "n"(kSoftWarps * 32) : "memory");
    return any;
}
// q_row: the thread's query row; seen, mask: the positions that exist, those that the row sees; ts: tensor memory for its scores;
// out: its half of its output, m and l: its maximum and its sum of weights
template <int DP> __device__ __forceinline__ void exact_tile(const WinParams &p, const Segment &keys, uint32_t kvh, uint32_t j0, const uint4 &seen,
                                                             const uint32_t (&mask)[4], const float *q_row, uint32_t ts, unsigned char *smem,
                                                             float *out, float &m, float &l)
{
    using Smem = ExactSmem<DP>;
    const uint32_t t = threadIdx.x, wg = t / 128, D = p.head_dim;
    uint32_t *rows = reinterpret_cast<uint32_t *>(smem + Smem::kRowOf);
    float4 *ks = reinterpret_cast<float4 *>(smem + Smem::kK), *vs = reinterpret_cast<float4 *>(smem + Smem::kV);
    const auto word = [](const uint32_t (&w)[4], int i) { return i < 2 ? (i ? w[1] : w[0]) : (i == 2 ? w[2] : w[3]); };
    const uint32_t there[4] = {seen.x, seen.y, seen.z, seen.w};
    const auto any = [&](int w) { return (word(there, w / 4) >> (w % 4 * 8)) & 255; };       // of the w-th eight positions
    soft_sync();                                         // (the tile before this one is done with)
    if (t < kKeys)
        rows[t] = (word(there, t / 32) >> (t & 31)) & 1
                      ? win_cache_row(p, p.pages ? p.pages + (size_t)keys.seq * p.max_pages : nullptr, j0 + t) : 0xffffffffu;
    soft_sync();
    for (uint32_t i = t; i < kKeys * DP / 4; i += kSoftWarps * 32) {
        const uint32_t row = rows[i / (DP / 4)], d = i % (DP / 4) * 4;
        const uint64_t at = ((uint64_t)row * p.kv_heads + kvh) * D + d;
        const bool on = row != 0xffffffffu && d < D;
        ks[i] = on ? *reinterpret_cast<const float4 *>(static_cast<const float *>(p.k) + at) : make_float4(0.f, 0.f, 0.f, 0.f);
        vs[i] = on ? *reinterpret_cast<const float4 *>(static_cast<const float *>(p.v) + at) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    soft_sync();
    {
        float4 q[DP / 4];
#pragma unroll
        for (int i = 0; i < DP / 4; i++) {
            q[i] = 4u * i < D ? *reinterpret_cast<const float4 *>(q_row + 4 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
            q[i].x *= p.scale_log2; q[i].y *= p.scale_log2; q[i].z *= p.scale_log2; q[i].w *= p.scale_log2;
        }
#pragma unroll 1
        for (int w = wg * 8; w < (int)wg * 8 + 8; w++) {
            if (!any(w)) continue;
            uint32_t s[8];
#pragma unroll 2
            for (int e = 0; e < 8; e += 4) {
                float2 x[4] = {}, y[4] = {};
#pragma unroll
                for (int i = 0; i < DP / 4; i++)
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        const float4 k = ks[(8 * w + e + n) * (DP / 4) + i];
                        x[n] = ab_fma2(make_float2(q[i].x, q[i].y), make_float2(k.x, k.y), x[n]);
                        y[n] = ab_fma2(make_float2(q[i].z, q[i].w), make_float2(k.z, k.w), y[n]);
                    }
#pragma unroll
                for (int n = 0; n < 4; n++) s[e + n] = __float_as_uint((x[n].x + x[n].y) + (y[n].x + y[n].y));
            }
            tmem_st8(ts + 8 * w, s);
        }
    }
    soft_sync();
    const auto eight = [&](int w, uint32_t (&s)[8]) {    // scores, -inf where the row does not look
        const uint32_t bits = word(mask, w / 4) >> (w % 4 * 8);
        tmem_ld8(ts + 8 * w, s);
#pragma unroll
        for (int e = 0; e < 8; e++) s[e] = (bits >> e) & 1 ? s[e] : 0xff800000u;
    };
    float top = -CUDART_INF_F;
#pragma unroll 1
    for (int w = 0; w < 16; w++) {
        if (!any(w)) continue;
        uint32_t s[8];
        eight(w, s);
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, __uint_as_float(s[e]));
    }
    const float m1 = fmaxf(m, top), ms = m1 == -CUDART_INF_F ? 0.f : m1, a = m == m1 ? 1.f : ab_ex2(m - m1);
    float sum = 0.f;
    float4 o[DP / 8];
#pragma unroll
    for (int i = 0; i < DP / 8; i++) {
        o[i] = reinterpret_cast<const float4 *>(out)[i];
        o[i].x *= a; o[i].y *= a; o[i].z *= a; o[i].w *= a;
    }
#pragma unroll 1
    for (int w = 0; w < 16; w++) {
        if (!any(w)) continue;
        uint32_t s[8];
        eight(w, s);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float x = ab_ex2(__uint_as_float(s[e]) - ms);
            sum += x;
            if (x != 0.f) {                              // (a value that is not finite stays with the rows that see it)
                const float4 *v = vs + (8 * w + e) * (DP / 4) + wg * (DP / 8);
#pragma unroll
                for (int i = 0; i < DP / 8; i++) {
                    const float4 y = v[i];
                    const float2 lo = ab_fma2(make_float2(x, x), make_float2(y.x, y.y), make_float2(o[i].x, o[i].y));
                    const float2 hi = ab_fma2(make_float2(x, x), make_float2(y.z, y.w), make_float2(o[i].z, o[i].w));
                    o[i] = make_float4(lo.x, lo.y, hi.x, hi.y);
                }
            }
        }
        __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < DP / 8; i++) reinterpret_cast<float4 *>(out)[i] = o[i];
    m = m1;
    l = fmaf(l, a, sum);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kTileThreads, 1)
win_tile_kernel(const WinParams p, const TilePlan plan, const unsigned char *tiles, const TileHead *heads, uint32_t kvh0,
                uint32_t split)
{
    using Smem = TileSmem<T, DP>;
    constexpr uint32_t kSlot = kSlotBytes<T, DP>;
    constexpr uint32_t kLboRows = kRows * 16, kLboDims = DP * 16;
    constexpr int kP = kParts<T>;
    extern __shared__ __align__(128) unsigned char smem[];
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + Smem::kBars), *freeb = full + kSlots;
    uint64_t *s_ready = freeb + kSlots, *p_ready = s_ready + 2, *d_ready = p_ready + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(d_ready + 2);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // the rows: tokens x heads of the group; the last tokens, which see most, first
    const uint32_t group = p.q_heads / p.kv_heads, per_tile = kRows / group, D = p.head_dim;
    const uint32_t index = blockIdx.x / split, part = blockIdx.x % split, kv = index / plan.max_row_tiles;
    Segment keys = plan.one;
    uint32_t rt = plan.max_row_tiles - 1 - index % plan.max_row_tiles;
    if (plan.segments) {
        const uint2 e = rt < plan.counts[1] ? plan.row_tiles[rt] : make_uint2(0xffffffffu, 0);
        if (e.x == 0xffffffffu) {
            pdl_wait();                                  // (this kernel is done when all before it is, whatever it had to do)
            return;
        }
        keys = plan.segments[e.x];
        rt = e.y;
    }
    const uint32_t first = rt * per_tile, tok0 = keys.row0 + first, tokens = min(per_tile, keys.rows - first);
    // The query rows.  A warp takes 16 of them, eight at a time, four lanes to a row: 64 bytes of each of eight rows a load.
    // All are on their way before anything else is worked out
    float4 both[2][DP / 16];
    if (warp < kSoftWarps) {
#pragma unroll
        for (int g = 0; g < 2; g++) {
            const uint32_t row = warp * 16 + g * 8 + (lane >> 2), at = (lane & 3) * 4;
            const bool on = row < tokens * group;
            const float *q = p.q + ((uint64_t)(tok0 + (on ? row / group : 0)) * p.q_heads + (kvh0 + kv) * group + (on ? row % group : 0)) * D;
#pragma unroll
            for (int i = 0; i < DP / 16; i++) {
                both[g][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (on && 16 * i + at < D)
                    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(both[g][i].x), "=f"(both[g][i].y), "=f"(both[g][i].z), "=f"(both[g][i].w) : "l"(q + 16 * i + at));
            }
        }
    }
    const uint64_t pa = (uint64_t)keys.base + first;
    const Range range = win_range(p, keys, pa, pa + tokens - 1);
    // of the tiles that they see, this CTA of the cluster takes n, from the i0-th on
    const uint32_t all = range.sinks_end + (range.end - range.begin), share = (all + split - 1) / split, i0 = min(part * share, all);
    const uint32_t n = min(share, all - i0);
    const auto tile_of = [&](uint32_t i) { return i0 + i < range.sinks_end ? i0 + i : range.begin + (i0 + i - range.sinks_end); };
    tiles += ((size_t)kv * plan.max_key_tiles + keys.tile0) * kTileBytes<T, DP>;
    heads += (size_t)kv * plan.max_key_tiles + keys.tile0;

    // The copies: parts of operands, in the order the MMAs take them: K(0) K(1) V(0) K(2) V(1) ... K(n-1) V(n-2) V(n-1)
    const uint32_t items = 2 * n * kP;
    const auto copy = [&](uint32_t i) {
        const uint32_t op = i / kP, part = i % kP, slot = i % kSlots;
        const bool key = op == 0 || ((op & 1) && op < 2 * n - 1);
        const uint32_t t = key ? (op + 1) / 2 : (op == 2 * n - 1 ? n - 1 : op / 2 - 1);
        sx_bar_expect_tx(&full[slot], kSlot);
        sx_bulk_load(smem + Smem::kRing + slot * kSlot, tiles + (size_t)tile_of(t) * kTileBytes<T, DP> + ((key ? 0 : kP) + part) * kSlot,
                     kSlot, &full[slot]);
    };
    if (warp == kSoftWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(sx_smem(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if (warp == kSoftWarps + 1 && lane == 0) {
        for (int i = 0; i < kSlots; i++) { sx_bar_init(&full[i], 1); sx_bar_init(&freeb[i], 1); }
        for (int i = 0; i < 2; i++) { sx_bar_init(&s_ready[i], 1); sx_bar_init(&p_ready[i], 4); sx_bar_init(&d_ready[i], 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        // the ring's first fill: nothing to wait for but the pack kernel
        pdl_wait();
        for (uint32_t i = 0; i < kSlots && i < items; i++) copy(i);
    }
    const uint32_t r = tid & (kRows - 1);
    const bool live = r < tokens * group;
    float *row_scale = reinterpret_cast<float *>(smem + Smem::kScale);
    // scaled, split, stored as the A operand (the stores meet every bank twice)
    if (warp < kSoftWarps) {
        const uint32_t at = (lane & 3) * 4;
#pragma unroll
        for (int g = 0; g < 2; g++) {
            const uint32_t row = warp * 16 + g * 8 + (lane >> 2);
            const float4 (&x)[DP / 16] = both[g];
            float amax = 0.f, sum = 0.f;
#pragma unroll
            for (int i = 0; i < DP / 16; i++) {
                sum += (fabsf(x[i].x) + fabsf(x[i].y)) + (fabsf(x[i].z) + fabsf(x[i].w));
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            amax = fminf(amax * fabsf(p.scale_log2), 3.402823466e38f);
            // [2^13, 2^14), as the keys: an element down to 2^-16 of the row's largest keeps all its bits, and the products (2^37 with
            // f16's largest keys) stay far inside f32.  (Near one, 2^-25 of the largest was all that the small ones were held to)
            const int e = fit_exponent(amax);
            const float f = ab_pow2(e);
            if ((lane & 3) == 0) {
                row_scale[row] = ab_pow2(-e);
                row_scale[kRows + row] = amax;
                row_scale[2 * kRows + row] = sum * fabsf(p.scale_log2);
            }
#pragma unroll
            for (int i = 0; i < DP / 16; i++) {
                uint2 hi, lo;
                split_f16x2(x[i].x * p.scale_log2 * f, x[i].y * p.scale_log2 * f, hi.x, lo.x);
                split_f16x2(x[i].z * p.scale_log2 * f, x[i].w * p.scale_log2 * f, hi.y, lo.y);
                unsigned char *to = smem + (16 * i + at) / 8 * kLboRows + row * 16 + (at & 4) * 2;
                *reinterpret_cast<uint2 *>(to) = hi;
                *reinterpret_cast<uint2 *>(to + Smem::kQ) = lo;
            }
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;

    // 168 registers a thread at launch; the softmax groups take what the other four warps do not need:
    // 2 x 128 x 224 + 128 x 56 = 384 x 168
    if (warp >= kSoftWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == kSoftWarps + 1) {
            // ---- the copies that do not fit at once
            if (lane == 0) {
                bool ok = true;
                uint32_t i = kSlots;
                for (; i < items && ok; i++) {
                    ok = bar_wait(&freeb[i % kSlots], (i / kSlots - 1) & 1);
                    if (ok) copy(i);
                }
                // nothing may be in flight when the CTA's shared memory goes to another
                const uint32_t issued = ok ? max(i, min(items, (uint32_t)kSlots)) : i - 1;
                const uint32_t last = min(issued, items);
                for (uint32_t k = last > kSlots ? last - kSlots : 0; k < last; k++) bar_wait(&full[k % kSlots], (k / kSlots) & 1);
            }
        } else if (warp == kSoftWarps) {
            // ---- the MMAs
            if (lane == 0) {
                constexpr uint32_t kS = (1u << 4) | ((kKeys >> 3) << 17) | ((kRows >> 4) << 24);
                constexpr uint32_t kO = (1u << 4) | ((uint32_t)(DP >> 3) << 17) | ((kRows >> 4) << 24);
                uint32_t slot = 0, use = 0;
                bool ok = true;
                const uint32_t q_at = sx_smem(smem), ring = sx_smem(smem + Smem::kRing);
                uint32_t at[kP], sl[kP];
                const auto take = [&]() {                           // the next operand's parts
                    for (int part = 0; part < kP && ok; part++) {
                        ok = bar_wait(&full[slot], use & 1);
                        at[part] = ring + slot * kSlot;
                        sl[part] = slot;
                        if (++slot == kSlots) { slot = 0; use++; }
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                };
                const auto scores = [&](uint32_t i) {
                    take();
                    if (!ok) return;
                    const uint32_t d = tmem + (i & 1) * 256;
                    const auto pass = [&](uint32_t q, uint32_t k, uint32_t first) {
#pragma unroll
                        for (int j = 0; j < DP / 16; j++)
                            mma_ss(d, sx_desc(q + j * 2 * kLboRows, kLboRows, 128), sx_desc(k + j * 2 * kKeys * 16, kKeys * 16, 128), kS,
                                   !(first && j == 0));
                    };
                    pass(q_at + Smem::kQ, at[0], 1);
                    if (kP == 2) { pass(q_at, at[kP - 1], 0); sx_commit(&freeb[sl[kP - 1]]); }
                    pass(q_at, at[0], 0);
                    sx_commit(&freeb[sl[0]]);
                    sx_commit(&s_ready[i & 1]);
                };
                const auto values = [&](uint32_t i) {
                    take();
                    ok = ok && bar_wait(&p_ready[i & 1], (i >> 1) & 1);
                    if (!ok) return;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t w = tmem + (i & 1) * 256, d = w + 128;
                    // 16 positions' weights: 8 columns of high parts, 8 of low ones
                    const auto pass = [&](uint32_t lo, uint32_t v, uint32_t first) {
#pragma unroll
                        for (int j = 0; j < kKeys / 16; j++)
                            sx_mma_ts(d, w + j * 16 + lo, sx_desc(v + j * 2 * kLboDims, kLboDims, 128), kO,
                                      !(first && j == 0));
                    };
                    pass(8, at[0], 1);
                    if (kP == 2) { pass(0, at[kP - 1], 0); sx_commit(&freeb[sl[kP - 1]]); }
                    pass(0, at[0], 0);
                    sx_commit(&freeb[sl[0]]);
                    sx_commit(&d_ready[i & 1]);
                };
                if (n) scores(0);
                for (uint32_t i = 0; i < n && ok; i++) {
                    if (i + 1 < n) scores(i + 1);
                    if (ok) values(i);
                }
            }
        }
    } else {
        // ---- the softmax of every other tile; a thread has a row
        pdl_wait();                                      // (for what follows of the pack kernel's)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const float q_scale = row_scale[r];
        float q_max = 0.f, q_sum = 0.f;                  // of the CTA's rows
        if constexpr (sizeof(T) == 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(row_scale + kRows + 4 * lane), y = *reinterpret_cast<const uint4 *>(row_scale + 2 * kRows + 4 * lane);
            q_max = __uint_as_float(__reduce_max_sync(0xffffffffu, max(max(x.x, x.y), max(x.z, x.w))));
            q_sum = __uint_as_float(__reduce_max_sync(0xffffffffu, max(max(y.x, y.y), max(y.z, y.w))));
        }
        float m = -CUDART_INF_F, l = 0.f, o[DP];
        uint32_t bad = 0;
        const int wg = warp >> 2;
        const uint32_t ts = tmem + wg * 256 + ((uint32_t)(warp & 3) << 21), td = ts + 128;
        const int64_t pos = (int64_t)pa + (live ? r / group : 0);
        const int64_t lo_row = pos + 1 > (int64_t)p.window ? pos + 1 - (int64_t)p.window : 0;
        bool ok = true;
#pragma unroll
        for (int i = 0; i < DP; i++) o[i] = 0.f;
        uint4 next_scale = make_uint4(0, 0, 0, 0), next_seen = next_scale;
        const auto look = [&](uint32_t i) {                         // a tile's header, a tile ahead of its use
            const TileHead *h = heads + tile_of(i);
            asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(next_scale.x), "=r"(next_scale.y), "=r"(next_scale.z), "=r"(next_scale.w) : "l"(h));
            asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4 + 16];"
                         : "=r"(next_seen.x), "=r"(next_seen.y), "=r"(next_seen.z), "=r"(next_seen.w) : "l"(h));
        };
        // do the rows take the tile in f32, after the others?
        const auto exact = [&](const uint4 &head) {
            return sizeof(T) == 4 && (!(q_sum * 16384.f * __uint_as_float(head.x) + q_max * __uint_as_float(head.w) <= kReach) || (head.z & kApart));
        };
        const auto rows_mask = [&](int64_t j0, uint32_t (&mask)[4]) {
            const int top = (int)min(max(pos - j0 + 1, (int64_t)0), (int64_t)kKeys);
            const int low = (int)min(max(lo_row - j0, (int64_t)0), (int64_t)kKeys);
            const int snk = (int)min(max((int64_t)p.sinks - j0, (int64_t)0), (int64_t)kKeys);
#pragma unroll
            for (int w = 0; w < 4; w++)
                mask[w] &= bit_range(0, top - 32 * w) & (bit_range(low - 32 * w, 32) | bit_range(0, snk - 32 * w));
        };
        if ((uint32_t)wg < n) look(wg);
        for (uint32_t i = wg; i < n; i += 2) {
            const int64_t j0 = win_tile_start(keys, tile_of(i));
            const uint32_t flags = next_scale.z;
            const float c = fmaxf(q_scale * __uint_as_float(next_scale.x), 1.2e-38f);
            float vs = __uint_as_float(next_scale.y);
            const bool later = exact(next_scale);
            bad |= (flags & kBad) | (later ? kApart : 0);
            const uint4 seen = next_seen;
            if (i + 2 < n) look(i + 2);
            // does every row of the CTA see the whole tile?
            const bool whole = !later && (seen.x & seen.y & seen.z & seen.w) == 0xffffffffu && j0 + kKeys - 1 <= (int64_t)pa &&
                               j0 + (int64_t)p.window > (int64_t)(pa + tokens - 1);
            uint32_t mask[4] = {seen.x, seen.y, seen.z, seen.w};
            if (later) {
                mask[0] = mask[1] = mask[2] = mask[3] = 0;
            } else if (!whole) {
                rows_mask(j0, mask);
            }
            const auto word = [&](int w) { return w < 2 ? (w ? mask[1] : mask[0]) : (w == 2 ? mask[2] : mask[3]); };
            ok = __all_sync(0xffffffffu, bar_wait(&s_ready[wg], (i >> 1) & 1));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float top = -CUDART_INF_F;
#pragma unroll 1
            for (int w = 0; w < 4; w++) {
                uint32_t s[32];
                tmem_ld32(ts + 32 * w, s);
                if (!whole) hide(s, word(w));
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = __uint_as_float(s[e]);
#pragma unroll
                for (int e = 4; e < 32; e++) x[e & 3] = fmaxf(x[e & 3], __uint_as_float(s[e]));
                top = fmaxf(top, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
            }
            // (rounded up to a whole number: m1 - 14 is then exact, so are the factors between maxima, and the weights of all tiles are
            // relative to the same ones.)  An f32 cache's weights are relative to their own tile's maximum, and its product is
            // brought to the row's afterwards: a tile of large values under small weights keeps its bits
            const float mt = ceilf(top * c), m1 = fmaxf(m, mt), mw = sizeof(T) == 4 ? mt : m1;
            const float ms = (mw == -CUDART_INF_F ? 0.f : mw) - kBias;
            const float a = m == m1 ? 1.f : ab_ex2(m - m1);
            const float down = sizeof(T) == 2 || mw == m1 ? 1.f : ab_ex2(mw - m1);
            m = m1;
            vs *= down;
            float2 sum = make_float2(0.f, 0.f);
            const float2 c2 = make_float2(c, c), ms2 = make_float2(-ms, -ms);
#pragma unroll 1
            for (int w = 0; w < 4; w++) {
                uint32_t s[32];
                tmem_ld32(ts + 32 * w, s);
                if (!whole) hide(s, word(w));
#pragma unroll
                for (int k = 0; k < 32; k += 16) {
                    uint32_t out[16];
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const float2 z = ab_fma2(make_float2(__uint_as_float(s[k + e]), __uint_as_float(s[k + e + 1])), c2, ms2);
                        const float2 x = make_float2(ab_ex2(z.x), ab_ex2(z.y));
                        sum = ab_add2(sum, x);
                        // the high part is cut off (11 bits), what is left of it rounded
                        const float2 h = make_float2(cut(x.x), cut(x.y)), d = ab_add2(x, make_float2(-h.x, -h.y));
                        out[e / 2] = pack_f16x2(h.x, h.y);
                        out[8 + e / 2] = pack_f16x2(d.x, d.y);
                    }
                    sx_tmem_st16(ts + 32 * w + k, out);
                }
            }
            l = fmaf(l, a, sizeof(T) == 4 ? (sum.x + sum.y) * (down * (1.f / 16384.f)) : sum.x + sum.y);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) sx_bar_arrive(&p_ready[wg]);
            ok = __all_sync(0xffffffffu, bar_wait(&d_ready[wg], (i >> 1) & 1));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int w = 0; w < DP / 32; w++) {
                uint32_t d[32];
                tmem_ld32(td + 32 * w, d);
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float2 x = make_float2(__uint_as_float(d[e]), __uint_as_float(d[e + 1]));
                    if (sizeof(T) == 4) x = ab_mul2(x, make_float2(vs, vs));
                    x = ab_fma2(make_float2(o[32 * w + e], o[32 * w + e + 1]), make_float2(a, a), x);
                    o[32 * w + e] = x.x;
                    o[32 * w + e + 1] = x.y;
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        }
        // ---- both groups' parts of a row: each gives away half of its dimensions through shared memory, finishes the other
        // half there, and whole rows go out (row stride DP + 4: 16 bytes of eight neighbouring rows meet every bank once)
        constexpr uint32_t kPitch = DP + 4;
        float *rows = reinterpret_cast<float *>(smem), *mine = rows + r * kPitch + wg * (DP / 2);
        float *give = rows + r * kPitch + (wg ^ 1) * (DP / 2), *ml = rows + kRows * kPitch + r;      // [group][m, l, bad][row]
        asm volatile("bar.sync 1, %0;" ::"n"(kSoftWarps * 32) : "memory");
#pragma unroll
        for (int i = 0; i < DP / 2; i += 4)
            *reinterpret_cast<float4 *>(give + i) = wg ? make_float4(o[i], o[i + 1], o[i + 2], o[i + 3])
                                                       : make_float4(o[DP / 2 + i], o[DP / 2 + i + 1], o[DP / 2 + i + 2], o[DP / 2 + i + 3]);
        ml[wg * 3 * kRows] = m;
        ml[(wg * 3 + 1) * kRows] = l;
        ml[(wg * 3 + 2) * kRows] = __uint_as_float(bad);
        const bool apart = soft_sync_or(bad & kApart);   // (one answer for all: what hangs on it has barriers)
        const float m0 = ml[0], m1 = ml[3 * kRows];
        float M = fmaxf(m0, m1);
        const float f0 = m0 == -CUDART_INF_F ? 0.f : ab_ex2(m0 - M), f1 = m1 == -CUDART_INF_F ? 0.f : ab_ex2(m1 - M);
        const float fm = wg ? f1 : f0, fo = wg ? f0 : f1;
#pragma unroll
        for (int i = 0; i < DP / 2; i += 4) {
            float4 x = *reinterpret_cast<float4 *>(mine + i);
            x.x = fmaf(x.x, fo, (wg ? o[DP / 2 + i] : o[i]) * fm);
            x.y = fmaf(x.y, fo, (wg ? o[DP / 2 + i + 1] : o[i + 1]) * fm);
            x.z = fmaf(x.z, fo, (wg ? o[DP / 2 + i + 2] : o[i + 2]) * fm);
            x.w = fmaf(x.w, fo, (wg ? o[DP / 2 + i + 3] : o[i + 3]) * fm);
            *reinterpret_cast<float4 *>(mine + i) = x;
        }
        float L = fmaf(ml[kRows], f0, ml[4 * kRows] * f1);
        bad |= __float_as_uint(ml[(2 + 3 * (wg ^ 1)) * kRows]);
        if constexpr (sizeof(T) == 4) {
            if (apart) {
                const uint32_t row = live ? r : 0;
                const float *q = p.q + ((uint64_t)(tok0 + row / group) * p.q_heads + (kvh0 + kv) * group + row % group) * D;
                uint32_t left = 0;                       // of 32 tiles, a lane asking about one each
                for (uint32_t i = 0; i < n; i++) {
                    if (i % 32 == 0) left = __ballot_sync(0xffffffffu, i + lane < n && exact(*reinterpret_cast<const uint4 *>(heads + tile_of(i + lane))));
                    if (!((left >> (i & 31)) & 1)) continue;
                    look(i);
                    const uint32_t j0 = win_tile_start(keys, tile_of(i));
                    uint32_t mask[4] = {next_seen.x, next_seen.y, next_seen.z, next_seen.w};
                    rows_mask(j0, mask);
                    exact_tile<DP>(p, keys, kvh0 + kv, j0, next_seen, mask, q, tmem + ((uint32_t)(warp & 3) << 21), smem, mine, M, L);
                }
            }
        }
        if (live && (bad & kBad)) {
            // values that are not finite were left out of the tiles: a row that sees one gets it added
            const uint64_t end = min((uint64_t)win_end(p, plan, keys), (uint64_t)pos + 1);
            const uint32_t *pages = p.pages ? p.pages + (size_t)keys.seq * p.max_pages : nullptr;
            for (uint32_t i = 0; i < n; i++) {
                const uint32_t tile = tile_of(i);
                if (!(heads[tile].flags & kBad)) continue;
                for (uint32_t x = 0; x < (uint32_t)kKeys; x++) {
                    const uint64_t j = (uint64_t)win_tile_start(keys, tile) + x;
                    if (!((heads[tile].seen[x >> 5] >> (x & 31)) & 1) || j >= end || (pos - (int64_t)j >= (int64_t)p.window && j >= p.sinks))
                        continue;
                    const T *v = static_cast<const T *>(p.v) +
                                 ((uint64_t)win_cache_row(p, pages, (uint32_t)j) * p.kv_heads + kvh0 + kv) * D + wg * (DP / 2);
                    for (uint32_t d = 0; d < DP / 2 && wg * (DP / 2) + d < D; d++) {
                        const float y = to_f32(v[d]);
                        if (!(fabsf(y) <= 3.402823466e38f)) mine[d] += y;
                    }
                }
            }
        }
        if (wg == 0) {
            float *total = rows + kRows * kPitch + 6 * kRows + r;      // [m, l][row]
            total[0] = M;
            total[kRows] = L;
        }
    }
    // ---- the CTAs' parts of a row, in their order, and out: a warp writes a row (two, of a head of 64) at a time
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == kSoftWarps) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    if (split > 1) cluster_sync();
    if (warp < kSoftWarps) {
        constexpr uint32_t kPitch = DP + 4, kWarpRows = kRows / kSoftWarps, kLanes = DP / 4, kTogether = 32 / kLanes;
        const float *rows = reinterpret_cast<const float *>(smem), *total = rows + kRows * kPitch + 6 * kRows;
        // a lane knows one of its warp's 16 rows: where it goes, and what each CTA's part is multiplied by
        const uint32_t mine = warp * kWarpRows + (lane & 15);
        const uint32_t to = mine < tokens * group ? (mine / group) * p.q_heads + mine % group : 0xffffffffu;
        float *out = p.out + ((uint64_t)tok0 * p.q_heads + (kvh0 + kv) * group) * D;
        const uint32_t d = lane % kLanes * 4;
        if (split == 1) {
            const float f = 1.f / total[kRows + mine];
#pragma unroll 4
            for (uint32_t i = 0; i < kWarpRows; i += kTogether) {
                const uint32_t row = i + lane / kLanes, at = __shfl_sync(0xffffffffu, to, row);
                const float g = __shfl_sync(0xffffffffu, f, row);
                const float4 x = *reinterpret_cast<const float4 *>(rows + (warp * kWarpRows + row) * kPitch + d);
                if (at != 0xffffffffu && d < D)
                    *reinterpret_cast<float4 *>(out + (uint64_t)at * D + d) = make_float4(x.x * g, x.y * g, x.z * g, x.w * g);
            }
        } else {
            // (the warp's rows are shared out too: every CTA of the cluster writes some of them)
            const auto join = [&](auto cs) {
                constexpr uint32_t S = decltype(cs)::value, kSome = kWarpRows / S;
                float m[S], l[S], M = -CUDART_INF_F, sum = 0.f;
#pragma unroll
                for (uint32_t c = 0; c < S; c++) {
                    m[c] = ld_cluster(sx_smem(total + mine), c);
                    l[c] = ld_cluster(sx_smem(total + kRows + mine), c);
                }
#pragma unroll
                for (uint32_t c = 0; c < S; c++) M = fmaxf(M, m[c]);
#pragma unroll
                for (uint32_t c = 0; c < S; c++) {
                    m[c] = m[c] == -CUDART_INF_F ? 0.f : ab_ex2(m[c] - M);
                    sum = fmaf(l[c], m[c], sum);
                }
#pragma unroll
                for (uint32_t c = 0; c < S; c++) m[c] /= sum;
#pragma unroll
                for (uint32_t i = 0; i < kSome; i += kTogether) {
                    const uint32_t row = part * kSome + i + lane / kLanes, at = __shfl_sync(0xffffffffu, to, row);
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y[S];
#pragma unroll
                    for (uint32_t c = 0; c < S; c++) y[c] = ld_cluster4(sx_smem(rows + (warp * kWarpRows + row) * kPitch + d), c);
#pragma unroll
                    for (uint32_t c = 0; c < S; c++) {
                        const float f = __shfl_sync(0xffffffffu, m[c], row);
                        x.x = fmaf(y[c].x, f, x.x); x.y = fmaf(y[c].y, f, x.y); x.z = fmaf(y[c].z, f, x.z); x.w = fmaf(y[c].w, f, x.w);
                    }
                    if (at != 0xffffffffu && d < D) *reinterpret_cast<float4 *>(out + (uint64_t)at * D + d) = x;
                }
            };
            if (split == 2) join(std::integral_constant<uint32_t, 2>());
            else if (split == 4) join(std::integral_constant<uint32_t, 4>());
            else join(std::integral_constant<uint32_t, 8>());
        }
    }
    if (split > 1) cluster_sync();                       // nobody leaves while its parts are being read
}

template <typename T, int DP> int tile_prepare(const char *name)
{
    static std::mutex mu;
    static uint64_t done[4];                             // a bit per device
    int dev = 0;
    cudaGetDevice(&dev);
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 0 && dev < 256 && (done[dev / 64] >> (dev % 64) & 1)) return AB_OK;
    const int rc = check_cuda(cudaFuncSetAttribute(win_tile_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   TileSmem<T, DP>::kBytes), name);
    if (rc == AB_OK && dev >= 0 && dev < 256) done[dev / 64] |= 1ull << (dev % 64);
    return rc;
}

// ------------------------------------------------------------------------------------------------
// A ragged step: the sequences whose rows pay for tiles (on_tiles) become segments, as many of the first as there is room
// for; the rows of the others, and those behind the last sequence, are left to the row kernel (WinParams::left).  One block.
__global__ void __launch_bounds__(256) win_plan_kernel(const WinParams p, uint32_t max_segments, Segment *segments,
                                                       uint4 *key_tiles, uint2 *row_tiles, uint32_t *counts, uint32_t max_key_tiles,
                                                       uint32_t max_row_tiles, uint4 *left)
{
    __shared__ uint4 part[8];
    __shared__ uint32_t part_left[8];
    const uint32_t t = threadIdx.x, lane = t & 31, group = p.q_heads / p.kv_heads, per_tile = kRows / group;
    pdl_enter();                                         // (the rows' kernel may come and wait)
    uint4 before = make_uint4(0, 0, 0, 0);               // segments, key tiles, row tiles, rows left of the sequences so far
    for (uint32_t s0 = 0; s0 < p.batch; s0 += 256) {
        const uint32_t s = s0 + t;
        Segment g{};
        uint4 mine = make_uint4(0, 0, 0, 0);
        uint32_t first = 0, len = 0, count = 0, mine_left = 0;
        if (s < p.batch) {
            const uint32_t a = min(p.offsets[s], p.rows), b = min(p.offsets[s + 1], p.rows);
            len = p.lengths[s];
            first = a;
            count = p.offsets[s + 1] - p.offsets[s];
            mine_left = b > a ? b - a : 0;
            // (a sequence with more tokens than positions has rows of zeros: the row kernel knows)
            if (b > a && b == p.offsets[s + 1] && len >= b - a &&
                on_tiles((uint64_t)(b - a) * group, min((uint64_t)p.window + p.sinks, (uint64_t)min(len, p.reach)), p.kv_heads)) {
                g.row0 = a; g.rows = b - a; g.base = len - (b - a); g.seq = s;
                g.end = min(len, p.reach);
                segment_list(g, p.window, p.sinks);
                mine = make_uint4(1, g.tiles, (g.rows + per_tile - 1) / per_tile, 0);
            }
        }
        uint4 sum = mine;                                // inclusive scan over the warp, then over the warps
#pragma unroll
        for (int w = 1; w < 32; w *= 2) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, sum.x, w), y = __shfl_up_sync(0xffffffffu, sum.y, w),
                           z = __shfl_up_sync(0xffffffffu, sum.z, w);
            if (lane >= (uint32_t)w) { sum.x += x; sum.y += y; sum.z += z; }
        }
        if (lane == 31) part[t >> 5] = sum;
        __syncthreads();
        uint4 at = before;
        for (uint32_t w = 0; w < 8; w++) {
            if (w < t >> 5) { at.x += part[w].x; at.y += part[w].y; at.z += part[w].z; }
            before.x += part[w].x; before.y += part[w].y; before.z += part[w].z;
        }
        at.x += sum.x - mine.x; at.y += sum.y - mine.y; at.z += sum.z - mine.z;
        // (once one does not fit none behind it does: the sums go on)
        if (mine.x && at.x < max_segments && (uint64_t)at.y + mine.y <= max_key_tiles && (uint64_t)at.z + mine.z <= max_row_tiles) {
            mine_left = 0;
            g.tile0 = at.y;
            segments[at.x] = g;
            for (uint32_t i = 0; i < mine.y; i++)
                key_tiles[at.y + i] = make_uint4(win_tile_start(g, i), i < g.sink_tiles ? g.ns : g.end, s, 0);
            for (uint32_t i = 0; i < mine.z; i++) row_tiles[at.z + i] = make_uint2(at.x, i);
        } else if (mine.x) {
            for (uint32_t i = at.y; i < max_key_tiles && i - at.y < mine.y; i++) key_tiles[i] = make_uint4(0, 0, 0, 0);
            for (uint32_t i = at.z; i < max_row_tiles && i - at.z < mine.z; i++) row_tiles[i] = make_uint2(0xffffffffu, 0);
        }
        uint32_t sum_left = mine_left;
#pragma unroll
        for (int w = 1; w < 32; w *= 2) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, sum_left, w);
            if (lane >= (uint32_t)w) sum_left += x;
        }
        if (lane == 31) part_left[t >> 5] = sum_left;
        __syncthreads();
        uint32_t at_left = before.w + sum_left - mine_left;
        for (uint32_t w = 0; w < 8; w++) {
            if (w < t >> 5) at_left += part_left[w];
            before.w += part_left[w];
        }
        for (uint32_t i = 0; i < mine_left && at_left + i < p.rows; i++) {
            // (the first tokens of a sequence with fewer positions than tokens have none)
            const uint64_t pos1 = (uint64_t)len + i + 1;
            left[1 + at_left + i] = make_uint4(first + i, pos1 > count ? s : 0xffffffffu, (uint32_t)(pos1 - count), len);
        }
        __syncthreads();
    }
    const uint32_t end = min(p.offsets[p.batch], p.rows);
    for (uint32_t i = end + t; i < p.rows && before.w + (i - end) < p.rows; i += 256) left[1 + before.w + (i - end)] = make_uint4(i, 0xffffffffu, 0, 0);
    if (t == 0) left[0] = make_uint4(min(before.w + (p.rows - end), p.rows), 0, 0, 0);
    if (t == 0) { counts[0] = min(before.y, max_key_tiles); counts[1] = min(before.z, max_row_tiles); }
}

constexpr uint64_t kPassBytes = 1ull << 30;              // tiles of one pass over KV heads; a prefill takes more where one head's list does

template <typename T, int DP> int run_tiles(Launch &l, WinParams &p, WindowRows rows_kernel, const char *name)
{
    static_assert(TileSmem<T, DP>::kBytes <= 232448, "shared memory of a CTA");
    static_assert(kRows * (DP + 4) * 4 + 8 * kRows * 4 <= TileSmem<T, DP>::kBars, "the parts of all groups fit where the operands were");
    static_assert(ExactSmem<DP>::kEnd <= TileSmem<T, DP>::kBars, "and a tile in f32 behind them");
    const uint32_t group = p.q_heads / p.kv_heads, per_tile = kRows / group;
    const bool ragged = p.form == kRaggedStep;
    TilePlan plan{};
    uint64_t key_tiles, row_tiles, segments = 0;
    if (ragged) {
        // at most: a segment has kTileFrom rows; its list ends in two unfilled tiles, its rows in one
        segments = std::min<uint64_t>(p.batch, (uint64_t)p.rows * group / kTileFrom);
        key_tiles = segments * ((uint64_t)std::min(p.sinks, p.reach) / kKeys + std::min<uint64_t>(p.window, p.reach) / kKeys + 3) + p.rows / kKeys;
        key_tiles = std::min<uint64_t>(key_tiles, kPassBytes / kTileBytes<T, DP>);      // (long lists: the plan stops where they are full)
        row_tiles = segments + p.rows / per_tile;
    } else {
        plan.one.rows = p.rows;
        plan.one.base = p.base;
        plan.one.end = (uint32_t)std::min<uint64_t>((uint64_t)p.base + p.rows, p.reach);
        segment_list(plan.one, p.window, p.sinks);
        key_tiles = plan.one.tiles;
        row_tiles = (p.rows + per_tile - 1) / per_tile;
    }
    const uint64_t per_head = std::max<uint64_t>(1, key_tiles) * kTileBytes<T, DP>;
    const uint32_t pass = (uint32_t)std::min<uint64_t>(p.kv_heads, std::max<uint64_t>(1, kPassBytes / per_head));
    const size_t head_bytes = align_up((size_t)(pass * key_tiles) * sizeof(TileHead), 256);
    const size_t seg_bytes = align_up((size_t)segments * sizeof(Segment), 256), key_bytes = ragged ? align_up((size_t)key_tiles * 16, 256) : 0;
    const size_t row_bytes = ragged ? align_up((size_t)row_tiles * 8, 256) : 0, left_bytes = ragged ? align_up((size_t)p.rows * 16 + 32, 256) : 0;
    l.ws_need = seg_bytes + key_bytes + row_bytes + left_bytes + head_bytes + (size_t)(pass * per_head);
    if (row_tiles * pass > 0x7fffffffull || key_tiles > 0x7fffffffull || pass > 65535)
        return fail(AB_ERR_INVALID, "%s: %u rows of %u heads", name, p.rows, p.q_heads);
    if (l.query_ws) return AB_OK;
    if (l.ws_need > l.ws_bytes || !l.ws)
        return fail(AB_ERR_INVALID, "%s: needs %zu bytes of workspace, given %zu", name, l.ws_need, l.ws_bytes);
    int rc = tile_prepare<T, DP>(name);
    if (rc) return rc;
    unsigned char *ws = static_cast<unsigned char *>(l.ws);
    plan.max_key_tiles = (uint32_t)key_tiles;
    plan.max_row_tiles = (uint32_t)row_tiles;
    if (ragged) {
        Segment *segs = reinterpret_cast<Segment *>(ws);
        uint4 *kt = reinterpret_cast<uint4 *>(ws + seg_bytes);
        uint2 *rt = reinterpret_cast<uint2 *>(ws + seg_bytes + key_bytes);
        uint32_t *counts = reinterpret_cast<uint32_t *>(ws + seg_bytes + key_bytes + row_bytes);
        plan.segments = segs;
        plan.key_tiles = kt;
        plan.row_tiles = rt;
        plan.counts = counts;
        uint4 *left = reinterpret_cast<uint4 *>(counts + 4);
        p.left = left;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(1);
        cfg.blockDim = dim3(256);
        cfg.stream = l.stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, win_plan_kernel, p, (uint32_t)segments, segs, kt, rt, counts, plan.max_key_tiles,
                                                 plan.max_row_tiles, left);
        count_launch();
        rc = check_cuda(e, name);
        if (rc == AB_OK) rc = rows_kernel(l, p, name);
        if (rc) return rc;
    }
    // few row tiles: a cluster shares the positions of each, as long as all CTAs run at once and have four tiles or more.
    // (8 KV heads, groups of 4, f32, with its packing: 64 tokens that see 1024 positions 30.6 us split, 40.5 whole, 40.2 split
    // without the limit of four tiles; 64 tokens that see 300 21.3, 21.5 and 34.5 us; 32 tokens of one KV head that see 16384
    // 57.3 us split over eight, 304 whole)
    uint32_t split = 1;
    {
        const uint64_t ctas = (ragged ? p.rows / per_tile + 1 : row_tiles) * pass;
        const uint64_t seen = std::min<uint64_t>((uint64_t)std::min(p.window, p.reach) + per_tile + p.sinks, ragged ? p.reach : plan.one.end) / kKeys;
        while (split < 8 && ctas * split * 2 <= (uint64_t)sm_count() && seen >= (uint64_t)split * 2 * 4) split *= 2;
    }
    if (row_tiles * pass * split > 0x7fffffffull) return fail(AB_ERR_INVALID, "%s: %u rows of %u heads", name, p.rows, p.q_heads);
    TileHead *heads = reinterpret_cast<TileHead *>(ws + seg_bytes + key_bytes + row_bytes + left_bytes);
    unsigned char *tiles = reinterpret_cast<unsigned char *>(heads) + head_bytes;
    for (uint32_t h = 0; h < p.kv_heads && row_tiles; h += pass) {
        const uint32_t now = std::min(pass, p.kv_heads - h);
        // A ragged step's rows left run beside the packing, which waits for them at its end: it is their programmatic dependent,
        // and they let it start once the plan, which both read, is complete.  Its grid is two rounds of CTAs, which take what tiles there are by
        // turns (the bound on their number is many times that).  8 single tokens and 4 chunks of 64 over windows of 1024, f16:
        // rows 19 and packing 21 us one after the other, 29 us together
        if (key_tiles) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3((uint32_t)(ragged ? std::min<uint64_t>(key_tiles, (uint64_t)sm_count() * (sizeof(T) == 2 ? 3 : 2) / now + 1) : key_tiles), now, 2);
            cfg.blockDim = dim3(kPackThreads);
            cfg.stream = l.stream;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[0].val.programmaticStreamSerializationAllowed = 1;
            cfg.attrs = attr;
            cfg.numAttrs = !ragged || h == 0 ? 1 : 0;
            const cudaError_t e = cudaLaunchKernelEx(&cfg, ragged ? win_pack_kernel<T, DP, true> : win_pack_kernel<T, DP, false>, p, plan, tiles, heads, h);
            count_launch();
            rc = check_cuda(e, name);
            if (rc) return rc;
        }
        // a programmatic dependent of the pack kernel: its set-up and query rows (which no kernel of this call writes) overlap it;
        // a plan was complete before the packing began
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((uint32_t)row_tiles * now * split);
        cfg.blockDim = dim3(kTileThreads);
        cfg.dynamicSmemBytes = TileSmem<T, DP>::kBytes;
        cfg.stream = l.stream;
        cudaLaunchAttribute attr[2];
        cfg.attrs = attr;
        if (key_tiles) {
            attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
        }
        if (split > 1) {
            attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
            attr[cfg.numAttrs].val.clusterDim.x = split;
            attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
            cfg.numAttrs++;
        }
        const cudaError_t e = cudaLaunchKernelEx(&cfg, win_tile_kernel<T, DP>, p, plan, static_cast<const unsigned char *>(tiles),
                                                 static_cast<const TileHead *>(heads), h, split);
        count_launch();
        rc = check_cuda(e, name);
        if (rc) return rc;
    }
    note_selection("%s: tcgen05 tiles, up to %u tiles of 128 positions and %u of 128 rows, split over %u CTA(s), %u pass(es)", name,
                   plan.max_key_tiles, plan.max_row_tiles, split, (p.kv_heads + pass - 1) / pass);
    return AB_OK;
}

}  // namespace

int run_window_tiles(Launch &l, WinParams &p, bool f16, WindowRows rows, const char *name)
{
    if (f16) return p.head_dim <= 64 ? run_tiles<__half, 64>(l, p, rows, name) : run_tiles<__half, 128>(l, p, rows, name);
    return p.head_dim <= 64 ? run_tiles<float, 64>(l, p, rows, name) : run_tiles<float, 128>(l, p, rows, name);
}

int window_error_flag()
{
    int v = 0;
    return cudaMemcpyFromSymbol(&v, g_sm100_error, sizeof v) == cudaSuccess ? v : -1;
}

}  // namespace ab
