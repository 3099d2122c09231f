// Attention with a sliding window and sink positions, over the same caches and in the same forms as
// attention.cu: one token over a contiguous cache, a batch of single tokens, a ragged step, and a
// causal prefill (contiguous or paged).  No counterpart in the reference.
//
// A query at position p sees the positions j < hi = min(p + 1, length, reach) with
//
//     j >= lo = max(p + 1 - Window, 0)    or    j < Sinks,
//
// which is one list of ns = min(Sinks, lo, hi) sinks followed by [lo, hi):
//
//     position(i) = i < ns ? i : lo + (i - ns),   i < n = ns + max(hi - lo, 0)
//
//     out = sum_i softmax(Scale * q . k_position(i)) v_position(i)
//
// A length past the page table's reach is cut to it, the window is still measured from p.
// Nothing outside the list is read, so page-table entries of pages wholly outside it may hold
// anything (a pool that frees the pages behind the window leaves 0xffffffff there).  A visible
// position whose page lies outside the cache is left out as if it were masked.  A row that sees
// nothing is 0/0 = NaN, as in attention.cu; ragged padding rows are zeros.
#include <algorithm>
#include <math_constants.h>

#include <mutex>

#include "common.cuh"
#include "window.cuh"

namespace ab {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// What one query row sees.
struct WinView {
    const uint32_t *pages;
    uint32_t lo, ns, n;
    bool zero;                                     // a ragged padding row: written as zeros
};

__device__ __forceinline__ WinView win_view(const WinParams &p, uint32_t &row)
{
    WinView w{p.pages, 0, 0, 0, false};
    uint64_t pos1;                                 // the row's position + 1
    uint32_t len;
    if (p.left) {
        const uint4 e = p.left[1 + row];           // row, sequence, position + 1, length
        row = e.x;
        if (e.y == 0xffffffffu) { w.zero = true; return w; }
        pos1 = e.z;
        len = min(e.w, p.reach);
        w.pages = p.pages + (size_t)e.y * p.max_pages;
    } else if (p.form == kRaggedStep) {
        // the sequence whose [offsets[s], offsets[s + 1]) holds the row; empty sequences hold none
        uint32_t a = 0, b = p.batch;
        while (a < b) {
            const uint32_t m = (a + b) / 2;
            if (p.offsets[m + 1] <= row) a = m + 1; else b = m;
        }
        if (a >= p.batch) { w.zero = true; return w; }
        const uint32_t i = row - p.offsets[a], n = p.offsets[a + 1] - p.offsets[a];
        len = p.lengths[a];
        if ((uint64_t)len + i < n) { w.zero = true; return w; }
        pos1 = (uint64_t)len + i - n + 1;
        w.pages = p.pages + (size_t)a * p.max_pages;
        len = min(len, p.reach);
    } else if (p.form == kPrefillRows) {
        pos1 = (uint64_t)p.base + row + 1;
        len = min(p.lengths[0], p.reach);
    } else {
        // a single token is its sequence's last position
        pos1 = p.lengths[p.form == kBatch ? row : 0];
        len = (uint32_t)min(pos1, (uint64_t)p.reach);
        if (p.form == kBatch) w.pages = p.pages + (size_t)row * p.max_pages;
    }
    const uint32_t hi = (uint32_t)min(pos1, (uint64_t)len);
    const uint64_t lo64 = pos1 > p.window ? pos1 - p.window : 0;
    w.lo = (uint32_t)min(lo64, (uint64_t)0xffffffffu);
    w.ns = min(min(p.sinks, w.lo), hi);
    w.n = w.ns + (hi > w.lo ? hi - w.lo : 0u);
    return w;
}

// The rows of a launch: all of the call's, or those that are left beside tiles.
__device__ __forceinline__ uint32_t win_rows(const WinParams &p) { return p.left ? p.left[0].x : p.rows; }

// The list's entry i: its position; the page that holds it (loaded now, looked at later: a page's number is asked for
// two tiles ahead of its rows, so that nothing waits for the table); its cache row, 0xffffffff where that page lies outside
// the cache.
__device__ __forceinline__ uint32_t win_position(const WinView &w, uint32_t i) { return i < w.ns ? i : w.lo + (i - w.ns); }
__device__ __forceinline__ uint32_t win_page(const WinParams &p, const WinView &w, uint32_t i)
{
    uint32_t pg = 0xffffffffu;
    if (i < w.n && w.pages)
        asm volatile("ld.global.u32 %0, [%1];" : "=r"(pg) : "l"(w.pages + win_position(w, i) / p.block));
    return pg;
}
__device__ __forceinline__ uint32_t win_row(const WinParams &p, const WinView &w, uint32_t i, uint32_t page)
{
    if (i >= w.n) return 0xffffffffu;
    const uint32_t j = win_position(w, i);
    const uint64_t r = w.pages ? (uint64_t)page * p.block + j % p.block : j;
    return r < p.capacity ? (uint32_t)r : 0xffffffffu;
}

// ------------------------------------------------------------------------------------------------
// The row kernel: a few query heads against one list of positions.
//
// A cluster of CTAs takes one (row, KV head, up to eight of its query heads); every warp takes tiles of 16
// positions of the list in turn, with the heads as the 8-wide dimension of mma.sync:
//     S^T[16 positions x 8 heads] = K Q^T,      O^T[dims x 8 heads] += V^T P^T
// and a running maximum and sum per warp; the warps are joined through shared memory and the CTAs of the
// cluster through distributed shared memory, in a fixed order, so one launch does it all without a
// workspace and repeats its bits.  HBM bounds it: the list is read once for up to eight heads of a group.  (An f32 cache with
// groups above four is bound by splitting its operands instead: see the lane kernel.)
//
// The products keep f32 accuracy.  An operand is held as a high and a low part of 11 bits each (tf32 for
// an f32 cache, f16 for an f16 cache, whose K and V are exact in one part); the product of the two low
// parts, 2^-22, is dropped.  (f16 has fewer exponents: QFrag, kWeightBias.)  Every tile's products start from zero and the smaller ones come first; the
// sums over tiles are f32 additions outside the tensor core.
//
// Measured: 32 rows over up to 4112 f16 positions of 8 KV heads, groups of 4, 536 MB: 96 to 99 us, 5.5 TB/s.
// ------------------------------------------------------------------------------------------------
constexpr int kRowWarps = 4;
constexpr int kTile = 16;
// an f16 cache's weights are carried times 2^14: the low part of a small one would otherwise meet f16's
// smallest step; they are at most 1, and the quotient by their sum does not change.  One below 2^-17 of the largest so far is off
// by 2^-39 of that
constexpr float kWeightBias = 14.f;

// Row strides of the tiles in shared memory, in bytes: f32 K is read as 16 bytes of two neighbouring rows by a quarter
// warp (stride = 64 mod 128), f32 V as 32 bytes of four (32 mod 128), f16 by ldmatrix as 16 bytes of eight (16 mod 128).
template <typename T, int DP> struct RowTile {
    static constexpr int kRow = DP * (int)sizeof(T);
    static constexpr int kStrideK = sizeof(T) == 4 ? kRow + 64 : kRow + 16;
    static constexpr int kStrideV = sizeof(T) == 4 ? kRow + 32 : kRow + 16;
    static constexpr int kBytesK = kTile * kStrideK, kBytesV = kTile * kStrideV;
    static constexpr int kWarpBytes = kBytesK + kBytesV;
    static constexpr int kMergeBytes = kRowWarps * 8 * (DP + 2) * 4 + 8 * (DP + 2) * 4;
    static constexpr int kSmem = kRowWarps * kWarpBytes > kMergeBytes ? kRowWarps * kWarpBytes : kMergeBytes;
};

__device__ __forceinline__ void cp16(uint32_t smem, const void *gmem, bool on)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float4 lds128(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
// x = hi + lo with hi of 11 bits.  Cut off (K and V, two instructions): the low part is exact and keeps the sign of x.
// Rounded (q and the weights): the low part has either sign, so the dropped product of two low parts averages out.
__device__ __forceinline__ void cut_tf32(float x, uint32_t &hi, uint32_t &lo)
{
    hi = __float_as_uint(x) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void round_tf32(float x, uint32_t &hi, uint32_t &lo)
{
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void round_f16x2(float x, float y, uint32_t &hi, uint32_t &lo)
{
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// A group of query heads in the B fragments of S^T = K Q^T, with Scale * log2(e) applied; column g = lane / 4.
template <typename T, int DP> struct QFrag;
template <int DP> struct QFrag<float, DP> {
    uint32_t hi[DP / 4], lo[DP / 4];
    // of every 16 dimensions a thread holds four neighbouring ones of K and of q: the order of a sum's terms is free
    __device__ __forceinline__ void load(const float *q, bool on, uint32_t D, int t, float scale, float (&undo)[2])
    {
#pragma unroll
        for (int j = 0; j < DP / 16; j++) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (on && (uint32_t)(16 * j + 4 * t) < D) x = *reinterpret_cast<const float4 *>(q + 16 * j + 4 * t);
            round_tf32(x.x * scale, hi[4 * j], lo[4 * j]);
            round_tf32(x.y * scale, hi[4 * j + 1], lo[4 * j + 1]);
            round_tf32(x.z * scale, hi[4 * j + 2], lo[4 * j + 2]);
            round_tf32(x.w * scale, hi[4 * j + 3], lo[4 * j + 3]);
        }
        undo[0] = undo[1] = 1.f;
    }
};
template <int DP> struct QFrag<__half, DP> {
    uint32_t hi[DP / 8], lo[DP / 8];
    // f16 has 5 bits of exponent: a head's q is scaled by a power of two that brings its largest element into [2^13, 2^14),
    // so that one of 2^-16 of it still keeps 22 bits in its two parts, and one below that 2^-38 of the largest.  (The sums stay
    // below 2^38.  Near one instead, the channels of a query at a thousandth of its largest would keep 15 bits)
    __device__ __forceinline__ void load(const float *q, bool on, uint32_t D, int t, float scale, float (&undo)[2])
    {
        float2 x[DP / 8];
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < DP / 8; j++) {
            x[j] = make_float2(0.f, 0.f);
            if (on && (uint32_t)(8 * j + 2 * t) < D) x[j] = *reinterpret_cast<const float2 *>(q + 8 * j + 2 * t);
            x[j].x *= scale;
            x[j].y *= scale;
            amax = fmaxf(amax, fmaxf(fabsf(x[j].x), fabsf(x[j].y)));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127 - 13, -126), 113);
#pragma unroll
        for (int j = 0; j < DP / 8; j++) round_f16x2(x[j].x * ab_pow2(-e), x[j].y * ab_pow2(-e), hi[j], lo[j]);
        const float back = ab_pow2(e);
        undo[0] = __shfl_sync(0xffffffffu, back, 8 * t);            // columns 2t and 2t + 1 are held by lanes 8t and 8t + 4
        undo[1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
    }
};

template <typename T, int DP> struct RowMath;
template <int DP> struct RowMath<float, DP> {
    static __device__ __forceinline__ void scores(const QFrag<float, DP> &q, uint32_t k, int g, int t, float (&s)[4])
    {
        float small[2][4] = {}, big[2][4] = {};
        const uint32_t r0 = k + g * RowTile<float, DP>::kStrideK + t * 16, r1 = r0 + 8 * RowTile<float, DP>::kStrideK;
#pragma unroll
        for (int j = 0; j < DP / 16; j++) {
            const float4 x = lds128(r0 + 64 * j), y = lds128(r1 + 64 * j);
            uint32_t h[4], l[4];
            cut_tf32(x.x, h[0], l[0]); cut_tf32(y.x, h[1], l[1]); cut_tf32(x.y, h[2], l[2]); cut_tf32(y.y, h[3], l[3]);
            mma_tf32(small[0], l, q.hi[4 * j], q.hi[4 * j + 1]);
            mma_tf32(small[1], h, q.lo[4 * j], q.lo[4 * j + 1]);
            mma_tf32(big[0], h, q.hi[4 * j], q.hi[4 * j + 1]);
            cut_tf32(x.z, h[0], l[0]); cut_tf32(y.z, h[1], l[1]); cut_tf32(x.w, h[2], l[2]); cut_tf32(y.w, h[3], l[3]);
            mma_tf32(small[0], l, q.hi[4 * j + 2], q.hi[4 * j + 3]);
            mma_tf32(small[1], h, q.lo[4 * j + 2], q.lo[4 * j + 3]);
            mma_tf32(big[1], h, q.hi[4 * j + 2], q.hi[4 * j + 3]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = (small[0][i] + small[1][i]) + (big[0][i] + big[1][i]);
    }
    // o[dims] = o * alpha + V^T P^T; the 16 positions as 2 x 8 with a thread on t, t + 4 | t + 8, t + 12
    static __device__ __forceinline__ void values(const float (&p)[4], uint32_t v, int g, int t, int lane, const float (&a)[2],
                                                  float (&o)[DP / 16][4])
    {
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {                               // weight of (position t + 4 i, column g)
            const int from = ((t + 4 * i) & 7) * 4 + (g >> 1);
            const float even = __shfl_sync(0xffffffffu, p[(i >> 1) * 2], from), odd = __shfl_sync(0xffffffffu, p[(i >> 1) * 2 + 1], from);
            round_tf32((g & 1) ? odd : even, ph[i], pl[i]);
        }
        const uint32_t row = v + t * RowTile<float, DP>::kStrideV + g * 16;
#pragma unroll
        for (int jj = 0; jj < DP / 32; jj++) {
            float x[4][4];                                          // [position t + 4 i][dimension 32 jj + 4 g + e]
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float4 y = lds128(row + 4 * i * RowTile<float, DP>::kStrideV + 128 * jj);
                x[i][0] = y.x; x[i][1] = y.y; x[i][2] = y.z; x[i][3] = y.w;
            }
#pragma unroll
            for (int m = 0; m < 2; m++) {                           // rows g and g + 8 of an MMA are elements 2 m and 2 m + 1
                float small[4] = {}, big[4] = {};
                uint32_t h[2][4], l[2][4];
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    cut_tf32(x[2 * ks][2 * m], h[ks][0], l[ks][0]);
                    cut_tf32(x[2 * ks][2 * m + 1], h[ks][1], l[ks][1]);
                    cut_tf32(x[2 * ks + 1][2 * m], h[ks][2], l[ks][2]);
                    cut_tf32(x[2 * ks + 1][2 * m + 1], h[ks][3], l[ks][3]);
                    mma_tf32(small, l[ks], ph[2 * ks], ph[2 * ks + 1]);
                    mma_tf32(small, h[ks], pl[2 * ks], pl[2 * ks + 1]);
                    mma_tf32(big, h[ks], ph[2 * ks], ph[2 * ks + 1]);
                }
                float (&d)[4] = o[2 * jj + m];
#pragma unroll
                for (int i = 0; i < 4; i++) d[i] = fmaf(d[i], a[i & 1], small[i] + big[i]);
            }
        }
    }
    // the dimension of o[m][i]
    static __device__ __forceinline__ int dim(int m, int i, int g) { return 32 * (m >> 1) + 4 * g + 2 * (m & 1) + (i >> 1); }
};
template <int DP> struct RowMath<__half, DP> {
    static __device__ __forceinline__ void scores(const QFrag<__half, DP> &q, uint32_t k, int, int, float (&s)[4])
    {
        const int lane = threadIdx.x & 31;
        float small[4] = {}, big[2][4] = {};
        const uint32_t at = k + (lane & 15) * RowTile<__half, DP>::kStrideK + (lane >> 4) * 16;
#pragma unroll
        for (int j = 0; j < DP / 16; j++) {
            uint32_t a[4];
            ldsm4(a, at + 32 * j);
            mma_f16(small, a, q.lo[2 * j], q.lo[2 * j + 1]);
            mma_f16(big[j & 1], a, q.hi[2 * j], q.hi[2 * j + 1]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = small[i] + (big[0][i] + big[1][i]);
    }
    static __device__ __forceinline__ void values(const float (&p)[4], uint32_t v, int, int, int lane, const float (&a)[2],
                                                  float (&o)[DP / 16][4])
    {
        uint32_t h0, l0, h1, l1;
        round_f16x2(p[0], p[1], h0, l0);
        round_f16x2(p[2], p[3], h1, l1);
        h0 = transpose8x8(h0); l0 = transpose8x8(l0); h1 = transpose8x8(h1); l1 = transpose8x8(l1);
        const uint32_t at = v + ((lane & 7) + ((lane >> 4) & 1) * 8) * RowTile<__half, DP>::kStrideV + ((lane >> 3) & 1) * 16;
#pragma unroll
        for (int m = 0; m < DP / 16; m++) {
            uint32_t x[4];
            float c[4] = {};
            ldsm4_t(x, at + 32 * m);
            mma_f16(c, x, l0, l1);
            mma_f16(c, x, h0, h1);
#pragma unroll
            for (int i = 0; i < 4; i++) o[m][i] = fmaf(o[m][i], a[i & 1], c[i]);
        }
    }
    static __device__ __forceinline__ int dim(int m, int i, int g) { return 16 * m + g + 8 * (i >> 1); }
};

// The parts of a row's heads, one per warp (or group of lanes), then one per CTA of the cluster, joined in their order:
// [part][maxima of C columns, sums of C columns] and [part][C][DP] in shared memory, the CTA's own result behind them.
template <int N, int C, int DP>
__device__ __forceinline__ void join_parts(const WinParams &p, float *part_ml, float *part_o, uint32_t row, uint32_t h0, uint32_t heads,
                                           uint32_t part, uint32_t parts, bool zero)
{
    float *cta_ml = part_o + N * C * DP, *cta_o = cta_ml + 2 * C;
    const uint32_t D = p.head_dim;
    __syncthreads();
    for (uint32_t x = threadIdx.x; x < heads * DP; x += blockDim.x) {
        const uint32_t c = x / DP, d = x % DP;
        float M = part_ml[c];
        for (int i = 1; i < N; i++) M = fmaxf(M, part_ml[i * 2 * C + c]);
        float ls = 0.f, os = 0.f;
        for (int i = 0; i < N; i++) {
            const float mi = part_ml[i * 2 * C + c], f = mi == -CUDART_INF_F ? 0.f : ab_ex2(mi - M);
            ls = fmaf(part_ml[i * 2 * C + C + c], f, ls);
            os = fmaf(part_o[(i * C + c) * DP + d], f, os);
        }
        if (parts == 1) {
            if (d < D) p.out[((uint64_t)row * p.q_heads + h0 + c) * D + d] = zero ? 0.f : os / ls;
        } else {
            cta_o[c * DP + d] = os;
            if (d == 0) { cta_ml[c] = M; cta_ml[C + c] = ls; }
        }
    }
    if (parts == 1) return;
    cluster_sync();
    const uint32_t ml_at = (uint32_t)__cvta_generic_to_shared(cta_ml), o_at = (uint32_t)__cvta_generic_to_shared(cta_o);
    for (uint32_t x = part * blockDim.x + threadIdx.x; x < heads * DP; x += parts * blockDim.x) {
        const uint32_t c = x / DP, d = x % DP;
        if (d >= D) continue;
        float M = -CUDART_INF_F;
        for (uint32_t i = 0; i < parts; i++) M = fmaxf(M, ld_cluster(ml_at + c * 4, i));
        float ls = 0.f, os = 0.f;
        for (uint32_t i = 0; i < parts; i++) {
            const float mi = ld_cluster(ml_at + c * 4, i), f = mi == -CUDART_INF_F ? 0.f : ab_ex2(mi - M);
            ls = fmaf(ld_cluster(ml_at + (C + c) * 4, i), f, ls);
            os = fmaf(ld_cluster(o_at + (c * DP + d) * 4, i), f, os);
        }
        p.out[((uint64_t)row * p.q_heads + h0 + c) * D + d] = zero ? 0.f : os / ls;
    }
    cluster_sync();                                                 // nobody leaves while its parts are being read
}

template <typename T, int DP>
__global__ void __launch_bounds__(kRowWarps * 32, sizeof(T) == 4 ? 3 : 4) win_rows_kernel(const WinParams p, const uint32_t parts)
{
    using Tile = RowTile<T, DP>;
    using Math = RowMath<T, DP>;
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t part = blockIdx.x % parts;
    const uint32_t D = p.head_dim, group = p.q_heads / p.kv_heads, per_kv = (group + 7) / 8;
    const uint32_t set = blockIdx.x / parts, kvh = set / per_kv, h0 = kvh * group + (set % per_kv) * 8;
    const uint32_t heads = min(8u, (kvh + 1) * group - h0);
    const uint32_t tile_k = (uint32_t)__cvta_generic_to_shared(smem) + warp * Tile::kWarpBytes, tile_v = tile_k + Tile::kBytesK;

    pdl_wait();
    if (p.left) pdl_trigger();                                      // the plan is there: the packing may run beside this
    for (uint32_t turn = blockIdx.y; turn < win_rows(p); turn += gridDim.y) {
    uint32_t row = turn;
    const WinView w = win_view(p, row);
    const uint32_t n_tiles = (w.n + kTile - 1) / kTile, step = parts * kRowWarps;
    uint32_t tile = part * kRowWarps + warp;

    // lanes 0..15 know the cache rows of a tile's positions (lanes 16..31 the same again)
    const auto rows_of = [&](uint32_t tl) -> uint32_t {
        const uint32_t i = tl * kTile + (lane & 15);
        return win_row(p, w, i, win_page(p, w, i));
    };
    const uint32_t row_bytes = D * sizeof(T), chunks = row_bytes / 16;
    const int span = chunks > 16 ? 32 : (chunks > 8 ? 16 : 8);      // lanes that copy one row
    const uint32_t chunk = lane & (span - 1);
    const uint64_t pitch = (uint64_t)p.kv_heads * row_bytes;
    const char *kb = static_cast<const char *>(p.k) + (uint64_t)kvh * row_bytes + chunk * 16;
    const char *vb = static_cast<const char *>(p.v) + (uint64_t)kvh * row_bytes + chunk * 16;
    const auto copy = [&](const char *base, uint32_t dst, uint32_t stride, uint32_t rows) {
        if (span == 32) {
#pragma unroll
            for (int r = 0; r < kTile; r++) {
                const uint32_t x = __shfl_sync(0xffffffffu, rows, r);
                if (chunk < chunks) cp16(dst + r * stride + chunk * 16, base + (x == 0xffffffffu ? 0 : x * pitch), x != 0xffffffffu);
            }
        } else {
            const int per = 32 / span;
            for (int r0 = 0; r0 < kTile; r0 += per) {
                const int r = r0 + lane / span;
                const uint32_t x = __shfl_sync(0xffffffffu, rows, r);
                if (chunk < chunks) cp16(dst + r * stride + chunk * 16, base + (x == 0xffffffffu ? 0 : x * pitch), x != 0xffffffffu);
            }
        }
        cp_commit();
    };

    if (D < DP) {                                                   // what a shorter head leaves unwritten of a tile is zero
        for (uint32_t i = lane; i < Tile::kWarpBytes / 16; i += 32)
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(tile_k + i * 16), "r"(0) : "memory");
        __syncwarp();
    }
    uint32_t rows = 0xffffffffu, next = 0xffffffffu;
    if (tile < n_tiles) {
        rows = rows_of(tile);
        copy(kb, tile_k, Tile::kStrideK, rows);
        copy(vb, tile_v, Tile::kStrideV, rows);
        if (tile + step < n_tiles) next = rows_of(tile + step);
    }
    QFrag<T, DP> q;
    float undo[2];
    q.load(p.q + ((uint64_t)row * p.q_heads + h0 + min((uint32_t)g, heads - 1)) * D, (uint32_t)g < heads, D, t, p.scale_log2, undo);

    float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f}, o[DP / 16][4];
#pragma unroll
    for (int i = 0; i < DP / 16; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    for (; tile < n_tiles; tile += step) {
        const bool more = tile + step < n_tiles;
        const uint32_t seen = __ballot_sync(0xffffffffu, rows != 0xffffffffu);
        cp_wait<1>();
        __syncwarp();
        float s[4];
        Math::scores(q, tile_k, g, t, s);
        __syncwarp();
        rows = next;
        if (more) {
            copy(kb, tile_k, Tile::kStrideK, rows);
            next = tile + 2 * step < n_tiles ? rows_of(tile + 2 * step) : 0xffffffffu;
        } else {
            cp_commit();
        }
        if (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 4; i++) s[i] *= undo[i & 1];
        }
        if (!((seen >> g) & 1)) s[0] = s[1] = -CUDART_INF_F;
        if (!((seen >> (g + 8)) & 1)) s[2] = s[3] = -CUDART_INF_F;
        float a[2], pr[4];
#pragma unroll
        for (int c = 0; c < 2; c++) {
            float x = fmaxf(s[c], s[c + 2]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float m1 = fmaxf(m[c], x), ms = m1 == -CUDART_INF_F ? 0.f : m1;
            const float bias = sizeof(T) == 2 ? kWeightBias : 0.f;
            a[c] = m[c] == m1 ? 1.f : ab_ex2(m[c] - ms);
            pr[c] = ab_ex2(s[c] - ms + bias);
            pr[c + 2] = ab_ex2(s[c + 2] - ms + bias);
            m[c] = m1;
            l[c] = fmaf(l[c], a[c], pr[c] + pr[c + 2]);
        }
        cp_wait<1>();
        __syncwarp();
        Math::values(pr, tile_v, g, t, lane, a, o);
        __syncwarp();
        if (more) copy(vb, tile_v, Tile::kStrideV, rows);
        else cp_commit();
    }
    cp_wait<0>();
    __syncthreads();

    // ---- the warps' parts, then the CTAs'
    float *part_ml = reinterpret_cast<float *>(smem), *part_o = part_ml + kRowWarps * 16;
#pragma unroll
    for (int c = 0; c < 2; c++) {
        l[c] += __shfl_xor_sync(0xffffffffu, l[c], 4);
        l[c] += __shfl_xor_sync(0xffffffffu, l[c], 8);
        l[c] += __shfl_xor_sync(0xffffffffu, l[c], 16);
        if (g == 0) { part_ml[warp * 16 + 2 * t + c] = m[c]; part_ml[warp * 16 + 8 + 2 * t + c] = l[c]; }
    }
#pragma unroll
    for (int i = 0; i < DP / 16; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) part_o[(warp * 8 + 2 * t + (e & 1)) * DP + Math::dim(i, e, g)] = o[i][e];
    join_parts<kRowWarps, 8, DP>(p, part_ml, part_o, row, h0, heads, part, parts, w.zero);
    __syncthreads();                                                // (the next turn's rows go where the parts are)
    }
}

// ------------------------------------------------------------------------------------------------
// The lane kernel: an f32 cache and one to four query heads per KV head, on the CUDA cores.
//
// LR lanes hold a position's row, four dimensions each (LR = 32 for a head of up to 128, 16 of up to 64, 8 of up to
// 32), and take eight positions at a time: the eight dot products of a head are reduced over the lanes together (4 + 2
// + 1 exchanges that halve what is left, then whole ones), so that a lane ends with one position's score and takes one
// exponential for it.  Every group of LR lanes has its own maximum, sum and output.  f32 throughout.
//
// The rows come by cp.async into a ring of two stages per warp, and a lane reads back what it copied itself, so a stage
// needs no barrier, and one is in flight while the other is worked on.  (In registers, loads for the next eight
// positions cost more than they hid: 148 us for the f32 batch, and 97 us without them.)
//
// Per position 25 warp instructions with one head and 70 with four, where the tensor-core form above takes 84
// whatever the heads (up to eight) and is bound by them: it stays for more heads and for f16 caches.  (16 rows over
// 4096 positions of 8 f32 KV heads, 537 MB: 90.7, 92.7, 97.4 and 103.7 us for one to four heads here, 5.9 to 5.2 TB/s, and
// 120.6 to 121.7 us there.)
// ------------------------------------------------------------------------------------------------
constexpr uint32_t kStageBytes = 8192;                              // of a warp: eight positions' rows of K and V in every group of lanes
constexpr uint32_t kLanesSmem = kRowWarps * 2 * kStageBytes;

template <int G, int LR>
__global__ void __launch_bounds__(kRowWarps * 32, 3) win_lanes_kernel(const WinParams p, const uint32_t parts)
{
    constexpr int S = 32 / LR, DP = 4 * LR, kPart = kRowWarps * S;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    static_assert((kPart + 1) * G * (DP + 2) * 4 <= kLanesSmem, "the parts fit where the rows were");
    float *smem = reinterpret_cast<float *>(smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LR, ll = lane % LR;
    const uint32_t part = blockIdx.x % parts, kvh = blockIdx.x / parts, h0 = kvh * G, D = p.head_dim;
    const bool on = (uint32_t)ll * 4 < D;
    pdl_wait();
    if (p.left) pdl_trigger();                                      // the plan is there: the packing may run beside this
    for (uint32_t turn = blockIdx.y; turn < win_rows(p); turn += gridDim.y) {
    uint32_t row = turn;
    const WinView w = win_view(p, row);
    const uint32_t n_batches = (w.n + 7) / 8, step = parts * kPart;
    // lanes 0..7 of a group: its eight positions (past the last batch there is nothing to see)
    const auto page_of = [&](uint32_t b) { return win_page(p, w, (b + sub) * 8 + (ll & 7)); };
    const auto rows_of = [&](uint32_t b, uint32_t page) { return win_row(p, w, (b + sub) * 8 + (ll & 7), page); };
    const uint64_t pitch = (uint64_t)p.kv_heads * D;
    const float *kb = static_cast<const float *>(p.k) + (uint64_t)kvh * D + ll * 4, *vb = static_cast<const float *>(p.v) + (uint64_t)kvh * D + ll * 4;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem_raw) + warp * 2 * kStageBytes + lane * 16;
    const auto copy = [&](uint32_t stage, uint32_t rows) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t r = __shfl_sync(0xffffffffu, rows, sub * LR + j);
            const bool load = on && r != 0xffffffffu;
            const uint64_t at = load ? r * pitch : 0;
            cp16(ring + stage * kStageBytes + j * 512, kb + at, load);
            cp16(ring + stage * kStageBytes + 4096 + j * 512, vb + at, load);
        }
        cp_commit();
    };
    uint32_t b0 = (part * kRowWarps + warp) * S, seen0, seen1;
    {
        const uint32_t page0 = page_of(b0), page1 = page_of(b0 + step);
        seen0 = rows_of(b0, page0);
        copy(0, seen0);
        seen1 = rows_of(b0 + step, page1);
        copy(1, seen1);
    }
    uint32_t page = page_of(b0 + 2 * step);
    float4 q[G], o[G];
    float m[G], l[G];
#pragma unroll
    for (int h = 0; h < G; h++) {
        q[h] = on ? *reinterpret_cast<const float4 *>(p.q + ((uint64_t)row * p.q_heads + h0 + h) * D + ll * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
        q[h].x *= p.scale_log2; q[h].y *= p.scale_log2; q[h].z *= p.scale_log2; q[h].w *= p.scale_log2;
        o[h] = make_float4(0.f, 0.f, 0.f, 0.f);
        m[h] = -CUDART_INF_F;
        l[h] = 0.f;
    }
    uint32_t stage = 0;
    for (; b0 < n_batches; b0 += step, stage ^= 1) {
        // the position whose score a lane ends with
        const bool seen = __shfl_sync(0xffffffffu, seen0, sub * LR + ll / (LR / 8)) != 0xffffffffu;
        float4 k[8];
        float x[G];
        cp_wait<1>();
#pragma unroll
        for (int j = 0; j < 8; j++) k[j] = lds128(ring + stage * kStageBytes + j * 512);
#pragma unroll
        for (int h = 0; h < G; h++) {
            float s[8];
#pragma unroll
            for (int j = 0; j < 8; j++) s[j] = fmaf(q[h].w, k[j].w, fmaf(q[h].z, k[j].z, fmaf(q[h].y, k[j].y, q[h].x * k[j].x)));
#pragma unroll
            for (int i = 0; i < 3; i++) {                              // a group's halves keep half of the scores each
                const int width = LR >> (i + 1), n = 4 >> i;
                const bool upper = (ll & width) != 0;
#pragma unroll
                for (int j = 0; j < n; j++) {
                    const float give = upper ? s[j] : s[j + n], keep = upper ? s[j + n] : s[j];
                    s[j] = keep + __shfl_xor_sync(0xffffffffu, give, width);
                }
            }
            x[h] = s[0];
#pragma unroll
            for (int width = LR / 16; width; width /= 2) x[h] += __shfl_xor_sync(0xffffffffu, x[h], width);
            if (!seen) x[h] = -CUDART_INF_F;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) k[j] = lds128(ring + stage * kStageBytes + 4096 + j * 512);
        seen0 = seen1;
        seen1 = rows_of(b0 + 2 * step, page);
        copy(stage, seen1);
        page = page_of(b0 + 3 * step);
#pragma unroll
        for (int h = 0; h < G; h++) {
            float top = x[h];
#pragma unroll
            for (int i = 1; i <= 3; i++) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, LR >> i));
            const float m1 = fmaxf(m[h], top), ms = m1 == -CUDART_INF_F ? 0.f : m1;
            const float a = m[h] == m1 ? 1.f : ab_ex2(m[h] - ms), e = ab_ex2(x[h] - ms);
            m[h] = m1;
            l[h] = fmaf(l[h], a, e);
            o[h].x *= a; o[h].y *= a; o[h].z *= a; o[h].w *= a;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float pj = __shfl_sync(0xffffffffu, e, sub * LR + j * (LR / 8));
                o[h].x = fmaf(pj, k[j].x, o[h].x); o[h].y = fmaf(pj, k[j].y, o[h].y);
                o[h].z = fmaf(pj, k[j].z, o[h].z); o[h].w = fmaf(pj, k[j].w, o[h].w);
            }
        }
    }
    cp_wait<0>();
    __syncthreads();
    float *part_ml = smem, *part_o = part_ml + kPart * 2 * G;
    const int unit = warp * S + sub;
#pragma unroll
    for (int h = 0; h < G; h++) {
#pragma unroll
        for (int i = 1; i <= 3; i++) l[h] += __shfl_xor_sync(0xffffffffu, l[h], LR >> i);
        if (ll == 0) { part_ml[unit * 2 * G + h] = m[h]; part_ml[unit * 2 * G + G + h] = l[h]; }
        *reinterpret_cast<float4 *>(part_o + (unit * G + h) * DP + ll * 4) = o[h];
    }
    join_parts<kPart, G, DP>(p, part_ml, part_o, row, h0, G, part, parts, w.zero);
    __syncthreads();
    }
}

// a kernel's shared memory and clusters of 16 CTAs, beyond what it gets unasked: once per device (`done`: a bit for each)
int prepare(void (*kernel)(const WinParams, const uint32_t), size_t bytes, uint64_t (&done)[4], const char *name)
{
    static std::mutex mu;
    int dev = 0;
    cudaGetDevice(&dev);
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 0 && dev < 256 && (done[dev / 64] >> (dev % 64) & 1)) return AB_OK;
    int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), name);
    if (rc == AB_OK) rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), name);
    if (rc == AB_OK && dev >= 0 && dev < 256) done[dev / 64] |= 1ull << (dev % 64);
    return rc;
}

// Grid: a cluster of `parts` CTAs that share the list of a row (blockIdx.y) and group of heads (blockIdx.x: the heads' parts of
// a position are neighbours in memory, and so in time; 91.0 -> 89.8 us for the f32 batch above, 97.2 -> 96.6 for the f16 one).  The time of a
// launch is about the rounds of resident CTAs it takes times the steps of a CTA, `unit` positions each, and three more
// to start and to join, and an eighth of one per part; parts is what makes that least.  (The f32 batch above, 512 x parts CTAs on 444 places: 98.6, 91.7,
// 94.8 and 119 us for 1, 2, 4 and 8 parts; the f16 one, 256 x parts on 592: 109, 101, 102 and 112 us.)
int launch_split(Launch &l, const WinParams &p, void (*kernel)(const WinParams, const uint32_t), uint32_t groups, uint32_t resident,
                 uint32_t unit, size_t smem, const char *how, const char *name)
{
    // (beside tiles, the rows left are mostly one of each sequence; the device knows how many)
    const uint64_t rows = p.left ? std::min(p.rows, p.batch) : p.rows;
    const uint64_t longest = std::min<uint64_t>((uint64_t)p.window + p.sinks, p.reach), places = (uint64_t)resident * sm_count();
    uint32_t parts = 1;
    uint64_t least = ~0ull;
    for (uint32_t n = 1; n <= 16; n *= 2) {
        const uint64_t rounds = (rows * groups * n + places - 1) / places, steps = (longest + (uint64_t)n * unit - 1) / ((uint64_t)n * unit);
        const uint64_t cost = rounds * (8 * (steps + 3) + n);
        if (cost < least) { least = cost; parts = n; }
    }
    const uint64_t turns = p.left ? std::min<uint64_t>(p.rows, std::max<uint64_t>(rows, places / ((uint64_t)groups * parts) + 1)) : rows;
    if ((uint64_t)groups * parts > 0x7fffffffull)
        return fail(AB_ERR_INVALID, "%s: %u rows of %u heads", name, p.rows, p.q_heads);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(groups * parts, (uint32_t)std::min<uint64_t>(turns, 65535));
    cfg.blockDim = dim3(kRowWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = l.stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (parts > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = parts;
        attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
        cfg.numAttrs++;
    }
    // (its CTAs are there when the kernel before it ends: 91.7 -> 89.9 us a call for the f32 batch, 106.2 -> 105.0 for the f16 one)
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, parts);
    count_launch();
    note_selection("%s: %s, %u rows, %u group(s) of heads, a list split over %u CTA(s)", name, how, p.rows, groups, parts);
    return check_cuda(e, name);
}

template <typename T, int DP> int launch_rows(Launch &l, const WinParams &p, const char *name)
{
    const uint32_t group = p.q_heads / p.kv_heads;
    static uint64_t done[4];
    const int rc = prepare(win_rows_kernel<T, DP>, RowTile<T, DP>::kSmem, done, name);
    if (rc) return rc;
    return launch_split(l, p, win_rows_kernel<T, DP>, p.kv_heads * ((group + 7) / 8), sizeof(T) == 4 ? 3 : 4, kRowWarps * kTile, RowTile<T, DP>::kSmem,
                        "up to 8 heads a CTA on the tensor cores", name);
}

template <int G, int LR> int launch_lanes(Launch &l, const WinParams &p, const char *name)
{
    static uint64_t done[4];
    const int rc = prepare(win_lanes_kernel<G, LR>, kLanesSmem, done, name);
    if (rc) return rc;
    return launch_split(l, p, win_lanes_kernel<G, LR>, p.kv_heads, 3, kRowWarps * 8 * (32 / LR), kLanesSmem, "a row a group of lanes", name);
}
template <int G> int launch_lanes(Launch &l, const WinParams &p, const char *name)
{
    return p.head_dim > 64 ? launch_lanes<G, 32>(l, p, name) : (p.head_dim > 32 ? launch_lanes<G, 16>(l, p, name) : launch_lanes<G, 8>(l, p, name));
}

template <typename T> int run_rows(Launch &l, const WinParams &p, const char *name)
{
    const uint32_t group = p.q_heads / p.kv_heads;
    if (sizeof(T) == 4) {
        switch (group) {
        case 1: return launch_lanes<1>(l, p, name);
        case 2: return launch_lanes<2>(l, p, name);
        case 3: return launch_lanes<3>(l, p, name);
        case 4: return launch_lanes<4>(l, p, name);
        default: break;
        }
    }
    return p.head_dim <= 64 ? launch_rows<T, 64>(l, p, name) : launch_rows<T, 128>(l, p, name);
}

template <typename T> int run_window(Launch &l, WinParams &p, const char *name)
{
    if ((uint64_t)p.base + p.rows > 0xffffffffull)
        return fail(AB_ERR_INVALID, "%s: Base=%u and %u rows pass 32 bits", name, p.base, p.rows);
    l.ws_need = 0;
    if (p.rows == 0) return AB_OK;
    const uint32_t group = p.q_heads / p.kv_heads;
    // (the device alone knows how a ragged step's rows are dealt out; with one or more to each sequence, the most that one
    // has is what the host assumes, and a step of single tokens needs no plan: 16 of them over 1024 positions take 29.6 us of the
    // row kernel's time, and took 7.0 us more of kernels without work)
    const uint64_t most = p.form == kPrefillRows ? p.rows : (p.form == kRaggedStep && p.rows >= p.batch ? p.rows - p.batch + 1 : 0);
    const uint64_t seen = std::min<uint64_t>((uint64_t)p.window + p.sinks, p.form == kPrefillRows ? std::min<uint64_t>((uint64_t)p.base + p.rows, p.reach) : p.reach);
    if (group <= 128 && on_tiles(most * group, seen, p.kv_heads)) return run_window_tiles(l, p, sizeof(T) == 2, run_rows<T>, name);
    return l.query_ws ? AB_OK : run_rows<T>(l, p, name);
}

// WindowDims{Batch,QHeads,KVHeads,HeadDim,Block,MaxPages,Scale f32,Window,Sinks,Capacity,QSeq,Base}, 48 bytes.
// The lengths block is u32 and a cache may hold more elements than that: its rows are Capacity, and a
// length of 0xffffffff stands for that many or more.
int window_form(Launch &l, Form form, bool paged, bool f16, const char *name)
{
    WinParams p{};
    p.form = form;
    p.batch = u32_at(l.u, 0);
    p.q_heads = u32_at(l.u, 4); p.kv_heads = u32_at(l.u, 8); p.head_dim = u32_at(l.u, 12);
    p.block = paged ? u32_at(l.u, 16) : 1;
    p.max_pages = paged ? u32_at(l.u, 20) : 0;
    p.scale_log2 = f32_at(l.u, 24) * kLog2e;
    p.window = u32_at(l.u, 28); p.sinks = u32_at(l.u, 32); p.capacity = u32_at(l.u, 36);
    if (form == kPrefillRows) { p.rows = u32_at(l.u, 40); p.base = u32_at(l.u, 44); p.batch = 1; }
    if (form == kDecode) p.rows = p.batch = 1;
    if (form == kBatch) p.rows = p.batch;
    if (p.kv_heads == 0 || p.q_heads == 0 || p.q_heads % p.kv_heads != 0)
        return fail(AB_ERR_INVALID, "%s: %u query heads over %u key/value heads", name, p.q_heads, p.kv_heads);
    if (p.head_dim == 0 || p.head_dim % 8 != 0 || p.head_dim > 128)
        return fail(AB_ERR_INVALID, "%s: head dimension %u; it is a multiple of eight and at most 128", name, p.head_dim);
    if (p.block == 0) return fail(AB_ERR_INVALID, "%s: a page table addresses blocks, and Block is 0", name);
    if (p.window == 0)
        return fail(AB_ERR_INVALID, "%s: a window of 0 positions; a query sees at least its own (without a window: "
                    "the Attention kernels)", name);
    const uint64_t per = (uint64_t)p.q_heads * p.head_dim, kvper = (uint64_t)p.kv_heads * p.head_dim;
    if (form == kRaggedStep && l.len[0] == 0xffffffffu)
        return fail(AB_ERR_INVALID, "%s: q's length, which says how many rows there are, does not fit 32 bits", name);
    if (form == kRaggedStep) p.rows = per ? (uint32_t)(l.len[0] / per) : 0;
    int i = 3;
    const int pages_i = paged ? i++ : -1, len_i = i++, off_i = form == kRaggedStep ? i++ : -1, out_i = i;
    p.reach = paged ? (uint32_t)std::min<uint64_t>((uint64_t)p.max_pages * p.block, 0xffffffffull) : p.capacity;
    const auto holds = [&](int b, uint64_t n) { return l.len[b] == 0xffffffffu || l.len[b] >= n; };
    if (!holds(0, p.rows * per) || !holds(out_i, p.rows * per) || !holds(1, p.capacity * kvper) || !holds(2, p.capacity * kvper) ||
        !holds(len_i, p.batch) || (paged && !holds(pages_i, (uint64_t)p.batch * p.max_pages)) ||
        (off_i >= 0 && !holds(off_i, (uint64_t)p.batch + 1)))
        return fail(AB_ERR_INVALID, "%s: Batch=%u QHeads=%u KVHeads=%u HeadDim=%u MaxPages=%u Capacity=%u rows=%u and the "
                    "lengths block says q[%u] k[%u] v[%u] lengths[%u] out[%u]", name, p.batch, p.q_heads, p.kv_heads,
                    p.head_dim, p.max_pages, p.capacity, p.rows, l.len[0], l.len[1], l.len[2], l.len[len_i], l.len[out_i]);
    if (!l.query_ws) {
        p.q = ptr<const float>(l, 0); p.k = l.b[1]; p.v = l.b[2];
        p.pages = paged ? ptr<const uint32_t>(l, pages_i) : nullptr;
        p.lengths = ptr<const uint32_t>(l, len_i);
        p.offsets = off_i >= 0 ? ptr<const uint32_t>(l, off_i) : nullptr;
        p.out = ptr<float>(l, out_i);
    }
    return f16 ? run_window<__half>(l, p, name) : run_window<float>(l, p, name);
}

}  // namespace

int launch_attention_window(Launch &l) { return window_form(l, kDecode, false, false, "AttentionWindow"); }
int launch_attention_window_f16(Launch &l) { return window_form(l, kDecode, false, true, "AttentionWindowF16"); }
int launch_attention_window_batched(Launch &l) { return window_form(l, kBatch, true, false, "AttentionWindowBatched"); }
int launch_attention_window_batched_f16(Launch &l) { return window_form(l, kBatch, true, true, "AttentionWindowBatchedF16"); }
int launch_attention_window_ragged(Launch &l) { return window_form(l, kRaggedStep, true, false, "AttentionWindowRagged"); }
int launch_attention_window_ragged_f16(Launch &l) { return window_form(l, kRaggedStep, true, true, "AttentionWindowRaggedF16"); }
int launch_attention_window_prefill(Launch &l) { return window_form(l, kPrefillRows, false, false, "AttentionWindowPrefill"); }
int launch_attention_window_prefill_f16(Launch &l) { return window_form(l, kPrefillRows, false, true, "AttentionWindowPrefillF16"); }
int launch_attention_window_prefill_paged(Launch &l) { return window_form(l, kPrefillRows, true, false, "AttentionWindowPrefillPaged"); }
int launch_attention_window_prefill_paged_f16(Launch &l) { return window_form(l, kPrefillRows, true, true, "AttentionWindowPrefillPagedF16"); }

}  // namespace ab
