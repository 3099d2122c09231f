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

#include "common.cuh"

namespace ab {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

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
    float scale_log2;                              // Scale * log2(e)
    int form;
};

// What one query row sees.
struct WinView {
    const uint32_t *pages;
    uint32_t lo, ns, n;
    bool zero;                                     // a ragged padding row: written as zeros
};

__device__ __forceinline__ WinView win_view(const WinParams &p, uint32_t row)
{
    WinView w{p.pages, 0, 0, 0, false};
    uint64_t pos1;                                 // the row's position + 1
    uint32_t len;
    if (p.form == kRaggedStep) {
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

// the cache row of the list's entry i; 0xffffffff where its page lies outside the cache
__device__ __forceinline__ uint32_t win_row(const WinParams &p, const WinView &w, uint32_t i)
{
    const uint32_t j = i < w.ns ? i : w.lo + (i - w.ns);
    uint64_t r = j;
    if (w.pages) {
        const uint32_t pg = j / p.block;
        r = (uint64_t)w.pages[pg] * p.block + (j - pg * p.block);
    }
    return r < p.capacity ? (uint32_t)r : 0xffffffffu;
}

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }

// One warp per (row, query head), a lane holds the dimensions lane, lane + 32, ...
template <typename T>
__global__ void __launch_bounds__(128) win_simple_kernel(const WinParams p)
{
    const uint64_t item = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= (uint64_t)p.rows * p.q_heads) return;
    const uint32_t row = (uint32_t)(item / p.q_heads), h = (uint32_t)(item % p.q_heads);
    const int lane = threadIdx.x & 31;
    const uint32_t D = p.head_dim, kvh = h / (p.q_heads / p.kv_heads);
    const WinView w = win_view(p, row);
    const T *k = static_cast<const T *>(p.k), *v = static_cast<const T *>(p.v);
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, oc[4];
    for (int e = 0; e < 4; e++) q[e] = (uint32_t)(lane + 32 * e) < D ? p.q[item * D + lane + 32 * e] * p.scale_log2 : 0.f;
    // sums over runs of 64 positions are joined by the same recurrence: a run of thousands of additions
    // into one accumulator would lose two more bits of it
    float m = -CUDART_INF_F, l = 0.f;
    for (uint32_t i0 = 0; i0 < w.n; i0 += 64) {
        float mc = -CUDART_INF_F, lc = 0.f;
        for (int e = 0; e < 4; e++) oc[e] = 0.f;
        for (uint32_t i = i0; i < min(i0 + 64, w.n); i++) {
            const uint32_t r = win_row(p, w, i);
            if (r == 0xffffffffu) continue;
            const size_t at = ((size_t)r * p.kv_heads + kvh) * D;
            float s = 0.f;
            for (int e = 0; e < 4; e++) if ((uint32_t)(lane + 32 * e) < D) s = fmaf(q[e], to_f32(k[at + lane + 32 * e]), s);
            for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            const float m1 = fmaxf(mc, s), a = mc == m1 ? 1.f : exp2f(mc - m1), pr = exp2f(s - m1);
            mc = m1;
            lc = fmaf(lc, a, pr);
            for (int e = 0; e < 4; e++)
                if ((uint32_t)(lane + 32 * e) < D) oc[e] = fmaf(oc[e], a, pr * to_f32(v[at + lane + 32 * e]));
        }
        if (mc == -CUDART_INF_F && lc == 0.f) continue;
        const float m1 = fmaxf(m, mc), a = m == m1 ? 1.f : exp2f(m - m1), c = mc == m1 ? 1.f : exp2f(mc - m1);
        m = m1;
        l = fmaf(l, a, lc * c);
        for (int e = 0; e < 4; e++) o[e] = fmaf(o[e], a, oc[e] * c);
    }
    for (int e = 0; e < 4; e++)
        if ((uint32_t)(lane + 32 * e) < D) p.out[item * D + lane + 32 * e] = w.zero ? 0.f : o[e] / l;
}

template <typename T> int run_window(Launch &l, WinParams &p, const char *name)
{
    if ((uint64_t)p.base + p.rows > 0xffffffffull)
        return fail(AB_ERR_INVALID, "%s: Base=%u and %u rows pass 32 bits", name, p.base, p.rows);
    l.ws_need = 0;
    if (l.query_ws) return AB_OK;
    const uint64_t items = (uint64_t)p.rows * p.q_heads;
    if (items == 0) return AB_OK;
    if ((items + 3) / 4 > 0x7fffffffull) return fail(AB_ERR_INVALID, "%s: %u rows of %u heads", name, p.rows, p.q_heads);
    win_simple_kernel<T><<<(uint32_t)((items + 3) / 4), 128, 0, l.stream>>>(p);
    count_launch();
    note_selection("%s: a warp per row and head", name);
    return check_cuda(cudaGetLastError(), name);
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
