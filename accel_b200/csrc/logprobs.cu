// Log probabilities of given tokens, the distribution's entropy, and the most probable alternatives,
// of every row of logits.  No counterpart in the reference.
//
//     m = max x,  s = sum e^(x - m),  logprob(t) = (x_t - m) - log s,
//     entropy = -sum p log p = log s - u / s,  u = sum (x - m) e^(x - m)
//
// and the Top largest logits in (value descending, index ascending) order with their log
// probabilities; -0 equals +0 and a NaN is larger than every number.  A logit of -inf is a token of
// probability 0 and adds nothing to the entropy.  A row that holds a NaN or a +inf, or nothing above
// -inf, has no distribution: its log probabilities and entropy are NaN (its indices still stand).  A
// target at or past Vocab has the log probability NaN.
//
// The row is read once: a thread carries (m, s, u) over its pieces, moving to a new maximum m' by
//     s' = s e^(m - m'),  u' = (u + (m - m') s) e^(m - m'),
// once per 16 elements, and threads, warps and CTAs are joined by the same rule in a fixed order.  One
// exponential and seven instructions per element: HBM bounds it.
//
// The alternatives cost no second pass.  With `each` = ceil(Top / warps) + 2 the warps' `each` largest thread maxima
// are at least Top numbers, every one reached by an element of its own, so at least Top elements reach
// the Top-th largest of them, the floor.  Only threads whose maximum reaches it can hold an alternative (about
// Top of 256); their pieces are read again (L2, all at once), what reaches the floor is listed, and an
// element's place among the alternatives is the number of listed ones before it.
#include <math_constants.h>

#include <algorithm>

#include "common.cuh"

namespace ab {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kMaxTop = 32;
constexpr uint32_t kList = 1024;           // candidates a CTA can list; more (a shape made for it) takes the slow way
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;

typedef unsigned long long u64;

// values in the order of their magnitude as unsigned numbers; 0 is below every value
__device__ __forceinline__ uint32_t lp_key(float x)
{
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.f);          // -0 + 0 = +0
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t key)
{
    if (key == 0xffffffffu) return CUDART_NAN_F;
    return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}
// an element as one number: the larger comes first
__device__ __forceinline__ u64 lp_rank(float x, uint32_t index) { return (u64)lp_key(x) << 32 | (0xffffffffu - index); }

struct LpParams {
    const void *x;
    const uint32_t *targets;
    float *logprobs, *entropy;
    uint32_t *top_ids;
    float *top_logprobs;
    uint32_t vocab, rows, n_targets, top;
};

// 16 aligned bytes of a row
template <typename T> struct Piece;
template <> struct Piece<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ float one(const float *p) { return *p; }
    static constexpr uint32_t kNone = 0xff800000u;        // -inf in every element
    static __device__ __forceinline__ void open(const uint4 &v, float *x)
    {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
};
template <> struct Piece<__half> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ float one(const __half *p) { return __half2float(*p); }
    static constexpr uint32_t kNone = 0xfc00fc00u;
    static __device__ __forceinline__ void open(const uint4 &v, float *x)
    {
        const uint32_t r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r[i]));
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
    }
};

struct Sums { float m, s, u; };
__device__ __forceinline__ float lp_exp(float d) { return ab_ex2(d * kLog2e); }
// below -1e4 e^d is 0, and (-inf) * 0 would be a NaN
__device__ __forceinline__ float lp_clamp(float d) { return fmaxf(d, -1e4f); }
// moves the sums to a maximum M >= m
__device__ __forceinline__ void lp_move(Sums &a, float M)
{
    const float d = a.m - M, f = lp_exp(d);
    a.u = fmaf(lp_clamp(d), a.s, a.u) * f;
    a.s *= f;
    a.m = M;
}
__device__ __forceinline__ void lp_join(Sums &a, Sums b)
{
    const float M = fmaxf(a.m, b.m);
    if (a.m != M) lp_move(a, M);
    if (b.m != M) lp_move(b, M);
    a.s += b.s;
    a.u += b.u;
}
// two elements, into sums of their own
__device__ __forceinline__ void lp_add(float2 x, float2 m, float2 &s, float2 &u)
{
    const float2 d = ab_add2(x, make_float2(-m.x, -m.y)), z = ab_mul2(d, make_float2(kLog2e, kLog2e));
    const float2 e = make_float2(ab_ex2(z.x), ab_ex2(z.y));
    s = ab_add2(s, e);
    u = ab_fma2(make_float2(lp_clamp(d.x), lp_clamp(d.y)), e, u);
}

__device__ __forceinline__ uint32_t lp_mapa(const void *p, uint32_t rank)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ float lp_remote_f32(uint32_t a)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ u64 lp_remote_u64(uint32_t a)
{
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void lp_cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A cluster of `parts` CTAs per row, a contiguous run of the row's pieces each; the first also takes the few elements
// before the first and behind the last whole piece.
template <typename T> __global__ void __launch_bounds__(kThreads, 6) logprobs_kernel(const LpParams p, const uint32_t parts)
{
    constexpr int N = Piece<T>::kN, U = 16 / N;
    __shared__ Sums sums[kWarps];
    __shared__ Sums whole;
    __shared__ uint32_t maxima[kWarps * (kMaxTop / kWarps + 2)], at_floor, n_list, n_held;
    __shared__ uint8_t held[kThreads];
    __shared__ u64 list[kList], best[kMaxTop], all[16 * kMaxTop], slow[kWarps];
    pdl_wait();
    const uint32_t row = blockIdx.x / parts, part = blockIdx.x % parts, V = p.vocab, t = threadIdx.x;
    const int warp = t >> 5, lane = t & 31;
    const T *x = static_cast<const T *>(p.x) + (size_t)row * V;
    const uint32_t head = min(V, (uint32_t)((0 - reinterpret_cast<uintptr_t>(x)) & 15) / (uint32_t)sizeof(T));
    const uint32_t pieces = (V - head) / N, tail = head + pieces * N, n_extra = part == 0 ? head + (V - tail) : 0;
    const uint32_t per = (pieces + parts - 1) / parts, p0 = min(part * per, pieces), p1 = min(p0 + per, pieces);
    const T *xp = x + head;
    const auto extra = [&](uint32_t i) { return i < head ? i : tail + (i - head); };

    // ---- one pass
    Sums a{kLowest, 0.f, 0.f};
    const auto fetch = [&](uint32_t i) {
        return i < p1 ? reinterpret_cast<const uint4 *>(xp)[i] : make_uint4(Piece<T>::kNone, Piece<T>::kNone, Piece<T>::kNone, Piece<T>::kNone);
    };
    uint4 next[U];
#pragma unroll
    for (int j = 0; j < U; j++) next[j] = fetch(p0 + t + j * kThreads);
    for (uint32_t i = p0 + t; i < p1; i += kThreads * U) {
        float v[16];
#pragma unroll
        for (int j = 0; j < U; j++) {
            Piece<T>::open(next[j], v + j * N);
            next[j] = fetch(i + (U + j) * kThreads);                // the next 16 are on their way
        }
        float c = v[0];
#pragma unroll
        for (int e = 1; e < 16; e++) c = fmaxf(c, v[e]);
        lp_move(a, fmaxf(a.m, c));
        float2 s = make_float2(a.s, 0.f), u = make_float2(a.u, 0.f);
#pragma unroll
        for (int e = 0; e < 16; e += 2) lp_add(make_float2(v[e], v[e + 1]), make_float2(a.m, a.m), s, u);
        a.s = s.x + s.y;
        a.u = u.x + u.y;
    }
    if (t < n_extra) {
        const float v = Piece<T>::one(x + extra(t));
        lp_move(a, fmaxf(a.m, v));
        const float d = v - a.m, e = lp_exp(d);
        a.s += e;
        a.u = fmaf(lp_clamp(d), e, a.u);
    }
    // the thread's largest element.  a.m says it but for a NaN (which s shows), and where nothing is above -FLT_MAX
    const bool any = p0 + t < p1 || t < n_extra;
    uint32_t key = 0;
    if (p.top && any) {
        key = lp_key(a.m);
        if (a.s != a.s || a.m == kLowest) {
            key = 0;
            for (uint32_t i = p0 + t; i < p1; i += kThreads)
                for (int e = 0; e < N; e++) key = max(key, lp_key(Piece<T>::one(xp + (size_t)i * N + e)));
            if (t < n_extra) key = max(key, lp_key(Piece<T>::one(x + extra(t))));
        }
    }
#pragma unroll
    for (int w = 16; w; w /= 2) {
        Sums b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, w);
        b.s = __shfl_xor_sync(0xffffffffu, a.s, w);
        b.u = __shfl_xor_sync(0xffffffffu, a.u, w);
        // both sides of a pair add in the same order, so that every lane holds the same bits
        if (lane & w) { const Sums c = a; a = b; b = c; }
        lp_join(a, b);
    }
    if (lane == 0) sums[warp] = a;
    if (p.top) {
        const uint32_t each = (p.top + kWarps - 1) / kWarps + 2;
        uint32_t k = key;
        for (uint32_t r = 0; r < each; r++) {
            const uint32_t f = __reduce_max_sync(0xffffffffu, k), at = __ballot_sync(0xffffffffu, k == f);
            if (lane == __ffs(at) - 1) k = 0;
            if (lane == 0) maxima[warp * each + r] = f;
        }
        if (t == 0) { n_list = 0; n_held = 0; }
    }
    __syncthreads();
    if (t == 0) {
        Sums b = sums[0];
        for (int i = 1; i < kWarps; i++) lp_join(b, sums[i]);
        whole = b;
    }

    // ---- the CTA's Top largest elements, in order, into best[] (0: it has fewer)
    if (p.top) {
        const uint32_t n_max = kWarps * ((p.top + kWarps - 1) / kWarps + 2);
        if (t < n_max) {
            const uint32_t mine = maxima[t];
            uint32_t before = 0;
            for (uint32_t j = 0; j < n_max; j++) before += maxima[j] > mine || (maxima[j] == mine && j < t);
            if (before == p.top - 1) at_floor = mine;
        }
        __syncthreads();
        const uint32_t floor = at_floor;
        {
            // the threads to look at (a floor of 0: fewer than Top threads have elements at all)
            const uint32_t b = __ballot_sync(0xffffffffu, key >= floor && key != 0);
            uint32_t at = 0;
            if (lane == 0 && b) at = atomicAdd(&n_held, __popc(b));
            at = __shfl_sync(0xffffffffu, at, 0);
            if ((b >> lane) & 1) held[at + __popc(b & ((1u << lane) - 1))] = (uint8_t)t;
        }
        __syncthreads();
        const uint32_t n_who = n_held, todo = n_who * ((p1 - p0 + kThreads - 1) / kThreads);
        if (t < kMaxTop) best[t] = 0;
        // what reaches the floor; where that is more than the list holds (many ties at the floor) what passes it, and
        // where that is too, nothing: the alternatives are then found one by one
        bool ties = false;
        uint32_t n;
        for (int pass = 0;; pass++) {
            const auto reaches = [&](uint32_t k) { return pass ? k > floor : k >= floor; };
            const auto put = [&](float v, uint32_t index) {
                const uint32_t k = lp_key(v);
                if (reaches(k)) {
                    const uint32_t at = atomicAdd(&n_list, 1);  // the places differ from run to run, what is listed does not
                    if (at < kList) list[at] = (u64)k << 32 | (0xffffffffu - index);
                }
            };
            for (uint32_t j0 = t; j0 < todo; j0 += U * kThreads) {
                uint4 raw[U];
                uint32_t at[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const uint32_t j = j0 + u * kThreads, i = p0 + j / n_who * kThreads + held[j % n_who];
                    at[u] = j < todo && i < p1 ? i : 0xffffffffu;
                    raw[u] = fetch(at[u]);
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float v[N];
                    Piece<T>::open(raw[u], v);
                    if (at[u] != 0xffffffffu)
#pragma unroll
                        for (int e = 0; e < N; e++) put(v[e], head + at[u] * N + e);
                }
            }
            if (t < n_extra) put(Piece<T>::one(x + extra(t)), extra(t));
            __syncthreads();
            n = n_list;
            if (n <= kList || pass) break;
            ties = true;
            __syncthreads();
            if (t == 0) n_list = 0;
            __syncthreads();
        }
        if (n > kList) {
            // the largest, then the largest below it, and so on over the run
            u64 last = ~0ull;
            for (uint32_t r = 0; r < p.top; r++) {
                u64 b = 0;
                const auto take = [&](float v, uint32_t index) {
                    const u64 k = lp_rank(v, index);
                    if (k < last && k > b) b = k;
                };
                for (uint32_t i = p0 + t; i < p1; i += kThreads)
                    for (int e = 0; e < N; e++) take(Piece<T>::one(xp + (size_t)i * N + e), head + i * N + e);
                if (t < n_extra) take(Piece<T>::one(x + extra(t)), extra(t));
                for (int w = 16; w; w /= 2) b = max(b, __shfl_xor_sync(0xffffffffu, b, w));
                if (lane == 0) slow[warp] = b;
                __syncthreads();
                b = slow[0];
                for (int i = 1; i < kWarps; i++) b = max(b, slow[i]);
                if (t == 0) best[r] = b;
                last = b;
                __syncthreads();
                if (b == 0) break;
            }
        } else {
            for (uint32_t i = t; i < n; i += kThreads) {
                const u64 mine = list[i];
                uint32_t before = 0;
                for (uint32_t j = 0; j < n; j++) before += list[j] > mine;
                if (before < p.top) best[before] = mine;
            }
            if (ties && n < p.top) {
                // and the lowest indices that equal the floor: every warp looks for them in an eighth of the run, in order
                const uint32_t want = p.top - n;
                const uint32_t first = part == 0 ? 0 : head + p0 * N, end = part == 0 && p1 == pieces ? V : head + p1 * N;
                const uint32_t run = ((end - first + kWarps - 1) / kWarps + 31) & ~31u;
                uint32_t have = 0;
                __syncthreads();                                // list is free for them: kMaxTop to a warp
                for (uint32_t i0 = warp * run; i0 < (warp + 1) * run && i0 < end - first && have < want; i0 += 32) {
                    const uint32_t i = first + i0 + lane;
                    const bool eq = i < end && lp_key(Piece<T>::one(x + i)) == floor;
                    const uint32_t b = __ballot_sync(0xffffffffu, eq), at = have + __popc(b & ((1u << lane) - 1));
                    if (eq && at < want) list[warp * kMaxTop + at] = (u64)floor << 32 | (0xffffffffu - i);
                    have += __popc(b);
                }
                if (lane == 0) slow[warp] = min(have, want);
                __syncthreads();
                if (t == 0) {
                    uint32_t at = n;
                    for (int i = 0; i < kWarps; i++)
                        for (uint32_t j = 0; j < (uint32_t)slow[i] && at < p.top; j++) best[at++] = list[i * kMaxTop + j];
                    // (the first CTA of several also holds the elements behind the last whole piece)
                    for (uint32_t i = max(tail, end); part == 0 && i < V && at < p.top; i++)
                        if (lp_key(Piece<T>::one(x + i)) == floor) best[at++] = (u64)floor << 32 | (0xffffffffu - i);
                }
            }
        }
    }
    __syncthreads();

    // ---- the row
    Sums r = whole;
    const u64 *order = best;
    if (parts > 1) {
        lp_cluster_sync();
        if (part == 0) {
            for (uint32_t i = 1; i < parts; i++) {
                const uint32_t at = lp_mapa(&whole, i);
                lp_join(r, Sums{lp_remote_f32(at), lp_remote_f32(at + 4), lp_remote_f32(at + 8)});
            }
            for (uint32_t i = t; i < parts * p.top; i += kThreads)
                all[i] = lp_remote_u64(lp_mapa(best + i % p.top, i / p.top));
        }
        __syncthreads();
        lp_cluster_sync();                                // nobody leaves while its part is being read
        if (part != 0) return;
        for (uint32_t i = t; i < parts * p.top; i += kThreads) {
            const u64 mine = all[i];
            uint32_t before = 0;
            for (uint32_t j = 0; j < parts * p.top; j++) before += all[j] > mine;
            if (mine && before < p.top) list[before] = mine;
        }
        __syncthreads();
        order = list;
    }
    const float log_s = logf(r.s);
    if (t == 0) p.entropy[row] = log_s - r.u / r.s;
    for (uint32_t j = t; j < p.n_targets; j += kThreads) {
        const uint32_t id = p.targets[(size_t)row * p.n_targets + j];
        p.logprobs[(size_t)row * p.n_targets + j] = id < V ? (Piece<T>::one(x + id) - r.m) - log_s : CUDART_NAN_F;
    }
    if (t < p.top) {
        const u64 o = order[t];
        const size_t at = (size_t)row * p.top + t;
        p.top_ids[at] = 0xffffffffu - (uint32_t)o;
        p.top_logprobs[at] = (lp_value((uint32_t)(o >> 32)) - r.m) - log_s;
    }
}

// TokenLogprobs(F16): logits [Rows, Vocab], targets u32[Rows * Targets], logprobs f32[Rows * Targets],
// entropy f32[Rows], top_ids u32[Rows * Top], top_logprobs f32[Rows * Top]; {Vocab, Rows, Targets, Top}
template <typename T> int run_logprobs(Launch &l, const char *name)
{
    LpParams p{};
    p.vocab = u32_at(l.u, 0); p.rows = u32_at(l.u, 4); p.n_targets = u32_at(l.u, 8); p.top = u32_at(l.u, 12);
    l.ws_need = 0;
    const auto holds = [&](int b, uint64_t n) { return l.len[b] == 0xffffffffu || l.len[b] >= n; };
    const uint64_t rows = p.rows;
    if (p.vocab == 0 || !holds(0, rows * p.vocab) || !holds(1, rows * p.n_targets) || !holds(2, rows * p.n_targets) ||
        !holds(3, rows) || !holds(4, rows * p.top) || !holds(5, rows * p.top))
        return fail(AB_ERR_INVALID, "%s: Vocab=%u Rows=%u Targets=%u Top=%u and the lengths block says logits[%u] targets[%u] "
                    "logprobs[%u] entropy[%u] top_ids[%u] top_logprobs[%u]", name, p.vocab, p.rows, p.n_targets, p.top,
                    l.len[0], l.len[1], l.len[2], l.len[3], l.len[4], l.len[5]);
    if (p.top > kMaxTop || p.top > p.vocab)
        return fail(AB_ERR_INVALID, "%s: %u alternatives of a vocabulary of %u; at most %u", name, p.top, p.vocab, kMaxTop);
    if (p.rows > 0x0fffffffu || p.vocab > 0x7fffffffu)
        return fail(AB_ERR_INVALID, "%s: %u rows of %u logits", name, p.rows, p.vocab);
    if (l.query_ws || p.rows == 0) return AB_OK;
    p.x = l.b[0];
    p.targets = ptr<const uint32_t>(l, 1);
    p.logprobs = ptr<float>(l, 2); p.entropy = ptr<float>(l, 3);
    p.top_ids = ptr<uint32_t>(l, 4); p.top_logprobs = ptr<float>(l, 5);
    // few rows: a row over several CTAs, as long as each has a step of every thread to do (16 rows of 128256 logits: 9.0 us
    // against 19.1 with a CTA a row; 1 of 32000: 7.1 against 7.5; 148 of 32000: 11.1 against 11.4)
    uint32_t parts = 1;
    while (parts < 8 && rows * parts * 2 <= 2ull * sm_count() && p.vocab >= parts * 2 * kThreads * 16 / 2) parts *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.rows * parts);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = l.stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = parts > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, p, parts);
    count_launch();
    note_selection("%s: %u CTA(s) per row", name, parts);
    return check_cuda(e, name);
}

}  // namespace

int launch_token_logprobs(Launch &l) { return run_logprobs<float>(l, "TokenLogprobs"); }
int launch_token_logprobs_f16(Launch &l) { return run_logprobs<__half>(l, "TokenLogprobsF16"); }

}  // namespace ab
