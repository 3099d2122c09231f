// Log probabilities of given tokens, the distribution's entropy, and the most probable alternatives,
// of every row of logits.  No counterpart in the reference.
//
//     m = max x,  s = sum e^(x - m),  logprob(t) = (x_t - m) - log s,
//     entropy = -sum p log p = log s - (sum (x - m) e^(x - m)) / s
//
// and the Top largest logits in (value descending, index ascending) order with their log
// probabilities; -0 equals +0 and a NaN is larger than every number.  A logit of -inf is a token of
// probability 0 and adds nothing to the entropy.  A row that holds a NaN or a +inf, or nothing above
// -inf, has no distribution: its log probabilities and entropy are NaN (its indices still stand).  A
// target at or past Vocab has the log probability NaN.
#include <math_constants.h>

#include "common.cuh"

namespace ab {

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxTop = 32;

template <typename T> __device__ __forceinline__ float lp_f32(T x);
template <> __device__ __forceinline__ float lp_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float lp_f32<__half>(__half x) { return __half2float(x); }

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

struct LpParams {
    const void *x;
    const uint32_t *targets;
    float *logprobs, *entropy;
    uint32_t *top_ids;
    float *top_logprobs;
    uint32_t vocab, rows, n_targets, top;
};

// One CTA per row, the row read once for the maximum, once for the sums and once for each alternative.
template <typename T> __global__ void __launch_bounds__(kThreads) logprobs_simple_kernel(const LpParams p)
{
    __shared__ float shf[2][kThreads];
    __shared__ unsigned long long shk[kThreads];
    const uint32_t row = blockIdx.x, t = threadIdx.x, V = p.vocab;
    const T *x = static_cast<const T *>(p.x) + (size_t)row * V;
    uint32_t best = 0;
    for (uint32_t i = t; i < V; i += kThreads) best = max(best, lp_key(lp_f32(x[i])));
    shk[t] = best;
    __syncthreads();
    for (int w = kThreads / 2; w; w /= 2) {
        if (t < (uint32_t)w) shk[t] = max(shk[t], shk[t + w]);
        __syncthreads();
    }
    const float m = lp_value((uint32_t)shk[0]);
    __syncthreads();
    float s = 0.f, u = 0.f;
    for (uint32_t i = t; i < V; i += kThreads) {
        const float d = lp_f32(x[i]) - m, e = expf(d);
        s += e;
        u = fmaf(fmaxf(d, -1000.f), e, u);               // -inf * 0 is a NaN
    }
    shf[0][t] = s; shf[1][t] = u;
    __syncthreads();
    for (int w = kThreads / 2; w; w /= 2) {
        if (t < (uint32_t)w) { shf[0][t] += shf[0][t + w]; shf[1][t] += shf[1][t + w]; }
        __syncthreads();
    }
    const float log_s = logf(shf[0][0]);
    if (t == 0) p.entropy[row] = log_s - shf[1][0] / shf[0][0];
    for (uint32_t j = t; j < p.n_targets; j += kThreads) {
        const uint32_t id = p.targets[(size_t)row * p.n_targets + j];
        p.logprobs[(size_t)row * p.n_targets + j] = id < V ? (lp_f32(x[id]) - m) - log_s : CUDART_NAN_F;
    }
    unsigned long long last = ~0ull;                      // key and the index's complement: larger comes first
    for (uint32_t r = 0; r < p.top; r++) {
        unsigned long long b = 0;
        for (uint32_t i = t; i < V; i += kThreads) {
            const unsigned long long k = (unsigned long long)lp_key(lp_f32(x[i])) << 32 | (0xffffffffu - i);
            if ((r == 0 || k < last) && k > b) b = k;
        }
        __syncthreads();
        shk[t] = b;
        __syncthreads();
        for (int w = kThreads / 2; w; w /= 2) {
            if (t < (uint32_t)w) shk[t] = max(shk[t], shk[t + w]);
            __syncthreads();
        }
        last = shk[0];
        if (t == 0) {
            const size_t o = (size_t)row * p.top + r;
            p.top_ids[o] = 0xffffffffu - (uint32_t)last;
            p.top_logprobs[o] = (lp_value((uint32_t)(last >> 32)) - m) - log_s;
        }
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
    if (p.rows > 0x7fffffffu) return fail(AB_ERR_INVALID, "%s: %u rows", name, p.rows);
    if (l.query_ws || p.rows == 0) return AB_OK;
    p.x = l.b[0];
    p.targets = ptr<const uint32_t>(l, 1);
    p.logprobs = ptr<float>(l, 2); p.entropy = ptr<float>(l, 3);
    p.top_ids = ptr<uint32_t>(l, 4); p.top_logprobs = ptr<float>(l, 5);
    logprobs_simple_kernel<T><<<p.rows, kThreads, 0, l.stream>>>(p);
    count_launch();
    note_selection("%s: a CTA per row", name);
    return check_cuda(cudaGetLastError(), name);
}

}  // namespace

int launch_token_logprobs(Launch &l) { return run_logprobs<float>(l, "TokenLogprobs"); }
int launch_token_logprobs_f16(Launch &l) { return run_logprobs<__half>(l, "TokenLogprobsF16"); }

}  // namespace ab
