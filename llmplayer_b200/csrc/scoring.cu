// Log probabilities of given tokens, with the entropy of each distribution and its most likely tokens.
//
// For a row x of V logits and a token t:
//   log p[t] = x[t] - ln(sum_i exp(x[i])),   entropy = -sum_i p[i] ln p[i],
//   rank = how many tokens come before t in the order of falling logits (equal logits: the lower token first; a logit that
//   is not a number comes behind all others), and the first k tokens of that order with their log probabilities.
// Sums are taken against the row's maximum m over the others only: with c logits equal to m and r = sum of exp(x[i] - m) over
// the rest, ln(sum) = m + ln(c + r) is formed as log1p(c - 1 + r), so that a nearly certain token's log probability keeps its digits.
// A row without a distribution (it holds +inf or no number at all, or nothing but -inf) gets no number everywhere but in ranks and tokens.
#include "common.cuh"

namespace {

constexpr int THREADS = 512;
constexpr int MOST_TOP = 32;

// x before y in the order of the tokens
__device__ __forceinline__ bool before(float x, int i, float y, int j) {
    const bool nx = x != x, ny = y != y;
    if (nx || ny) return nx == ny ? i < j : ny;
    return x > y || (x == y && i < j);
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
token_logprobs_kernel(const T* __restrict__ logits, long long ld, const int* __restrict__ targets, float* __restrict__ logprob,
                      float* __restrict__ entropy, int* __restrict__ rank, int* __restrict__ top_ids, float* __restrict__ top_logprobs,
                      int V, int top) {
    __shared__ float scratch[32];
    __shared__ int best_at[32];
    lp_grid_wait();
    lp_grid_release();
    const T* x = logits + (long long)blockIdx.x * ld;
    const int target = targets[blockIdx.x];
    const bool real = target >= 0 && target < V;
    const float xt = real ? lp_to_float(x[target]) : 0.f;
    float m = -INFINITY;
    for (int i = threadIdx.x; i < V; i += THREADS) m = fmaxf(m, lp_to_float(x[i]));
    m = lp_block_max(m, scratch);
    float c = 0.f, r = 0.f, u = 0.f, ahead = 0.f;
    for (int i = threadIdx.x; i < V; i += THREADS) {
        const float v = lp_to_float(x[i]);
        if (v == m) c += 1.f;
        else {
            const float d = v - m, e = expf(d);
            r += e;
            if (e != 0.f) u += e * d;
        }
        if (real && before(v, i, xt, target)) ahead += 1.f;
    }
    c = lp_block_sum(c, scratch);
    r = lp_block_sum(r, scratch);
    u = lp_block_sum(u, scratch);
    ahead = lp_block_sum(ahead, scratch);
    const bool none = !(m > -INFINITY && m < INFINITY) || r != r;
    const float log_s = none ? NAN : log1pf((c - 1.f) + r);
    if (threadIdx.x == 0) {
        logprob[blockIdx.x] = real ? (xt - m) - log_s : NAN;
        entropy[blockIdx.x] = log_s - u / (c + r);
        rank[blockIdx.x] = real ? (int)ahead : -1;
    }
    float last = INFINITY;
    int last_at = -1;
    for (int k = 0; k < top; ++k) {                     // the first token behind the last one found
        float v = NAN;
        int at = V;
        for (int i = threadIdx.x; i < V; i += THREADS) {
            const float w = lp_to_float(x[i]);
            if ((k == 0 || before(last, last_at, w, i)) && (at == V || before(w, i, v, at))) { v = w; at = i; }
        }
        for (int o = 16; o > 0; o >>= 1) {
            const float w = __shfl_xor_sync(0xffffffffu, v, o);
            const int j = __shfl_xor_sync(0xffffffffu, at, o);
            if (j < V && (at == V || before(w, j, v, at))) { v = w; at = j; }
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 0) { scratch[threadIdx.x >> 5] = v; best_at[threadIdx.x >> 5] = at; }
        __syncthreads();
        for (int w = 0; w < THREADS / 32; ++w)
            if (best_at[w] < V && (at == V || before(scratch[w], best_at[w], v, at))) { v = scratch[w]; at = best_at[w]; }
        last = v;
        last_at = at;
        if (threadIdx.x == 0) {
            top_ids[(long long)blockIdx.x * top + k] = at;
            top_logprobs[(long long)blockIdx.x * top + k] = (v - m) - log_s;
        }
    }
}

}  // namespace

extern "C" int lp_token_logprobs_most_top() { return MOST_TOP; }

// logits: rows of `ld` elements (float32 or bfloat16); targets, rank int32 [rows]; logprob, entropy float32 [rows];
// top_ids int32, top_logprobs float32 [rows, top] (null for top == 0).
extern "C" int lp_token_logprobs(const void* logits, int dtype, long long ld, const int* targets, float* logprob, float* entropy, int* rank,
                                 int* top_ids, float* top_logprobs, int rows, int V, int top, cudaStream_t stream) {
    if (rows <= 0 || V <= 0 || top < 0 || top > MOST_TOP || top > V || ld < V) LP_REFUSE("token_logprobs: %d rows of %d logits, the %d most likely", rows, V, top);
    if (dtype == LP_F32)
        lp_launch(token_logprobs_kernel<float>, dim3(rows), dim3(THREADS), 0, stream, (const float*)logits, ld, targets, logprob, entropy, rank,
                  top_ids, top_logprobs, V, top);
    else
        lp_launch(token_logprobs_kernel<__nv_bfloat16>, dim3(rows), dim3(THREADS), 0, stream, (const __nv_bfloat16*)logits, ld, targets, logprob,
                  entropy, rank, top_ids, top_logprobs, V, top);
    return lp_check_launch("token_logprobs");
}
