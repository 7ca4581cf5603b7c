// What a batch of sequences that continue one prompt needs beside its products: a step's tables built from the sequences'
// lengths, pages of the cache copied for new forks, and attention over pages that all sequences share.
#include "common.cuh"

namespace {

// ============================================================================ tables of a step
// Sequence b holds first[b] positions and brings count[b] new tokens. Its blocks of page_size positions lie in the shared
// pages as far as these reach and behind them in pages of its own, which `own` lists sequence after sequence.
__device__ __forceinline__ int blocks_of(int length, int page_size) { return length > 0 ? (length + page_size - 1) / page_size : 0; }

__device__ __forceinline__ int block_sum_int(int v, int* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < (blockDim.x >> 5); ++w) total += scratch[w];
    return total;
}

__global__ void __launch_bounds__(256)
step_tables_kernel(const int* __restrict__ first, const int* __restrict__ count, const int* __restrict__ shared, int num_shared,
                   const int* __restrict__ own, int num_own, int* __restrict__ q_start, int* __restrict__ kv_len,
                   int* __restrict__ positions, int* __restrict__ seq_ids, int tokens, int* __restrict__ table, int width, int B, int page_size) {
    __shared__ int scratch[32];
    lp_grid_wait();
    lp_grid_release();
    const int b = blockIdx.x;
    int before = 0, own_before = 0;
    for (int i = threadIdx.x; i < b; i += blockDim.x) {
        before += max(count[i], 0);
        own_before += max(0, blocks_of(first[i] + count[i], page_size) - num_shared);
    }
    before = block_sum_int(before, scratch);
    own_before = block_sum_int(own_before, scratch);
    const int from = first[b], n = max(count[b], 0), length = from + n, blocks = blocks_of(length, page_size);
    if (q_start && threadIdx.x == 0) {
        q_start[b] = before;
        kv_len[b] = length;
        if (b == B - 1) q_start[B] = before + n;
    }
    if (positions)
        for (int i = threadIdx.x; i < n; i += blockDim.x)
            if (before + i < tokens) {
                positions[before + i] = from + i;
                seq_ids[before + i] = b;
            }
    for (int i = threadIdx.x; i < width; i += blockDim.x) {
        int page = 0;
        if (i < blocks) {
            const int at = own_before + i - num_shared;
            page = i < num_shared ? shared[i] : (at < num_own ? own[at] : 0);
        }
        table[(long long)b * width + i] = page;
    }
}

// ============================================================================ copies of pages
// Pairs of pages travel as an argument of the launch: nothing is uploaded, and what the host checked is what is copied.
constexpr int PAIRS = 448;
struct PagePairs { int from[PAIRS], to[PAIRS]; };

__global__ void __launch_bounds__(256)
copy_pages_kernel(uint4* __restrict__ storage, long long run_stride, int page_vectors, const __grid_constant__ PagePairs pairs) {
    lp_grid_wait();
    lp_grid_release();
    uint4* run = storage + blockIdx.z * run_stride;
    const uint4* src = run + (long long)pairs.from[blockIdx.y] * page_vectors;
    uint4* dst = run + (long long)pairs.to[blockIdx.y] * page_vectors;
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < page_vectors; i += gridDim.x * blockDim.x) dst[i] = src[i];
}

// ============================================================================ attention
// One warp per query token and head: keys 32 at a time, a lane per key for the scores, a lane per features for the values.
__global__ void __launch_bounds__(128)
attention_shared_kernel(const __nv_bfloat16* __restrict__ q, __nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ pages,
                        const int* __restrict__ table, int width, const int* __restrict__ q_start, const int* __restrict__ kv_len, int B, int T,
                        int H, int G, int hd, int shared_pages, float scale_log2) {
    lp_grid_wait();
    lp_grid_release();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int at = blockIdx.x * 4 + warp;
    const int t = at / H, h = at % H, g = h / (H / G);
    if (t >= T) return;
    int b = 0;
    while (b < B && q_start[b + 1] <= t) ++b;
    if (b >= B) return;                                      // behind the last sequence
    const int pos = kv_len[b] - (q_start[b + 1] - t);
    const __nv_bfloat16* query = q + ((long long)t * H + h) * hd;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 <= pos; k0 += 32) {
        const int block = k0 >> 6;
        const int page = table[(long long)(block < shared_pages ? 0 : b) * width + block];
        const __nv_bfloat16* k = pages + (((long long)page * 2 * G + g) * 64 + (k0 & 63)) * hd;
        const __nv_bfloat16* v = k + (long long)G * 64 * hd;
        float s = 0.f;
        for (int d = 0; d < hd; ++d) s += __bfloat162float(query[d]) * __bfloat162float(k[lane * hd + d]);
        s = k0 + lane <= pos ? s * scale_log2 : -INFINITY;
        const float mn = fmaxf(m, lp_warp_max(s));
        const float f = exp2f(m - mn), e = exp2f(s - mn);
        m = mn;
        l = l * f + lp_warp_sum(e);
        for (int u = 0; u < hd / 32; ++u) o[u] *= f;
        for (int j = 0; j < 32 && k0 + j <= pos; ++j) {
            const float w = __shfl_sync(0xffffffffu, e, j);
            for (int u = 0; u < hd / 32; ++u) o[u] += w * __bfloat162float(v[j * hd + u * 32 + lane]);
        }
    }
    for (int u = 0; u < hd / 32; ++u)
        out[((long long)t * H + h) * hd + u * 32 + lane] = __float2bfloat16_rn(l > 0.f ? o[u] / l : 0.f);
}

}  // namespace

// first, count int32 [B]; shared [num_shared], own [num_own] page numbers; table [B, width]; the others may be null, together:
// q_start [B + 1], kv_len [B], positions and seq_ids [tokens].
extern "C" int lp_step_tables(const int* first, const int* count, const int* shared, int num_shared, const int* own, int num_own, int* q_start,
                              int* kv_len, int* positions, int* seq_ids, int tokens, int* table, int width, int B, int page_size, cudaStream_t stream) {
    if (B <= 0 || width <= 0 || num_shared < 0 || num_own < 0 || tokens < 0 || page_size <= 0) LP_REFUSE("step_tables: %d sequences, tables of %d pages", B, width);
    lp_launch(step_tables_kernel, dim3(B), dim3(256), 0, stream, first, count, shared, num_shared, own, num_own, q_start, kv_len, positions,
              seq_ids, tokens, table, width, B, page_size);
    return lp_check_launch("step_tables");
}

extern "C" int lp_copy_pages_most() { return PAIRS; }

// storage: [runs, num_pages, page_bytes]; pairs of page numbers on the host.
extern "C" int lp_copy_pages(void* storage, int runs, long long num_pages, long long page_bytes, const int* from, const int* to, int n, cudaStream_t stream) {
    if (runs <= 0 || runs > 65535 || n <= 0 || n > PAIRS || page_bytes <= 0 || page_bytes % 16 || page_bytes / 16 > 0x7fffffff || ((uintptr_t)storage & 15))
        LP_REFUSE("copy_pages: %d pairs of pages of %lld bytes in %d runs", n, page_bytes, runs);
    PagePairs pairs = {};
    for (int i = 0; i < n; ++i) {
        if (from[i] < 0 || from[i] >= num_pages || to[i] < 0 || to[i] >= num_pages) LP_REFUSE("copy_pages: pages %d and %d of %lld", from[i], to[i], num_pages);
        pairs.from[i] = from[i];
        pairs.to[i] = to[i];
    }
    const int vectors = (int)(page_bytes / 16);
    lp_launch(copy_pages_kernel, dim3((vectors + 1023) / 1024, n, runs), dim3(256), 0, stream, (uint4*)storage, num_pages * (page_bytes / 16), vectors, pairs);
    return lp_check_launch("copy_pages");
}

// q, out: bf16 [T, H, hd]; pages bf16 [num_pages, 2, G, 64, hd]; table int32 [B, width], whose first shared_pages columns are
// the same in every row; q_start int32 [B + 1]; kv_len int32 [B], lengths with the new tokens.
extern "C" int lp_attention_shared(const void* q, void* out, const void* pages, const int* table, int width, const int* q_start, const int* kv_len,
                                   int B, int T, int H, int G, int hd, int shared_pages, float scale, cudaStream_t stream) {
    if (B <= 0 || T <= 0 || G <= 0 || H % G || (hd != 64 && hd != 128) || shared_pages < 0 || shared_pages > width)
        LP_REFUSE("attention_shared: %d sequences, %d tokens, %d heads on %d of %d, %d shared pages", B, T, H, G, hd, shared_pages);
    lp_launch(attention_shared_kernel, dim3((T * H + 3) / 4), dim3(128), 0, stream, (const __nv_bfloat16*)q, (__nv_bfloat16*)out,
              (const __nv_bfloat16*)pages, table, width, q_start, kv_len, B, T, H, G, hd, shared_pages, scale * 1.4426950408889634f);
    return lp_check_launch("attention_shared");
}
