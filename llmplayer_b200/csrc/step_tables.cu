// What a batch of sequences that continue one prompt needs of its cache: a step's tables built from the sequences' lengths, and
// pages copied for new forks.
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
