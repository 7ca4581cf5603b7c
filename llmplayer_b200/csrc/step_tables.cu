// What a batch of sequences that continue one prompt needs of its cache: a step's tables built from the sequences' lengths, and
// pages copied for new forks.
#include "common.cuh"

namespace {

// ============================================================================ tables of a step
// Sequence b holds first[b] positions and brings count[b] new tokens. Its blocks of page_size positions lie in the shared
// pages as far as these reach and behind them in pages of its own, which `own` lists sequence after sequence. Where a sequence's tokens
// and own pages begin are sums over the sequences before it; every CTA forms those it needs itself (a few thousand integers at most,
// from L2), so one launch does and nothing has to be zero before it. Bound by latency: 3 us for 8 sequences, 4.3 us for 250 sequences of
// up to 130 tokens on 500 shared pages (B200; 0.67 MB, 0.1 us of memory time). A long sequence is shared by the CTAs along y.
__device__ __forceinline__ int blocks_of(int length, int page_size) { return length > 0 ? (length - 1) / page_size + 1 : 0; }
// Lengths that no cache has wrap around: what lies outside a tensor is left out by its unsigned index.
__device__ __forceinline__ int plus(int a, int b) { return (int)((unsigned)a + (unsigned)b); }

__device__ __forceinline__ int block_sum_int(int v, int* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = plus(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < (blockDim.x >> 5); ++w) total = plus(total, scratch[w]);
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
        const int more = max(count[i], 0);
        before = plus(before, more);
        own_before = plus(own_before, max(0, blocks_of(plus(first[i], more), page_size) - num_shared));
    }
    before = block_sum_int(before, scratch);
    own_before = block_sum_int(own_before, scratch);
    const int from = first[b], n = max(count[b], 0), length = plus(from, n), blocks = blocks_of(length, page_size);
    const int step = gridDim.y * blockDim.x, i0 = blockIdx.y * blockDim.x + threadIdx.x;
    if (q_start && i0 == 0) {
        q_start[b] = before;
        kv_len[b] = length;
        if (b == B - 1) q_start[B] = plus(before, n);
    }
    if (positions)
        for (int i = i0; i < min(n, tokens); i += step)
            if ((unsigned)plus(before, i) < (unsigned)tokens) {
                positions[plus(before, i)] = plus(from, i);
                seq_ids[plus(before, i)] = b;
            }
    for (int i = i0; i < width; i += step) {
        int page = 0;
        if (i < blocks) {
            const int at = plus(own_before, i - num_shared);
            page = i < num_shared ? shared[i] : ((unsigned)at < (unsigned)num_own ? own[at] : 0);
        }
        table[(long long)b * width + i] = page;
    }
}

// ============================================================================ copies of pages
// Pairs of pages travel as an argument of the launch: nothing is uploaded, and what the host checked is what is copied. Bound by memory:
// a page of a run is 32 to 256 KB, read once (its further copies come from L2) and written once per target. B200: 60 copies in 32 runs of
// 256 KB (512 MB) 84 us, 93 % of the measured copy rate.
constexpr int PAIRS = 448, FEW_PAIRS = 16;
template <int N> struct PagePairs { int from[N], to[N]; };

template <int N>
__global__ void __launch_bounds__(256)
copy_pages_kernel(uint4* __restrict__ storage, long long run_stride, int page_vectors, const __grid_constant__ PagePairs<N> pairs) {
    lp_grid_wait();
    lp_grid_release();
    uint4* run = storage + blockIdx.z * run_stride;
    const uint4* src = run + (long long)pairs.from[blockIdx.y] * page_vectors;
    uint4* dst = run + (long long)pairs.to[blockIdx.y] * page_vectors;
    const int i0 = blockIdx.x * 1024 + threadIdx.x;              // four vectors per thread, asked for together
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (i0 + u * 256 < page_vectors) v[u] = src[i0 + u * 256];
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (i0 + u * 256 < page_vectors) dst[i0 + u * 256] = v[u];
}

template <int N>
int launch_copies(void* storage, int runs, long long run_stride, int vectors, const int* from, const int* to, int n, cudaStream_t stream) {
    PagePairs<N> pairs = {};
    for (int i = 0; i < n; ++i) {
        pairs.from[i] = from[i];
        pairs.to[i] = to[i];
    }
    lp_launch(copy_pages_kernel<N>, dim3((vectors + 1023) / 1024, n, runs), dim3(256), 0, stream, (uint4*)storage, run_stride, vectors, pairs);
    return lp_check_launch("copy_pages");
}

}  // namespace

// first, count int32 [B]; shared [num_shared], own [num_own] page numbers; table [B, width]; the others may be null, together:
// q_start [B + 1], kv_len [B], positions and seq_ids [tokens].
extern "C" int lp_step_tables(const int* first, const int* count, const int* shared, int num_shared, const int* own, int num_own, int* q_start,
                              int* kv_len, int* positions, int* seq_ids, int tokens, int* table, int width, int B, int page_size, cudaStream_t stream) {
    // indexes run past an end by a step of the grid at most
    const int most = 0x7fffffff - 64 * 256;
    if (B <= 0 || width <= 0 || width > most || num_shared < 0 || num_own < 0 || tokens < 0 || tokens > most || page_size <= 0)
        LP_REFUSE("step_tables: %d sequences, tables of %d pages, %d tokens", B, width, tokens);
    // four entries per thread or more
    const long long per_sequence = (tokens > (long long)B * width ? tokens / B : width) / 1024;
    const unsigned shares = (unsigned)(per_sequence < 1 ? 1 : per_sequence > 64 ? 64 : per_sequence);
    lp_launch(step_tables_kernel, dim3(B, shares), dim3(256), 0, stream, first, count, shared, num_shared, own, num_own, q_start, kv_len, positions,
              seq_ids, tokens, table, width, B, page_size);
    return lp_check_launch("step_tables");
}

extern "C" int lp_copy_pages_most() { return PAIRS; }

// storage: [runs, num_pages, page_bytes]; n page numbers to copy from and n to copy to, on the host.
extern "C" int lp_copy_pages(void* storage, int runs, long long num_pages, long long page_bytes, const int* pages, int n, cudaStream_t stream) {
    if (runs <= 0 || runs > 65535 || n <= 0 || n > PAIRS || page_bytes <= 0 || page_bytes % 16 || page_bytes / 16 > 0x7ffffbff || ((uintptr_t)storage & 15))
        LP_REFUSE("copy_pages: %d pairs of pages of %lld bytes in %d runs", n, page_bytes, runs);
    for (int i = 0; i < 2 * n; ++i)
        if (pages[i] < 0 || pages[i] >= num_pages) LP_REFUSE("copy_pages: page %d of %lld", pages[i], num_pages);
    const long long vectors = page_bytes / 16;
    if (n <= FEW_PAIRS) return launch_copies<FEW_PAIRS>(storage, runs, num_pages * vectors, (int)vectors, pages, pages + n, n, stream);
    return launch_copies<PAIRS>(storage, runs, num_pages * vectors, (int)vectors, pages, pages + n, n, stream);
}
