// Attention of a batch whose sequences share their first pages: the shared pages are read once for the whole batch.
//
//   out[t, h] = softmax(scale * q[t, h] . K) V over the keys up to the token's own position. The keys fall into two ranges, the shared
//   pages and the sequence's own pages behind them; a range gives (m, l, o) = (maximum, sum of exp(s - m), sum of exp(s - m) v), and
//   ranges are joined by bringing their sums to the common maximum.
//
//   shared pages   One kernel over the new tokens of ALL sequences at once: for a key/value head the rows of the products are the
//                  (token, query head) pairs, and neither the products nor the softmax knows sequences. With 64 sequences and 4 query heads
//                  per key head that is 256 rows on one read of the keys, instead of 64 reads. Tensor memory, tcgen05.
//   own pages      One kernel per step form (a single token per sequence, several tokens) takes the sequence's own pages with
//                  mma.sync, then joins its result with what the first kernel left in float32. Its reads of its own pages
//                  begin before the first kernel's results are there (programmatic launch), as far as the SMs have room. Few rows of
//                  several tokens have many results, which a third kernel joins.
//
// B200, 32 query heads on 8, calls one behind the other in a graph, each on a cache that has left L2, against attention that reads every sequence's pages:
//   64 single tokens, heads of 128, 128 shared pages, up to 250 own positions each: 26.7 us against 427; the two kernels by
//       themselves 21 and 15 us for 70 MB (10.8 us at the measured copy rate).
//   24 sequences of 9 to 37 tokens, heads of 64, 50 shared pages: 33.8 against 223; 33 and 12 us, by themselves and cold, for 15 GFLOP.
//   40 sequences of 47 to 190 tokens, heads of 128, 500 shared pages: 1,890 against 5,500, 1,298 TFLOP/s, 80 % of the measured rate of
//       dense products (96 us of it the second kernel); 2,100 over a long run, where the power limit holds the clock down.
//
// All sums, maxima and partial results are float32. The softmax weights enter the products with the values as bfloat16, rounded
// against a reference maximum (as in the other attention kernels here); the row sums use the float32 weights.
// Every mbarrier wait is bounded; a wait that runs out sets *status and the CTA winds down.
#include "tcgen05_utils.cuh"
#include "attention_decode.cuh"

namespace {

constexpr int ROWS = 128;                 // rows of a product: (token, query head) pairs of one key/value head
constexpr int THREADS = 384;              // warp 0: loader, warps 1 and 2: the chains' products (3: nothing), warps 4-7 and 8-11: their softmaxes
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_ABOVE = 8.0f;     // log2: how far a row's reference maximum may lag behind its maximum (a factor of 256)

// ============================================================================ the shared pages
// A CTA has two chains of products and softmaxes, so that the tensor cores and the exponential units are both busy. With two tiles of
// rows each chain has one, and both read each page from the same stage; with a single tile the chains share it and take
// alternate pages (their results are two partial ones). Per page and chain:
//   S[128 x 64] = Q K^T (tensor memory)  ->  a thread per row: maximum, exp2, sum, weights as bfloat16 over S in tensor memory
//   ->  O[128 x HD] += P V (P from tensor memory, V from shared memory, contiguous in N).
// A chain has two S tiles: the scores of its next page are asked for before it has finished with one. (With one tile of 128 keys
// per chain the two chains' softmaxes ran one behind the other: 4,000 cycles per 128 keys at heads of 128.)
// What bounds it: a page of 64 keys takes both chains 1,550 to 1,600 cycles. The products alone take 1,650 back to back at heads of 128 (half of
// that at 64); a chain's page has 600 cycles of exponentials (64 per thread, 8 cycles per warp: the exp2 unit's rate) and 600 of waiting,
// loading, the maximum and the store. At the 500 pages above these took longer than the 1,870 to 1,900 us: chains that take no turns 2,060 (and 529
// against 472 at heads of 64, 300 pages), turns of whole chains 2,386, two groups of softmax warps per chain 2,061, blocks of 128 keys on
// two threads per row 2,526, weights in tiles of their own and scores given back early 2,150. A polynomial for a quarter of the
// exponentials gained 5 % at heads of 64 without turns, and lost with them.
template <int HD> struct Shape {
    static constexpr int BLOCKS = HD / 64;                          // blocks of 64 features (one swizzle row each)
    static constexpr int TILE = PAGE * HD * 2;                      // keys or values of a page
    static constexpr int Q_TILE = ROWS * HD * 2;
    static constexpr int SLOTS = HD == 64 ? 16 : 8;                 // a power of two: which slot and which round are bits of a tile's place
    static constexpr int SMEM = 2 * Q_TILE + SLOTS * TILE + 1024 /* alignment */ + 512 /* barriers */ + 2 * ROWS * 4 /* positions */;
    static constexpr int OUT_ROW = HD * 4 + 16;                     // a row of results on its way out: where queries and ring were
    static_assert(SMEM <= 227 * 1024 && 2 * ROWS * OUT_ROW <= 2 * Q_TILE + SLOTS * TILE && (SLOTS & (SLOTS - 1)) == 0, "");
    static constexpr int S_COL = 0, O_COL = 256;                    // chain c: S at 128 c and 128 c + 64, O at 256 + HD c
    static constexpr int TMEM_COLS = 512;
};

// The products are issued by a whole warp of which one thread is elected: values that the compiler knows to be alike in all lanes stay
// in uniform registers.
__device__ __forceinline__ bool elect_one() {
    uint32_t leader;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
    return leader != 0;
}
// A product whose first operand lies in tensor memory.
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Two float32 operations in one instruction (Blackwell's packed forms).
__device__ __forceinline__ void fma2(float& x0, float& x1, float a, float b) {            // x = x * a + b
    uint64_t vx, va, vb;
    asm("mov.b64 %0, {%1, %2};" : "=l"(vx) : "f"(x0), "f"(x1));
    asm("mov.b64 %0, {%1, %1};" : "=l"(va) : "f"(a));
    asm("mov.b64 %0, {%1, %1};" : "=l"(vb) : "f"(b));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(vx) : "l"(vx), "l"(va), "l"(vb));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x0), "=f"(x1) : "l"(vx));
}
__device__ __forceinline__ void add2(float& x0, float& x1, float y0, float y1) {
    uint64_t vx, vy;
    asm("mov.b64 %0, {%1, %2};" : "=l"(vx) : "f"(x0), "f"(x1));
    asm("mov.b64 %0, {%1, %2};" : "=l"(vy) : "f"(y0), "f"(y1));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(vx) : "l"(vx), "l"(vy));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x0), "=f"(x1) : "l"(vx));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

struct SharedArgs {
    const __nv_bfloat16* kv;     // [num_pages, 2, G, PAGE, HD]
    long long num_pages;
    const int* table;            // the first row of the page table: its first `pages` entries are the shared pages
    const int* q_start;          // [B + 1]
    const int* kv_len;           // [B]
    float* part_o;               // [slots][T][H][HD]
    float* part_ml;              // [slots][T][H][2]: maximum (log2 units of the scaled scores) and sum
    int B, T, H, G, R, pages, splits;
    float scale_log2;
    int* status;
};

// grid: (splits x pairs of row tiles, G); a split takes consecutive pages.
template <int HD>
__global__ void __launch_bounds__(THREADS, 1)
attention_shared_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv, const SharedArgs a) {
    using SH = Shape<HD>;
    constexpr int SLOTS = SH::SLOTS, TILE = SH::TILE;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* q_tiles = smem;
    uint8_t* ring = smem + 2 * SH::Q_TILE;
    uint64_t* full = (uint64_t*)(ring + SLOTS * TILE);             // [SLOTS]
    uint64_t* empty = full + SLOTS;                                // [SLOTS]
    uint64_t* q_full = empty + SLOTS;
    uint64_t* s_ready = q_full + 1;                                // [chain][tile] scores are in tensor memory
    uint64_t* p_ready = s_ready + 4;                               // [chain][tile] weights are
    uint64_t* o_ready = p_ready + 4;                               // [chain] weights times values have been added
    uint32_t* tmem_slot = (uint32_t*)(o_ready + 2);
    int* position = (int*)((uint8_t*)full + 512);                  // [2 ROWS]: of the CTA's tokens, -1: nobody's
    static_assert((2 * SLOTS + 11) * 8 + 4 <= 512, "");

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;       // alike in all lanes
    const int per_tile = ROWS / a.R, tiles = (a.T + per_tile - 1) / per_tile;
    const int pair = blockIdx.x / a.splits, split = blockIdx.x - pair * a.splits, g = blockIdx.y;
    const bool alone = tiles == 1;                                 // one tile of rows: the chains take alternate pages
    const int chains = alone || pair * 2 + 1 < tiles ? 2 : 1;
    const int t0 = pair * 2 * per_tile;
    const int first = (int)((long long)a.pages * split / a.splits), n = (int)((long long)a.pages * (split + 1) / a.splits) - first;
    // A chain's k-th page is page k of the share, or every second one. Tiles come in the order in which the products take them: two
    // pages' keys, then the values of a page and the keys of the page two behind it. Chains that take alternate pages have half of the
    // slots each: whoever waits for a slot's tile must have seen the tile before it there, as a parity tells only a round from the last.
    const int streams = alone ? 2 : 1, slots = SLOTS / streams, slots_log2 = 31 - __clz(slots);
    auto page_of = [&](int k, int c) { return alone ? 2 * k + c : k; };
    auto turns = [&](int c) { return alone ? (n + 1 - c) / 2 : c < chains ? n : 0; };
    auto keys_at = [&](int k) { return k < 2 ? k : 2 * k - 1; };
    auto values_at = [&](int k, int count) { return min(count, 2 + k) + k; };
    auto slot_of = [&](int at, int c) { return (alone ? c * slots : 0) + (at & (slots - 1)); };
    auto round_of = [&](int at) { return (at >> slots_log2) & 1; };

    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_kv) : "memory");
        mbar_init(q_full, 1);
        for (int s = 0; s < SLOTS; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], alone ? 1 : chains); }
        for (int i = 0; i < 4; ++i) { mbar_init(&s_ready[i], 1); mbar_init(&p_ready[i], 4); }
        mbar_init(&o_ready[0], 1);
        mbar_init(&o_ready[1], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)SH::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    lp_grid_wait();
    lp_grid_release();             // behind the wait: what the kernel for the own pages reads early is then there

    if (warp == 0) {
        // ------------------------------------------------------------ loader
        if (lane == 0) {
            const int q_tiles_here = alone ? 1 : chains;
            const uint32_t q_bytes = (uint32_t)(per_tile * a.R * 128 * SH::BLOCKS);
            mbar_expect_tx(q_full, q_bytes * q_tiles_here);
            for (int c = 0; c < q_tiles_here; ++c)
#pragma unroll
                for (int f = 0; f < SH::BLOCKS; ++f)
                    tma_load_3d(q_tiles + c * SH::Q_TILE + f * (ROWS * 128), &map_q, f * 64, g * a.R, t0 + c * per_tile, q_full);
        }
        // The lanes hold page numbers (lane j those of pages j, j + 32, ... of the share, the last two of them), so that a request does not
        // begin with a round trip to memory.
        int held = lane < n ? a.table[first + lane] : 0, before = 0, loaded = 32;
        int at[2] = {0, 0};                                        // tiles asked for, per stream
        int reached = 0;                                           // the greatest length
        bool ok = true;
        auto request = [&](int k, int c, int which) {
            const int i = page_of(k, c);
            if (i >= loaded) {                                     // keys run ahead of values by less than 32 pages
                before = held;
                held = loaded + lane < n ? a.table[first + loaded + lane] : 0;
                loaded += 32;
            }
            const int page = __shfl_sync(0xffffffffu, i >= loaded - 32 ? held : before, i & 31);
            const int s = slot_of(at[c], c);
            ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], round_of(at[c]) ^ 1));
            if (!ok) { if (lane == 0) atomicExch(a.status, 81); return; }
            const int filled = which ? reached - (first + i) * PAGE : PAGE;
            if (filled < PAGE) {
                // Behind the longest sequence values may be no numbers, and no weight of zero takes them out: the page is brought in by hand.
                const __nv_bfloat16* from = a.kv + ((long long)(page * 2ll + 1) * a.G + g) * (PAGE * HD);
                for (int x = lane; x < PAGE * (HD / 8); x += 32) {
                    const int r = x / (HD / 8), chunk = x % (HD / 8);
                    const bool there = r < filled && page >= 0 && page < a.num_pages;
                    *reinterpret_cast<uint4*>(ring + s * TILE + tile_offset<true>(r, chunk, HD, HD / 8)) =
                        there ? *reinterpret_cast<const uint4*>(from + r * HD + chunk * 8) : make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[s]);
            } else if (lane == 0) {
                mbar_expect_tx(&full[s], (uint32_t)TILE);
                const int row = ((page * 2 + which) * a.G + g) * PAGE;
#pragma unroll
                for (int f = 0; f < SH::BLOCKS; ++f) tma_load_2d(ring + s * TILE + f * (PAGE * 128), &map_kv, f * 64, row, &full[s]);
            }
            ++at[c];
        };
        const int counts[2] = {turns(0), streams == 2 ? turns(1) : 0};
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int c = 0; c < 2; ++c)
                if (ok && k < counts[c]) request(k, c, 0);
#pragma unroll 4
        for (int b = lane; b < a.B; b += 32) reached = max(reached, a.kv_len[b]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) reached = max(reached, __shfl_xor_sync(0xffffffffu, reached, o));
        for (int k = 0; k < counts[0] && ok; ++k)                  // the first stream has as many pages as the second, or one more
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (ok && k < counts[c]) request(k, c, 1);
                if (ok && k + 2 < counts[c]) request(k + 2, c, 0);
            }
        if (!ok)                                                   // the copies in flight land before the CTA ends
#pragma unroll
            for (int c = 0; c < 2; ++c)
                for (int i = max(0, at[c] - slots); i < at[c]; ++i) mbar_wait(&full[slot_of(i, c)], round_of(i));
        __syncwarp();
    } else if (warp < 3) {
        // ------------------------------------------------------------ products, a warp per chain
        // (Waiting and committing cost a warp more than issuing: one warp for both chains took 2,350 cycles per page.)
        constexpr uint32_t base_idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(ROWS >> 4) << 24);
        constexpr uint32_t idesc_s = base_idesc | ((uint32_t)(PAGE >> 3) << 17);
        constexpr uint32_t idesc_pv = base_idesc | (1u << 16) | ((uint32_t)(HD >> 3) << 17);                  // V: contiguous in N
        const int c = warp - 1, count = turns(c);
        const bool leader = elect_one();
        const uint64_t desc_q = smem_desc(smem_u32(q_tiles + (alone ? 0 : c) * SH::Q_TILE)), desc_k = smem_desc(smem_u32(ring));
        const uint64_t desc_v = smem_desc_mn(smem_u32(ring), PAGE * 128);
        const uint32_t s_col = tmem_base + SH::S_COL + c * 128, o_col = tmem_base + SH::O_COL + c * HD;
        bool ok = count > 0;
        auto await = [&](uint64_t* bar, uint32_t parity, int code) {
            if (!mbar_test(bar, parity) && !mbar_wait(bar, parity)) { ok = false; atomicExch(a.status, code); }
        };
        auto scores = [&](int k) {
            const int at = keys_at(k), s = slot_of(at, c);
            await(&full[s], round_of(at), 83);
            tcgen05_fence_after();
            const uint64_t dk = desc_k + (uint64_t)(s * (TILE >> 4));
            if (ok && leader) {
#pragma unroll
                for (int j = 0; j < HD / 16; ++j)              // 16 features per instruction; 4 instructions per block of 64
                    tcgen05_mma(s_col + (k & 1) * PAGE, desc_q + (uint64_t)((j >> 2) * (ROWS * 128 >> 4) + (j & 3) * 2),
                                dk + (uint64_t)((j >> 2) * (PAGE * 128 >> 4) + (j & 3) * 2), idesc_s, j > 0 ? 1u : 0u);
                tcgen05_commit(&s_ready[c * 2 + (k & 1)]);
                tcgen05_commit(&empty[s]);
            }
            __syncwarp();
        };
        auto values = [&](int k) {
            const int at = values_at(k, count), s = slot_of(at, c);
            await(&full[s], round_of(at), 83);
            const uint64_t dv = desc_v + (uint64_t)(s * (TILE >> 4));
            await(&p_ready[c * 2 + (k & 1)], (k >> 1) & 1, 84);
            tcgen05_fence_after();
            if (ok && leader) {
#pragma unroll
                for (int j = 0; j < PAGE / 16; ++j)
                    mma_ts(o_col, s_col + (k & 1) * PAGE + j * 8, dv + (uint64_t)(j * (2048 >> 4)), idesc_pv, (j > 0 || k > 0) ? 1u : 0u);
                tcgen05_commit(&o_ready[c]);
                tcgen05_commit(&empty[s]);
            }
            __syncwarp();
        };
        // A chain's scores go over the weights of two pages before, which the products issued before them have read.
        if (ok) await(q_full, 0, 82);
        for (int k = 0; k < 2; ++k)
            if (__all_sync(0xffffffffu, ok) && k < count) scores(k);
        for (int k = 0; k < count && __all_sync(0xffffffffu, ok); ++k) {
            values(k);
            if (k + 2 < count) scores(k + 2);
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ------------------------------------------------------------ softmax: a thread per row
        const int c = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        // the positions of the CTA's tokens: a token that itself lies among the shared pages sees them up to its own
        for (int i = threadIdx.x - 128; i < 2 * per_tile; i += 256) position[i] = -1;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        for (int b = threadIdx.x - 128; b < a.B; b += 256) {
            const int from = a.q_start[b], to = a.q_start[b + 1], len = a.kv_len[b];
            for (int t = max(from, t0); t < min(to, t0 + 2 * per_tile); ++t) position[t - t0] = len - (to - t);
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const int token = t0 + (alone ? 0 : c) * per_tile + r / a.R, head = g * a.R + r % a.R;
        const bool real = r < per_tile * a.R && token < a.T && c < chains;
        const int seen = real ? min(position[token - t0] + 1, a.pages * PAGE) : 0;      // shared keys that the row sees
        const float scale = a.scale_log2;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16), o_addr = lane_addr + SH::O_COL + c * HD;
        const int count = turns(c);
        float m = NEG_BIG, l = 0.f;
        bool ok = true;
        // The two chains' warps of a scheduler take turns at the exponentials (named barriers of 64): while one has the exp2 unit the other loads,
        // looks for its maximum and stores. Left to themselves both come to their exponentials together and then leave the unit idle together.
        const bool take_turns = !alone && chains == 2;
        const int mine = 2 + quarter * 2 + c, theirs = 2 + quarter * 2 + (c ^ 1);
        auto await_turn = [&]() { if (take_turns) asm volatile("bar.sync %0, 64;" ::"r"(mine) : "memory"); };
        auto hand_on = [&](int k) { if (take_turns && (c == 0 || k + 1 < count)) asm volatile("bar.arrive %0, 64;" ::"r"(theirs) : "memory"); };
        auto give_up = [&](int k) {                                // at page k: the other chain goes on, without an end to its waits otherwise
            for (; take_turns && k < count; ++k) {
                await_turn();
                hand_on(k);
            }
        };
        if (c == 1) hand_on(-1);
        for (int k = 0; k < count; ++k) {
            const uint32_t s_addr = lane_addr + SH::S_COL + c * 128 + (k & 1) * PAGE;
            ok = __all_sync(0xffffffffu, mbar_wait(&s_ready[c * 2 + (k & 1)], (k >> 1) & 1));
            if (!ok) { if (lane == 0) atomicExch(a.status, 85); give_up(k); break; }
            tcgen05_fence_after();
            uint32_t s[PAGE];
            tmem_ld32(s_addr, s);
            tmem_ld32(s_addr + 32, s + 32);
            tmem_ld_wait();
            const int key0 = (first + page_of(k, c)) * PAGE;
            if (__any_sync(0xffffffffu, seen < key0 + PAGE)) {
#pragma unroll
                for (int j = 0; j < PAGE; ++j)
                    if (key0 + j >= seen) s[j] = 0xff800000u;
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < PAGE; j += 8)
#pragma unroll
                for (int u = 0; u < 4; ++u) mx4[u] = max3(mx4[u], __uint_as_float(s[j + 2 * u]), __uint_as_float(s[j + 2 * u + 1]));
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale;
            // The reference follows only when the row's maximum has outgrown it by more than RESCALE_ABOVE; then the output so far comes
            // down to it, which must have been added up before and waits for nothing else (the next product follows p_ready).
            const bool moves = mx > m + RESCALE_ABOVE;
            if (__any_sync(0xffffffffu, moves)) {
                if (k > 0) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&o_ready[c], (k - 1) & 1));
                    if (!ok) { if (lane == 0) atomicExch(a.status, 86); give_up(k); break; }
                    tcgen05_fence_after();
                    const float factor = moves ? fast_exp2(m - mx) : 1.0f;
#pragma unroll
                    for (int d = 0; d < HD; d += 32) {
                        uint32_t o[32];
                        tmem_ld32(o_addr + d, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * factor);
                        tmem_st32(o_addr + d, o);
                    }
                }
                if (moves) {
                    l *= fast_exp2(m - mx);
                    m = mx;
                }
            }
            await_turn();
            float sum4[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t p[PAGE / 2];
#pragma unroll
            for (int j = 0; j < PAGE / 2; ++j) {
                float e0 = __uint_as_float(s[2 * j]), e1 = __uint_as_float(s[2 * j + 1]);
                fma2(e0, e1, scale, -m);
                e0 = fast_exp2(e0);
                e1 = fast_exp2(e1);
                add2(sum4[(j & 1) * 2], sum4[(j & 1) * 2 + 1], e0, e1);
                p[j] = pack_bf16(e0, e1);
            }
            tmem_st32(s_addr, p);
            hand_on(k);
            tmem_st_wait();
            l += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
            // A parity tells only a phase from the one before it. The scores of page k say that the products up to page k - 2 have been
            // added; before the last page's product is let go the one before it is awaited, so that the last can be awaited by itself.
            if (k > 0 && k == count - 1) {
                ok = __all_sync(0xffffffffu, mbar_wait(&o_ready[c], (k - 1) & 1));
                if (!ok) { if (lane == 0) atomicExch(a.status, 86); break; }
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[c * 2 + (k & 1)]);
        }
        if (count > 0 && ok && !__all_sync(0xffffffffu, mbar_wait(&o_ready[c], (count - 1) & 1))) { if (lane == 0) atomicExch(a.status, 86); ok = false; }
        tcgen05_fence_after();
        const int slot = alone ? split * 2 + c : split;
        const long long row = ((long long)slot * a.T + token) * a.H + head;
        if (real) *reinterpret_cast<float2*>(a.part_ml + row * 2) = make_float2(count > 0 ? m : NEG_BIG, count > 0 && ok ? l : 0.f);
        // The results leave through shared memory, a row per copy: stored from the registers they took 10,000 cycles. Both
        // chains have had their last product when all are here.
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (count > 0 && ok) {
            uint8_t* mine = q_tiles + (c * ROWS + r) * SH::OUT_ROW;
#pragma unroll
            for (int d = 0; d < HD; d += 32) {
                uint32_t o[32];
                tmem_ld32(o_addr + d, o);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; j += 4) *reinterpret_cast<uint4*>(mine + (d + j) * 4) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            if (real) {
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(a.part_o + row * HD), "r"(smem_u32(mine)), "n"(HD * 4) : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
            }
        }
        tcgen05_fence_before();
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)SH::TMEM_COLS));
    }
}

// ============================================================================ the own pages, and the join
struct OwnArgs {
    const __nv_bfloat16* q;
    __nv_bfloat16* out;
    const int* table;
    int width;
    const int* q_start;
    const int* kv_len;
    float* part_o;
    float* part_ml;
    int B, T, H, G, R, pages, slots;           // slots: partial results per row from the shared pages
    int waits_first;                           // nothing runs before it that would have waited
    float scale_log2;
    int* status;
};

// A page of 64 keys and its 64 values into a stage (K, then V; panels of 64 features with the 128-byte swizzle).
template <int HD>
__device__ __forceinline__ void request_page(uint8_t* stage, uint64_t* bar, const CUtensorMap* map, int page, int G, int g) {
    mbar_expect_tx(bar, 2 * PAGE * HD * 2);
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int f = 0; f < HD / 64; ++f)
            tma_load_2d(stage + which * (PAGE * HD * 2) + f * (PAGE * 128), map, f * 64, ((page * 2 + which) * G + g) * PAGE, bar);
}
// Values behind the sequence's last position may hold anything, and zero times no number is no number: rows [from, to) become zero.
template <int HD>
__device__ __forceinline__ void clear_values(uint8_t* v_tile, int from, int to, int i, int step) {
    for (; i < (to - from) * (HD / 8); i += step) {
        const int row = from + i / (HD / 8), chunk = i % (HD / 8);
        *reinterpret_cast<uint4*>(v_tile + (chunk >> 3) * (PAGE * 128) + row * 128 + (chunk & 7) * 16) = make_uint4(0, 0, 0, 0);
    }
}

// A single new token per sequence: the keys are the rows of the products and the (up to 8) query heads of a key/value head their
// columns (see attention_decode.cuh); four warps share a page, 16 keys each. grid: (G x head groups, B); 128 threads. Keys and values of a
// page come one by one through a ring of three tiles (two pages at heads of 64), so that four CTAs share an SM at heads of 128.
// Bound by the latency of a page's way (number, tiles, products) and of the join at one or two rounds of pages per CTA: 15 us for the 64
// sequences above, whose own pages are 37 MB (5.6 us), with 17 MB of results that mostly come from L2.
template <int HD> struct OwnShape {
    static constexpr int TILE = PAGE * HD * 2;
    static constexpr int TILES = HD == 64 ? 4 : 3;
    static constexpr int SMEM = TILES * TILE + 1024;
    static_assert(TILES * TILE >= 4 * HEAD_ROWS * (HD + 2) * 4, "the warps' results lie where the pages were");
};
constexpr int MOST_SLOTS = 64;
template <int HD>
__global__ void __launch_bounds__(128)
attention_own_single_kernel(const __grid_constant__ CUtensorMap map_kv, const OwnArgs a) {
    using SH = OwnShape<HD>;
    constexpr int KSTEPS = HD / 16, TILES = SH::TILES, TILE = SH::TILE;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t full[TILES];
    __shared__ float factor[HEAD_ROWS][MOST_SLOTS + 4];
    __shared__ float total[HEAD_ROWS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int b = blockIdx.y, groups = gridDim.x / a.G, g = blockIdx.x / groups, hg = blockIdx.x - g * groups;
    const int head0 = g * a.R + hg * HEAD_ROWS, nrows = min(HEAD_ROWS, a.R - hg * HEAD_ROWS);
    if (a.waits_first) lp_grid_wait();
    const int* table = a.table + (long long)b * a.width + a.pages;
    // asked for together; the first own pages' numbers as well (a sequence without any has none there to use)
    const int t = a.q_start[b], t_end = a.q_start[b + 1], len = a.kv_len[b];
    const int held = lane < a.width - a.pages ? table[lane] : 0;
    const bool real = t_end > t && t >= 0 && t < a.T;              // one new token, or none
    const int pos = real ? len - 1 : -1;
    const int last = pos >= 0 ? pos / PAGE : -1, npages = max(0, min(last + 1, a.width) - a.pages);
    auto request = [&](int n) {                                    // by the whole first warp: tile n = keys or values of page n / 2
        const int p = n >> 1, page = p < 32 ? __shfl_sync(0xffffffffu, held, p) : table[p];
        if (lane == 0) {
            uint64_t* bar = &full[n % TILES];
            mbar_expect_tx(bar, TILE);
#pragma unroll
            for (int f = 0; f < HD / 64; ++f)
                tma_load_2d(smem + (n % TILES) * TILE + f * (PAGE * 128), &map_kv, f * 64, ((page * 2 + (n & 1)) * a.G + g) * PAGE, bar);
        }
    };
    if (warp == 0) {
        if (lane == 0) {
            for (int s = 0; s < TILES; ++s) mbar_init(&full[s], 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        for (int n = 0; n < TILES && n < 2 * npages; ++n) request(n);
    }
    __syncthreads();
    const int g8 = lane >> 2, t4 = lane & 3;
    uint32_t qf[KSTEPS][2];
    if (real) {
        const __nv_bfloat16* q_row = a.q + ((long long)t * a.H + head0 + min(g8, nrows - 1)) * HD;
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
            qf[kk][0] = *reinterpret_cast<const uint32_t*>(q_row + kk * 16 + t4 * 2);
            qf[kk][1] = *reinterpret_cast<const uint32_t*>(q_row + kk * 16 + t4 * 2 + 8);
        }
    }
    float o[KSTEPS][4];
#pragma unroll
    for (int i = 0; i < KSTEPS; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = NEG_BIG, m1 = NEG_BIG, l0 = 0.f, l1 = 0.f;          // of heads 2 t4 and 2 t4 + 1
    const int frag_row = (lane & 7) + ((lane >> 3) & 1) * 8, frag_chunk = lane >> 4, key0 = warp * 16;
    auto arrived = [&](int n) {
        const bool yes = mbar_wait(&full[n % TILES], (n / TILES) & 1);
        if (!yes && lane == 0) atomicExch(a.status, 87);
        return yes;
    };
    auto refill = [&](int n) {                                     // tile n has been read by all: tile n + TILES goes there
        __syncthreads();
        if (warp == 0 && n + TILES < 2 * npages) {
            // what was written here by stores comes before what the copy writes
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            request(n + TILES);
        }
    };
    for (int p = 0; p < npages; ++p) {
        const int key_base = (a.pages + p) * PAGE;
        const bool active = key_base + key0 <= pos;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        bool there = arrived(2 * p);
        if (there && active) {
            const uint32_t k_tile = smem_u32(smem + (2 * p % TILES) * TILE);
#pragma unroll
            for (int kk = 0; kk < KSTEPS; ++kk) {
                uint32_t x[4];
                ldmatrix_x4(k_tile + tile_offset<true>(key0 + frag_row, kk * 2 + frag_chunk, HD, HD / 8), x[0], x[1], x[2], x[3]);
                mma_bf16(s, x, qf[kk][0], qf[kk][1]);
            }
        }
        refill(2 * p);
        there = arrived(2 * p + 1) && there;
        if (there && active) {
            uint8_t* values = smem + ((2 * p + 1) % TILES) * TILE;
            const uint32_t v_tile = smem_u32(values);
            if (key_base + key0 + 15 > pos) {                      // the warp's own rows of the page
                clear_values<HD>(values, pos + 1 - key_base, key0 + 16, lane, 32);
                __syncwarp();
            }
            const bool out_a = key_base + key0 + g8 > pos, out_b = key_base + key0 + g8 + 8 > pos;
            s[0] = out_a ? NEG_BIG : s[0] * a.scale_log2;
            s[1] = out_a ? NEG_BIG : s[1] * a.scale_log2;
            s[2] = out_b ? NEG_BIG : s[2] * a.scale_log2;
            s[3] = out_b ? NEG_BIG : s[3] * a.scale_log2;
            float mx0 = fmaxf(s[0], s[2]), mx1 = fmaxf(s[1], s[3]);
#pragma unroll
            for (int sh = 4; sh < 32; sh <<= 1) {
                mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, sh));
                mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, sh));
            }
            const float mn0 = fmaxf(m0, mx0), mn1 = fmaxf(m1, mx1);
            const float f0 = fast_exp2(m0 - mn0), f1 = fast_exp2(m1 - mn1);
            m0 = mn0; m1 = mn1;
            const float e0 = out_a ? 0.f : fast_exp2(s[0] - mn0), e1 = out_a ? 0.f : fast_exp2(s[1] - mn1);
            const float e2 = out_b ? 0.f : fast_exp2(s[2] - mn0), e3 = out_b ? 0.f : fast_exp2(s[3] - mn1);
            l0 = l0 * f0 + (e0 + e2);
            l1 = l1 * f1 + (e1 + e3);
            const uint32_t p0 = transpose_8x8(pack_bf16(e0, e1)), p1 = transpose_8x8(pack_bf16(e2, e3));
            const int v_row = key0 + (lane & 7) + (lane >> 4) * 8, v_chunk = (lane >> 3) & 1;
#pragma unroll
            for (int mt = 0; mt < KSTEPS; ++mt) {
                o[mt][0] *= f0; o[mt][1] *= f1; o[mt][2] *= f0; o[mt][3] *= f1;
                uint32_t x[4];
                ldmatrix_x4_trans(v_tile + tile_offset<true>(v_row, mt * 2 + v_chunk, HD, HD / 8), x[0], x[1], x[2], x[3]);
                mma_bf16(o[mt], x, p0, p1);
            }
        }
        refill(2 * p + 1);
    }
#pragma unroll
    for (int sh = 4; sh < 32; sh <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, sh);
        l1 += __shfl_xor_sync(0xffffffffu, l1, sh);
    }
    // the warps' results, where the pages were: all have arrived and been read
    float* sm_m = reinterpret_cast<float*>(smem);                  // [4][8]
    float* sm_l = sm_m + 4 * HEAD_ROWS;                            // [4][8]
    float* sm_o = sm_l + 4 * HEAD_ROWS;                            // [4][8][HD]
    if (g8 == 0) {
        sm_m[warp * HEAD_ROWS + 2 * t4] = m0; sm_m[warp * HEAD_ROWS + 2 * t4 + 1] = m1;
        sm_l[warp * HEAD_ROWS + 2 * t4] = l0; sm_l[warp * HEAD_ROWS + 2 * t4 + 1] = l1;
    }
#pragma unroll
    for (int mt = 0; mt < KSTEPS; ++mt) {
        float* head_a = sm_o + (warp * HEAD_ROWS + 2 * t4) * HD + mt * 16 + g8;
        head_a[0] = o[mt][0]; head_a[HD] = o[mt][1];
        head_a[8] = o[mt][2]; head_a[HD + 8] = o[mt][3];
    }
    if (!a.waits_first) lp_grid_wait();                            // the shared pages' results
    lp_grid_release();
    __syncthreads();
    if (!real) return;
    // per head the factor of each partial result: the four warps' and the shared pages'
    for (int r = warp; r < nrows; r += 4) {
        const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + (long long)t * a.H + head0 + r;
        const long long step = (long long)a.T * a.H;
        constexpr int PER = (MOST_SLOTS + 4 + 31) / 32;
        float mi[PER], li[PER], m = NEG_BIG, l = 0.f;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int i = k * 32 + lane;
            float2 x = make_float2(NEG_BIG, 0.f);
            if (i < 4) x = make_float2(sm_m[i * HEAD_ROWS + r], sm_l[i * HEAD_ROWS + r]);
            else if (i < 4 + a.slots) x = __ldcg(ml + (i - 4) * step);
            mi[k] = x.x;
            li[k] = x.y;
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) m = fmaxf(m, li[k] != 0.f ? mi[k] : NEG_BIG);      // nothing lies where the sum is zero
        m = lp_warp_max(m);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const float f = li[k] != 0.f ? fast_exp2(mi[k] - m) : 0.f;
            l += li[k] * f;
            if (k * 32 + lane < 4 + a.slots) factor[r][k * 32 + lane] = f;
        }
        l = lp_warp_sum(l);
        if (lane == 0) total[r] = l;
    }
    __syncthreads();
    for (int idx = tid; idx < nrows * (HD / 4); idx += 128) {      // four features per thread; sixteen results are asked for at a time
        const int r = idx / (HD / 4), d = (idx - r * (HD / 4)) * 4;
        const float* po = a.part_o + ((long long)t * a.H + head0 + r) * HD + d;
        const long long step = (long long)a.T * a.H * HD;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](const float4& x, float f) {
            acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
        };
#pragma unroll
        for (int w = 0; w < 4; ++w) add(*reinterpret_cast<const float4*>(&sm_o[(w * HEAD_ROWS + r) * HD + d]), factor[r][w]);
        for (int s0 = 0; s0 < a.slots; s0 += 16) {
            float4 x[16];
#pragma unroll
            for (int u = 0; u < 16; ++u)
                x[u] = s0 + u < a.slots && factor[r][4 + s0 + u] != 0.f ? __ldcg(reinterpret_cast<const float4*>(po + (s0 + u) * step)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int u = 0; u < 16; ++u)
                if (s0 + u < a.slots) add(x[u], factor[r][4 + s0 + u]);
        }
        const float l = total[r], inv = l != 0.f ? 1.0f / l : 0.f;
        uint2 packed = l != 0.f ? make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv)) : make_uint2(0, 0);
        *reinterpret_cast<uint2*>(a.out + ((long long)t * a.H + head0 + r) * HD + d) = packed;
    }
}

// Several new tokens: 64 rows of (token, query head) pairs of one sequence, 16 per warp, over its own pages, causal. These are few next
// to the shared ones, so mma.sync does. Bound by latency: lengths, page numbers, tiles, then the shared pages' results (each of a row's two
// rounds of values asked for at once: 4 sequences of 20 tokens behind 30 shared pages 16.4 us in all, 20.7 row by row). Three CTAs per SM:
// two with registers to spare took 41.8 instead of 35.9 us for 100 sequences of 2 tokens. At 40 sequences of up to 190 tokens above it
// takes 96 us, 5 % of the call, and most of what it moves are the shared pages' results (77 MB); to take those first, while the pages
// are on their way, gained nothing there and cost 5 us where the first kernel leaves SMs free.
// grid: (row tiles, G, B); 128 threads.
template <int HD> struct OwnRows {
    static constexpr int STAGE = 2 * PAGE * HD * 2, STAGES = 2, SMEM = STAGES * STAGE + 1024;
};
// APART: the results go behind the shared pages', for the kernel below.
template <int HD, bool APART>
__global__ void __launch_bounds__(128, 3)
attention_own_rows_kernel(const __grid_constant__ CUtensorMap map_kv, const OwnArgs a) {
    using SH = OwnRows<HD>;
    constexpr int KSTEPS = HD / 16, STAGES = SH::STAGES;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t full[STAGES];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
    const int b = blockIdx.z, g = blockIdx.y;
    if (a.waits_first) lp_grid_wait();
    const int t0 = a.q_start[b], n = a.q_start[b + 1] - t0;
    const int row0 = (gridDim.x - 1 - blockIdx.x) * 64;            // the rows with the most keys first
    const int rows = t0 >= 0 ? min(64, min(n, a.T - t0) * a.R - row0) : 0;
    if (rows <= 0) {
        if (!a.waits_first) lp_grid_wait();
        return;
    }
    const int len = a.kv_len[b], pos0 = len - n;
    const int last_pos = pos0 + (row0 + rows - 1) / a.R;
    const int npages = last_pos >= 0 ? max(0, min(last_pos / PAGE + 1, a.width) - a.pages) : 0;
    const int* table = a.table + (long long)b * a.width + a.pages;
    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(&full[s], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int p = 0; p < STAGES && p < npages; ++p) request_page<HD>(smem + p * SH::STAGE, &full[p], &map_kv, table[p], a.G, g);
    }
    __syncthreads();
    // the lane's two rows
    int token[2], head[2], pos[2];
    bool real[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int r = warp * 16 + g8 + 8 * k, at = row0 + min(r, rows - 1);
        token[k] = t0 + at / a.R;
        head[k] = g * a.R + at % a.R;
        pos[k] = pos0 + at / a.R;
        real[k] = r < rows;
    }
    const int warp_first = pos0 + (row0 + min(warp * 16, rows - 1)) / a.R, warp_last = pos0 + (row0 + min(warp * 16 + 15, rows - 1)) / a.R;
    uint32_t qf[KSTEPS][4];
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const __nv_bfloat16* row = a.q + ((long long)token[k] * a.H + head[k]) * HD + kk * 16 + t4 * 2;
            qf[kk][k] = *reinterpret_cast<const uint32_t*>(row);
            qf[kk][2 + k] = *reinterpret_cast<const uint32_t*>(row + 8);
        }
    float o[KSTEPS * 2][4];
#pragma unroll
    for (int i = 0; i < KSTEPS * 2; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {NEG_BIG, NEG_BIG}, l[2] = {0.f, 0.f};             // the sum: a part in each of a row's four lanes
    for (int p = 0; p < npages; ++p) {
        uint8_t* stage = smem + (p % STAGES) * SH::STAGE;
        const bool arrived = mbar_wait(&full[p % STAGES], (p / STAGES) & 1);
        if (!arrived && lane == 0) atomicExch(a.status, 88);
        const int key_base = (a.pages + p) * PAGE;
        if (key_base + PAGE > len) {
            clear_values<HD>(stage + PAGE * HD * 2, max(0, len - key_base), PAGE, tid, 128);
            __syncthreads();
        }
        if (arrived && key_base <= warp_last) {
            const uint32_t k_tile = smem_u32(stage), v_tile = k_tile + PAGE * HD * 2;
            const int mat = lane >> 3, in_mat = lane & 7;
            float s[8][4];
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                s[2 * ks][0] = s[2 * ks][1] = s[2 * ks][2] = s[2 * ks][3] = 0.f;
                s[2 * ks + 1][0] = s[2 * ks + 1][1] = s[2 * ks + 1][2] = s[2 * ks + 1][3] = 0.f;
                const int key = ks * 16 + (mat >> 1) * 8 + in_mat;
#pragma unroll
                for (int kk = 0; kk < KSTEPS; ++kk) {
                    uint32_t x[4];
                    ldmatrix_x4(k_tile + tile_offset<true>(key, kk * 2 + (mat & 1), HD, HD / 8), x[0], x[1], x[2], x[3]);
                    mma_bf16(s[2 * ks], qf[kk], x[0], x[1]);
                    mma_bf16(s[2 * ks + 1], qf[kk], x[2], x[3]);
                }
            }
            const bool edge = key_base + PAGE - 1 > warp_first;
            float mx[2] = {NEG_BIG, NEG_BIG};
#pragma unroll
            for (int nt = 0; nt < 8; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = s[nt][e] * a.scale_log2;
                    if (edge && key_base + nt * 8 + t4 * 2 + (e & 1) > pos[e >> 1]) v = -INFINITY;
                    s[nt][e] = v;
                    mx[e >> 1] = fmaxf(mx[e >> 1], v);
                }
            float f[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], 1));
                mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], 2));
                const float mn = fmaxf(m[k], mx[k]);
                f[k] = fast_exp2(m[k] - mn);
                m[k] = mn;
                l[k] *= f[k];
            }
            uint32_t pf[4][4];
#pragma unroll
            for (int nt = 0; nt < 8; ++nt) {
                const float e0 = fast_exp2(s[nt][0] - m[0]), e1 = fast_exp2(s[nt][1] - m[0]);
                const float e2 = fast_exp2(s[nt][2] - m[1]), e3 = fast_exp2(s[nt][3] - m[1]);
                l[0] += e0 + e1;
                l[1] += e2 + e3;
                pf[nt >> 1][(nt & 1) * 2] = pack_bf16(e0, e1);
                pf[nt >> 1][(nt & 1) * 2 + 1] = pack_bf16(e2, e3);
            }
#pragma unroll
            for (int i = 0; i < KSTEPS * 2; ++i) { o[i][0] *= f[0]; o[i][1] *= f[0]; o[i][2] *= f[1]; o[i][3] *= f[1]; }
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                const int key = ks * 16 + (mat & 1) * 8 + in_mat;
#pragma unroll
                for (int dd = 0; dd < KSTEPS; ++dd) {
                    uint32_t x[4];
                    ldmatrix_x4_trans(v_tile + tile_offset<true>(key, dd * 2 + (mat >> 1), HD, HD / 8), x[0], x[1], x[2], x[3]);
                    mma_bf16(o[dd * 2], pf[ks], x[0], x[1]);
                    mma_bf16(o[dd * 2 + 1], pf[ks], x[2], x[3]);
                }
            }
        }
        __syncthreads();
        if (tid == 0 && p + STAGES < npages) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            request_page<HD>(stage, &full[p % STAGES], &map_kv, table[p + STAGES], a.G, g);
        }
    }
    if (APART) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            l[k] += __shfl_xor_sync(0xffffffffu, l[k], 1);
            l[k] += __shfl_xor_sync(0xffffffffu, l[k], 2);
            if (!real[k]) continue;
            const long long row = ((long long)a.slots * a.T + token[k]) * a.H + head[k];
            if (t4 == 0) *reinterpret_cast<float2*>(a.part_ml + row * 2) = make_float2(m[k], l[k]);
#pragma unroll
            for (int i = 0; i < KSTEPS * 2; ++i)
                *reinterpret_cast<float2*>(a.part_o + row * HD + i * 8 + t4 * 2) = make_float2(o[i][2 * k], o[i][2 * k + 1]);
        }
        lp_grid_wait();
        lp_grid_release();
        return;
    }
    // what the shared pages gave
    if (!a.waits_first) lp_grid_wait();
    lp_grid_release();
    const float* po[2];
    const float* ml[2];
    const long long row_step = (long long)a.T * a.H;
    float f[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const long long row = (long long)token[k] * a.H + head[k];
        po[k] = a.part_o + row * HD + t4 * 2;
        ml[k] = a.part_ml + row * 2;
        float most = m[k];
#pragma unroll 2
        for (int s = t4; s < a.slots; s += 4) {                    // the row's four lanes share them
            const float2 x = __ldcg(reinterpret_cast<const float2*>(ml[k] + s * row_step * 2));
            if (x.y != 0.f) most = fmaxf(most, x.x);
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        f[k] = fast_exp2(m[k] - most);
        m[k] = most;
        l[k] *= f[k];
    }
#pragma unroll
    for (int i = 0; i < KSTEPS * 2; ++i) { o[i][0] *= f[0]; o[i][1] *= f[0]; o[i][2] *= f[1]; o[i][3] *= f[1]; }
    for (int s = 0; s < a.slots; ++s) {                            // both rows' values asked for together
        float2 x[2], v[2][KSTEPS * 2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            x[k] = __ldcg(reinterpret_cast<const float2*>(ml[k] + s * row_step * 2));
#pragma unroll
            for (int i = 0; i < KSTEPS * 2; ++i) v[k][i] = __ldcg(reinterpret_cast<const float2*>(po[k] + s * row_step * HD + i * 8));
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (x[k].y == 0.f) continue;                           // nothing there
            const float weight = fast_exp2(x[k].x - m[k]);
            if (t4 == 0) l[k] += x[k].y * weight;
#pragma unroll
            for (int i = 0; i < KSTEPS * 2; ++i) {
                o[i][2 * k] += v[k][i].x * weight;
                o[i][2 * k + 1] += v[k][i].y * weight;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        l[k] += __shfl_xor_sync(0xffffffffu, l[k], 1);
        l[k] += __shfl_xor_sync(0xffffffffu, l[k], 2);
        const float inv = l[k] != 0.f ? 1.0f / l[k] : 0.f;
        if (real[k]) {
            __nv_bfloat16* dst = a.out + ((long long)token[k] * a.H + head[k]) * HD + t4 * 2;
#pragma unroll
            for (int i = 0; i < KSTEPS * 2; ++i)
                *reinterpret_cast<uint32_t*>(dst + i * 8) = l[k] != 0.f ? pack_bf16(o[i][2 * k] * inv, o[i][2 * k + 1] * inv) : 0u;
        }
    }
}

// Many results per row and few rows: all of a row's results, the own pages' last, joined by a thread per four features. In the kernel above,
// whose CTAs are as few as the rows, a result costs a round trip each.
// grid: rows of (token, query head) in portions of 128 / (HD / 4); 128 threads.
template <int HD>
__global__ void __launch_bounds__(128)
attention_join_kernel(const OwnArgs a) {
    constexpr int LANES = HD / 4, PER = (MOST_SLOTS + 1 + LANES - 1) / LANES;
    const int lane = threadIdx.x % LANES;
    const long long row = (long long)blockIdx.x * (128 / LANES) + threadIdx.x / LANES, step = (long long)a.T * a.H;
    lp_grid_wait();
    lp_grid_release();
    const bool real = row < (long long)min(a.T, a.q_start[a.B]) * a.H;       // rows behind the last sequence stay as they are
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + (real ? row : 0);
    float2 x[PER];
    float m = NEG_BIG, l = 0.f;
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] = k * LANES + lane <= a.slots ? __ldcg(ml + (k * LANES + lane) * step) : make_float2(NEG_BIG, 0.f);
#pragma unroll
    for (int k = 0; k < PER; ++k) m = fmaxf(m, x[k].y != 0.f ? x[k].x : NEG_BIG);        // nothing lies where the sum is zero
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float factor[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        factor[k] = x[k].y != 0.f ? fast_exp2(x[k].x - m) : 0.f;
        l += x[k].y * factor[k];
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const float4* po = reinterpret_cast<const float4*>(a.part_o) + (real ? row : 0) * LANES + lane;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < PER; ++k)
        for (int j = 0; j < LANES && k * LANES + j <= a.slots; j += 8) {
            float4 v[8];
            float f[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                f[u] = __shfl_sync(0xffffffffu, factor[k], j + u, LANES);
                v[u] = f[u] != 0.f ? __ldcg(po + (long long)(k * LANES + j + u) * step * LANES) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) { sum.x += v[u].x * f[u]; sum.y += v[u].y * f[u]; sum.z += v[u].z * f[u]; sum.w += v[u].w * f[u]; }
        }
    const float inv = l != 0.f ? 1.0f / l : 0.f;
    if (real)
        *reinterpret_cast<uint2*>(a.out + row * HD + lane * 4) =
            l != 0.f ? make_uint2(pack_bf16(sum.x * inv, sum.y * inv), pack_bf16(sum.z * inv, sum.w * inv)) : make_uint2(0, 0);
}

// ============================================================================ launches
int make_query_map(CUtensorMap* map, const void* q, int T, int H, int hd, int R, int tokens) {
    EncodeTiled enc = encode_fn();
    if (!enc) LP_REFUSE("attention_shared: the driver does not offer cuTensorMapEncodeTiled");
    cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)H, (cuuint64_t)T};
    cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)H * hd * 2};
    cuuint32_t box[3] = {64u, (cuuint32_t)R, (cuuint32_t)tokens};
    cuuint32_t elem[3] = {1, 1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) LP_REFUSE("attention_shared: cuTensorMapEncodeTiled failed with code %d for %d tokens of %d heads of %d", (int)r, T, H, hd);
    return 0;
}

template <typename K> int reserve(K kernel, int bytes) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) LP_REFUSE("attention_shared: cannot reserve %d bytes of shared memory: %s", bytes, cudaGetErrorString(e));
    return 0;
}

template <int HD>
int run(const void* q, const void* pages, long long num_pages, int max_new, bool apart, SharedArgs s, OwnArgs o, cudaStream_t stream) {
    static bool configured = false;
    if (!configured) {
        int rc = reserve(attention_shared_kernel<HD>, Shape<HD>::SMEM);
        if (!rc) rc = reserve(attention_own_single_kernel<HD>, OwnShape<HD>::SMEM);
        if (!rc) rc = reserve(attention_own_rows_kernel<HD, false>, OwnRows<HD>::SMEM);
        if (!rc) rc = reserve(attention_own_rows_kernel<HD, true>, OwnRows<HD>::SMEM);
        if (rc) return rc;
        configured = true;
    }
    CUtensorMap mq, mkv;
    int rc = make_map(&mkv, pages, num_pages * 2 * s.G * PAGE, HD, HD, PAGE);
    if (rc) return rc;
    if (o.slots > 0) {
        const int per_tile = ROWS / s.R, tiles = (s.T + per_tile - 1) / per_tile;
        rc = make_query_map(&mq, q, s.T, s.H, HD, s.R, per_tile);
        if (rc) return rc;
        cudaError_t err = lp_launch(attention_shared_kernel<HD>, dim3((unsigned)(s.splits * ((tiles + 1) / 2)), s.G), dim3(THREADS), Shape<HD>::SMEM, stream, mq, mkv, s);
        if (err != cudaSuccess) return lp_check_launch("attention_shared");
    }
    if (max_new == 1) {
        const int groups = (s.R + HEAD_ROWS - 1) / HEAD_ROWS;
        lp_launch(attention_own_single_kernel<HD>, dim3(s.G * groups, s.B), dim3(128), OwnShape<HD>::SMEM, stream, mkv, o);
    } else {
        const dim3 grid((unsigned)(((long long)max_new * s.R + 63) / 64), s.G, s.B);
        if (!apart) {
            lp_launch(attention_own_rows_kernel<HD, false>, grid, dim3(128), OwnRows<HD>::SMEM, stream, mkv, o);
        } else {
            lp_launch(attention_own_rows_kernel<HD, true>, grid, dim3(128), OwnRows<HD>::SMEM, stream, mkv, o);
            rc = lp_check_launch("attention_shared");
            if (rc) return rc;
            const long long rows = 128 / (HD / 4);
            lp_launch(attention_join_kernel<HD>, dim3((unsigned)(((long long)s.T * s.H + rows - 1) / rows)), dim3(128), 0, stream, o);
        }
    }
    return lp_check_launch("attention_shared");
}

}  // namespace

// q, out: bf16 [T, H, hd]; pages bf16 [num_pages, 2, G, 64, hd]; table int32 [B, width], whose first shared_pages columns are
// the same in every row; q_start int32 [B + 1]; kv_len int32 [B], lengths with the new tokens, at most max_new of which a sequence
// has. splits: into how many CTAs the shared pages are cut (0: there is nothing for them); part_o, part_ml float32 [slots, T, H, hd] and
// [slots, T, H, 2] with slots = splits, or 2 splits if the tokens fill one tile of rows (T <= 128 / (H / G)), and room for one more if the
// own pages' results are to be joined `apart`.
extern "C" int lp_attention_shared(const void* q, void* out, const void* pages, long long num_pages, const int* table, int width, const int* q_start,
                                   const int* kv_len, int B, int T, int max_new, int H, int G, int hd, int shared_pages, float scale, int splits, int apart,
                                   float* part_o, float* part_ml, int* status, cudaStream_t stream) {
    if (B <= 0 || T <= 0 || max_new <= 0 || G <= 0 || H <= 0 || H % G || H / G > ROWS || (hd != 64 && hd != 128) || shared_pages < 0 || shared_pages > width)
        LP_REFUSE("attention_shared: %d sequences, %d tokens, %d heads on %d of %d, %d shared pages", B, T, H, G, hd, shared_pages);
    if (!(scale > 0.f)) LP_REFUSE("attention_shared: a scale of %g", (double)scale);
    if (splits < 0 || splits > 32 || (splits > 0) != (shared_pages > 0) || splits > shared_pages)
        LP_REFUSE("attention_shared: %d shares of %d pages", splits, shared_pages);
    if (B > 65535 || G > 65535 || num_pages * 2 * G * PAGE > 0x7fffffffll || ((uintptr_t)q | (uintptr_t)pages | (uintptr_t)out) & 15)
        LP_REFUSE("attention_shared: %d sequences, %lld pages for %d heads, or operands that are not aligned to 16 bytes", B, num_pages, G);
    const int R = H / G, one_tile = T <= ROWS / R;
    SharedArgs s = {(const __nv_bfloat16*)pages, num_pages, table, q_start, kv_len, part_o, part_ml, B, T, H, G, R, shared_pages, splits > 0 ? splits : 1, scale * LOG2E, status};
    OwnArgs o = {(const __nv_bfloat16*)q, (__nv_bfloat16*)out, table, width, q_start, kv_len, part_o, part_ml, B, T, H, G, R, shared_pages,
                 one_tile ? 2 * splits : splits, splits == 0, scale * LOG2E, status};
    return hd == 64 ? run<64>(q, pages, num_pages, max_new, apart && splits > 0, s, o, stream) : run<128>(q, pages, num_pages, max_new, apart && splits > 0, s, o, stream);
}
