// Log probabilities of given tokens, with the entropy of each distribution and its most likely tokens.
//
// For a row x of V logits and a token t:
//   log p[t] = x[t] - ln(sum_i exp(x[i])),   entropy = -sum_i p[i] ln p[i],
//   rank = how many tokens come before t in the order of falling logits (equal logits: the lower token first; a logit that
//   is not a number comes behind all others), and the first k tokens of that order with their log probabilities.
// Sums are taken against the row's maximum m over the others only: with c logits equal to m and r = sum of exp(x[i] - m) over
// the rest, ln(sum) = m + ln(c + r) is formed as log1p(c - 1 + r), so that a nearly certain token's log probability keeps its
// digits; the entropy is ln(c + r) - u / (c + r) with u = sum of (x[i] - m) exp(x[i] - m).
// A row without a distribution (it holds +inf or no number at all, or nothing but -inf) gets no number everywhere but in ranks and tokens.
//
// A row is read once. Every thread keeps (c, r, u) of what it has seen against its warp's maximum m and brings them down when that
// moves, which it does a few times per row: only then, and where a logit is -inf, are logits compared with m one by one. A
// warp keeps its k first tokens sorted over its lanes, and a logit is looked at again only if it is not below a bound that the
// warps' largest logits so far give. A cluster of CTAs shares a long row when the rows are few; their parts meet in the first CTA's
// registers through distributed shared memory, so there is no scratch in memory and no order of arrival: results repeat bit for bit.
//
// Bound by memory at many rows: 2,000 rows of 128,256 float32 logits (1.03 GB, 157 us at the measured copy rate) take 163 us without
// a list, 96 %, 180 with the most likely token and 211 with the 20 most likely ones (B200, one call behind the other): a row's first loads
// fill the lists of its eight warps, and its end is nobody's memory time. At few rows bound by latency: 6.6 us for one row of 32,000, 9.5 for 4
// and 13.5 for 48 of 128,256, with 5 tokens. Between them by the turns of a CTA, 1,200 cycles for 4,096 logits: 333 rows of 50,257
// bfloat16 logits (33 MB, 5.1 us) take 16 us without a list, 20 with one token and 28 with 20.
#include "common.cuh"

#include <type_traits>

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int CTAS_PER_SM = 3;
constexpr int MOST_TOP = 32;
constexpr int MOST_CLUSTER = 8;
constexpr int PENDING = 64;
constexpr int VALUES = 16;                       // logits that a thread has in hand at a time
constexpr uint32_t ALL = 0xffffffffu;

// ------------------------------------------------------------------ the order of the tokens
// A logit as an unsigned number of the same order (both zeros alike, no number below everything), and with its token: the larger
// comes first. 0 is nobody.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return x != x ? 0u : ((int)u < 0 ? ~u : u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return k == 0 ? __uint_as_float(0x7fffffffu) : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t entry(float x, int i) { return ((uint64_t)order_key(x) << 32) | (uint32_t)~i; }
__device__ __forceinline__ bool before(float x, int i, float y, int j) { return entry(x, i) > entry(y, j); }

// 32 entries, one per lane, in falling order
__device__ __forceinline__ uint64_t sort32(uint64_t v, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            const uint64_t w = __shfl_xor_sync(ALL, v, stride);
            const bool larger = ((lane & stride) == 0) == ((lane & size) == 0);
            v = (v > w) == larger ? v : w;
        }
    return v;
}
// the first 32 of two sorted lists
__device__ __forceinline__ uint64_t merge32(uint64_t a, uint64_t b, int lane) {
    const uint64_t w = __shfl_sync(ALL, b, 31 - lane);
    a = a > w ? a : w;
#pragma unroll
    for (int stride = 16; stride > 0; stride >>= 1) {
        const uint64_t p = __shfl_xor_sync(ALL, a, stride);
        a = (a > p) == ((lane & stride) == 0) ? a : p;
    }
    return a;
}
// ------------------------------------------------------------------ sums against a maximum
constexpr float LOG2E = 1.4426950408889634f;
// the hardware's exp2: within 2^-22 of the value, and each term is rounded by as much already
__device__ __forceinline__ float fast_exp2(float t) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
    return y;
}
__device__ __forceinline__ float fast_exp(float d) { return fast_exp2(d * LOG2E); }
// Two float32 operations in one instruction (Blackwell's packed forms); each half is rounded as by the scalar operation.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void halves(float& a, float& b, uint64_t v) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ void add2(float& x0, float& x1, float y0, float y1) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(pair(x0, x1)), "l"(pair(y0, y1)));
    halves(x0, x1, v);
}
__device__ __forceinline__ void add2(float& x0, float& x1, float y) { add2(x0, x1, y, y); }
__device__ __forceinline__ void mul2(float& z0, float& z1, float x0, float x1, float y) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(pair(x0, x1)), "l"(pair(y, y)));
    halves(z0, z1, v);
}
__device__ __forceinline__ void fma2(float& z0, float& z1, float x0, float x1, float y0, float y1) {      // z += x * y
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(pair(x0, x1)), "l"(pair(y0, y1)), "l"(pair(z0, z1)));
    halves(z0, z1, v);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
struct Sums {
    float m, c, r, u;           // maximum, how often it occurs, the others' sum and weighted sum against it
    int ahead;                  // logits before the target's
    // The same against a larger maximum. A part that has seen nothing but -inf adds nothing, one that has seen no numbers passes that on.
    __device__ __forceinline__ void lower(float to) {
        const float d = fmaxf(m - to, -1e30f), f = m == to ? 1.f : expf(d), w = (m == -INFINITY ? 0.f : c) + r;
        u = f * (u + w * d);
        r = f * w;
        c = 0.f;
        m = to;
    }
};

// ------------------------------------------------------------------ loads: 16 bytes at a time, the row's ends one by one
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void spread(const uint4& v, float* x) {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 gather(const float* row, int i0, int V) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = i0 + e >= 0 && i0 + e < V ? row[i0 + e] : -INFINITY;
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
    static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void spread(const uint4& v, float* x) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[2 * e] = __uint_as_float(w[e] << 16); x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
    }
    static __device__ __forceinline__ uint4 gather(const __nv_bfloat16* row, int i0, int V) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int a = i0 + 2 * e, b = a + 1;
            const uint32_t lo = a >= 0 && a < V ? __bfloat16_as_ushort(row[a]) : 0xff80u;
            const uint32_t hi = b >= 0 && b < V ? __bfloat16_as_ushort(row[b]) : 0xff80u;
            w[e] = lo | hi << 16;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
};
__device__ __forceinline__ uint4 load_once(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(const void* p, int cta) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(cta));
    return a;
}
__device__ __forceinline__ uint32_t remote_word(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

// The candidates of a CTA (in the first CTA of a cluster: of all) and the first k of them; its sums.
struct Found {
    __align__(16) uint64_t pool[WARPS * (MOST_TOP + PENDING)];
    uint64_t best[MOST_TOP];
    int count;
};
static_assert(WARPS * (MOST_TOP + PENDING) >= MOST_CLUSTER * MOST_TOP && MOST_CLUSTER <= 32 && WARPS <= 32, "one lane per part, room for all lists");

// grid: (rows x cluster); the CTAs of a cluster take consecutive slices of one row.
template <typename T, bool TOP>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM)
token_logprobs_kernel(const T* __restrict__ logits, long long ld, const int* __restrict__ targets, float* __restrict__ logprob,
                      float* __restrict__ entropy, int* __restrict__ rank, int* __restrict__ top_ids, float* __restrict__ top_logprobs,
                      int V, int top, int cluster) {
    constexpr int N = Vec<T>::N, PER = VALUES / N;             // logits per vector, vectors in hand
    __shared__ Sums parts[WARPS];
    __shared__ Sums whole;
    __shared__ Found found;
    __shared__ uint64_t pending[TOP ? WARPS : 1][PENDING];       // candidates of a warp, not yet in its list
    __shared__ __align__(16) float offers[TOP ? WARPS : 1][32][VALUES];
    __shared__ uint32_t posts[WARPS];                            // each warp has `per_warp` logits that are not below this key
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.x / cluster, share = blockIdx.x - row * cluster;
    lp_grid_wait();
    const T* x = logits + (long long)row * ld;
    const int lead = (int)(((uintptr_t)x & 15) / sizeof(T));     // logits of the first vector that lie before the row
    const int vectors = (int)(((long long)V + lead + N - 1) / N);
    const int each = (vectors + cluster - 1) / cluster;
    const int from = share * each, to = min(vectors, from + each);
    // Vectors that lie wholly in the row and the share need no look at their ends.
    const int whole_from = max(from, lead > 0 ? 1 : 0), whole_to = min(to, (int)(((long long)V + lead) / N));
    const T* mine = x - lead + (long long)threadIdx.x * N;
    uint4 next[PER];
    auto fetch = [&](int w0) {
        if (w0 >= whole_from && w0 + PER * THREADS <= whole_to) {
            const T* p0 = mine + (long long)w0 * N;
#pragma unroll
            for (int p = 0; p < PER; ++p) next[p] = load_once(p0 + p * THREADS * N);
        } else {
#pragma unroll
            for (int p = 0; p < PER; ++p) {
                const int w = w0 + p * THREADS + (int)threadIdx.x;
                next[p] = w >= to ? Vec<T>::nothing() : (w >= whole_from && w < whole_to) ? load_once(mine + (long long)(w0 + p * THREADS) * N)
                                                                                           : Vec<T>::gather(x, w * N - lead, V);
            }
        }
    };
    fetch(from);
    const int target = targets[row];
    const bool real = target >= 0 && target < V;
    const float xt = real ? lp_to_float(x[target]) : INFINITY;
    // A logit comes before the target's if it is larger, and if it is equal and its token lower: in front of the target it is larger than the
    // number below the target's. -inf has none below and also stands for what is not in the row: in front of it all numbers count, where
    // all are in the row. One by one only what is left: around such a target, and where the target's logit is no number.
    const bool in_order = !real || xt > -INFINITY;
    const float below = xt == 0.f ? -__uint_as_float(1u) : __int_as_float(__float_as_int(xt) + (xt > 0.f ? -1 : 1));

    Sums s = {-INFINITY, 0.f, 0.f, 0.f, 0};
    uint64_t list = 0, kth = 0;          // the warp's first tokens over its lanes, and the last of the first k
    int held = 0;                        // candidates in `pending`
    auto flush = [&]() {                 // up to 32 of them into the list
        __syncwarp();
        const int n = min(held, 32);
        const uint64_t v = lane < n ? pending[warp][held - n + lane] : 0;
        held -= n;
        list = merge32(list, sort32(v, lane), lane);
        kth = __shfl_sync(ALL, list, top - 1);
        __syncwarp();
    };
    const int per_warp = (top + WARPS - 1) / WARPS, warps_needed = per_warp ? (top + per_warp - 1) / per_warp : 0;
    float lane_most = -INFINITY;
    uint32_t bound = 0;                  // no logit below this key is among the first k
    // Each warp posts a key that per_warp of its lanes have a logit at or above: enough warps' keys are below k logits or are them.
    // (-inf may stand for no logit at all.)
    auto warps_key = [&]() {
        uint32_t key = order_key(lane_most), most = 0;
        if (key <= 0x007fffffu) key = 0;
        for (int i = 0; i < per_warp; ++i) {
            most = __reduce_max_sync(ALL, key);
            if (lane == __ffs(__ballot_sync(ALL, key == most)) - 1) key = 0;
        }
        return most;
    };
    auto posts_bound = [&]() {
        const volatile uint32_t* const posted = posts;
        const uint32_t post = lane < WARPS ? posted[lane] : 0u;
        int place = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const uint32_t other = __shfl_sync(ALL, post, w);
            if (other > post || (other == post && w < lane)) ++place;
        }
        const uint32_t who = __ballot_sync(ALL, lane < WARPS && place == warps_needed - 1);
        return __shfl_sync(ALL, post, __ffs(who) - 1);
    };
    float cut = key_value(0);
    int turn = 0, again = 0;
    bool offered = false;
    for (int w0 = from; w0 < to; w0 += PER * THREADS) {
        float v[VALUES];
#pragma unroll
        for (int p = 0; p < PER; ++p) Vec<T>::spread(next[p], v + p * N);
        if (w0 + PER * THREADS < to) fetch(w0 + PER * THREADS);
        float most = max3(v[0], v[1], v[2]), least = min3(v[0], v[1], v[2]);
#pragma unroll
        for (int j = 3; j + 1 < VALUES; j += 2) {
            most = max3(most, v[j], v[j + 1]);
            least = min3(least, v[j], v[j + 1]);
        }
        most = fmaxf(most, v[VALUES - 1]);
        least = fminf(least, v[VALUES - 1]);
        // Against the warp's maximum, two logits at a time. Where a logit is -inf (or so low that the difference overflows) the
        // weighted sum takes its term, zero times that, against a finite difference.
        auto add_up = [&](auto masked) {
            float r0 = 0.f, r1 = 0.f, u0 = 0.f, u1 = 0.f;
#pragma unroll
            for (int j = 0; j < VALUES; j += 2) {
                float d0 = v[j], d1 = v[j + 1], t0, t1;
                add2(d0, d1, -s.m);
                mul2(t0, t1, d0, d1, LOG2E);
                t0 = fast_exp2(t0);
                t1 = fast_exp2(t1);
                add2(r0, r1, t0, t1);
                if (masked.value) { d0 = fmaxf(d0, -1e30f); d1 = fmaxf(d1, -1e30f); }
                fma2(u0, u1, t0, t1, d0, d1);
            }
            s.r += r0 + r1;
            s.u += u0 + u1;
        };
        if (__any_sync(ALL, most >= s.m)) {
            // a logit that reaches the warp's maximum: one by one
            const float peak = key_value(max(__reduce_max_sync(ALL, order_key(most)), 0x007fffffu));
            if (peak > s.m) s.lower(peak);
            const float ref = fmaxf(s.m, -3.402823466e38f);          // so that -inf - ref is -inf
#pragma unroll
            for (int j = 0; j < VALUES; ++j) {
                const float d = v[j] - ref, e = fast_exp(d);
                if (v[j] == s.m) s.c += 1.f;
                else s.r += e;
                s.u = fmaf(e, fmaxf(d, -1e30f), s.u);
            }
        } else if (__any_sync(ALL, least - s.m < -3e38f)) add_up(std::true_type());
        else add_up(std::false_type());
        // the target's rank
        const int at0 = w0 * N - lead;                                // the first logit in the CTA's hands
        const bool behind = at0 > target, in_front = at0 + PER * THREADS * N <= target;
        if (in_order || (xt == -INFINITY && behind)) {
            if (__any_sync(ALL, most >= xt)) {
                if (behind || in_front) {
                    const float limit = behind ? xt : below;
#pragma unroll
                    for (int j = 0; j < VALUES; ++j)
                        if (v[j] > limit) ++s.ahead;
                } else {
#pragma unroll
                    for (int j = 0; j < VALUES; ++j)
                        if (v[j] > (at0 + (j / N * THREADS + (int)threadIdx.x) * N + j % N < target ? below : xt)) ++s.ahead;
                }
            }
        } else if (xt == -INFINITY && in_front && w0 >= whole_from && w0 + PER * THREADS <= whole_to) {
#pragma unroll
            for (int j = 0; j < VALUES; ++j)
                if (v[j] == v[j]) ++s.ahead;
        } else {
#pragma unroll
            for (int j = 0; j < VALUES; ++j) {
                const int w = w0 + j / N * THREADS + (int)threadIdx.x, i = w * N - lead + j % N;
                if (i >= 0 && i < V && w < to && before(v[j], i, xt, target)) ++s.ahead;
            }
        }
        if (TOP) {
            lane_most = fmaxf(lane_most, most);
            if (turn == 0 || (offered && turn >= again)) {
                again = 2 * turn + 1;
                offered = false;
                // At first, and when something was offered since and as much has been seen again as before. Posts only rise, so an old one
                // holds as well.
                const uint32_t key = warps_key();
                volatile uint32_t* const posted = posts;
                if (lane == 0) posted[warp] = key;
                if (turn == 0) __syncthreads();
                bound = max(bound, posts_bound());
                cut = key_value(max(bound, (uint32_t)(kth >> 32)));
            }
            ++turn;
            uint32_t who = __ballot_sync(ALL, !(most < cut));
            if (who) {
                offered = true;
                // The lanes with something to offer lay out what they hold, and the warp goes through two lanes' logits at a time.
                if (!(most < cut)) {
#pragma unroll
                    for (int j = 0; j < VALUES; j += 4)
                        *reinterpret_cast<float4*>(&offers[warp][lane][j]) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                }
                __syncwarp();
                while (who) {
                    const int a = __ffs(who) - 1;
                    who &= who - 1;
                    const int b = who ? __ffs(who) - 1 : -1;
                    who &= who - 1;
                    const int from_lane = lane < 16 ? a : b, j = lane & 15;
                    uint64_t mine = 0;
                    if (from_lane >= 0) {
                        const int w = w0 + j / N * THREADS + warp * 32 + from_lane, i = w * N - lead + j % N;
                        if (i >= 0 && i < V && w < to) mine = entry(offers[warp][from_lane][j], i);
                    }
                    const bool in = mine > kth && (uint32_t)(mine >> 32) >= bound;
                    const uint32_t all = __ballot_sync(ALL, in);
                    if (in) pending[warp][held + __popc(all & ((1u << lane) - 1))] = mine;
                    held += __popc(all);
                    if (held >= 32) flush();
                }
                __syncwarp();
                cut = key_value(max(bound, (uint32_t)(kth >> 32)));
            }
        }
    }
    lp_grid_release();

    // ---------------------------------------------------------------- the warps' parts, then the CTAs'
    // a warp's lanes have one maximum
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s.c += __shfl_xor_sync(ALL, s.c, o);
        s.r += __shfl_xor_sync(ALL, s.r, o);
        s.u += __shfl_xor_sync(ALL, s.u, o);
    }
    s.ahead = __reduce_add_sync(ALL, s.ahead);
    if (lane == 0) parts[warp] = s;
    if (TOP) {
        const uint32_t key = warps_key();
        if (lane == 0) posts[warp] = key;
        if (threadIdx.x == 0) found.count = 0;
    }
    __syncthreads();
    const Sums nothing = {-INFINITY, 0.f, 0.f, 0.f, 0};
    static_assert(WARPS <= 8 && MOST_CLUSTER <= 8, "parts meet in eight lanes");
    auto sums_meet = [&]() {                                     // those of a warp's first eight lanes
        float most = s.m;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(ALL, most, o));
        if (s.m < most) s.lower(most);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            s.c += __shfl_xor_sync(ALL, s.c, o);
            s.r += __shfl_xor_sync(ALL, s.r, o);
            s.u += __shfl_xor_sync(ALL, s.u, o);
            s.ahead += __shfl_xor_sync(ALL, s.ahead, o);
        }
    };
    if (warp == 0) {
        s = lane < WARPS ? parts[lane] : nothing;
        sums_meet();
        if (lane == 0) whole = s;
    }
    // A candidate's place is the number of candidates before it: no sorting, and the order in which they lie does not matter.
    auto place_of = [&](uint64_t mine, int n) {
        int place = 0;
#pragma unroll 4
        for (int i = 0; i < n; i += 2) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&found.pool[i]);
            place += (two.x > mine ? 1 : 0) + (two.y > mine && i + 1 < n ? 1 : 0);
        }
        return place;
    };
    int candidates = 0;
    if (TOP) {
        bound = max(bound, posts_bound());
        const uint64_t other = lane < held ? pending[warp][lane] : 0;        // fewer than 32
        const bool a = lane < top && list != 0 && (uint32_t)(list >> 32) >= bound, b = other != 0 && (uint32_t)(other >> 32) >= bound;
        const uint32_t listed = __ballot_sync(ALL, a), others = __ballot_sync(ALL, b), before_me = (1u << lane) - 1;
        int at = 0;
        if (lane == 0) at = atomicAdd(&found.count, __popc(listed) + __popc(others));
        at = __shfl_sync(ALL, at, 0);
        if (a) found.pool[at + __popc(listed & before_me)] = list;
        if (b) found.pool[at + __popc(listed) + __popc(others & before_me)] = other;
        if (warp == 0) found.best[lane] = 0;
        __syncthreads();
        candidates = found.count;
    }
    if (cluster > 1) {
        if (TOP)
            for (int i = threadIdx.x; i < candidates; i += THREADS) {
                const uint64_t mine = found.pool[i];
                const int place = place_of(mine, candidates);
                if (place < top) found.best[place] = mine;
            }
        cluster_sync();
        if (share == 0) {
            if (warp == 0) {
                s = nothing;
                if (lane < cluster) {
                    const uint32_t a = remote(&whole, lane);
                    s = {__uint_as_float(remote_word(a)), __uint_as_float(remote_word(a + 4)), __uint_as_float(remote_word(a + 8)),
                         __uint_as_float(remote_word(a + 12)), (int)remote_word(a + 16)};
                }
                sums_meet();
                __syncwarp();
                if (lane == 0) whole = s;                        // nobody else reads this CTA's
            }
            if (TOP) {
                candidates = cluster * top;
                for (int i = threadIdx.x; i < candidates; i += THREADS) {
                    const uint32_t a = remote(&found.best[i % top], i / top);
                    found.pool[i] = (uint64_t)remote_word(a + 4) << 32 | remote_word(a);
                }
            }
        }
        cluster_sync();                                          // the others' shared memory stays until it has been read
    } else __syncthreads();
    if (share == 0) {
        s = whole;
        const bool none = !(s.m > -INFINITY && s.m < INFINITY) || s.r != s.r;
        const float log_s = none ? NAN : log1pf((s.c - 1.f) + s.r);
        if (threadIdx.x == 0) {
            logprob[row] = real ? (xt - s.m) - log_s : NAN;
            entropy[row] = log_s - s.u / (s.c + s.r);
            rank[row] = real ? s.ahead : -1;
        }
        if (TOP)
            for (int i = threadIdx.x; i < candidates; i += THREADS) {
                const uint64_t mine = found.pool[i];
                const int place = mine != 0 ? place_of(mine, candidates) : top;
                if (place < top) {
                    top_ids[(long long)row * top + place] = (int)~(uint32_t)mine;
                    top_logprobs[(long long)row * top + place] = (key_value((uint32_t)(mine >> 32)) - s.m) - log_s;
                }
            }
    }
}

template <typename T>
int launch(const void* logits, long long ld, const int* targets, float* logprob, float* entropy, int* rank, int* top_ids, float* top_logprobs,
           int rows, int V, int top, int cluster, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * cluster));
    cfg.blockDim = dim3(THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (lp_pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    cudaLaunchKernelEx(&cfg, top ? token_logprobs_kernel<T, true> : token_logprobs_kernel<T, false>, (const T*)logits, ld, targets, logprob, entropy,
                       rank, top_ids, top_logprobs, V, top, cluster);
    return lp_check_launch("token_logprobs");
}

}  // namespace

// logits: rows of `ld` elements (float32 or bfloat16); targets, rank int32 [rows]; logprob, entropy float32 [rows];
// top_ids int32, top_logprobs float32 [rows, top] (null for top == 0).
extern "C" int lp_token_logprobs(const void* logits, int dtype, long long ld, const int* targets, float* logprob, float* entropy, int* rank,
                                 int* top_ids, float* top_logprobs, int rows, int V, int top, cudaStream_t stream) {
    if (rows <= 0 || V <= 0 || top < 0 || top > MOST_TOP || top > V || ld < V || rows > 0x7fffffff / MOST_CLUSTER || V > 0x7fffffff - 4 * THREADS * VALUES)
        LP_REFUSE("token_logprobs: %d rows of %d logits, the %d most likely", rows, V, top);
    // Few rows: as many CTAs per row as the GPU holds at once, each with half a load of its threads at least. B200, 128,256 float32 logits,
    // 5 tokens, us (cold) with 1, 2, 4 and 8 CTAs per row: 1 row 31, 23, 18, 14; 48 rows 33, 25, 21, 21; 100 rows 33, 29, 25, 37;
    // 220 rows 39, 35, 49, 61; 300 rows 49, 51, 57, 78; 8 rows of 2,000 10, 12, 12, 12; 1 row of 32,000 14, 14, 12, 12.
    int cluster = 1;
    while (cluster < MOST_CLUSTER && (long long)rows * cluster * 2 <= (long long)lp_sm_count() * CTAS_PER_SM && V / (cluster * 2) >= THREADS * VALUES / 2) cluster *= 2;
    if (dtype == LP_F32)
        return launch<float>(logits, ld, targets, logprob, entropy, rank, top_ids, top_logprobs, rows, V, top, cluster, stream);
    return launch<__nv_bfloat16>(logits, ld, targets, logprob, entropy, rank, top_ids, top_logprobs, rows, V, top, cluster, stream);
}
