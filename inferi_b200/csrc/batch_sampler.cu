// A token for every row of logits, each row with settings of its own: temperature, top-k, top-p, min-p (ib_sample_batch).
//
//   w_i = exp((x_i - max x) / temperature), the rows sorted by (x descending, index ascending), S_m = sum of the first m weights
//   kept: the first min(k, m_min, m_p) of them; m_min = how many w_i >= min_p; m_p = the first m with S_m > top_p * S_k
//   token: the first one with S_m > coin * S_kept.  Rows without a filter: the same over the tokens in index order.
// That is what `Sampler` does where it offers the same (temperature and top-p; crates/inferi/src/models/sampler.rs:32-130).
//
// Which token it is hangs on sums of up to half a million weights next to a border, and on a flat distribution the border is 1e-5 of the sum away.  So weights are whole numbers, in units
// of 2^-44 of the largest, good to 3e-10 of themselves: (x - max) log2(e) / T is one product of doubles, added to 1.5 * 2^20 so that its whole and fractional parts
// are words of the result; 2^fraction is a table of 256 and three steps of a series in 32-bit fixed point.  Sums of whole numbers do not depend on their order.  Of a row with filters, the weights
// below the histogram (below) mostly matter as one sum only, and that only to top_p's bound: there ex2.approx in 32 bits will do, with a bound on what their sum is off by (BS_LOOSE).  Where the element
// that top_p's border falls on is the same with that much more and less, it is the one that the exact sum gives; where it is not, or the whole is what the coin is held against, the sums are formed anew
// from whole numbers (BS_EXACT).  Rows without a filter have nothing but exact sums.
//
// A row is a thread-block cluster of up to 8 CTAs, each with a slice of the row in shared memory: one read of the row from HBM, and what follows passes over shared memory.  A warp goes over its
// stretch of the slice once, adds up the small weights and lists the places of the others, which it takes together then (a few per cent of a language model's logits: with some of them
// among the 32 lanes of every step, all of it ran at the price of the large ones).
// Nothing is sorted but a list of at most 1024 elements: every border asks for the element at which a running count or sum in sorted order crosses a bound, and a histogram
// (count and weight over 1024 equal stretches of x, those of the largest 16 factors of two) says which bin that is; its elements - or, where they fit, all up to
// there, so that one list answers every question - are listed and sorted.  Bins too full for the list (ties) or below the histogram: the same by digits of x's order, to the last
// tie in index order.  The first CTA of the cluster leads: it looks at the merged histogram and says what all do next (BsStep).  Its threads carry the same state and search sums by
// bisection, each for itself, without barriers.
// What bounds it, at 128,256 logits: a chain of barriers, scans and short lists for few rows (one row with top-p 36 us, without a filter 13; 33 rows of 32,003 44 us); for many the passes over logits that
// have left the caches and the arithmetic of the elements in the histogram: 250 rows 173 us with settings of every row's own (one that takes BS_EXACT late lengthens that: 192 to 229 by the numbers drawn); all of them without a filter 111, top-k up to 200 163, top-p 0.5 to 0.99 259.
#include "op_launch.cuh"

#include <cooperative_groups.h>
#include <float.h>
#include <math.h>

namespace ib {

namespace cg = cooperative_groups;

constexpr uint32_t BS_THREADS = 512, BS_WARPS = BS_THREADS / 32, BS_CLUSTER = 8;
constexpr uint32_t BS_BINS = 1024, BS_LIST = 1024;
constexpr uint32_t BS_MAX_VOCAB = 1u << 19;   // S < 2^63
constexpr int BS_ONE = 44;                    // the largest weight is 2^44 units
// The histogram's reach below the largest weight, in factors of two, where no sample says better.  A border below it is looked for in a second one, of the stretch behind the first.  (Normal logits of
// deviation 3.  One row, top-k 50, reach 11 or 16: 29 and 36 us.)
constexpr double BS_OCTAVES = 16.0, BS_OCTAVES_K = 11.0;
// What a sum of small weights may be off by.  A weight t octaves below the largest: by 2^-24 t octaves in its difference and as many in its product with log2(e) / T, which is t 2^-23 ln 2 of it, by
// ex2.approx's 2^-22, and eight of them are added up in 32 bits, 7 * 2^-24.  That is 2.64e-6 of it at 24 octaves, 4.4e-6 at 44, where a weight is a unit; those behind 24 octaves are below 2^20 units each, so
// it is 4.6 units of each of them, and on the other side there is half a unit for every whole number.
constexpr double BS_LOOSE = 2.7e-6;
constexpr uint32_t BS_LOOSE_EACH = 6;
constexpr uint32_t BS_WINDOWS = 4;                  // such stretches, at most
// Vocabularies up to this size are one CTA's work, up to twice this size two CTAs' and so on: what a cluster's barriers cost is not less than what a small slice saves.  (Top-k 50, slices of 8192
// or 4096 at most: one row of 8000 20 and 23 us, 33 rows of 32,003 25 and 35; 12,000 at most: the same, but top-p 0.9 of one row of 20,000 35 and 39.)
constexpr uint32_t BS_ONE_CTA = 8192;
constexpr uint32_t BS_QUEUE = 16, BS_STEP = 8;  // a thread's elements that wait to be taken; those that come together
constexpr uint32_t BS_KEPT = 768;             // the histogram's elements whose places a warp keeps
constexpr uint32_t BS_SAMPLE = 4096, BS_SAMPLED = 20000;   // logits that say how far the histogram should reach, for slices above that size (250 rows, top-p 0.9: 236 us, without 306; one row in slices of 16,032: 44 and 45, top-k 50 30 and 29)
constexpr uint32_t BS_SMEM_LIMIT = 227 * 1024;

struct BatchSampleParams {
    const float *logits;
    uint64_t stride;
    uint32_t n, slice, resident, sampled;   // tokens of a row, of a CTA; whether a slice is held in shared memory; whether some logits say how far the histogram goes
    const float *temperature, *top_p, *min_p, *coin;
    const int32_t *top_k;
    int32_t *token;
    float *prob;
};

// 2^(i / 256) with 31 fractional bits
struct BsTable { uint32_t t[256]; };
constexpr BsTable bs_make_table() {
    BsTable r = {};
    double x = 2147483648.0;
    for (int i = 0; i < 256; i++) {
        r.t[i] = (uint32_t)(x + 0.5);
        x *= 1.0027112750502025;   // 2^(1 / 256)
    }
    return r;
}
__device__ const BsTable bs_table = bs_make_table();

enum BsStep : uint32_t { BS_DONE, BS_HISTOGRAM, BS_EXACT, BS_DIGIT, BS_LIST_BINS, BS_LIST_DIGITS, BS_COUNT_TIES, BS_PICK_TIE };

struct BsShared {
    uint32_t table[256];                                // 2^(i / 256), 31 fractional bits
    uint32_t cnt[BS_BINS];                              // this CTA's histogram: elements ...
    union {
        uint2 mass[BS_BINS];                            // ... and their weight, as two words; in the first CTA, when a list is there,
        unsigned long long run[BS_LIST];                // the running weight through each of its elements
    };
    union {
        struct {
            unsigned long long tot_mass[BS_BINS];       // first CTA: the cluster's histogram, then the sums ahead of each bin
            uint32_t tot_cnt[BS_BINS];
            unsigned long long list[BS_LIST];           // listed elements, (~order of x, index)
        };
        struct {                                        // before there is any of these, by threads: elements that wait to be taken, and their places in the warp's stretch
            float wait_x[BS_WARPS][BS_QUEUE][32];
            uint16_t wait_at[BS_WARPS][BS_QUEUE][32];
        };
    };
    uint16_t kept[BS_WARPS][BS_KEPT];                   // places in its stretch of a warp's elements that are in the histogram
    unsigned long long seg[BS_CLUSTER * BS_WARPS];      // weight of every warp's stretch of the row; in the first CTA, or a count
    unsigned long long red[2][BS_WARPS];
    float lo[BS_CLUSTER];                               // of every CTA's slice: its smallest finite logit
    unsigned long long best[BS_CLUSTER];                // ... and its arg-max
    unsigned long long loose[BS_WARPS];                 // of every warp's small weights: their sum in 32 bits
    unsigned long long part_loose[BS_CLUSTER], part_min[BS_CLUSTER];   // first CTA: of each slice, its small weights, and its elements with w >= min_p
    uint32_t part_cnt[BS_CLUSTER], part_min_cnt[BS_CLUSTER];
    // what the first CTA says
    uint32_t step, a, b, prefix;
    unsigned long long arg;
    uint32_t listed;
    // first CTA: the whole histogram's sums
    unsigned long long all_mass;
    uint32_t all_cnt;
};

// the order of x as a number: larger x, larger number
__device__ __forceinline__ uint32_t bs_order(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float bs_value(uint32_t order) { return __uint_as_float(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order); }
// what is no number is never drawn; an infinity is the largest number; the zeros are the same
__device__ __forceinline__ float bs_clean(float x) { return x > -INFINITY ? fminf(x, FLT_MAX) + 0.f : -INFINITY; }

// Sum over a warp of numbers below 2^44: the halves in the reduction unit
__device__ __forceinline__ unsigned long long bs_sum(unsigned long long w) {
    return (unsigned long long)__reduce_add_sync(0xffffffffu, (uint32_t)w & 0x3FFFFFu) + ((unsigned long long)__reduce_add_sync(0xffffffffu, (uint32_t)(w >> 22)) << 22);
}

static_assert(BS_MAX_VOCAB / BS_WARPS <= 65536, "places are 16 bits");

struct BsWeight {
    float hi;
    double c;   // log2(e) / temperature
    // of x <= hi; 0 for -infinity only
    __device__ __forceinline__ unsigned long long operator()(float x, const uint32_t *table) const {
        const double d = ((double)x - (double)hi) * c;
        if (!(d > -(double)BS_ONE)) return x == -INFINITY ? 0ull : 1ull;
        const double y = d + 1572864.0;   // 1.5 * 2^20: a step of the sum is 2^-32
        const uint32_t f = (uint32_t)__double2loint(y), down = 0x80000u - ((uint32_t)__double2hiint(y) & 0xFFFFFu);   // d = f / 2^32 - down
        const uint32_t r = f << 8, t = table[f >> 24];
        // 2^(r / 2^40) - 1 = z + z^2 / 2 + z^3 / 6, z = ln 2 * r / 2^40, times 2^40
        const uint32_t q = __umulhi(r, __umulhi(r, __umulhi(r, 3638u) + 4030416u) + 2977044472u);
        const uint32_t w = t + (__umulhi(t, q) >> 8);   // 31 fractional bits
        return (((unsigned long long)w << (BS_ONE - 30)) >> down) + 1ull >> 1;   // (1 at least: down is 44 at most)
    }
};

// Sums ahead of each thread over the block, of two values; the totals.  Ends with a barrier.
__device__ __forceinline__ void bs_scan(unsigned long long &a, unsigned long long &b, unsigned long long &a_all, unsigned long long &b_all, BsShared &S) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned long long a0 = a, b0 = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= (uint32_t)o) { a += x; b += y; }
    }
    if (lane == 31) { S.red[0][warp] = a; S.red[1][warp] = b; }
    __syncthreads();
    unsigned long long ahead_a = 0, ahead_b = 0;
    a_all = b_all = 0;
#pragma unroll
    for (uint32_t w = 0; w < BS_WARPS; w++) {
        if (w == warp) { ahead_a = a_all; ahead_b = b_all; }
        a_all += S.red[0][w];
        b_all += S.red[1][w];
    }
    a += ahead_a - a0;
    b += ahead_b - b0;
    __syncthreads();
}

// Ascending sort of list[0 .. cap), cap a power of two: exchanges over fewer than 32 places are shuffles
__device__ __forceinline__ void bs_sort(unsigned long long *list, uint32_t cap) {
    const uint32_t tid = threadIdx.x;
    auto in_warps = [&](uint32_t k, uint32_t from) {
        for (uint32_t t = tid; t - (tid & 31) < cap; t += BS_THREADS) {
            unsigned long long v = t < cap ? list[t] : ~0ull;
            for (uint32_t j = from; j > 0; j >>= 1) {
                const unsigned long long o = __shfl_xor_sync(0xffffffffu, v, j);
                const bool keep_min = ((t & k) == 0) == ((t & j) == 0);
                v = keep_min ? (v < o ? v : o) : (v < o ? o : v);
            }
            if (t < cap) list[t] = v;
        }
        __syncthreads();
    };
    for (uint32_t k = 2; k <= cap; k <<= 1) {
        for (uint32_t j = k >> 1; j >= 32; j >>= 1) {
            for (uint32_t t = tid; t < cap / 2; t += BS_THREADS) {
                const uint32_t a = ((t & ~(j - 1)) << 1) | (t & (j - 1)), b = a | j;
                const unsigned long long x = list[a], y = list[b];
                if ((x > y) == ((a & k) == 0)) { list[a] = y; list[b] = x; }
            }
            __syncthreads();
        }
        in_warps(k, k < 64 ? k >> 1 : 16);
    }
}

__global__ void __launch_bounds__(BS_THREADS, 2) batch_sample_kernel(const __grid_constant__ BatchSampleParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    BsShared &S = *reinterpret_cast<BsShared *>(smem);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t C = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    BsShared &L = *cluster.map_shared_rank(&S, 0);   // the first CTA's
    auto barrier = [&]() { if (C > 1) cluster.sync(); else __syncthreads(); };
    const uint32_t i0 = min(p.n, rank * p.slice), len = min(p.n, i0 + p.slice) - i0;
    const float *from = p.logits + row * p.stride + i0;
    float *held = reinterpret_cast<float *>(smem + sizeof(BsShared));
    if (tid < 256) S.table[tid] = bs_table.t[tid];
    pdl_enter();

    const float T = p.temperature[row];
    const bool greedy = !(T > 0.f);
    const float coin = p.coin[row], top_p = p.top_p ? p.top_p[row] : 1.f, min_p = p.min_p ? p.min_p[row] : 0.f;
    const int32_t k = p.top_k ? p.top_k[row] : 0;
    const bool by_k = k > 0 && (uint32_t)k < p.n, by_p = top_p > 0.f && top_p < 1.f, by_min = min_p > 0.f, filtered = by_k || by_p || by_min;

    // the slice, its largest logit (lowest index on ties) and its smallest finite one
    float top = -INFINITY, lo = INFINITY;
    uint32_t top_at = i0 + tid;   // (a thread's first element, if it has one)
    constexpr uint32_t AT_ONCE = 16;
    auto look = [&](uint32_t i, float y) {
        const float x = bs_clean(y);
        const bool more = x > top;
        top = more ? x : top;
        top_at = more ? i0 + i : top_at;
        if (x > -INFINITY) lo = fminf(lo, x);
    };
    uint32_t done = 0;
    for (; done + AT_ONCE * BS_THREADS <= len; done += AT_ONCE * BS_THREADS) {   // (without a check for every element)
        const float *y = from + done + tid;
        float v[AT_ONCE];
#pragma unroll
        for (uint32_t e = 0; e < AT_ONCE; e++) v[e] = __ldg(y + e * BS_THREADS);
#pragma unroll
        for (uint32_t e = 0; e < AT_ONCE; e++) {
            if (p.resident) held[done + tid + e * BS_THREADS] = v[e];
            look(done + tid + e * BS_THREADS, v[e]);
        }
    }
    {
        float v[AT_ONCE];
#pragma unroll
        for (uint32_t e = 0; e < AT_ONCE; e++) v[e] = done + tid + e * BS_THREADS < len ? __ldg(from + done + tid + e * BS_THREADS) : -INFINITY;
#pragma unroll
        for (uint32_t e = 0; e < AT_ONCE; e++) {
            if (p.resident && done + tid + e * BS_THREADS < len) held[done + tid + e * BS_THREADS] = v[e];
            look(done + tid + e * BS_THREADS, v[e]);
        }
    }
    unsigned long long best = tid >= len ? 0ull : (unsigned long long)bs_order(top) << 32 | (0xFFFFFFFFu - top_at);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    if (lane == 0) {
        S.red[0][warp] = best;
        S.red[1][warp] = __float_as_uint(lo);
    }
    __syncthreads();
    if (C > 1) cluster.sync();   // every CTA of the cluster runs: its shared memory may be written
    if (tid < C) {
        for (uint32_t w = 0; w < BS_WARPS; w++) {
            best = max(best, S.red[0][w]);
            lo = fminf(lo, __uint_as_float((uint32_t)S.red[1][w]));
        }
        BsShared &to = *cluster.map_shared_rank(&S, tid);
        to.best[rank] = best;
        to.lo[rank] = lo;
    }
    barrier();
    for (uint32_t r = 0; r < C; r++) {
        best = r ? max(best, S.best[r]) : S.best[r];
        lo = r ? fminf(lo, S.lo[r]) : S.lo[r];
    }
    const float hi = bs_value((uint32_t)(best >> 32));
    if (greedy || hi == -INFINITY) {   // (uniform over the cluster)
        if (rank == 0 && tid == 0) {
            p.token[row] = (int32_t)(0xFFFFFFFFu - (uint32_t)best);
            if (p.prob) p.prob[row] = 1.f;
        }
        return;   // nobody reads another CTA's memory from here on
    }
    const BsWeight weight = {hi, 1.4426950408889634074 / (double)T};
    const float *here = p.resident ? held : from;   // (as they came)
    auto logit = [&](uint32_t i) { return bs_clean(here[i]); };
    // `body` for `many` elements of a warp, number k at place(k) of the slice; the loads of eight steps are in flight together (a slice that is not held comes from L2)
    auto sweep = [&](uint32_t many, auto place, auto body) {
        constexpr uint32_t K = 8;
        for (uint32_t k = lane; k - lane < many; k += 32 * K) {
            uint32_t at[K];
            float x[K];
#pragma unroll
            for (uint32_t e = 0; e < K; e++) at[e] = place(min(k + 32 * e, many - 1));
#pragma unroll
            for (uint32_t e = 0; e < K; e++) x[e] = here[at[e]];   // (without a condition: a branch each would wait for each)
#pragma unroll
            for (uint32_t e = 0; e < K; e++) body(at[e], k + 32 * e < many ? bs_clean(x[e]) : -INFINITY);
        }
    };
    // a warp's elements: a stretch of the slice
    const uint32_t stretch = ((len + BS_WARPS - 1) / BS_WARPS + 31) & ~31u, w0 = min(len, warp * stretch), w1 = min(len, w0 + stretch);

    auto scaled = [](float f, unsigned long long m) { return f > 0.f ? min((unsigned long long)((double)f * (double)m), m - 1) : 0ull; };   // f < 1
    auto exact_sums = [&]() {   // of the warp's stretch, for every CTA
        unsigned long long sum = 0ull;
        sweep(w1 - w0, [&](uint32_t k) { return w0 + k; }, [&](uint32_t, float x) { sum += weight(x, S.table); });
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane < C) cluster.map_shared_rank(&S, lane)->seg[rank * BS_WARPS + warp] = sum;
    };

    // ---- a row without a filter: index order ----
    if (!filtered) {
        exact_sums();
        barrier();
        // every warp finds the stretch of the crossing, from four sums a lane
        constexpr uint32_t E = BS_CLUSTER * BS_WARPS / 32;
        unsigned long long seg[E], upto = 0ull;
#pragma unroll
        for (uint32_t e = 0; e < E; e++) {
            seg[e] = E * lane + e < C * BS_WARPS ? S.seg[E * lane + e] : 0ull;
            upto += seg[e];
        }
        unsigned long long ahead = upto;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long t = __shfl_up_sync(0xffffffffu, upto, o);
            if ((int)lane >= o) upto += t;
        }
        ahead = upto - ahead;
        const unsigned long long total = __shfl_sync(0xffffffffu, upto, 31), bound = scaled(coin, total);
        uint32_t s = 0;
        for (; s + 1 < E && bound >= ahead + seg[s]; s++) ahead += seg[s];
        const int who = __ffs(__ballot_sync(0xffffffffu, bound < upto)) - 1;
        s = __shfl_sync(0xffffffffu, E * lane + s, who);
        ahead = __shfl_sync(0xffffffffu, ahead, who);
        if (rank == s / BS_WARPS) {
            // The CTA's warps share that stretch; the one whose part the crossing is in goes through it element by element.
            const uint32_t o = s % BS_WARPS, s0 = min(len, o * stretch), s1 = min(len, s0 + stretch), part = ((s1 - s0 + BS_WARPS - 1) / BS_WARPS + 31) & ~31u;
            const uint32_t p0 = min(s1, s0 + warp * part), p1 = min(s1, p0 + part);
            unsigned long long sum = 0ull, left = bound - ahead;
            sweep(p1 - p0, [&](uint32_t k) { return p0 + k; }, [&](uint32_t, float x) { sum += weight(x, S.table); });
#pragma unroll
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (lane == 0) S.red[0][warp] = sum;
            __syncthreads();
            uint32_t mine = 0;
            while (mine + 1 < BS_WARPS && left >= S.red[0][mine]) left -= S.red[0][mine++];
            if (warp == mine) {
                bool found = false;
                sweep(p1 - p0, [&](uint32_t k) { return p0 + k; }, [&](uint32_t i, float x) {
                    if (found) return;
                    const unsigned long long w = weight(x, S.table), all = bs_sum(w);
                    found = left < all;
                    if (!found) {
                        left -= all;
                        return;
                    }
                    unsigned long long run = w;
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const unsigned long long t = __shfl_up_sync(0xffffffffu, run, d);
                        if ((int)lane >= d) run += t;
                    }
                    if ((int)lane == __ffs(__ballot_sync(0xffffffffu, left < run)) - 1) {
                        p.token[row] = (int32_t)(i0 + i);
                        if (p.prob) p.prob[row] = (float)((double)w / (double)total);
                    }
                });
            }
        }
        return;   // nobody reads another CTA's memory from here on
    }

    // ---- what a step does ----
    // bins of x: equal stretches down from the largest logit
    // As far as the borders, if that can be told: min_p says so itself; where rank k or the mass top_p lies is seen from some of the row's logits, by half octaves.
    // (Every CTA of the row takes the same ones.  A border behind the reach costs another histogram, no more.)
    double octaves = by_k ? BS_OCTAVES_K : BS_OCTAVES;
    if (p.sampled && (by_k || by_p)) {
        octaves = BS_OCTAVES;
        constexpr uint32_t HALVES = 64, E = BS_SAMPLE / BS_THREADS;
        const bool all = p.n <= BS_SAMPLE;
        if (tid < HALVES) S.cnt[tid] = 0u;
        float x[E];
#pragma unroll
        for (uint32_t e = 0; e < E; e++) {
            const uint32_t j = e * BS_THREADS + tid, at = all ? j : (uint32_t)((uint64_t)(j >> 3) * p.n / (BS_SAMPLE / 8)) + (j & 7);   // (eight neighbours are a sector of memory)
            x[e] = at < p.n ? bs_clean(__ldg(p.logits + row * p.stride + at)) : -INFINITY;
        }
        __syncthreads();
        const float scale = 2.f * (float)weight.c;
#pragma unroll
        for (uint32_t e = 0; e < E; e++) {
            const float h = (hi - x[e]) * scale;
            if (h < (float)HALVES) atomicAdd(&S.cnt[(uint32_t)h], 1u);
        }
        __syncthreads();
        const float share = all ? 1.f : (float)p.n / (float)BS_SAMPLE;   // a sampled one stands for so many
        const float n0 = (float)S.cnt[2 * lane] * share, n1 = (float)S.cnt[2 * lane + 1] * share, octave = exp2f(-(float)lane);
        // By rank: where there are a quarter more, and six sampled ones.  By mass: where what is behind is less than 1 - top_p of the whole.  Many sampled ones are behind, few perhaps
        // in front, so the whole is taken as low as their scatter allows: 1.5 times the root of the sum of squares less.
        const float m0 = n0 * 0.84f * octave, m1 = n1 * 0.59f * octave;
        float sum = by_k ? n0 + n1 : m0 + m1, whole = m0 + m1, scatter = all ? 0.f : (m0 * 0.84f + m1 * 0.59f) * octave * share;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float t = by_k ? __shfl_up_sync(0xffffffffu, sum, o) : __shfl_down_sync(0xffffffffu, sum, o);
            if (by_k ? (int)lane >= o : (int)lane + o < 32) sum += t;
            whole += __shfl_xor_sync(0xffffffffu, whole, o);
            scatter += __shfl_xor_sync(0xffffffffu, scatter, o);
        }
        const float far = (1.f - top_p) * fmaxf(1.f, whole - 1.5f * sqrtf(scatter));
        const uint32_t in0 = __ballot_sync(0xffffffffu, by_k ? sum - n1 >= (float)k * 1.25f + 6.f * share : sum - m0 <= far);
        const uint32_t in1 = __ballot_sync(0xffffffffu, by_k ? sum >= (float)k * 1.25f + 6.f * share : sum - m0 - m1 <= far);
        const uint32_t l0 = in0 ? __ffs(in0) - 1 : 32, l1 = in1 ? __ffs(in1) - 1 : 32;
        octaves = fmin(octaves, fmin((double)l0 + 0.5, (double)l1 + 1.0) + 0.5);
        __syncthreads();   // (the counters are cleared for the histogram)
    }
    if (by_min && !(by_k && by_p)) octaves = fmin(octaves, 0.01 - log2((double)fmaxf(min_p, 1e-30f)));
    auto reach_of = [&](double octaves) { return (float)fmin(fmax(octaves, 0.01) / weight.c, (double)hi - (double)lo); };
    auto bins_of = [&](float reach) { return reach > 0.f && isfinite(reach) ? (float)BS_BINS * (1.f - 0x1p-20f) / reach : 0.f; };
    const float reach = reach_of(octaves);
    float per_bin = bins_of(reach);
    uint32_t window = 0;           // of the row's stretches of that length
    auto bin_of = [&](float x) {   // >= BS_BINS: not in this window
        const float d = (hi - x) * per_bin;
        const uint32_t u = (d < (float)(BS_BINS * BS_WINDOWS) ? (uint32_t)d : BS_BINS * BS_WINDOWS) - BS_BINS * window;
        return u < BS_BINS ? u : BS_BINS;
    };
    auto add = [&](uint32_t bin, unsigned long long w) {
        atomicAdd(&S.cnt[bin], 1u);
        const uint32_t l = (uint32_t)w, old = atomicAdd(&S.mass[bin].x, l), h = (uint32_t)(w >> 32) + ((uint32_t)(old + l) < old ? 1u : 0u);
        if (h) atomicAdd(&S.mass[bin].y, h);
    };
    auto clear = [&]() {
        for (uint32_t b = tid; b < BS_BINS; b += BS_THREADS) {
            S.cnt[b] = 0u;
            S.mass[b] = make_uint2(0u, 0u);
        }
        __syncthreads();
    };
    // the CTAs' histograms together in the first CTA: each adds up a part of the bins
    auto merge = [&]() {
        barrier();
        const uint32_t share = (BS_BINS + C - 1) / C;
        for (uint32_t b = rank * share + tid; b < min(BS_BINS, (rank + 1) * share); b += BS_THREADS) {
            unsigned long long m = 0ull;
            uint32_t n = 0u;
#pragma unroll
            for (uint32_t r = 0; r < BS_CLUSTER; r++)
                if (r < C) {
                    const BsShared &o = *cluster.map_shared_rank(&S, r);
                    const uint2 x = o.mass[b];
                    m += ((unsigned long long)x.y << 32) + x.x;
                    n += o.cnt[b];
                }
            L.tot_mass[b] = m;
            L.tot_cnt[b] = n;
        }
        barrier();
        // sums ahead of each bin (a thread's two bins follow one another)
        if (rank == 0) {
            static_assert(BS_BINS == 2 * BS_THREADS, "two bins per thread");
            const unsigned long long m0 = S.tot_mass[2 * tid], n0 = S.tot_cnt[2 * tid];
            unsigned long long m = m0 + S.tot_mass[2 * tid + 1], n = n0 + S.tot_cnt[2 * tid + 1], all_m, all_n;
            bs_scan(m, n, all_m, all_n, S);
            S.tot_mass[2 * tid] = m; S.tot_cnt[2 * tid] = (uint32_t)n;
            S.tot_mass[2 * tid + 1] = m + m0; S.tot_cnt[2 * tid + 1] = (uint32_t)(n + n0);
            if (tid == 0) { S.all_mass = all_m; S.all_cnt = (uint32_t)all_n; }
            __syncthreads();
        }
    };

    // ---- the weights: sums of every stretch and slice, and the histogram ----
    const unsigned long long least = by_min ? (min_p > 1.f ? (1ull << BS_ONE) + 1 : (unsigned long long)ceil((double)min_p * (double)(1ull << BS_ONE))) : 0ull;
    // elements that are looked at one by one: those of the histogram (and a little more), and what may reach min_p (a factor of two more: rounding)
    const float near = fmaxf(per_bin > 0.f && weight.c < (double)FLT_MAX ? reach * (1.f + 0x1p-18f) : INFINITY, by_min ? (float)((1.0 - log2((double)fmaxf(min_p, 1e-30f))) / weight.c) : 0.f);
    const float c_hi = (float)weight.c, c_lo = (float)(weight.c - (double)c_hi);
    uint32_t n_places = 0;      // the warp's kept places
    bool all_kept = true;     // they are those of all of its elements of the histogram
    {
        clear();
        unsigned long long sum = 0ull, above = 0ull;
        uint32_t n = 0u, n_above = 0u, waiting = 0u;
        double small = 0.0;
        auto take = [&]() {
            // one behind the other, from the front: a place that is written has been read
            float *queue_x = &S.wait_x[warp][0][0];
            uint16_t *queue_at = &S.wait_at[warp][0][0];
            const uint32_t below = (1u << lane) - 1u;
            uint32_t many = 0;
            for (uint32_t k = 0;; k++) {
                const uint32_t here = __ballot_sync(0xffffffffu, k < waiting);
                if (!here) break;
                const float x = queue_x[32 * k + lane];
                const uint16_t at = queue_at[32 * k + lane];
                __syncwarp();
                if (k < waiting) {
                    const uint32_t to = many + __popc(here & below);
                    queue_x[to] = x;
                    queue_at[to] = at;
                }
                many += __popc(here);
            }
            waiting = 0;
            __syncwarp();
            constexpr uint32_t K = 4;   // a chain of some hundred clocks each: several at once
            for (uint32_t i = lane; i - lane < many; i += 32 * K) {
                unsigned long long w[K];
                uint32_t bin[K];
#pragma unroll
                for (uint32_t e = 0; e < K; e++) {
                    const float x = i + 32 * e < many ? queue_x[i + 32 * e] : -INFINITY;
                    w[e] = weight(x, S.table);
                    bin[e] = w[e] ? bin_of(x) : BS_BINS;
                }
#pragma unroll
                for (uint32_t e = 0; e < K; e++) {
                    sum += w[e];
                    if (by_min && w[e] >= least) { above += w[e]; n_above++; }
                    const bool in = bin[e] < BS_BINS;
                    if (in) add(bin[e], w[e]);
                    const uint32_t stay = __ballot_sync(0xffffffffu, in);
                    all_kept = all_kept && n_places + __popc(stay) <= BS_KEPT;
                    if (!all_kept) continue;
                    if (in) S.kept[warp][n_places + __popc(stay & below)] = queue_at[i + 32 * e];
                    n_places += __popc(stay);
                }
            }
            __syncwarp();
        };
        constexpr uint32_t U = BS_STEP;
        auto some = [&](uint32_t i, const float (&x)[U]) {   // elements i + 32 e of the stretch.  (What is no number is not above -infinity; an infinity is FLT_MAX.)
            if (__any_sync(0xffffffffu, waiting > BS_QUEUE - U)) take();
            float few = 0.f;
#pragma unroll
            for (uint32_t e = 0; e < U; e++) {
                const float d = x[e] - hi;
                const bool any = x[e] > -INFINITY, far = d < -near;
                float w;
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(fmaf(d, c_hi, d * c_lo)));
                n += any;
                if (any && far) few += fmaxf(w, 0x1p-44f);
                if (any && !far) {
                    S.wait_x[warp][waiting][lane] = fminf(x[e], FLT_MAX);
                    S.wait_at[warp][waiting++][lane] = (uint16_t)(i + 32 * e);
                }
            }
            small += few;   // (32 bits for eight only)
        };
        // (without a check for every element; the next ones are requested before these are looked at)
        const float *mine = here + w0 + lane;
        const uint32_t many = w1 - w0, whole = many / (32 * U) * (32 * U);
        float x[U];
        if (whole) {
#pragma unroll
            for (uint32_t e = 0; e < U; e++) x[e] = mine[32 * e];
        }
        for (uint32_t i = 0; i < whole; i += 32 * U) {
            float y[U];
            const bool more = i + 32 * U < whole;
#pragma unroll
            for (uint32_t e = 0; e < U; e++) y[e] = more ? mine[i + 32 * (U + e)] : 0.f;
            some(i + lane, x);
#pragma unroll
            for (uint32_t e = 0; e < U; e++) x[e] = y[e];
        }
        if (whole < many) {
#pragma unroll
            for (uint32_t e = 0; e < U; e++) x[e] = whole + lane + 32 * e < many ? mine[whole + 32 * e] : -INFINITY;
            some(whole + lane, x);
        }
        take();
        unsigned long long loose = (unsigned long long)(small * (double)(1ull << BS_ONE));   // (one of them is a unit at least)
        sum += loose;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            above += __shfl_xor_sync(0xffffffffu, above, o);
            loose += __shfl_xor_sync(0xffffffffu, loose, o);
            n += __shfl_xor_sync(0xffffffffu, n, o);
            n_above += __shfl_xor_sync(0xffffffffu, n_above, o);
        }
        if (lane == 0) {
            L.seg[rank * BS_WARPS + warp] = sum;
            S.loose[warp] = loose;
            S.red[0][warp] = above;
            S.red[1][warp] = (unsigned long long)n << 32 | n_above;
        }
        __syncthreads();
        if (tid == 0) {
            unsigned long long a = 0ull, c = 0ull, l = 0ull;
            for (uint32_t w = 0; w < BS_WARPS; w++) { a += S.red[0][w]; c += S.red[1][w]; l += S.loose[w]; }
            L.part_loose[rank] = l;
            L.part_min[rank] = a;
            L.part_min_cnt[rank] = (uint32_t)c;
            L.part_cnt[rank] = (uint32_t)(c >> 32);
        }
    }

    // ---- the first CTA leads ----
    // Every one of its threads carries the same state; the questions: 0 the k-th element, 1 top_p's, 2 the coin's (3: one whose answer hangs on what
    // the sums are off by).
    unsigned long long kept = 0ull, n_kept = 0ull, bound = 0ull, base = 0ull, n_base = 0ull, n_min = 0ull, S_min = 0ull, there = 0ull, loose = 0ull;   // kept: what is left so far
    uint32_t question = 0, list_lo = 1, list_hi = 0, list_n = 0, shift = 32, prefix = 0;   // the list: bins list_lo .. list_hi
    bool histogram = true, exact = false;   // tot_* are those of the bins of x; the sums are those of whole numbers
    unsigned long long list_mass = 0ull, list_cnt = 0ull;   // ahead of the list
    unsigned long long win_mass = 0ull, win_cnt = 0ull;     // ahead of the window
    auto add_up = [&]() {
        kept = 0ull;
        for (uint32_t s = lane; s < C * BS_WARPS; s += 32) kept += S.seg[s];
#pragma unroll
        for (int o = 16; o; o >>= 1) kept += __shfl_xor_sync(0xffffffffu, kept, o);
        n_kept = p.n;
        question = 0;
    };
    // what `kept` may be off by: while it is the sum of all, and that is not of whole numbers
    auto slack = [&]() { return exact || n_kept != p.n ? 0ull : loose; };
    auto say = [&](uint32_t step, uint32_t a, uint32_t b, uint32_t pre, unsigned long long arg) {
        if (tid == 0) { S.step = step; S.a = a; S.b = b; S.prefix = pre; S.arg = arg; }
    };
    // the next question that this row has; its bound (0: a rank, counted from 0; otherwise a weight)
    auto ask = [&]() {
        for (;; question++) {
            if (question == 0 && by_k) {
                if ((unsigned long long)k >= there || (by_min && !by_p && n_min <= (unsigned long long)k)) continue;   // all that have a weight; min_p leaves no more
                bound = (unsigned long long)k - 1;
                return;
            }
            if (question == 1 && by_p) {
                const unsigned long long off = slack();
                bound = scaled(top_p, kept - off);   // (the least that it can be)
                if (by_min && n_min && bound >= S_min) continue;   // min_p leaves less
                if (by_min && n_min && off && scaled(top_p, kept + off) >= S_min) question = 3;
                return;
            }
            if (question == 2) {
                if (by_min && n_min < n_kept) { n_kept = max(n_min, 1ull); kept = n_min ? S_min : 1ull << BS_ONE; }
                bound = scaled(coin, kept);
                if (slack()) question = 3;
                return;
            }
        }
    };
    // What the answer - the element `key` with running weight and count through it - means; true: the row is done
    auto answered = [&](unsigned long long key, unsigned long long sum, unsigned long long cnt) {
        if (question < 2) {
            kept = sum;
            n_kept = cnt;
        } else {
            if (tid == 0) {
                p.token[row] = (int32_t)(uint32_t)key;
                if (p.prob) p.prob[row] = (float)((double)weight(bs_value(~(uint32_t)(key >> 32)), S.table) / (double)kept);
            }
            return true;
        }
        question++;
        return false;
    };
    auto by_count = [&]() { return question == 0; };
    auto sum_upto = [&](uint32_t b) -> unsigned long long {
        if (by_count()) return b + 1 < BS_BINS ? S.tot_cnt[b + 1] : S.all_cnt;
        return b + 1 < BS_BINS ? S.tot_mass[b + 1] : S.all_mass;
    };
    // the bin of the crossing in tot_* (BS_BINS: none); ahead: weight or count ahead of the histogram
    auto find = [&](unsigned long long ahead) {
        uint32_t lo = 0, hi = BS_BINS;   // the first bin whose sum exceeds the bound
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (bound < ahead + sum_upto(mid)) hi = mid; else lo = mid + 1;
        }
        return lo;
    };
    auto cnt_upto = [&](uint32_t b) { return b + 1 < BS_BINS ? S.tot_cnt[b + 1] : S.all_cnt; };
    // the crossing inside the sorted list, whose sums start behind list_mass, list_cnt
    auto from_list = [&]() {
        uint32_t lo = 0, hi = list_n - 1;
        if (by_count()) lo = (uint32_t)(bound - list_cnt);
        else
            while (lo < hi) {
                const uint32_t mid = (lo + hi) >> 1;
                if (bound < list_mass + S.run[mid]) hi = mid; else lo = mid + 1;
            }
        if (question == 1) {
            const unsigned long long off = slack();
            if (off && scaled(top_p, kept + off) >= list_mass + S.run[lo]) {   // (with the most that the bound can be it is not this element)
                question = 3;
                return false;
            }
        }
        return answered(S.list[lo], list_mass + S.run[lo], list_cnt + lo + 1);
    };
    // Goes on until the cluster is needed; says what for.
    uint32_t last = BS_HISTOGRAM;   // what the cluster has just done
    auto lead = [&]() {
        if (last == BS_DIGIT) {
            const uint32_t bin = find(by_count() ? n_base : base), at = bin < BS_BINS ? bin : 0;   // (there is one: the elements' sums are the same)
            const uint32_t n = cnt_upto(at) - S.tot_cnt[at], to = shift > 10 ? shift - 10 : 0;
            base += S.tot_mass[at];
            n_base += S.tot_cnt[at];
            prefix = (shift == 32 ? 0u : prefix << (shift - to)) | at;
            shift = to;
            if (n <= BS_LIST) {
                list_mass = base;
                list_cnt = n_base;
                say(BS_LIST_DIGITS, shift, 0, prefix, 0);
            } else if (shift == 0) say(BS_COUNT_TIES, 0, 0, prefix, 0);
            else say(BS_DIGIT, shift, shift > 10 ? shift - 10 : 0, prefix, 0);
            return;
        }
        bool done = false;
        if (last == BS_LIST_DIGITS) done = from_list();
        if (last == BS_COUNT_TIES) {
            const unsigned long long w = weight(bs_value(~prefix), S.table), th = by_count() ? bound - n_base : (bound - base) / w;   // number th of the equal ones
            if (question == 2) {
                unsigned long long left = th;
                uint32_t s = 0;
                while (s + 1 < C * BS_WARPS && left >= S.seg[s]) left -= S.seg[s++];
                if (tid == 0 && p.prob) p.prob[row] = (float)((double)w / (double)kept);
                say(BS_PICK_TIE, s, 0, prefix, left);
                return;
            }
            answered(0ull, base + (th + 1) * w, n_base + th + 1);   // (which one it is does not matter to the sums)
        }
        while (!done) {
            if (question < 3) ask();
            if (question == 3) {
                say(BS_EXACT, 0, 0, 0, 0);
                return;
            }
            const unsigned long long ahead = by_count() ? win_cnt : win_mass;
            if (!histogram || bound < ahead) {
                win_mass = win_cnt = 0ull;
                list_lo = 1;
                list_hi = 0;
                say(BS_HISTOGRAM, 0, 0, 0, 0);
                return;
            }
            const uint32_t b = find(ahead);
            if (b == BS_BINS && window + 1 < BS_WINDOWS && (hi - lo) * per_bin >= (float)(BS_BINS * (window + 1))) {   // behind this window
                win_mass += S.all_mass;
                win_cnt += S.all_cnt;
                list_lo = 1;
                list_hi = 0;
                if (octaves < BS_OCTAVES) {
                    win_mass = win_cnt = 0ull;
                    say(BS_HISTOGRAM, 0, 1, 0, 0);
                } else say(BS_HISTOGRAM, window + 1, 0, 0, 0);
                return;
            }
            if (b < BS_BINS) {
                if (b >= list_lo && b <= list_hi) {
                    done = from_list();
                    continue;
                }
                const uint32_t first = cnt_upto(b) <= BS_LIST ? 0 : b;
                if (cnt_upto(b) - S.tot_cnt[first] <= BS_LIST) {
                    list_lo = first;
                    list_hi = b;
                    list_mass = win_mass + S.tot_mass[first];
                    list_cnt = win_cnt + S.tot_cnt[first];
                    say(BS_LIST_BINS, first, b, 0, 0);
                    return;
                }
            }
            if (!exact) { say(BS_EXACT, 0, 0, 0, 0); return; }   // below the histogram, or a bin too full for the list
            // by digits of x's order
            shift = 32;
            prefix = 0;
            base = n_base = 0ull;
            list_lo = 1;
            list_hi = 0;
            say(BS_DIGIT, 32, 22, 0, 0);
            return;
        }
        say(BS_DONE, 0, 0, 0, 0);
    };
    auto sorted = [&]() {   // the first CTA's list has arrived
        list_n = min(S.listed, BS_LIST);
        uint32_t cap = 2;
        while (cap < list_n) cap <<= 1;
        for (uint32_t i = list_n + tid; i < cap; i += BS_THREADS) S.list[i] = ~0ull;
        __syncthreads();
        bs_sort(S.list, cap);
        unsigned long long w0 = 0, w1 = 0, none = 0, all, all_none;
        if (2 * tid < list_n) w0 = weight(bs_value(~(uint32_t)(S.list[2 * tid] >> 32)), S.table);
        if (2 * tid + 1 < list_n) w1 = weight(bs_value(~(uint32_t)(S.list[2 * tid + 1] >> 32)), S.table);
        unsigned long long before = w0 + w1;
        bs_scan(before, none, all, all_none, S);
        static_assert(BS_LIST == 2 * BS_THREADS, "two elements per thread");
        S.run[2 * tid] = before + w0;
        S.run[2 * tid + 1] = before + w0 + w1;
        __syncthreads();
    };

    // (Every part of this stands here once: code that runs once costs 12 clocks an instruction, and a row comes through here a few times only.)
    bool merging = true;
#pragma unroll 1
    for (bool first = true;; first = false) {
        if (merging) merge();
        else if (last == BS_EXACT || last == BS_COUNT_TIES) barrier();   // the stretches' sums are there
        if (rank == 0) {
            if (first || last == BS_EXACT) {
                add_up();
                exact = !first;
            }
            if (first) {
                for (uint32_t r = 0; r < C; r++) {
                    n_min += S.part_min_cnt[r];
                    S_min += S.part_min[r];
                    there += S.part_cnt[r];
                    loose += S.part_loose[r];
                }
                if (loose) loose = (unsigned long long)((double)loose * BS_LOOSE) + BS_LOOSE_EACH * p.n + C * BS_THREADS;   // (a thread makes a whole number of its sum)
            }
            if (last == BS_LIST_BINS || last == BS_LIST_DIGITS) sorted();
            lead();
        }
        barrier();
        const uint32_t step = L.step, a = L.a, b = L.b, pre = L.prefix;
        const unsigned long long arg = L.arg;
        last = step;
        merging = step == BS_HISTOGRAM || step == BS_DIGIT;
        if (step == BS_DONE) break;
        if (merging) {
            // the histogram by stretches of x; or, of the elements whose order's bits from a on are `pre`, by their bits from b to a
            clear();
            histogram = step == BS_HISTOGRAM;
            if (histogram) window = a;
            if (histogram && b) {   // as far as a histogram goes
                per_bin = bins_of(reach_of(BS_OCTAVES));
                octaves = BS_OCTAVES;
                all_kept = false;
            }
            sweep(w1 - w0, [&](uint32_t k) { return w0 + k; }, [&](uint32_t, float x) {
                const uint32_t order = ~bs_order(x);   // (ascending: the largest x first)
                const uint32_t bin = histogram ? bin_of(x) : (order >> b) & ((1u << (a - b)) - 1u);
                if (x > -INFINITY && (histogram ? bin < BS_BINS : a == 32 || order >> a == pre)) add(bin, weight(x, S.table));
            });
        } else if (step == BS_EXACT) {   // the stretches' sums from whole numbers; then all questions again
            exact_sums();
        } else if (step == BS_LIST_BINS || step == BS_LIST_DIGITS) {
            // into this CTA's own list, a place for every warp's elements together; the first CTA fetches them from all
            if (tid == 0) S.listed = 0;
            __syncthreads();
            const float from_bin = (float)(a + BS_BINS * window), to_bin = (float)(b + 1 + BS_BINS * window);
            auto list = [&](uint32_t i, float x) {
                const uint32_t order = ~bs_order(x);
                const float d = (hi - x) * per_bin;   // (bins a to b, without forming the bin)
                if (step == BS_LIST_BINS ? d >= from_bin && d < to_bin : x > -INFINITY && (a == 32 || order >> a == pre)) {
                    const uint32_t at = atomicAdd(&S.listed, 1u);
                    if (at < BS_LIST) S.list[at] = (unsigned long long)order << 32 | (i0 + i);
                }
            };
            const bool by_place = step == BS_LIST_BINS && all_kept && window == 0;
            if (by_place) sweep(n_places, [&](uint32_t k) { return w0 + S.kept[warp][k]; }, list);
            else sweep(w1 - w0, [&](uint32_t k) { return w0 + k; }, list);
            barrier();
            if (rank == 0 && C > 1) {
                // all CTAs' counts at once, then two warps per CTA
                static_assert(BS_WARPS / 2 >= BS_CLUSTER - 1, "two warps for every other CTA");
                const uint32_t n = lane < C ? min(cluster.map_shared_rank(&S, lane)->listed, BS_LIST) : 0u;
                uint32_t upto = n;
#pragma unroll
                for (int o = 1; o < (int)BS_CLUSTER; o <<= 1) {
                    const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
                    if ((int)lane >= o) upto += t;
                }
                const uint32_t r = 1 + warp / 2, many = __shfl_sync(0xffffffffu, n, r), to = __shfl_sync(0xffffffffu, upto, r) - many, all = __shfl_sync(0xffffffffu, upto, C - 1);
                if (r < C) {
                    const BsShared &o = *cluster.map_shared_rank(&S, r);
                    for (uint32_t i = lane + 32 * (warp & 1); i < many && to + i < BS_LIST; i += 64) S.list[to + i] = o.list[i];
                }
                __syncthreads();
                if (tid == 0) S.listed = min(all, BS_LIST);
                __syncthreads();
            }
        } else if (step == BS_COUNT_TIES) {   // more equal elements than the list holds: how many in every stretch
            uint32_t n = 0;
            for (uint32_t i = w0 + lane; i < w1; i += 32) n += ~bs_order(logit(i)) == pre;
            n = __reduce_add_sync(0xffffffffu, n);
            if (lane == 0) L.seg[rank * BS_WARPS + warp] = n;
        } else {   // BS_PICK_TIE: number arg of warp a's stretch
            if (rank == a / BS_WARPS && warp == a % BS_WARPS) {
                uint32_t left = (uint32_t)arg;
                for (uint32_t i = w0 + lane; i - lane < w1; i += 32) {
                    const uint32_t hit = __ballot_sync(0xffffffffu, i < w1 && ~bs_order(logit(i)) == pre);
                    if (left < (uint32_t)__popc(hit)) {
                        if (lane == 0) p.token[row] = (int32_t)(i0 + i + __fns(hit, 0, (int)left + 1));
                        break;
                    }
                    left -= (uint32_t)__popc(hit);
                }
            }
            break;
        }
    }
    if (C > 1) cluster.sync();   // no CTA leaves while another may still read its shared memory
}

}  // namespace ib

using namespace ib;

extern "C" int32_t ib_sample_batch(ib_ctx *ctx, void *stream, const ib_sample_batch_args *args) {
    IB_ENTER(ctx);
    IB_REQUIRE(args, "ib_sample_batch: null argument");
    const ib_sample_batch_args &a = *args;
    IB_REQUIRE(a.vocab >= 1 && a.vocab <= BS_MAX_VOCAB, "ib_sample_batch: %u tokens (1 to %u)", a.vocab, BS_MAX_VOCAB);
    IB_REQUIRE(a.stride >= a.vocab && a.stride < (1ull << 40), "ib_sample_batch: rows overlap (a stride below %u), or a stride above 2^40", a.vocab);
    IB_REQUIRE(a.rows < (1u << 28), "ib_sample_batch: %u rows (below 2^28)", a.rows);
    if (a.rows == 0) return IB_OK;
    IB_REQUIRE(a.logits_dev && a.temperature && a.coin && a.token, "ib_sample_batch: null pointer");
    BatchSampleParams p = {};
    p.logits = a.logits_dev; p.stride = a.stride; p.n = a.vocab;
    p.temperature = a.temperature; p.top_p = a.top_p; p.min_p = a.min_p; p.top_k = a.top_k; p.coin = a.coin;
    p.token = a.token; p.prob = a.prob;
    // CTAs of a row: up to 8, while all rows' have a place at once (two on an SM); a slice has 65536 tokens at most.  (250 rows of 128,256: one CTA each 279 us, two 190, four 195: with one, the
    // rows that take longest are alone at the end.)
    uint32_t ctas = BS_CLUSTER;
    while (ctas > 1 && (a.vocab <= BS_ONE_CTA * ctas / 2 || ((uint64_t)a.rows * ctas > 2 * (uint64_t)ctx->sm_count && a.vocab <= 65536 * ctas / 2))) ctas /= 2;
    p.slice = (a.vocab + ctas - 1) / ctas;
    p.sampled = p.slice > BS_SAMPLED;
    // held in shared memory where that costs no CTA its place
    const size_t without = sizeof(BsShared), with = without + p.slice * sizeof(float);
    p.resident = with <= BS_SMEM_LIMIT && ((uint64_t)a.rows * ctas <= (uint64_t)ctx->sm_count || 2 * (with + 1024) <= BS_SMEM_LIMIT + 1024);
    static bool attr_set[16] = {false};
    const bool beyond = ctx->device >= 16;
    if (beyond || !attr_set[ctx->device]) {
        IB_CHECK_CUDA(cudaFuncSetAttribute(batch_sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)BS_SMEM_LIMIT));
        if (!beyond) attr_set[ctx->device] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(a.rows * ctas);
    cfg.blockDim = dim3(BS_THREADS);
    cfg.dynamicSmemBytes = p.resident ? with : without;
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    IB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, batch_sample_kernel, p));
    ctx->launches++;
    return IB_OK;
}
