// A token for every row of logits, each row with settings of its own: temperature, top-k, top-p, min-p (ib_sample_batch).
//
//   w_i = exp((x_i - max x) / temperature), the rows sorted by (x descending, index ascending), S_m = sum of the first m weights
//   kept: the first min(k, m_min, m_p) of them; m_min = how many w_i >= min_p; m_p = the first m with S_m > top_p * S_k
//   token: the first one with S_m > coin * S_kept.  Rows without a filter: the same over the tokens in index order.
// That is what `Sampler` does where it offers the same (temperature and top-p; crates/inferi/src/models/sampler.rs:32-130).
//
// Which token it is hangs on sums of up to half a million weights next to a border, and on a flat distribution the border is 1e-5 of the sum away.  So weights are whole numbers, in units
// of 2^-44 of the largest, good to 3e-10 of themselves: (x - max) log2(e) / T is one product of doubles, added to 1.5 * 2^20 so that its whole and fractional parts
// are words of the result; 2^fraction is a table of 256 and three steps of a series in 32-bit fixed point.  Sums of whole numbers do not depend on their order.
//
// A row is a thread-block cluster of up to 8 CTAs, each with a slice of the row in shared memory: one read of the row from HBM, and what follows passes over shared memory.
// Nothing is sorted but a list of at most 1024 elements: every border asks for the element at which a running count or sum in sorted order crosses a bound, and a histogram
// (count and weight over 1024 equal stretches of x, those of the largest 11 factors of two) says which bin that is; its elements - or, where they fit, all up to
// there, so that one list answers every question - are listed and sorted.  Bins too full for the list (ties) or below the histogram: the same by digits of x's order, to the last
// tie in index order.  The first CTA of the cluster leads: it looks at the merged histogram and says what all do next (Step).
// What bounds it: a batch of many rows, the 25 instructions a token; few rows, the cluster's barriers.
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
constexpr double BS_OCTAVES = 11.0;           // the histogram's reach below the largest weight, at most
// Vocabularies up to this size are one CTA's work
constexpr uint32_t BS_ONE_CTA = 4096;
constexpr uint32_t BS_SMEM_LIMIT = 227 * 1024;

struct BatchSampleParams {
    const float *logits;
    uint64_t stride;
    uint32_t n, slice, resident;   // tokens of a row, of a CTA; whether a slice is held in shared memory
    const float *temperature, *top_p, *min_p, *coin;
    const int32_t *top_k;
    int32_t *token;
    float *prob;
};

enum BsStep : uint32_t { BS_DONE, BS_HISTOGRAM, BS_DIGIT, BS_LIST_BINS, BS_LIST_DIGITS, BS_SEGMENT, BS_COUNT_TIES, BS_PICK_TIE };

struct BsShared {
    uint32_t table[256];                                // 2^(i / 256), 31 fractional bits
    uint32_t cnt[BS_BINS];                              // this CTA's histogram: elements ...
    uint2 mass[BS_BINS];                                // ... and their weight, as two words
    unsigned long long tot_mass[BS_BINS];               // first CTA: the cluster's histogram, then the sums ahead of each bin
    uint32_t tot_cnt[BS_BINS];
    unsigned long long list[BS_LIST], run[BS_LIST];     // first CTA: listed elements, (~order of x, index); running weight through each
    unsigned long long seg[BS_CLUSTER * BS_WARPS];      // first CTA: weight or count of every warp's stretch of the row
    unsigned long long red[2][BS_WARPS];
    float lo[BS_CLUSTER];                               // of every CTA's slice: its smallest finite logit
    unsigned long long best[BS_CLUSTER];                // ... and its arg-max
    unsigned long long part_mass[BS_CLUSTER], part_min[BS_CLUSTER];   // first CTA: weight of each slice, of its elements with w >= min_p
    uint32_t part_cnt[BS_CLUSTER], part_min_cnt[BS_CLUSTER];
    // what the first CTA says
    uint32_t step, a, b, prefix;
    unsigned long long arg;
    uint32_t listed;
    // first CTA: the whole histogram's sums; scratch of its searches
    unsigned long long all_mass;
    uint32_t all_cnt, at;
};

// the order of x as a number: larger x, larger number
__device__ __forceinline__ uint32_t bs_order(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float bs_value(uint32_t order) { return __uint_as_float(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order); }
// what is no number is never drawn; an infinity is the largest number
__device__ __forceinline__ float bs_clean(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }

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
        return max((((unsigned long long)w << (BS_ONE - 30)) >> down) + 1ull >> 1, 1ull);
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

// Ascending sort of list[0 .. cap), cap a power of two
__device__ __forceinline__ void bs_sort(unsigned long long *list, uint32_t cap) {
    for (uint32_t k = 2; k <= cap; k <<= 1)
        for (uint32_t j = k >> 1; j > 0; j >>= 1) {
            for (uint32_t t = threadIdx.x; t < cap / 2; t += BS_THREADS) {
                const uint32_t a = ((t & ~(j - 1)) << 1) | (t & (j - 1)), b = a | j;
                const unsigned long long x = list[a], y = list[b];
                if ((x > y) == ((a & k) == 0)) { list[a] = y; list[b] = x; }
            }
            __syncthreads();
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
    if (tid < 256) S.table[tid] = (uint32_t)__double2uint_rn(exp2((double)tid * (1.0 / 256)) * 2147483648.0);
    pdl_enter();

    const float T = p.temperature[row];
    const bool greedy = !(T > 0.f);
    const float coin = p.coin[row], top_p = p.top_p ? p.top_p[row] : 1.f, min_p = p.min_p ? p.min_p[row] : 0.f;
    const int32_t k = p.top_k ? p.top_k[row] : 0;
    const bool by_k = k > 0 && (uint32_t)k < p.n, by_p = top_p > 0.f && top_p < 1.f, by_min = min_p > 0.f, filtered = by_k || by_p || by_min;

    // the slice, its largest logit (lowest index on ties) and its smallest finite one
    unsigned long long best = 0ull;
    float lo = INFINITY;
    constexpr uint32_t AT_ONCE = 8;
    for (uint32_t base = tid; base < len; base += AT_ONCE * BS_THREADS) {
        float v[AT_ONCE];
#pragma unroll
        for (uint32_t e = 0; e < AT_ONCE; e++) v[e] = base + e * BS_THREADS < len ? __ldg(from + base + e * BS_THREADS) : 0.f;
#pragma unroll
        for (uint32_t e = 0; e < AT_ONCE; e++) {
            const uint32_t i = base + e * BS_THREADS;
            if (i >= len) continue;
            const float x = bs_clean(v[e]);
            if (p.resident) held[i] = x;
            best = max(best, (unsigned long long)bs_order(x) << 32 | (0xFFFFFFFFu - (i0 + i)));
            if (x > -INFINITY) lo = fminf(lo, x);
        }
    }
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
    auto logit = [&](uint32_t i) { return p.resident ? held[i] : bs_clean(__ldg(from + i)); };
    // a warp's elements: a stretch of the slice
    const uint32_t stretch = ((len + BS_WARPS - 1) / BS_WARPS + 31) & ~31u, w0 = min(len, warp * stretch), w1 = min(len, w0 + stretch);

    // ---- what a step does ----
    // bins of x: equal stretches down from the largest logit
    const float reach = (float)fmin(BS_OCTAVES / weight.c, (double)hi - (double)lo), per_bin = reach > 0.f && isfinite(reach) ? (float)BS_BINS * (1.f - 0x1p-20f) / reach : 0.f;
    auto bin_of = [&](float x) {   // >= BS_BINS: below the histogram
        const float d = (hi - x) * per_bin;
        return d < (float)BS_BINS ? (uint32_t)d : BS_BINS;
    };
    auto add = [&](uint32_t bin, unsigned long long w) {
        atomicAdd(&S.cnt[bin], 1u);
        const uint32_t l = (uint32_t)w, old = atomicAdd(&S.mass[bin].x, l), h = (uint32_t)(w >> 32) + ((uint32_t)(old + l) < old ? 1u : 0u);
        if (h) atomicAdd(&S.mass[bin].y, h);
    };
    // a warp's 32 elements; where all of them fall into one bin (a row of equal logits), one addition
    auto add_warp = [&](uint32_t bin, unsigned long long w, bool in) {
        const uint32_t who = __ballot_sync(0xffffffffu, in);
        if (!who) return;
        const uint32_t one = __shfl_sync(0xffffffffu, bin, __ffs(who) - 1);
        if (__popc(who) > 8 && __all_sync(0xffffffffu, !in || bin == one)) {
            unsigned long long sum = in ? w : 0ull;
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) {
                atomicAdd(&S.cnt[one], (uint32_t)__popc(who));
                const uint32_t l = (uint32_t)sum, old = atomicAdd(&S.mass[one].x, l), h = (uint32_t)(sum >> 32) + ((uint32_t)(old + l) < old ? 1u : 0u);
                if (h) atomicAdd(&S.mass[one].y, h);
            }
        } else if (in) add(bin, w);
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
            for (uint32_t r = 0; r < C; r++) {
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

    // ---- the weights: sums of every stretch and slice, and for filtered rows the histogram ----
    if (filtered) clear();
    const unsigned long long least = by_min ? (min_p > 1.f ? (1ull << BS_ONE) + 1 : (unsigned long long)ceil((double)min_p * (double)(1ull << BS_ONE))) : 0ull;
    {
        unsigned long long sum = 0ull, above = 0ull;
        uint32_t n = 0u, n_above = 0u;
        for (uint32_t i = w0 + lane; i - lane < w1; i += 32) {
            const bool in = i < w1;
            const float x = in ? logit(i) : -INFINITY;
            const unsigned long long w = weight(x, S.table);
            sum += w;
            if (w) n++;
            if (by_min && w >= least) { above += w; n_above++; }
            if (filtered) {
                const uint32_t bin = bin_of(x);
                add_warp(bin, w, w != 0ull && bin < BS_BINS);
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            above += __shfl_xor_sync(0xffffffffu, above, o);
            n += __shfl_xor_sync(0xffffffffu, n, o);
            n_above += __shfl_xor_sync(0xffffffffu, n_above, o);
        }
        if (lane == 0) {
            L.seg[rank * BS_WARPS + warp] = sum;
            S.red[0][warp] = above;
            S.red[1][warp] = (unsigned long long)n << 32 | n_above;
        }
        __syncthreads();
        if (tid == 0) {
            unsigned long long a = 0ull, c = 0ull;
            for (uint32_t w = 0; w < BS_WARPS; w++) { a += S.red[0][w]; c += S.red[1][w]; }
            L.part_min[rank] = a;
            L.part_min_cnt[rank] = (uint32_t)c;
            L.part_cnt[rank] = (uint32_t)(c >> 32);
        }
    }
    if (filtered) merge(); else barrier();

    // ---- the first CTA leads ----
    // Every one of its threads carries the same state; the questions: 0 the k-th element, 1 top_p's, 2 the coin's.
    unsigned long long total = 0ull, kept = 0ull, n_kept = 0ull, S_k = 0ull, bound = 0ull, base = 0ull, n_base = 0ull;
    uint32_t question = 0, list_lo = 1, list_hi = 0, list_n = 0, shift = 32, prefix = 0;   // the list: bins list_lo .. list_hi
    bool histogram = true;   // tot_* are those of the bins of x
    unsigned long long list_mass = 0ull, list_cnt = 0ull;   // ahead of the list
    if (rank == 0) {
        for (uint32_t s = 0; s < C * BS_WARPS; s++) total += S.seg[s];
        kept = S_k = total;
        n_kept = p.n;
    }
    const unsigned long long n_min = rank == 0 && by_min ? [&]() { unsigned long long c = 0; for (uint32_t r = 0; r < C; r++) c += S.part_min_cnt[r]; return c; }() : 0ull;
    const unsigned long long S_min = rank == 0 && by_min ? [&]() { unsigned long long m = 0; for (uint32_t r = 0; r < C; r++) m += S.part_min[r]; return m; }() : 0ull;
    auto scaled = [](float f, unsigned long long m) { return f > 0.f ? min((unsigned long long)((double)f * (double)m), m - 1) : 0ull; };   // f < 1
    auto say = [&](uint32_t step, uint32_t a, uint32_t b, uint32_t pre, unsigned long long arg) {
        if (tid == 0) { S.step = step; S.a = a; S.b = b; S.prefix = pre; S.arg = arg; }
    };
    // the next question that this row has; its bound (0: a rank, counted from 0; otherwise a weight)
    auto ask = [&]() {
        for (;; question++) {
            if (question == 0 && by_k) {
                unsigned long long there = 0;
                for (uint32_t r = 0; r < C; r++) there += S.part_cnt[r];
                if ((unsigned long long)k >= there) continue;   // all that have a weight
                bound = (unsigned long long)k - 1;
                return;
            }
            if (question == 1 && by_p) { bound = scaled(top_p, S_k); return; }
            if (question == 2) {
                if (by_min && n_min < n_kept) { n_kept = max(n_min, 1ull); kept = n_min ? S_min : 1ull << BS_ONE; }
                bound = scaled(coin, kept);
                return;
            }
        }
    };
    // What the answer - the element `key` with running weight and count through it - means; true: the row is done
    auto answered = [&](unsigned long long key, unsigned long long sum, unsigned long long cnt) {
        if (question == 0) { S_k = kept = sum; n_kept = cnt; }
        else if (question == 1) { kept = sum; n_kept = cnt; }
        else {
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
    // the bin of the crossing in tot_* -> S.at (BS_BINS: none); ahead: weight or count ahead of the histogram
    auto find = [&](unsigned long long ahead) {
        if (tid == 0) S.at = BS_BINS;
        __syncthreads();
        for (uint32_t b = tid; b < BS_BINS; b += BS_THREADS) {
            const unsigned long long upto = b + 1 < BS_BINS ? (by_count() ? S.tot_cnt[b + 1] : S.tot_mass[b + 1]) : (by_count() ? S.all_cnt : S.all_mass);
            const unsigned long long before = by_count() ? S.tot_cnt[b] : S.tot_mass[b];
            if (bound >= ahead + before && bound < ahead + upto) S.at = b;
        }
        __syncthreads();
        const uint32_t b = S.at;
        __syncthreads();
        return b;
    };
    auto cnt_upto = [&](uint32_t b) { return b + 1 < BS_BINS ? S.tot_cnt[b + 1] : S.all_cnt; };
    // the crossing inside the sorted list, whose sums start behind list_mass, list_cnt
    auto from_list = [&]() {
        if (tid == 0) S.at = list_n - 1;
        __syncthreads();
        if (by_count()) { if (tid == 0) S.at = (uint32_t)(bound - list_cnt); }
        else
            for (uint32_t i = tid; i < list_n; i += BS_THREADS) {
                const unsigned long long upto = list_mass + S.run[i], before = list_mass + (i ? S.run[i - 1] : 0ull);
                if (bound >= before && bound < upto) S.at = i;
            }
        __syncthreads();
        const uint32_t i = S.at;
        __syncthreads();
        return answered(S.list[i], list_mass + S.run[i], list_cnt + i + 1);
    };
    // Goes on until the cluster is needed; says what for.
    auto lead = [&]() {
        for (;;) {
            ask();
            if (!filtered) {   // index order: the stretch of the crossing
                unsigned long long ahead = 0ull;
                uint32_t s = 0;
                while (s + 1 < C * BS_WARPS && bound >= ahead + S.seg[s]) ahead += S.seg[s++];
                say(BS_SEGMENT, s, 0, 0, bound - ahead);
                return;
            }
            if (!histogram) { say(BS_HISTOGRAM, 0, 0, 0, 0); return; }
            const uint32_t b = find(0ull);
            if (b < BS_BINS) {
                if (b >= list_lo && b <= list_hi) {
                    if (from_list()) { say(BS_DONE, 0, 0, 0, 0); return; }
                    continue;
                }
                const uint32_t first = cnt_upto(b) <= BS_LIST ? 0 : b;
                if (cnt_upto(b) - S.tot_cnt[first] <= BS_LIST) {
                    list_lo = first;
                    list_hi = b;
                    list_mass = S.tot_mass[first];
                    list_cnt = S.tot_cnt[first];
                    if (tid == 0) S.listed = 0;
                    say(BS_LIST_BINS, first, b, 0, 0);
                    return;
                }
            }
            // by digits of x's order
            shift = 32;
            prefix = 0;
            base = n_base = 0ull;
            histogram = false;
            list_lo = 1;
            list_hi = 0;
            say(BS_DIGIT, 32, 22, 0, 0);
            return;
        }
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

    if (rank == 0) lead();
    for (;;) {
        barrier();
        const uint32_t step = L.step, a = L.a, b = L.b, pre = L.prefix;
        const unsigned long long arg = L.arg;
        if (step == BS_DONE) break;
        if (step == BS_HISTOGRAM) {
            clear();
            for (uint32_t i = w0 + lane; i - lane < w1; i += 32) {
                const float x = i < w1 ? logit(i) : -INFINITY;
                const uint32_t bin = bin_of(x);
                add_warp(bin, weight(x, S.table), x > -INFINITY && bin < BS_BINS);
            }
            merge();
            histogram = true;
            if (rank == 0) lead();
        } else if (step == BS_DIGIT) {   // elements whose order's bits from a on are `pre`: by their bits from b to a
            clear();
            for (uint32_t i = w0 + lane; i - lane < w1; i += 32) {
                const float x = i < w1 ? logit(i) : -INFINITY;
                const uint32_t order = ~bs_order(x);   // (ascending: the largest x first)
                add_warp((order >> b) & ((1u << (a - b)) - 1u), weight(x, S.table), x > -INFINITY && (a == 32 || order >> a == pre));
            }
            merge();
            if (rank == 0) {
                const unsigned long long ahead = by_count() ? n_base : base;
                const uint32_t bin = find(ahead);   // (there is one: the elements' sums are the same)
                const uint32_t at = bin < BS_BINS ? bin : 0;
                const uint32_t n = cnt_upto(at) - S.tot_cnt[at];
                base += S.tot_mass[at];
                n_base += S.tot_cnt[at];
                prefix = (shift == 32 ? 0u : prefix << (a - b)) | at;
                shift = b;
                if (n <= BS_LIST) {
                    list_mass = base;
                    list_cnt = n_base;
                    if (tid == 0) S.listed = 0;
                    __syncthreads();
                    say(BS_LIST_DIGITS, shift, 0, prefix, 0);
                } else if (shift == 0) say(BS_COUNT_TIES, 0, 0, prefix, 0);
                else say(BS_DIGIT, shift, shift > 10 ? shift - 10 : 0, prefix, 0);
                __syncthreads();
            }
        } else if (step == BS_LIST_BINS || step == BS_LIST_DIGITS) {
            for (uint32_t i = w0 + lane; i < w1; i += 32) {
                const float x = logit(i);
                const uint32_t order = ~bs_order(x);
                bool in = x > -INFINITY;
                if (step == BS_LIST_BINS) {
                    const uint32_t bin = bin_of(x);
                    in = in && bin >= a && bin <= b;
                } else in = in && (a == 32 || order >> a == pre);
                if (in) {
                    const uint32_t at = atomicAdd(&L.listed, 1u);
                    if (at < BS_LIST) L.list[at] = (unsigned long long)order << 32 | (i0 + i);
                }
            }
            barrier();
            if (rank == 0) {
                sorted();
                if (step == BS_LIST_BINS) lead();   // (finds its bin in the list now)
                else if (from_list()) say(BS_DONE, 0, 0, 0, 0);
                else lead();
                __syncthreads();
            }
        } else if (step == BS_SEGMENT) {   // index order: the element of warp a's stretch at which the running weight exceeds arg
            if (rank == a / BS_WARPS && warp == a % BS_WARPS) {
                unsigned long long left = arg;
                uint32_t last = 0xFFFFFFFFu;
                unsigned long long last_w = 0ull;
                for (uint32_t i = w0 + lane; i - lane < w1; i += 32) {
                    const unsigned long long w = i < w1 ? weight(logit(i), S.table) : 0ull;
                    unsigned long long run = w;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned long long t = __shfl_up_sync(0xffffffffu, run, o);
                        if ((int)lane >= o) run += t;
                    }
                    const uint32_t hit = __ballot_sync(0xffffffffu, left < run);
                    const uint32_t some = __ballot_sync(0xffffffffu, w != 0ull);
                    if (hit || some) {
                        const int l = hit ? __ffs(hit) - 1 : 31 - __clz(some);
                        last = i0 + i - lane + l;
                        last_w = __shfl_sync(0xffffffffu, w, l);
                    }
                    if (hit) break;
                    left -= __shfl_sync(0xffffffffu, run, 31);
                }
                if (lane == 0) {
                    p.token[row] = (int32_t)(last == 0xFFFFFFFFu ? 0u : last);
                    unsigned long long all = 0ull;
                    for (uint32_t s = 0; s < C * BS_WARPS; s++) all += L.seg[s];
                    if (p.prob) p.prob[row] = (float)((double)last_w / (double)all);
                }
            }
            break;
        } else if (step == BS_COUNT_TIES) {   // more equal elements than the list holds: how many in every stretch
            uint32_t n = 0;
            for (uint32_t i = w0 + lane; i < w1; i += 32) n += ~bs_order(logit(i)) == pre;
            n = __reduce_add_sync(0xffffffffu, n);
            if (lane == 0) L.seg[rank * BS_WARPS + warp] = n;
            barrier();
            if (rank == 0) {
                const unsigned long long w = weight(bs_value(~pre), S.table), th = by_count() ? bound - n_base : (bound - base) / w;   // number th of them
                if (question == 2) {
                    unsigned long long left = th;
                    uint32_t s = 0;
                    while (s + 1 < C * BS_WARPS && left >= S.seg[s]) left -= S.seg[s++];
                    if (tid == 0 && p.prob) p.prob[row] = (float)((double)w / (double)kept);
                    say(BS_PICK_TIE, s, 0, pre, left);
                } else {   // (which one it is does not matter to the sums)
                    answered(0ull, base + (th + 1) * w, n_base + th + 1);
                    lead();
                }
                __syncthreads();
            }
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
    const uint32_t ctas = a.vocab <= BS_ONE_CTA ? 1u : BS_CLUSTER;
    p.slice = (a.vocab + ctas - 1) / ctas;
    p.resident = sizeof(BsShared) + p.slice * sizeof(float) <= BS_SMEM_LIMIT;
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
    cfg.dynamicSmemBytes = sizeof(BsShared) + (p.resident ? p.slice * sizeof(float) : 0);
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    IB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, batch_sample_kernel, p));
    ctx->launches++;
    return IB_OK;
}
