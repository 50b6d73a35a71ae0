// Attention of new tokens over a paged cache: what its kernels share - a launch's arguments, how the work is handed out, and the rows that are done again.
//
// Rows and tiles.  The query heads of a kv head see the same positions, so a request's tokens and those heads together are the rows of a product with K: row t * heads + g is
// head g of token t.  A query tile is some tokens of a request with all heads of a group (TileShape); the positions it sees are cut into key tiles of KT.
//
// The units (request, head group, query tile, key tile), in that order, are cut into contiguous, equally long ranges, one per CTA of a grid that fills the GPU once, whatever
// the requests' lengths: the requests of a launch may be one long and many short ones, or equal ones.  (Requests with few new rows and those with many are two launches, one behind the other, each of which
// walks over all of them: paged_attention.cu.)  A query tile whose key tiles fall to several CTAs gets a
// partial (maximum, sum, accumulator) from each; a CTA has at most two such tiles, the one that its range begins in and the one that it ends in, so the scratch has
// two places per CTA whatever the lengths.  The last CTA of a tile to arrive (an atomic counter; nobody waits) adds up the partials in the order of the CTAs: the result does not depend on who
// was last.  Every CTA finds its range by itself from row_start and kv_len, by a sum over the requests: lengths never have to come to the host, and no launch ahead
// has to prepare the work.
#pragma once

#include "common.cuh"

#include <math.h>

namespace ib {

struct PagedAttn {
    const float *q;
    float *out;
    uint64_t q_stride, out_stride;
    const int32_t *table, *row_start, *kv_len;
    const void *k, *v;
    uint64_t page_stride;
    uint32_t n_requests, n_tokens, max_pages, n_pages, page_log2;
    uint32_t kv_heads, kv_mul, kv_dim;
    int32_t window, sinks;         // 0: no window
    uint32_t rows_from, rows_to;   // the launch takes the requests with that many rows (new tokens * kv_mul)
    float merge_cost;              // of a partial, in units' time
    uint32_t vec;                  // q and out are on 16-byte boundaries
    float *scratch;                // two partials per CTA
    uint32_t *counters;            // of arrivals, one per CTA and half of its tiles; zero between launches
    uint32_t *err;
    unsigned long long wait_ns;
};

struct PagedRequest {
    uint32_t start, n;   // first row of q, new tokens
    int32_t p0;          // position of the first one (below 0: lengths that do not fit together; such tokens see nothing)
};
// Lengths come from the caller's arrays: whatever they hold, rows stay inside q and positions inside the row of the table.
__device__ __forceinline__ PagedRequest paged_request(const PagedAttn &a, uint32_t r) {
    PagedRequest q;
    const int32_t s = a.row_start[r], e = a.row_start[r + 1], top = (int32_t)a.n_tokens, kv = a.kv_len[r];
    const int32_t s1 = min(max(s, 0), top), e1 = min(max(e, s1), top);
    q.start = (uint32_t)s1;
    q.n = (uint32_t)(e1 - s1);
    if ((uint64_t)q.n * a.kv_mul < a.rows_from || (uint64_t)q.n * a.kv_mul > a.rows_to) q.n = 0;   // not of this launch
    q.p0 = min(max(kv, 0), (int32_t)(a.max_pages << a.page_log2)) - (int32_t)(e1 - s1);
    return q;
}

// How rows are grouped: `heads` query heads of a kv head at a time (`groups` times per kv head), with `tokens` tokens per query tile
struct TileShape { uint32_t heads, groups, tokens; };

// The key tiles of a query tile: the first `sink_tiles` ones, then those from `first` on; `units` together (one at least: a tile whose tokens see nothing
// still has its rows written)
struct KeySpan { uint32_t sink_tiles, first, units, end; };   // end: positions before it are seen by some row
template <uint32_t KT>
__device__ __forceinline__ KeySpan key_span(const PagedAttn &a, const PagedRequest &q, uint32_t tokens, uint32_t j) {
    const int32_t lo = q.p0 + (int32_t)(j * tokens), hi = q.p0 + (int32_t)min((j + 1) * tokens, q.n);   // positions of the tile's tokens: lo .. hi - 1
    KeySpan s = {0, 0, 1, hi > 0 ? (uint32_t)hi : 0u};
    const uint32_t tiles = (s.end + KT - 1) / KT;
    if (a.window && lo >= a.window) {
        const int32_t from = lo - a.window + 1;
        s.first = (uint32_t)from / KT;
        s.sink_tiles = ((uint32_t)min(a.sinks, from) + KT - 1) / KT;
        if (s.sink_tiles >= s.first) s.first = s.sink_tiles = 0;
    }
    const uint32_t n = s.sink_tiles + tiles - s.first;
    if (n > 1) s.units = n;
    return s;
}
__device__ __forceinline__ uint32_t key_tile(const KeySpan &s, uint32_t unit) { return unit < s.sink_tiles ? unit : s.first + unit - s.sink_tiles; }

// Units of a head group of every lane's own request.  Called by a whole warp: long requests are shared among the lanes.
template <uint32_t KT>
__device__ __forceinline__ unsigned long long request_units(const PagedAttn &a, const PagedRequest &q, uint32_t tokens) {
    const uint32_t lane = threadIdx.x & 31, tiles = (q.n + tokens - 1) / tokens;
    unsigned long long sum = 0;
    if (tiles <= 4)
        for (uint32_t j = 0; j < tiles; j++) sum += key_span<KT>(a, q, tokens, j).units;
    for (uint32_t who = __ballot_sync(0xffffffffu, tiles > 4); who; who &= who - 1) {
        const int l = __ffs(who) - 1;
        PagedRequest b;
        b.start = 0;
        b.n = __shfl_sync(0xffffffffu, q.n, l);
        b.p0 = __shfl_sync(0xffffffffu, q.p0, l);
        const uint32_t t = (b.n + tokens - 1) / tokens;
        unsigned long long part = 0;
        for (uint32_t j = lane; j < t; j += 32) part += key_span<KT>(a, b, tokens, j).units;
#pragma unroll
        for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
        if ((int)lane == l) sum = part;
    }
    return sum;
}

// Quotients whose operands mostly fit 32 bits
__device__ __forceinline__ unsigned long long paged_div(unsigned long long a, unsigned long long b) {
    return ((a | b) >> 32) == 0 ? (unsigned long long)((uint32_t)a / (uint32_t)b) : a / b;
}
// One arrival of a CTA whose threads have met at a barrier, and will again: what they wrote before is there for whoever counts it, and what the others wrote for this one
__device__ __forceinline__ uint32_t paged_arrive(uint32_t *counter) {
    uint32_t before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
    return before;
}

// ---- a CTA's range ----
// Ranges of equal length, the last one shorter.  (Written without divisions where it can be: this is the code that a launch begins with, and code that runs once costs 12 clocks an instruction.)
struct PagedRange {
    unsigned long long total, length, offset;   // units of the launch, of a range; the range's first unit, counted inside its request
    unsigned long long per_group;               // units of a head group of that request, where they are known (0: not)
    uint32_t ranges, request;
    __device__ __forceinline__ unsigned long long first_unit(uint32_t c) const { return min(c * length, total); }
    __device__ __forceinline__ uint32_t range_of(unsigned long long unit) const { return (uint32_t)paged_div(unit, length); }
};
struct PagedRangeShared { unsigned long long sum[32], offset, per_group; uint32_t owner, request; };

// Called by a whole CTA of THREADS threads; ends with a barrier.  MERGE_COST: partials cost something (a.merge_cost).  total == 0: nothing to do in this launch.
template <uint32_t KT, uint32_t THREADS, bool MERGE_COST>
__device__ __forceinline__ PagedRange paged_range(const PagedAttn &a, const TileShape &shape, PagedRangeShared &sh) {
    constexpr uint32_t WARPS = THREADS / 32;
    static_assert(WARPS <= 32, "one sum per warp");
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, head_groups = a.kv_heads * shape.groups;
    // Few requests: a warp each, whose lanes share the request's tiles.  Otherwise every thread has a stretch of them.
    const bool by_warp = a.n_requests <= WARPS;
    const uint32_t per = by_warp ? 1 : (a.n_requests + THREADS - 1) / THREADS;
    auto units_of = [&](uint32_t r) {
        PagedRequest q = {0, 0, 0};
        if (r < a.n_requests) q = paged_request(a, r);
        return request_units<KT>(a, q, shape.tokens) * head_groups;
    };
    unsigned long long mine = 0, group_units = 0;
    uint32_t most = 0;   // units of a tile (by_warp)
    if (by_warp) {
        if (warp < a.n_requests) {
            const PagedRequest q = paged_request(a, warp);
            const uint32_t tiles = (q.n + shape.tokens - 1) / shape.tokens;
            for (uint32_t j = lane; j < tiles; j += 32) {
                const uint32_t units = key_span<KT>(a, q, shape.tokens, j).units;
                group_units += units;
                if constexpr (MERGE_COST) most = max(most, units);
            }
            mine = group_units * head_groups;
        }
    } else
        for (uint32_t b = 0; b < per; b++) mine += units_of(tid * per + b);
    unsigned long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= (uint32_t)o) upto += t;
    }
    if constexpr (MERGE_COST) most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 31) sh.sum[warp] = upto | (unsigned long long)min(most, 0xFFFFu) << 48;   // (2^48 units would take years)
    __syncthreads();
    // every warp: the sums of all warps
    unsigned long long sums = lane < WARPS ? sh.sum[lane] : 0ull;
    if constexpr (MERGE_COST) {
        most = __reduce_max_sync(0xffffffffu, (uint32_t)(sums >> 48));
        sums &= (1ull << 48) - 1;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, sums, o);
        if (lane >= (uint32_t)o) sums += t;
    }
    PagedRange g = {__shfl_sync(0xffffffffu, sums, 31), 1, 0, 0, 0, 0};
    if (g.total == 0) return g;
    g.length = paged_div(g.total + gridDim.x - 1, gridDim.x);
    // A tile of u units in ranges of L is done in the time of L units and of u / L partials, one after the other: L is the root of u times a partial's cost, at least.  (Where there are more
    // requests than warps the tiles are more than the CTAs, mostly, and have one or two each.)
    if (MERGE_COST && by_warp && a.merge_cost > 0.f) {
        const uint32_t least = (uint32_t)sqrtf((float)most * a.merge_cost);
        if (g.length < least) g.length = least;
    }
    g.ranges = (uint32_t)paged_div(g.total + g.length - 1, g.length);
    const unsigned long long first = g.first_unit(blockIdx.x);
    unsigned long long before = __shfl_sync(0xffffffffu, sums, warp ? warp - 1 : 0);
    if (warp == 0) before = 0;
    if (by_warp) {
        const unsigned long long all = __shfl_sync(0xffffffffu, upto, 31);
#pragma unroll
        for (int o = 16; o; o >>= 1) group_units += __shfl_xor_sync(0xffffffffu, group_units, o);
        if (lane == 0 && first >= before && first < before + all) {
            sh.offset = first - before;
            sh.request = warp;
            sh.per_group = group_units;
        }
    } else {
        before += upto - mine;
        if (first >= before && first < before + mine) {
            sh.owner = tid;
            sh.offset = first - before;
            sh.request = tid;
        }
    }
    __syncthreads();
    if (per > 1) {   // which of the owner's requests
        if (warp == 0 && blockIdx.x < g.ranges) {
            const uint32_t base = sh.owner * per;
            unsigned long long left = sh.offset;
            __syncwarp();   // (everyone has read what the finder overwrites)
            for (uint32_t b = 0; b < per; b += 32) {
                const unsigned long long u = units_of(b + lane < per ? base + b + lane : a.n_requests);
                unsigned long long run = u;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long t = __shfl_up_sync(0xffffffffu, run, o);
                    if (lane >= (uint32_t)o) run += t;
                }
                const bool here = left >= run - u && left < run;
                if (here) {
                    sh.request = base + b + lane;
                    sh.offset = left - (run - u);
                }
                if (__any_sync(0xffffffffu, here)) break;
                left -= __shfl_sync(0xffffffffu, run, 31);
            }
        }
        __syncthreads();
    }
    g.request = sh.request;
    g.offset = sh.offset;
    if (by_warp) g.per_group = sh.per_group;
    return g;
}

// ---- a walk over the range, piece by piece; every warp that needs it walks for itself ----
template <uint32_t KT>
struct PagedWalk {
    PagedRequest q;
    KeySpan span;
    unsigned long long unit, end, per_group;   // the current unit and the range's end, counted over the launch; units of the request's head groups
    uint32_t request, group, tile, tiles;      // group: of all kv heads' groups
    uint32_t at, count;                        // the piece: units at .. at + count - 1 of its query tile

    __device__ __forceinline__ void load(const PagedAttn &a, const TileShape &s, uint32_t r) {
        request = r;
        q = paged_request(a, r);
        tiles = (q.n + s.tokens - 1) / s.tokens;
    }
    __device__ __forceinline__ void cut() {
        const unsigned long long left = end - unit;
        count = span.units - at < left ? span.units - at : (uint32_t)left;
    }
    __device__ __forceinline__ void begin(const PagedAttn &a, const TileShape &s, const PagedRange &g) {
        const uint32_t lane = threadIdx.x & 31;
        unit = g.first_unit(blockIdx.x);
        end = g.first_unit(blockIdx.x + 1);
        load(a, s, g.request);
        per_group = g.per_group;
        if (per_group == 0) {
            PagedRequest one = q;
            if (lane) one.n = 0;   // (the others help)
            per_group = __shfl_sync(0xffffffffu, request_units<KT>(a, one, s.tokens), 0);
        }
        group = (uint32_t)paged_div(g.offset, per_group);
        unsigned long long left = g.offset - group * per_group;
        for (uint32_t j = 0;; j += 32) {   // the query tile
            const uint32_t u = j + lane < tiles ? key_span<KT>(a, q, s.tokens, j + lane).units : 0u;
            unsigned long long run = u;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long t = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= (uint32_t)o) run += t;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, left < run);
            if (hit || j + 32 >= tiles) {
                const int l = hit ? __ffs(hit) - 1 : 0;
                tile = j + l;
                at = (uint32_t)(left - __shfl_sync(0xffffffffu, run - u, l));
                break;
            }
            left -= __shfl_sync(0xffffffffu, run, 31);
        }
        span = key_span<KT>(a, q, s.tokens, tile);
        cut();
    }
    // the next piece; false: the range is done
    __device__ __forceinline__ bool next(const PagedAttn &a, const TileShape &s) {
        unit += count;
        if (unit >= end) return false;
        at = 0;
        if (++tile == tiles) {
            tile = 0;
            if (++group == a.kv_heads * s.groups) {
                group = 0;
                const uint32_t lane = threadIdx.x & 31;
                for (uint32_t r = request + 1;; r += 32) {   // the next request of this launch (there is one: the range goes on)
                    const bool some = r + lane < a.n_requests && paged_request(a, r + lane).n > 0;
                    const uint32_t who = __ballot_sync(0xffffffffu, some);
                    if (who || r + 32 >= a.n_requests) {
                        load(a, s, who ? r + __ffs(who) - 1 : a.n_requests - 1);
                        break;
                    }
                }
            }
        }
        span = key_span<KT>(a, q, s.tokens, tile);
        cut();
        return true;
    }
    __device__ __forceinline__ bool whole() const { return count == span.units; }
    // Of a tile that is not whole: where this CTA leaves its partial, and who else has one.  A piece that begins the range goes to the CTA's first place, one that ends it to
    // the second.
    __device__ __forceinline__ unsigned long long tile_unit() const { return unit - at; }
};
// The place of CTA c's partial of the tile that starts at unit `tile_unit`
__device__ __forceinline__ uint32_t paged_place(const PagedRange &g, unsigned long long tile_unit, uint32_t c) { return 2 * c + (g.first_unit(c) < tile_unit ? 1u : 0u); }

__device__ __forceinline__ bool paged_sees(const PagedAttn &a, int32_t p, uint32_t j) {   // (j: a position, below 2^31)
    return (int32_t)j <= p && (a.window == 0 || p - (int32_t)j < a.window || (int32_t)j < a.sinks);
}

__device__ __forceinline__ float paged_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A row's power of two for its f16 halves: q * 2^-e is below 2 in magnitude, whatever q's range (no scaling for rows that hold no numbers)
__device__ __forceinline__ int paged_exponent(float most) {
    const int e = (int)(__float_as_uint(most) >> 23) - 127;   // most >= 0
    return e > 127 || most == 0.f ? 0 : (e < -100 ? -100 : e);
}

// ---- rows that hold something that is not a finite number ----
// A masked position's weight is 0, but 0 times an infinity or NaN in its row of V is not, and the tiles' products run over all of a tile's positions (those that no
// row of the tile sees are zeroed on their way); a weight's remainder may be 0 or negative where the weight is not.  And q's two operands times an infinity in K are infinities of either sign, whose sum is
// NaN where the score is an infinity.  So a row that sees something and has such a result, or no sum of weights, is computed anew, position by position and in one product each: a score of -infinity weighs
// nothing, one that is NaN or infinity makes all of the row NaN, and so do scores that are all -infinity.
// most: the row's largest score (rounded up, in units of log2), -infinity where the sum of weights says that it is not known.  Called by a whole warp.
// 8 positions at a time, of 32 which lie in two pages at most: a lane has HS / 32 columns of each row of K, the sums over the lanes are formed for all 8 together (9 exchanges), which leaves four lanes each
// the score of a position; then the weights are handed round, and a lane adds up its columns of V.  (More at a time takes registers, which the callers' own loops pay for.)
// L2's bandwidth bounds it where all rows of many tiles are done again: 2400 tokens after 40,000, 32 heads of 128: 410 ms, 0.2 s for a tile's 256 rows (a position per lane: 905); one token after 40,000: 14 ms.
// Of more than 400,000 positions a chunk's tile takes longer than the 2 s that the warps of its CTA wait for it by default, and the launch gives up.
template <uint32_t E>
__device__ __forceinline__ void paged_elements(const __half *from, float (&x)[E]) {
    uint32_t w[E / 2];
    if constexpr (E == 4) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(from));
        w[0] = v.x; w[1] = v.y;
    } else w[0] = __ldg(reinterpret_cast<const uint32_t *>(from));
#pragma unroll
    for (uint32_t e = 0; e < E; e += 2) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[e / 2]));
        x[e] = f.x; x[e + 1] = f.y;
    }
}
template <uint32_t E>
__device__ __forceinline__ void paged_elements(const float *from, float (&x)[E]) {
#pragma unroll
    for (uint32_t e = 0; e < E; e += 2) {
        const float2 f = __ldg(reinterpret_cast<const float2 *>(from + e));
        x[e] = f.x; x[e + 1] = f.y;
    }
}
template <typename T, uint32_t HS>
__device__ __forceinline__ void paged_repair(const PagedAttn &a, uint32_t KT, uint32_t request, uint32_t kv_head, const KeySpan span, int32_t p, float most, const float *q, float *out) {
    constexpr uint32_t E = HS / 32;
    const uint32_t lane = threadIdx.x & 31, column = lane * E, kv_dim = a.kv_dim;
    const float scale = 1.4426950408889634f / sqrtf((float)HS);
    const T *k = static_cast<const T *>(a.k) + kv_head * HS + column, *v = static_cast<const T *>(a.v) + kv_head * HS + column;
    const int32_t *table = a.table + (size_t)request * a.max_pages;
    float qr[E];
#pragma unroll
    for (uint32_t e = 0; e < E; e++) qr[e] = q[column + e];
    unsigned long long row0 = 0, row1 = 0;   // of 32 positions: the first and the 17th one's (of pages that are none: the cache's first)
    uint32_t mask = 0;                    // which of them are seen
    auto score = [&](uint32_t g) {        // of position 8 g + lane / 4 of those
        const T *from = k + (g < 2 ? row0 : row1) + (unsigned long long)(g % 2 * 8) * kv_dim;
        float s[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            float x[E];
            paged_elements(from + (unsigned long long)i * kv_dim, x);
            s[i] = qr[0] * x[0];
#pragma unroll
            for (uint32_t e = 1; e < E; e++) s[i] += qr[e] * x[e];
        }
#pragma unroll
        for (uint32_t o = 4; o; o >>= 1)
#pragma unroll
            for (uint32_t i = 0; i < o; i++) {
                const bool upper = lane & (4 * o);
                const float send = upper ? s[i] : s[i + o], keep = upper ? s[i + o] : s[i];
                s[i] = keep + __shfl_xor_sync(0xffffffffu, send, 4 * o);
            }
        s[0] += __shfl_xor_sync(0xffffffffu, s[0], 2);
        s[0] += __shfl_xor_sync(0xffffffffu, s[0], 1);
        return mask >> (8 * g + lane / 4) & 1 ? s[0] : -INFINITY;
    };
    auto positions = [&](auto body) {   // 8 at a time; false: enough
        for (uint32_t u = 0; u < span.units; u++)
            for (uint32_t j0 = key_tile(span, u) * KT; j0 < min(key_tile(span, u) * KT + KT, span.end); j0 += 32) {
                const uint32_t j = j0 + lane;
                const int32_t page = j < span.end ? table[j >> a.page_log2] : -1;
                const bool there = page >= 0 && (uint32_t)page < a.n_pages;
                const unsigned long long at = there ? (unsigned long long)page * a.page_stride + (unsigned long long)(j & ((1u << a.page_log2) - 1)) * kv_dim : 0ull;
                row0 = __shfl_sync(0xffffffffu, at, 0);
                row1 = __shfl_sync(0xffffffffu, at, 16);
                mask = __ballot_sync(0xffffffffu, there && paged_sees(a, p, j));
#pragma unroll 1
                for (uint32_t g = 0; g < 4; g++)
                    if ((mask >> 8 * g & 0xFFu) && !body(g)) return;
            }
    };
    if (most == -INFINITY) {
        float top = -INFINITY;
        bool some = false, none = false;   // sees something; has a score that is none
        positions([&](uint32_t g) {
            const float s = score(g);
            some = true;
            none = __any_sync(0xffffffffu, !(s < INFINITY));
            top = fmaxf(top, s);
            return !none;
        });
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (none || top == -INFINITY) {
#pragma unroll
            for (uint32_t e = 0; e < E; e++) out[column + e] = some ? NAN : 0.f;   // (nothing: pages outside the cache)
            return;
        }
        most = ceilf(top * scale);
    }
    float l = 0.f, acc[E];
#pragma unroll
    for (uint32_t e = 0; e < E; e++) acc[e] = 0.f;
    positions([&](uint32_t g) {
        const float s = score(g);
        const uint32_t seen = mask >> 8 * g;
        const float w = !(seen >> lane / 4 & 1) || s == -INFINITY ? 0.f : fmaxf(paged_ex2(s * scale - most), 1e-38f);   // (not nothing: an infinity that is seen counts, however small its weight)
        const T *from = v + (g < 2 ? row0 : row1) + (unsigned long long)(g % 2 * 8) * kv_dim;
        l += w;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            float x[E];
            paged_elements(from + (unsigned long long)i * kv_dim, x);
            const float wi = __shfl_sync(0xffffffffu, w, 4 * i);
#pragma unroll
            for (uint32_t e = 0; e < E; e++) acc[e] += seen >> i & 1 ? wi * x[e] : 0.f;
        }
        return true;
    });
#pragma unroll
    for (int o = 16; o > 2; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);   // (four lanes have the same)
#pragma unroll
    for (uint32_t e = 0; e < E; e++) out[column + e] = acc[e] / l;
}

// paged_decode.cu
constexpr uint32_t PAGED_DECODE_ROWS = 8;
size_t paged_decode_scratch_floats(const ib_ctx *ctx, uint32_t head_size);
uint32_t paged_decode_ctas(const ib_ctx *ctx);
int32_t launch_paged_decode(ib_ctx *ctx, cudaStream_t s, PagedAttn a, uint32_t head_size, int kv_dtype);


// paged_chunk.cu
uint32_t paged_chunk_ctas(const ib_ctx *ctx);
size_t paged_chunk_scratch_floats(const ib_ctx *ctx, uint32_t head_size);
bool paged_chunk_takes(const PagedAttn &a, int kv_dtype);
int32_t launch_paged_chunk(ib_ctx *ctx, cudaStream_t s, PagedAttn a, uint32_t head_size);

}  // namespace ib
