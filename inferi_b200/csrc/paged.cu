// A paged cache's bookkeeping on the GPU: block tables, positions and slots of a step from the requests' lengths (ib_page_plan), and the rows that a step
// adds, rotated at their positions and put into their slots (ib_paged_append).  The reference holds one sequence in a contiguous cache.
#include "op_launch.cuh"

#include <cooperative_groups.h>
#include <math.h>

namespace ib {

namespace cg = cooperative_groups;

// ---- ib_page_plan ----
// Four sums over the requests, each taken ahead of a request: of the pages that ended requests return, of the new tokens (who has room among the rows), of the
// pages that those need (who gets pages), and of the tokens of the requests that remain.  Everything written follows from these sums and the inputs, element by
// element, so the launch is one cluster: every CTA forms the sums of all requests for itself in shared memory (a scan is 0.5 us, an exchange between CTAs not
// less), and they share out what is written.  They meet twice: once all lengths have been read, which is what lets kv_len be cached_len, and once the table's new
// entries are written, from which a token's page is read as those of before are.  A page from the stack's old part is read from there, a returned one from
// the ended request's row of the table; no entry that this launch puts on the stack is read.
// Latency bounds it: a chain of some scans, then binary searches in shared memory and reads of the table.
// 16 decoding requests take 4.8 us; 2000 with 40,000 tokens in chunks of prompts, 104,400 rows, 15.4 us: the sums 5, pages 4, tokens 5.
// How many threads (decoding requests, us; 128 threads / 1024 / a cluster of 8): 16: 5.1 / 5.6 / 6.7; 100: 9.4 / 6.2 / 6.8; 250: 17.5 / 7.4 / 6.9; 2000: - / 28 / 12.6.
constexpr uint32_t PLAN_MAX_REQUESTS = 8192, PLAN_THREADS = 1024, PLAN_FEW = 128, PLAN_CLUSTER = 8;

struct PlanRequest { int32_t cached, tokens_end; uint32_t need_before, back_before; };   // sums ahead of it (tokens: including it)

// Sums over the block ahead of each thread, of two values at once; *a_all, *b_all get the totals.  Ends with a barrier.
template <uint32_t THREADS>
__device__ __forceinline__ void plan_scan(unsigned long long &a, unsigned long long &b, unsigned long long *a_all, unsigned long long *b_all, unsigned long long (&red)[2][32]) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned long long a0 = a, b0 = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= (uint32_t)o) { a += x; b += y; }
    }
    if (lane == 31) { red[0][warp] = a; red[1][warp] = b; }
    __syncthreads();
    unsigned long long x = lane < THREADS / 32 ? red[0][lane] : 0ull, y = lane < THREADS / 32 ? red[1][lane] : 0ull;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long u = __shfl_up_sync(0xffffffffu, x, o), w = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= (uint32_t)o) { x += u; y += w; }
    }
    *a_all = __shfl_sync(0xffffffffu, x, 31);
    *b_all = __shfl_sync(0xffffffffu, y, 31);
    const unsigned long long xa = __shfl_sync(0xffffffffu, x, warp ? warp - 1 : 0), yb = __shfl_sync(0xffffffffu, y, warp ? warp - 1 : 0);
    a += (warp ? xa : 0ull) - a0;
    b += (warp ? yb : 0ull) - b0;
    __syncthreads();
}

// THREADS: a few requests are a small CTA's work, whose barriers are cheaper
template <uint32_t THREADS>
__global__ void __launch_bounds__(THREADS) page_plan_kernel(const ib_page_plan_args p, uint32_t page_log2) {
    extern __shared__ __align__(16) PlanRequest R[];   // [n_requests]
    __shared__ unsigned long long red[2][32];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, n = p.n_requests, P = p.page_size, width = p.max_pages;
    pdl_enter();
    const long long n_free = min(max((long long)*p.n_free, 0ll), (long long)p.n_pages);
    auto pages_of = [&](long long positions) { return (positions + P - 1) >> page_log2; };
    struct Lens { long long have, want, need; int32_t status; bool ended, bad; };
    auto lens_of = [&](uint32_t i) {   // of a request, as far as its own lengths go
        Lens l = {0, 0, 0, IB_PLAN_OK, false, false};
        const int32_t cached = R[i].cached, add = R[i].tokens_end;   // (as loaded)
        l.ended = add < 0;
        l.bad = cached < 0 || pages_of(cached) > width;
        if (l.bad) { l.status = IB_PLAN_INVALID; return l; }
        l.have = pages_of(cached);
        if (l.ended || add == 0) return l;
        l.need = pages_of((long long)cached + add) - l.have;
        l.want = add;
        if (l.have + l.need > width) { l.status = IB_PLAN_TABLE_FULL; l.want = l.need = 0; }
        return l;
    };
    // A thread's requests follow one another, so that a scan over the threads is one over all of them.
    const uint32_t each = (n + THREADS - 1) / THREADS, mine = min(tid * each, n), mine_end = min(mine + each, n);
#pragma unroll 2
    for (uint32_t i = mine; i < mine_end; i++) {
        R[i].cached = p.cached_len[i];
        R[i].tokens_end = p.new_len[i];
    }
    // Sums ahead of a request: returned pages; new tokens.  Then, where there is room for the tokens, needed pages; then, if anyone is refused, tokens again, of those that got pages.
    unsigned long long back = 0, want = 0, need = 0, none = 0, returns, wants, needs, all_none;
    for (uint32_t i = mine; i < mine_end; i++) {
        const Lens l = lens_of(i);
        back += l.ended ? l.have : 0;
        want += l.want;
    }
    plan_scan<THREADS>(back, want, &returns, &wants, red);
    const unsigned long long size = min((unsigned long long)n_free + returns, (unsigned long long)p.n_pages), returned = size - n_free;   // (more than n_pages: pages returned twice)
    auto has_room = [&](const Lens &l, unsigned long long &ahead) {   // ahead: the tokens wanted ahead of it
        ahead += l.want;
        return l.want == 0 || ahead <= p.max_tokens;
    };
    unsigned long long ahead = want;
    for (uint32_t i = mine; i < mine_end; i++) {
        const Lens l = lens_of(i);
        if (has_room(l, ahead)) need += l.need;
    }
    plan_scan<THREADS>(need, none, &needs, &all_none, red);
    unsigned long long tokens = 0, taken = 0, got = need;
    bool out = false;
    ahead = want;
    for (uint32_t i = mine; i < mine_end; i++) {
        const Lens l = lens_of(i);
        const bool room = has_room(l, ahead);
        if (room) got += l.need;
        if (room && (l.need == 0 || got <= size)) { tokens += l.want; taken += l.need; }
        else out = true;
    }
    unsigned long long n_all = wants, takens = needs;
    if (__syncthreads_or(out)) plan_scan<THREADS>(tokens, taken, &n_all, &takens, red);
    else tokens = want;
    ahead = want;
    for (uint32_t i = mine; i < mine_end; i++) {
        const Lens l = lens_of(i);
        const bool room = has_room(l, ahead), pages = l.need == 0 || need + l.need <= size;
        PlanRequest r;
        if (room && pages) tokens += l.want;
        r.cached = l.bad || l.ended ? 0 : R[i].cached;
        r.tokens_end = (int32_t)tokens;
        r.need_before = (uint32_t)min(need, size);   // (those that get pages are ahead of all that do not: the sum ahead of one is the sum of what is taken)
        r.back_before = (uint32_t)min(back, 0xFFFFFFFFull);
        if (room) need += l.need;
        back += l.ended ? l.have : 0;
        R[i] = r;
        if (cluster.block_rank() == 0) p.status[i] = !room ? IB_PLAN_NO_ROOM : (!pages ? IB_PLAN_NO_PAGES : l.status);
    }
    const uint32_t n_tokens = (uint32_t)n_all;
    __syncthreads();
    if (cluster.num_blocks() > 1) cluster.sync();   // everyone has read the lengths
    const uint32_t worker = cluster.block_rank() * THREADS + tid, workers = cluster.num_blocks() * THREADS;

    auto owner = [&](uint32_t PlanRequest::*sum, uint32_t x) {   // the last request with its sum ahead <= x (requests without pages share their successor's)
        uint32_t lo = 0, hi = n;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (R[mid].*sum <= x) lo = mid; else hi = mid;
        }
        return lo;
    };
    auto returned_page = [&](uint32_t r) {   // number r of the returned pages
        const uint32_t i = owner(&PlanRequest::back_before, r);
        return p.block_table[(size_t)i * width + (r - R[i].back_before)];
    };
    auto stack = [&](uint32_t at) { return at < (uint32_t)n_free ? p.free_pages[at] : returned_page(at - (uint32_t)n_free); };
    auto tokens_before = [&](uint32_t i) { return i ? (uint32_t)R[i - 1].tokens_end : 0u; };

    // pages taken and lengths
    for (uint32_t i = worker; i < n; i += workers) {
        const uint32_t add = (uint32_t)R[i].tokens_end - tokens_before(i);
        p.kv_len[i] = R[i].cached + (int32_t)add;
        p.row_start[i + 1] = R[i].tokens_end;
    }
    if (worker == 0) p.row_start[0] = 0;
    for (uint32_t g = worker; g < (uint32_t)takens; g += workers) {   // a thread per page: chunks of a prompt need many
        const uint32_t i = owner(&PlanRequest::need_before, g);
        p.block_table[(size_t)i * width + (uint32_t)pages_of(R[i].cached) + (g - R[i].need_before)] = stack((uint32_t)size - 1 - g);
    }
    if (worker == 0) *p.n_free_out = (int32_t)(size - takens);
    for (uint32_t r = worker; r < (uint32_t)returned; r += workers) p.free_pages[n_free + r] = returned_page(r);
    __syncthreads();
    if (cluster.num_blocks() > 1) cluster.sync();   // the table is whole
    // Tokens, four to a thread: one search, and their table entries are requested together
    const bool whole = (((uintptr_t)p.positions | (uintptr_t)p.slots) & 15) == 0;
    for (uint32_t t0 = 4 * worker; t0 < p.max_tokens; t0 += 4 * workers) {
        int32_t pos[4] = {0, 0, 0, 0}, slot[4] = {-1, -1, -1, -1}, page[4];
        if (t0 < n_tokens) {
            uint32_t lo = 0, hi = n - 1;   // the first request whose tokens end behind t0
            while (lo < hi) {
                const uint32_t mid = (lo + hi) >> 1;
                if ((uint32_t)R[mid].tokens_end > t0) hi = mid; else lo = mid + 1;
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                page[e] = -1;
                if (t0 + e >= n_tokens) continue;
                while (lo + 1 < n && (uint32_t)R[lo].tokens_end <= t0 + e) lo++;
                pos[e] = R[lo].cached + (int32_t)(t0 + e - tokens_before(lo));
                page[e] = p.block_table[(size_t)lo * width + ((uint32_t)pos[e] >> page_log2)];
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; e++)
                if (page[e] >= 0 && (uint32_t)page[e] < p.n_pages) slot[e] = (int32_t)(((uint32_t)page[e] << page_log2) + ((uint32_t)pos[e] & (P - 1)));
        }
        if (whole && t0 + 4 <= p.max_tokens) {
            *reinterpret_cast<int4 *>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
            *reinterpret_cast<int4 *>(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        } else
            for (uint32_t e = 0; e < 4 && t0 + e < p.max_tokens; e++) {
                p.positions[t0 + e] = pos[e];
                p.slots[t0 + e] = slot[e];
            }
    }
}

// ---- ib_paged_append ----
// A CTA per row.  It requests all of its data, computes the row's (cos, sin) pairs meanwhile, and rotates: every element is read and written once, and HBM bounds it: 8001 rows of 32 heads of 128
// (360 MB) take 57.5 us, 6.3 TB/s; 64 rows of 64 take 2.6 us, a launch.
// An item is eight elements as two vectors of four: four pairs of the rotation (ORIGINAL: (0, 1), (2, 3) of each; NEOX: element i of the first with i of the second).
constexpr uint32_t APPEND_ITEMS = 3;   // items of a thread that are in flight together
// Threads of a CTA: 256 while the rows' CTAs have a place together, more or less; behind that 128, of which twice as many rows are under way.  (32 heads of 128, 128 or 256: one row 3.8 and 2.9 us, 500
// 9.2 and 5.6, 2000 17.9 and 18.7, 8001 57.5 and 64.)
constexpr uint32_t APPEND_FEW = 256, APPEND_MANY = 128, APPEND_ROWS_PER_SM = 12;
constexpr uint32_t APPEND_MAX_HEAD = 256;

struct AppendParams {
    ib_paged_append_args a;
    void *k, *v;
    uint64_t page_stride;
    uint32_t kv_dim, page_log2, n_slots;
    double turns[APPEND_MAX_HEAD / 2];   // the frequencies in turns (of 2 pi) per position
};

__device__ __forceinline__ void put4(float *p, float4 x) { *reinterpret_cast<float4 *>(p) = x; }
__device__ __forceinline__ void put4(__half *p, float4 x) {
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
__device__ __forceinline__ void put1(float *p, float x) { *p = x; }
__device__ __forceinline__ void put1(__half *p, float x) { *p = __float2half_rn(x); }

// VEC: everything is on 16-byte boundaries and head_size is a multiple of 8; otherwise a pair at a time
template <typename T, bool VEC, uint32_t THREADS>
__global__ void __launch_bounds__(THREADS) paged_append_kernel(const __grid_constant__ AppendParams p) {
    __shared__ float2 cs[APPEND_MAX_HEAD / 2];
    const uint32_t tid = threadIdx.x, row = blockIdx.x, hs = p.a.head_size, half = hs / 2, q_dim = p.a.q_dim, kv_dim = p.kv_dim;
    const bool neox = p.a.variant == IB_ROPE_NEOX;
    pdl_enter();
    const int32_t slot = p.a.slots[row], pos = p.a.positions[row];
    if (slot < 0 || (uint32_t)slot >= p.n_slots) return;
    const uint64_t at = (uint64_t)((uint32_t)slot >> p.page_log2) * p.page_stride + (uint64_t)((uint32_t)slot & ((1u << p.page_log2) - 1)) * kv_dim;
    const float *q = p.a.q_dev + row * p.a.q_stride, *k = p.a.k_dev + row * p.a.k_stride, *v = p.a.v_dev + row * p.a.v_stride;
    float *q_out = p.a.q_out_dev + row * p.a.q_out_stride;
    T *kc = static_cast<T *>(p.k) + at, *vc = static_cast<T *>(p.v) + at;
    auto angles = [&]() {
        for (uint32_t j = tid; j < half; j += THREADS) {
            const double t = (double)pos * p.turns[j];
            float s, c;
            sincospif((float)(2.0 * (t - rint(t))), &s, &c);
            cs[j] = make_float2(c, s);
        }
        __syncthreads();
    };
    auto turn = [&](float x, float y, uint32_t j) {
        const float2 w = cs[j];
        return make_float2(w.x * x - w.y * y, w.y * x + w.x * y);
    };
    if constexpr (VEC) {
        // items of q, then k, then v; an item's two vectors
        const uint32_t n_q = q_dim / 8, n_k = kv_dim / 8, n_items = n_q + 2 * n_k;
        auto places = [&](uint32_t e, bool rotated, uint32_t &x, uint32_t &y, uint32_t &j) {
            if (!rotated || !neox) { x = 8 * e; y = x + 4; j = (x % hs) / 2; return; }
            const uint32_t per = hs / 8, head = e / per;
            j = (e % per) * 4;
            x = head * hs + j;
            y = x + half;
        };
        bool first = true;
        for (uint32_t base = tid; base < n_items || first; base += THREADS * APPEND_ITEMS) {
            float4 f[APPEND_ITEMS][2];
#pragma unroll
            for (uint32_t i = 0; i < APPEND_ITEMS; i++) {
                const uint32_t e = base + i * THREADS;
                if (e >= n_items) continue;
                const float *src = e < n_q ? q : (e < n_q + n_k ? k : v);
                uint32_t x, y, j;
                places(e < n_q ? e : (e < n_q + n_k ? e - n_q : e - n_q - n_k), e < n_q + n_k, x, y, j);
                f[i][0] = __ldcs(reinterpret_cast<const float4 *>(src + x));
                f[i][1] = __ldcs(reinterpret_cast<const float4 *>(src + y));
            }
            if (first) { angles(); first = false; }
#pragma unroll
            for (uint32_t i = 0; i < APPEND_ITEMS; i++) {
                const uint32_t e = base + i * THREADS;
                if (e >= n_items) continue;
                const bool rotated = e < n_q + n_k;
                uint32_t x, y, j;
                places(e < n_q ? e : (rotated ? e - n_q : e - n_q - n_k), rotated, x, y, j);
                float4 a = f[i][0], b = f[i][1];
                if (rotated) {
                    if (neox) {
                        const float2 r0 = turn(a.x, b.x, j), r1 = turn(a.y, b.y, j + 1), r2 = turn(a.z, b.z, j + 2), r3 = turn(a.w, b.w, j + 3);
                        a = make_float4(r0.x, r1.x, r2.x, r3.x);
                        b = make_float4(r0.y, r1.y, r2.y, r3.y);
                    } else {
                        const float2 r0 = turn(a.x, a.y, j), r1 = turn(a.z, a.w, j + 1), r2 = turn(b.x, b.y, j + 2), r3 = turn(b.z, b.w, j + 3);
                        a = make_float4(r0.x, r0.y, r1.x, r1.y);
                        b = make_float4(r2.x, r2.y, r3.x, r3.y);
                    }
                }
                if (e < n_q) { put4(q_out + x, a); put4(q_out + y, b); }
                else {
                    T *to = rotated ? kc : vc;
                    put4(to + x, a);
                    put4(to + y, b);
                }
            }
        }
    } else {
        angles();
        const uint32_t n_q = q_dim / 2, n_k = kv_dim / 2;
        for (uint32_t e = tid; e < n_q + n_k; e += THREADS) {
            const bool of_q = e < n_q;
            const uint32_t i = of_q ? e : e - n_q, j = i % half, x = neox ? (i / half) * hs + j : 2 * i, y = neox ? x + half : x + 1;
            const float *src = of_q ? q : k;
            const float2 r = turn(src[x], src[y], j);
            if (of_q) { q_out[x] = r.x; q_out[y] = r.y; }
            else { put1(kc + x, r.x); put1(kc + y, r.y); }
        }
        for (uint32_t e = tid; e < kv_dim; e += THREADS) put1(vc + e, v[e]);
    }
}

}  // namespace ib

using namespace ib;

namespace ib {
int32_t check_paged_cache(const char *who, const ib_paged_cache *c) {
    IB_REQUIRE(c && c->k_dev && c->v_dev, "%s: null cache", who);
    IB_REQUIRE(c->kv_dtype == IB_KV_F32 || c->kv_dtype == IB_KV_F16, "%s: unknown kv dtype %d", who, c->kv_dtype);
    IB_REQUIRE(c->page_size >= 16 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0, "%s: page_size=%u must be a power of two from 16 to 1024", who, c->page_size);
    IB_REQUIRE(c->n_pages >= 1 && (uint64_t)c->n_pages * c->page_size < (1ull << 31), "%s: %u pages of %u positions (1 to 2^31 - 1 slots)", who, c->n_pages, c->page_size);
    IB_REQUIRE(c->kv_dim >= 1, "%s: kv_dim is 0", who);
    const uint64_t elem = c->kv_dtype == IB_KV_F16 ? 2 : 4;
    IB_REQUIRE(c->page_stride >= (uint64_t)c->page_size * c->kv_dim && c->page_stride < (1ull << 40), "%s: page_stride=%llu below page_size * kv_dim=%llu, or above 2^40", who,
               (unsigned long long)c->page_stride, (unsigned long long)c->page_size * c->kv_dim);
    IB_REQUIRE(c->page_stride * elem % 16 == 0 && c->kv_dim * elem % 16 == 0, "%s: pages and rows of the cache must be multiples of 16 bytes", who);
    IB_REQUIRE((uintptr_t)c->k_dev % 16 == 0 && (uintptr_t)c->v_dev % 16 == 0, "%s: the caches must be 16-byte aligned", who);
    return IB_OK;
}
uint32_t log2_of(uint32_t power) {
    uint32_t l = 0;
    while ((1u << l) < power) l++;
    return l;
}
}  // namespace ib

extern "C" {

int32_t ib_page_plan(ib_ctx *ctx, void *stream, const ib_page_plan_args *args) {
    IB_ENTER(ctx);
    IB_REQUIRE(args, "ib_page_plan: null argument");
    const ib_page_plan_args &a = *args;
    IB_REQUIRE(a.page_size >= 16 && a.page_size <= 1024 && (a.page_size & (a.page_size - 1)) == 0, "ib_page_plan: page_size=%u must be a power of two from 16 to 1024", a.page_size);
    IB_REQUIRE(a.n_pages >= 1 && (uint64_t)a.n_pages * a.page_size < (1ull << 31), "ib_page_plan: %u pages of %u positions (1 to 2^31 - 1 slots)", a.n_pages, a.page_size);
    IB_REQUIRE(a.max_pages >= 1 && (uint64_t)a.max_pages * a.page_size < (1ull << 31), "ib_page_plan: rows of %u pages of %u positions (1 to 2^31 - 1 positions)", a.max_pages, a.page_size);
    IB_REQUIRE(a.n_requests <= PLAN_MAX_REQUESTS, "ib_page_plan: %u requests (up to %u)", a.n_requests, PLAN_MAX_REQUESTS);
    IB_REQUIRE(a.max_tokens >= 1 && a.max_tokens < (1u << 31), "ib_page_plan: room for %u tokens (1 to 2^31 - 1)", a.max_tokens);
    IB_REQUIRE(a.n_free && a.free_pages && a.row_start && a.positions && a.slots && a.n_free_out && (a.n_requests == 0 || (a.cached_len && a.new_len && a.block_table && a.kv_len && a.status)),
               "ib_page_plan: null array");
    static bool attr_set[16] = {false};
    const bool beyond = ctx->device >= 16;
    if (beyond || !attr_set[ctx->device]) {
        IB_CHECK_CUDA(cudaFuncSetAttribute(page_plan_kernel<PLAN_THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(PLAN_MAX_REQUESTS * sizeof(PlanRequest))));
        if (!beyond) attr_set[ctx->device] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    const bool few = a.n_requests <= PLAN_FEW / 4 && a.max_tokens <= 8 * PLAN_FEW;
    const uint32_t ctas = few || (a.n_requests <= PLAN_FEW && a.max_tokens <= 4 * PLAN_THREADS) ? 1 : PLAN_CLUSTER;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(few ? PLAN_FEW : PLAN_THREADS);
    cfg.dynamicSmemBytes = a.n_requests * sizeof(PlanRequest);
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    IB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, few ? page_plan_kernel<PLAN_FEW> : page_plan_kernel<PLAN_THREADS>, a, log2_of(a.page_size)));
    ctx->launches++;
    return IB_OK;
}

int32_t ib_paged_append(ib_ctx *ctx, void *stream, const ib_paged_append_args *args, const ib_paged_cache *cache) {
    IB_ENTER(ctx);
    IB_REQUIRE(args, "ib_paged_append: null argument");
    const ib_paged_append_args &a = *args;
    int32_t rc = check_paged_cache("ib_paged_append", cache);
    if (rc) return rc;
    if (a.n == 0) return IB_OK;
    IB_REQUIRE(a.q_dev && a.k_dev && a.v_dev && a.q_out_dev && a.positions && a.slots, "ib_paged_append: null pointer");
    IB_REQUIRE(a.variant == IB_ROPE_ORIGINAL || a.variant == IB_ROPE_NEOX, "ib_paged_append: unknown variant %d", a.variant);
    IB_REQUIRE(a.head_size >= 2 && a.head_size % 2 == 0 && a.head_size <= APPEND_MAX_HEAD && a.q_dim >= a.head_size && a.q_dim % a.head_size == 0 && cache->kv_dim % a.head_size == 0,
               "ib_paged_append: head_size=%u must be even, <= %u and divide q_dim=%u and kv_dim=%u", a.head_size, APPEND_MAX_HEAD, a.q_dim, cache->kv_dim);
    IB_REQUIRE(a.q_dim <= (1u << 24) && cache->kv_dim <= (1u << 24), "ib_paged_append: rows of %u and %u elements (up to 2^24)", a.q_dim, cache->kv_dim);
    IB_REQUIRE(a.q_stride >= a.q_dim && a.q_out_stride >= a.q_dim && a.k_stride >= cache->kv_dim && a.v_stride >= cache->kv_dim, "ib_paged_append: rows overlap (a stride below the row's length)");
    IB_REQUIRE(a.base_freq > 0.f && isfinite(a.base_freq), "ib_paged_append: base_freq=%g must be positive", (double)a.base_freq);
    IB_REQUIRE(a.n < (1u << 31), "ib_paged_append: %u rows", a.n);
    AppendParams p;
    p.a = a;
    p.k = cache->k_dev; p.v = cache->v_dev;
    p.page_stride = cache->page_stride;
    p.kv_dim = cache->kv_dim;
    p.page_log2 = log2_of(cache->page_size);
    p.n_slots = cache->n_pages * cache->page_size;
    // a model's constants: a thread keeps those of the last model it launched for
    static thread_local double turns[APPEND_MAX_HEAD / 2];
    static thread_local float of_base = 0.f;
    static thread_local uint32_t of_size = 0;
    if (of_size != a.head_size || of_base != a.base_freq) {
        for (uint32_t j = 0; j < a.head_size / 2; j++) turns[j] = pow((double)a.base_freq, -(double)(2 * j) / (double)a.head_size) / 6.283185307179586476925;
        of_size = a.head_size;
        of_base = a.base_freq;
    }
    for (uint32_t j = 0; j < a.head_size / 2; j++) p.turns[j] = turns[j];
    auto whole = [](const void *ptr, uint64_t stride) { return (uintptr_t)ptr % 16 == 0 && stride % 4 == 0; };
    const bool vec = a.head_size % 8 == 0 && whole(a.q_dev, a.q_stride) && whole(a.k_dev, a.k_stride) && whole(a.v_dev, a.v_stride) && whole(a.q_out_dev, a.q_out_stride);
    const bool f16 = cache->kv_dtype == IB_KV_F16, many = vec && a.n > APPEND_ROWS_PER_SM * (uint32_t)ctx->sm_count;
    void (*kernel)(AppendParams) = many  ? (f16 ? paged_append_kernel<__half, true, APPEND_MANY> : paged_append_kernel<float, true, APPEND_MANY>)
                                   : vec ? (f16 ? paged_append_kernel<__half, true, APPEND_FEW> : paged_append_kernel<float, true, APPEND_FEW>)
                                         : (f16 ? paged_append_kernel<__half, false, APPEND_FEW> : paged_append_kernel<float, false, APPEND_FEW>);
    return launch_op(ctx, (cudaStream_t)stream, kernel, a.n, many ? APPEND_MANY : APPEND_FEW, p);
}

}  // extern "C"
