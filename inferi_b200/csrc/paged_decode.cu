// Attention over a paged cache for requests with few rows: single tokens, or some proposed ones.
//
// A query tile is up to 8 rows (tokens x heads of a kv head) on 4 warps; a key tile is 64 positions, 16 of each warp, which lie in one page.  What bounds it is HBM: every
// row of K and V is read once per 8 rows, straight into the registers of the warp that uses it, in 16-byte pieces that follow one another across the lanes; nothing passes through
// shared memory.  The products run on the tensor cores (mma.sync): at 8 rows they are bound by neither instructions nor operands, and a tile through tensor memory would be
// 128 rows of which 120 are empty.
//
// The 16 rows of an MMA's A operand are the 8 rows twice: their f16 values and, below, the remainders (q = hi + lo, about 22 bits), so one MMA makes both products and the sum of
// an accumulator's upper and lower half is the result.  The probabilities are split the same way (times 2^14: the remainders of small ones stay above f16's
// smallest step).  A 32-bit cache: tf32 in the place of f16, and K and V are two operands each (hi, lo).  Every tile's accumulators start from zero and are added to the running
// ones in f32 arithmetic: the tensor core adds with truncation, and a long chain of such additions shrinks.
//
// Which element goes where.  A sum may run in any order, so what an MMA calls columns k of A and B are whatever elements a lane's 16-byte pieces hold, the same for both:
//   K   lane (n, c) = (lane / 4, lane % 4) has elements 32 i + 8 c .. + 7 of position n: of the i-th piece two MMAs' columns {2c, 2c+1, 2c+8, 2c+9}.  q's lanes hold the same elements.
//   V   lane (n, c) has elements 64 i + 8 n .. + 7 of positions 2c, 2c + 1, 2c + 8, 2c + 9: MMA t of a piece makes the result's elements 64 i + 8 n + t, n = 0 .. 7,
//       from pairs of positions that a byte permute puts together.  A lane's results are elements 64 i + 16 c .. + 15 of row n.
// 64 requests over up to 8000 positions, 32 heads of 128, four to a kv head (1.57 GB): 250 us, 6.3 TB/s.  One over 500: 7.2 us, of which a launch is 2.5; the rest is the chain of lengths,
// pages, K, softmax, V, arrival and merge.  24 requests with 5 tokens and 8 heads to a kv head over 3000 positions of a 32-bit cache (224 MB): 134 us: up to five
// tiles of 8 rows read and cut every row again, and a warp's step is a chain (data, K's products, softmax, V's products) that 12 warps on an SM do not hide.
// (32-bit: pieces of 4 elements, MMAs of 8 columns: K elements 16 i + 4 c .. + 3, V elements 32 i + 4 n .. + 3 of positions 2c, 2c + 1; results 32 i + 8 c .. + 7.)
#include "paged_attention.cuh"

namespace ib {

constexpr uint32_t PD_THREADS = 128, PD_WARPS = 4, PD_KT = 64, PD_ROWS = PAGED_DECODE_ROWS;
constexpr float PD_SHIFT = 14.f;   // f16 probabilities are held times 2^14

__device__ __forceinline__ void pd_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pd_mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo: two f16 each of a pair; two tf32
__device__ __forceinline__ void pd_split(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
__device__ __forceinline__ void pd_split_tf32(float x, uint32_t &hi, uint32_t &lo) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));   // (the MMA would drop its lower bits, always towards zero)
}
// The same for what the cache holds, without conversions (16 a clock and SM): the upper bits, as which the MMA takes x itself, and what is left of x, rounded by half a step of what the MMA drops.
// A value that is no finite number is none in hi, whatever lo becomes; but a NaN whose payload is in the lower bits only is an infinity there.  In V its products are no finite numbers all the same, and
// their rows are done again from the cache's own values (paged_repair); of K's see the scores.
__device__ __forceinline__ void pd_cut_tf32(uint32_t x, uint32_t &hi, uint32_t &lo) {
    hi = x & 0xFFFFE000u;
    lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi)) + 0x1000u;
}
__device__ __forceinline__ uint4 pd_load(const void *p) { return __ldcg(reinterpret_cast<const uint4 *>(p)); }
__device__ __forceinline__ uint32_t pd_word(const uint4 &v, int i) { return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)); }

// A call, so that what it takes in registers is not the loop's
template <typename T, uint32_t HS>
static __device__ __noinline__ void pd_repair(const PagedAttn &a, uint32_t request, uint32_t kv_head, uint32_t sink_tiles, uint32_t first, uint32_t units, uint32_t end, int32_t p, float most, uint32_t row,
                                              uint32_t head) {
    paged_repair<T, HS>(a, PD_KT, request, kv_head, {sink_tiles, first, units, end}, p, most, a.q + row * a.q_stride + head * HS, a.out + row * a.out_stride + head * HS);
}

constexpr uint32_t pd_partial_floats(uint32_t hs) { return PD_ROWS * (hs + 2); }
constexpr uint32_t PD_CTAS_PER_SM = 3;   // (32-bit, with two of 237 registers a thread: 140 us instead of 133, see above)

template <typename T, int HS>
__global__ void __launch_bounds__(PD_THREADS, PD_CTAS_PER_SM) paged_decode_kernel(const __grid_constant__ PagedAttn a, const TileShape shape) {
    constexpr bool F16 = sizeof(T) == 2;
    constexpr int NP = F16 ? 16 : 8;               // positions of a warp's step
    constexpr int KP = HS * sizeof(T) / 64;        // a lane's pieces of a position of K (the row's 16-byte pieces over four lanes)
    constexpr int VP = HS * sizeof(T) / 128;       // ... of V (over eight lanes)
    constexpr int VN = 16 / sizeof(T);             // elements of a piece
    constexpr int ACC = HS / 4;                    // results of a lane
    __shared__ PagedRangeShared range_sh;
    __shared__ __align__(16) float sm_acc[PD_WARPS][PD_ROWS][HS];
    __shared__ float sm_m[PD_WARPS][PD_ROWS], sm_l[PD_WARPS][PD_ROWS];
    __shared__ uint32_t sm_last;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = lane >> 2, c = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const PagedRange range = paged_range<PD_KT, PD_THREADS, false>(a, shape, range_sh);
    if (range.total == 0 || blockIdx.x >= range.ranges) return;
    PagedWalk<PD_KT> w;
    w.begin(a, shape, range);
    const uint32_t page_mask = (1u << a.page_log2) - 1;
    do {
        const uint32_t kv_head = w.group / shape.groups, head0 = kv_head * a.kv_mul + (w.group % shape.groups) * shape.heads;
        const uint32_t heads = min(shape.heads, a.kv_mul - (w.group % shape.groups) * shape.heads);   // (the last group may have fewer)
        const uint32_t t0 = w.tile * shape.tokens, tokens = min(shape.tokens, w.q.n - t0);
        // the lane's row: token t0 + n / shape.heads, head n % shape.heads of the group
        const uint32_t tt = n / shape.heads, g = n % shape.heads;
        const bool there = tt < tokens && g < heads;
        const int32_t p_lo = w.q.p0 + (int32_t)t0, p = p_lo + (int32_t)tt, p_hi = p_lo + (int32_t)tokens - 1;
        const float *q = a.q + (uint64_t)(w.q.start + t0 + (there ? tt : 0)) * a.q_stride + (uint64_t)(head0 + (there ? g : 0)) * HS;
        const int32_t *table = a.table + (size_t)w.request * a.max_pages;

        uint32_t qa[F16 ? 2 * KP : 4 * KP][F16 ? 4 : 2];   // A operands: f16 {hi, lo, hi, lo} of two column pairs; tf32 {hi, lo} per column
        float f;
        {
            float x[KP][VN], most = 0.f;
#pragma unroll
            for (int i = 0; i < KP; i++) {
                const float *from = q + i * 4 * VN + c * VN;
                if (a.vec)
#pragma unroll
                    for (int e = 0; e < VN; e += 4) {
                        const float4 v = *reinterpret_cast<const float4 *>(from + e);
                        x[i][e] = v.x; x[i][e + 1] = v.y; x[i][e + 2] = v.z; x[i][e + 3] = v.w;
                    }
                else
#pragma unroll
                    for (int e = 0; e < VN; e++) x[i][e] = from[e];
#pragma unroll
                for (int e = 0; e < VN; e++) most = fmaxf(most, fabsf(x[i][e]));
            }
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int e2 = paged_exponent(most);
            const float down = exp2f((float)-e2);
            f = exp2f((float)e2) * (1.4426950408889634f / sqrtf((float)HS));
#pragma unroll
            for (int i = 0; i < KP; i++) {
                if constexpr (F16) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        pd_split(x[i][4 * h] * down, x[i][4 * h + 1] * down, qa[2 * i + h][0], qa[2 * i + h][1]);
                        pd_split(x[i][4 * h + 2] * down, x[i][4 * h + 3] * down, qa[2 * i + h][2], qa[2 * i + h][3]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) pd_split_tf32(x[i][e] * down, qa[4 * i + e][0], qa[4 * i + e][1]);
                }
            }
        }
        float acc[ACC], m = -INFINITY, l = 0.f;   // m: the largest score in units of log2, rounded up to a whole number: rescaling is exact, here and where partials meet
#pragma unroll
        for (int i = 0; i < ACC; i++) acc[i] = 0.f;

        const uint32_t end = w.span.end, steps = w.count * (16 / NP);
        auto position = [&](uint32_t step) { return key_tile(w.span, w.at + step / (16 / NP)) * PD_KT + warp * 16 + (step % (16 / NP)) * NP; };
        auto page_of = [&](uint32_t step) {
            const uint32_t j = step < steps ? position(step) : end;
            return j < end ? table[j >> a.page_log2] : -1;
        };
        int32_t page = page_of(0);
        for (uint32_t step = 0; step < steps; step++) {
            const uint32_t j0 = position(step);
            const int32_t mine = page;
            page = page_of(step + 1);
            if (mine < 0 || (uint32_t)mine >= a.n_pages) continue;   // no position to see here, or a page outside the cache
            const uint64_t at = (uint64_t)mine * a.page_stride + (uint64_t)(j0 & page_mask) * a.kv_dim + kv_head * HS;
            const T *kp = static_cast<const T *>(a.k) + at + (uint64_t)n * a.kv_dim + c * VN, *vp = static_cast<const T *>(a.v) + at + (uint64_t)(2 * c) * a.kv_dim + n * VN;
            uint4 kr[NP / 8][KP], vr[NP / 4][VP];
#pragma unroll
            for (int i = 0; i < NP / 8; i++)
#pragma unroll
                for (int s = 0; s < KP; s++) kr[i][s] = pd_load(kp + (uint64_t)(8 * i) * a.kv_dim + s * 4 * VN);
#pragma unroll
            for (int i = 0; i < NP / 4; i++)
#pragma unroll
                for (int s = 0; s < VP; s++) vr[i][s] = pd_load(vp + (uint64_t)(8 * (i / 2) + i % 2) * a.kv_dim + s * 8 * VN);

            // scores of the lane's row at positions j0 + 8 i + 2 c, + 1
            float x[NP / 8][2];
#pragma unroll
            for (int i = 0; i < NP / 8; i++) {
                if constexpr (F16) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int s = 0; s < KP; s++) {
                        pd_mma(d, qa[2 * s], kr[i][s].x, kr[i][s].y);
                        pd_mma(d, qa[2 * s + 1], kr[i][s].z, kr[i][s].w);
                    }
                    x[i][0] = d[0] + d[2];
                    x[i][1] = d[1] + d[3];
                } else {
                    // K's remainders have sums of their own, four as its upper parts have: short chains drop less and take less time (one for the remainders: 157 us instead of 140)
                    float d[8][4] = {};
#pragma unroll
                    for (int s = 0; s < KP; s++)
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const uint32_t qq[4] = {qa[4 * s + e][0], qa[4 * s + e][1], qa[4 * s + e + 1][0], qa[4 * s + e + 1][1]};
                            uint32_t h0, l0, h1, l1;
                            pd_cut_tf32(pd_word(kr[i][s], e), h0, l0);
                            pd_cut_tf32(pd_word(kr[i][s], e + 1), h1, l1);
                            pd_mma_tf32(d[s & 3], qq, h0, h1);
                            pd_mma_tf32(d[4 + (s & 3)], qq, l0, l1);
                        }
                    x[i][0] = ((d[0][0] + d[1][0]) + (d[2][0] + d[3][0])) + (((d[0][2] + d[1][2]) + (d[2][2] + d[3][2])) + (((d[4][0] + d[5][0]) + (d[6][0] + d[7][0])) + ((d[4][2] + d[5][2]) + (d[6][2] + d[7][2]))));
                    x[i][1] = ((d[0][1] + d[1][1]) + (d[2][1] + d[3][1])) + (((d[0][3] + d[1][3]) + (d[2][3] + d[3][3])) + (((d[4][1] + d[5][1]) + (d[6][1] + d[7][1])) + ((d[4][3] + d[5][3]) + (d[6][3] + d[7][3]))));
                    // -infinity: perhaps a NaN's, so the row is to be done again.  (Here it is two instructions for 8 positions; in the cut of K's elements, two for each: 150 us instead of 146)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        if (x[i][e] == -INFINITY) x[i][e] = NAN;
                }
            }
            if ((int32_t)j0 + NP - 1 > p_lo || (a.window && p_hi - (int32_t)j0 >= a.window)) {   // not every row sees all of these positions
#pragma unroll
                for (int i = 0; i < NP / 8; i++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        if (!paged_sees(a, p, j0 + 8 * i + 2 * c + e)) x[i][e] = -INFINITY;
                if (j0 + NP > end) {   // what nobody sees may be anything
#pragma unroll
                    for (int i = 0; i < NP / 4; i++)
                        if (j0 + 2 * c + 8 * (i / 2) + i % 2 >= end)
#pragma unroll
                            for (int s = 0; s < VP; s++) vr[i][s] = make_uint4(0u, 0u, 0u, 0u);
                }
            }
            float top = x[0][0];
#pragma unroll
            for (int i = 0; i < NP / 8; i++) top = fmaxf(top, fmaxf(x[i][0], x[i][1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float m1 = fmaxf(m, ceilf(top * f)), from = m1 == -INFINITY ? 0.f : m1, alpha = paged_ex2(m - from), shift = F16 ? PD_SHIFT - from : -from;
            m = m1;
            l *= alpha;
            uint32_t pa[4];
#pragma unroll
            for (int i = 0; i < NP / 8; i++) {
                const float u = paged_ex2(fmaf(x[i][0], f, shift)), v = paged_ex2(fmaf(x[i][1], f, shift));
                l += u + v;
                if constexpr (F16) pd_split(u, v, pa[2 * i], pa[2 * i + 1]);
                else {
                    pd_split_tf32(u, pa[0], pa[1]);
                    pd_split_tf32(v, pa[2], pa[3]);
                }
            }
#pragma unroll
            for (int s = 0; s < VP; s++) {
#pragma unroll
                for (int t = 0; t < VN; t++) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
                    if constexpr (F16) {
                        const uint32_t sel = t & 1 ? 0x7632u : 0x5410u;
                        pd_mma(d, pa, __byte_perm(pd_word(vr[0][s], t / 2), pd_word(vr[1][s], t / 2), sel), __byte_perm(pd_word(vr[2][s], t / 2), pd_word(vr[3][s], t / 2), sel));
                    } else {
                        uint32_t h0, l0, h1, l1;
                        pd_cut_tf32(pd_word(vr[0][s], t), h0, l0);
                        pd_cut_tf32(pd_word(vr[1][s], t), h1, l1);
                        pd_mma_tf32(d, pa, l0, l1);   // (the remainders first: what the second addition drops is all)
                        pd_mma_tf32(d, pa, h0, h1);
                    }
                    acc[2 * VN * s + t] = fmaf(acc[2 * VN * s + t], alpha, d[0] + d[2]);
                    acc[2 * VN * s + VN + t] = fmaf(acc[2 * VN * s + VN + t], alpha, d[1] + d[3]);
                }
            }
        }
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);

        // the warps' parts meet
        if (c == 0) { sm_m[warp][n] = m; sm_l[warp][n] = l; }
#pragma unroll
        for (int s = 0; s < VP; s++)
#pragma unroll
            for (int t = 0; t < 2 * VN; t += 4)
                *reinterpret_cast<float4 *>(&sm_acc[warp][n][s * 8 * VN + c * 2 * VN + t]) = make_float4(acc[2 * VN * s + t], acc[2 * VN * s + t + 1], acc[2 * VN * s + t + 2], acc[2 * VN * s + t + 3]);
        __syncthreads();
        constexpr int D = HS / 16;   // a thread's elements of row tid / 16
        const uint32_t row = tid >> 4, d0 = (tid & 15) * D;
        float mx = -INFINITY, sum = 0.f, y[D];
#pragma unroll
        for (int i = 0; i < D; i++) y[i] = 0.f;
#pragma unroll
        for (uint32_t k = 0; k < PD_WARPS; k++) mx = fmaxf(mx, sm_m[k][row]);
#pragma unroll
        for (uint32_t k = 0; k < PD_WARPS; k++) {
            const float wt = mx == -INFINITY ? 0.f : paged_ex2(sm_m[k][row] - mx);
            sum += wt * sm_l[k][row];
#pragma unroll
            for (int i = 0; i < D; i += 4) {
                const float4 v = *reinterpret_cast<const float4 *>(&sm_acc[k][row][d0 + i]);
                y[i] += wt * v.x; y[i + 1] += wt * v.y; y[i + 2] += wt * v.z; y[i + 3] += wt * v.w;
            }
        }
        bool finish = w.whole();
        if (!finish) {
            const uint32_t c0 = range.range_of(w.tile_unit()), c1 = range.range_of(w.tile_unit() + w.span.units - 1);
            float *part = a.scratch + (size_t)paged_place(range, w.tile_unit(), blockIdx.x) * pd_partial_floats(HS);
#pragma unroll
            for (int i = 0; i < D; i += 4) __stcg(reinterpret_cast<float4 *>(part + 2 * PD_ROWS + row * HS + d0 + i), make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]));
            if ((tid & 15) == 0) __stcg(reinterpret_cast<float2 *>(part) + row, make_float2(mx, sum));
            __syncthreads();
            if (tid == 0) {
                const uint32_t last = paged_arrive(a.counters + c0) == c1 - c0;
                if (last) a.counters[c0] = 0u;   // for the next launch
                sm_last = last;
            }
            __syncthreads();
            finish = sm_last != 0;
            if (finish) {
                // the pieces in their order, some at a time: their loads are in flight together
                constexpr uint32_t AT_ONCE = HS == 128 ? 4 : 8;
                mx = -INFINITY;
                sum = 0.f;
#pragma unroll
                for (int i = 0; i < D; i++) y[i] = 0.f;
                for (uint32_t k0 = c0; k0 <= c1; k0 += AT_ONCE) {
                    float2 ml[AT_ONCE];
                    float4 v[AT_ONCE][D / 4];
                    float top = mx;
#pragma unroll
                    for (uint32_t k = 0; k < AT_ONCE; k++) {
                        const float *from = a.scratch + (size_t)paged_place(range, w.tile_unit(), min(k0 + k, c1)) * pd_partial_floats(HS);
                        ml[k] = __ldcg(reinterpret_cast<const float2 *>(from) + row);
#pragma unroll
                        for (int i = 0; i < D / 4; i++) v[k][i] = __ldcg(reinterpret_cast<const float4 *>(from + 2 * PD_ROWS + row * HS + d0) + i);
                    }
#pragma unroll
                    for (uint32_t k = 0; k < AT_ONCE; k++) top = fmaxf(top, ml[k].x);
                    const float keep = mx == -INFINITY ? 0.f : paged_ex2(mx - top);
                    mx = top;
                    sum *= keep;
#pragma unroll
                    for (int i = 0; i < D; i++) y[i] *= keep;
#pragma unroll
                    for (uint32_t k = 0; k < AT_ONCE; k++) {
                        const float wt = k0 + k > c1 || ml[k].x == -INFINITY ? 0.f : paged_ex2(ml[k].x - mx);
                        sum += wt * ml[k].y;
#pragma unroll
                        for (int i = 0; i < D / 4; i++) {
                            y[4 * i] += wt * v[k][i].x; y[4 * i + 1] += wt * v[k][i].y; y[4 * i + 2] += wt * v[k][i].z; y[4 * i + 3] += wt * v[k][i].w;
                        }
                    }
                }
            }
        }
        if (finish) {
            const uint32_t rt = row / shape.heads, rg = row % shape.heads;
            const bool store = rt < tokens && rg < heads;
            const uint64_t q_row = w.q.start + t0 + rt;
            float *out = a.out + q_row * a.out_stride + (uint64_t)(head0 + rg) * HS;
            const bool sees = p_lo + (int32_t)rt >= 0;   // (a token ahead of the first position sees nothing: 0, whatever the tile's values are)
            const float inv = 1.f / sum;
            bool odd = !(sum > 0.f);
#pragma unroll
            for (int i = 0; i < D; i++) {
                y[i] = sees ? y[i] * inv : 0.f;
                odd |= !isfinite(y[i]);
            }
            odd = odd && sees;
            const float most = sum > 0.f ? mx : -INFINITY;
            if (store) {
                if (a.vec)
#pragma unroll
                    for (int i = 0; i < D; i += 4) *reinterpret_cast<float4 *>(out + d0 + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                else
#pragma unroll
                    for (int i = 0; i < D; i++) out[d0 + i] = y[i];
            }
            const uint32_t rows = __ballot_sync(0xffffffffu, odd && store);   // of the warp's two
#pragma unroll 1
            for (uint32_t h = 0; h < 2; h++)
                if (rows & (0xFFFFu << (16 * h))) {
                    const uint32_t r = 2 * warp + h, ft = r / shape.heads, fg = r % shape.heads;
                    __syncwarp();
                    pd_repair<T, HS>(a, w.request, kv_head, w.span.sink_tiles, w.span.first, w.span.units, w.span.end, p_lo + (int32_t)ft, __shfl_sync(0xffffffffu, most, 16 * h),
                                     w.q.start + t0 + ft, head0 + fg);
                }
        }
        __syncthreads();   // shared memory is used again
    } while (w.next(a, shape));
}

uint32_t paged_decode_ctas(const ib_ctx *ctx) { return (uint32_t)ctx->sm_count * PD_CTAS_PER_SM; }
size_t paged_decode_scratch_floats(const ib_ctx *ctx, uint32_t head_size) { return (size_t)paged_decode_ctas(ctx) * 2 * pd_partial_floats(head_size); }

int32_t launch_paged_decode(ib_ctx *ctx, cudaStream_t s, PagedAttn a, uint32_t head_size, int kv_dtype) {
    TileShape shape;
    shape.heads = a.kv_mul < PD_ROWS ? a.kv_mul : PD_ROWS;
    shape.groups = (a.kv_mul + shape.heads - 1) / shape.heads;
    shape.tokens = PD_ROWS / shape.heads;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(paged_decode_ctas(ctx));
    cfg.blockDim = dim3(PD_THREADS);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    void (*kernel)(PagedAttn, TileShape) = kv_dtype == IB_KV_F16 ? (head_size == 128 ? paged_decode_kernel<__half, 128> : paged_decode_kernel<__half, 64>)
                                                                 : (head_size == 128 ? paged_decode_kernel<float, 128> : paged_decode_kernel<float, 64>);
    IB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, shape));
    ctx->launches++;
    return IB_OK;
}

}  // namespace ib
