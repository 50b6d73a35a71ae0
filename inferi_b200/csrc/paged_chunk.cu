// Attention over a paged cache (f16) for requests with many rows: chunks of a prompt, on the 5th-generation tensor cores.
//
// A query tile is 256 rows (tokens x heads of a kv head), two halves of 128 rows; a key tile is 128 positions.  Per half and key tile:
//     S[128 x 128] = Q K^T        Q from shared memory (two operands, hi and lo), K from shared memory; f32 sums in tensor memory
//     P = 2^(S f - m)             a thread per row; P replaces S in tensor memory, as two f16 operands, hi and lo
//     O[128 x HS] = P V           P from tensor memory, V from shared memory, f32 sums in tensor memory
//     acc = 2^(m' - m) acc + O    in registers, HS of them per thread
// q = hi + lo and P = hi + lo hold about 22 bits, K and V are exact, so the result is as good as 32-bit arithmetic makes it; each product is two MMAs.  The sums of a tile go from tensor
// memory to registers before the next one's: the tensor core truncates, and a chain of its additions over a long context would shrink the result.  With whole numbers m rescaling is exact.
//
// What bounds it at head size 128: the MMAs, and what they wait for.  Twice 4 * 128 * 128 * HS operations per half and key tile are 2048 clocks (HS 128); the exponentials are 1024 of the SM's special function units, and the
// remaining work of a thread's 128 scores about 1000.  The halves take turns: while one is in softmax, the tensor cores do the other's products.  Two halves share a key tile's 64 KB, 16
// bytes a clock and SM; a tile of 128 rows would take twice as much from L2, which is all that L2 has.
//
// Who does what (20 warps, one CTA per SM):
//   warps 0-7, 8-15  a half each: two threads per row, each with half of the key tile's scores and of the result's columns.  Load and split q, softmax, fold, result.  (A thread per row
//                    had a chain of 4600 clocks from the scores to the next product, 128 sums in registers and no room for the rest)
//   warps 16, 17     MMA issue, of a half each
//   warp 18          TMA copies of K and V: a ring of tiles, a copy per page and 64 columns, swizzled by 128 bytes
//   warp 19          nothing (registers change hands by groups of four warps)
// They hand over through mbarriers.  Order of the MMAs: S0 S1 | O0 S0' O1 S1' | O0' S0'' ...: a half's softmax has the time of the other's two products.  The tensor cores take no more than
// three or four MMAs ahead, so what the issuing warp does between two products is time that they stand still (700 clocks of every 2600 with one warp for both halves): there are two, which take
// turns, and each waits for its operands while the other one's products run.  From a product with A in shared memory to one with A in tensor memory the tensor cores lose 215 clocks.
// Tensor memory (512 columns): S0 / P0, S1 / P1, O0, O1 of 128 columns each.  P's operands are interleaved by 16 positions, hi then lo, so that a thread overwrites only scores that it has read.
//
// 1000 tokens after 15,000, 32 heads of 128, four to a kv head (254 GFLOP): 451 us, 0.56 PFLOP/s of results and 1.12 of products, two thirds of the measured 1.68; the SM clock is at 1.4 GHz then,
// by the power limit, and the tensor pipe busy for 56 % of the time.  7 chunks of up to 700 with a window of 1024 and 4 sinks, heads of 64: 132 us, 26 %; there the exponentials and the rest of softmax take as
// long as the products, and each CTA has a tile of 10 key tiles, whose start and end count.
//
// Every wait for a copy or a product is bounded; a wait that gives up raises the context's error word, and the kernel returns after freeing its tensor memory.  Barriers are only waited at where all
// who take part come: a half's warps leave as one, the remaining warps meet nobody until the end.
#include "paged_attention.cuh"
#include "tensor_core.cuh"

namespace ib {

constexpr uint32_t PC_THREADS = 640, PC_KT = 128, PC_ROWS = 256, PC_W_MMA = 16, PC_W_TMA = 18;
// Registers: 640 threads at 96 are what the block is launched with; the halves' warps take 104 of them, the others keep 64 (512 * 104 + 128 * 64 = 640 * 96).
constexpr uint32_t PC_REGS_HALF = 104, PC_REGS_OTHER = 64;
constexpr uint32_t PC_S = 0, PC_O = 256;   // tensor memory columns; the halves' are 128 apart
constexpr uint32_t PC_SMEM_LIMIT = 227 * 1024;
constexpr float PC_SHIFT = 14.f;           // probabilities are held times 2^14 (the remainders of small ones stay above f16's smallest step)
constexpr uint32_t pc_half(uint32_t hs) { return 128 * hs * 2; }       // bytes of 128 rows: a half's hi (= lo) operand, a tile of K or V
constexpr uint32_t pc_slots(uint32_t hs) { return hs == 128 ? 3u : 8u; }
constexpr uint32_t PC_MAX_SLOTS = 8;
struct PcShared {   // behind Q and the ring
    uint64_t bars[2 * PC_MAX_SLOTS + 12];
    uint32_t tmem, last[2], odd[2][2][4];
    int32_t lo[2], hi[2];          // positions of the halves' first tokens, and of their query tile's last one
    float x[2][2][128];            // what the two threads of a row tell one another
    PagedWalk<PC_KT> walk[5];      // the walks of the halves, of the MMA warps and of the TMA warp, while registers have other things to hold
    PagedRangeShared range;
};
constexpr uint32_t pc_smem(uint32_t hs) { return (4 + pc_slots(hs)) * pc_half(hs) + (uint32_t)sizeof(PcShared); }
static_assert(pc_smem(128) <= PC_SMEM_LIMIT && pc_smem(64) <= PC_SMEM_LIMIT && pc_slots(64) <= PC_MAX_SLOTS, "shared memory");
constexpr uint32_t pc_partial_floats(uint32_t hs) { return 128 * (hs + 2); }   // of a half

// Descriptors of operands in shared memory: rows of 64 f16 (128 bytes), eight of them 1024 bytes, swizzled by 128 bytes.  K-major: further columns lie behind all rows, so a descriptor covers 64
// columns.  MN-major (V: the product's columns run along the rows): `next` bytes to the following 64 columns, 1024 to the following 8 positions.
__device__ __forceinline__ uint64_t pc_desc_k(uint32_t addr) { return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61; }
__device__ __forceinline__ uint64_t pc_desc_mn(uint32_t addr, uint32_t next) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(next >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// D[128 x N] (+)= A x B, both in shared memory
__device__ __forceinline__ void pc_mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc),
                 "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void pc_tma3d(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, int32_t z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}

// 16 or 32 consecutive tensor-memory columns of the warp's 32 lanes.  The wait names the registers that the load fills: nothing that reads those can be moved ahead of it.
#define PC_REGS32(C, r) \
    C(r[0]), C(r[1]), C(r[2]), C(r[3]), C(r[4]), C(r[5]), C(r[6]), C(r[7]), C(r[8]), C(r[9]), C(r[10]), C(r[11]), C(r[12]), C(r[13]), C(r[14]), C(r[15]), C(r[16]), C(r[17]), C(r[18]), \
        C(r[19]), C(r[20]), C(r[21]), C(r[22]), C(r[23]), C(r[24]), C(r[25]), C(r[26]), C(r[27]), C(r[28]), C(r[29]), C(r[30]), C(r[31])
#define PC_NAMES32 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}"
#define PC_OUT(x) "=r"(x)
#define PC_BOTH(x) "+r"(x)
__device__ __forceinline__ void pc_load(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 " PC_NAMES32 ", [%32];" : PC_REGS32(PC_OUT, r) : "r"(taddr) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" : PC_REGS32(PC_BOTH, r) : : "memory");
}
#undef PC_REGS32
#undef PC_NAMES32
#undef PC_OUT
#undef PC_BOTH
__device__ __forceinline__ void pc_load(uint32_t taddr, uint32_t (&r)[16]) {
    pg_ld16(taddr, r);
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                   "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void pc_sync_half(uint32_t half) {
    if (half) asm volatile("bar.sync 2, 256;" ::: "memory");
    else asm volatile("bar.sync 1, 256;" ::: "memory");
}
// The same barrier; whether all threads of the half hold `ok`
__device__ __forceinline__ bool pc_agree_half(uint32_t half, bool ok) {
    uint32_t all;
    if (half) asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 2, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(all) : "r"((uint32_t)ok) : "memory");
    else asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(all) : "r"((uint32_t)ok) : "memory");
    return all != 0;
}

// Bounded wait without a function call: ptxas does not keep a caller's registers beyond the launch's number across one
__device__ __forceinline__ bool pc_wait(uint32_t bar, uint32_t parity, const PagedAttn &a, uint32_t code) {
    unsigned long long t0 = 0;
    for (uint32_t tries = 1; !pg_try(bar, parity); tries++) {
        if (tries & 1023) continue;   // (the clock takes a microsecond to read)
        const unsigned long long t = pg_ns();
        if (t0 == 0) t0 = t;
        else if (t - t0 > a.wait_ns) {
            *(volatile uint32_t *)a.err = code;
            __threadfence_system();
            return false;
        }
    }
    return true;
}

// A value that all lanes hold, in a uniform register.  MMAs take their operands from those; of what comes from memory the compiler does not know that it is uniform, nor of what hangs on it, and
// moves every operand of every MMA over by itself (70 clocks an MMA instead of 20).
__device__ __forceinline__ uint32_t pc_uniform(uint32_t x) { return __reduce_or_sync(0xffffffffu, x); }

// The CTA's range, as far as places and arrivals go, while registers have other things to hold
__device__ __forceinline__ PagedRange pc_range(const PcShared &S) {
    PagedRange range = {};
    range.total = S.range.sum[0];
    range.length = S.range.sum[1];
    return range;
}
// Rows `who` of a warp's 32 of the kept walk's tile, anew.  (A call that needs nothing of its caller's registers: the loops around it would pay for each.)
template <int HS>
static __device__ __noinline__ void pc_repair(const PagedAttn &a, const TileShape &shape, const PcShared &S, uint32_t half, uint32_t first, uint32_t who, int32_t p, float m) {
    const PagedWalk<PC_KT> &w = S.walk[half];
    for (; who; who &= who - 1) {
        const int b = __ffs(who) - 1;
        const uint32_t at = first + b, token = at / a.kv_mul;
        if (token >= shape.tokens || w.tile * shape.tokens + token >= w.q.n) break;
        const uint64_t q_row = w.q.start + w.tile * shape.tokens + token, from = (uint64_t)(w.group * a.kv_mul + at - token * a.kv_mul) * HS;
        paged_repair<__half, HS>(a, PC_KT, w.request, w.group, w.span, __shfl_sync(0xffffffffu, p, b), __shfl_sync(0xffffffffu, m, b), a.q + q_row * a.q_stride + from, a.out + q_row * a.out_stride + from);
    }
}
// A half that gave up arrives at the tiles that it would still have had a part of, from the one that it was at on (it gives up before it arrives there): the counters are zero again when the launch
// ends, whoever gave up, and launches that follow, replayed ones too, find their last arrivals where they are.  Called by a warp.
static __device__ __noinline__ void pc_arrive_at_rest(const PagedAttn &a, const TileShape &shape, const PcShared &S, uint32_t half) {
    const PagedRange range = pc_range(S);
    PagedWalk<PC_KT> w = S.walk[half];
    do {
        if (w.whole() || (half == 1 && min(shape.tokens, w.q.n - w.tile * shape.tokens) * a.kv_mul <= 128)) continue;
        const uint32_t c0 = range.range_of(w.tile_unit()), c1 = range.range_of(w.tile_unit() + w.span.units - 1);
        if ((threadIdx.x & 31) == 0 && paged_arrive(a.counters + 2 * c0 + half) == c1 - c0) a.counters[2 * c0 + half] = 0u;
    } while (w.next(a, shape));
}

struct PcMaps { CUtensorMap k, v; };

template <int HS>
__global__ void __launch_bounds__(PC_THREADS, 1) paged_chunk_kernel(const __grid_constant__ PagedAttn a, const TileShape shape, const __grid_constant__ PcMaps maps) {
    constexpr uint32_t HALF = pc_half(HS), SLOTS = pc_slots(HS), COLS = HS / 64;   // column blocks of 64
    extern __shared__ __align__(1024) uint8_t smem[];   // (the swizzle's alignment; there is no static shared memory ahead of it)
    PcShared &S = *reinterpret_cast<PcShared *>(smem + (4 + SLOTS) * HALF);
    const uint32_t q0 = pg_smem(smem), ring = q0 + 4 * HALF, bars = pg_smem(S.bars);   // Q: [half][hi, lo]
    const uint32_t b_full = bars, b_empty = b_full + 8 * SLOTS, b_q = b_empty + 8 * SLOTS, b_s = b_q + 16, b_p = b_s + 16, b_o = b_p + 16, b_free = b_o + 16, b_turn = b_free + 16;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const PagedRange range = paged_range<PC_KT, PC_THREADS, true>(a, shape, S.range);
    if (range.total == 0 || blockIdx.x >= range.ranges) return;
    if (warp == 0 && lane == 0) {
        S.range.sum[0] = range.total;   // (free from here on: pc_range)
        S.range.sum[1] = range.length;
        for (uint32_t i = 0; i < SLOTS; i++) {
            pg_bar_init(b_full + 8 * i, 1);
            pg_bar_init(b_empty + 8 * i, 2);   // both MMA warps
        }
        for (uint32_t h = 0; h < 2; h++) {
            pg_bar_init(b_q + 8 * h, 8);      // a half's warps
            pg_bar_init(b_s + 8 * h, 1);      // the MMAs' completion
            pg_bar_init(b_p + 8 * h, 8);
            pg_bar_init(b_o + 8 * h, 1);
            pg_bar_init(b_free + 8 * h, 8);
            pg_bar_init(b_turn + 8 * h, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == PC_W_MMA) pg_alloc<false>(pg_smem(&S.tmem));
    pg_fence_before();
    __syncthreads();
    pg_fence_after();
    const uint32_t tmem = pc_uniform(*const_cast<volatile uint32_t *>(&S.tmem));
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity, uint32_t code) {
        ok = __all_sync(0xffffffffu, pc_wait(bar, parity, a, code));
        return ok;
    };
    PagedWalk<PC_KT> w;
    w.begin(a, shape, range);
    PagedWalk<PC_KT> &kept = S.walk[warp < PC_W_MMA ? warp >> 3 : 2 + (warp - PC_W_MMA) % 3];
    auto park = [&]() {
        __syncwarp();
        if (lane == 0) kept = w;
        __syncwarp();
    };
    auto unpark = [&]() { w = *const_cast<const PagedWalk<PC_KT> *>(&kept); };
    // row r of a tile is token r / kv_mul of it (r < 256, kv_mul <= 64: exact)
    const uint32_t inverse = (65535 + a.kv_mul) / a.kv_mul;
    auto token_of = [&](uint32_t r) { return r * inverse >> 16; };
    auto rows_of = [&]() { return min(shape.tokens, w.q.n - w.tile * shape.tokens) * a.kv_mul; };

    if (warp < PC_W_MMA) {
        // ===== a half: two threads per row =====
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PC_REGS_HALF));
        constexpr uint32_t D = HS / 2;   // a thread's columns of the result
        const uint32_t half = warp >> 3, side = (warp >> 2) & 1, row = tid & 127, tl = tmem + ((warp & 3) << 21);   // the warp's 32 lanes of tensor memory
        const uint32_t t_s = tl + PC_S + 128 * half + 64 * side, t_o = tl + PC_O + 128 * half + D * side;
        const uint32_t bs = b_s + 8 * half, bp = b_p + 8 * half, bo = b_o + 8 * half, bf = b_free + 8 * half;
        // The value of the row's other thread.  (Between an exchange and the next one there is a barrier that every warp of the half arrives at only when it is through with this one: of the
        // scores, of the products, or the half's own.)
        auto other = [&](float x) {
            S.x[half][side][row] = x;
            pc_sync_half(half);
            return S.x[half][side ^ 1][row];
        };
        uint32_t ps = 0;   // parity of the scores; that of the products before them is the other one
        do {
            if (half == 1 && rows_of() <= 128) continue;
            const int32_t p = w.q.p0 + (int32_t)(w.tile * shape.tokens + token_of(128 * half + row));
            if (side == 0 && (warp & 3) == 0) {   // (read behind the exchanges)
                park();
                if (lane == 0) {
                    S.lo[half] = w.q.p0 + (int32_t)(w.tile * shape.tokens + token_of(128 * half));
                    S.hi[half] = w.q.p0 + (int32_t)min((w.tile + 1) * shape.tokens, w.q.n) - 1;
                }
            }
            // q: a warp takes rows as they lie in memory (a thread with a row of its own would touch 32 lines with every load), 16 of the half's
            constexpr uint32_t LANES = HS / 4, AT_ONCE = 32 / LANES, LOADS = 8;   // lanes of a row, rows of a load, loads in flight
            const uint32_t column = 4 * (lane % LANES);
#pragma unroll 1
            for (uint32_t i = 0; i < 16; i += LOADS * AT_ONCE) {
                float4 v[LOADS];
#pragma unroll
                for (uint32_t k = 0; k < LOADS; k++) {
                    const uint32_t rr = 16 * (warp & 7) + i + k * AT_ONCE + lane / LANES, at = 128 * half + rr, token = token_of(at);
                    v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (token < shape.tokens && w.tile * shape.tokens + token < w.q.n) {
                        const float *q = a.q + (uint64_t)(w.q.start + w.tile * shape.tokens + token) * a.q_stride + (uint64_t)(w.group * a.kv_mul + at - token * a.kv_mul) * HS + column;
                        if (a.vec) v[k] = *reinterpret_cast<const float4 *>(q);
                        else v[k] = make_float4(q[0], q[1], q[2], q[3]);
                    }
                }
#pragma unroll
                for (uint32_t k = 0; k < LOADS; k++) {
                    const uint32_t rr = 16 * (warp & 7) + i + k * AT_ONCE + lane / LANES;
                    float most = fmaxf(fmaxf(fabsf(v[k].x), fabsf(v[k].y)), fmaxf(fabsf(v[k].z), fabsf(v[k].w)));
#pragma unroll
                    for (uint32_t o = LANES / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                    const int e2 = paged_exponent(most);
                    const float down = exp2f((float)-e2);
                    if (column == 0) S.x[half][0][rr] = exp2f((float)e2) * (1.4426950408889634f / sqrtf((float)HS));
                    const float x[4] = {v[k].x * down, v[k].y * down, v[k].z * down, v[k].w * down};
                    uint32_t hi[2], lo[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const __half2 h = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
                        const float2 g = __half22float2(h);
                        const __half2 l = __floats2half2_rn(x[2 * e] - g.x, x[2 * e + 1] - g.y);
                        hi[e] = *reinterpret_cast<const uint32_t *>(&h);
                        lo[e] = *reinterpret_cast<const uint32_t *>(&l);
                    }
                    // 16-byte piece c of a row lies at piece c ^ (row % 8)
                    const uint32_t to = q0 + half * 2 * HALF + (column / 64) * 16384 + rr * 128 + (((column % 64 / 8) ^ (rr & 7)) << 4) + 2 * (column % 8);
                    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(hi[0]), "r"(hi[1]) : "memory");
                    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to + HALF), "r"(lo[0]), "r"(lo[1]) : "memory");
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            pc_sync_half(half);
            float acc[D];
            const float f = S.x[half][0][row];   // a score's unit, in those of log2
            __syncwarp();
            if (lane == 0) pg_arrive(b_q + 8 * half);
#pragma unroll
            for (int i = 0; i < (int)D; i++) acc[i] = 0.f;
            float m = -INFINITY, l = 0.f, alpha = 1.f;
            const volatile PagedWalk<PC_KT> &now = kept;   // (registers are short: what is read once per key tile is read from there)
            auto fold = [&]() {   // acc = alpha acc + O
                if (!ok || !wait(bo, ps ^ 1, 12)) return;
                pg_fence_after();
#pragma unroll
                for (int c = 0; c < (int)D / 32; c++) {
                    uint32_t o[32];
                    pc_load(t_o + 32 * c, o);
#pragma unroll
                    for (int e = 0; e < 32; e++) acc[32 * c + e] = fmaf(acc[32 * c + e], alpha, __uint_as_float(o[e]));
                }
                pg_fence_before();
                __syncwarp();
                if (lane == 0) pg_arrive(bf);
            };
            // Each warp sees for itself that a wait gave up, and one that left by itself would keep the others at the half's next barrier for ever.  So it goes on without waiting, with whatever tensor
            // memory holds, and the half leaves as one behind its last key tile.
            for (uint32_t i = 0; i < now.count; i++) {
                if (i) fold();   // of the tile before: its products are done before this one's scores
                const uint32_t unit = now.at + i, sink_tiles = now.span.sink_tiles;
                const int32_t base = (int32_t)((unit < sink_tiles ? unit : now.span.first + unit - sink_tiles) * PC_KT + 64 * side);
                const bool masked = base + 63 > *const_cast<volatile int32_t *>(&S.lo[half]) || (a.window && *const_cast<volatile int32_t *>(&S.hi[half]) - base >= a.window);
                if (ok) wait(bs, ps, 12);
                ps ^= 1;
                pg_fence_after();
                uint64_t seen = ~0ull;   // which of its 64 columns the row sees: up to its own position, and of those the window's and the sinks
                if (masked) {
                    const int32_t last = p - base;
                    if (a.window) {
                        const int32_t from = last - a.window + 1, sinks = a.sinks - base;
                        seen = (from <= 0 ? ~0ull : (from > 63 ? 0ull : ~0ull << from)) | (sinks <= 0 ? 0ull : (sinks > 63 ? ~0ull : ~(~0ull << sinks)));
                    }
                    seen &= last < 0 ? 0ull : (last > 62 ? ~0ull : ~(~0ull << (last + 1)));
                }
                auto sees = [&](int c) { return ((c < 32 ? (uint32_t)seen : (uint32_t)(seen >> 32)) & (1u << (c & 31))) != 0; };
                // A load from tensor memory takes 200 clocks and more whatever its size (while products run), so it is of as many columns as there are registers for; those that are looked at
                // last for the maximum are the first to become weights.
                constexpr int ST = HS == 128 ? 16 : 32, NC = 64 / ST;   // (HS 128, in pieces of 32: 474 us instead of 464; HS 64, of 16: 165 instead of 155)
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, sums[2];
                uint32_t s[ST];
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    pc_load(t_s + ST * c, s);
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < ST; e++) {
                            if (!sees(ST * c + e)) s[e] = 0xFF800000u;
                            tops[e & 3] = fmaxf(tops[e & 3], __uint_as_float(s[e]));
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < ST; e++) tops[e & 3] = fmaxf(tops[e & 3], __uint_as_float(s[e]));
                    }
                }
                const float own = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), top = fmaxf(own, other(own));
                const float m1 = fmaxf(m, ceilf(top * f)), bottom = m1 == -INFINITY ? 0.f : m1, alpha1 = paged_ex2(m - bottom), shift = PC_SHIFT - bottom;
                m = m1;
                sums[0] = sums[1] = 0.f;
#pragma unroll
                for (int c = NC - 1; c >= 0; c--) {
                    if (c < NC - 1) {
                        pc_load(t_s + ST * c, s);
                        if (masked) {
#pragma unroll
                            for (int e = 0; e < ST; e++)
                                if (!sees(ST * c + e)) s[e] = 0xFF800000u;
                        }
                    }
#pragma unroll
                    for (int b = 0; b < ST; b += 16) {   // by 16 positions: their upper parts, then their remainders
                        uint32_t o[16];
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float x = paged_ex2(fmaf(__uint_as_float(s[b + e]), f, shift)), y = paged_ex2(fmaf(__uint_as_float(s[b + e + 1]), f, shift));
                            sums[0] += x;
                            sums[1] += y;
                            const __half2 h = __floats2half2_rn(x, y);
                            const float2 g = __half22float2(h);
                            const __half2 d = __floats2half2_rn(x - g.x, y - g.y);
                            o[e / 2] = *reinterpret_cast<const uint32_t *>(&h);
                            o[8 + e / 2] = *reinterpret_cast<const uint32_t *>(&d);
                        }
                        pg_st16(t_s + ST * c + b, o);
                    }
                }
                l = fmaf(l, alpha1, sums[0] + sums[1]);
                pg_wait_st();
                pg_fence_before();
                __syncwarp();
                if (lane == 0) pg_arrive(bp);
                alpha = alpha1;
            }
            fold();
            S.x[half][side][row] = l;
            ok = pc_agree_half(half, ok);   // (also: the kept walk is there)
            if (!ok) break;
            l += S.x[half][side ^ 1][row];
            unpark();

            // ---- the half's result, or its part of it ----
            bool finish = w.whole();
            if (!finish) {
                const PagedRange range = pc_range(S);
                const uint32_t c0 = range.range_of(w.tile_unit()), c1 = range.range_of(w.tile_unit() + w.span.units - 1);
                float *part = a.scratch + ((size_t)paged_place(range, w.tile_unit(), blockIdx.x) * 2 + half) * pc_partial_floats(HS);
#pragma unroll
                for (int i = 0; i < (int)D; i++) __stcg(part + 128 * (D * side + i) + row, acc[i]);
                if (side == 0) {
                    __stcg(part + 128 * HS + row, m);
                    __stcg(part + 128 * (HS + 1) + row, l);
                }
                pc_sync_half(half);
                if (row == 0 && side == 0) {
                    const uint32_t is_last = paged_arrive(a.counters + 2 * c0 + half) == c1 - c0;
                    if (is_last) a.counters[2 * c0 + half] = 0u;   // for the next launch
                    S.last[half] = is_last;
                }
                pc_sync_half(half);
                finish = S.last[half] != 0;
                if (finish) {
                    m = -INFINITY;
                    l = 0.f;
#pragma unroll
                    for (int i = 0; i < (int)D; i++) acc[i] = 0.f;
                    for (uint32_t k = c0; k <= c1; k++) m = fmaxf(m, __ldcg(a.scratch + ((size_t)paged_place(range, w.tile_unit(), k) * 2 + half) * pc_partial_floats(HS) + 128 * HS + row));
                    for (uint32_t k = c0; k <= c1; k++) {
                        const float *from = a.scratch + ((size_t)paged_place(range, w.tile_unit(), k) * 2 + half) * pc_partial_floats(HS);
                        const float wt = m == -INFINITY ? 0.f : paged_ex2(__ldcg(from + 128 * HS + row) - m);
                        l += wt * __ldcg(from + 128 * (HS + 1) + row);
#pragma unroll
                        for (int i = 0; i < (int)D; i++) acc[i] = fmaf(wt, __ldcg(from + 128 * (D * side + i) + row), acc[i]);
                    }
                }
            }
            if (finish) {   // (the same for all of the half)
                // through q's place in shared memory, from which warps store whole rows; column c of row r lies at c ^ (r % 32)
                float *rows = reinterpret_cast<float *>(smem + half * 2 * HALF);
                const bool sees = p >= 0;   // (a token ahead of the first position sees nothing: 0, whatever the tile's values are)
                const float inv = 1.f / l;
                bool odd = !(l > 0.f);
                if (odd) m = -INFINITY;
#pragma unroll
                for (int i = 0; i < (int)D; i++) {
                    const float y = sees ? acc[i] * inv : 0.f;
                    odd |= !isfinite(y);
                    rows[row * HS + ((D * side + i) ^ (row & 31))] = y;
                }
                const uint32_t mine = __ballot_sync(0xffffffffu, odd && sees);
                if (lane == 0) S.odd[half][side][warp & 3] = mine;
                pc_sync_half(half);
#pragma unroll 4
                for (uint32_t i = 0; i < 16; i++) {
                    const uint32_t rr = 16 * (warp & 7) + i, at = 128 * half + rr, token = token_of(at);
                    if (token >= shape.tokens || w.tile * shape.tokens + token >= w.q.n) break;   // (so are the rows behind it)
                    float *out = a.out + (uint64_t)(w.q.start + w.tile * shape.tokens + token) * a.out_stride + (uint64_t)(w.group * a.kv_mul + at - token * a.kv_mul) * HS;
#pragma unroll
                    for (uint32_t c = lane; c < HS; c += 32) out[c] = rows[rr * HS + (c ^ (rr & 31))];
                }
                uint32_t any = 0;
                for (uint32_t i = 0; i < 8; i++) any |= S.odd[half][i >> 2][i & 3];
                if (any) {
                    pc_sync_half(half);   // (the rows are stored)
                    // (the two warps of the rows share them)
                    pc_repair<HS>(a, shape, S, half, 128 * half + 32 * (warp & 3), (mine | S.odd[half][side ^ 1][warp & 3]) & (side ? 0xFFFF0000u : 0xFFFFu), p, m);
                    unpark();
                }
            }
            pc_sync_half(half);   // (what is shared may be written again)
        } while (w.next(a, shape));
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PC_REGS_OTHER));
      if (warp < PC_W_TMA) {
        // ===== MMA issue of a half =====
        // Every product stands here once: this code competes with the halves' for the instruction caches.
        const uint32_t h = pc_uniform(warp - PC_W_MMA), id_s = pg_idesc(128, 128), id_o = pg_idesc(128, HS) | 1u << 16;   // (V: MN-major)
        const uint32_t t_s = tmem + PC_S + 128 * h, t_o = tmem + PC_O + 128 * h;
        const uint64_t q_lo = pc_desc_k(q0 + h * 2 * HALF + HALF);
        uint32_t slot = 0, phase = 0;                        // of the ring
        uint32_t pq = 0, pp = 0, po = 0, pf = 1, pt = h ^ 1;  // parities: of q's arrival, of P's, of O, of O's release (nobody has to be waited for at first), of the turn (the first half begins)
        auto take = [&]() {   // the next tile of the ring
            const uint32_t at = slot;
            if (wait(b_full + 8 * slot, phase, 11) && ++slot == SLOTS) { slot = 0; phase ^= 1; }
            return at;
        };
        // The walk is the same for both; a half without rows passes its turns on.
        bool now = false, two = pc_uniform(rows_of() > 128), more = true, fresh = true;   // now: the half has rows in this key tile's query tile; two: both have in the next one's
        uint32_t left = 0, vs = 0, ks = 0;                                               // left: key tiles of the query tile
        uint32_t unit = 0, sink_tiles = 0, first_tile = 0;
        int32_t kv_end = 0;
        bool began = false;   // the first round has scores to make only
#pragma unroll 1
        while (ok) {
            const bool products = began;
            if (began) {
                vs = take();
                if (!ok) break;
                const int32_t base = (int32_t)(key_tile({sink_tiles, first_tile, 0, 0}, unit++) * PC_KT);
                if (__any_sync(0xffffffffu, base + (int32_t)PC_KT > kv_end)) {   // rows of the last page that hold nothing: zeros (both warps write them)
                    const uint32_t first = (uint32_t)max(kv_end - base, 0);
                    for (uint32_t c = 0; c < COLS; c++)
#pragma unroll 1
                        for (uint32_t at = first * 128 + lane * 16; at < 16384; at += 512)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring + vs * HALF + c * 16384 + at), "r"(0u) : "memory");
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                now = h == 0 || two;
                fresh = --left == 0;   // the next key tile is another query tile's
                if (fresh) {
                    unpark();
                    more = __any_sync(0xffffffffu, w.next(a, shape));
                    if (more) two = pc_uniform(rows_of() > 128);
                }
            }
            began = true;
            if (fresh && more) {
                left = pc_uniform(w.count);
                unit = w.at;
                kv_end = w.q.p0 + (int32_t)w.q.n;
                sink_tiles = w.span.sink_tiles;
                first_tile = w.span.first;
                park();
            }
            const bool next = more && (h == 0 || two);
            if (more) ks = take();
            if (!ok) break;
            if (products && now) {   // P is there, and O's place is free
                if (!wait(b_p + 8 * h, pp, 12) || !wait(b_free + 8 * h, pf, 12)) break;
                pp ^= 1;
                pf ^= 1;
            }
            if (!wait(b_turn + 8 * h, pt, 12)) break;
            pt ^= 1;
            pg_fence_after();
            if (products && now) {   // O = P V
                if (pg_elect()) {
                    const uint64_t vd = pc_desc_mn(ring + vs * HALF, 16384);
#pragma unroll 1
                    for (uint32_t hi = 0; hi < 2; hi++)   // the remainders first: the sums are small then, and what their additions drop too
#pragma unroll
                        for (uint32_t k = 0; k < 8; k++) pg_mma<false>(t_o, t_s + 8 - 8 * hi + 16 * k, vd + k * (2048 >> 4), id_o, hi | k);
                    pg_commit<false>(b_o + 8 * h);
                    pg_commit<false>(b_empty + 8 * vs);
                }
                __syncwarp();
                // The scores take P's place: only when the products are through with it.  (MMAs with different accumulators are not ordered among themselves.)
                if (!wait(b_o + 8 * h, po, 12)) break;
                po ^= 1;
            }
            if (fresh && products && more) {   // The half has to write this query tile's result before it brings the next one's q; the other half's products do not wait for that.
                if (pg_elect()) pg_arrive(b_turn + 8 * (h ^ 1));
                __syncwarp();
                if (next && !wait(b_q + 8 * h, pq, 12)) break;
                if (!wait(b_turn + 8 * h, pt, 12)) break;
                pt ^= 1;
            } else if (fresh && next && !wait(b_q + 8 * h, pq, 12)) break;   // (the first one)
            if (fresh && next) pq ^= 1;
            pg_fence_after();
            if (pg_elect()) {
                if (next) {   // S = Q K^T of the next key tile
                    const uint64_t kd = pc_desc_k(ring + ks * HALF);
#pragma unroll 1
                    for (uint32_t hi = 0; hi < 2; hi++) {
                        const uint64_t qd = q_lo - hi * (HALF >> 4);
#pragma unroll
                        for (uint32_t k = 0; k < HS / 16; k++) {
                            const uint32_t at = (k / 4) * (16384 >> 4) + (k % 4) * (32 >> 4);
                            pc_mma_ss(t_s, qd + at, kd + at, id_s, hi | k);
                        }
                    }
                    pg_commit<false>(b_s + 8 * h);
                    pg_commit<false>(b_empty + 8 * ks);
                }
                pg_arrive(b_turn + 8 * (h ^ 1));
                if (products && !now) pg_arrive(b_empty + 8 * vs);   // (without rows: the tiles are not needed)
                if (more && !next) pg_arrive(b_empty + 8 * ks);
            }
            __syncwarp();
            if (!more) break;
        }
        if (ok) {   // the last commits arrive in shared memory: let them, before the CTA ends
            const uint32_t last = (slot + SLOTS - 1) % SLOTS;
            wait(b_empty + 8 * last, slot == 0 ? phase ^ 1 : phase, 12);
        }
      } else if (warp == PC_W_TMA) {
        // ===== TMA: K and V of a key tile, one slot of the ring each =====
        const uint32_t page_size = 1u << a.page_log2, box = page_size < PC_KT ? page_size : PC_KT, boxes = PC_KT / box;
        uint32_t slot = 0, use = 0;
        bool more = true;
        do {
            const int32_t *table = a.table + (size_t)w.request * a.max_pages;
            const int32_t kv_end = w.q.p0 + (int32_t)w.q.n, x = (int32_t)(w.group * HS);
            const uint32_t at = w.at, end = w.at + w.count, sink_tiles = w.span.sink_tiles, first_tile = w.span.first;
            park();
            for (uint32_t i = at; i < end && ok; i++) {
                const uint32_t j = key_tile({sink_tiles, first_tile, 0, 0}, i) * PC_KT + lane * box;   // a lane per page
                int32_t page = -1;
                if (lane < boxes && (int32_t)j < kv_end) page = table[j >> a.page_log2];
                const bool there = page >= 0 && (uint32_t)page < a.n_pages;
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, there)) * box * HS * 2;
#pragma unroll
                for (uint32_t v = 0; v < 2; v++) {
                    if (use && !wait(b_empty + 8 * slot, (use - 1) & 1, 12)) break;
                    const uint32_t full = b_full + 8 * slot, dst = ring + slot * HALF + lane * box * 128;
                    if (lane == 0) pg_expect(full, bytes);
                    __syncwarp();
                    if (there)
                        for (uint32_t c = 0; c < COLS; c++)
                            pc_tma3d(dst + c * 16384, v ? &maps.v : &maps.k, x + (int32_t)(64 * c), (int32_t)(j & (page_size - 1)), page, full);
                    __syncwarp();
                    if (++slot == SLOTS) { slot = 0; use++; }
                }
            }
            unpark();
            more = ok && w.next(a, shape);
        } while (more);
      }
    }
    if (!ok) {   // a wait gave up: copies and products of this CTA may still be in flight; give them time to land before the CTA ends
        if (warp == 0 || warp == 8) pc_arrive_at_rest(a, shape, S, warp >> 3);
        const unsigned long long t0 = pg_ns();
        while (pg_ns() - t0 < 100000ull) {}
    }
    __syncwarp();
    pg_fence_before();
    __syncthreads();
    if (warp == PC_W_MMA) pg_dealloc<false>(tmem);
}

uint32_t paged_chunk_ctas(const ib_ctx *ctx) { return (uint32_t)ctx->sm_count; }
size_t paged_chunk_scratch_floats(const ib_ctx *ctx, uint32_t head_size) { return (size_t)paged_chunk_ctas(ctx) * 4 * pc_partial_floats(head_size); }

// Pages of a cache as boxes of up to 128 rows x 64 columns
static int32_t pc_encode(const PagedAttn &a, const void *cache, CUtensorMap *map) {
    EncodeTiledFn encode = encode_tiled();
    IB_REQUIRE(encode, "ib_paged_attention: the driver does not export cuTensorMapEncodeTiled");
    const cuuint32_t page_size = 1u << a.page_log2, box[3] = {64, page_size < PC_KT ? page_size : PC_KT, 1}, estr[3] = {1, 1, 1};
    const cuuint64_t dims[3] = {a.kv_dim, page_size, a.n_pages}, strides[2] = {(cuuint64_t)a.kv_dim * 2, a.page_stride * 2};
    const CUresult cr = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(cache), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    IB_REQUIRE(cr == CUDA_SUCCESS, "ib_paged_attention: cuTensorMapEncodeTiled failed with %d", (int)cr);
    return IB_OK;
}

bool paged_chunk_takes(const PagedAttn &a, int kv_dtype) { return kv_dtype == IB_KV_F16 && a.page_stride * 2 < (1ull << 40); }

int32_t launch_paged_chunk(ib_ctx *ctx, cudaStream_t s, PagedAttn a, uint32_t head_size) {
    const TileShape shape = {a.kv_mul, 1, PC_ROWS / a.kv_mul};
    // Head size 128: 132 KB of a partial through one SM take 2.5 us, a key tile 3.3.  256 rows over 1500, 2000, 4000, 8000 positions: 44, 49, 49, 76 us, with ranges of one key tile 50, 60, 62, 77.
    // Head size 64: a partial takes 1 us, and the ends of ranges that do not meet those of query tiles cost as much as the fewer partials save (25.8 us instead of 22.4 at 1000 positions).
    a.merge_cost = head_size == 128 ? 0.75f : 0.f;
    PcMaps maps;
    int32_t rc = pc_encode(a, a.k, &maps.k);
    if (rc == IB_OK) rc = pc_encode(a, a.v, &maps.v);
    if (rc) return rc;
    void (*kernel)(PagedAttn, TileShape, PcMaps) = head_size == 128 ? paged_chunk_kernel<128> : paged_chunk_kernel<64>;
    static bool attr_set[16] = {false};
    const bool beyond = ctx->device >= 16;
    if (beyond || !attr_set[ctx->device]) {
        IB_CHECK_CUDA(cudaFuncSetAttribute(paged_chunk_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pc_smem(128)));
        IB_CHECK_CUDA(cudaFuncSetAttribute(paged_chunk_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pc_smem(64)));
        if (!beyond) attr_set[ctx->device] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(paged_chunk_ctas(ctx));
    cfg.blockDim = dim3(PC_THREADS);
    cfg.dynamicSmemBytes = pc_smem(head_size);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    IB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, shape, maps));
    ctx->launches++;
    return IB_OK;
}

}  // namespace ib
