// ib_paged_attention: checks, scratch, and which kernel takes which requests.
#include "paged_attention.cuh"

namespace ib {

int32_t check_paged_cache(const char *who, const ib_paged_cache *c);   // paged.cu
uint32_t log2_of(uint32_t power);

// Rows (new tokens * kv_mul) up to which a request is the decode kernel's.  At 32 requests over 4000 positions the two take the same at 20 rows (head size 64: 125 us and 131, 128: 187 and 181);
// 16 rows 83 and 131, 117 and 181; 32 rows 155 and 132, 243 and 181.  One request alone is faster with the decode kernel (17 us and 28, 27 and 49 at 64 rows), until it is long: 249 us and 86 at 256 rows over 16,000 positions.
constexpr uint32_t PAGED_FEW_ROWS = 24;

// Scratch of a context, of one size whatever the arguments: made once and never moved, so a captured launch may be replayed at any time.  (Made while a stream is being
// captured, it is cleared on a stream of its own: the capture does not get the clearing as a node.)
static int32_t ensure_paged_scratch(ib_ctx *ctx) {
    if (ctx->paged_scratch) return IB_OK;
    const size_t of_decode = paged_decode_scratch_floats(ctx, 128), floats = of_decode + paged_chunk_scratch_floats(ctx, 128), counters = paged_decode_ctas(ctx) + 2 * paged_chunk_ctas(ctx);
    BesideCaptures beside;
    float *scratch = nullptr;
    cudaStream_t own = nullptr;
    IB_CHECK_CUDA(cudaMalloc(&scratch, floats * sizeof(float) + counters * sizeof(uint32_t)));
    cudaError_t e = cudaStreamCreateWithFlags(&own, cudaStreamNonBlocking);
    if (e == cudaSuccess) e = cudaMemsetAsync(scratch + floats, 0, counters * sizeof(uint32_t), own);
    if (e == cudaSuccess) e = cudaStreamSynchronize(own);
    if (own) cudaStreamDestroy(own);
    if (e != cudaSuccess) {
        cudaFree(scratch);
        return set_error(IB_ERR_CUDA, "ib_paged_attention: clearing the counters failed: %s", cudaGetErrorString(e));
    }
    ctx->paged_scratch = scratch;
    ctx->paged_counters = reinterpret_cast<uint32_t *>(scratch + floats);
    return IB_OK;
}

}  // namespace ib

using namespace ib;

extern "C" int32_t ib_paged_attention(ib_ctx *ctx, void *stream, const ib_paged_attn_args *args, const ib_paged_cache *cache) {
    IB_ENTER(ctx);
    IB_REQUIRE(args, "ib_paged_attention: null argument");
    const ib_paged_attn_args &p = *args;
    int32_t rc = check_paged_cache("ib_paged_attention", cache);
    if (rc) return rc;
    if (p.n_requests == 0 || p.n_tokens == 0) return IB_OK;
    IB_REQUIRE(p.q_dev && p.out_dev && p.block_table && p.row_start && p.kv_len, "ib_paged_attention: null pointer");
    IB_REQUIRE((const float *)p.out_dev != p.q_dev, "ib_paged_attention: out is q");
    IB_REQUIRE(p.kv_mul >= 1 && p.kv_mul <= 64 && p.n_heads >= p.kv_mul && p.n_heads % p.kv_mul == 0, "ib_paged_attention: n_heads=%u is not a multiple of kv_mul=%u (1 to 64)", p.n_heads, p.kv_mul);
    if (p.head_size != 64 && p.head_size != 128) return set_error(IB_ERR_UNSUPPORTED, "ib_paged_attention: head_size=%u (supported: 64, 128)", p.head_size);
    IB_REQUIRE(p.n_heads <= (1u << 16), "ib_paged_attention: %u heads (up to 65536)", p.n_heads);
    IB_REQUIRE(cache->kv_dim == p.n_heads / p.kv_mul * p.head_size, "ib_paged_attention: kv_dim=%u != n_kv_heads*head_size=%u", cache->kv_dim, p.n_heads / p.kv_mul * p.head_size);
    const uint32_t dim = p.n_heads * p.head_size;
    IB_REQUIRE(p.q_stride >= dim && p.out_stride >= dim && p.q_stride < (1ull << 40) && p.out_stride < (1ull << 40), "ib_paged_attention: rows overlap (a stride below %u), or a stride above 2^40", dim);
    IB_REQUIRE(p.n_requests <= 65536 && p.n_tokens < (1u << 25), "ib_paged_attention: %u requests (up to 65536) with %u rows (below 2^25)", p.n_requests, p.n_tokens);
    IB_REQUIRE(p.max_pages >= 1 && (uint64_t)p.max_pages * cache->page_size < (1ull << 31), "ib_paged_attention: rows of %u pages of %u positions (1 to 2^31 - 1 positions)", p.max_pages, cache->page_size);
    rc = ensure_paged_scratch(ctx);
    if (rc) return rc;
    PagedAttn a = {};
    a.q = p.q_dev; a.out = p.out_dev; a.q_stride = p.q_stride; a.out_stride = p.out_stride;
    a.table = p.block_table; a.row_start = p.row_start; a.kv_len = p.kv_len;
    a.k = cache->k_dev; a.v = cache->v_dev; a.page_stride = cache->page_stride;
    a.n_requests = p.n_requests; a.n_tokens = p.n_tokens; a.max_pages = p.max_pages; a.n_pages = cache->n_pages; a.page_log2 = log2_of(cache->page_size);
    a.kv_heads = p.n_heads / p.kv_mul; a.kv_mul = p.kv_mul; a.kv_dim = cache->kv_dim;
    a.window = p.window < (1u << 31) ? (int32_t)p.window : 0;   // (positions are below 2^31: a longer window is none)
    a.sinks = p.sinks < (1u << 31) ? (int32_t)p.sinks : 0x7FFFFFFF;
    a.vec = (uintptr_t)p.q_dev % 16 == 0 && (uintptr_t)p.out_dev % 16 == 0 && p.q_stride % 4 == 0 && p.out_stride % 4 == 0;
    a.err = ctx->err_dev; a.wait_ns = ctx->wait_limit_ns;
    // Requests with few rows go through tiles of 8, the others through tiles of 256.  The host knows no lengths: where requests of either kind can be there, both kernels are launched, each for
    // its own.  One that is alone takes all of them, whatever they turn out to be.
    const uint64_t most = (uint64_t)(p.longest_new && p.longest_new < p.n_tokens ? p.longest_new : p.n_tokens) * p.kv_mul;
    const bool chunks = most > PAGED_FEW_ROWS && paged_chunk_takes(a, cache->kv_dtype), few = !chunks || p.n_requests > 1;
    const uint32_t border = chunks && few ? PAGED_FEW_ROWS : (chunks ? 0u : 0xFFFFFFFFu);
    if (few) {
        a.scratch = ctx->paged_scratch;
        a.counters = ctx->paged_counters;
        a.rows_from = 1;
        a.rows_to = border;
        rc = launch_paged_decode(ctx, (cudaStream_t)stream, a, p.head_size, cache->kv_dtype);
        if (rc) return rc;
    }
    if (!chunks) return IB_OK;
    a.scratch = ctx->paged_scratch + paged_decode_scratch_floats(ctx, 128);
    a.counters = ctx->paged_counters + paged_decode_ctas(ctx);
    a.rows_from = border + 1;
    a.rows_to = 0xFFFFFFFFu;
    return launch_paged_chunk(ctx, (cudaStream_t)stream, a, p.head_size);
}
