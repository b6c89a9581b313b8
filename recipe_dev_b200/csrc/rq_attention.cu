// Attention of new tokens over the paged cache.
//
//   y = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale * q . k_j - m),  over the keys j that the token sees
//
// A warp takes one query head of one token and walks its keys once: scores by shuffles, the running maximum m and sum of the weights
// in fp32, the accumulated values scaled down when m grows.
#include "rq_serve.cuh"

using namespace rqserve;

namespace {

constexpr int kWarps = 8;

struct AttentionParams {
    const float* q;
    float* y;
    const uint16_t *k, *v;
    const int32_t *block_table, *starts, *lengths;
    int64_t q_stride, y_stride, table_stride, page_stride, head_stride, line_stride, pages;
    int tokens, requests, q_heads, kv_heads, table_width, page_shift, window;
    float scale;
};

template <int D, int TYPE>
__global__ void __launch_bounds__(kWarps * 32) rq_attention_kernel(AttentionParams p) {
    constexpr int E = D / 32;
    launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    wait_for_previous();
    if (item >= (int64_t)p.tokens * p.q_heads) return;
    const int t = (int)(item / p.q_heads), head = (int)(item % p.q_heads), kv = head / (p.q_heads / p.kv_heads);
    if (t < p.starts[0] || t >= p.starts[p.requests]) return;
    const int r = owner_of(p.starts, p.requests, t), length = p.lengths[r];
    const int64_t position = (int64_t)length - (p.starts[r + 1] - t);
    const int64_t end = min(position + 1, min((int64_t)length, (int64_t)p.table_width << p.page_shift));
    const int64_t begin = p.window > 0 ? max(position - p.window + 1, (int64_t)0) : 0;
    float q[E], acc[E], m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) { q[i] = p.q[t * p.q_stride + (int64_t)head * D + i * 32 + lane] * p.scale; acc[i] = 0.0f; }
    for (int64_t j = begin; j < end; ++j) {
        const int64_t page = p.block_table[r * p.table_stride + (j >> p.page_shift)];
        if (page < 0 || page >= p.pages) continue;
        const int64_t at = page * p.page_stride + kv * p.head_stride + (j & ((1 << p.page_shift) - 1)) * p.line_stride + lane;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) s = fmaf(q[i], to_float<TYPE>(p.k[at + i * 32]), s);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        const float top = fmaxf(m, s), old = m == top ? 1.0f : expf(m - top), w = s == top ? 1.0f : expf(s - top);
        sum = sum * old + w;
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] = fmaf(acc[i], old, w * to_float<TYPE>(p.v[at + i * 32]));
        m = top;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) p.y[t * p.y_stride + (int64_t)head * D + i * 32 + lane] = sum > 0.0f ? acc[i] / sum : (sum == 0.0f ? 0.0f : sum);
}

}  // namespace

extern "C" int rq_attention_reserve(rq_ctx* ctx) {
    if (!ctx) return rq_fail(RQ_ERR_INVALID, "rq_attention_reserve: null context");
    return RQ_OK;
}

extern "C" int rq_attention(rq_ctx* ctx, const float* q, int64_t q_t_stride, int q_heads, const rq_kv_cache* cache, const int32_t* block_table, int64_t table_stride,
                            int table_width, const int32_t* starts, const int32_t* lengths, int requests, int tokens, int max_fresh, float scale, int window, float* y,
                            int64_t y_t_stride, void* stream) {
    if (!ctx || !q || !block_table || !starts || !lengths || !y) return rq_fail(RQ_ERR_INVALID, "rq_attention: null argument");
    int rc = check_cache("rq_attention", cache);
    if (rc) return rc;
    if (requests <= 0 || tokens <= 0 || q_heads <= 0 || table_width <= 0 || table_stride < table_width)
        return rq_fail(RQ_ERR_INVALID, "rq_attention: requests, tokens, q_heads and table_width must be positive and table_stride at least table_width");
    if (q_heads % cache->heads) return rq_fail(RQ_ERR_INVALID, "rq_attention: %d query heads are not a multiple of the cache's %d", q_heads, cache->heads);
    if (tokens > 1 && (q_t_stride <= 0 || y_t_stride <= 0)) return rq_fail(RQ_ERR_INVALID, "rq_attention: token strides must be positive");
    if (max_fresh < 0 || window < 0) return rq_fail(RQ_ERR_INVALID, "rq_attention: max_fresh and window must not be negative");
    if (!(scale > 0.0f) || scale > 3e38f) return rq_fail(RQ_ERR_INVALID, "rq_attention: scale must be finite and positive");
    if (requests > RQ_MAX_REQUESTS) return rq_fail(RQ_ERR_LIMIT, "rq_attention: %d requests; at most %d", requests, RQ_MAX_REQUESTS);
    if (q_heads / cache->heads > 128) return rq_fail(RQ_ERR_LIMIT, "rq_attention: %d query heads share a key head; at most 128", q_heads / cache->heads);
    DeviceGuard guard(ctx->device);
    AttentionParams p = {};
    p.q = q; p.y = y; p.k = (const uint16_t*)cache->k; p.v = (const uint16_t*)cache->v; p.block_table = block_table; p.starts = starts; p.lengths = lengths;
    p.q_stride = q_t_stride; p.y_stride = y_t_stride; p.table_stride = table_stride; p.page_stride = cache->page_stride; p.head_stride = cache->head_stride;
    p.line_stride = cache->line_stride; p.pages = cache->pages; p.tokens = tokens; p.requests = requests; p.q_heads = q_heads; p.kv_heads = cache->heads;
    p.table_width = table_width; p.window = window; p.scale = scale;
    while (1 << p.page_shift < cache->page_size) ++p.page_shift;
    const int64_t items = (int64_t)tokens * q_heads;
    const dim3 grid((unsigned)((items + kWarps - 1) / kWarps));
    auto pick = [&](auto f16, auto bf16) { return cache->type == RQ_KV_F16 ? f16 : bf16; };
    auto kernel = cache->head_dim == 64 ? pick(rq_attention_kernel<64, RQ_KV_F16>, rq_attention_kernel<64, RQ_KV_BF16>)
                  : cache->head_dim == 128 ? pick(rq_attention_kernel<128, RQ_KV_F16>, rq_attention_kernel<128, RQ_KV_BF16>)
                                           : pick(rq_attention_kernel<256, RQ_KV_F16>, rq_attention_kernel<256, RQ_KV_BF16>);
    return launch(kernel, grid, kWarps * 32, 0, (cudaStream_t)stream, p);
}
