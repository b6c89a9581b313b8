// Norm and rotation of queries and keys, and the store of keys and values into the paged cache, in one pass over the projections' outputs.
//
//   x' = x / sqrt(mean(x^2) + epsilon) * gain;  (a, b) -> (a cos - b sin, a sin + b cos) over the pairs of the first `rotary` elements
//
// Bound by bytes for a prompt (everything is read once and written once) and by latency for a few tokens: a warp takes one head of one token, its
// lanes hold head_dim / 32 neighbouring elements each, so that a head is one contiguous access, the sum of squares five shuffles
// and the other element of a pair half a head apart one more. Everything is held in fp32 and a key or value is rounded once.
#include "rq_serve.cuh"

using namespace rqserve;

namespace {

constexpr int kWarps = 8;

struct RopeParams {
    const float *q, *k, *v, *q_gain, *k_gain, *table;
    float* q_out;
    const int32_t *positions, *slots;
    uint16_t *k_cache, *v_cache;
    int64_t q_stride, k_stride, v_stride, out_stride, table_rows, page_stride, head_stride, line_stride, pages;
    int tokens, q_heads, kv_heads, rotary, style, page_shift;
    float epsilon;
};

// E neighbouring fp32 numbers, in 16-byte (E = 2: 8-byte) accesses where the caller's planes allow them
template <int E, bool WIDE> __device__ __forceinline__ void load(const float* p, float (&x)[E]) {
    if (WIDE && E == 2) { const float2 a = __ldcg((const float2*)p); x[0] = a.x; x[1] = a.y; }
    else if (WIDE) {
#pragma unroll
        for (int i = 0; i < E; i += 4) { const float4 a = __ldcg((const float4*)(p + i)); x[i] = a.x; x[i + 1] = a.y; x[i + 2] = a.z; x[i + 3] = a.w; }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = __ldcg(p + i);
    }
}
template <int E, bool WIDE> __device__ __forceinline__ void store(float* p, const float (&x)[E]) {
    if (WIDE && E == 2) *(float2*)p = make_float2(x[0], x[1]);
    else if (WIDE) {
#pragma unroll
        for (int i = 0; i < E; i += 4) *(float4*)(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) p[i] = x[i];
    }
}

template <int D, int TYPE, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32) rq_rope_kernel(RopeParams p) {
    constexpr int E = D / 32;
    launch_dependents();
    const int heads = p.q_heads + 2 * p.kv_heads, lane = threadIdx.x & 31, first = lane * E;
    const int64_t item = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    wait_for_previous();
    if (item >= (int64_t)p.tokens * heads) return;
    const int t = (int)(item / heads), head = (int)(item % heads);
    const int kind = head < p.q_heads ? 0 : (head < p.q_heads + p.kv_heads ? 1 : 2), h = kind == 0 ? head : (head - p.q_heads) % p.kv_heads;
    const int slot = kind == 0 ? 0 : p.slots[t];
    const int64_t page = slot >> p.page_shift;
    if (slot < 0 || (kind != 0 && page >= p.pages)) return;  // passed over: a padding token, or one whose page is lacking
    float x[E];
    load<E, WIDE>((kind == 0 ? p.q + t * p.q_stride : (kind == 1 ? p.k + t * p.k_stride : p.v + t * p.v_stride)) + (int64_t)h * D + first, x);
    if (kind < 2) {
        const float* gain = kind == 0 ? p.q_gain : p.k_gain;
        if (gain) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < E; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            const float scale = 1.0f / sqrtf(sum / (float)D + p.epsilon);
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = x[i] * scale * __ldcg(gain + first + i);
        }
        if (p.rotary) {
            const int64_t position = max((int64_t)0, min((int64_t)p.positions[t], p.table_rows - 1));
            const float* row = p.table + position * p.rotary;
            const int half = p.rotary / 2;
            if (p.style == RQ_ROPE_PAIRS) {
                if (first < p.rotary) {
#pragma unroll
                    for (int i = 0; i < E; i += 2) {
                        const float c = __ldcg(row + (first + i) / 2), s = __ldcg(row + half + (first + i) / 2), a = x[i], b = x[i + 1];
                        x[i] = a * c - b * s;
                        x[i + 1] = a * s + b * c;
                    }
                }
            } else {
                // half is a whole number of lanes: the lane that holds the other elements of this lane's pairs
                const bool low = first < half;
                const int other = low ? lane + half / E : lane - half / E;
                const int i0 = low ? first : first - half;
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float y = __shfl_sync(0xffffffffu, x[i], other & 31);
                    if (first < p.rotary) {
                        const float c = __ldcg(row + i0 + i), s = __ldcg(row + half + i0 + i);
                        x[i] = low ? x[i] * c - y * s : y * s + x[i] * c;
                    }
                }
            }
        }
    }
    if (kind == 0) {
        store<E, WIDE>(p.q_out + t * p.out_stride + (int64_t)h * D + first, x);
    } else {
        uint16_t* to = (kind == 1 ? p.k_cache : p.v_cache) + page * p.page_stride + h * p.head_stride + (slot & ((1 << p.page_shift) - 1)) * p.line_stride + first;
        uint32_t w[E / 2];
#pragma unroll
        for (int i = 0; i < E; i += 2) w[i / 2] = from_float<TYPE>(x[i]) | (uint32_t)from_float<TYPE>(x[i + 1]) << 16;
        if (E == 2) *(uint32_t*)to = w[0];
        else if (E == 4) *(uint2*)to = make_uint2(w[0], w[1 % (E / 2)]);
        else *(uint4*)to = make_uint4(w[0], w[1 % (E / 2)], w[2 % (E / 2)], w[3 % (E / 2)]);
    }
}

__global__ void __launch_bounds__(256) rq_rope_table_kernel(double base, double scale, int half, int64_t rows, float* table) {
    launch_dependents();
    wait_for_previous();
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < rows * half; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / half;
        const int at = (int)(i % half);
        double s, c;
        sincos((double)row * scale * pow(base, -(double)at / half), &s, &c);
        table[row * 2 * half + at] = (float)c;
        table[row * 2 * half + half + at] = (float)s;
    }
}

template <int D>
int launch_rope(const RopeParams& p, int type, bool wide, cudaStream_t s) {
    const int64_t items = (int64_t)p.tokens * (p.q_heads + 2 * p.kv_heads);
    const dim3 grid((unsigned)((items + kWarps - 1) / kWarps));
    auto kernel = type == RQ_KV_F16 ? (wide ? rq_rope_kernel<D, RQ_KV_F16, true> : rq_rope_kernel<D, RQ_KV_F16, false>)
                                    : (wide ? rq_rope_kernel<D, RQ_KV_BF16, true> : rq_rope_kernel<D, RQ_KV_BF16, false>);
    return launch(kernel, grid, kWarps * 32, 0, s, p);
}

}  // namespace

extern "C" int rq_rope_table(rq_ctx* ctx, double base, double frequency_scale, int rotary, int64_t rows, float* table, void* stream) {
    if (!ctx || !table) return rq_fail(RQ_ERR_INVALID, "rq_rope_table: null argument");
    if (!(base > 0.0) || !(frequency_scale > 0.0) || base > 1e300 || frequency_scale > 1e300) return rq_fail(RQ_ERR_INVALID, "rq_rope_table: base and frequency_scale must be finite and positive");
    if (rotary <= 0 || rotary > 256 || rotary % 16) return rq_fail(RQ_ERR_INVALID, "rq_rope_table: rotary=%d is not a multiple of 16 up to 256", rotary);
    if (rows <= 0 || rows > (int64_t)1 << 31) return rq_fail(RQ_ERR_INVALID, "rq_rope_table: rows=%lld is not in 1 .. 2^31", (long long)rows);
    DeviceGuard guard(ctx->device);
    const int64_t want = (rows * (rotary / 2) + 255) / 256;
    return launch(rq_rope_table_kernel, dim3((unsigned)(want < 148 * 8 ? want : 148 * 8)), 256, 0, (cudaStream_t)stream, base, frequency_scale, rotary / 2, rows, table);
}

extern "C" int rq_rope_store(rq_ctx* ctx, const float* q, int64_t q_t_stride, int q_heads, const float* k, int64_t k_t_stride, const float* v, int64_t v_t_stride, int tokens,
                             const float* q_gain, const float* k_gain, float epsilon, const float* table, int64_t table_rows, int rotary, int style,
                             const int32_t* positions, const int32_t* slots, float* q_out, int64_t q_out_t_stride, const rq_kv_cache* cache, void* stream) {
    if (!ctx || !q || !k || !v || !positions || !slots || !q_out || (rotary != 0 && !table)) return rq_fail(RQ_ERR_INVALID, "rq_rope_store: null argument");
    const int rc = check_cache("rq_rope_store", cache);
    if (rc) return rc;
    const int d = cache->head_dim;
    if (tokens <= 0 || q_heads <= 0) return rq_fail(RQ_ERR_INVALID, "rq_rope_store: tokens and q_heads must be positive");
    if (tokens > 1 && (q_t_stride <= 0 || k_t_stride <= 0 || v_t_stride <= 0 || q_out_t_stride <= 0)) return rq_fail(RQ_ERR_INVALID, "rq_rope_store: token strides must be positive");
    if (rotary < 0 || rotary > d || rotary % 16) return rq_fail(RQ_ERR_INVALID, "rq_rope_store: rotary=%d is not a multiple of 16 up to head_dim=%d", rotary, d);
    if (rotary && table_rows <= 0) return rq_fail(RQ_ERR_INVALID, "rq_rope_store: table_rows must be positive");
    if (style != RQ_ROPE_HALVES && style != RQ_ROPE_PAIRS) return rq_fail(RQ_ERR_INVALID, "rq_rope_store: style=%d is neither HALVES(0) nor PAIRS(1)", style);
    if (!(epsilon >= 0.0f)) return rq_fail(RQ_ERR_INVALID, "rq_rope_store: epsilon must be non-negative");
    if ((int64_t)tokens * ((int64_t)q_heads + 2 * (int64_t)cache->heads) > (int64_t)1 << 31) return rq_fail(RQ_ERR_LIMIT, "rq_rope_store: %d tokens of %d + 2 * %d heads are beyond 2^31", tokens, q_heads, cache->heads);
    DeviceGuard guard(ctx->device);
    RopeParams p = {};
    p.q = q; p.k = k; p.v = v; p.q_gain = q_gain; p.k_gain = k_gain; p.table = table; p.q_out = q_out; p.positions = positions; p.slots = slots;
    p.k_cache = (uint16_t*)cache->k; p.v_cache = (uint16_t*)cache->v;
    p.q_stride = q_t_stride; p.k_stride = k_t_stride; p.v_stride = v_t_stride; p.out_stride = q_out_t_stride; p.table_rows = table_rows;
    p.page_stride = cache->page_stride; p.head_stride = cache->head_stride; p.line_stride = cache->line_stride; p.pages = cache->pages;
    p.tokens = tokens; p.q_heads = q_heads; p.kv_heads = cache->heads; p.rotary = rotary; p.style = style; p.epsilon = epsilon;
    while (1 << p.page_shift < cache->page_size) ++p.page_shift;
    const bool wide = (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out) & 15) == 0 && (tokens == 1 || ((q_t_stride | k_t_stride | v_t_stride | q_out_t_stride) & 3) == 0);
    if (d == 64) return launch_rope<64>(p, cache->type, wide, (cudaStream_t)stream);
    if (d == 128) return launch_rope<128>(p, cache->type, wide, (cudaStream_t)stream);
    return launch_rope<256>(p, cache->type, wide, (cudaStream_t)stream);
}
