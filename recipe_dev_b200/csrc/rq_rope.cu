// Norm and rotation of queries and keys, and the store of keys and values into the paged cache, in one pass over the projections' outputs.
//
//   x' = x / sqrt(mean(x^2) + epsilon) * gain;  (a, b) -> (a cos - b sin, a sin + b cos) over the pairs of the first `rotary` elements
//
// Bound by bytes for a prompt (everything is read once and written once) and by the launch for a few tokens: a warp takes four heads of one token, all of them on
// their way at once and with one reading of the token's row of the table; its lanes hold head_dim / 32 neighbouring elements of each, so that a head is one
// contiguous access and the other element of a pair half a head apart one shuffle; the four sums of squares are added up together. Everything is held in fp32 and a
// key or value is rounded once, to the cache's type. (In place: a warp has read what it writes.) 2039 tokens of 32 + 2 x 8 heads of 128: 22.0 us, 4.2 TB/s; with five
// shuffles and a square root a head 23.8, and of that form with two heads a warp 24.4, eight 27.7, CTAs of eight warps 24.9; one head a warp 30.3. 64 tokens 10.1 us, one
// 9.4, which is what a call from Python takes.
#include "rq_serve.cuh"

using namespace rqserve;

namespace {

constexpr int kWarps = 4, kHeads = 4;

struct RopeParams {
    const float *q, *k, *v, *q_gain, *k_gain, *table;
    float* q_out;
    const int32_t *positions, *slots;
    uint16_t *k_cache, *v_cache;
    int64_t q_stride, k_stride, v_stride, out_stride, table_rows, page_stride, head_stride, line_stride, pages;
    int tokens, q_heads, kv_heads, rotary, style, page_shift;
    float epsilon;
};

// N neighbouring fp32 numbers, in 16-byte (two: 8-byte) accesses where the caller's planes allow them; KEEP: through the L1 cache, for what other warps read too
// (through L2 alone, the few lines of the gains are asked for by every warp: 102 us in place of 25 for 2039 tokens)
template <int N, bool WIDE, bool KEEP = false> __device__ __forceinline__ void load(const float* p, float (&x)[N]) {
    if (WIDE && N >= 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 a = KEEP ? *(const float4*)(p + i) : __ldcg((const float4*)(p + i));
            x[i] = a.x; x[(i + 1) % N] = a.y; x[(i + 2) % N] = a.z; x[(i + 3) % N] = a.w;
        }
    } else if (WIDE && N == 2) {
        const float2 a = KEEP ? *(const float2*)p : __ldcg((const float2*)p);
        x[0] = a.x; x[1 % N] = a.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = KEEP ? p[i] : __ldcg(p + i);
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
    const int heads = p.q_heads + 2 * p.kv_heads, groups = (heads + kHeads - 1) / kHeads, lane = threadIdx.x & 31, first = lane * E, half = p.rotary / 2;
    const uint32_t item = blockIdx.x * kWarps + (threadIdx.x >> 5), t = item / (uint32_t)groups;
    const int head0 = (int)(item % (uint32_t)groups) * kHeads;
    wait_for_previous();
    if (t >= (uint32_t)p.tokens) return;
    // every head's elements on their way at once, with the token's place and position
    float x[kHeads][E];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int head = min(head0 + i, heads - 1);  // (one past the last is loaded for nothing)
        const bool is_q = head < p.q_heads, is_k = head < p.q_heads + p.kv_heads;
        const float* from = is_q ? p.q + t * p.q_stride + (int64_t)head * D
                                 : (is_k ? p.k + t * p.k_stride + (int64_t)(head - p.q_heads) * D : p.v + t * p.v_stride + (int64_t)(head - p.q_heads - p.kv_heads) * D);
        load<E, WIDE>(from + first, x[i]);
    }
    const int slot = __ldcg(p.slots + t);
    const bool turns = first < p.rotary && head0 < p.q_heads + p.kv_heads, low = first < half;
    float c[E], s[E];
    if (turns) {
        const int64_t position = max((int64_t)0, min((int64_t)__ldcg(p.positions + t), p.table_rows - 1));
        const float* row = p.table + position * p.rotary;
        if (p.style == RQ_ROPE_PAIRS) {
            float cs[E / 2], ss[E / 2];
            load<E / 2, WIDE, true>(row + first / 2, cs);
            load<E / 2, WIDE, true>(row + half + first / 2, ss);
#pragma unroll
            for (int i = 0; i < E; i += 2) { c[i] = cs[i / 2]; s[i] = ss[i / 2]; }
        } else {
            const int at = low ? first : first - half;
            load<E, WIDE, true>(row + at, c);
            load<E, WIDE, true>(row + half + at, s);
        }
    }
    // The heads' sums of squares, added up together: each exchange leaves a lane half as many heads to go on with, and at the end one of the four, by bits 4 and 3 of
    // the lane, whose scale it makes for all
    float scale = 0.0f;
    if (p.q_gain || p.k_gain) {
        static_assert(kHeads == 4, "two exchanges of heads");
        float sum[kHeads];
#pragma unroll
        for (int n = 0; n < kHeads; ++n) {
            sum[n] = 0.0f;
#pragma unroll
            for (int i = 0; i < E; ++i) sum[n] = fmaf(x[n][i], x[n][i], sum[n]);
        }
        const bool second = lane & 16, odd = lane & 8;
        const float a0 = (second ? sum[2] : sum[0]) + __shfl_xor_sync(0xffffffffu, second ? sum[0] : sum[2], 16);
        const float a1 = (second ? sum[3] : sum[1]) + __shfl_xor_sync(0xffffffffu, second ? sum[1] : sum[3], 16);
        float all = (odd ? a1 : a0) + __shfl_xor_sync(0xffffffffu, odd ? a0 : a1, 8);
#pragma unroll
        for (int off = 4; off > 0; off >>= 1) all += __shfl_xor_sync(0xffffffffu, all, off);
        scale = 1.0f / sqrtf(all / (float)D + p.epsilon);
    }
    const int64_t page = slot >> p.page_shift;
    const bool stored = slot >= 0 && page < p.pages;  // else passed over: a padding token, or one whose page is lacking
    const int64_t line = page * p.page_stride + (slot & ((1 << p.page_shift) - 1)) * p.line_stride + first;
#pragma unroll
    for (int n = 0; n < kHeads; ++n) {
        const int head = head0 + n;
        if (head >= heads) break;
        const bool is_q = head < p.q_heads, is_k = !is_q && head < p.q_heads + p.kv_heads;
        if (is_q || is_k) {
            const float* gain = is_q ? p.q_gain : p.k_gain;
            if (gain) {
                const float own = __shfl_sync(0xffffffffu, scale, (n >> 1) * 16 + (n & 1) * 8);
                float g[E];
                load<E, WIDE, true>(gain + first, g);
#pragma unroll
                for (int i = 0; i < E; ++i) x[n][i] = x[n][i] * own * g[i];
            }
            if (p.rotary && p.style == RQ_ROPE_PAIRS) {
                if (turns) {
#pragma unroll
                    for (int i = 0; i < E; i += 2) {
                        const float a = x[n][i], b = x[n][i + 1];
                        x[n][i] = a * c[i] - b * s[i];
                        x[n][i + 1] = a * s[i] + b * c[i];
                    }
                }
            } else if (p.rotary) {
                // half is a whole number of lanes: the lane that holds the other elements of this lane's pairs
                const int other = (low ? lane + half / E : lane - half / E) & 31;
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float y = __shfl_sync(0xffffffffu, x[n][i], other);
                    if (turns) x[n][i] = low ? x[n][i] * c[i] - y * s[i] : y * s[i] + x[n][i] * c[i];
                }
            }
        }
        if (is_q) {
            store<E, WIDE>(p.q_out + t * p.out_stride + (int64_t)head * D + first, x[n]);
        } else if (stored) {
            uint16_t* to = (is_k ? p.k_cache + (head - p.q_heads) * p.head_stride : p.v_cache + (head - p.q_heads - p.kv_heads) * p.head_stride) + line;
            uint32_t w[E / 2];
#pragma unroll
            for (int i = 0; i < E; i += 2) w[i / 2] = from_float<TYPE>(x[n][i]) | (uint32_t)from_float<TYPE>(x[n][i + 1]) << 16;
            if (E == 2) *(uint32_t*)to = w[0];
            else if (E == 4) *(uint2*)to = make_uint2(w[0], w[1 % (E / 2)]);
            else *(uint4*)to = make_uint4(w[0], w[1 % (E / 2)], w[2 % (E / 2)], w[3 % (E / 2)]);
        }
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
    const int64_t items = (int64_t)p.tokens * ((p.q_heads + 2 * p.kv_heads + kHeads - 1) / kHeads);
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
    const bool wide = (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)q_gain | (uintptr_t)k_gain | (uintptr_t)table) & 15) == 0 && (tokens == 1 || ((q_t_stride | k_t_stride | v_t_stride | q_out_t_stride) & 3) == 0);
    if (d == 64) return launch_rope<64>(p, cache->type, wide, (cudaStream_t)stream);
    if (d == 128) return launch_rope<128>(p, cache->type, wide, (cudaStream_t)stream);
    return launch_rope<256>(p, cache->type, wide, (cudaStream_t)stream);
}
