// What the kernels of a few rows at a time share (rq_attention.cu over 16-bit caches, rq_attention_int8.cu over 8-bit codes): copies into shared memory, how
// the requests' keys are dealt out over CTAs, and how the sums of a CTA's warps, and of CTAs that share rows, are joined.
#pragma once
#include "rq_attention.cuh"
#include "rq_mma.cuh"

namespace rqattn {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kRequestStep = 128;  // requests' places in shared memory are taken by so many

#ifdef __CUDACC__
// a * b + c, two numbers an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
// four matrices of eight lines x sixteen bytes, lane l giving line l % 8 of matrix l / 8
__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_transposed(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// sixteen bytes, or zeros
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A request's rows and keys, as a CTA deals with them: ROWS rows at a time, a warp takes TILE keys
struct Request {
    int fresh, here, length, begin, end, tiles;  // new tokens, those with queries; keys [begin, end) are seen by some row; row tiles
    int64_t units;                         // of one row tile and head
};
template <int ROWS, int TILE> __device__ __forceinline__ Request request_of(const AttentionParams& p, int r) {
    Request q;
    const int start = p.starts[r];
    const int next = p.starts[r + 1];
    q.fresh = max(next - start, 0);
    q.here = tokens_here(p, start, next);
    q.length = p.lengths[r];
    q.end = (int)min((int64_t)max(q.length, 0), (int64_t)p.table_width << p.page_shift);
    q.begin = p.window > 0 ? (int)max((int64_t)0, (int64_t)q.length - q.fresh - p.window + 1) : 0;
    q.begin = min(q.begin, q.end) & ~(TILE - 1);
    q.tiles = (q.here * (p.q_heads / p.kv_heads) + ROWS - 1) / ROWS;
    q.units = max((q.end - q.begin + kWarps * TILE - 1) / (kWarps * TILE), 1);  // (a row that sees no key is written all the same)
    return q;
}

// Where this CTA's units lie: [begin, end) of `total` over `ctas` CTAs (0: there are none)
struct Deal {
    int64_t total, ctas, begin, end;
};
// before: the units before each request, left behind; sums: a number a warp. LEAD: units that each row tile and head counts for in the dealing beside its own
template <int ROWS, int TILE, int LEAD = 0> __device__ __forceinline__ Deal deal_units(const AttentionParams& p, int64_t* before, int64_t* sums) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = p.q_heads / p.kv_heads;
    int64_t total = 0;
    if (tid == 0) before[0] = 0;
    for (int r0 = 0; r0 < p.requests; r0 += kThreads) {
        int64_t units = 0;
        if (r0 + tid < p.requests) { const Request q = request_of<ROWS, TILE>(p, r0 + tid); units = (int64_t)q.here * group > p.few ? 0 : (LEAD + q.units) * q.tiles * p.kv_heads; }
        int64_t scan = units;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) { const int64_t o = __shfl_up_sync(0xffffffffu, scan, off); if (lane >= off) scan += o; }
        __syncthreads();
        if (lane == 31) sums[warp] = scan;
        __syncthreads();
        scan += total;
        for (int w = 0; w < kWarps; ++w) { if (w < warp) scan += sums[w]; total += sums[w]; }
        if (r0 + tid < p.requests) before[r0 + tid + 1] = scan;
    }
    __syncthreads();
    Deal d = {total, min((int64_t)gridDim.x, total), 0, 0};
    if (blockIdx.x < d.ctas) { d.begin = blockIdx.x * total / d.ctas; d.end = (blockIdx.x + 1) * total / d.ctas; }
    return d;
}

// A row's results: sums over the sum of weights
template <int D> __device__ __forceinline__ void put_row(const AttentionParams& p, int group, int start, int at, int kv, int e, float4 v, float total_weight) {
    float* y = p.y + (int64_t)(start + at / group) * p.y_stride + (int64_t)(kv * group + at % group) * D;
    const float inverse = total_weight == 0.0f ? 0.0f : 1.0f / total_weight;
    v.x *= inverse; v.y *= inverse; v.z *= inverse; v.w *= inverse;
    if (p.wide) *(float4*)(y + e) = v;
    else { y[e] = v.x; y[e + 1] = v.y; y[e + 2] = v.z; y[e + 3] = v.w; }
}

// The parts that CTAs first_cta .. last_cta have left of some rows, joined: many of them. (Of few, each thread is done by itself sooner than through shared memory: a token over 1001 keys
// 9.1 us, 10.4 so.)
template <int D, int ROWS>
__device__ __forceinline__ void join_parts(const AttentionParams& p, float* out, int64_t first_cta, int64_t last_cta, int start, int row0, int rows, int kv) {
    const int tid = threadIdx.x;
    const int64_t stride = ROWS * (D + 2);
    // The parts' bases and sums of weights are brought by all threads side by side, some parts at a time, and their sums many at once; they are added up in CTA order. (Each thread
    // for itself, a few loads at a time, took the last CTA of 55 ten microseconds.)
    constexpr int ITEMS = (ROWS * (D / 4) + kThreads - 1) / kThreads, kParts = 64;
    static_assert(kThreads % ROWS == 0 && 2 * kParts * ROWS <= kWarps * ROWS * (D + 8) && kThreads <= kWarps * ROWS * (D + 8), "the place of the warps' sums");
    const int parts = (int)(last_cta - first_cta) + 1, my_row = tid % ROWS;
    auto part = [&](int c) { return p.partial + ((first_cta + c) * 2 + (c == 0)) * stride; };
    float top = -INFINITY;
#pragma unroll 4
    for (int c = tid / ROWS; c < parts; c += kThreads / ROWS) top = fmaxf(top, __ldcg(part(c) + ROWS * D + my_row));
    out[tid] = top;
    __syncthreads();
#pragma unroll
    for (int i = my_row; i < kThreads; i += ROWS) top = fmaxf(top, out[i]);
    const float to = top == -INFINITY ? 0.0f : top;
    float4 v[ITEMS];
    float weight[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) { v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f); weight[i] = 0.0f; }
    for (int c0 = 0; c0 < parts; c0 += kParts) {
        const int here = min(kParts, parts - c0);
        __syncthreads();
#pragma unroll 4
        for (int c = tid / ROWS; c < here; c += kThreads / ROWS) {
            const float* from = part(c0 + c) + ROWS * D + my_row;
            *(float2*)(out + 2 * (c * ROWS + my_row)) = make_float2(exp2_fast(__ldcg(from) - to), __ldcg(from + ROWS));
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int item = tid + i * kThreads, row = item / (D / 4), e = 4 * (item % (D / 4));
            if (row >= rows) break;
#pragma unroll 28
            for (int c = 0; c < here; ++c) {
                const float4 o = __ldcg((const float4*)(part(c0 + c) + row * D + e));
                const float2 f = *(const float2*)(out + 2 * (c * ROWS + row));
                v[i].x = fmaf(o.x, f.x, v[i].x); v[i].y = fmaf(o.y, f.x, v[i].y); v[i].z = fmaf(o.z, f.x, v[i].z); v[i].w = fmaf(o.w, f.x, v[i].w);
                weight[i] = fmaf(f.y, f.x, weight[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int item = tid + i * kThreads, row = item / (D / 4), e = 4 * (item % (D / 4));
        if (row < rows) put_row<D>(p, p.q_heads / p.kv_heads, start, row0 + row, kv, e, v[i], weight[i]);
    }
}

// The warps' sums of rows (out: [warp][row][D + 8]; their bases and sums of weights) to y, or, where other CTAs have parts of the rows' units [item_begin, item_end), to the
// work area; the last of those CTAs joins the parts in CTA order (LEAD: as dealt, the first units of an item are nobody's work; MANY: of more than kFewParts by join_parts). start: the
// request's first token. Begins behind a barrier that all have written before.
constexpr int kFewParts = 16;
template <int D, int ROWS, int LEAD = 0, bool MANY = false>
__device__ __forceinline__ void join_rows(const AttentionParams& p, float* out, const float (&warp_base)[kWarps][ROWS], const float (&warp_sum)[kWarps][ROWS], int64_t item_begin,
                                          int64_t item_end, const Deal& deal, int start, int row0, int rows, int kv, uint32_t& last_arrival) {
    const int tid = threadIdx.x, group = p.q_heads / p.kv_heads;
    const int64_t first_cta = ((item_begin + LEAD + 1) * deal.ctas - 1) / deal.total, last_cta = (item_end * deal.ctas - 1) / deal.total;
    const bool whole = first_cta == last_cta;
    const int64_t stride = ROWS * (D + 2);
    float* mine = p.partial + ((int64_t)blockIdx.x * 2 + (blockIdx.x == first_cta)) * stride;
    for (int i = tid; i < ROWS * (D / 4); i += kThreads) {
        const int row = i / (D / 4), e = 4 * (i % (D / 4));
        if (row >= rows) break;
        float top = warp_base[0][row];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, warp_base[w][row]);
        const float to = top == -INFINITY ? 0.0f : top;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float weight = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = exp2_fast(warp_base[w][row] - to);
            const float4 o = *(const float4*)&out[(w * ROWS + row) * (D + 8) + e];
            v.x = fmaf(o.x, f, v.x); v.y = fmaf(o.y, f, v.y); v.z = fmaf(o.z, f, v.z); v.w = fmaf(o.w, f, v.w);
            weight = fmaf(warp_sum[w][row], f, weight);
        }
        if (whole) {
            put_row<D>(p, group, start, row0 + row, kv, e, v, weight);
        } else {
            __stcg((float4*)(mine + row * D + e), v);
            if (e == 0) { __stcg(mine + ROWS * D + row, top); __stcg(mine + ROWS * D + ROWS + row, weight); }
        }
    }
    if (!whole) {
        __threadfence();
        __syncthreads();
        if (tid == 0) last_arrival = atomicAdd(&p.arrived[first_cta], 1);
        __syncthreads();
        if (last_arrival == (uint32_t)(last_cta - first_cta)) {
            if (tid == 0) p.arrived[first_cta] = 0;
            __threadfence();
            if (MANY && last_cta - first_cta >= kFewParts) {
                join_parts<D, ROWS>(p, out, first_cta, last_cta, start, row0, rows, kv);
                return;
            }
            for (int i = tid; i < ROWS * (D / 4); i += kThreads) {
                const int row = i / (D / 4), e = 4 * (i % (D / 4));
                if (row >= rows) break;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float weight = 0.0f, top = -INFINITY;
#pragma unroll 8
                for (int64_t c = first_cta; c <= last_cta; ++c) top = fmaxf(top, __ldcg(p.partial + (c * 2 + (c == first_cta)) * stride + ROWS * D + row));
                const float to = top == -INFINITY ? 0.0f : top;
#pragma unroll 8
                for (int64_t c = first_cta; c <= last_cta; ++c) {
                    const float* from = p.partial + (c * 2 + (c == first_cta)) * stride;
                    const float f = exp2_fast(__ldcg(from + ROWS * D + row) - to);
                    const float4 o = __ldcg((const float4*)(from + row * D + e));
                    v.x = fmaf(o.x, f, v.x); v.y = fmaf(o.y, f, v.y); v.z = fmaf(o.z, f, v.z); v.w = fmaf(o.w, f, v.w);
                    weight = fmaf(__ldcg(from + ROWS * D + ROWS + row), f, weight);
                }
                put_row<D>(p, group, start, row0 + row, kv, e, v, weight);
            }
        }
    }
}
#endif

}  // namespace rqattn
