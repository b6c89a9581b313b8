// Attention of new tokens over the paged cache.
//
//   y = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale * q . k_j - m),  over the keys j that the token sees
//
// rq_attention_rows_kernel, for up to sixteen rows (new tokens x the query heads that share a key head) at a time: a decode step. It is bound by the bytes of
// the cache, read once, so everything else is arranged around loads:
//   * a warp takes 32 keys at a time (16 of 256 elements) straight from global memory into the operand registers of mma.sync: which elements
//     the tensor core takes together is free as long as both operands agree, so a thread loads sixteen bytes of a key (or of a value, for four
//     keys, whose halves a byte permute pairs up) and nothing passes through shared memory. The keys of the next tile are under way while
//     the values of this one are used.
//   * fp32 activations: queries and weights are taken apart into 16-bit parts, hi + lo over f16 (22 bits), hi + mid + lo over
//     bf16 (24 bits). The sixteen rows of an operand are eight rows' hi parts above their lo parts: one instruction does both.
//   * The tensor core adds by truncation, a bias that grows with the length of a chain: a sum stays in it for one tile and is then added, with
//     round-to-nearest, to the row's fp32 sums, which are scaled by 2^(old max - new max) in the same multiply-add.
//   * The keys of all requests and heads, in units of 128, are dealt out evenly: every CTA takes an equal range of units, wherever it begins and ends.
//     Rows whose units fall to several CTAs are joined, in CTA order, by whichever of these is the last to leave its sums: the same bits on every run.
#include "rq_attention.cuh"

using namespace rqserve;
using namespace rqattn;

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kUnit = 128;  // keys

template <int TYPE> __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (TYPE == RQ_KV_F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Whether a word's two 16-bit numbers are both finite
template <int TYPE> __device__ __forceinline__ bool finite2(uint32_t w) {
    const uint32_t e = TYPE == RQ_KV_F16 ? 0x7c00u : 0x7f80u;
    return (w & e) != e && ((w >> 16) & e) != e;
}

__device__ __forceinline__ uint4 load16(const uint16_t* p) { return __ldcg((const uint4*)p); }

// A request's rows and keys, as a CTA deals with them
struct Request {
    int fresh, length, begin, end, tiles;  // keys [begin, end) are seen by some row; row tiles
    int64_t units;                         // of one row tile and head
};
template <int ROWS> __device__ __forceinline__ Request request_of(const AttentionParams& p, int r) {
    Request q;
    const int start = p.starts[r];
    q.fresh = max(p.starts[r + 1] - start, 0);
    q.length = p.lengths[r];
    q.end = (int)min((int64_t)max(q.length, 0), (int64_t)p.table_width << p.page_shift);
    q.begin = p.window > 0 ? (int)max((int64_t)0, (int64_t)q.length - q.fresh - p.window + 1) : 0;
    q.begin = min(q.begin, q.end) & ~31;  // tiles begin at whole multiples of 32 keys
    q.tiles = (q.fresh * (p.q_heads / p.kv_heads) + ROWS - 1) / ROWS;
    q.units = max((q.end - q.begin + kUnit - 1) / kUnit, 1);  // (a row that sees no key is written all the same)
    return q;
}

template <int D, int TYPE, int RT> struct Tiles {
    uint4 q_hi[RT][D / 16][32];                          // operand registers of the queries: hi above lo (f16), hi above mid (bf16)
    uint2 q_lo[TYPE == RQ_KV_BF16 ? RT : 1][D / 16][32];  // the third parts
    float out[kWarps][8 * RT][D + 4];                    // the warps' sums
};

template <int D, int TYPE, int RT>
__global__ void __launch_bounds__(kThreads, D == 64 ? 4 : 2) rq_attention_rows_kernel(AttentionParams p) {
    constexpr int ROWS = 8 * RT, TK = D == 256 ? 16 : 32, NT = TK / 8, STEPS = D / 16, KC = D / 32, VC = D / 64, PARTS = TYPE == RQ_KV_F16 ? 2 : 3;
    extern __shared__ __align__(16) unsigned char dynamic[];
    Tiles<D, TYPE, RT>& sh = *(Tiles<D, TYPE, RT>*)dynamic;
    auto& q_hi = sh.q_hi;
    auto& q_lo = sh.q_lo;
    auto& out = sh.out;
    int64_t* before = (int64_t*)(dynamic + sizeof(sh));  // units before each request
    __shared__ float warp_max[kWarps][ROWS], warp_sum[kWarps][ROWS];
    __shared__ int64_t sums[kWarps];
    __shared__ uint32_t last_arrival;
    launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int group = p.q_heads / p.kv_heads;
    wait_for_previous();

    // ---- where this CTA's units lie -----------------------------------------------------------------
    int64_t total = 0;
    if (tid == 0) before[0] = 0;
    for (int r0 = 0; r0 < p.requests; r0 += kThreads) {
        int64_t units = 0;
        if (r0 + tid < p.requests) { const Request q = request_of<ROWS>(p, r0 + tid); units = q.units * q.tiles * p.kv_heads; }
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
    if (total == 0) return;
    const int64_t ctas = min((int64_t)gridDim.x, total);
    if (blockIdx.x >= ctas) return;
    const int64_t my_end = (blockIdx.x + 1) * total / ctas;
    int64_t u = blockIdx.x * total / ctas;

    while (u < my_end) {
        // the rows that unit u belongs to
        int r = 0;
        for (int hi = p.requests - 1; r < hi;) { const int mid = (r + hi + 1) >> 1; if (before[mid] <= u) r = mid; else hi = mid - 1; }
        const Request rq = request_of<ROWS>(p, r);
        const int64_t in_request = u - before[r], item = in_request / rq.units, first_unit = in_request % rq.units;
        const int kv = (int)(item % p.kv_heads), row0 = (int)(item / p.kv_heads) * ROWS, rows = min(ROWS, rq.fresh * group - row0);
        const int64_t item_begin = u - first_unit, item_end = item_begin + rq.units, stop = min(item_end, my_end);
        const int key_first = rq.begin + (int)first_unit * kUnit, key_stop = min(rq.end, rq.begin + (int)(stop - item_begin) * kUnit);
        u = stop;

        // queries: scaled, taken apart, in the order in which the tensor core takes a key's elements (see the loads below)
        for (int i = tid; i < RT * STEPS * 32; i += kThreads) {
            const int l = i & 31, step = (i >> 5) % STEPS, rt = i / (32 * STEPS), row = rt * 8 + (l >> 2);
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (row < rows) {
                const int at = row0 + row;
                const float* from = p.q + (int64_t)(p.starts[r] + at / group) * p.q_stride + (int64_t)(kv * group + at % group) * D + 8 * ((l & 3) + 4 * (step >> 1)) + 4 * (step & 1);
                if (p.wide) { const float4 v = __ldcg((const float4*)from); x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
                else { for (int e = 0; e < 4; ++e) x[e] = __ldcg(from + e); }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] *= p.scale * kLog2e;
            uint4 a;
            a.x = take_pair<TYPE>(x[0], x[1]);
            a.z = take_pair<TYPE>(x[2], x[3]);
            a.y = take_pair<TYPE>(x[0], x[1]);
            a.w = take_pair<TYPE>(x[2], x[3]);
            q_hi[rt][step][l] = a;
            if (PARTS == 3) q_lo[rt % (PARTS == 3 ? RT : 1)][step][l] = make_uint2(pair_of<TYPE>(x[0], x[1]), pair_of<TYPE>(x[2], x[3]));
        }
        __syncthreads();

        // the keys that this thread's rows see: [low, high)
        int low[RT], high[RT];
        const int position0 = rq.length - rq.fresh, seen_high = min(rq.end, position0 + (row0 + max(rows, 1) - 1) / group + 1);
        const int seen_low = p.window > 0 ? max(0, position0 + row0 / group - p.window + 1) : 0;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int position = position0 + (row0 + rt * 8 + g) / group;
            high[rt] = rt * 8 + g < rows ? min(position + 1, rq.end) : 0;
            low[rt] = p.window > 0 ? max(position - p.window + 1, 0) : 0;
        }
        const bool one_token = row0 / group == (row0 + max(rows, 1) - 1) / group;

        float m[RT], sum[RT], acc[RT][VC][16];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = -INFINITY;
            sum[rt] = 0.0f;
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[rt][c][i] = 0.0f;
        }

        // where a tile's keys lie: lane l finds key l's, -1 for a key that no row sees
        auto entry_of = [&](int key0) -> int {
            const int key = key0 + (lane & (TK - 1));
            return key < key_stop ? __ldcg(p.block_table + r * p.table_stride + (key >> p.page_shift)) : -1;
        };
        auto place_of = [&](int key0, int entry) -> int64_t {
            const int key = key0 + (lane & (TK - 1));
            if (key < seen_low || key >= min(key_stop, seen_high) || entry < 0 || entry >= p.pages) return -1;
            return entry * p.page_stride + (key & ((1 << p.page_shift) - 1)) * p.line_stride;
        };
        const uint16_t *k_head = p.k + kv * p.head_stride, *v_head = p.v + kv * p.head_stride;
        uint4 kreg[NT][KC];
        auto load_keys = [&](int64_t place) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int64_t at = __shfl_sync(0xffffffffu, place, 8 * i + g);
#pragma unroll
                for (int c = 0; c < KC; ++c) kreg[i][c] = at >= 0 ? load16(k_head + at + 8 * (t4 + 4 * c)) : make_uint4(0, 0, 0, 0);
            }
        };

        int key0 = key_first + warp * TK;
        int64_t place = -1;
        int entry = -1;
        if (key0 < key_stop) {
            place = place_of(key0, entry_of(key0));
            load_keys(place);
            entry = entry_of(key0 + kWarps * TK);
        }
        for (; key0 < key_stop; key0 += kWarps * TK) {
            const uint32_t valid = __ballot_sync(0xffffffffu, place >= 0);
            // values, a chunk of 64 elements ahead of its use
            uint4 vreg[2][TK / 4];
            auto load_values = [&](int c) {
#pragma unroll
                for (int i = 0; i < TK / 4; ++i) {  // keys 16 s + 2 t4 + {0, 1, 8, 9}
                    const int64_t at = __shfl_sync(0xffffffffu, place, 16 * (i >> 2) + 2 * t4 + (i & 1) + 8 * ((i >> 1) & 1));
                    vreg[c & 1][i] = at >= 0 ? load16(v_head + at + 8 * (g + 8 * c)) : make_uint4(0, 0, 0, 0);
                }
            };
            load_values(0);

            // scores: of key 8 i + 2 t4 + {0, 1} and row g
            float s[RT][NT][2];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float c[NT][4];
#pragma unroll
                for (int i = 0; i < NT; ++i) c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0.0f;
#pragma unroll
                for (int step = 0; step < STEPS; ++step) {
                    const uint4 a = q_hi[rt][step][lane];
                    uint2 lo = make_uint2(0, 0);
                    if (PARTS == 3) lo = q_lo[rt % (PARTS == 3 ? RT : 1)][step][lane];
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        const uint4 b = kreg[i][step >> 1];
                        const uint32_t b0 = step & 1 ? b.z : b.x, b1 = step & 1 ? b.w : b.y;
                        if (PARTS == 3) mma<TYPE>(c[i], 0, lo.x, 0, lo.y, b0, b1);  // with the small parts
                        mma<TYPE>(c[i], a.x, a.y, a.z, a.w, b0, b1);
                    }
                }
#pragma unroll
                for (int i = 0; i < NT; ++i) { s[rt][i][0] = c[i][0] + c[i][2]; s[rt][i][1] = c[i][1] + c[i][3]; }
            }
            // the next tile's keys, under way from here on
            const int next = key0 + kWarps * TK;
            const int64_t next_place = next < key_stop ? place_of(next, entry) : -1;
            if (next < key_stop) {
                load_keys(next_place);
                entry = entry_of(next + kWarps * TK);
            }

            // weights
            uint32_t w_hi[RT][NT], w_mid[RT][NT], w_lo[RT][PARTS == 3 ? NT : 1];
            float old[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float top = m[rt];
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int at = 8 * i + 2 * t4 + e, key = key0 + at;
                        if (key < low[rt] || key >= high[rt] || !(valid >> at & 1)) s[rt][i][e] = -INFINITY;
                        top = fmaxf(top, s[rt][i][e]);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float base = (top == -INFINITY ? 0.0f : top) - kRaise;
                old[rt] = exp2_fast(m[rt] - (base + kRaise));
                m[rt] = top;
                float add = 0.0f;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    float a = exp2_fast(s[rt][i][0] - base), b = exp2_fast(s[rt][i][1] - base);
                    add += a + b;
                    w_hi[rt][i] = take_pair<TYPE>(a, b);
                    w_mid[rt][i] = take_pair<TYPE>(a, b);
                    if (PARTS == 3) w_lo[rt][i % (PARTS == 3 ? NT : 1)] = pair_of<TYPE>(a, b);
                }
                sum[rt] = fmaf(sum[rt], old[rt], add);
            }

            // A value that one row must not see may be infinite, and 0 * inf is no 0. Where a tile's rows do not see the same keys and a value
            // is not finite, the rows of each token meet the values by themselves, the unseen ones taken out.
            int token = -1, tokens = 0;
            const bool partial = !one_token && (key0 < seen_low + (rows - 1) / group + 1 || key0 + TK > position0 + row0 / group + 1);

#pragma unroll
            for (int c = 0; c < VC; ++c) {
                if (c + 1 < VC) load_values(c + 1);
                uint4* v = vreg[c & 1];
                if (partial) {
                    bool fine = true;
#pragma unroll
                    for (int i = 0; i < TK / 4; ++i) fine = fine && finite2<TYPE>(v[i].x) && finite2<TYPE>(v[i].y) && finite2<TYPE>(v[i].z) && finite2<TYPE>(v[i].w);
                    token = __all_sync(0xffffffffu, fine) ? -1 : row0 / group;
                    tokens = token < 0 ? 0 : (row0 + rows - 1) / group - token;
                }
                float scaled[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) scaled[rt] = old[rt];
                for (int pass = 0; pass <= tokens; ++pass) {
                    uint32_t shown = 0xffffffffu, row_on[RT];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) row_on[rt] = 0xffffffffu;
                    if (token >= 0) {
                        const int position = position0 + token + pass, from = p.window > 0 ? max(position - p.window + 1, 0) : 0;
                        shown = 0;
#pragma unroll
                        for (int i = 0; i < TK; ++i) shown |= (key0 + i >= from && key0 + i <= position ? 1u : 0u) << i;
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) row_on[rt] = (row0 + rt * 8 + g) / group == token + pass ? 0xffffffffu : 0;
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float d[RT][4];
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) d[rt][0] = d[rt][1] = d[rt][2] = d[rt][3] = 0.0f;
#pragma unroll
                        for (int step = 0; step < TK / 16; ++step) {
                            uint32_t x[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint4 line = v[4 * step + i];
                                x[i] = j / 2 == 0 ? line.x : (j / 2 == 1 ? line.y : (j / 2 == 2 ? line.z : line.w));
                                if (token >= 0 && !(shown >> (16 * step + 2 * t4 + (i & 1) + 8 * (i >> 1)) & 1)) x[i] = 0;
                            }
                            const uint32_t b0 = __byte_perm(x[0], x[1], j & 1 ? 0x7632 : 0x5410), b1 = __byte_perm(x[2], x[3], j & 1 ? 0x7632 : 0x5410);
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) {
                                const uint32_t on = row_on[rt];
                                if (PARTS == 3) mma<TYPE>(d[rt], 0, w_lo[rt][(2 * step) % (PARTS == 3 ? NT : 1)] & on, 0, w_lo[rt][(2 * step + 1) % (PARTS == 3 ? NT : 1)] & on, b0, b1);
                                mma<TYPE>(d[rt], w_hi[rt][2 * step] & on, w_mid[rt][2 * step] & on, w_hi[rt][2 * step + 1] & on, w_mid[rt][2 * step + 1] & on, b0, b1);
                            }
                        }
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) {
                            const bool on = row_on[rt] != 0;
                            acc[rt][c][j] = fmaf(acc[rt][c][j], scaled[rt], on ? d[rt][0] + d[rt][2] : 0.0f);
                            acc[rt][c][8 + j] = fmaf(acc[rt][c][8 + j], scaled[rt], on ? d[rt][1] + d[rt][3] : 0.0f);
                        }
                    }
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) scaled[rt] = 1.0f;
                }
            }
            place = next_place;
        }

        // ---- the four warps' sums, and other CTAs' ------------------------------------------------------
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            sum[rt] += __shfl_xor_sync(0xffffffffu, sum[rt], 1);
            sum[rt] += __shfl_xor_sync(0xffffffffu, sum[rt], 2);
            if (t4 == 0) { warp_max[warp][rt * 8 + g] = m[rt]; warp_sum[warp][rt * 8 + g] = sum[rt]; }
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *(float4*)&out[warp][rt * 8 + g][64 * c + 16 * t4 + i] = make_float4(acc[rt][c][i], acc[rt][c][i + 1], acc[rt][c][i + 2], acc[rt][c][i + 3]);
        }
        __syncthreads();
        const int64_t first_cta = ((item_begin + 1) * ctas - 1) / total, last_cta = (item_end * ctas - 1) / total;
        const bool whole = first_cta == last_cta;
        const int64_t stride = ROWS * (D + 2);
        float* mine = p.partial + ((int64_t)blockIdx.x * 2 + (blockIdx.x == first_cta)) * stride;
        auto row_of = [&](int row) { const int at = row0 + row; return p.y + (int64_t)(p.starts[r] + at / group) * p.y_stride + (int64_t)(kv * group + at % group) * D; };
        auto put = [&](float* y, int e, float4 v, float total_weight) {
            const float inverse = total_weight == 0.0f ? 0.0f : 1.0f / total_weight;
            v.x *= inverse; v.y *= inverse; v.z *= inverse; v.w *= inverse;
            if (p.wide) *(float4*)(y + e) = v;
            else { y[e] = v.x; y[e + 1] = v.y; y[e + 2] = v.z; y[e + 3] = v.w; }
        };
        for (int i = tid; i < ROWS * (D / 4); i += kThreads) {
            const int row = i / (D / 4), e = 4 * (i % (D / 4));
            if (row >= rows) break;
            float top = warp_max[0][row];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) top = fmaxf(top, warp_max[w][row]);
            const float base = top == -INFINITY ? 0.0f : top;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float weight = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = exp2_fast(warp_max[w][row] - base);
                const float4 o = *(const float4*)&out[w][row][e];
                v.x = fmaf(o.x, f, v.x); v.y = fmaf(o.y, f, v.y); v.z = fmaf(o.z, f, v.z); v.w = fmaf(o.w, f, v.w);
                weight = fmaf(warp_sum[w][row], f, weight);
            }
            if (whole) {
                put(row_of(row), e, v, weight);
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
                for (int i = tid; i < ROWS * (D / 4); i += kThreads) {
                    const int row = i / (D / 4), e = 4 * (i % (D / 4));
                    if (row >= rows) break;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    float weight = 0.0f, top = -INFINITY;
#pragma unroll 8
                    for (int64_t c = first_cta; c <= last_cta; ++c) top = fmaxf(top, __ldcg(p.partial + (c * 2 + (c == first_cta)) * stride + ROWS * D + row));
                    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll 8
                    for (int64_t c = first_cta; c <= last_cta; ++c) {
                        const float* from = p.partial + (c * 2 + (c == first_cta)) * stride;
                        const float f = exp2_fast(__ldcg(from + ROWS * D + row) - base);
                        const float4 o = __ldcg((const float4*)(from + row * D + e));
                        v.x = fmaf(o.x, f, v.x); v.y = fmaf(o.y, f, v.y); v.z = fmaf(o.z, f, v.z); v.w = fmaf(o.w, f, v.w);
                        weight = fmaf(__ldcg(from + ROWS * D + ROWS + row), f, weight);
                    }
                    put(row_of(row), e, v, weight);
                }
            }
        }
        __syncthreads();  // the shared sums are free again
    }
}

// The work area: parts of rows for every CTA of the largest grid, and the counts of those that have left theirs
constexpr int kMostCtas = 148 * 4;
size_t partial_bytes() { return (size_t)kMostCtas * 2 * 16 * (256 + 2) * sizeof(float); }

int ensure_work_area(rq_ctx* ctx) {
    if (ctx->attn_scratch) return RQ_OK;
    if (ctx->recording) return rq_fail(RQ_ERR_INVALID, "a recorded rq_attention needs its work area: call rq_attention_reserve before rq_sequence_begin");
    const size_t bytes = partial_bytes() + kMostCtas * sizeof(uint32_t);
    uint8_t* area = nullptr;
    cudaError_t e = cudaMalloc(&area, bytes);
    if (e != cudaSuccess) return rq_fail(RQ_ERR_ALLOC, "attention's work area of %zu bytes: %s", bytes, cudaGetErrorString(e));
    e = cudaMemset(area + partial_bytes(), 0, kMostCtas * sizeof(uint32_t));
    if (e == cudaSuccess) e = cudaDeviceSynchronize();  // streams that do not wait for the default one may use it next
    if (e != cudaSuccess) { cudaFree(area); return rq_fail(RQ_ERR_CUDA, "attention's work area: %s", cudaGetErrorString(e)); }
    ctx->attn_scratch = area;
    return RQ_OK;
}

template <int D, int TYPE, int RT>
int launch_rows(rq_ctx* ctx, const AttentionParams& p, cudaStream_t s) {
    static int resident = 0;  // CTAs an SM holds
    auto kernel = rq_attention_rows_kernel<D, TYPE, RT>;
    const size_t smem = sizeof(Tiles<D, TYPE, RT>) + sizeof(int64_t) * ((size_t)p.requests + 1);
    if (!resident) {
        RQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(Tiles<D, TYPE, RT>) + sizeof(int64_t) * (RQ_MAX_REQUESTS + 1))));
        int n = 0;
        RQ_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, smem));
        resident = n < 1 ? 1 : (n > 4 ? 4 : n);
    }
    const int ctas = ctx->sm_count * resident;
    return launch(kernel, dim3((unsigned)(ctas < kMostCtas ? ctas : kMostCtas)), kThreads, smem, s, p);
}

template <int D>
int launch_rows(rq_ctx* ctx, const AttentionParams& p, int type, bool two, cudaStream_t s) {
    if (type == RQ_KV_F16) return two ? launch_rows<D, RQ_KV_F16, 2>(ctx, p, s) : launch_rows<D, RQ_KV_F16, 1>(ctx, p, s);
    return two ? launch_rows<D, RQ_KV_BF16, 2>(ctx, p, s) : launch_rows<D, RQ_KV_BF16, 1>(ctx, p, s);
}

}  // namespace

extern "C" int rq_attention_reserve(rq_ctx* ctx) {
    if (!ctx) return rq_fail(RQ_ERR_INVALID, "rq_attention_reserve: null context");
    DeviceGuard guard(ctx->device);
    return ensure_work_area(ctx);
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
    const int group = q_heads / cache->heads;
    if (group > 128) return rq_fail(RQ_ERR_LIMIT, "rq_attention: %d query heads share a key head; at most 128", group);
    DeviceGuard guard(ctx->device);
    cudaStream_t s = (cudaStream_t)stream;
    rc = ensure_work_area(ctx);
    if (rc) return rc;
    rc = rq_order_work_areas(ctx, s);
    if (rc) return rc;
    AttentionParams p = {};
    p.q = q; p.y = y; p.k = (const uint16_t*)cache->k; p.v = (const uint16_t*)cache->v; p.block_table = block_table; p.starts = starts; p.lengths = lengths;
    p.partial = (float*)ctx->attn_scratch; p.arrived = (uint32_t*)(ctx->attn_scratch + partial_bytes());
    p.q_stride = q_t_stride; p.y_stride = y_t_stride; p.table_stride = table_stride; p.page_stride = cache->page_stride; p.head_stride = cache->head_stride;
    p.line_stride = cache->line_stride; p.pages = cache->pages; p.tokens = tokens; p.requests = requests; p.q_heads = q_heads; p.kv_heads = cache->heads;
    p.table_width = table_width; p.window = window; p.scale = scale;
    p.wide = (((uintptr_t)q | (uintptr_t)y) & 15) == 0 && (tokens == 1 || ((q_t_stride | y_t_stride) & 3) == 0);
    while (1 << p.page_shift < cache->page_size) ++p.page_shift;
    // rows that meet a key together: eight, or sixteen where a request may have more
    const bool two = (int64_t)(max_fresh > 0 ? max_fresh : tokens) * group > 8;
    if (cache->head_dim == 64) return launch_rows<64>(ctx, p, cache->type, two, s);
    if (cache->head_dim == 128) return launch_rows<128>(ctx, p, cache->type, two, s);
    return launch_rows<256>(ctx, p, cache->type, two, s);
}
