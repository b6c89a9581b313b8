// Attention of new tokens over the paged cache.
//
//   y = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale * q . k_j - m),  over the keys j that the token sees
//
// rq_attention_rows_kernel, for up to sixteen rows (new tokens x the query heads that share a key head) at a time: a decode step. It is bound by the bytes of
// the cache, read once, so everything else is arranged around loads:
//   * a warp takes sixteen keys at a time through a ring of its own in shared memory, filled by 16-byte asynchronous copies a tile ahead: any
//     page size, order and stride, and what no row sees arrives as zeros. Chunks of a line are permuted (chunk ^ line % 8) so that
//     the matrix loads meet no bank twice. (Loads into registers instead, without shared memory, kept too little under way: 140 us for 131071 keys.)
//   * fp32 activations: queries and weights are taken apart into 16-bit parts, hi + lo over f16 (22 bits, a row of queries brought to f16's range by a power of two
//     first), hi + mid + lo over bf16 (24 bits). The sixteen rows of an operand are eight rows' hi parts above their lo parts: one mma.sync does both.
//   * The tensor core adds by truncation, a bias that grows with the length of a chain: a sum stays in it for one tile and is then added, with
//     round-to-nearest, to the row's fp32 sums, which are scaled by 2^(old base - new base) in the same multiply-add. A row's base is what its weights are made
//     against, its maximum less 12 (bf16: 0) as rounded: kept itself, the factor is exactly one where the base stays. (Of the maximum, and the 12 added and taken off
//     again, it was one rounding off on every tile, the same one: 64 requests of 32768 keys, flat heads of 128 elements, 4.2e-5 of a
//     head's outputs in place of 5e-7.)
//   * The keys of all requests and heads, in units of 64, are dealt out evenly: every CTA takes an equal range of units, wherever it begins and ends.
//     Rows whose units fall to several CTAs are joined, in CTA order, by whichever of these is the last to leave its sums: the same bits on every run.
// One token over 131071 keys, 32 + 2 x 8 heads of 128, f16: 94.5 us, 0.87 of the measured copy's bandwidth (another GPU 96.5); 64 requests of up to 8191 keys, bf16: 176 us, 0.93 (184).
#include <cmath>

#include "rq_attention_rows.cuh"

using namespace rqserve;
using namespace rqattn;
using rqmma::smem_u32;

namespace {

constexpr int kTile = 16, kUnit = kWarps * kTile;  // keys a warp and a CTA take at a time
constexpr int kStages = 2;  // of a warp's ring: one tile under way while the other is used

// c = (first ? 0 : c) + a b for sixteen rows, eight columns and sixteen products each
template <int TYPE> __device__ __forceinline__ void mma(float (&c)[4], bool first, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    const float c0 = first ? 0.0f : c[0], c1 = first ? 0.0f : c[1], c2 = first ? 0.0f : c[2], c3 = first ? 0.0f : c[3];
    if (TYPE == RQ_KV_F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
// acc = acc * f + d
__device__ __forceinline__ void add_scaled(float2 (&acc)[2], float f, const float (&d)[4]) {
    acc[0] = fma2(acc[0], make_float2(f, f), make_float2(d[0], d[1]));
    acc[1] = fma2(acc[1], make_float2(f, f), make_float2(d[2], d[3]));
}
// Whether a word's two 16-bit numbers are both finite
template <int TYPE> __device__ __forceinline__ bool finite2(uint32_t w) {
    const uint32_t e = TYPE == RQ_KV_F16 ? 0x7c00u : 0x7f80u;
    return (w & e) != e && ((w >> 16) & e) != e;
}

template <int D, int TYPE, int RT> struct Tiles {
    union {
        uint16_t ring[kWarps][kStages][2][kTile][D];  // keys, values
        float out[kWarps][8 * RT][D + 8];             // the warps' sums
    };
    uint4 q_hi[RT][D / 16][32];                           // operand registers of the queries: hi above lo (f16), hi above mid (bf16)
    uint2 q_lo[TYPE == RQ_KV_BF16 ? RT : 1][D / 16][32];  // the third parts
};

template <int D, int TYPE, int RT>
__global__ void __launch_bounds__(kThreads) rq_attention_rows_kernel(AttentionParams p) {
    constexpr int ROWS = 8 * RT, STEPS = D / 16, PARTS = TYPE == RQ_KV_F16 ? 2 : 3, CHUNKS = D / 8, LINES = 32 / CHUNKS > 0 ? 32 / CHUNKS : 1;
    extern __shared__ __align__(128) unsigned char dynamic[];
    Tiles<D, TYPE, RT>& sh = *(Tiles<D, TYPE, RT>*)dynamic;
    int64_t* before = (int64_t*)(dynamic + sizeof(sh));  // units before each request
    __shared__ float warp_base[kWarps][ROWS], warp_sum[kWarps][ROWS];
    __shared__ uint32_t row_largest[kWarps][ROWS];
    __shared__ int64_t sums[kWarps];
    __shared__ uint32_t last_arrival;
    launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int group = p.q_heads / p.kv_heads;
    wait_for_previous();

    const Deal deal = deal_units<ROWS, kTile>(p, before, sums);
    if (blockIdx.x >= deal.ctas) return;
    int64_t u = deal.begin;

    while (u < deal.end) {
        // the rows that unit u belongs to
        int r = 0;
        for (int hi = p.requests - 1; r < hi;) { const int mid = (r + hi + 1) >> 1; if (before[mid] <= u) r = mid; else hi = mid - 1; }
        const Request rq = request_of<ROWS, kTile>(p, r);
        const int64_t in_request = u - before[r], item = in_request / rq.units, first_unit = in_request % rq.units;
        const int kv = (int)(item % p.kv_heads), row0 = (int)(item / p.kv_heads) * ROWS, rows = min(ROWS, rq.here * group - row0);
        const int64_t item_begin = u - first_unit, item_end = item_begin + rq.units, stop = min(item_end, deal.end);
        const int key_first = rq.begin + (int)first_unit * kUnit, key_stop = min(rq.end, rq.begin + (int)(stop - item_begin) * kUnit);
        u = stop;

        // the keys that some row sees and that this thread's rows see: [low, high)
        int low[RT], high[RT];
        const int position0 = rq.length - rq.fresh, seen_high = min(key_stop, position0 + (row0 + max(rows, 1) - 1) / group + 1);
        const int seen_low = p.window > 0 ? max(0, position0 + row0 / group - p.window + 1) : 0;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int position = position0 + (row0 + rt * 8 + g) / group;
            high[rt] = rt * 8 + g < rows ? min(position + 1, rq.end) : 0;
            low[rt] = p.window > 0 ? max(position - p.window + 1, 0) : 0;
        }
        const bool one_token = row0 / group == (row0 + max(rows, 1) - 1) / group;

        const int32_t* table = p.block_table + r * p.table_stride;
        const int line_mask = (1 << p.page_shift) - 1, lane_chunk = lane % CHUNKS, lane_line = lane / CHUNKS;
        const char* k_lane = (const char*)(p.k + kv * p.head_stride + 8 * lane_chunk) + (int64_t)lane_line * p.line_bytes;
        const int64_t k_to_v = (const char*)p.v - (const char*)p.k;
        const uint32_t ring = smem_u32(&sh.ring[warp][0][0][0][0]);
        // where a tile's keys lie: lanes l and l + 16 find key l's page, -1 for a key that no row sees
        auto page_of = [&](int key0) -> int {
            const int key = key0 + (lane & 15);
            const int entry = key >= seen_low && key < seen_high ? __ldcg(table + (key >> p.page_shift)) : -1;
            return entry < p.pages ? max(entry, -1) : -1;
        };
        // A warp copies LINES lines an instruction, this lane one chunk of one of them
        const uint32_t stage_at = ring + lane_line * (D * 2);
        auto fetch = [&](int key0, int page, uint32_t seen, int stage) {
            const uint32_t to = stage_at + stage * (2 * kTile * D * 2);
            if (p.page_shift >= 4) {  // the tile's keys, sixteen of a multiple of sixteen, share a page
                const int first = __shfl_sync(0xffffffffu, page, seen ? __ffs(seen) - 1 : 0);
                const char* from = k_lane + (uint64_t)(uint32_t)max(first, 0) * p.page_bytes + (uint64_t)(uint32_t)(key0 & line_mask) * p.line_bytes;
#pragma unroll
                for (int i = 0; i < kTile / LINES; ++i) {
                    const uint32_t place = to + i * (LINES * D * 2) + ((lane_chunk ^ ((i * LINES + lane_line) & 7)) << 4);
                    const bool there = seen >> (i * LINES + lane_line) & 1;
                    copy16(place, from, there);
                    copy16(place + kTile * D * 2, from + k_to_v, there);
                    from += LINES * (uint64_t)p.line_bytes;
                }
            } else {
#pragma unroll
                for (int i = 0; i < kTile / LINES; ++i) {
                    const int line = i * LINES + lane_line, at = __shfl_sync(0xffffffffu, page, line);
                    const char* from = k_lane + (int64_t)max(at, 0) * p.page_bytes + ((int64_t)((key0 + line) & line_mask) - lane_line) * p.line_bytes;
                    const uint32_t place = to + i * (LINES * D * 2) + ((lane_chunk ^ (line & 7)) << 4);
                    copy16(place, from, at >= 0);
                    copy16(place + kTile * D * 2, from + k_to_v, at >= 0);
                }
            }
        };
        int key0 = key_first + warp * kTile, ahead = key0, stage = 0;
        int page = page_of(ahead);
        uint32_t seen = __ballot_sync(0xffffffffu, page >= 0) & 0xffff, seen_next = 0;  // the tile's keys that some row sees
        if (ahead < key_stop) fetch(ahead, page, seen, 0);
        copies_commit();
        ahead += kUnit;
        page = page_of(ahead);

        // queries: brought to one size (f16) and taken apart, as the tensor core's operand registers; a warp has every fourth step of all rows
        float factor[RT];  // of the scores of row g
        {
            constexpr int MINE = RT * STEPS / kWarps;
            float x[MINE][4];  // elements 16 step + 2 t4 + {0, 1, 8, 9}
            uint32_t largest[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) largest[rt] = 0;
#pragma unroll
            for (int n = 0; n < MINE; ++n) {
                const int rt = n * kWarps / STEPS, step = n * kWarps % STEPS + warp, row = rt * 8 + g;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[n][e] = 0.0f;
                if (row < rows) {
                    const int at = row0 + row;
                    const float* from = p.q + (int64_t)(p.starts[r] + at / group) * p.q_stride + (int64_t)(kv * group + at % group) * D + 16 * step + 2 * t4;
                    if (p.wide) {
                        const float2 v = __ldcg((const float2*)from), w = __ldcg((const float2*)(from + 8));
                        x[n][0] = v.x; x[n][1] = v.y; x[n][2] = w.x; x[n][3] = w.y;
                    } else { x[n][0] = __ldcg(from); x[n][1] = __ldcg(from + 1); x[n][2] = __ldcg(from + 8); x[n][3] = __ldcg(from + 9); }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) largest[rt] = max(largest[rt], __float_as_uint(x[n][e]) & 0x7fffffffu);
            }
            if (PARTS == 2) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    largest[rt] = max(largest[rt], __shfl_xor_sync(0xffffffffu, largest[rt], 1));
                    largest[rt] = max(largest[rt], __shfl_xor_sync(0xffffffffu, largest[rt], 2));
                    if (t4 == 0) row_largest[warp][rt * 8 + g] = largest[rt];
                }
                __syncthreads();
            }
            float raised[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                raised[rt] = 1.0f;
                factor[rt] = factor_of(p.scale, 0);
                if (PARTS == 2) {
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) largest[rt] = max(largest[rt], row_largest[w][rt * 8 + g]);
                    const int raise = raise_of(largest[rt]);
                    raised[rt] = power_of_two(raise);
                    factor[rt] = factor_of(p.scale, raise);
                }
            }
#pragma unroll
            for (int n = 0; n < MINE; ++n) {
                const int rt = n * kWarps / STEPS, step = n * kWarps % STEPS + warp;
                if (PARTS == 2)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][e] *= raised[rt];
                uint4 a;
                a.x = take_pair<TYPE>(x[n][0], x[n][1]);
                a.z = take_pair<TYPE>(x[n][2], x[n][3]);
                a.y = take_pair<TYPE>(x[n][0], x[n][1]);
                a.w = take_pair<TYPE>(x[n][2], x[n][3]);
                sh.q_hi[rt][step][lane] = a;
                if (PARTS == 3) sh.q_lo[PARTS == 3 ? rt : 0][step][lane] = make_uint2(pair_of<TYPE>(x[n][0], x[n][1]), pair_of<TYPE>(x[n][2], x[n][3]));
            }
        }
        __syncthreads();

        float base[RT], sum[RT];  // base: -inf while the row has seen no key
        float2 acc[RT][D / 8][2];  // sums of the hi parts, and of the parts below them
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            base[rt] = -INFINITY;
            sum[rt] = 0.0f;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) acc[rt][n][0] = acc[rt][n][1] = make_float2(0.0f, 0.0f);
        }
        for (; key0 < key_stop; key0 += kUnit, stage ^= 1, seen = seen_next) {
            const uint32_t keys = ring + stage * (2 * kTile * D * 2), values = keys + kTile * D * 2;
            __syncwarp();  // the other stage has been read
            seen_next = __ballot_sync(0xffffffffu, page >= 0) & 0xffff;
            if (ahead < key_stop) fetch(ahead, page, seen_next, stage ^ 1);
            copies_commit();
            ahead += kUnit;
            page = page_of(ahead);
            copies_wait<1>();
            __syncwarp();
            // scores: of keys 8 i + 2 t4 + {0, 1} and row g
            float s[RT][2][2];
            {
                float c[RT][2][4];
                const int line = (lane & 7) + (lane & 16 ? 8 : 0), half = lane >> 3 & 1;
#pragma unroll
                for (int step = 0; step < STEPS; ++step) {
                    uint32_t b[4];
                    ldmatrix(b, keys + line * (D * 2) + (((2 * step + half) ^ (line & 7)) << 4));
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const uint4 a = sh.q_hi[rt][step][lane];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            mma<TYPE>(c[rt][i], step == 0, a.x, a.y, a.z, a.w, b[2 * i], b[2 * i + 1]);
                            if (PARTS == 3) {
                                const uint2 lo = sh.q_lo[PARTS == 3 ? rt : 0][step][lane];
                                mma<TYPE>(c[rt][i], false, 0, lo.x, 0, lo.y, b[2 * i], b[2 * i + 1]);  // into the rows of the small parts
                            }
                        }
                    }
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) { s[rt][i][0] = c[rt][i][0] + c[rt][i][2]; s[rt][i][1] = c[rt][i][1] + c[rt][i][3]; }
            }
            // weights
            uint32_t w_hi[RT][2], w_mid[RT][2], w_lo[RT][2];
            float old[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int at = 8 * i + 2 * t4 + e, key = key0 + at;
                        if (key < low[rt] || key >= high[rt] || !(seen >> at & 1)) s[rt][i][e] = -INFINITY;
                        top = fmaxf(top, s[rt][i][e]);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                top = fmaxf(base[rt], fmaf(top, factor[rt], -kRaise<TYPE>));
                const float from = top == -INFINITY ? 0.0f : top;
                old[rt] = exp2_fast(base[rt] - from);
                base[rt] = top;
                float add = 0.0f;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float a = exp2_fast(fmaf(s[rt][i][0], factor[rt], -from)), b = exp2_fast(fmaf(s[rt][i][1], factor[rt], -from));
                    add += a + b;
                    w_hi[rt][i] = take_pair<TYPE>(a, b);
                    w_mid[rt][i] = take_pair<TYPE>(a, b);
                    w_lo[rt][i] = PARTS == 3 ? pair_of<TYPE>(a, b) : 0;
                }
                sum[rt] = fmaf(sum[rt], old[rt], add);
            }
            // A value that one row must not see may be infinite, and 0 * inf is no 0. Where a tile's rows do not see the same keys and a value
            // is not finite, the rows of each token meet the values by themselves, the unseen ones taken out.
            const int value_line = (lane & 7) + (lane & 8), value_half = lane >> 4;
            auto load_values = [&](int n2, uint32_t (&b)[4]) { ldmatrix_transposed(b, values + value_line * (D * 2) + (((2 * n2 + value_half) ^ (value_line & 7)) << 4)); };
            const int first_token = row0 / group, tokens = (row0 + max(rows, 1) - 1) / group - first_token + 1;
            bool apart = false;
            if (!one_token && (key0 < seen_low + tokens || key0 + kTile > position0 + first_token + 1)) {
                bool fine = true;
#pragma unroll
                for (int n2 = 0; n2 < D / 16; ++n2) {
                    uint32_t b[4];
                    load_values(n2, b);
                    fine = fine && finite2<TYPE>(b[0]) && finite2<TYPE>(b[1]) && finite2<TYPE>(b[2]) && finite2<TYPE>(b[3]);
                }
                apart = !__all_sync(0xffffffffu, fine);
            }
            if (!apart) {
#pragma unroll
                for (int n2 = 0; n2 < D / 16; ++n2) {
                    uint32_t b[4];
                    load_values(n2, b);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float d[4];
                            mma<TYPE>(d, true, w_hi[rt][0], w_mid[rt][0], w_hi[rt][1], w_mid[rt][1], b[2 * i], b[2 * i + 1]);
                            if (PARTS == 3) mma<TYPE>(d, false, 0, w_lo[rt][0], 0, w_lo[rt][1], b[2 * i], b[2 * i + 1]);
                            add_scaled(acc[rt][2 * n2 + i], old[rt], d);
                        }
                }
            } else {
                for (int token = first_token; token < first_token + tokens; ++token) {
                    const int position = position0 + token, from = p.window > 0 ? position - p.window + 1 : 0;
                    uint32_t shown[2];  // the words of keys 8 i + 2 t4 + {0, 1}
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int key = key0 + 8 * i + 2 * t4;
                        shown[i] = (key >= from && key <= position ? 0xffffu : 0) | (key + 1 >= from && key + 1 <= position ? 0xffff0000u : 0);
                    }
#pragma unroll
                    for (int n2 = 0; n2 < D / 16; ++n2) {
                        uint32_t b[4];
                        load_values(n2, b);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                float d[4];
                                const uint32_t b0 = b[2 * i] & shown[0], b1 = b[2 * i + 1] & shown[1];
                                mma<TYPE>(d, true, w_hi[rt][0], w_mid[rt][0], w_hi[rt][1], w_mid[rt][1], b0, b1);
                                if (PARTS == 3) mma<TYPE>(d, false, 0, w_lo[rt][0], 0, w_lo[rt][1], b0, b1);
                                if ((row0 + rt * 8 + g) / group != token) continue;
                                add_scaled(acc[rt][2 * n2 + i], old[rt], d);
                            }
                    }
                }
            }
        }
        copies_wait<0>();
        __syncthreads();  // the sums go where the ring was

        // ---- the four warps' sums, and other CTAs' ------------------------------------------------------
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            sum[rt] += __shfl_xor_sync(0xffffffffu, sum[rt], 1);
            sum[rt] += __shfl_xor_sync(0xffffffffu, sum[rt], 2);
            if (t4 == 0) { warp_base[warp][rt * 8 + g] = base[rt]; warp_sum[warp][rt * 8 + g] = sum[rt]; }
#pragma unroll
            for (int n = 0; n < D / 8; ++n) *(float2*)&sh.out[warp][rt * 8 + g][8 * n + 2 * t4] = make_float2(acc[rt][n][0].x + acc[rt][n][1].x, acc[rt][n][0].y + acc[rt][n][1].y);
        }
        __syncthreads();
        join_rows<D, ROWS>(p, &sh.out[0][0][0], warp_base, warp_sum, item_begin, item_end, deal, p.starts[r], row0, rows, kv, last_arrival);
        __syncthreads();  // the shared sums are free again
    }
}

int ensure_work_area(rq_ctx* ctx) {
    if (ctx->attn_scratch) return RQ_OK;
    if (ctx->recording) return rq_fail(RQ_ERR_INVALID, "a recorded rq_attention needs its work area: call rq_attention_reserve before rq_sequence_begin");
    const size_t bytes = kPartialBytes + kCounts * sizeof(uint32_t);
    uint8_t* area = nullptr;
    cudaError_t e = cudaMalloc(&area, bytes);
    if (e != cudaSuccess) return rq_fail(RQ_ERR_ALLOC, "attention's work area of %zu bytes: %s", bytes, cudaGetErrorString(e));
    e = cudaMemset(area + kPartialBytes, 0, kCounts * sizeof(uint32_t));
    if (e == cudaSuccess) e = cudaDeviceSynchronize();  // streams that do not wait for the default one may use it next
    if (e != cudaSuccess) { cudaFree(area); return rq_fail(RQ_ERR_CUDA, "attention's work area: %s", cudaGetErrorString(e)); }
    ctx->attn_scratch = area;
    return RQ_OK;
}

template <int D, int TYPE, int RT>
int launch_rows(rq_ctx* ctx, const AttentionParams& p, cudaStream_t s) {
    auto kernel = rq_attention_rows_kernel<D, TYPE, RT>;
    // The grid decides where rows are cut, and with it the last bits: it follows from the call alone. Shared memory holds eight bytes a request, by steps of 128 of them.
    const int step = (p.requests + kRequestStep - 1) / kRequestStep, dev = ctx->device;
    auto bytes = [](int steps) { return sizeof(Tiles<D, TYPE, RT>) + sizeof(int64_t) * ((size_t)steps * kRequestStep + 1); };
    constexpr int kSteps = RQ_MAX_REQUESTS / kRequestStep;
    static uint8_t resident[64][kSteps + 1] = {};  // by device: CTAs an SM holds; 0: not known yet
    int n = dev < 64 ? resident[dev][step] : 0;
    if (!n) {
        RQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes(kSteps)));
        RQ_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, bytes(step)));
        n = n < 1 ? 1 : (n > 4 ? 4 : n);
        if (dev < 64) resident[dev][step] = (uint8_t)n;
    }
    const int ctas = ctx->sm_count * n;
    return launch(kernel, dim3((unsigned)(ctas < kRowCtas ? ctas : kRowCtas)), kThreads, bytes(step), s, p);
}

// two: sixteen rows at a time. Not for 256 elements a head, whose sums of sixteen rows do not fit a thread's registers: 16 requests of eight tokens over 8192 keys, 8 + 2 x 4
// heads, f16, 240 us by sixteen rows and 178 by eight; 509 tokens over 7680, 16 + 2 x 4 heads, 1460 and 998.
template <int D>
int launch_rows(rq_ctx* ctx, const AttentionParams& p, int type, bool two, cudaStream_t s) {
    constexpr int MOST = D < 256 ? 2 : 1;
    if (type == RQ_KV_F16) return two ? launch_rows<D, RQ_KV_F16, MOST>(ctx, p, s) : launch_rows<D, RQ_KV_F16, 1>(ctx, p, s);
    return two ? launch_rows<D, RQ_KV_BF16, MOST>(ctx, p, s) : launch_rows<D, RQ_KV_BF16, 1>(ctx, p, s);
}
int launch_rows_of(rq_ctx* ctx, const CodesParams& p, const rq_kv_cache& cache, bool two, cudaStream_t s) {
    if (cache.type == RQ_KV_INT8) return launch_rows_int8(ctx, p, cache, two, s);
    if (cache.head_dim == 64) return launch_rows<64>(ctx, p, cache.type, two, s);
    if (cache.head_dim == 128) return launch_rows<128>(ctx, p, cache.type, two, s);
    return launch_rows<256>(ctx, p, cache.type, two, s);
}

}  // namespace

int rq_attention_forget(rq_ctx* ctx) {
    if (ctx->attn_scratch) RQ_CUDA(cudaMemset(ctx->attn_scratch + kPartialBytes, 0, kCounts * sizeof(uint32_t)));
    return RQ_OK;
}

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
    CodesParams p = {};
    p.q = q; p.y = y; p.k = (const uint16_t*)cache->k; p.v = (const uint16_t*)cache->v; p.block_table = block_table; p.starts = starts; p.lengths = lengths;
    p.partial = (float*)ctx->attn_scratch; p.arrived = (uint32_t*)(ctx->attn_scratch + kPartialBytes);
    p.q_stride = q_t_stride; p.y_stride = y_t_stride; p.table_stride = table_stride; p.head_stride = cache->head_stride; p.pages = cache->pages; p.tokens = tokens; p.requests = requests; p.q_heads = q_heads; p.kv_heads = cache->heads;
    p.table_width = table_width; p.window = window; p.scale = scale; p.page_bytes = (uint32_t)(2 * cache->page_stride); p.line_bytes = (uint32_t)(2 * cache->line_stride);
    auto aligned = [&](int bytes) { return (((uintptr_t)q | (uintptr_t)y) & (bytes - 1)) == 0 && (tokens == 1 || ((q_t_stride | y_t_stride) & (bytes / 4 - 1)) == 0); };
    p.wide = (aligned(16) ? 1 : 0) | (aligned(32) ? 2 : 0);
    while (1 << p.page_shift < cache->page_size) ++p.page_shift;
    p.error_flag = ctx->error_flag; p.wait_ns = ctx->wait_limit_ns;
    if (cache->type == RQ_KV_INT8) {
        p.page_bytes = (uint32_t)cache->page_stride; p.line_bytes = (uint32_t)cache->line_stride;
        p.k_scale = cache->k_scale; p.v_scale = cache->v_scale;
        p.scale_page = cache->scale_page_stride; p.scale_head = cache->scale_head_stride; p.scale_line = cache->scale_line_stride;
        p.scale_size = (float)(2.0 * frexp((double)scale * (double)kLog2e, &p.scale_exponent));
        --p.scale_exponent;
    }
    const int64_t rows = (int64_t)(max_fresh > 0 ? (max_fresh < tokens ? max_fresh : tokens) : tokens) * group;
    // The rows kernel reads a request's keys once for every sixteen rows (from L2, from the second time on), the tensor-core kernel makes scores of 128 whatever
    // there is. 8192 cached keys, 32 + 2 x 8 heads of 128, f16, rows kernel | tensor cores: 16 requests of 16 rows 102 | 217 us, 32 rows 180 | 219, 48 rows 259 | 219,
    // 128 rows 656 | 209; one request of 32 rows 35 | 44, 48 rows 39 | 44, 128 rows 71 | 45. bf16: 16 requests of 32 rows 265 | 371, 48 rows 407 | 373.
    // Over codes, whose widening the tensor-core kernel repeats for every 128 or 256 rows: 16 requests of 32 rows 143 | 206, 48 rows 213 | 206, 64 rows 285 | 207; one request of 48 rows 34 | 49, 64
    // rows 33 | 49, 128 rows 52 | 50; 64 elements a head, 16 requests of 48 rows 123 | 177, 64 rows 157 | 177.
    if (rows > (cache->type == RQ_KV_INT8 ? 48 : 32)) {
        // Where a request may be a decode step among prompts, the rows kernel takes those and the tensor-core kernel the rest: 63 decode steps over 4096 keys and
        // a chunk of 512 are 267 us in two launches, 509 by the tensor cores alone, 531 by the rows kernel alone; 7 over 300 keys and a prompt of 100: 33, 27, 22.
        const int few = requests > 1 && tokens < requests * (rows / group) ? (group <= 8 ? 8 : 32) : 0;
        p.few = group <= few ? few : 0;
        rc = launch_tensor(ctx, p, *cache, rows <= 128, s);
        if (rc != RQ_ERR_UNSUPPORTED && (rc != RQ_OK || !p.few)) return rc;
        if (rc == RQ_OK) return launch_rows_of(ctx, p, *cache, group > 8, s);
    }
    p.few = 0x7fffffff;
    // rows that meet a key together: eight, or sixteen where a request may have more
    return launch_rows_of(ctx, p, *cache, rows > 8, s);
}
