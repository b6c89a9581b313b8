// Attention of a few rows at a time (decode steps) over a cache of 8-bit codes with a scale for each position's head:
//
//   y = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale * q . k_j - m),  k_j = sk_j ck_j,  v_j = sv_j cv_j
//
// The form of rq_attention.cu's kernel: a warp takes its keys through a ring of its own in shared memory, queries and weights are taken apart into parts that mma.sync takes,
// sums are added up in fp32. What differs, since a tile is half the bytes:
//   * Scores are products of bytes: a query is a whole number of 32 bits (of its row's step, a power of two), four digits of eight bits; the sixteen rows of an operand are eight
//     rows' first digits above their second ones, or third above fourth. Sums are exact, and joined and multiplied by factor and key's scale in fp32.
//   * The elements of a product's thirty-two may be any, if the queries' are the same: a thread's operands of two steps are sixteen neighbouring codes of a key, one 16-byte load.
//   * Values become f16 numbers on their way into operand registers, exactly (a byte permute and a subtraction a pair), weights times their scales hi + lo f16 parts. A transposing
//     matrix load moves pairs of neighbouring elements: the even ones make one column of the product, the odd ones the next.
//   * A warp's tile is 32 keys (16 for heads of 256): the same bytes on their way as there, and half the work on sums for each key. A lane brings its key's scales through registers.
//   * A row's base is the largest score plus its value's scale's exponent, less 12: hi parts of weight * sv lie below 2^13 whatever the scales are.
// Bound by the bytes of the cache while the loop runs (at 7 TB/s of reading), and by both ends of a launch: the first tiles 4 to 5 us after its beginning, CTAs that are done 4 us apart, and
// 3 to 8 us for the parts of rows. One token over 131071 keys, 32 + 2 x 8 heads of 128: 57.4 us, 0.74 of the measured copy's bandwidth (f16: 94); 64 requests of up to 8191 keys: 111 us, 0.76
// (bf16: 185); one token over 1001 keys 9.4 (in a recorded sequence 9.0). With scores of f16 numbers too (as values are taken), 1130 instructions a tile in place of 750, 80 and 143 us.
#include <type_traits>

#include "rq_attention_rows.cuh"
#include "rq_pairs.cuh"

using namespace rqserve;
using namespace rqattn;
using rqmma::smem_u32;

namespace {

// c = (first ? 0 : c) + a b for sixteen rows, eight columns and sixteen products each
__device__ __forceinline__ void mma(float (&c)[4], bool first, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    const float c0 = first ? 0.0f : c[0], c1 = first ? 0.0f : c[1], c2 = first ? 0.0f : c[2], c3 = first ? 0.0f : c[3];
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
// the same over bytes: thirty-two products each, exact
__device__ __forceinline__ void mma(int (&c)[4], bool first, uint4 a, uint32_t b0, uint32_t b1) {
    const int c0 = first ? 0 : c[0], c1 = first ? 0 : c[1], c2 = first ? 0 : c[2], c3 = first ? 0 : c[3];
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}
// Queries as whole numbers of 32 bits, n = 2^24 d0 + 2^16 d1 + 2^8 d2 + d3 with digits of -128 .. 127: |n| < 2^30, a row's largest element at least 2^29 (a power of two
// brings it there; one below 2^-126 stays below, exactly)
__device__ __forceinline__ int digits_raise(uint32_t largest) { return 156 - (int)(largest >> 23); }  // from -99 to 156: in two steps
// byte i of a word: digit of x[i]
__device__ __forceinline__ void take_digits(const int (&n)[4], uint32_t (&digit)[4]) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = ((uint32_t)n[i] + 0x00808080u) ^ 0x00808080u;  // (carries go up, a byte of 128 and more is the digit less 256)
    const uint32_t x = __byte_perm(b[0], b[1], 0x5140), y = __byte_perm(b[2], b[3], 0x5140), z = __byte_perm(b[0], b[1], 0x7362), w = __byte_perm(b[2], b[3], 0x7362);
    digit[3] = __byte_perm(x, y, 0x5410); digit[2] = __byte_perm(x, y, 0x7632); digit[1] = __byte_perm(z, w, 0x5410); digit[0] = __byte_perm(z, w, 0x7632);
}

// Taking up the rows of a request and head (their queries, the first tile, the sums at the end) costs a CTA as much as some units: so many lead each one's own in the dealing
// (64 requests of up to 8191 keys: none 119 us, one 115, two 112, four 113).
constexpr int kLead = 2;

template <int D> struct Form {
    static constexpr int TILE = D == 256 ? 16 : 32, STAGES = 2;  // keys a warp takes at a time; tiles of its ring
    static constexpr int CHUNKS = D / 16, LINES = 32 / CHUNKS;   // 16-byte pieces of a line; lines that a warp copies an instruction
    static constexpr int STAGE = 2 * TILE * D;                   // bytes: keys, values
};
// Where a line's pieces lie, so that neither eight lines' same piece (matrix loads) nor four pieces each of two lines meet a bank twice
template <int D> __device__ __forceinline__ int placed(int line, int chunk) { return chunk ^ (D == 64 ? line >> 1 & 3 : (line & 1) << 2 | (line >> 1 & 3)); }

// a / b, neither negative: mostly small ones
__device__ __forceinline__ int64_t divided(int64_t a, int64_t b) { return ((uint64_t)a | (uint64_t)b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b); }

template <int D, int RT> struct Tiles {
    union {
        struct {
            uint8_t codes[kWarps][Form<D>::STAGES][2][Form<D>::TILE][D];
        };
        float out[kWarps][8 * RT][D + 8];  // the warps' sums
    };
    uint4 q[RT][D / 32][2][32];                // operand registers of the queries: first digits above second, third above fourth
    float scales[kWarps][3][Form<D>::TILE];   // of a warp's tile: of the keys, of the values, and these's exponents
};

// CTAs that an SM holds, by what their shared memory and their sums in registers leave room for
template <int D, int RT> constexpr int kResident = D == 256 || (D == 128 && RT == 2) ? 2 : (D == 64 && RT == 1 ? 4 : 3);

template <int D, int RT>
__global__ void __launch_bounds__(kThreads, kResident<D, RT>) rq_attention_int8_kernel(CodesParams p) {
    using F = Form<D>;
    constexpr int ROWS = 8 * RT, STEPS = D / 32, TILE = F::TILE, UNIT = kWarps * TILE, NT = TILE / 8, LINES = F::LINES;
    constexpr uint32_t ALL = TILE == 32 ? 0xffffffffu : 0xffffu;
    extern __shared__ __align__(128) unsigned char dynamic[];
    Tiles<D, RT>& sh = *(Tiles<D, RT>*)dynamic;
    int64_t* before = (int64_t*)(dynamic + sizeof(sh));  // units before each request
    __shared__ float warp_base[kWarps][ROWS], warp_sum[kWarps][ROWS];
    __shared__ uint32_t row_largest[kWarps][ROWS];
    __shared__ int64_t sums[kWarps];
    __shared__ uint32_t last_arrival;
    launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int group = p.q_heads / p.kv_heads;
    wait_for_previous();

    const Deal deal = deal_units<ROWS, TILE, kLead>(p, before, sums);
    if (blockIdx.x >= deal.ctas) return;
    int64_t u = deal.begin;

    while (u < deal.end) {
        // the rows that unit u belongs to
        int r = 0;
        for (int hi = p.requests - 1; r < hi;) { const int mid = (r + hi + 1) >> 1; if (before[mid] <= u) r = mid; else hi = mid - 1; }
        const Request rq = request_of<ROWS, TILE>(p, r);
        const int64_t in_request = u - before[r], item_units = kLead + rq.units, item = divided(in_request, item_units), item_begin = before[r] + item * item_units, item_end = item_begin + item_units;
        const int64_t tile = divided(item, p.kv_heads), stop = min(item_end, deal.end);
        const int kv = (int)(item - tile * p.kv_heads), row0 = (int)tile * ROWS, rows = min(ROWS, rq.here * group - row0), offset = (int)(u - item_begin), first_unit = max(offset - kLead, 0);
        const int units = (int)(stop - item_begin) - kLead - first_unit;
        u = stop;
        if (units <= 0) continue;  // (a range that ends in the lead: the next CTA has it all)
        const int key_first = rq.begin + first_unit * UNIT, key_stop = min(rq.end, key_first + units * UNIT), start = p.starts[r];

        // the queries, on their way while the first keys are found
        constexpr int MINE = (RT * STEPS + kWarps - 1) / kWarps;
        float x[MINE][8];
#pragma unroll
        for (int n = 0; n < MINE; ++n) {
            const int of = n * kWarps + warp, step = of % STEPS, row = of / STEPS * 8 + g;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[n][e] = 0.0f;
            if (of < RT * STEPS && row < rows) {
                const int at = row0 + row;
                const float* from = p.q + (int64_t)(start + at / group) * p.q_stride + (int64_t)(kv * group + at % group) * D + 64 * (step >> 1) + 16 * t4 + 8 * (step & 1);
                if (p.wide) {
                    const float4 v = __ldcg((const float4*)from), w = __ldcg((const float4*)from + 1);
                    x[n][0] = v.x; x[n][1] = v.y; x[n][2] = v.z; x[n][3] = v.w; x[n][4] = w.x; x[n][5] = w.y; x[n][6] = w.z; x[n][7] = w.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[n][e] = __ldcg(from + e);
                }
            }
        }

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

        const int32_t* table = p.block_table + r * p.table_stride;
        const int line_mask = (1 << p.page_shift) - 1, lane_chunk = lane % F::CHUNKS, lane_line = lane / F::CHUNKS, lane_key = lane & (TILE - 1);
        const char* k_lane = (const char*)p.k + kv * p.head_stride + 16 * lane_chunk;
        const int64_t k_to_v = (const char*)p.v - (const char*)p.k;
        const float *k_scale = p.k_scale + kv * p.scale_head, *v_scale = p.v_scale + kv * p.scale_head;
        const uint32_t ring = smem_u32(&sh.codes[warp][0][0][0][0]);
        // the keys that every row sees
        const int every_high = min(key_stop, position0 + row0 / group + 1);
        const int every_low = p.window > 0 ? position0 + (row0 + max(rows, 1) - 1) / group - p.window + 1 : 0;
        // where a tile's keys lie: lane l finds key l's page, -1 for a key that no row sees
        auto page_of = [&](int key0) -> int {
            const int key = key0 + lane_key;
            const int entry = key >= seen_low && key < seen_high ? __ldcg(table + (key >> p.page_shift)) : -1;
            return entry < p.pages ? max(entry, -1) : -1;
        };
        // A warp copies LINES lines an instruction, this lane one piece of one of them
        const bool plain = p.page_shift >= 4 && p.line_bytes == D;
        auto fetch = [&](int key0, int page, uint32_t seen, int stage) {
            const uint32_t to = ring + stage * F::STAGE + lane_line * D;
            if (plain && seen == ALL) {  // nothing but the pages' addresses changes from tile to tile
#pragma unroll
                for (int half = 0; half < TILE / 16; ++half) {
                    const int at = __shfl_sync(0xffffffffu, page, 16 * half);
                    const char* from = k_lane + (uint64_t)(uint32_t)at * p.page_bytes + (uint32_t)((((key0 + 16 * half) & line_mask) + lane_line) * D);
                    const char* values_from = from + k_to_v;
#pragma unroll
                    for (int i = 0; i < 16 / LINES; ++i) {
                        const uint32_t place = to + (16 * half + i * LINES) * D + (placed<D>(i * LINES + lane_line, lane_chunk) << 4);
                        copy16(place, from + i * LINES * D, true);
                        copy16(place + TILE * D, values_from + i * LINES * D, true);
                    }
                }
                return;
            }
#pragma unroll
            for (int half = 0; half < TILE / 16; ++half) {
                if (p.page_shift >= 4) {  // sixteen keys of a multiple of sixteen share a page
                    const uint32_t here = seen >> (16 * half) & 0xffffu;
                    const int first = __shfl_sync(0xffffffffu, page, 16 * half + (here ? __ffs(here) - 1 : 0));
                    const char* from = k_lane + (uint64_t)(uint32_t)max(first, 0) * p.page_bytes + (uint64_t)(uint32_t)(((key0 + 16 * half) & line_mask) + lane_line) * p.line_bytes;
#pragma unroll
                    for (int i = 0; i < 16 / LINES; ++i) {
                        const int line = 16 * half + i * LINES;
                        const uint32_t place = to + line * D + (placed<D>(line + lane_line, lane_chunk) << 4);
                        const bool there = seen >> (line + lane_line) & 1;
                        copy16(place, from, there);
                        copy16(place + TILE * D, from + k_to_v, there);
                        from += LINES * (uint64_t)p.line_bytes;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16 / LINES; ++i) {
                        const int line = 16 * half + i * LINES + lane_line, at = __shfl_sync(0xffffffffu, page, line);
                        const char* from = k_lane + (uint64_t)(uint32_t)max(at, 0) * p.page_bytes + (uint64_t)(uint32_t)((key0 + line) & line_mask) * p.line_bytes;
                        const uint32_t place = to + (line - lane_line) * D + (placed<D>(line, lane_chunk) << 4);
                        copy16(place, from, at >= 0);
                        copy16(place + TILE * D, from + k_to_v, at >= 0);
                    }
                }
            }
        };
        // a lane's key's scales
        float key_scale = 0.0f, value_scale = 0.0f;
        auto load_scales = [&](int key0, int page) {
            const int64_t at = (int64_t)page * p.scale_page + (int64_t)((key0 + lane_key) & line_mask) * p.scale_line;
            key_scale = page >= 0 ? __ldcg(k_scale + at) : 0.0f;
            value_scale = page >= 0 ? __ldcg(v_scale + at) : 0.0f;
        };
        int key0 = key_first + warp * TILE, ahead = key0, stage = 0;
        int page = page_of(ahead);
        uint32_t seen = __ballot_sync(0xffffffffu, page >= 0) & ALL, seen_next = 0;  // the tile's keys that some row sees
        if (ahead < key_stop) fetch(ahead, page, seen, 0);
        copies_commit();
        load_scales(ahead, page);
        ahead += UNIT;
        page = page_of(ahead);

        // queries: brought to one size and taken apart, as the tensor core's operand registers (a thread's of step 2 j + i: elements 64 j + 16 t4 + 8 i + 0 .. 7); a warp
        // has every fourth step of all rows
        float lift[RT], factor[RT];  // of the sums of row g, and of their products with keys' scales
        {
            uint32_t largest[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) largest[rt] = 0;
#pragma unroll
            for (int n = 0; n < MINE; ++n)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    if ((n * kWarps + warp) / STEPS == rt)
#pragma unroll
                        for (int e = 0; e < 8; ++e) largest[rt] = max(largest[rt], __float_as_uint(x[n][e]) & 0x7fffffffu);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                largest[rt] = max(largest[rt], __shfl_xor_sync(0xffffffffu, largest[rt], 1));
                largest[rt] = max(largest[rt], __shfl_xor_sync(0xffffffffu, largest[rt], 2));
                if (t4 == 0) row_largest[warp][rt * 8 + g] = largest[rt];
            }
            __syncthreads();
            float raised[RT], more[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                for (int w = 0; w < kWarps; ++w) largest[rt] = max(largest[rt], row_largest[w][rt * 8 + g]);
                const int raise = digits_raise(largest[rt]);
                raised[rt] = power_of_two(min(raise, 126));
                more[rt] = power_of_two(max(raise - 126, 0));
                const PowerParts parts = power_parts(p.scale_size, p.scale_exponent - raise);
                lift[rt] = parts.first;
                factor[rt] = parts.rest;
            }
#pragma unroll
            for (int n = 0; n < MINE; ++n) {
                const int item = n * kWarps + warp, rt = item / STEPS, step = item % STEPS;
                if (item >= RT * STEPS) break;
                const float f = RT == 2 && rt ? raised[RT - 1] : raised[0], f2 = RT == 2 && rt ? more[RT - 1] : more[0];
                uint32_t d[2][4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    int whole[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) whole[i] = __float2int_rn(x[n][4 * e + i] * f * f2);
                    take_digits(whole, d[e]);
                }
                sh.q[rt][step][0][lane] = make_uint4(d[0][0], d[0][1], d[1][0], d[1][1]);
                sh.q[rt][step][1][lane] = make_uint4(d[0][2], d[0][3], d[1][2], d[1][3]);
            }
        }
        __syncthreads();

        float base[RT], sum[RT];  // base: -inf while the row has seen no key
        Pair acc[RT][D / 8];      // elements 16 c + 4 t4 + {0, 2} (2 c), + {1, 3} (2 c + 1)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            base[rt] = -INFINITY;
            sum[rt] = 0.0f;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) acc[rt][n] = ::pair_of(0.0f, 0.0f);
        }
        for (; key0 < key_stop; key0 += UNIT, stage = stage + 1 == F::STAGES ? 0 : stage + 1, seen = seen_next) {
            const uint32_t keys = ring + stage * F::STAGE, values = keys + TILE * D;
            __syncwarp();  // the other stage, and the scales, have been read
            if (TILE == 32 || lane < TILE) {
                sh.scales[warp][0][lane_key] = key_scale;
                sh.scales[warp][1][lane_key] = value_scale;
                sh.scales[warp][2][lane_key] = exponent_of(value_scale);
            }
            seen_next = __ballot_sync(0xffffffffu, page >= 0) & ALL;
            if (ahead < key_stop) fetch(ahead, page, seen_next, stage ^ 1);
            copies_commit();
            load_scales(ahead, page);
            ahead += UNIT;
            page = page_of(ahead);
            copies_wait<1>();
            __syncwarp();
            // scores: of keys 8 i + 2 t4 + {0, 1} and row g
            float s[RT][NT][2];
            {
                int c[RT][NT][2][4];
#pragma unroll
                for (int j = 0; j < D / 64; ++j) {
                    uint4 w[NT];
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        const uint32_t from = keys + (8 * i + g) * D + (placed<D>(8 * i + g, 4 * j + t4) << 4);
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w) : "r"(from) : "memory");
                    }
#pragma unroll
                    for (int step = 0; step < 2; ++step)
#pragma unroll
                        for (int part = 0; part < 2; ++part)
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) {
                                const uint4 a = sh.q[rt][2 * j + step][part][lane];
#pragma unroll
                                for (int i = 0; i < NT; ++i) mma(c[rt][i][part], j == 0 && step == 0, a, step ? w[i].z : w[i].x, step ? w[i].w : w[i].y);
                            }
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int e = 0; e < 2; ++e) s[rt][i][e] = fmaf((float)(c[rt][i][0][e] * 256 + c[rt][i][0][2 + e]), 65536.0f * lift[rt], (float)(c[rt][i][1][e] * 256 + c[rt][i][1][2 + e]) * lift[rt]);
            }
            // weights
            uint32_t w_hi[RT][NT], w_lo[RT][NT];
            float old[RT];
            auto weigh = [&](auto masked) {
                constexpr bool kMasked = decltype(masked)::value;
                float top[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) top[rt] = -INFINITY;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const float2 ks = *(const float2*)&sh.scales[warp][0][8 * i + 2 * t4], level = *(const float2*)&sh.scales[warp][2][8 * i + 2 * t4];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int at = 8 * i + 2 * t4 + e, key = key0 + at;
                            s[rt][i][e] *= e ? ks.y : ks.x;
                            if (kMasked && (key < low[rt] || key >= high[rt] || !(seen >> at & 1))) s[rt][i][e] = -INFINITY;
                            top[rt] = fmaxf(top[rt], fmaf(s[rt][i][e], factor[rt], e ? level.y : level.x));
                        }
                }
                float from[RT], add[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    top[rt] = fmaxf(top[rt], __shfl_xor_sync(0xffffffffu, top[rt], 1));
                    top[rt] = fmaxf(top[rt], __shfl_xor_sync(0xffffffffu, top[rt], 2));
                    top[rt] = fmaxf(base[rt], top[rt] - kRaise<RQ_KV_F16>);
                    from[rt] = top[rt] == -INFINITY ? 0.0f : top[rt];
                    old[rt] = exp2_fast(base[rt] - from[rt]);
                    base[rt] = top[rt];
                    add[rt] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const float2 vs = *(const float2*)&sh.scales[warp][1][8 * i + 2 * t4];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const float a = exp2_fast(fmaf(s[rt][i][0], factor[rt], -from[rt])), b = exp2_fast(fmaf(s[rt][i][1], factor[rt], -from[rt]));
                        add[rt] += a + b;
                        float x = a * vs.x, y = b * vs.y;
                        if (kMasked) {  // (a scale that the row must not see may be infinite, and 0 * inf is no 0)
                            x = s[rt][i][0] == -INFINITY ? 0.0f : x;
                            y = s[rt][i][1] == -INFINITY ? 0.0f : y;
                        }
                        w_hi[rt][i] = take_pair<RQ_KV_F16>(x, y);
                        w_lo[rt][i] = rqattn::pair_of<RQ_KV_F16>(x, y);
                    }
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) sum[rt] = fmaf(sum[rt], old[rt], add[rt]);
            };
            if (key0 >= every_low && key0 + TILE <= every_high && seen == ALL) weigh(std::false_type());
            else weigh(std::true_type());
            const int value_line = lane & 15, value_half = lane >> 4;
#pragma unroll
            for (int n2 = 0; n2 < D / 32; ++n2) {
                uint32_t b[TILE / 16][4];
#pragma unroll
                for (int half = 0; half < TILE / 16; ++half) {
                    const int line = 16 * half + value_line;
                    ldmatrix_transposed(b[half], values + line * D + (placed<D>(line, 2 * n2 + value_half) << 4));
#pragma unroll
                    for (int i = 0; i < 4; ++i) b[half][i] = turn_codes(b[half][i]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // sixteen elements, even ones, odd ones
                    uint32_t b0[TILE / 16], b1[TILE / 16];
#pragma unroll
                    for (int half = 0; half < TILE / 16; ++half) {
                        const uint32_t x = b[half][i & 2], y = b[half][(i & 2) + 1];
                        b0[half] = i & 1 ? widen_codes<1, 3>(x) : widen_codes<0, 2>(x);
                        b1[half] = i & 1 ? widen_codes<1, 3>(y) : widen_codes<0, 2>(y);
                    }
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        float d[4];
#pragma unroll
                        for (int half = 0; half < TILE / 16; ++half)
                            mma(d, half == 0, w_hi[rt][2 * half], w_lo[rt][2 * half], w_hi[rt][2 * half + 1], w_lo[rt][2 * half + 1], b0[half], b1[half]);
                        acc[rt][4 * n2 + i] = pair_fma(acc[rt][4 * n2 + i], ::pair_of(old[rt], old[rt]), pair_add(::pair_of(d[0], d[1]), ::pair_of(d[2], d[3])));
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
            for (int n = 0; n < D / 16; ++n)
                *(float4*)&sh.out[warp][rt * 8 + g][16 * n + 4 * t4] = make_float4(pair_at(acc[rt][2 * n], 0), pair_at(acc[rt][2 * n + 1], 0), pair_at(acc[rt][2 * n], 1), pair_at(acc[rt][2 * n + 1], 1));
        }
        __syncthreads();
        join_rows<D, ROWS, kLead, true>(p, &sh.out[0][0][0], warp_base, warp_sum, item_begin, item_end, deal, start, row0, rows, kv, last_arrival);
        __syncthreads();  // the shared sums are free again
    }
}

template <int D, int RT>
int launch_rows(rq_ctx* ctx, const CodesParams& p, cudaStream_t s) {
    auto kernel = rq_attention_int8_kernel<D, RT>;
    // The grid decides where rows are cut, and with it the last bits: it follows from the call alone. Shared memory holds eight bytes a request, by steps of 128 of them.
    const int step = (p.requests + kRequestStep - 1) / kRequestStep, dev = ctx->device;
    auto bytes = [](int steps) { return sizeof(Tiles<D, RT>) + sizeof(int64_t) * ((size_t)steps * kRequestStep + 1); };
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

}  // namespace

int rqattn::launch_rows_int8(rq_ctx* ctx, const CodesParams& p, const rq_kv_cache& cache, bool two, cudaStream_t s) {
    if (cache.head_dim == 64) return two ? launch_rows<64, 2>(ctx, p, s) : launch_rows<64, 1>(ctx, p, s);
    if (cache.head_dim == 128) return two ? launch_rows<128, 2>(ctx, p, s) : launch_rows<128, 1>(ctx, p, s);
    return launch_rows<256, 1>(ctx, p, s);
}
