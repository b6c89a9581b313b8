// Attention of chunks and prompts over the paged cache: rows by the hundred, on the 5th-generation tensor cores.
//
// A row is one query head of one new token; the rows of the heads that share a key head lie together, tokens after tokens, so that they
// meet a tile of keys and values together. A CTA has two PIPES, each with 128 rows' scores and sums in tensor memory and a
// warpgroup of softmax threads (a thread has one row to itself):
//   rows form (f16): the pipes are two tiles of 128 rows, which share every tile of 128 keys;
//   keys form (few rows; bf16, whose third parts leave no room for a second row tile): one row tile, the pipes take alternate tiles of keys and
//     are joined at the end, through tensor memory.
// Per tile of keys: S = Q K^T (tcgen05.mma, Q and K in shared memory), weights P = 2^(S - base) from and to tensor memory, T = P V (P in tensor memory,
// V in shared memory as it lies in the cache, keys times elements), sums O = O 2^(old base - base) + T in fp32 registers, base = max - 12 (bf16: 0) as rounded
// (kept itself, so that the factor is exactly one where the base stays).
//   * fp32 activations: Q and P are taken apart into 16-bit parts (hi + lo over f16, 22 bits, Q brought to f16's range by a power of two a row; hi + mid + lo over
//     bf16), each part a product of its own into the same accumulator, the smallest first. Products double (treble) against 16-bit activations; with one part the
//     results would be off by 2^-11 (2^-8) where the framework's fp32 activations are good for 1e-6.
//   * The tensor core adds by truncation: T is one tile's sum only, and O is added up with round-to-nearest.
//   * P takes the place of its S in tensor memory, 32 keys' hi and lo parts over the 32 scores they came from.
// The issuing warp's order is Q K_A(j + 1), P V_B(j), Q K_B(j + 1), P V_A(j + 1), ..: while the tensor core is busy with one pipe's
// products the other pipe's softmax runs. A thread issues a product of 128 columns every 71 cycles, 64 of them a unit: 4.5 thousand cycles.
//
// Work is counted in units, one tile of keys (keys form: two) of one block of rows; every CTA takes an equal range of them, wherever it begins and ends, and
// rows whose keys fall to several CTAs are joined in CTA order by the last of these (the same bits on every run). Keys and values come by TMA, a
// page (at most a tile) of 64 elements a copy, into a ring of stages; an entry of the page table that names no page becomes a coordinate outside, which reads zeros.
//
// A value that a row does not see may be infinite, and 0 * inf is no 0: where a tile is not seen by all rows, the mending warp takes what is not
// finite out of it, and the softmax threads add it to the sums of the rows that do see it.
//
// A cache of 8-bit codes (CODES): TMA brings whole lines of codes into a part of the place that their f16 numbers take, four more warps widen them there, exactly, and bring the tile's
// scales. The softmax multiplies scores by the keys' scales and weights, before they are taken apart, by the values'; a value's scale counts by its exponent in the row's base,
// by the tile's largest where they lie within 2^12 of each other. A tile is half the bytes and 40 % more work: 8.8 thousand cycles in place of 6.1 (the first pass over
// scores 1.7 in place of 0.8, the second 4.1 in place of 3.1, the rest waits for tiles). Two of the twelve warps as wideners: 509 tokens over 7680 keys 183 us in place of 172; codes kept as codes
// and multiplied as bytes would need P in digits.
//
// Every wait between the roles is bounded; a wait that runs out records a code in the context's error word, and the warp waits no more and hands nothing on, so that
// the others' waits run out too and all meet at the end. The loading warp leaves when every copy has landed.
//
// 509 tokens over 7680 keys, 32 + 2 x 8 heads of 128, f16: 137 us, 66 GFLOP of them useful (0.29 of the measured peak, 0.59 with both parts), products under way
// 56 % of the time; four prompts of 1021 to 3001 tokens 378 us, 150 GFLOP (both called among other cases; over the same two batches again and again 123 and 350). Over codes 160 and 440 us,
// products under way 41 % of the time; that form spills 746 bytes of stores a thread and 964 of loads (over f16 606 and 800), half of them in the issuing warp.
#include <type_traits>

#include "rq_attention.cuh"
#include "rq_mma.cuh"
#include "rq_pairs.cuh"

using namespace rqserve;
using namespace rqattn;
using namespace rqmma;

namespace {

constexpr int kSoftmaxWarps = 8, kIssuer = 8, kLoader = 9, kFetcher = 10, kMender = 11, kWidener = 12;
constexpr int kCodesShift = 4;  // a copy of codes brings at most sixteen lines
constexpr int kEven = 12;       // exponents of a tile's scales of values that lie no further apart need no look at each
// Keys' scales of 2^-60 to 2^61 meet a row's sum (at most 2^30) before its power of two does: neither is past fp32's range, and a score that the power's lower end, 2^-126, is
// too large for is less than 2^-34. Other tiles, and rows of powers above 2^126, take it in two parts.
constexpr int kUsual = 60;
constexpr int kItems = 4, kWords = 16;  // rings in shared memory: items, words on tiles of keys

// Taking a block up (its queries, the first scores, the sums at the end: 21 us) costs as much as some units (3.9 us): so many lead each block's own in the dealing.
// Without it the CTAs that got a prompt's first blocks, short ones, were the last to end. 32 + 2 x 8 heads of 128, f16, without | with, over the same batches again and
// again: four prompts of 1021 to 3001 tokens 620 | 350 us, one of 12001 2816 | 1883, eight of 512 138 | 120, two of 3001 with windows of 1000 425 | 244, 509 tokens over 7680 125 |
// 123; 32 of 128, all blocks of one unit, 67 | 68; 16 requests of 48 rows over 8192 keys 205 | 219.
// Over codes a unit takes longer: by three 509 tokens over 7680 keys 164 us, the four prompts 452, by four 164 and 461, by two 164 and 467.

// CODES: the cache holds 8-bit codes, TYPE is what they become
template <int D, int TYPE, bool KEYS_, bool CODES_> struct Form {
    static constexpr bool KEYS = KEYS_, CODES = CODES_;
    using Params = std::conditional_t<CODES, CodesParams, AttentionParams>;
    // registers that the block is launched with are dealt out anew: 2 * 224 + 56 = 3 * 168; 2 * 200 + 2 * 56 = 4 * 128 (208 and 48: the four prompts 469 us in place of 461)
    static constexpr int WIDENERS = CODES ? 4 : 0, THREADS = (12 + WIDENERS) * 32, SOFTMAX_REGS = CODES ? 200 : 224, OTHER_REGS = 56, LEAD = CODES ? 3 : 4;
    static constexpr int PARTS = TYPE == RQ_KV_F16 ? 2 : 3;
    static constexpr int KT = TYPE == RQ_KV_F16 || D == 64 ? 128 : 64;  // keys a tile (bf16, 128 elements: 2 KT + 2 D + KT columns are what tensor memory holds with 64)
    static constexpr int TILE_BYTES = KT * D * 2, Q_PART = 128 * D * 2, Q_BYTES = (KEYS ? 1 : 2) * PARTS * Q_PART;
    static constexpr int STAGES_FIT = ((227 - 3) * 1024 - Q_BYTES) / TILE_BYTES, STAGES = CODES ? (D == 64 ? 6 : (KEYS ? 4 : 3)) : (STAGES_FIT > 8 ? 8 : STAGES_FIT);
    // Codes: tiles whose scales are held. A tile's are written once its keys have landed, where the slot's tile before has been used: of three slots that is the values two
    // tiles back, of six at most the ones five back.
    static constexpr int SCALE_TILES = !CODES ? 1 : (STAGES == 3 ? 2 : 8);
    static constexpr int LANDED_BYTES = CODES ? TILE_BYTES / 2 : TILE_BYTES;
    static constexpr int BLOCK = KEYS ? 128 : 256;                // rows
    static constexpr int UNIT = KEYS ? 2 * KT : KT;               // keys
    static constexpr int T_COL = 2 * KT, LO_COL = T_COL + 2 * D;  // tensor memory: scores (then weights), tile sums, bf16's third parts
    static_assert(STAGES >= (KEYS ? 4 : 3) && STAGES <= STAGES_FIT, "ring");
    static_assert(LO_COL + (PARTS == 3 ? KT : 0) <= 512, "tensor memory");
};

// A block of rows of one request and key head, and the keys that some row of it sees
struct Block {
    int start, row0, rows, position0, begin, low, high, end;  // keys [low, high), from the tile at begin; end: the request's keys
    int units;
};
template <typename F> __device__ __forceinline__ int blocks_of(const AttentionParams& p, int r, int group) {
    const int rows = tokens_here(p, p.starts[r], p.starts[r + 1]) * group;
    return rows > p.few ? (rows + F::BLOCK - 1) / F::BLOCK : 0;
}
template <typename F> __device__ __forceinline__ Block block_of(const AttentionParams& p, int r, int b, int group) {
    Block k;
    k.start = p.starts[r];
    const int next = p.starts[r + 1];
    const int length = p.lengths[r];
    k.end = (int)min((int64_t)max(length, 0), (int64_t)p.table_width << p.page_shift);
    k.position0 = length - max(next - k.start, 0);
    k.row0 = b * F::BLOCK;
    k.rows = min(F::BLOCK, tokens_here(p, k.start, next) * group - k.row0);
    const int first = k.row0 / group, last = (k.row0 + k.rows - 1) / group;
    k.high = max(0, min(k.end, k.position0 + last + 1));
    k.low = p.window > 0 ? min(k.high, max(0, k.position0 + first - p.window + 1)) : 0;
    k.begin = k.low & ~(F::KT - 1);
    k.units = max(1, (k.high - k.begin + F::UNIT - 1) / F::UNIT);
    return k;
}

// One block's part of a CTA's range of units, as the roles need it; take = 0: there are no more
struct Item {
    int take;                                    // units
    int first_key, low, high, end;               // as in Block, from the first key of the part
    int start, row0, rows, position0, kv, r;
    int first_cta, last_cta;                     // that share the block
};

// B as it lies in the cache, elements of a key contiguous: 64 elements a 128-byte swizzled line, lines of eight keys 1024 bytes, the
// next 64 elements `half` bytes on
__device__ __forceinline__ uint64_t values_desc(uint32_t addr, uint32_t half) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(half >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void mma_f16_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u)
        : "memory");
}
// 32 columns of this warp's 32 rows: under way, and (tmem_ld_wait) there
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, "
        "%26, %27, %28, %29, %30, %31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {  // the registers pass through: nothing that uses them can move ahead of it
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30])
                 :
                 : "memory");
    asm volatile("" : "+r"(r[31])::"memory");
}
// eight fp32 numbers, 32 bytes: a whole sector for a thread whose neighbours are a row away
__device__ __forceinline__ void store32(float* p, const float* x, float f) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0] * f), "f"(x[1] * f), "f"(x[2] * f), "f"(x[3] * f), "f"(x[4] * f), "f"(x[5] * f), "f"(x[6] * f),
                 "f"(x[7] * f)
                 : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_to_tensor_core() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <typename F> struct Shared {
    uint64_t full[F::STAGES], empty[F::STAGES], item_full[kItems], item_empty[kItems], q_full[2], s_full[2], p_full[2][2], t_full[2], t_empty[2], q_empty, landed[F::STAGES], joined[4], ended;
    int64_t warp_sums[F::THREADS / 32], range[2];
    int where[4];
    Item items[kItems];
    uint32_t pages_there[kWords];  // a tile's pages that the cache has, a bit each; all ones: all of them
    uint32_t odd[kWords];          // whether something was taken out of a tile's values
    uint32_t tmem_slot;
    float factors[2][F::KEYS && F::PARTS == 2 ? 128 : 1];  // keys form over f16: of the rows' scores (codes: their powers of two, as bits), the items in turn
    float joint[2][F::KEYS ? 128 : 1];  // keys form: the second pipe's base and sum of each row
    alignas(16) float scales[F::SCALE_TILES][2][F::CODES ? F::KT : 1];  // codes: of a tile's keys, of its values
    int levels[F::SCALE_TILES][4][2];                                     // codes: the largest and the least exponent of the scales of either half of its keys, and of its values
};

__device__ __forceinline__ bool finite16(uint32_t v, int type) { const uint32_t e = type == RQ_KV_F16 ? 0x7c00u : 0x7f80u; return (v & e) != e; }
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int line, int head, int page, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map), "r"(x), "r"(line), "r"(head),
                 "r"(page), "r"(smem_u32(bar))
                 : "memory");
}

__device__ __forceinline__ uint32_t max_pairs(uint32_t a, uint32_t b) { uint32_t r; asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }

// The rows of a warp's share, each brought to one size by its own largest element; returns what that of the lane's row was raised by. (Over codes rows below 2^-112 too, in two
// steps: keys may be as large as they are small. f16 keys may not.) A call of its own: in line, it takes registers from the softmax around it (a prompt of 3001 tokens,
// windows of 1000, 259 us in place of 247).
template <int D, int TYPE, bool KEYS, bool CODES> __device__ __noinline__ int rescale_queries(const AttentionParams& p, int64_t mine, uint8_t* to, int first) {
    using F = Form<D, TYPE, KEYS, CODES>;
    constexpr int SHARE = 128 / D, ROWS = KEYS ? 16 : 32, BATCH = 4;
    const int lane = threadIdx.x & 31, e = 4 * (lane % (D / 4));
    int raise = 0;
#pragma unroll 1
    for (int r0 = 0; r0 < ROWS; r0 += BATCH * SHARE) {
        float4 x[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int64_t from = __shfl_sync(0xffffffffu, mine, r0 + i * SHARE + lane / (D / 4));
            x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (from >= 0) {
                const float* q = p.q + from + e;
                if (p.wide) x[i] = __ldcg((const float4*)q);
                else x[i] = make_float4(__ldcg(q), __ldcg(q + 1), __ldcg(q + 2), __ldcg(q + 3));
            }
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int r = r0 + i * SHARE;
            float top = fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w)));
#pragma unroll
            for (int off = D / 8; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            const int here = CODES ? 141 - (int)(__float_as_uint(top) >> 23) : raise_of(__float_as_uint(top)), told = __shfl_sync(0xffffffffu, here, (lane % SHARE) * (D / 4));
            if ((lane & (ROWS - SHARE)) == r) raise = told;
            const float raised = power_of_two(CODES ? min(here, 126) : here);
            const int row = first + r + lane / (D / 4);
            uint8_t* place = to + (e >> 6) * (128 * 128) + swizzled(row, (e & 63) >> 3) + 2 * (e & 7);
            x[i].x *= raised; x[i].y *= raised; x[i].z *= raised; x[i].w *= raised;
            if (CODES) {
                const float more = power_of_two(max(here - 126, 0));
                x[i].x *= more; x[i].y *= more; x[i].z *= more; x[i].w *= more;
            }
#pragma unroll
            for (int part = 0; part < F::PARTS; ++part) *(uint2*)(place + part * F::Q_PART) = make_uint2(take_pair<TYPE>(x[i].x, x[i].y), take_pair<TYPE>(x[i].z, x[i].w));
        }
    }
    return raise;
}

// Queries of a warp's share of the block's rows, brought to one size (f16) and taken apart, as the tensor core reads them: a row is one contiguous access, eight
// accesses on their way at a time. (A thread that reads a row of its own meets 32 lines an instruction.) Returns what the lane's row was raised by.
// Over f16 all rows are multiplied by the same power of two first, and the parts themselves say whether that was the right one for each: a row's largest element has
// to be 2 or more, and finite, as an f16 number. Where it is not, the warp's rows are taken once more. (Every row by its own largest element at once made a block's
// take-up 1.7 us longer: 32 prompts of 128 tokens 71 us in place of 68. Queries a thousandth of the usual size: 88 us, and the four prompts 402 in place of 356.)
template <int D, int TYPE, bool KEYS, bool CODES> __device__ __forceinline__ int load_queries(const AttentionParams& p, const Item& it, uint8_t* to, int block_row, int first, int group) {
    using F = Form<D, TYPE, KEYS, CODES>;
    constexpr int SHARE = 128 / D, ROWS = KEYS ? 16 : 32, BATCH = ROWS / SHARE < 8 ? ROWS / SHARE : 8;  // rows an access; rows a warp; accesses at a time
    const int lane = threadIdx.x & 31, own = block_row + first + (lane & (ROWS - 1)), at = it.row0 + own, e = 4 * (lane % (D / 4));
    const int64_t mine = own < it.rows ? (int64_t)(it.start + at / group) * p.q_stride + (int64_t)(it.kv * group + at % group) * D : -1;
    auto load = [&](int row) {
        const int64_t from = __shfl_sync(0xffffffffu, mine, row + lane / (D / 4));
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (from >= 0) {
            const float* q = p.q + from + e;
            if (p.wide) x = __ldcg((const float4*)q);
            else x = make_float4(__ldcg(q), __ldcg(q + 1), __ldcg(q + 2), __ldcg(q + 3));
        }
        return x;
    };
    uint32_t large = 0, most = 0;  // a bit an access: whether it holds a number of 2 or more; the largest numbers
#pragma unroll 1
    for (int r0 = 0; r0 < ROWS; r0 += BATCH * SHARE) {
        float4 x[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) x[i] = load(r0 + i * SHARE);
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int row = first + r0 + i * SHARE + lane / (D / 4);
            uint8_t* place = to + (e >> 6) * (128 * 128) + swizzled(row, (e & 63) >> 3) + 2 * (e & 7);
            if (F::PARTS == 2) {
                constexpr float kRaised = 1 << kUsualRaise;
                x[i].x *= kRaised; x[i].y *= kRaised; x[i].z *= kRaised; x[i].w *= kRaised;
            }
#pragma unroll
            for (int part = 0; part < F::PARTS; ++part) {
                const uint2 w = make_uint2(take_pair<TYPE>(x[i].x, x[i].y), take_pair<TYPE>(x[i].z, x[i].w));
                *(uint2*)(place + part * F::Q_PART) = w;
                if (F::PARTS == 2 && part == 0) {
                    if ((w.x | w.y) & 0x40004000u) bits |= 1u << i;
                    most = max_pairs(most, max_pairs(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu));
                }
            }
        }
        large |= bits << (r0 / SHARE);
    }
    int raise = F::PARTS == 2 ? kUsualRaise : 0;
    if (F::PARTS == 2) {
        const uint32_t rows_there = __ballot_sync(0xffffffffu, mine >= 0) & (uint32_t)((1ull << ROWS) - 1);
        const bool too_large = ((most & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
        uint32_t lacking;  // rows without a large number
        if (SHARE == 1) {
            lacking = rows_there & ~__reduce_or_sync(0xffffffffu, large);
        } else {
            const uint32_t all = __reduce_or_sync(0xffffffffu, lane < 16 ? large : large << 16), row = lane & (ROWS - 1);  // even rows, odd rows
            lacking = __ballot_sync(0xffffffffu, !(all >> ((row >> 1) + (row & 1) * 16) & 1)) & rows_there;
        }
        if (__any_sync(0xffffffffu, too_large) || lacking) {
            raise = rescale_queries<D, TYPE, KEYS, CODES>(p, mine, to, first);
        }
    }
    fence_to_tensor_core();
    return raise;
}

template <int D, int TYPE, bool KEYS, bool CODES>
__global__ void __launch_bounds__(Form<D, TYPE, KEYS, CODES>::THREADS, 1) rq_attention_tc_kernel(const __grid_constant__ typename Form<D, TYPE, KEYS, CODES>::Params p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    using F = Form<D, TYPE, KEYS, CODES>;
    constexpr int PARTS = F::PARTS, KT = F::KT, STAGES = F::STAGES;
    extern __shared__ __align__(1024) unsigned char dynamic[];
    uint8_t* const smem = dynamic;  // (there is no other shared memory in front of it)
    uint8_t* const ring = smem + F::Q_BYTES;
    auto& sh = *(Shared<F>*)(ring + STAGES * F::TILE_BYTES);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int group = p.q_heads / p.kv_heads;

    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(&sh.full[i], CODES ? F::WIDENERS : 1); mbar_init(&sh.empty[i], 1); mbar_init(&sh.landed[i], 1); }
        for (int i = 0; i < kItems; ++i) { mbar_init(&sh.item_full[i], 1); mbar_init(&sh.item_empty[i], kSoftmaxWarps + (CODES ? 2 + F::WIDENERS : 3)); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.q_full[i], KEYS ? 8 : 4);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i][0], 4);
            mbar_init(&sh.p_full[i][1], 4);
            mbar_init(&sh.t_full[i], 1);
            mbar_init(&sh.t_empty[i], 4);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&sh.joined[i], 1);
        mbar_init(&sh.q_empty, 1);
        mbar_init(&sh.ended, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kIssuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    launch_dependents();
    wait_for_previous();

    // ---- where this CTA's units lie: requests' units are added up once, a request a thread and round ------
    {
        int64_t* const before = (int64_t*)smem;  // (the queries' place and, at most, the ring's first bytes)
        int64_t total = 0;
        if (tid == 0) before[0] = 0;
        for (int r0 = 0; r0 < p.requests; r0 += F::THREADS) {
            const int r = r0 + tid;
            int64_t units = 0;
            if (r < p.requests)
                for (int b = blocks_of<F>(p, r, group) - 1; b >= 0; --b) units += F::LEAD + block_of<F>(p, r, b, group).units;
            units *= p.kv_heads;
            int64_t scan = units;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) { const int64_t o = __shfl_up_sync(0xffffffffu, scan, off); if (lane >= off) scan += o; }
            __syncthreads();
            if (lane == 31) sh.warp_sums[warp] = scan;
            __syncthreads();
            scan += total;
            for (int w = 0; w < F::THREADS / 32; ++w) { if (w < warp) scan += sh.warp_sums[w]; total += sh.warp_sums[w]; }
            if (r < p.requests) before[r + 1] = scan;
        }
        __syncthreads();
        if (tid == 0) {
            const int64_t ctas = min((int64_t)gridDim.x, total), u = blockIdx.x < ctas ? blockIdx.x * total / ctas : 0;
            sh.range[0] = u;
            sh.range[1] = blockIdx.x < ctas ? (blockIdx.x + 1) * total / ctas : 0;
            int r = 0, b = 0;
            for (int hi = p.requests - 1; r < hi;) { const int mid = (r + hi + 1) >> 1; if (before[mid] <= u) r = mid; else hi = mid - 1; }
            int64_t left = u - before[r];
            int units = 1;
            if (total)
                while (true) {
                    units = F::LEAD + block_of<F>(p, r, b, group).units;
                    if (left < (int64_t)units * p.kv_heads) break;
                    left -= (int64_t)units * p.kv_heads;
                    ++b;
                }
            sh.where[0] = r;
            sh.where[1] = b;
            sh.where[2] = (int)(left / units);
            sh.where[3] = (int)(left % units);
            sh.warp_sums[0] = total;
            sh.warp_sums[1] = ctas;
        }
        fence_to_tensor_core();  // copies write where these sums were
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem_slot;
    // The CTA's items, one after another: each role waits for one, reads what it needs of it and gives it back
    Ring item_at(kItems);
    bool dead = false;
    auto next_item = [&]() -> const Item* {
        if (!mbar_wait_warp(&sh.item_full[item_at.slot], item_at.phase, p.wait_ns, dead)) atomicExch(p.error_flag, 40);
        const Item* i = &sh.items[item_at.slot];
        return !dead && i->take ? i : nullptr;
    };

    // An item's tiles of keys and values in the order of their use: K0 V0 K1 V1 .. (rows form), K0 K1 V0 K2 V1 K3 .. (keys form); n-th of 2 * tiles
    auto is_values = [](int n, int tiles) { return KEYS ? n > 1 && (!(n & 1) || (n + 1) / 2 >= tiles) : (n & 1) != 0; };
    auto tile_of = [](int n, int tiles) { return KEYS ? (n < 2 ? n : (n & 1 ? min((n + 1) / 2, tiles - 1) : n / 2 - 1)) : n >> 1; };
    // A tile that not every row sees: its values are looked at before they are used
    auto is_edge = [&](const Item& i, int key0) {
        const int every_high = min(i.high, i.position0 + i.row0 / group + 1);
        const int every_low = p.window > 0 ? max(i.low, i.position0 + (i.row0 + i.rows - 1) / group - p.window + 1) : i.low;
        return key0 < every_low || key0 + KT > every_high;
    };

    // Codes: four warps bring each tile from where it landed to what the tensor core reads, every fourth sixteen lines each, and a half each of the scales of its keys (0, 1) and
    // of its values (2, 3) beside it. Sixteen lines landed in a part of the place that their f16 numbers take (128 elements: where the second 64 go; 64: in the upper half, pages
    // of eight lines in that of their own): a warp has read them before it writes there. A lane's pieces are 16 codes, one load, two stores, so that no eight lanes meet a
    // bank twice.
    auto widen = [&](int which) {
        if constexpr (CODES) {
            constexpr int SHARE = KT / 64, PIECES = D / 32;  // scales, pieces of sixteen lines, of a lane
            Ring at(STAGES);
            uint32_t key_tiles = 0;
            while (const Item* it = next_item()) {
                const int tiles = it->take * (KEYS ? 2 : 1);
                const int32_t* table = p.block_table + (int64_t)it->r * p.table_stride + (it->first_key >> p.page_shift);
                const float* scales = (which < 2 ? p.k_scale : p.v_scale) + it->kv * p.scale_head;
                const int first = (which & 1) * (KT / 2) + lane, line0 = it->first_key & ((1 << p.page_shift) - 1), low = it->low - it->first_key, high = it->high - it->first_key;  // keys from the item's first
                // Scales are on their way while the tile before is widened, and their pages' entries while the one before that is
                int page[SHARE];
                float scale[SHARE];
                auto find = [&](int tile) {
#pragma unroll
                    for (int i = 0; i < SHARE; ++i) {
                        const int key = tile * KT + first + 32 * i;
                        page[i] = key >= low && key < high ? __ldcg(table + ((line0 + key) >> p.page_shift)) : -1;
                    }
                };
                auto load = [&](int tile) {
#pragma unroll
                    for (int i = 0; i < SHARE; ++i) {
                        const int line = (line0 + tile * KT + first + 32 * i) & ((1 << p.page_shift) - 1);
                        scale[i] = page[i] >= 0 && page[i] < p.pages ? __ldcg(scales + page[i] * p.scale_page + line * p.scale_line) : 0.0f;
                    }
                };
                find(0);
                load(0);
                find(1);
                for (int n = 0, tile = 0; n < 2 * tiles; ++n, at.next()) {
                    const bool values = is_values(n, tiles);
                    const int slot = at.slot;
                    if (!mbar_wait_warp(&sh.landed[slot], at.phase, p.wait_ns, dead)) atomicExch(p.error_flag, 54);
                    if (dead) break;  // (the tile may be on its way: it is not touched, and not handed on)
                    // (a short loop: laid out in a line it took the softmax's place in the instruction caches, 259 us in place of 236 then)
#pragma unroll 1
                    for (int block = which; block < KT / 16; block += F::WIDENERS) {
                        uint8_t* const out = ring + slot * F::TILE_BYTES + block * 2048;
                        uint4 raw[PIECES];
#pragma unroll
                        for (int i = 0; i < PIECES; ++i) {
                            if (D == 64) raw[i] = *(const uint4*)(out + (p.page_shift == 3 ? 512 * (2 * i + 1) : 1024 + 512 * i) + 16 * lane);
                            else raw[i] = *(const uint4*)(out + KT * 128 + (8 * (i >> 1) + (lane >> 2)) * 128 + ((i & 1) ^ (lane >> 2 & 1)) * 64 + (lane & 3) * 16);
                        }
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < PIECES; ++i) {
                            const int line = 8 * (D == 64 ? i : i >> 1) + (lane >> 2);
                            uint8_t* const to = out + (D == 64 ? 0 : (i & 1) ^ (lane >> 2 & 1)) * (KT * 128);
                            const uint32_t x = turn_codes(raw[i].x), y = turn_codes(raw[i].y), z = turn_codes(raw[i].z), w = turn_codes(raw[i].w);
                            *(uint4*)(to + swizzled(line, 2 * (lane & 3))) = make_uint4(widen_codes<0, 1>(x), widen_codes<2, 3>(x), widen_codes<0, 1>(y), widen_codes<2, 3>(y));
                            *(uint4*)(to + swizzled(line, 2 * (lane & 3) + 1)) = make_uint4(widen_codes<0, 1>(z), widen_codes<2, 3>(z), widen_codes<0, 1>(w), widen_codes<2, 3>(w));
                        }
                    }
                    if (!values) {
                        const int place = key_tiles++ % F::SCALE_TILES;
                        int most = 0, least = 254;
#pragma unroll
                        for (int i = 0; i < SHARE; ++i) {
                            sh.scales[place][which >> 1][first + 32 * i] = scale[i];
                            const int e = (int)(__float_as_uint(scale[i]) >> 23 & 0xff);
                            most = max(most, e);
                            least = min(least, scale[i] == 0.0f ? 254 : e);  // (a value of zero takes no weight's bits, a key of zero is none of an extreme size)
                        }
                        most = __reduce_max_sync(0xffffffffu, most);
                        least = __reduce_min_sync(0xffffffffu, least);
                        if (lane == 0) { sh.levels[place][which][0] = most; sh.levels[place][which][1] = least; }
                    }
                    fence_to_tensor_core();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.full[slot]);
                    if (!values) {
                        load(++tile);
                        find(tile + 1);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.item_empty[item_at.slot]);
                item_at.next();
            }
        }
    };

    if (warp < kSoftmaxWarps) {
        // ------------------------------------------------------------ softmax: a thread a row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F::SOFTMAX_REGS));
        const int pipe = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t rows_at = tmem + ((uint32_t)(quarter * 32) << 16), scores = rows_at + pipe * KT, sums_at = rows_at + F::T_COL + pipe * D, lo_at = rows_at + F::LO_COL + pipe * (KT / 2);
        const int in_block = KEYS ? row : pipe * 128 + row;
        uint32_t tiles_done = 0, keys_before = 0, items_done = 0;  // this pipe's tiles; the items' tiles of keys; items
        float factor = 1.0f;  // of this row's scores
        int exponent = 0;     // codes: their power of two
        auto queries = [&](const Item& of, uint32_t n) {  // of the n-th item
            const int first = quarter * 32 + (KEYS ? pipe * 16 : 0);
            const int raise = load_queries<D, TYPE, KEYS, CODES>(p, of, smem + (KEYS ? 0 : pipe * PARTS * F::Q_PART), KEYS ? 0 : pipe * 128, first, group);
            if constexpr (CODES) exponent = p.scale_exponent - raise;
            else factor = factor_of(p.scale, raise);
            if (KEYS && PARTS == 2 && lane < 16) sh.factors[n & 1][first + lane] = CODES ? __int_as_float(exponent) : factor;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full[KEYS ? 0 : pipe]);
        };

        float o[D];
        const Item* it = next_item();
        if (it) queries(*it, 0);
        while (it) {
            const Item* following = nullptr;
            const int tiles = it->take;
            int low, high;  // the keys that this row sees
            {
                const int position = it->position0 + (it->row0 + in_block) / group;
                high = in_block < it->rows ? min(position + 1, it->end) : 0;
                low = p.window > 0 ? max(position - p.window + 1, 0) : 0;
            }
            // (keys form: the rows' queries are brought by the warps of both pipes)
            if (KEYS && PARTS == 2) {
                if (!mbar_wait_warp(&sh.q_full[0], items_done & 1, p.wait_ns, dead)) atomicExch(p.error_flag, 53);
                if (CODES) exponent = __float_as_int(sh.factors[items_done & 1][row]);
                else factor = sh.factors[items_done & 1][row];
            }
            float base = -INFINITY, sum = 0.0f, old = 1.0f;  // base: -inf while the row has seen no key
#pragma unroll
            for (int i = 0; i < D; ++i) o[i] = 0.0f;
            // The values of a tile that are not finite, to the sums of the rows that see them
            auto add_odd = [&](int first) {
                const int32_t* table = p.block_table + (int64_t)it->r * p.table_stride;
                for (int key = max(first, it->low); key < min(first + KT, it->high); ++key) {
                    const int page = __ldcg(table + (key >> p.page_shift));
                    if (page < 0 || page >= p.pages) continue;
                    const uint16_t* v = p.v + it->kv * p.head_stride + (int64_t)page * (p.page_bytes / 2) + (int64_t)(key & ((1 << p.page_shift) - 1)) * (p.line_bytes / 2);
                    bool fine = true;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) fine = fine && finite16(__ldcg(v + 32 * i + lane), TYPE);
                    if (__all_sync(0xffffffffu, fine)) continue;
                    const bool sees = key >= low && key < high;
#pragma unroll
                    for (int i = 0; i < D; ++i) {
                        const uint16_t x = __ldcg(v + i);
                        if (sees && !finite16(x, TYPE)) o[i] += to_float<TYPE>(x);
                    }
                }
            };
            int key0 = it->first_key + (KEYS ? pipe * KT : 0);
            constexpr int kStep = (KEYS ? 2 : 1) * KT;
#pragma unroll 1
            for (int j = 0;; ++j, key0 += kStep) {
                if (j > 0) {
                    // O = O f + T, the sums of this pipe's tile before, while the tensor core makes the next one's scores
                    if (!mbar_wait_warp(&sh.t_full[pipe], (tiles_done - 1) & 1, p.wait_ns, dead)) atomicExch(p.error_flag, 41);
                    fence_after();
                    const Pair ff = pair_of(old, old);
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t t[32];
                        tmem_ld32(sums_at + 32 * c, t);
                        tmem_ld_wait(t);
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            float* to = o + 32 * c + i;
                            const Pair v = pair_fma(pair_of(to[0], to[1]), ff, pair_of(t[i], t[i + 1]));
                            to[0] = pair_at(v, 0);
                            to[1] = pair_at(v, 1);
                        }
                    }
                    fence_before();
                    __syncwarp();
                    // (the loading warp took what is not finite out of the tile)
                    if (!CODES && *(volatile uint32_t*)&sh.odd[(keys_before + (KEYS ? 2 * (j - 1) + pipe : j - 1)) % kWords]) add_odd(key0 - kStep);
                    if (j == tiles) break;
                    if (lane == 0) mbar_arrive(&sh.t_empty[pipe]);
                }
                if (!mbar_wait_warp(&sh.s_full[pipe], tiles_done & 1, p.wait_ns, dead)) atomicExch(p.error_flag, 42);
                fence_after();
                const uint32_t there = *(volatile uint32_t*)&sh.pages_there[(keys_before + (KEYS ? 2 * j + pipe : j)) % kWords];
                const int place = (keys_before + (KEYS ? 2 * j + pipe : j)) % F::SCALE_TILES;
                const float *of_keys = sh.scales[place][0], *of_values = sh.scales[place][1];
                // (the exponent that counts for the tile: the largest, where they lie close together)
                int level = 0;
                bool even = true;
                if (CODES) {
                    const volatile int* l = &sh.levels[place][0][0];
                    const int most = max(l[4], l[6]);
                    even = most < 255 && most - min(l[5], l[7]) <= kEven && max(l[0], l[2]) <= 127 + kUsual && min(l[1], l[3]) >= 127 - kUsual && exponent <= 126;
                    level = min(max(most, 127 - 80), 127 + 90) - 127;
                }
                // (codes: rows past the block's last, whose results nobody reads, hide nothing)
                const bool all = (key0 >= low && key0 + KT <= high && there == 0xffffffffu) || (CODES && in_block >= it->rows);
                // the columns of 32 keys that this row sees
                auto shown = [&](int c) -> uint32_t {
                    const int from = key0 + 32 * c, a = min(max(high - from, 0), 32), b = min(max(low - from, 0), 32);
                    uint32_t on = (a == 32 ? 0xffffffffu : (1u << a) - 1) & ~(b == 32 ? 0xffffffffu : (1u << b) - 1);
                    if (there != 0xffffffffu)
                        for (int i = 0; i < 32; ++i)
                            if (!(there >> ((from - key0 + i) >> (CODES ? min(p.page_shift, kCodesShift) : p.page_shift)) & 1)) on &= ~(1u << i);
                    return on;
                };
                float f;
                auto weights_there = [&](int half) {
                    tmem_st_wait();
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.p_full[pipe][half]);
                };
                // The loops over columns are loops: laid out in a line, with the masks, they were longer than the instruction caches are.
                auto tile = [&](auto masked, auto uneven) {
                    constexpr bool kMasked = decltype(masked)::value, kUneven = decltype(uneven)::value;
                    float top = -INFINITY, top2 = -INFINITY, lift = 1.0f;
                    // (keys of usual sizes: the power of two may wait)
                    if constexpr (CODES) {
                        const PowerParts parts = power_parts(p.scale_size, exponent);
                        lift = parts.first;
                        factor = kUneven ? parts.rest : p.scale_size * power_of_two(max(exponent, -126));
                    }
#pragma unroll 1
                    for (int c = 0; c < KT / 32; ++c) {
                        uint32_t s[32];
                        tmem_ld32(scores + 32 * c, s);
                        tmem_ld_wait(s);
                        if (CODES) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                if (kUneven)
#pragma unroll
                                    for (int n = 0; n < 4; ++n) s[i + n] = __float_as_uint(__uint_as_float(s[i + n]) * lift);
                                const float4 k = *(const float4*)(of_keys + 32 * c + i);
                                const Pair a = pair_mul(pair_of(s[i], s[i + 1]), pair_of(k.x, k.y)), b = pair_mul(pair_of(s[i + 2], s[i + 3]), pair_of(k.z, k.w));
                                s[i] = __float_as_uint(pair_at(a, 0)); s[i + 1] = __float_as_uint(pair_at(a, 1)); s[i + 2] = __float_as_uint(pair_at(b, 0)); s[i + 3] = __float_as_uint(pair_at(b, 1));
                            }
                        }
                        if (kMasked) {
                            const uint32_t on = shown(c);
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                s[i] = on >> i & 1 ? s[i] : 0xff800000u;
                                if (kUneven) s[i] = __float_as_uint(fmaf(__uint_as_float(s[i]), factor, exponent_of(of_values[32 * c + i])));  // (each scale's exponent counts)
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            top = fmaxf(fmaxf(top, __uint_as_float(s[i])), __uint_as_float(s[i + 1]));
                            top2 = fmaxf(fmaxf(top2, __uint_as_float(s[i + 2])), __uint_as_float(s[i + 3]));
                        }
                    }
                    top = kUneven ? fmaxf(base, fmaxf(top, top2) - kRaise<TYPE>) : fmaxf(base, fmaf(fmaxf(top, top2), factor, (float)level - kRaise<TYPE>));
                    const float from = top == -INFINITY ? 0.0f : top;
                    f = exp2_fast(base - from);
                    base = top;
                    const Pair down = pair_of(-from, -from), factors = pair_of(factor, factor), minus = pair_of(-1.0f, -1.0f);
                    Pair add[2] = {pair_of(0.0f, 0.0f), pair_of(0.0f, 0.0f)};
#pragma unroll 1
                    for (int c = 0; c < KT / 32; ++c) {
                        uint32_t s[32];
                        tmem_ld32(scores + 32 * c, s);
                        tmem_ld_wait(s);
                        const uint32_t on = kMasked ? shown(c) : 0;
                        uint32_t hi[16], mid[16], lo[16];
                        float4 two_keys, two_values;  // the scales of two pairs
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            if (CODES) {
                                if (!(i & 1)) {
                                    two_keys = *(const float4*)(of_keys + 32 * c + 2 * i);
                                    two_values = *(const float4*)(of_values + 32 * c + 2 * i);
                                }
                                if (kUneven) {
                                    s[2 * i] = __float_as_uint(__uint_as_float(s[2 * i]) * lift);
                                    s[2 * i + 1] = __float_as_uint(__uint_as_float(s[2 * i + 1]) * lift);
                                }
                                const Pair scaled = pair_mul(pair_of(s[2 * i], s[2 * i + 1]), i & 1 ? pair_of(two_keys.z, two_keys.w) : pair_of(two_keys.x, two_keys.y));
                                s[2 * i] = __float_as_uint(pair_at(scaled, 0));
                                s[2 * i + 1] = __float_as_uint(pair_at(scaled, 1));
                            }
                            if (kMasked) {
                                s[2 * i] = on >> (2 * i) & 1 ? s[2 * i] : 0xff800000u;
                                s[2 * i + 1] = on >> (2 * i + 1) & 1 ? s[2 * i + 1] : 0xff800000u;
                            }
                            const Pair x = pair_fma(pair_of(s[2 * i], s[2 * i + 1]), factors, down);
                            float a = exp2_fast(pair_at(x, 0)), b = exp2_fast(pair_at(x, 1));
                            Pair v = pair_of(a, b);
                            add[i & 1] = pair_add(add[i & 1], v);
                            if (CODES) {
                                v = pair_mul(v, i & 1 ? pair_of(two_values.z, two_values.w) : pair_of(two_values.x, two_values.y));
                                a = pair_at(v, 0);
                                b = pair_at(v, 1);
                                if (kUneven) {  // (a scale that the row does not see may be infinite, and 0 * inf is no 0)
                                    a = on >> (2 * i) & 1 ? a : 0.0f;
                                    b = on >> (2 * i + 1) & 1 ? b : 0.0f;
                                    v = pair_of(a, b);
                                }
                            }
                            hi[i] = rqattn::pair_of<TYPE>(a, b);
                            v = pair_fma(pair_of(to_float<TYPE>((uint16_t)hi[i]), to_float<TYPE>((uint16_t)(hi[i] >> 16))), minus, v);
                            mid[i] = rqattn::pair_of<TYPE>(pair_at(v, 0), pair_at(v, 1));
                            if (PARTS == 3) {
                                v = pair_fma(pair_of(to_float<TYPE>((uint16_t)mid[i]), to_float<TYPE>((uint16_t)(mid[i] >> 16))), minus, v);
                                lo[i] = rqattn::pair_of<TYPE>(pair_at(v, 0), pair_at(v, 1));
                            }
                        }
                        tmem_st16(scores + 32 * c, hi);
                        tmem_st16(scores + 32 * c + 16, mid);
                        if (PARTS == 3) tmem_st16(lo_at + 16 * c, lo);
                        if (c == KT / 64 - 1) weights_there(0);  // the tensor core may begin with the first half
                    }
                    add[0] = pair_add(add[0], add[1]);
                    sum = fmaf(sum, f, pair_at(add[0], 0) + pair_at(add[0], 1));
                };
                if (CODES && !__all_sync(0xffffffffu, even)) tile(std::true_type(), std::bool_constant<CODES>());
                else if (__all_sync(0xffffffffu, all)) tile(std::false_type(), std::false_type());
                else tile(std::true_type(), std::false_type());
                weights_there(1);
                // behind the last scores the queries' place is free: the next item's, before this one's sums are finished
                if (j + 1 == tiles) {
                    if (KEYS && !mbar_wait_warp(&sh.q_empty, items_done & 1, p.wait_ns, dead)) atomicExch(p.error_flag, 43);
                    item_at.next();
                    following = next_item();
                    if (following) queries(*following, items_done + 1);
                }
                old = f;
                ++tiles_done;
            }
            keys_before += (KEYS ? 2 : 1) * tiles;
            if ((!KEYS || pipe == 0) && lane == 0) mbar_arrive(&sh.t_empty[pipe]);

            // ---- the row is finished, or this CTA's part of it -----------------------------------------
            if (KEYS) {
                // the second pipe leaves its sums where its tiles' sums were; the first one joins them
                if (pipe == 1) {
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t t[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) t[i] = __float_as_uint(o[16 * c + i]);
                        tmem_st16(sums_at + 16 * c, t);
                    }
                    tmem_st_wait();
                    sh.joint[0][row] = base;
                    sh.joint[1][row] = sum;
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.joined[quarter]);
                } else {
                    if (!mbar_wait_warp(&sh.joined[quarter], items_done & 1, p.wait_ns, dead)) atomicExch(p.error_flag, 52);
                    fence_after();
                    const float other = sh.joint[0][row], top = fmaxf(base, other), to = top == -INFINITY ? 0.0f : top;
                    const float fa = exp2_fast(base - to), fb = exp2_fast(other - to);
                    sum = sum * fa + sh.joint[1][row] * fb;
                    base = top;
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t t[32];
                        tmem_ld32(sums_at + D + 32 * c, t);
                        tmem_ld_wait(t);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[32 * c + i] = o[32 * c + i] * fa + __uint_as_float(t[i]) * fb;
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.t_empty[1]);
                }
            }
            if (!KEYS || pipe == 0) {
                const int at = it->row0 + in_block, first_cta = it->first_cta, last_cta = it->last_cta;
                const bool active = in_block < it->rows;
                float* y = p.y + (active ? (int64_t)(it->start + at / group) * p.y_stride + (int64_t)(it->kv * group + at % group) * D : 0);
                auto put = [&]() {
                    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
                    if (!active) return;
                    if (p.wide & 2) {
#pragma unroll
                        for (int i = 0; i < D; i += 8) store32(y + i, o + i, inverse);
                    } else {
#pragma unroll
                        for (int i = 0; i < D; ++i) y[i] = o[i] * inverse;
                    }
                };
                if (first_cta == last_cta) {
                    put();
                } else {
                    // [CTA][first or last of its items][pipe]: sums four elements a row, bases, sums of weights
                    constexpr int64_t PART = 128 * (D + 2);
                    auto part = [&](int cta) { return p.partial + (((int64_t)cta * 2 + (cta == first_cta)) * 2 + pipe) * PART; };
                    const int mine = row * 4;
                    float* to = part((int)blockIdx.x);
#pragma unroll
                    for (int i = 0; i < D; i += 4) __stcg((float4*)(to + mine + i * 128), make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]));
                    __stcg(to + 128 * D + row, base);
                    __stcg(to + 128 * (D + 1) + row, sum);
                    // (a warp's rows are joined by themselves: it waits for no other warp of its CTA)
                    uint32_t* const count = p.arrived + (first_cta * 2 + pipe) * 4 + quarter;
                    __threadfence();
                    __syncwarp();
                    uint32_t before = 0;
                    if (lane == 0) before = atomicAdd(count, 1);
                    if (__shfl_sync(0xffffffffu, before, 0) == (uint32_t)(last_cta - first_cta)) {
                        if (lane == 0) *count = 0;
                        __threadfence();
                        base = -INFINITY;
                        for (int c = first_cta; c <= last_cta; ++c) base = fmaxf(base, __ldcg(part(c) + 128 * D + row));
                        const float at_all = base == -INFINITY ? 0.0f : base;
                        sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < D; ++i) o[i] = 0.0f;
                        for (int c = first_cta; c <= last_cta; ++c) {
                            const float* from = part(c);
                            const float f = exp2_fast(__ldcg(from + 128 * D + row) - at_all);
                            sum = fmaf(__ldcg(from + 128 * (D + 1) + row), f, sum);
#pragma unroll
                            for (int i = 0; i < D; i += 4) {
                                const float4 v = __ldcg((const float4*)(from + mine + i * 128));
                                o[i] = fmaf(v.x, f, o[i]);
                                o[i + 1] = fmaf(v.y, f, o[i + 1]);
                                o[i + 2] = fmaf(v.z, f, o[i + 2]);
                                o[i + 3] = fmaf(v.w, f, o[i + 3]);
                            }
                        }
                        put();
                    }
                }
            }
            // (the ring of items is already at the following one)
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.item_empty[it - sh.items]);
            it = following;
            ++items_done;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::OTHER_REGS));
    }
    if (CODES && warp >= kMender) {
        // ------------------------------------------------------------ the widening warps (nothing is mended: a code is a number)
        if (warp >= kWidener) widen(warp - kWidener);
    } else if (warp == kIssuer) {
        // ------------------------------------------------------------ the issuing warp
        Ring at(STAGES);
        uint32_t sums[2] = {0, 0}, item_count = 0;
        const uint32_t q_at = smem_u32(smem), ring_at = smem_u32(ring);
        constexpr uint32_t kFormat = TYPE == RQ_KV_F16 ? 0u : (1u << 7 | 1u << 10);  // of A and B: f16, bf16
        const uint32_t scores_desc = instr_desc(KT) | kFormat, sums_desc = instr_desc(D) | kFormat | 1u << 16;  // (bit 16: B is given elements first)
        auto arrived = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_warp(bar, parity, p.wait_ns, dead); };
        auto take_slot = [&]() {
            const int slot = at.slot;
            if (!arrived(&sh.full[slot], at.phase)) atomicExch(p.error_flag, 45);
            at.next();
            return slot;
        };
        auto issue_scores = [&](int pipe, int slot) {
            fence_after();
            if (elect_one() && !dead) {
                const uint64_t b = smem_desc(ring_at + slot * F::TILE_BYTES);
#pragma unroll
                for (int part = PARTS - 1; part >= 0; --part) {
                    const uint64_t a = smem_desc(q_at + ((KEYS ? 0 : pipe * PARTS) + part) * F::Q_PART);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        mma_f16_ss(tmem + pipe * KT, a + (k >> 2) * (128 * 128 >> 4) + 2 * (k & 3), b + (k >> 2) * (KT * 128 >> 4) + 2 * (k & 3), scores_desc, part < PARTS - 1 || k > 0);
                }
                mma_commit(&sh.s_full[pipe]);
            }
            __syncwarp();
        };
        auto issue_sums = [&](int pipe, int slot) {
            if (!arrived(&sh.t_empty[pipe], (sums[pipe] & 1) ^ 1)) atomicExch(p.error_flag, 48);
            const uint64_t b = values_desc(ring_at + slot * F::TILE_BYTES, KT * 128);
            const uint32_t to = tmem + F::T_COL + pipe * D, weights = tmem + pipe * KT, third = tmem + F::LO_COL + pipe * (KT / 2);
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // of the tile's keys
                if (!arrived(&sh.p_full[pipe][half], sums[pipe] & 1)) atomicExch(p.error_flag, 47);
                fence_after();
                if (elect_one() && !dead) {
                    constexpr int N = KT / 32;  // steps of sixteen keys
                    if (PARTS == 3)
#pragma unroll
                        for (int k = half * N; k < (half + 1) * N; ++k) mma_f16_ts(to, third + 8 * k, b + k * (16 * 128 >> 4), sums_desc, k > 0);
#pragma unroll
                    for (int part = 1; part >= 0; --part)
#pragma unroll
                        for (int k = half * N; k < (half + 1) * N; ++k)
                            mma_f16_ts(to, weights + 32 * (k >> 1) + 16 * part + 8 * (k & 1), b + k * (16 * 128 >> 4), sums_desc, PARTS == 3 || part == 0 || k > 0);
                    if (half) mma_commit(&sh.t_full[pipe]);
                }
                __syncwarp();
            }
            ++sums[pipe];
        };
        // (once a wait has run out nothing is handed on: who waits for it gives up as well, and no barrier sees an arrival that it does not expect)
        auto release = [&](uint64_t* bar) {
            if (elect_one() && !dead) mma_commit(bar);
            __syncwarp();
        };
        while (const Item* it = next_item()) {
            const int tiles = it->take;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.item_empty[item_at.slot]);
            item_at.next();
            if (!arrived(&sh.q_full[0], item_count & 1)) atomicExch(p.error_flag, 46);
            int slot = take_slot();
            issue_scores(0, slot);
            if (KEYS) {
                release(&sh.empty[slot]);
                slot = take_slot();
            } else {
                if (!arrived(&sh.q_full[1], item_count & 1)) atomicExch(p.error_flag, 46);
            }
            issue_scores(1, slot);
            release(&sh.empty[slot]);
            if (KEYS && tiles == 1) release(&sh.q_empty);
            for (int j = 0; j < tiles; ++j) {
                const bool another = j + 1 < tiles;
                int values = take_slot(), keys = 0;
                issue_sums(0, values);
                if (KEYS) release(&sh.empty[values]);
                if (another) {
                    keys = take_slot();
                    issue_scores(0, keys);
                    if (KEYS) release(&sh.empty[keys]);
                }
                if (KEYS) values = take_slot();
                issue_sums(1, values);
                release(&sh.empty[values]);
                if (another) {
                    if (KEYS) keys = take_slot();
                    issue_scores(1, keys);
                    release(&sh.empty[keys]);
                    if (KEYS && j + 2 == tiles) release(&sh.q_empty);
                }
            }
            ++item_count;
        }
        // nothing may be in flight when tensor memory is freed
        dead = false;
        release(&sh.ended);
        if (!arrived(&sh.ended, 0)) atomicExch(p.error_flag, 49);
    } else if (warp == kFetcher) {
        // ------------------------------------------------------------ the items' queries, into L2 ahead of their use
        while (const Item* it = next_item()) {
            for (int row = lane; row < it->rows; row += 32) {
                const int at = it->row0 + row;
                const char* q = (const char*)(p.q + (int64_t)(it->start + at / group) * p.q_stride + (int64_t)(it->kv * group + at % group) * D);
#pragma unroll
                for (int line = 0; line < D * 4; line += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + line));
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.item_empty[item_at.slot]);
            item_at.next();
        }
    } else if (warp == kMender) {
        // ------------------------------------------------------------ tiles of values that not every row sees, between their arrival and their use: past the keys that
        // some row sees they become zeros (a page's end may never have been written), and what is not finite is taken out (0 * inf is no 0)
        Ring at(STAGES);
        uint32_t value_tiles = 0, phases = 0;  // phases: a bit a slot
        while (const Item* it = next_item()) {
            const int tiles = it->take * (KEYS ? 2 : 1);
            for (int n = 0; n < 2 * tiles; ++n, at.next()) {
                if (!is_values(n, tiles)) continue;
                const int key0 = it->first_key + tile_of(n, tiles) * KT, slot = at.slot;
                if (is_edge(*it, key0)) {
                    if (!mbar_wait_warp(&sh.landed[slot], phases >> slot & 1, p.wait_ns, dead)) atomicExch(p.error_flag, 51);
                    if (dead) break;  // (the tile may be on its way: it is not touched, and not handed on)
                    phases ^= 1u << slot;
                    const int first = min(max(it->low - key0, 0), KT), last = min(max(it->high - key0, 0), KT);
                    constexpr uint32_t kExponent = TYPE == RQ_KV_F16 ? 0x7c007c00u : 0x7f807f80u, kCarry = 0x80008000u - kExponent;
                    bool fine = true;
                    // (a line's chunks are looked at in any order: the swizzle does not matter)
#pragma unroll 4
                    for (int c = lane; c < KT * (D / 8); c += 32) {
                        const int line = c / 8 % KT;
                        uint4* v = (uint4*)(ring + slot * F::TILE_BYTES + c * 16);
                        const uint4 was = *v;
                        const uint32_t bad = (((was.x & kExponent) + kCarry) | ((was.y & kExponent) + kCarry) | ((was.z & kExponent) + kCarry) | ((was.w & kExponent) + kCarry)) & 0x80008000u;
                        if (line < first || line >= last) {
                            *v = make_uint4(0, 0, 0, 0);
                        } else if (bad) {
                            uint32_t x[4] = {was.x, was.y, was.z, was.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[e] &= (finite16(x[e], TYPE) ? 0xffffu : 0) | (finite16(x[e] >> 16, TYPE) ? 0xffff0000u : 0);
                            *v = make_uint4(x[0], x[1], x[2], x[3]);
                            fine = false;
                        }
                    }
                    if (!__all_sync(0xffffffffu, fine) && lane == 0) sh.odd[value_tiles % kWords] = 1;
                    fence_to_tensor_core();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.full[slot]);
                }
                ++value_tiles;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.item_empty[item_at.slot]);
            item_at.next();
        }
    } else if (warp == kLoader) {
        // ------------------------------------------------------------ the loading warp: deals the items out, and copies their tiles in the order of their use
        const int64_t total = sh.warp_sums[0], ctas = sh.warp_sums[1], end = sh.range[1];
        int64_t u = sh.range[0];
        int r = sh.where[0], b = sh.where[1], kv = sh.where[2], offset = sh.where[3];
        auto deal = [&]() {
            if (!mbar_wait_warp(&sh.item_empty[item_at.slot], item_at.phase ^ 1, p.wait_ns, dead)) atomicExch(p.error_flag, 50);
            Item i = {};
            if (u < end && !dead) {
                const Block k = block_of<F>(p, r, b, group);
                const int64_t item_begin = u - offset, item_end = item_begin + F::LEAD + k.units;
                const int first_unit = max(offset - F::LEAD, 0);
                u = min(item_end, end);
                i.take = max((int)(u - item_begin) - F::LEAD - first_unit, 0);  // (none where a range ends in a block's lead: the next CTA has it all)
                i.first_key = k.begin + first_unit * F::UNIT;
                i.low = k.low; i.high = k.high; i.end = k.end; i.start = k.start; i.row0 = k.row0; i.rows = k.rows; i.position0 = k.position0; i.kv = kv; i.r = r;
                const bool all = offset <= F::LEAD && u == item_end;  // nobody else's
                i.first_cta = all ? blockIdx.x : (int)(((item_begin + F::LEAD + 1) * ctas - 1) / total);
                i.last_cta = all ? blockIdx.x : (int)((item_end * ctas - 1) / total);
                offset = 0;
                if (++kv == p.kv_heads) {
                    kv = 0;
                    if (++b >= blocks_of<F>(p, r, group)) {
                        b = 0;
                        do ++r; while (r < p.requests - 1 && blocks_of<F>(p, r, group) == 0);
                    }
                }
            }
            if (lane == 0 && !dead) {
                sh.items[item_at.slot] = i;
                mbar_arrive(&sh.item_full[item_at.slot]);
            }
            item_at.next();
            return i;
        };
        const int box_shift = min(p.page_shift, CODES ? kCodesShift : (KT == 128 ? 7 : 6)), boxes = KT >> box_shift;  // a copy brings 64 elements of a page, or of a tile
        const int box = lane & (boxes - 1), column = lane / boxes;                               // this lane's copy
        Ring at(STAGES);
        uint32_t key_tiles = 0, value_tiles = 0;
        uint32_t landings = 0;  // a bit a slot: the parity of its next copies that go to the mending warp
        Item following = deal();
        while (following.take && !dead) {
            const Item i = following;
            const int tiles = i.take * (KEYS ? 2 : 1);
            const int32_t* table = p.block_table + (int64_t)i.r * p.table_stride;
            auto page_of = [&](int tile) -> int {  // of this lane's copy; one past the last for none: such a copy reads zeros
                const int key = i.first_key + tile * KT + (box << box_shift);
                const int page = key < i.high && key + (1 << box_shift) > i.low ? __ldcg(table + (key >> p.page_shift)) : -1;
                return page < 0 || page >= p.pages ? (int)p.pages : page;
            };
            int page = page_of(0);
#pragma unroll 1
            for (int n = 0; n < 2 * tiles; ++n) {
                const bool values = is_values(n, tiles);
                const int tile = tile_of(n, tiles), key0 = i.first_key + tile * KT, slot = at.slot;
                const int now = page;
                if (n + 1 < 2 * tiles) page = page_of(tile_of(n + 1, tiles));
                if (!mbar_wait_warp(&sh.empty[slot], at.phase ^ 1, p.wait_ns, dead)) atomicExch(p.error_flag, 44);
                if (dead) break;  // (a slot that never came free is not armed again)
                if (!values) {
                    const uint32_t ok = __ballot_sync(0xffffffffu, now < p.pages || lane >= boxes), all = boxes == 32 ? 0xffffffffu : (1u << boxes) - 1;
                    // (keys past the last one that some row sees have no page here: they are masked by their position)
                    uint32_t word = ok & all;
                    const int in_range = min(max((i.high - key0 + (1 << box_shift) - 1) >> box_shift, 0), boxes), before = min(max(i.low - key0, 0) >> box_shift, boxes);
                    word |= all & ~((1u << in_range) - 1);
                    word |= (1u << before) - 1;
                    if (lane == 0) sh.pages_there[key_tiles % kWords] = word == all ? 0xffffffffu : word;
                    ++key_tiles;
                }
                if (values) {
                    if (lane == 0) sh.odd[value_tiles % kWords] = 0;
                    ++value_tiles;
                }
                uint64_t* bar = &sh.full[slot];
                if (CODES || (values && is_edge(i, key0))) {  // (to the mending or the widening warps first, which hand it on)
                    bar = &sh.landed[slot];
                    landings ^= 1u << slot;
                }
                if (lane == 0) mbar_expect_tx(bar, F::LANDED_BYTES);
                __syncwarp();
                if (column < (CODES ? 1 : D / 64)) {
                    const uint32_t to = smem_u32(ring) + slot * F::TILE_BYTES + (CODES ? D / 64 - 1 : column) * (KT * 128) + box * (128 << box_shift) + (CODES && D == 64 ? 64 << box_shift : 0);
                    tma_load_4d(to, values ? &v_map : &k_map, column * 64, (key0 + (box << box_shift)) & ((1 << p.page_shift) - 1), i.kv, now, bar);
                }
                __syncwarp();
                at.next();
                if (n == 1) following = deal();  // ahead of its use: its queries are fetched while this one's tiles are
            }
        }
        // Every copy has landed before the CTA ends, whoever gave up: the last ones to the mending warp, and the last ones of each slot (a barrier that nothing was
        // counted by looks as if it had; where the mending warp gave up, a slot's own wait runs out)
#pragma unroll 1
        for (int n = 0; n < 2 * STAGES; ++n) {
            const int slot = n >> 1;
            bool late = false;
            if (n & 1) mbar_wait_warp(&sh.landed[slot], (landings >> slot & 1) ^ 1, p.wait_ns, late);
            else mbar_wait_warp(&sh.full[slot], slot < at.slot ? at.phase : at.phase ^ 1, p.wait_ns, late);
        }
    }
    fence_before();
    __syncthreads();
    if (warp == kIssuer) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <int D, int TYPE, bool KEYS, bool CODES = false>
int launch_form(rq_ctx* ctx, const CodesParams& p, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
    using F = Form<D, TYPE, KEYS, CODES>;
    auto kernel = rq_attention_tc_kernel<D, TYPE, KEYS, CODES>;
    constexpr size_t smem = F::Q_BYTES + F::STAGES * F::TILE_BYTES + sizeof(Shared<F>);
    static_assert(smem <= 227 * 1024, "shared memory");
    static bool configured[64] = {};  // by device: the opt-in to large shared memory
    if (ctx->device >= 64 || !configured[ctx->device]) {
        RQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        if (ctx->device < 64) configured[ctx->device] = true;
    }
    const int ctas = ctx->sm_count < kTensorCtas ? ctx->sm_count : kTensorCtas;
    return launch(kernel, dim3((unsigned)ctas), F::THREADS, smem, s, (const typename F::Params&)p, k, v);
}

// The cache as a TMA reads it: elements, lines, heads, pages; a copy is 64 elements of `lines` lines, swizzled as the tensor core reads them (codes: whole lines, as they are)
int make_map(CUtensorMap* map, const void* base, const rq_kv_cache& c, int lines) {
    rq_encode_tiled encode = nullptr;
    const int rc = rq_tensor_map_encoder(&encode);
    if (rc) return rc;
    const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_size, (cuuint64_t)c.heads, (cuuint64_t)c.pages};
    const bool codes = c.type == RQ_KV_INT8;
    const cuuint64_t bytes = codes ? 1 : 2;
    const cuuint64_t strides[3] = {bytes * (cuuint64_t)c.line_stride, c.heads > 1 ? bytes * (cuuint64_t)c.head_stride : 16, c.pages > 1 ? bytes * (cuuint64_t)c.page_stride : 16};
    const cuuint32_t box[4] = {codes ? (cuuint32_t)c.head_dim : 64, (cuuint32_t)lines, 1, 1}, step[4] = {1, 1, 1, 1};
    const CUresult e = encode(map, codes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, (void*)base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              codes ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (e != CUDA_SUCCESS) return rq_fail(RQ_ERR_CUDA, "rq_attention: cuTensorMapEncodeTiled failed with %d", (int)e);
    return RQ_OK;
}

}  // namespace

int rqattn::launch_tensor(rq_ctx* ctx, const CodesParams& p, const rq_kv_cache& c, bool one_tile, cudaStream_t s) {
    // pages of whole groups of eight lines (the swizzle's), and strides that a tensor map can hold
    if (c.head_dim > 128 || c.page_size < 8 || c.line_stride <= 0 || (c.heads > 1 && c.head_stride <= 0) || (c.pages > 1 && c.page_stride <= 0) || c.head_stride >= (int64_t)1 << 38) return RQ_ERR_UNSUPPORTED;
    const int tile = c.type == RQ_KV_INT8 ? 1 << kCodesShift : (c.type == RQ_KV_F16 || c.head_dim == 64 ? 128 : 64), lines = c.page_size < tile ? c.page_size : tile;
    alignas(64) CUtensorMap k, v;
    int rc = make_map(&k, c.k, c, lines);
    if (!rc) rc = make_map(&v, c.v, c, lines);
    if (rc) return rc;
    if (c.type == RQ_KV_INT8) {
        if (c.head_dim == 64) return one_tile ? launch_form<64, RQ_KV_F16, true, true>(ctx, p, k, v, s) : launch_form<64, RQ_KV_F16, false, true>(ctx, p, k, v, s);
        return one_tile ? launch_form<128, RQ_KV_F16, true, true>(ctx, p, k, v, s) : launch_form<128, RQ_KV_F16, false, true>(ctx, p, k, v, s);
    }
    if (c.type == RQ_KV_BF16) return c.head_dim == 64 ? launch_form<64, RQ_KV_BF16, true>(ctx, p, k, v, s) : launch_form<128, RQ_KV_BF16, true>(ctx, p, k, v, s);
    if (c.head_dim == 64) return one_tile ? launch_form<64, RQ_KV_F16, true>(ctx, p, k, v, s) : launch_form<64, RQ_KV_F16, false>(ctx, p, k, v, s);
    return one_tile ? launch_form<128, RQ_KV_F16, true>(ctx, p, k, v, s) : launch_form<128, RQ_KV_F16, false>(ctx, p, k, v, s);
}
