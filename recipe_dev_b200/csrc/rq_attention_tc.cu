// Attention of chunks and prompts over the paged cache: rows by the hundred, on the 5th-generation tensor cores.
//
// A row is one query head of one new token; the rows of the heads that share a key head lie together, tokens after tokens, so that they
// meet a tile of keys and values together. A CTA has two PIPES, each with 128 rows' scores and sums in tensor memory and a
// warpgroup of softmax threads (a thread has one row to itself):
//   rows form (f16): the pipes are two tiles of 128 rows, which share every tile of 128 keys;
//   keys form (few rows; bf16, whose third parts leave no room for a second row tile): one row tile, the pipes take alternate tiles of keys and
//     are joined at the end, through tensor memory.
// Per tile of keys: S = Q K^T (tcgen05.mma, Q and K in shared memory), weights P = 2^(S - max) from and to tensor memory, T = P V (P in tensor memory,
// V in shared memory as it lies in the cache, keys times elements), sums O = O 2^(old max - max) + T in fp32 registers.
//   * fp32 activations: Q and P are taken apart into 16-bit parts (hi + lo over f16, 22 bits; hi + mid + lo over bf16), each part a
//     product of its own into the same accumulator, the smallest first. Products double (treble) against 16-bit activations; with one part the
//     results would be off by 2^-11 (2^-8) where the framework's fp32 activations are good for 1e-6.
//   * The tensor core adds by truncation: T is one tile's sum only, and O is added up with round-to-nearest.
//   * P takes the place of its S in tensor memory, 32 keys' hi and lo parts over the 32 scores they came from.
// The issuing warp's order is Q K_A(j + 1), P V_B(j), Q K_B(j + 1), P V_A(j + 1), ..: while the tensor core is busy with one pipe's
// products the other pipe's softmax runs.
//
// Work is counted in units, one tile of keys (keys form: two) of one block of rows; every CTA takes an equal range of them, wherever it begins and ends, and
// rows whose keys fall to several CTAs are joined in CTA order by the last of these (the same bits on every run).
//
// Every wait is bounded; a wait that runs out records a code in the context's error word and the warp waits no more.
#include <type_traits>

#include "rq_attention.cuh"
#include "rq_mma.cuh"
#include "rq_pairs.cuh"

using namespace rqserve;
using namespace rqattn;
using namespace rqmma;

namespace {

constexpr int kSoftmaxWarps = 8, kLoadWarps = 4, kIssuer = 12, kDealer = 13, kThreads = 512;  // warps 14 and 15 complete a warpgroup
constexpr int kSoftmaxRegs = 208, kOtherRegs = 48;                // 2 * 208 + 2 * 48 = 4 * 128, what the block is launched with
constexpr int kOdd = 32;                                          // ring of "a value that some row does not see is not finite"

template <int D, int TYPE, bool KEYS_> struct Form {
    static constexpr bool KEYS = KEYS_;
    static constexpr int PARTS = TYPE == RQ_KV_F16 ? 2 : 3;
    static constexpr int KT = TYPE == RQ_KV_F16 || D == 64 ? 128 : 64;  // keys a tile (bf16, 128 elements: 2 KT + 2 D + KT columns are what tensor memory holds with 64)
    static constexpr int TILE_BYTES = KT * D * 2, Q_PART = 128 * D * 2, Q_BYTES = (KEYS ? 1 : 2) * PARTS * Q_PART;
    static constexpr int STAGES_FIT = (227 * 1024 - 3072 - Q_BYTES) / TILE_BYTES, STAGES = STAGES_FIT > 8 ? 8 : STAGES_FIT;
    static constexpr int BLOCK = KEYS ? 128 : 256;                      // rows
    static constexpr int UNIT = KEYS ? 2 * KT : KT;                     // keys
    static constexpr int T_COL = 2 * KT, LO_COL = T_COL + 2 * D;        // tensor memory: scores (then weights), tile sums, bf16's third parts
    static_assert(STAGES >= (KEYS ? 4 : 3), "ring");
    static_assert(LO_COL + (PARTS == 3 ? KT : 0) <= 512, "tensor memory");
};

// A block of rows of one request and key head, and the keys that some row of it sees
struct Block {
    int start, fresh, row0, rows, position0, begin, low, high, end;  // keys [low, high), from the tile at begin; end: the request's keys
    int units;
};
template <typename F> __device__ __forceinline__ int blocks_of(const AttentionParams& p, int r, int group) {
    return (max(p.starts[r + 1] - p.starts[r], 0) * group + F::BLOCK - 1) / F::BLOCK;
}
template <typename F> __device__ __forceinline__ Block block_of(const AttentionParams& p, int r, int b, int group) {
    Block k;
    k.start = p.starts[r];
    k.fresh = max(p.starts[r + 1] - k.start, 0);
    const int length = p.lengths[r];
    k.end = (int)min((int64_t)max(length, 0), (int64_t)p.table_width << p.page_shift);
    k.position0 = length - k.fresh;
    k.row0 = b * F::BLOCK;
    k.rows = min(F::BLOCK, k.fresh * group - k.row0);
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
constexpr int kItems = 4;  // a ring of them in shared memory, filled ahead by a warp of its own

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
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
                 "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16_start(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                   "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
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
__device__ __forceinline__ void load32(const float* p, float (&x)[8]) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]) : "l"(p) : "memory");
}
__device__ __forceinline__ void store32(float* p, const float* x, float f) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0] * f), "f"(x[1] * f), "f"(x[2] * f), "f"(x[3] * f), "f"(x[4] * f), "f"(x[5] * f), "f"(x[6] * f),
                 "f"(x[7] * f)
                 : "memory");
}
// a look that does not wait
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_to_tensor_core() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void warpgroup_sync(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool finite16(uint32_t v, int type) { const uint32_t e = type == RQ_KV_F16 ? 0x7c00u : 0x7f80u; return (v & e) != e; }

template <typename F> struct Shared {
    uint64_t full[F::STAGES], empty[F::STAGES], item_full[kItems], item_empty[kItems], q_full[2], s_full[2], p_full[2][2], t_full[2], t_empty[2], q_free, ended;
    int64_t warp_sums[kThreads / 32], range[2];
    int where[4];
    Item items[kItems];
    uint32_t valid[kOdd][F::KT / 32];  // which keys of a tile lie on a page of the cache and are seen by some row
    uint32_t odd[kOdd], arrival[2], tmem_slot;
    float joint[2][F::KEYS ? 128 : 1];  // keys form: the second pipe's maximum and sum of each row
};

template <int D, int TYPE, bool KEYS>
__global__ void __launch_bounds__(kThreads, 1) rq_attention_tc_kernel(AttentionParams p) {
    using F = Form<D, TYPE, KEYS>;
    constexpr int PARTS = F::PARTS, KT = F::KT, STAGES = F::STAGES, LEAD = KEYS ? 2 : 1;
    extern __shared__ __align__(1024) unsigned char dynamic[];
    uint8_t* const smem = dynamic;  // (there is no other shared memory in front of it)
    uint8_t* const ring = smem + F::Q_BYTES;
    auto& sh = *(Shared<F>*)(ring + STAGES * F::TILE_BYTES);
    auto& full = sh.full;
    auto& empty = sh.empty;
    auto& item_full = sh.item_full;
    auto& item_empty = sh.item_empty;
    auto& q_full = sh.q_full;
    auto& s_full = sh.s_full;
    auto& p_full = sh.p_full;
    auto& t_full = sh.t_full;
    auto& t_empty = sh.t_empty;
    auto& q_free = sh.q_free;
    auto& ended = sh.ended;
    auto& odd = sh.odd;
    auto& valid = sh.valid;
    auto& items = sh.items;
    auto& joint = sh.joint;
    auto& warp_sums = sh.warp_sums;
    auto& range = sh.range;
    auto& where = sh.where;
    auto& arrival = sh.arrival;
    auto& tmem_slot = sh.tmem_slot;
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int group = p.q_heads / p.kv_heads;

    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], kLoadWarps); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], KEYS ? 8 : 4); mbar_init(&s_full[i], 1); mbar_init(&p_full[i][0], 4); mbar_init(&p_full[i][1], 4); mbar_init(&t_full[i], 1); mbar_init(&t_empty[i], 4); }
        for (int i = 0; i < kItems; ++i) { mbar_init(&item_full[i], 1); mbar_init(&item_empty[i], kSoftmaxWarps + kLoadWarps + 1); }
        mbar_init(&q_free, 1);
        mbar_init(&ended, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid < kOdd) odd[tid] = 0;
    if (warp == kIssuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    launch_dependents();
    wait_for_previous();

    // ---- where this CTA's units lie: requests' units are added up once, a request a thread and round ------
    {
        int64_t* const before = (int64_t*)smem;  // (the queries' place; at most 32 KB)
        int64_t total = 0;
        if (tid == 0) before[0] = 0;
        for (int r0 = 0; r0 < p.requests; r0 += kThreads) {
            const int r = r0 + tid;
            int64_t units = 0;
            if (r < p.requests)
                for (int b = blocks_of<F>(p, r, group) - 1; b >= 0; --b) units += block_of<F>(p, r, b, group).units;
            units *= p.kv_heads;
            int64_t scan = units;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) { const int64_t o = __shfl_up_sync(0xffffffffu, scan, off); if (lane >= off) scan += o; }
            __syncthreads();
            if (lane == 31) warp_sums[warp] = scan;
            __syncthreads();
            scan += total;
            for (int w = 0; w < kThreads / 32; ++w) { if (w < warp) scan += warp_sums[w]; total += warp_sums[w]; }
            if (r < p.requests) before[r + 1] = scan;
        }
        __syncthreads();
        if (tid == 0) {
            const int64_t ctas = min((int64_t)gridDim.x, total), u = blockIdx.x < ctas ? blockIdx.x * total / ctas : 0;
            range[0] = blockIdx.x < ctas ? u : 0;
            range[1] = blockIdx.x < ctas ? (blockIdx.x + 1) * total / ctas : 0;
            int r = 0, b = 0;
            for (int hi = p.requests - 1; r < hi;) { const int mid = (r + hi + 1) >> 1; if (before[mid] <= u) r = mid; else hi = mid - 1; }
            int64_t left = u - before[r];
            int units = 1;
            if (total)
                while (true) {
                    units = block_of<F>(p, r, b, group).units;
                    if (left < (int64_t)units * p.kv_heads) break;
                    left -= (int64_t)units * p.kv_heads;
                    ++b;
                }
            where[0] = r;
            where[1] = b;
            where[2] = (int)(left / units);
            where[3] = (int)(left % units);
            warp_sums[0] = total;
            warp_sums[1] = ctas;
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    // The CTA's items, one after another: each role waits for one, reads what it needs of it and gives it back
    Ring item_at(kItems);
    bool dead = false;
    auto next_item = [&]() -> const Item* {
        if (!mbar_wait_warp(&item_full[item_at.slot], item_at.phase, p.wait_ns, dead)) atomicExch(p.error_flag, 40);
        const Item* i = &items[item_at.slot];
        return !dead && i->take ? i : nullptr;
    };
    auto item_done = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[item_at.slot]);
        item_at.next();
    };

    if (warp < kSoftmaxWarps) {
        // ------------------------------------------------------------ softmax: a thread a row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int pipe = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t rows_at = (uint32_t)((warp & 3) * 32) << 16, scores = tmem + rows_at + pipe * KT, sums_at = tmem + rows_at + F::T_COL + pipe * D,
                       lo_at = tmem + rows_at + F::LO_COL + pipe * (KT / 2);
        const int in_block = KEYS ? row : pipe * 128 + row;
        uint32_t tiles_done = 0, ring_tiles = 0;  // ring_tiles: of the items before
        bool odd_item = false;
        const float scale = p.scale * kLog2e;

        // this thread's query (keys form: its pipe's half of it) into shared memory, taken apart
        auto load_query = [&](const Item& it) {
            const bool active = in_block < it.rows;
            const int at = it.row0 + in_block;
            const float* from = p.q + (active ? (int64_t)(it.start + at / group) * p.q_stride + (int64_t)(it.kv * group + at % group) * D : 0);
            uint8_t* const to = smem + (KEYS ? 0 : pipe * PARTS * F::Q_PART);
            constexpr int CHUNKS = KEYS ? D / 16 : D / 8, BATCH = 4;  // chunks of eight elements, four on their way at a time
#pragma unroll 1
            for (int i0 = 0; i0 < CHUNKS; i0 += BATCH) {
                const int c0 = (KEYS ? pipe * CHUNKS : 0) + i0;
                float x[BATCH][8];
                if (!active) {
#pragma unroll
                    for (int i = 0; i < BATCH; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[i][e] = 0.0f;
                } else if (p.wide & 2) {
#pragma unroll
                    for (int i = 0; i < BATCH; ++i) load32(from + 8 * (c0 + i), x[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < BATCH; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[i][e] = __ldcg(from + 8 * (c0 + i) + e);
                }
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const int c = c0 + i;
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[i][e] *= scale;
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) {
                        uint4 v;
                        v.x = take_pair<TYPE>(x[i][0], x[i][1]);
                        v.y = take_pair<TYPE>(x[i][2], x[i][3]);
                        v.z = take_pair<TYPE>(x[i][4], x[i][5]);
                        v.w = take_pair<TYPE>(x[i][6], x[i][7]);
                        *(uint4*)(to + part * F::Q_PART + (c >> 3) * (128 * 128) + swizzled(row, c & 7)) = v;
                    }
                }
            }
            fence_to_tensor_core();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[KEYS ? 0 : pipe]);
        };

        float o[D];
        const Item* it = next_item();
        if (it) load_query(*it);
        while (it) {
            const int tiles = it->take;
            int low, high;  // the keys that this thread's row sees
            {
                const int position = it->position0 + (it->row0 + in_block) / group;
                high = in_block < it->rows ? min(position + 1, it->end) : 0;
                low = p.window > 0 ? max(position - p.window + 1, 0) : 0;
            }
            float m = -INFINITY, sum = 0.0f, old = 1.0f;
#pragma unroll
            for (int i = 0; i < D; ++i) o[i] = 0.0f;

            // The values of a tile that are not finite, to the sums of the rows that see them
            auto add_odd = [&](const Item& of, int key0) {
                const int32_t* table = p.block_table + (int64_t)of.r * p.table_stride;
                for (int key = max(key0, of.low); key < min(key0 + KT, of.high); ++key) {
                    const int page = __ldcg(table + (key >> p.page_shift));
                    if (page < 0 || page >= p.pages) continue;
                    const uint16_t* v = p.v + of.kv * p.head_stride + (int64_t)page * (p.page_bytes / 2) + (int64_t)(key & ((1 << p.page_shift) - 1)) * (p.line_bytes / 2);
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
            const Item* following = nullptr;
            int key0 = it->first_key + (KEYS ? pipe * KT : 0);
            constexpr int kStep = (KEYS ? 2 : 1) * KT;
#pragma unroll 1
            for (int j = 0;; ++j, key0 += kStep) {
                float f = 1.0f;
                if (j > 0) {
                    // O = O f + T, the sums of this pipe's tile before, while the tensor core makes the next one's scores
                    if (!mbar_wait_warp(&t_full[pipe], (tiles_done - 1) & 1, p.wait_ns, dead)) atomicExch(p.error_flag, 41);
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
                    // (the loading warps took what is not finite out of the tile)
                    const int i = KEYS ? 2 * (j - 1) + pipe : j - 1, values = KEYS ? min(2 * i + 2, 4 * tiles - 1) : 2 * i + 1;
                    if (*(volatile uint32_t*)&odd[(ring_tiles + values) % kOdd]) add_odd(*it, key0 - kStep);
                    if (j == tiles) break;
                    if (lane == 0) mbar_arrive(&t_empty[pipe]);
                }
                if (j < tiles) {
                    if (!mbar_wait_warp(&s_full[pipe], tiles_done & 1, p.wait_ns, dead)) atomicExch(p.error_flag, 42);
                    fence_after();
                    const int i = KEYS ? 2 * j + pipe : j, keys = KEYS ? (i < 2 ? i : 2 * i - 1) : 2 * i;
                    const volatile uint32_t* there = valid[(ring_tiles + keys) % kOdd];
                    bool all = key0 >= low && key0 + KT <= high;
#pragma unroll
                    for (int c = 0; c < KT / 32; ++c) all = all && there[c] == 0xffffffffu;
                    // the columns of 32 keys that this row sees
                    auto shown = [&](int c) -> uint32_t {
                        const int a = min(max(high - key0 - 32 * c, 0), 32), b = min(max(low - key0 - 32 * c, 0), 32);
                        return there[c] & (a == 32 ? 0xffffffffu : (1u << a) - 1) & ~(b == 32 ? 0xffffffffu : (1u << b) - 1);
                    };
                    auto weights_there = [&](int half) {
                        tmem_st_wait();
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_full[pipe][half]);
                    };
                    // The loops over columns are loops: laid out in a line, with the masks, they were longer than the instruction caches are.
                    auto tile = [&](auto masked) {
                        constexpr bool kMasked = decltype(masked)::value;
                        float top = m, top2 = -INFINITY;
#pragma unroll 1
                        for (int c = 0; c < KT / 32; ++c) {
                            uint32_t s[32];
                            tmem_ld32(scores + 32 * c, s);
                            tmem_ld_wait(s);
                            if (kMasked) {
                                const uint32_t on = shown(c);
#pragma unroll
                                for (int i = 0; i < 32; ++i) s[i] = on >> i & 1 ? s[i] : 0xff800000u;
                            }
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                top = fmaxf(fmaxf(top, __uint_as_float(s[i])), __uint_as_float(s[i + 1]));
                                top2 = fmaxf(fmaxf(top2, __uint_as_float(s[i + 2])), __uint_as_float(s[i + 3]));
                            }
                        }
                        top = fmaxf(top, top2);
                        const float base = (top == -INFINITY ? 0.0f : top) - kRaise;
                        f = exp2_fast(m - (base + kRaise));
                        m = top;
                        const Pair down = pair_of(-base, -base), minus = pair_of(-1.0f, -1.0f);
                        Pair add[2] = {pair_of(0.0f, 0.0f), pair_of(0.0f, 0.0f)};
                        // sixteen columns' weights, in parts
                        auto weigh = [&](uint32_t (&s)[16], uint32_t on, uint32_t (&hi)[8], uint32_t (&mid)[8], uint32_t (&lo)[8]) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                if (kMasked) {
                                    s[2 * i] = on >> (2 * i) & 1 ? s[2 * i] : 0xff800000u;
                                    s[2 * i + 1] = on >> (2 * i + 1) & 1 ? s[2 * i + 1] : 0xff800000u;
                                }
                                const Pair x = pair_add(pair_of(s[2 * i], s[2 * i + 1]), down);
                                const float a = exp2_fast(pair_at(x, 0)), b = exp2_fast(pair_at(x, 1));
                                Pair v = pair_of(a, b);
                                add[i & 1] = pair_add(add[i & 1], v);
                                hi[i] = rqattn::pair_of<TYPE>(a, b);
                                v = pair_fma(pair_of(to_float<TYPE>((uint16_t)hi[i]), to_float<TYPE>((uint16_t)(hi[i] >> 16))), minus, v);
                                mid[i] = rqattn::pair_of<TYPE>(pair_at(v, 0), pair_at(v, 1));
                                if (PARTS == 3) {
                                    v = pair_fma(pair_of(to_float<TYPE>((uint16_t)mid[i]), to_float<TYPE>((uint16_t)(mid[i] >> 16))), minus, v);
                                    lo[i] = rqattn::pair_of<TYPE>(pair_at(v, 0), pair_at(v, 1));
                                }
                            }
                        };
                        uint32_t s0[16], s1[16], hi[8], mid[8], lo[8];
                        tmem_ld16_start(scores, s0);
#pragma unroll 1
                        for (int c = 0; c < KT / 32; ++c) {
                            const uint32_t at = scores + 32 * c, on = kMasked ? shown(c) : 0;
                            tmem_ld16_wait(s0);
                            tmem_ld16_start(at + 16, s1);
                            weigh(s0, on, hi, mid, lo);
                            tmem_ld16_wait(s1);  // (they lie where some of these weights go)
                            if (c + 1 < KT / 32) tmem_ld16_start(at + 32, s0);
                            tmem_st8(at, hi);
                            tmem_st8(at + 16, mid);
                            if (PARTS == 3) tmem_st8(lo_at + 16 * c, lo);
                            weigh(s1, on >> 16, hi, mid, lo);
                            tmem_st8(at + 8, hi);
                            tmem_st8(at + 24, mid);
                            if (PARTS == 3) tmem_st8(lo_at + 16 * c + 8, lo);
                            if (c == KT / 64 - 1) weights_there(0);  // the tensor core may begin with the first half
                        }
                        add[0] = pair_add(add[0], add[1]);
                        sum = fmaf(sum, f, pair_at(add[0], 0) + pair_at(add[0], 1));
                    };
                    if (__all_sync(0xffffffffu, all)) tile(std::false_type());
                    else tile(std::true_type());
                    weights_there(1);
                    // behind the last scores the queries' place is free: the next item's, before this one's sums are finished
                    if (j + 1 == tiles) {
                        if (KEYS && !mbar_wait_warp(&q_free, odd_item, p.wait_ns, dead)) atomicExch(p.error_flag, 43);
                        item_at.next();
                        following = next_item();
                        if (following) load_query(*following);
                    }
                }
                old = f;
                ++tiles_done;
            }
            odd_item = !odd_item;
            ring_tiles += (KEYS ? 4 : 2) * tiles;

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
                    joint[0][row] = m;
                    joint[1][row] = sum;
                    fence_before();
                    asm volatile("bar.sync 3, 256;" ::: "memory");
                } else {
                    asm volatile("bar.sync 3, 256;" ::: "memory");
                    fence_after();
                    const float other = joint[0][row], top = fmaxf(m, other), base = top == -INFINITY ? 0.0f : top;
                    const float fa = exp2_fast(m - base), fb = exp2_fast(other - base);
                    sum = sum * fa + joint[1][row] * fb;
                    m = top;
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
                    if (lane == 0) mbar_arrive(&t_empty[1]);
                }
            }
            if (!KEYS || pipe == 0) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&t_empty[pipe]);
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
                    // [CTA][first or last of its items][pipe]: sums four elements a row, maxima, sums of weights
                    constexpr int64_t PART = 128 * (D + 2);
                    auto part = [&](int cta) { return p.partial + (((int64_t)cta * 2 + (cta == first_cta)) * 2 + pipe) * PART; };
                    float* to = part((int)blockIdx.x);
#pragma unroll
                    for (int i = 0; i < D; i += 4) __stcg((float4*)(to + (i / 4 * 128 + row) * 4), make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]));
                    __stcg(to + 128 * D + row, m);
                    __stcg(to + 128 * (D + 1) + row, sum);
                    __threadfence();
                    warpgroup_sync(1 + pipe);
                    if (row == 0) arrival[pipe] = atomicAdd(&p.arrived[first_cta * 2 + pipe], 1);
                    warpgroup_sync(1 + pipe);
                    if (arrival[pipe] == (uint32_t)(last_cta - first_cta)) {
                        if (row == 0) p.arrived[first_cta * 2 + pipe] = 0;
                        __threadfence();
                        m = -INFINITY;
                        for (int c = first_cta; c <= last_cta; ++c) m = fmaxf(m, __ldcg(part(c) + 128 * D + row));
                        const float base = m == -INFINITY ? 0.0f : m;
                        sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < D; ++i) o[i] = 0.0f;
                        for (int c = first_cta; c <= last_cta; ++c) {
                            const float* from = part(c);
                            const float f = exp2_fast(__ldcg(from + 128 * D + row) - base);
                            sum = fmaf(__ldcg(from + 128 * (D + 1) + row), f, sum);
#pragma unroll
                            for (int i = 0; i < D; i += 4) {
                                const float4 v = __ldcg((const float4*)(from + (i / 4 * 128 + row) * 4));
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
            // (the ring's place after this item's is the one in hand)
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[it - items]);
            it = following;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp < kIssuer) {
            // ------------------------------------------------------------ loads: tiles of keys and values, in the order in which they are used
            constexpr int CHUNKS = D / 8, LINES = 32 / CHUNKS, PASS = LINES * kLoadWarps;  // 16-byte chunks a line; lines a warp and all of them copy at a time
            const int loader = warp - kSoftmaxWarps, chunk = lane % CHUNKS, line0 = loader * LINES + lane / CHUNKS;
            const uint32_t ring_at = smem_u32(ring) + (chunk >> 3) * (KT * 128);
            Ring at(STAGES);
            uint32_t n = 0, pending_n = 0;  // tiles so far; the one whose copies are under way
            bool pending = false, pending_look = false;
            int pending_slot = 0;
            // A tile's copies have landed: hand it on. Values that some row does not see are looked at first: what is not finite (0 * inf is no 0)
            // is taken out here and met by the softmax threads.
            auto hand_on = [&]() {
                if (pending_look) {
                    bool fine = true;
#pragma unroll 1
                    for (int i = 0; i < KT / PASS; ++i) {
                        uint4* v = (uint4*)(ring + pending_slot * F::TILE_BYTES + (chunk >> 3) * (KT * 128) + swizzled(i * PASS + line0, chunk & 7));
                        const uint4 was = *v;
                        uint32_t x[4] = {was.x, was.y, was.z, was.w};
                        bool ok = true;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t keep = (finite16(x[e], TYPE) ? 0xffffu : 0) | (finite16(x[e] >> 16, TYPE) ? 0xffff0000u : 0);
                            ok = ok && keep == 0xffffffffu;
                            x[e] &= keep;
                        }
                        if (!ok) { *v = make_uint4(x[0], x[1], x[2], x[3]); fine = false; }
                    }
                    if (!__all_sync(0xffffffffu, fine) && lane == 0) odd[pending_n % kOdd] = 1;
                }
                fence_to_tensor_core();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[pending_slot]);
                pending = false;
            };
            const int line_mask = (1 << p.page_shift) - 1;
            while (const Item* it = next_item()) {
                const int32_t* table = p.block_table + (int64_t)it->r * p.table_stride;
                const int tiles = it->take * (KEYS ? 2 : 1), first_key = it->first_key, seen_low = it->low, seen_high = it->high;
                const int64_t head = it->kv * p.head_stride + 8 * chunk;
                // the keys that every row sees
                const int common_high = min(it->end, it->position0 + it->row0 / group + 1);
                const int common_low = p.window > 0 ? it->position0 + (it->row0 + it->rows - 1) / group - p.window + 1 : 0;
                item_done();
                int entry[KT / 32];  // lane l: the pages of keys l, l + 32, .. of the tile that is loaded next, -1 for none
                auto entries = [&](int key0) {
#pragma unroll
                    for (int i = 0; i < KT / 32; ++i) {
                        const int key = key0 + 32 * i + lane, e = key >= seen_low && key < seen_high ? __ldcg(table + (key >> p.page_shift)) : -1;
                        entry[i] = e < p.pages ? max(e, -1) : -1;
                    }
                };
                auto load = [&](int key0, bool values, int next_key0) {
                    if (!__all_sync(0xffffffffu, mbar_test(&empty[at.slot], at.phase ^ 1))) {
                        if (pending) {  // what has landed must not wait for a slot
                            asm volatile("cp.async.wait_all;" ::: "memory");
                            hand_on();
                        }
                        if (!mbar_wait_warp(&empty[at.slot], at.phase ^ 1, p.wait_ns, dead)) atomicExch(p.error_flag, 44);
                    }
                    if (loader == 0 && lane == 0) odd[(n + STAGES) % kOdd] = 0;
                    const char* base = (const char*)((values ? p.v : p.k) + head);
                    if (loader == 0 && !values) {
#pragma unroll
                        for (int i = 0; i < KT / 32; ++i) { const uint32_t ok = __ballot_sync(0xffffffffu, entry[i] >= 0); if (lane == 0) valid[n % kOdd][i] = ok; }
                    }
                    const uint32_t to = ring_at + at.slot * F::TILE_BYTES;
#pragma unroll
                    for (int i = 0; i < KT / PASS; ++i) {
                        const int line = i * PASS + line0, page = __shfl_sync(0xffffffffu, entry[i * PASS / 32], line & 31);
                        const char* from = base + (uint64_t)(uint32_t)max(page, 0) * p.page_bytes + (uint64_t)(uint32_t)((key0 + line) & line_mask) * p.line_bytes;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + swizzled(line, chunk & 7)), "l"(from), "r"(page >= 0 ? 16 : 0) : "memory");
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    entries(next_key0);
                    if (pending) {
                        asm volatile("cp.async.wait_group 1;" ::: "memory");
                        hand_on();
                    }
                    pending = true;
                    pending_slot = at.slot;
                    pending_n = n;
                    pending_look = values && (key0 < common_low || key0 + KT > common_high);
                    at.next();
                    ++n;
                };
                entries(first_key);
                if (KEYS) {
                    load(first_key, false, first_key + KT);
                    load(first_key + KT, false, first_key);
                } else {
                    load(first_key, false, first_key);
                }
                for (int i = 0; i < tiles; ++i) {
                    const int key0 = first_key + i * KT;
                    const bool another = i + LEAD < tiles;
                    load(key0, true, another ? key0 + LEAD * KT : key0 + KT);
                    if (another) load(key0 + LEAD * KT, false, key0 + KT);
                }
            }
            if (pending) {
                asm volatile("cp.async.wait_all;" ::: "memory");
                hand_on();
            }
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
                if (!arrived(&full[slot], at.phase)) atomicExch(p.error_flag, 45);
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
                    mma_commit(&s_full[pipe]);
                }
                __syncwarp();
            };
            auto issue_sums = [&](int pipe, int slot) {
                if (!arrived(&t_empty[pipe], (sums[pipe] & 1) ^ 1)) atomicExch(p.error_flag, 48);
                const uint64_t b = values_desc(ring_at + slot * F::TILE_BYTES, KT * 128);
                const uint32_t to = tmem + F::T_COL + pipe * D, weights = tmem + pipe * KT, third = tmem + F::LO_COL + pipe * (KT / 2);
#pragma unroll
                for (int half = 0; half < 2; ++half) {  // of the tile's keys
                    if (!arrived(&p_full[pipe][half], sums[pipe] & 1)) atomicExch(p.error_flag, 47);
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
                        if (half) mma_commit(&t_full[pipe]);
                    }
                    __syncwarp();
                }
                ++sums[pipe];
            };
            auto release = [&](uint64_t* bar) {
                if (elect_one()) mma_commit(bar);
                __syncwarp();
            };
            while (const Item* it = next_item()) {
                const int tiles = it->take;
                item_done();
                if (!arrived(&q_full[0], item_count & 1)) atomicExch(p.error_flag, 46);
                int slot = take_slot();
                issue_scores(0, slot);
                if (KEYS) {
                    release(&empty[slot]);
                    slot = take_slot();
                } else {
                    if (!arrived(&q_full[1], item_count & 1)) atomicExch(p.error_flag, 46);
                }
                issue_scores(1, slot);
                release(&empty[slot]);
                if (KEYS && tiles == 1) release(&q_free);
                for (int j = 0; j < tiles; ++j) {
                    const bool another = j + 1 < tiles;
                    int values = take_slot(), keys = 0;
                    issue_sums(0, values);
                    if (KEYS) release(&empty[values]);
                    if (another) {
                        keys = take_slot();
                        issue_scores(0, keys);
                        if (KEYS) release(&empty[keys]);
                    }
                    if (KEYS) values = take_slot();
                    issue_sums(1, values);
                    release(&empty[values]);
                    if (another) {
                        if (KEYS) keys = take_slot();
                        issue_scores(1, keys);
                        release(&empty[keys]);
                        if (KEYS && j + 2 == tiles) release(&q_free);
                    }
                }
                ++item_count;
            }
            // nothing may be in flight when tensor memory is freed
            release(&ended);
            dead = false;
            if (!arrived(&ended, 0)) atomicExch(p.error_flag, 49);
        } else if (warp == kDealer) {
            // ------------------------------------------------------------ the items, ahead of their use
            const int64_t total = warp_sums[0], ctas = warp_sums[1], end = range[1];
            int64_t u = range[0];
            int r = where[0], b = where[1], kv = where[2], offset = where[3];
            while (true) {
                if (!mbar_wait_warp(&item_empty[item_at.slot], item_at.phase ^ 1, p.wait_ns, dead)) atomicExch(p.error_flag, 50);
                Item i = {};
                if (u < end && !dead) {
                    const Block k = block_of<F>(p, r, b, group);
                    i.take = (int)min((int64_t)(k.units - offset), end - u);
                    i.first_key = k.begin + offset * F::UNIT;
                    i.low = k.low; i.high = k.high; i.end = k.end; i.start = k.start; i.row0 = k.row0; i.rows = k.rows; i.position0 = k.position0; i.kv = kv; i.r = r;
                    const int64_t item_begin = u - offset, item_end = item_begin + k.units;
                    i.first_cta = (int)(((item_begin + 1) * ctas - 1) / total);
                    i.last_cta = (int)((item_end * ctas - 1) / total);
                    u += i.take;
                    offset = 0;
                    for (int row = lane; row < k.rows; row += 32) {  // its queries, into L2: they are read when the item begins
                        const char* q = (const char*)(p.q + (int64_t)(k.start + (k.row0 + row) / group) * p.q_stride + (int64_t)(kv * group + (k.row0 + row) % group) * D);
#pragma unroll
                        for (int line = 0; line < D * 4; line += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + line));
                    }
                    if (++kv == p.kv_heads) {
                        kv = 0;
                        if (++b >= blocks_of<F>(p, r, group)) {
                            b = 0;
                            do ++r; while (r < p.requests - 1 && blocks_of<F>(p, r, group) == 0);
                        }
                    }
                }
                if (lane == 0) {
                    items[item_at.slot] = i;
                    mbar_arrive(&item_full[item_at.slot]);
                }
                item_at.next();
                if (!i.take) break;
            }
        }
    }
    fence_before();
    __syncthreads();
    if (warp == kIssuer) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <int D, int TYPE, bool KEYS>
int launch_form(rq_ctx* ctx, const AttentionParams& p, cudaStream_t s) {
    using F = Form<D, TYPE, KEYS>;
    auto kernel = rq_attention_tc_kernel<D, TYPE, KEYS>;
    constexpr size_t smem = F::Q_BYTES + F::STAGES * F::TILE_BYTES + sizeof(Shared<F>);
    static_assert(smem <= 227 * 1024, "shared memory");
    static bool allowed = false;
    if (!allowed) {
        RQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        allowed = true;
    }
    const int ctas = ctx->sm_count < kTensorCtas ? ctx->sm_count : kTensorCtas;
    return launch(kernel, dim3((unsigned)ctas), kThreads, smem, s, p);
}

}  // namespace

int rqattn::launch_tensor(rq_ctx* ctx, const AttentionParams& p, int head_dim, int type, bool one_tile, cudaStream_t s) {
    if (type == RQ_KV_BF16) return head_dim == 64 ? launch_form<64, RQ_KV_BF16, true>(ctx, p, s) : launch_form<128, RQ_KV_BF16, true>(ctx, p, s);
    if (head_dim == 64) return one_tile ? launch_form<64, RQ_KV_F16, true>(ctx, p, s) : launch_form<64, RQ_KV_F16, false>(ctx, p, s);
    return one_tile ? launch_form<128, RQ_KV_F16, true>(ctx, p, s) : launch_form<128, RQ_KV_F16, false>(ctx, p, s);
}
