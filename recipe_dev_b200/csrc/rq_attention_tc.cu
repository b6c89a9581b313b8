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
#include "rq_attention.cuh"
#include "rq_mma.cuh"
#include "rq_pairs.cuh"

using namespace rqserve;
using namespace rqattn;
using namespace rqmma;

namespace {

constexpr int kSoftmaxWarps = 8, kLoadWarps = 4, kThreads = 512;  // and the issuing warp; three warps complete its warpgroup
constexpr int kSoftmaxRegs = 208, kOtherRegs = 48;                // 2 * 208 + 2 * 48 = 4 * 128, what the block is launched with
constexpr int kOdd = 32;                                          // ring of "a value that some row does not see is not finite"

template <int D, int TYPE, bool KEYS> struct Form {
    static constexpr int PARTS = TYPE == RQ_KV_F16 ? 2 : 3;
    static constexpr int KT = TYPE == RQ_KV_F16 || D == 64 ? 128 : 64;  // keys a tile (bf16, 128 elements: 2 KT + 2 D + KT columns are what tensor memory holds with 64)
    static constexpr int TILE_BYTES = KT * D * 2, Q_PART = 128 * D * 2, Q_BYTES = (KEYS ? 1 : 2) * PARTS * Q_PART;
    static constexpr int STAGES_FIT = (227 * 1024 - 2048 - Q_BYTES) / TILE_BYTES, STAGES = STAGES_FIT > 8 ? 8 : STAGES_FIT;
    static constexpr int BLOCK = KEYS ? 128 : 256;                      // rows
    static constexpr int UNIT = KEYS ? 2 * KT : KT;                     // keys
    static constexpr int T_COL = 2 * KT, LO_COL = T_COL + 2 * D;        // tensor memory: scores (then weights), tile sums, bf16's third parts
    static constexpr int SMEM = 1024 + Q_BYTES + STAGES * TILE_BYTES;
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

// The blocks of a CTA's range of units, one after another; every role walks it for itself
template <typename F> struct Walk {
    const AttentionParams& p;
    int group, r, b, kv, offset, take;
    int64_t u, end;
    Block k;
    __device__ Walk(const AttentionParams& p_, int r_, int b_, int kv_, int offset_, int64_t u_, int64_t end_)
        : p(p_), group(p_.q_heads / p_.kv_heads), r(r_), b(b_), kv(kv_ - 1), offset(offset_), take(0), u(u_), end(end_) {}
    __device__ bool next() {
        u += take;
        if (u >= end) return false;
        if (take) offset = 0;
        if (++kv == p.kv_heads) {
            kv = 0;
            if (++b >= blocks_of<F>(p, r, group)) {
                b = 0;
                do ++r; while (r < p.requests - 1 && blocks_of<F>(p, r, group) == 0);
            }
        }
        k = block_of<F>(p, r, b, group);
        take = (int)min((int64_t)(k.units - offset), end - u);
        return true;
    }
    __device__ int first_key() const { return k.begin + offset * F::UNIT; }
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

template <int D, int TYPE, bool KEYS>
__global__ void __launch_bounds__(kThreads, 1) rq_attention_tc_kernel(AttentionParams p) {
    using F = Form<D, TYPE, KEYS>;
    constexpr int PARTS = F::PARTS, KT = F::KT, STAGES = F::STAGES, LEAD = KEYS ? 2 : 1;
    extern __shared__ __align__(16) unsigned char dynamic[];
    uint8_t* const smem = (uint8_t*)(((uintptr_t)dynamic + 1023) & ~(uintptr_t)1023);
    uint8_t* const ring = smem + F::Q_BYTES;
    __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], q_full[2], q_free, s_full[2], p_full[2], t_full[2], t_empty[2], ended;
    __shared__ uint32_t tmem_slot, odd[kOdd], arrival[2];
    __shared__ int64_t warp_sums[kThreads / 32], range[2];
    __shared__ int where[4];
    __shared__ float joint[2][128];  // keys form: the second pipe's maximum and sum of each row
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int group = p.q_heads / p.kv_heads;

    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], kLoadWarps); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], KEYS ? 8 : 4); mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&t_full[i], 1); mbar_init(&t_empty[i], 4); }
        mbar_init(&q_free, 1);
        mbar_init(&ended, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid < kOdd) odd[tid] = 0;
    if (warp == kSoftmaxWarps + kLoadWarps) {
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
    const int64_t total = warp_sums[0], ctas = warp_sums[1];
    Walk<F> walk(p, where[0], where[1], where[2], where[3], range[0], range[1]);

    if (warp < kSoftmaxWarps) {
        // ------------------------------------------------------------ softmax: a thread a row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int pipe = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t rows_at = (uint32_t)((warp & 3) * 32) << 16, scores = tmem + rows_at + pipe * KT, sums_at = tmem + rows_at + F::T_COL + pipe * D,
                       lo_at = tmem + rows_at + F::LO_COL + pipe * (KT / 2);
        const int in_block = KEYS ? row : pipe * 128 + row;
        bool dead = false;
        uint32_t tiles_done = 0, items_done = 0, ring_tiles = 0;  // ring_tiles: of the items before
        const float scale = p.scale * kLog2e;

        // this thread's query (keys form: its pipe's half of it) into shared memory, taken apart
        auto load_query = [&](const Walk<F>& w) {
            const bool active = in_block < w.k.rows;
            const int at = w.k.row0 + in_block;
            const float* from = p.q + (active ? (int64_t)(w.k.start + at / group) * p.q_stride + (int64_t)(w.kv * group + at % group) * D : 0);
            uint8_t* const to = smem + (KEYS ? 0 : pipe * PARTS * F::Q_PART);
            constexpr int CHUNKS = KEYS ? D / 16 : D / 8;
#pragma unroll 4
            for (int i = 0; i < CHUNKS; ++i) {
                const int c = KEYS ? pipe * CHUNKS + i : i;
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 0.0f;
                if (active) {
                    if (p.wide) {
                        const float4 a = __ldcg((const float4*)(from + 8 * c)), b = __ldcg((const float4*)(from + 8 * c + 4));
                        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = __ldcg(from + 8 * c + e);
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= scale;
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    uint4 v;
                    v.x = take_pair<TYPE>(x[0], x[1]);
                    v.y = take_pair<TYPE>(x[2], x[3]);
                    v.z = take_pair<TYPE>(x[4], x[5]);
                    v.w = take_pair<TYPE>(x[6], x[7]);
                    *(uint4*)(to + part * F::Q_PART + (c >> 3) * (128 * 128) + swizzled(row, c & 7)) = v;
                }
            }
            fence_to_tensor_core();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[KEYS ? 0 : pipe]);
        };

        float o[D];
        bool more = walk.next();
        if (more) load_query(walk);
        while (more) {
            const Walk<F> w = walk;  // this item; `walk` goes on to the next one when its query is due
            const Block& k = w.k;
            const int at = k.row0 + in_block, position = k.position0 + at / group;
            const bool active = in_block < k.rows;
            const int high = active ? min(position + 1, k.end) : 0, low = p.window > 0 ? max(position - p.window + 1, 0) : 0;
            const int32_t* table = p.block_table + (int64_t)w.r * p.table_stride;
            float m = -INFINITY, sum = 0.0f, old = 1.0f;
#pragma unroll
            for (int i = 0; i < D; ++i) o[i] = 0.0f;

            // which of a tile's keys lie on a page of the cache: 32 keys a word
            int entry[KT / 32];
            auto entries = [&](int key0) {
#pragma unroll
                for (int i = 0; i < KT / 32; ++i) {
                    const int key = key0 + 32 * i + lane;
                    entry[i] = key >= k.low && key < k.high ? __ldcg(table + (key >> p.page_shift)) : -1;
                }
            };
            // The values of a tile that are not finite, to the sums of the rows that see them
            auto add_odd = [&](int key0) {
                for (int key = max(key0, k.low); key < min(key0 + KT, k.high); ++key) {
                    const int page = __ldcg(table + (key >> p.page_shift));
                    if (page < 0 || page >= p.pages) continue;
                    const uint16_t* v = p.v + w.kv * p.head_stride + (int64_t)page * (p.page_bytes / 2) + (int64_t)(key & ((1 << p.page_shift) - 1)) * (p.line_bytes / 2);
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
            auto add_tile = [&](int key0, int j, float f) {
                if (!mbar_wait_warp(&t_full[pipe], (tiles_done - 1) & 1, p.wait_ns, dead)) atomicExch(p.error_flag, 41);
                fence_after();
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t t[32];
                    tmem_ld32(sums_at + 32 * c, t);
                    tmem_ld_wait(t);
                    const Pair ff = pair_of(f, f);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const Pair v = pair_fma(pair_of(o[32 * c + i], o[32 * c + i + 1]), ff, pair_of(t[i], t[i + 1]));
                        o[32 * c + i] = pair_at(v, 0);
                        o[32 * c + i + 1] = pair_at(v, 1);
                    }
                }
                fence_before();
                __syncwarp();
                // (the loading warps took what is not finite out of the tile)
                const int i = KEYS ? 2 * j + pipe : j, values = KEYS ? min(2 * i + 2, 4 * w.take - 1) : 2 * i + 1;
                if (*(volatile uint32_t*)&odd[(ring_tiles + values) % kOdd]) add_odd(key0);
            };
            const int stride = KEYS ? 2 : 1, tiles = w.take;  // this pipe's
            int key0 = w.first_key() + (KEYS ? pipe * KT : 0);
            entries(key0);
            for (int j = 0; j < tiles; ++j, key0 += stride * KT) {
                uint32_t there[KT / 32];
                bool all = key0 >= low && key0 + KT <= high;
#pragma unroll
                for (int i = 0; i < KT / 32; ++i) { there[i] = __ballot_sync(0xffffffffu, entry[i] >= 0 && entry[i] < p.pages); all = all && there[i] == 0xffffffffu; }
                if (j + 1 < tiles) entries(key0 + stride * KT);
                const bool plain = __all_sync(0xffffffffu, all);
                if (!mbar_wait_warp(&s_full[pipe], tiles_done & 1, p.wait_ns, dead)) atomicExch(p.error_flag, 42);
                fence_after();
                // the columns of 32 keys that this row sees
                auto shown = [&](int c) -> uint32_t {
                    const int a = min(max(high - key0 - 32 * c, 0), 32), b = min(max(low - key0 - 32 * c, 0), 32);
                    return there[c] & (a == 32 ? 0xffffffffu : (1u << a) - 1) & ~(b == 32 ? 0xffffffffu : (1u << b) - 1);
                };
                float top = m;
#pragma unroll
                for (int c = 0; c < KT / 32; ++c) {
                    uint32_t s[32];
                    tmem_ld32(scores + 32 * c, s);
                    tmem_ld_wait(s);
                    if (plain) {
#pragma unroll
                        for (int i = 0; i < 32; i += 2) top = fmaxf(fmaxf(top, __uint_as_float(s[i])), __uint_as_float(s[i + 1]));
                    } else {
                        const uint32_t on = shown(c);
#pragma unroll
                        for (int i = 0; i < 32; ++i) top = fmaxf(top, on >> i & 1 ? __uint_as_float(s[i]) : -INFINITY);
                    }
                }
                const float base = (top == -INFINITY ? 0.0f : top) - kRaise, f = exp2_fast(m - (base + kRaise));
                m = top;
                const Pair down = pair_of(-base, -base), minus = pair_of(-1.0f, -1.0f);
                Pair add = pair_of(0.0f, 0.0f);
#pragma unroll
                for (int c = 0; c < KT / 32; ++c) {
                    uint32_t s[32], hi[16], mid[16], lo[PARTS == 3 ? 16 : 1];
                    tmem_ld32(scores + 32 * c, s);
                    tmem_ld_wait(s);
                    if (!plain) {
                        const uint32_t on = shown(c);
#pragma unroll
                        for (int i = 0; i < 32; ++i) s[i] = on >> i & 1 ? s[i] : 0xff800000u;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const Pair x = pair_add(pair_of(s[2 * i], s[2 * i + 1]), down);
                        const float a = exp2_fast(pair_at(x, 0)), b = exp2_fast(pair_at(x, 1));
                        Pair v = pair_of(a, b);
                        add = pair_add(add, v);
                        hi[i] = rqattn::pair_of<TYPE>(a, b);
                        v = pair_fma(pair_of(to_float<TYPE>((uint16_t)hi[i]), to_float<TYPE>((uint16_t)(hi[i] >> 16))), minus, v);
                        mid[i] = rqattn::pair_of<TYPE>(pair_at(v, 0), pair_at(v, 1));
                        if (PARTS == 3) {
                            v = pair_fma(pair_of(to_float<TYPE>((uint16_t)mid[i]), to_float<TYPE>((uint16_t)(mid[i] >> 16))), minus, v);
                            lo[PARTS == 3 ? i : 0] = rqattn::pair_of<TYPE>(pair_at(v, 0), pair_at(v, 1));
                        }
                    }
                    tmem_st16(scores + 32 * c, hi);
                    tmem_st16(scores + 32 * c + 16, mid);
                    if (PARTS == 3) tmem_st16(lo_at + 16 * c, lo);
                }
                sum = fmaf(sum, f, pair_at(add, 0) + pair_at(add, 1));
                tmem_st_wait();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[pipe]);
                // behind the last scores the query's place is free: the next item's, before this one's sums are finished
                if (j + 1 == tiles) {
                    if (KEYS) {
                        if (!mbar_wait_warp(&q_free, items_done & 1, p.wait_ns, dead)) atomicExch(p.error_flag, 43);
                    }
                    more = walk.next();
                    if (more) load_query(walk);
                }
                if (j > 0) {
                    add_tile(key0 - stride * KT, j - 1, old);
                    if (lane == 0) mbar_arrive(&t_empty[pipe]);
                }
                old = f;
                ++tiles_done;
            }
            add_tile(key0 - stride * KT, tiles - 1, old);
            ++items_done;
            ring_tiles += (KEYS ? 4 : 2) * w.take;

            // ---- the row is finished, or this CTA's part of it -----------------------------------------
            bool mine = true;
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
                    mine = false;
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
            }
            if (mine) {
                const int64_t item_begin = w.u - w.offset, item_end = item_begin + k.units;
                const int64_t first_cta = ((item_begin + 1) * ctas - 1) / total, last_cta = (item_end * ctas - 1) / total;
                float* y = p.y + (active ? (int64_t)(k.start + at / group) * p.y_stride + (int64_t)(w.kv * group + at % group) * D : 0);
                auto put = [&]() {
                    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
                    if (!active) return;
                    if (p.wide) {
#pragma unroll
                        for (int i = 0; i < D; i += 4) *(float4*)(y + i) = make_float4(o[i] * inverse, o[i + 1] * inverse, o[i + 2] * inverse, o[i + 3] * inverse);
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
                    auto part = [&](int64_t cta) { return p.partial + ((cta * 2 + (cta == first_cta)) * 2 + pipe) * PART; };
                    float* to = part(blockIdx.x);
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
                        for (int64_t c = first_cta; c <= last_cta; ++c) m = fmaxf(m, __ldcg(part(c) + 128 * D + row));
                        const float base = m == -INFINITY ? 0.0f : m;
                        sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < D; ++i) o[i] = 0.0f;
                        for (int64_t c = first_cta; c <= last_cta; ++c) {
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
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp < kSoftmaxWarps + kLoadWarps) {
            // ------------------------------------------------------------ loads: tiles of keys and values, in the order in which they are used
            constexpr int CHUNKS = D / 8, LINES = 32 / CHUNKS, PASS = LINES * kLoadWarps;  // 16-byte chunks a line; lines a warp and all of them copy at a time
            const int loader = warp - kSoftmaxWarps, chunk = lane % CHUNKS, line0 = loader * LINES + lane / CHUNKS;
            const uint32_t ring_at = smem_u32(ring) + (chunk >> 3) * (KT * 128);
            Ring at(STAGES);
            uint32_t n = 0, pending_n = 0;  // tiles so far; the one whose copies are under way
            bool dead = false, pending = false, pending_look = false;
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
            while (walk.next()) {
                const Block& k = walk.k;
                const int32_t* table = p.block_table + (int64_t)walk.r * p.table_stride;
                const int tiles = walk.take * (KEYS ? 2 : 1), first_key = walk.first_key(), line_mask = (1 << p.page_shift) - 1;
                // the keys that every row sees
                const int common_high = min(k.end, k.position0 + k.row0 / group + 1);
                const int common_low = p.window > 0 ? k.position0 + (k.row0 + k.rows - 1) / group - p.window + 1 : 0;
                int entry[KT / 32];  // lane l: the pages of keys l, l + 32, .. of the tile that is loaded next, -1 for none
                auto entries = [&](int key0) {
#pragma unroll
                    for (int i = 0; i < KT / 32; ++i) {
                        const int key = key0 + 32 * i + lane, e = key >= k.low && key < k.high ? __ldcg(table + (key >> p.page_shift)) : -1;
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
                    const char* base = (const char*)((values ? p.v : p.k) + walk.kv * p.head_stride + 8 * chunk);
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
        } else if (warp == kSoftmaxWarps + kLoadWarps) {
            // ------------------------------------------------------------ the issuing warp
            Ring at(STAGES);
            bool dead = false;
            uint32_t sums[2] = {0, 0}, items = 0;
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
                if (!arrived(&p_full[pipe], sums[pipe] & 1)) atomicExch(p.error_flag, 47);
                if (!arrived(&t_empty[pipe], (sums[pipe] & 1) ^ 1)) atomicExch(p.error_flag, 48);
                ++sums[pipe];
                fence_after();
                if (elect_one() && !dead) {
                    const uint64_t b = values_desc(ring_at + slot * F::TILE_BYTES, KT * 128);
                    const uint32_t to = tmem + F::T_COL + pipe * D, weights = tmem + pipe * KT, third = tmem + F::LO_COL + pipe * (KT / 2);
                    if (PARTS == 3)
#pragma unroll
                        for (int k = 0; k < KT / 16; ++k) mma_f16_ts(to, third + 8 * k, b + k * (16 * 128 >> 4), sums_desc, k > 0);
#pragma unroll
                    for (int part = 1; part >= 0; --part)
#pragma unroll
                        for (int k = 0; k < KT / 16; ++k)
                            mma_f16_ts(to, weights + 32 * (k >> 1) + 16 * part + 8 * (k & 1), b + k * (16 * 128 >> 4), sums_desc, PARTS == 3 || part == 0 || k > 0);
                    mma_commit(&t_full[pipe]);
                }
                __syncwarp();
            };
            auto release = [&](uint64_t* bar) {
                if (elect_one()) mma_commit(bar);
                __syncwarp();
            };
            while (walk.next()) {
                const int tiles = walk.take;
                if (!arrived(&q_full[0], items & 1)) atomicExch(p.error_flag, 46);
                int slot = take_slot();
                issue_scores(0, slot);
                if (KEYS) {
                    release(&empty[slot]);
                    slot = take_slot();
                } else {
                    if (!arrived(&q_full[1], items & 1)) atomicExch(p.error_flag, 46);
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
                ++items;
            }
            // nothing may be in flight when tensor memory is freed
            release(&ended);
            dead = false;
            if (!arrived(&ended, 0)) atomicExch(p.error_flag, 49);
        }
    }
    fence_before();
    __syncthreads();
    if (warp == kSoftmaxWarps + kLoadWarps) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <int D, int TYPE, bool KEYS>
int launch_form(rq_ctx* ctx, const AttentionParams& p, cudaStream_t s) {
    using F = Form<D, TYPE, KEYS>;
    auto kernel = rq_attention_tc_kernel<D, TYPE, KEYS>;
    static bool allowed = false;
    if (!allowed) {
        RQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM));
        allowed = true;
    }
    const int ctas = ctx->sm_count < kTensorCtas ? ctx->sm_count : kTensorCtas;
    return launch(kernel, dim3((unsigned)ctas), kThreads, F::SMEM, s, p);
}

}  // namespace

int rqattn::launch_tensor(rq_ctx* ctx, const AttentionParams& p, int head_dim, int type, bool one_tile, cudaStream_t s) {
    if (type == RQ_KV_BF16) return head_dim == 64 ? launch_form<64, RQ_KV_BF16, true>(ctx, p, s) : launch_form<128, RQ_KV_BF16, true>(ctx, p, s);
    if (head_dim == 64) return one_tile ? launch_form<64, RQ_KV_F16, true>(ctx, p, s) : launch_form<64, RQ_KV_F16, false>(ctx, p, s);
    return one_tile ? launch_form<128, RQ_KV_F16, true>(ctx, p, s) : launch_form<128, RQ_KV_F16, false>(ctx, p, s);
}
