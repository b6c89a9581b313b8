// The next token of a row of logits, from one given random number.
//
// Weights are whole numbers, w = floor(2^40 exp((x - max) / T)), so that their sums are exact: which tokens top_k, top_p and min_p keep and
// which one the random number meets depend on no order of additions (and of atomics). Tokens are ranked by a 64-bit key, the logit's bits made
// ascending above the complement of the index; the kept tokens are those whose key is at least a bound.
//
// A row is dealt out over a cluster of up to sixteen CTAs, each with its share in shared memory, read once from HBM (or, of many long rows, again from L2). A bound is
// found from a histogram, over 1024 parts of the logits' distance from the largest, of counts (top_k) or of weights (top_p, over no more than the distance that
// the bound can have): the CTAs' histograms are added up through distributed shared memory, every CTA finds the part in which the sum is reached, the tokens of
// that part, some hundreds, are sent to the first CTA, which finds the one by a histogram of its own and comparison of the few that share a place in it. Where a
// part holds more than fit (equal logits), it is taken apart by its 1024ths and then ten bits of the key at a time until they do. Where top_k leaves at most 512,
// these are sent to the first CTA, sorted, and everything else happens there. The draw is by sums in index order: of CTAs, of warps, of threads.
//
// For one row it is bound by the chain of some ten cluster barriers with a pass over the share between them: 1 x 262144 with top_k = 64 and top_p = 0.95 20 us,
// with top_p alone 30, greedy 6. For many rows by instructions, some hundred a logit in four passes (an exponential in two of them, an addition in shared memory
// of two or three words): 64 x 262144 with top_p = 0.9 112 us, with min_p = 0.02 too 94, top_k = 64 52, no filter 47, greedy 22. With one CTA a row and seven
// rounds over ten bits of the key each it was 2054 us for one row and 1863 for 64; with parts over all 28 T, lists of 512 and weights made whole numbers by
// conversion 118 for the 64, at T = 1.2 191 (now 116).
#include <cooperative_groups.h>

#include <type_traits>

#include "rq_serve.cuh"

using namespace rqserve;
namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 1024, kList = 2 * kThreads, kMostCtas = 16;
constexpr int kShare = 16384;  // logits of a CTA in shared memory
constexpr float kFade = 28.0f; // exp(-28) < 2^-40

struct SampleParams {
    const float *logits, *temperature, *top_p, *min_p, *uniform;
    const int32_t* top_k;
    int32_t *token, *kept;
    float* probability;
    int64_t stride;
    int vocabulary, share;  // logits a CTA: a whole number of warps' shares
};

typedef unsigned long long u64;

// NaN as -inf, -0 as +0
__device__ __forceinline__ float cleaned(float x) { return x != x ? -INFINITY : x + 0.0f; }
__device__ __forceinline__ uint32_t ascending(float x) { const uint32_t u = __float_as_uint(x); return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u); }
__device__ __forceinline__ float value_of(u64 key) { const uint32_t b = (uint32_t)(key >> 32); return __uint_as_float(b >> 31 ? b ^ 0x80000000u : ~b); }
__device__ __forceinline__ u64 rank_key(float x, int index) { return (u64)ascending(x) << 32 | (uint32_t)~index; }
// the weight over 2^40; equal to the largest logit: one, also where that is +inf
__device__ __forceinline__ float weight(float x, float top, float temperature) {
    if (x == top) return 1.0f;
    return temperature > 0.0f ? expf((x - top) / temperature) : 0.0f;
}
__device__ __forceinline__ u64 mass_of(float e) { return (u64)(e * 1099511627776.0f); }
// floor(x), 0 <= x < 2^22, as the low bits of x + 2^23 rounded down; x = a * b. What is left of the product is exact.
__device__ __forceinline__ uint32_t take_whole(float a, float b, float& left) {
    const float t = __fmaf_rd(a, b, 8388608.0f);
    left = fmaf(a, b, 8388608.0f - t);
    return __float_as_uint(t) - 0x4b000000u;
}

struct Shared {
    // this CTA's sums, in words of 16, 13 and 12 bits of their terms: a 64-bit atomic addition in shared memory is a loop, and one that carries waits for an answer
    uint32_t low[kBins], mid[kBins], high[kBins];
    u64 list[kList], list_mass[kList];
    u64 merged[kBins], list_sum[kList];
    u64 warp_sum[kWarps], warp_count[kWarps];
    u64 sum, count;          // this CTA's kept weights and tokens
    u64 bound, before;       // the first CTA's answer; what lies before the part that was found
    int part, sharing, best;
    uint32_t listed[16];     // the first CTA's lists, one after another
    float warp_top[kWarps], top;
};

// Sum over the CTA; every thread gets it
__device__ __forceinline__ u64 block_sum(u64 v, u64* warp_sums) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    __syncthreads();
    if (lane == 0) warp_sums[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < kWarps ? warp_sums[lane] : 0;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// Sorts the first CTA's list by falling keys, the masses with them, and adds the masses up: list_sum[i] = those of keys above and at i. A bitonic network, a
// thread an entry: steps within a warp by shuffles, between warps through shared memory. (Ranks by comparison with all others took 9 us for 330.)
__device__ void sort_list(Shared& sh, int n) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int size = 32;
    while (size < n) size <<= 1;
    __syncthreads();
    u64 key = tid < n ? sh.list[tid] : 0, mass = tid < n ? sh.list_mass[tid] : 0;
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            u64 other, other_mass;
            if (j >= 32) {
                __syncthreads();
                sh.list[tid] = key;
                sh.list_mass[tid] = mass;
                __syncthreads();
                other = sh.list[tid ^ j];
                other_mass = sh.list_mass[tid ^ j];
            } else {
                other = __shfl_xor_sync(0xffffffffu, key, j);
                other_mass = __shfl_xor_sync(0xffffffffu, mass, j);
            }
            const bool larger_here = ((tid & k) == 0) == ((tid & j) == 0);
            if (key != other && (other > key) == larger_here) { key = other; mass = other_mass; }
        }
    u64 scan = mass;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) { const u64 o = __shfl_up_sync(0xffffffffu, scan, off); if (lane >= off) scan += o; }
    __syncthreads();
    if (lane == 31) sh.warp_sum[warp] = scan;
    __syncthreads();
    for (int w = 0; w < warp; ++w) scan += sh.warp_sum[w];
    sh.list[tid] = key;
    sh.list_mass[tid] = mass;
    sh.list_sum[tid] = scan;
    __syncthreads();
}

// Up to a thread's worth of candidates, every token of weight down to the last that top_k could keep among them: a thread has one and compares it with all
__device__ void draw_from_list(const SampleParams& p, Shared& sh, int row, float top, float temperature, int top_k, float top_p, float min_p) {
    const int tid = threadIdx.x, n = (int)sh.listed[0];
    if (tid < n) sh.list_mass[tid] = mass_of(weight(value_of(sh.list[tid]), top, temperature));
    sort_list(sh, n);
    const u64 key = tid < n ? sh.list[tid] : 0, mass = tid < n ? sh.list_mass[tid] : 0, before = tid < n ? sh.list_sum[tid] - mass : 0;
    const float x = value_of(key);
    const double target = (double)top_p * (double)sh.list_sum[min(top_k, n) - 1];
    const bool kept = tid < n && tid < top_k && (top_p >= 1.0f || (double)before < target || tid == 0) && (x == top || weight(x, top, temperature) >= min_p);
    const u64 mine = kept ? mass : 0;
    const u64 total = block_sum(mine, sh.warp_sum), tokens = block_sum(mine != 0, sh.warp_count);
    // in the order of their indices: those are the complement of the keys' low halves
    __syncthreads();
    if (tid < n) { sh.list[tid] = (uint32_t)key; sh.list_mass[tid] = mine; }
    sort_list(sh, n);
    u64 want = (u64)(fmin(fmax((double)p.uniform[row], 0.0), 1.0) * (double)total);
    if (want >= total) want = total - 1;
    if (tid < n) {
        const u64 w = sh.list_mass[tid], upto = sh.list_sum[tid];
        if (upto > want && upto - w <= want) {
            p.token[row] = (int32_t)~(uint32_t)sh.list[tid];
            if (p.probability) p.probability[row] = (float)((double)w / (double)total);
            if (p.kept) p.kept[row] = (int32_t)tokens;
        }
    }
}

// The weight's division by the temperature, one for a row, as a product with its reciprocal and a correction by the remainder (Markstein, 1990): rounded as
// the quotient is, unless the divisor's fraction is all ones; far from where a step of it could overflow or lose bits.
struct Weigher {
    float top, temperature, reciprocal;
    bool quick;
    __device__ Weigher(float top_, float temperature_) : top(top_), temperature(temperature_), reciprocal(1.0f / temperature_) {
        quick = top < INFINITY && temperature > 1e-15f && temperature < 1e15f && (__float_as_uint(temperature) & 0x7fffffu) != 0x7fffffu;
    }
    template <bool QUICK> __device__ __forceinline__ float share(float x) const {  // (of the largest logit itself: exp(0) = 1)
        if (!QUICK) return weight(x, top, temperature);
        const float n = x - top, q = n * reciprocal;
        return expf(fmaf(fmaf(-q, temperature, n), reciprocal, q));
    }
    __device__ u64 operator()(float x) const { return mass_of(quick ? share<true>(x) : share<false>(x)); }
};
__device__ __forceinline__ u64 sum_of(const Shared& sh, int bin) { return ((u64)sh.high[bin] << 29) + ((u64)sh.mid[bin] << 16) + sh.low[bin]; }
__device__ __forceinline__ void clear(Shared& sh) { *(uint2*)&sh.low[2 * threadIdx.x] = *(uint2*)&sh.mid[2 * threadIdx.x] = *(uint2*)&sh.high[2 * threadIdx.x] = make_uint2(0, 0); }
__device__ __forceinline__ void add_words(Shared& sh, int bin, uint32_t hi, uint32_t mid, uint32_t lo) {
    if (lo) atomicAdd(&sh.low[bin], lo);  // (at most 2^16 terms a CTA)
    if (mid) atomicAdd(&sh.mid[bin], mid);
    if (hi) atomicAdd(&sh.high[bin], hi);
}
// the same without a branch a word (three words of a part lie a plane apart), where `here`
__device__ __forceinline__ void add_words_if(bool here, uint32_t part_low, uint32_t hi, uint32_t mid, uint32_t lo) {
    asm volatile(
        "{\n.reg .pred h, p, q, r;\nsetp.ne.u32 h, %4, 0;\nsetp.ne.and.u32 p, %1, 0, h;\nsetp.ne.and.u32 q, %2, 0, h;\nsetp.ne.and.u32 r, %3, 0, h;\n"
        "@p red.shared.add.u32 [%0], %1;\n@q red.shared.add.u32 [%0 + %5], %2;\n@r red.shared.add.u32 [%0 + %6], %3;\n}" ::"r"(part_low), "r"(lo), "r"(mid), "r"(hi),
        "r"((uint32_t)here), "n"(4 * kBins), "n"(8 * kBins)
        : "memory");
}
__device__ __forceinline__ void add_to(Shared& sh, int bin, u64 v) { add_words(sh, bin, (uint32_t)(v >> 29), (uint32_t)(v >> 16) & 0x1fff, (uint32_t)v & 0xffff); }

// STAGED: the share lies in shared memory, cleaned; otherwise it is read again
template <bool STAGED>
__global__ void __launch_bounds__(kThreads, 2) rq_sample_kernel(SampleParams p) {
    extern __shared__ __align__(16) float staged[];
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = rank * p.share, count = max(min(p.vocabulary - first, p.share), 0);
    // a warp has neighbouring logits, so that sums in index order are sums of warps
    const int warp_share = p.share / kWarps, begin = warp * warp_share, stop = begin + warp_share, end = min(stop, count);  // (a multiple of 128)
    launch_dependents();
    for (int b = tid; b < kBins; b += kThreads) sh.low[b] = sh.mid[b] = sh.high[b] = 0;
    if (tid < 16) sh.listed[tid] = 0;
    if (tid == 0) sh.best = p.vocabulary;
    Shared* const leader = cluster.map_shared_rank(&sh, 0);
    wait_for_previous();
    const float* x = p.logits + row * p.stride + first;
    const float temperature = p.temperature ? p.temperature[row] : 1.0f, given_p = p.top_p ? p.top_p[row] : 1.0f, given_min = p.min_p ? p.min_p[row] : 0.0f;
    // into their ranges, NaN to the end that keeps all (the parts of a histogram are made for these: logf(V / (1 - top_p)) is not below 0)
    const float top_p = given_p < 1.0f ? fmaxf(given_p, 0.0f) : 1.0f, min_p = given_min > 0.0f ? fminf(given_min, 1.0f) : 0.0f;
    const int top_k = (p.top_k && p.top_k[row] > 0 ? p.top_k[row] : p.vocabulary);
    auto at = [&](int i) { return STAGED ? staged[i] : cleaned(__ldcg(x + i)); };

    // ---- the largest logit ----------------------------------------------------------------------------
    float top = -INFINITY;
    const bool wide = ((uintptr_t)x & 15) == 0;
    // four neighbours of the row; -inf past the end
    auto read = [&](int i, float (&v)[4]) {
        if (wide && i + 4 <= end) {
            const float4 a = __ldcg((const float4*)(x + i));
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = i + k < end ? __ldcg(x + i + k) : -INFINITY;
        }
    };
    constexpr int kAtOnce = 4;
    for (int i = begin + 4 * lane; i < stop; i += 128 * kAtOnce) {
        float v[kAtOnce][4];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) read(i + 128 * n, v[n]);
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[n][k] = cleaned(v[n][k]);
                top = fmaxf(top, v[n][k]);
            }
            if (STAGED && i + 128 * n < stop) *(float4*)(staged + i + 128 * n) = make_float4(v[n][0], v[n][1], v[n][2], v[n][3]);
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if (lane == 0) sh.warp_top[warp] = top;
    __syncthreads();
    top = sh.warp_top[lane % kWarps];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if (tid == 0) sh.top = top;
    cluster.sync();
    top = lane < ctas ? cluster.map_shared_rank(&sh, lane)->top : -INFINITY;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));

    // Four neighbouring logits of a thread at a time, -inf past the end. CLEAN: NaN as -inf and -0 as +0, which keys are made of; comparisons and
    // weights need neither.
    auto each_four = [&](auto clean, auto&& use) {
        float next[4];
        if (!STAGED) read(begin + 4 * lane, next);
#pragma unroll 1
        for (int i = begin + 4 * lane; i < stop; i += 128) {
            float v[4];
            if (STAGED) {
                const float4 a = *(const float4*)(staged + i);
                v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = decltype(clean)::value ? cleaned(next[k]) : next[k];
                read(i + 128, next);  // (on their way while these are looked at)
            }
            use(v, i);
        }
    };
    const std::true_type for_keys;
    const std::false_type for_sums;

    // ---- bounds ------------------------------------------------------------------------------------
    const Weigher weigh(top, temperature);
    const float limit = fminf(kFade * temperature, 3e38f);
    float scale = (float)kBins / limit;
    // 0 <= place (and NaN, which comes out as the last part): distances from the largest logit times a scale that is positive, since all of what it is made of is
    auto floor_of = [](float place) { return (int)(__float_as_uint(__fadd_rd(fminf(place, (float)(kBins - 1)), 8388608.0f)) & 0x7fffffu); };
    auto part_of = [&](float v) { return v == top ? 0 : floor_of((top - v) * scale); };
    auto sub_of = [&](float v) { const float place = (top - v) * scale; return v == top ? 0 : floor_of((place - (float)floor_of(place)) * (float)kBins); };
    // What lies so far below weighs nothing: by one comparison (the rounding of this value takes no logit's weight, for they are rounded alike)
    const float fade = top < INFINITY ? fmaxf(top - limit, -3.4e38f) : top;
    auto fades = [&](float v) { return v < fade; };
    // A pass's loop for either way to divide (a branch around each would keep the steps of four logits from overlapping)
    auto quickly = [&](auto&& pass) {
        if (weigh.quick) pass(std::true_type());
        else pass(std::false_type());
    };
    // Tokens whose key is at least a bound: (value, index), without putting the key together
    struct Floor { float value; int index; };
    auto floor_at = [&](u64 key, float least) -> Floor {
        const float v = key ? value_of(key) : -INFINITY;
        return v >= least ? Floor{v, (int)(~(uint32_t)key) - first} : Floor{least, 0x7fffffff};
    };
    auto above = [](const Floor& f, float v, int i) { return v > f.value || (v == f.value && i <= f.index); };
    int lists = 0;
    bool few = false;

    // Adds up the CTAs' histograms and finds the last key's part: where the sum from the largest keys down (bins in the order given by `down`) reaches what is wanted.
    // `before`: the sum above the interval. False: it is not reached.
    auto reached_by = [](bool by_mass, u64 want, double target) { return [=](u64 s) { return by_mass ? (double)s >= target : s >= want; }; };
    // Which of the parts, two a thread in falling order of their keys, is the one in which the sum is reached, and the sum before it
    auto reach_in = [&](u64 m0, u64 m1, int b0, int b1, auto&& reached, u64& before, int& part) -> bool {
        u64 scan = m0 + m1;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) { const u64 o = __shfl_up_sync(0xffffffffu, scan, off); if (lane >= off) scan += o; }
        if (lane == 31) sh.warp_sum[warp] = scan;
        if (tid == 0) sh.part = -1;
        __syncthreads();
        u64 others = lane < warp ? sh.warp_sum[lane % kWarps] : 0;
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) others += __shfl_xor_sync(0xffffffffu, others, off);
        scan += before + __shfl_sync(0xffffffffu, others, 0);
        const u64 low = scan - m0 - m1, mid = low + m0;
        if (m0 && reached(mid) && !reached(low)) { sh.part = b0; sh.before = low; }
        if (m1 && reached(scan) && !reached(mid)) { sh.part = b1; sh.before = mid; }
        __syncthreads();
        part = sh.part;
        if (part >= 0) before = sh.before;
        __syncthreads();
        return part >= 0;
    };
    auto find = [&](bool by_mass, u64 want, double& share_of_mass, bool first_round, bool down, u64& before, int& part) -> bool {
        cluster.sync();  // all histograms are complete
        // this CTA's parts, a lane per source: two rounds whatever the cluster's size
        const int source = tid & (ctas - 1);
        const Shared* const from = cluster.map_shared_rank(&sh, source);
        Shared* const to = cluster.map_shared_rank(&sh, source);
        u64 sum[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) sum[i] = sum_of(*from, (rank * kBins + i * kThreads + tid) / ctas);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            for (int off = ctas >> 1; off > 0; off >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], off);
            to->merged[(rank * kBins + i * kThreads + tid) / ctas] = sum[i];
        }
        cluster.sync();
        // two neighbouring parts a thread, from the largest keys down
        const int a = 2 * tid, b0 = down ? kBins - 1 - a : a, b1 = down ? b0 - 1 : a + 1;
        clear(sh);
        if (by_mass && first_round) {
            share_of_mass *= (double)block_sum(sh.merged[b0] + sh.merged[b1], sh.warp_count);
            if (!(share_of_mass > 0.0)) share_of_mass = 0.5;  // at least one token: any weight reaches a half
        }
        return reach_in(sh.merged[b0], sh.merged[b1], b0, b1, reached_by(by_mass, want, share_of_mass), before, part);
    };
    // The last key, in falling order, up to which the counts reach `want` or the weights the share top_p of all, among keys of at least `floor`
    auto reach = [&](bool by_mass, u64 want, u64 floor) -> u64 {
        const Floor from = floor_at(floor, fade);
        if (!by_mass) {
            each_four(for_sums, [&](const float (&v)[4], int i) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (above(from, v[k], i + k)) atomicAdd(&sh.low[part_of(v[k])], 1u);
            });
        } else {
            // Logits further off than T ln(V / (1 - top_p)) weigh less than 1 - top_p together, for the largest alone weighs 1: the parts are
            // finer by as much, and what lies in the last one is added up in registers. (One part more or less does no harm: what is found is looked up.)
            scale = (float)kBins / fminf(fminf(logf((float)p.vocabulary / (1.0f - top_p)) + 1.0f, kFade) * temperature, 3e38f);
            uint32_t far_hi = 0, far_mid = 0, far_low = 0;
            const uint32_t parts_at = (uint32_t)__cvta_generic_to_shared(sh.low);
            static_assert(offsetof(Shared, mid) == offsetof(Shared, low) + 4 * kBins && offsetof(Shared, high) == offsetof(Shared, mid) + 4 * kBins, "planes");
            auto add_up = [&](auto quick, auto ties) {
                each_four(for_sums, [&](const float (&v)[4], int i) {
                    uint32_t hi[4], mid[4], low[4];
                    int bin[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool on = decltype(ties)::value ? above(from, v[k], i + k) : v[k] >= from.value;
                        float left = on ? weigh.share<decltype(quick)::value>(v[k]) : 0.0f;
                        hi[k] = take_whole(left, 2048.0f, left);
                        mid[k] = take_whole(left, 8192.0f, left);
                        low[k] = take_whole(left, 65536.0f, left);
                        bin[k] = decltype(quick)::value ? floor_of((v[k] - top) * -scale) : part_of(v[k]);  // (the same: 0 for the largest, which is finite)
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool far = bin[k] == kBins - 1;
                        far_hi += far ? hi[k] : 0;
                        far_mid += far ? mid[k] : 0;
                        far_low += far ? low[k] : 0;
                        add_words_if(!far, parts_at + 4 * bin[k], hi[k], mid[k], low[k]);
                    }
                });
            };
            if (!weigh.quick) add_up(std::false_type(), std::true_type());
            else if (from.index == 0x7fffffff) add_up(std::true_type(), std::false_type());  // no token of that value is left out
            else add_up(std::true_type(), std::true_type());
            far_hi = __reduce_add_sync(0xffffffffu, far_hi); far_mid = __reduce_add_sync(0xffffffffu, far_mid); far_low = __reduce_add_sync(0xffffffffu, far_low);
            if (lane == 0) add_words(sh, kBins - 1, far_hi, far_mid, far_low);
        }
        u64 before = 0;
        int part;
        double target = top_p;
        if (!find(by_mass, want, target, true, false, before, part)) return floor;
        if (!by_mass && before + sh.merged[part] <= kThreads) {  // so few that they are drawn from where they are listed
            few = true;
            const float high_place = part < kBins - 1 ? (float)(part + 1) : INFINITY;
            each_four(for_keys, [&](const float (&v)[4], int i) {
                bool any = false;
#pragma unroll
                for (int k = 0; k < 4; ++k) any = any || (v[k] >= fade && !((top - v[k]) * scale >= high_place));
                if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (!fades(v[k]) && part_of(v[k]) <= part) leader->list[atomicAdd(&leader->listed[0], 1u)] = rank_key(v[k], first + i + k);
            });
            cluster.sync();
            return 0;
        }
        // the tokens of that part, or of an interval of keys in it, to the first CTA
        u64 base = 0;
        int shift = 64, sub_part = -1;
        while (true) {
            const int list = lists++ & 15;
            auto inside = [&](float v, u64 key) {
                return part_of(v) == part && key >= floor && (sub_part < 0 || sub_of(v) == sub_part) && key >= base && (shift == 64 || !((key - base) >> shift));
            };
            // the part's values and a little more; those between are asked for their part
            const float most = part > 0 ? top - ((float)part - 0.5f) / scale : top, least = part < kBins - 1 ? fmaxf(fade, top - ((float)part + 1.5f) / scale) : fade;
            each_four(for_sums, [&](const float (&raw)[4], int i) {
                bool on[4], any = false;
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    on[k] = raw[k] >= least && raw[k] <= most;
                    any = any || on[k];
                    v[k] = raw[k] + 0.0f;
                }
                if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (!on[k]) continue;
                    const u64 key = rank_key(v[k], first + i + k);
                    if (!inside(v[k], key)) continue;
                    const u64 mass = by_mass ? weigh(v[k]) : 1;
                    if (!mass) continue;
                    const uint32_t entry = atomicAdd(&leader->listed[list], 1u);
                    if (entry < kList) { leader->list[entry] = key; leader->list_mass[entry] = mass; }
                }
            });
            cluster.sync();
            const uint32_t n = leader->listed[list];
            if (n <= kList) {
                if (rank == 0) {
                    // the list by a 1024th of the part (or ten bits of the key), then the few that share one by comparison with each other
                    const int next = max(shift - 10, 0);
                    auto bin_of = [&](u64 key) { return sub_part < 0 ? kBins - 1 - sub_of(value_of(key)) : (int)((key - base) >> next); };  // rising with the key
                    for (int e = tid; e < (int)n; e += kThreads) add_to(sh, bin_of(sh.list[e]), sh.list_mass[e]);
                    __syncthreads();
                    int sub;
                    u64 above_all = before;
                    if (tid == 0) sh.sharing = 0;
                    const u64 a = sum_of(sh, kBins - 1 - 2 * tid), b = sum_of(sh, kBins - 2 - 2 * tid);
                    reach_in(a, b, kBins - 1 - 2 * tid, kBins - 2 - 2 * tid, reached_by(by_mass, want, target), above_all, sub);
                    for (int e = tid; e < (int)n; e += kThreads) {
                        if (bin_of(sh.list[e]) != sub) continue;
                        const int place = atomicAdd(&sh.sharing, 1);
                        sh.merged[place] = sh.list[e];
                        sh.list_sum[place] = sh.list_mass[e];
                    }
                    __syncthreads();
                    const int sharing = sh.sharing;
                    for (int e = tid; e < sharing; e += kThreads) {
                        const u64 key = sh.merged[e], mass = sh.list_sum[e];
                        u64 above_it = above_all;
                        for (int j = 0; j < sharing; ++j) above_it += sh.merged[j] > key ? sh.list_sum[j] : 0;
                        const auto reached = reached_by(by_mass, want, target);
                        if (reached(above_it + mass) && !reached(above_it)) sh.bound = key;
                    }
                    __syncthreads();
                    clear(sh);
                }
                cluster.sync();
                if (tid == 0 && rank == 0) sh.listed[(list + 8) & 15] = 0;  // (eight lists on: nobody looks at that one any more)
                return leader->bound;
            }
            // more than fit: a 1024th of the part, then ten bits of the key after ten
            const bool by_key = sub_part >= 0;
            const int next = max(shift - 10, 0);
            for (int i = begin + lane; i < end; i += 32) {
                const float v = at(i);
                if (fades(v)) continue;
                const u64 key = rank_key(v, first + i);
                if (!inside(v, key)) continue;
                const u64 mass = by_mass ? weigh(v) : 1;
                if (mass) add_to(sh, by_key ? (int)((key - base) >> next) : sub_of(v), mass);
            }
            int sub = 0;
            find(by_mass, want, target, false, by_key, before, sub);
            if (tid == 0 && rank == 0) sh.listed[(list + 8) & 15] = 0;
            if (!by_key) { sub_part = max(sub, 0); continue; }
            base += (u64)max(sub, 0) << next;
            shift = next;
        }
    };
    const bool nothing = top == -INFINITY;
    u64 bound = 0;
    if (!(temperature > 0.0f) && !nothing) {  // the largest logit, the first of equal ones
        int least = p.vocabulary;
        each_four(for_sums, [&](const float (&v)[4], int i) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (v[k] == top) least = min(least, first + i + k);
        });
        least = __reduce_min_sync(0xffffffffu, least);
        if (lane == 0) sh.warp_count[warp] = (u64)least;
        __syncthreads();
        if (warp == 0) {
            least = __reduce_min_sync(0xffffffffu, lane < kWarps ? (int)sh.warp_count[lane] : p.vocabulary);
            if (lane == 0) atomicMin(&leader->best, least);
        }
        cluster.sync();
        if (rank == 0 && tid == 0) {
            p.token[row] = sh.best;
            if (p.probability) p.probability[row] = 1.0f;
            if (p.kept) p.kept[row] = 1;
        }
        return;
    }
    if (!nothing && top_k < p.vocabulary) bound = reach(false, (u64)top_k, 0);
    if (few) {
        if (rank == 0) draw_from_list(p, sh, row, top, temperature, top_k, top_p, min_p);
        return;  // (nobody reads another CTA's memory any more)
    }
    if (!nothing && top_p < 1.0f) bound = reach(true, 0, bound);

    // ---- the draw -----------------------------------------------------------------------------------
    // (min_p as a value too, a little low: what lies below it is not looked at, what lies above is asked itself)
    const bool by_min = min_p > 0.0f;
    const float least = by_min && min_p < 1.0f && weigh.quick ? fmaxf(fade, top + temperature * (logf(min_p) * 1.001f - 0.001f)) : fade;
    const Floor from = floor_at(bound, least);
    const float enough = by_min ? fmaxf(min_p, 0x1p-40f) : 0x1p-40f;  // (of less than 2^-40 nothing is left as a whole number)
    auto weight_of = [&](auto quick, float v, bool on) {
        const float e = weigh.share<decltype(quick)::value>(v);
        return on && (e >= enough || v == top) ? e : 0.0f;
    };
    u64 sum = 0;
    uint32_t tokens = 0;
    if (!nothing) {
        uint32_t high = 0, low = 0;  // words of 20 bits of the weights of at most 2^7 logits
        quickly([&](auto quick) { each_four(for_sums, [&](const float (&v)[4], int i) {
            bool on[4], any = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) { on[k] = above(from, v[k], i + k); any = any || on[k]; }
            if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float e = weight_of(quick, v[k], on[k]);
                tokens += e > 0.0f;
                high += take_whole(e, 1048576.0f, e);
                low += take_whole(e, 1048576.0f, e);
            }
        }); });
        sum = ((u64)high << 20) + low;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) { sum += __shfl_xor_sync(0xffffffffu, sum, off); tokens += __shfl_xor_sync(0xffffffffu, tokens, off); }
    if (lane == 0) { sh.warp_sum[warp] = sum; sh.warp_count[warp] = tokens; }
    __syncthreads();
    if (tid == 0) {
        u64 s = 0, n = 0;
        for (int w = 0; w < kWarps; ++w) { s += sh.warp_sum[w]; n += sh.warp_count[w]; }
        sh.sum = s;
        sh.count = n;
    }
    cluster.sync();
    u64 total = 0, ahead = 0, all = 0;
    {
        const Shared* other = cluster.map_shared_rank(&sh, lane & (ctas - 1));
        const u64 s = lane < ctas ? other->sum : 0, n = lane < ctas ? other->count : 0;
        total = s;
        all = n;
        ahead = lane < rank ? s : 0;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            total += __shfl_xor_sync(0xffffffffu, total, off);
            all += __shfl_xor_sync(0xffffffffu, all, off);
            ahead += __shfl_xor_sync(0xffffffffu, ahead, off);
        }
    }
    if (nothing) {
        if (rank == 0 && tid == 0) { p.token[row] = -1; if (p.probability) p.probability[row] = 0.0f; if (p.kept) p.kept[row] = 0; }
    } else {
        const double u = fmin(fmax((double)p.uniform[row], 0.0), 1.0);
        u64 want = (u64)(u * (double)total);
        if (want >= total) want = total - 1;
        if (ahead <= want && want < ahead + sh.sum) {
            // this CTA's: the warp's share that it is in, neighbours a thread, and the one thread's neighbours one by one
            int in = 0;
            for (; in < kWarps - 1 && ahead + sh.warp_sum[in] <= want; ++in) ahead += sh.warp_sum[in];
            const int each = (warp_share + kThreads - 1) / kThreads, from_here = in * warp_share + tid * each, upto = min(min(from_here + each, (in + 1) * warp_share), count);
            u64 w = 0;
            quickly([&](auto quick) {
                for (int i = from_here; i < upto; i += 4) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float v = i + k < upto ? at(i + k) : -INFINITY;
                        w += mass_of(weight_of(quick, v, above(from, v, i + k)));
                    }
                }
            });
            u64 scan = w;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) { const u64 o = __shfl_up_sync(0xffffffffu, scan, off); if (lane >= off) scan += o; }
            if (lane == 31) sh.list_sum[warp] = scan;
            __syncthreads();
            for (int k = 0; k < warp; ++k) ahead += sh.list_sum[k];
            if (ahead + scan > want && ahead + scan - w <= want) {
                u64 run = ahead + scan - w;
                for (int i = from_here; i < upto; ++i) {
                    const float v = at(i);
                    const u64 m = mass_of(weigh.quick ? weight_of(std::true_type(), v, above(from, v, i)) : weight_of(std::false_type(), v, above(from, v, i)));
                    run += m;
                    if (run > want) {
                        p.token[row] = first + i;
                        if (p.probability) p.probability[row] = (float)((double)m / (double)total);
                        if (p.kept) p.kept[row] = (int32_t)all;
                        break;
                    }
                }
            }
        }
    }
    cluster.sync();  // nobody leaves while its shared memory may be read
}

template <bool STAGED>
int launch_sample(rq_ctx* ctx, const SampleParams& p, int rows, int ctas, cudaStream_t s) {
    auto kernel = rq_sample_kernel<STAGED>;
    static bool configured[64] = {};  // by device: the opt-ins to clusters of sixteen and to large shared memory
    if (ctx->device >= 64 || !configured[ctx->device]) {
        RQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        if (STAGED) RQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kShare * (int)sizeof(float)));
        if (ctx->device < 64) configured[ctx->device] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = STAGED ? (size_t)p.share * sizeof(float) : 0;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    RQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return RQ_OK;
}

}  // namespace

extern "C" int rq_sample(rq_ctx* ctx, const float* logits, int64_t row_stride, int rows, int64_t vocabulary, const float* temperature, const int32_t* top_k, const float* top_p,
                         const float* min_p, const float* uniform, int32_t* token, float* probability, int32_t* kept, void* stream) {
    if (!ctx || !logits || !uniform || !token) return rq_fail(RQ_ERR_INVALID, "rq_sample: null argument");
    if (rows <= 0 || vocabulary <= 0 || (rows > 1 && row_stride < vocabulary)) return rq_fail(RQ_ERR_INVALID, "rq_sample: rows and vocabulary must be positive and row_stride at least vocabulary");
    if (vocabulary > RQ_MAX_VOCABULARY) return rq_fail(RQ_ERR_LIMIT, "rq_sample: %lld tokens; at most %d", (long long)vocabulary, RQ_MAX_VOCABULARY);
    if (rows > (1 << 26)) return rq_fail(RQ_ERR_LIMIT, "rq_sample: %d rows; at most 2^26", rows);
    DeviceGuard guard(ctx->device);
    // CTAs a row: as many as hold it in shared memory, and more while the GPU holds them all at once (two an SM; of clusters of sixteen fourteen) and a share is some
    // thousand logits. Where they do not all fit, as few as let all rows run at once, and logits are read again from L2.
    // T = 0.9, top_p = 0.95: 64 x 32000 by two CTAs a row 34 us, by four 25; 24 x 64000 by four 36, by eight 28. Shares of two thousand: 4 x 32000 by sixteen 24, by
    // eight 16.
    int ctas = 1;
    while (ctas < kMostCtas && (vocabulary > (int64_t)ctas * kShare || ((int64_t)rows * ctas * 2 <= (ctas == 8 ? 14 * 16 : 2 * ctx->sm_count) && vocabulary > (int64_t)ctas * 4096))) ctas *= 2;
    if ((int64_t)rows * ctas > 14 * 16)
        while (ctas > 1 && (int64_t)rows * ctas > 2 * ctx->sm_count && (vocabulary + ctas / 2 - 1) / (ctas / 2) <= 65536) ctas /= 2;
    const int64_t unit = 4 * kThreads;  // a warp's share is a whole number of 128
    SampleParams p = {logits, temperature, top_p, min_p, uniform, top_k, token, kept, probability, row_stride, (int)vocabulary, 0};
    p.share = (int)(((vocabulary + ctas - 1) / ctas + unit - 1) / unit * unit);
    if (p.share <= kShare) return launch_sample<true>(ctx, p, rows, ctas, (cudaStream_t)stream);
    return launch_sample<false>(ctx, p, rows, ctas, (cudaStream_t)stream);
}
