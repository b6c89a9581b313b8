// The next token of a row of logits, from one given random number.
//
// Weights are whole numbers, w = floor(2^40 exp((x - max) / T)), so that their sums are exact: which tokens top_k, top_p and min_p keep and
// which one the random number meets depend on no order of additions (and of atomics). Tokens are ranked by a 64-bit key, the logit's bits made
// ascending above the complement of the index; the kept tokens are those whose key is at least a bound.
//
// A row is dealt out over a cluster of up to sixteen CTAs, each with its share in shared memory, read once from HBM. A bound is found from a histogram, over 1024 parts of the
// logits' distance from the largest (the weights fade within 28 T of it), of counts (top_k) or of weights (top_p): the CTAs'
// histograms are added up through distributed shared memory, every CTA finds the part in which the sum is reached, the tokens of that part, some
// hundreds, are sent to the first CTA, and there each finds its rank and the weights before it by comparison with all others. Where
// a part holds more than fit (equal logits), it is taken apart by ten bits of the key at a time until they do.
//
// For one row it is bound by the chain of some ten cluster barriers with a pass over the share between them; for many rows by instructions: an
// exponential, a division and an atomic addition in shared memory a token. One thread block a row, with seven rounds over ten bits of the key
// each: 2054 us for 1 x 262144 and 1863 us for 64 x 262144.
#include <cooperative_groups.h>

#include "rq_serve.cuh"

using namespace rqserve;
namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 1024, kList = 1024, kMostCtas = 16;
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
__device__ __forceinline__ u64 rank_key(float x, int index) { return (u64)ascending(x) << 32 | (uint32_t)~index; }
// the weight over 2^40; equal to the largest logit: one, also where that is +inf
__device__ __forceinline__ float weight(float x, float top, float temperature) {
    if (x == top) return 1.0f;
    return temperature > 0.0f ? expf((x - top) / temperature) : 0.0f;
}
__device__ __forceinline__ u64 mass_of(float e) { return (u64)(e * 1099511627776.0f); }

struct Shared {
    u64 hist[kBins], merged[kBins];
    u64 list[kList], list_mass[kList];
    u64 warp_sum[kWarps], warp_count[kWarps];
    u64 sum, count;          // this CTA's kept weights and tokens
    u64 bound, before;       // the first CTA's answer; what lies before the part that was found
    u64 total;
    int part;
    uint32_t listed[16];     // the first CTA's lists, one after another
    float warp_top[kWarps], top;
    int chosen_warp;
    u64 chosen_want;
};

// STAGED: the share lies in shared memory, cleaned; otherwise it is read again
template <bool STAGED>
__global__ void __launch_bounds__(kThreads) rq_sample_kernel(SampleParams p) {
    extern __shared__ __align__(16) float staged[];
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = rank * p.share, count = max(min(p.vocabulary - first, p.share), 0);
    // a warp has neighbouring logits, so that sums in index order are sums of warps
    const int warp_share = p.share / kWarps, begin = warp * warp_share, end = min(begin + warp_share, count);
    launch_dependents();
    for (int b = tid; b < kBins; b += kThreads) sh.hist[b] = 0;
    if (tid < 16) sh.listed[tid] = 0;
    Shared* const leader = cluster.map_shared_rank(&sh, 0);
    wait_for_previous();
    const float* x = p.logits + row * p.stride + first;
    const float temperature = p.temperature ? p.temperature[row] : 1.0f, top_p = p.top_p ? p.top_p[row] : 1.0f, min_p = p.min_p ? p.min_p[row] : 0.0f;
    const int top_k = !(temperature > 0.0f) ? 1 : (p.top_k && p.top_k[row] > 0 ? p.top_k[row] : p.vocabulary);
    auto at = [&](int i) { return STAGED ? staged[i] : cleaned(__ldcg(x + i)); };

    // ---- the largest logit ----------------------------------------------------------------------------
    float top = -INFINITY;
    {
        int i = begin + lane;
        for (; i + 7 * 32 < end; i += 8 * 32) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = __ldcg(x + i + 32 * k);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = cleaned(v[k]);
                if (STAGED) staged[i + 32 * k] = v[k];
                top = fmaxf(top, v[k]);
            }
        }
        for (; i < end; i += 32) {
            const float v = cleaned(__ldcg(x + i));
            if (STAGED) staged[i] = v;
            top = fmaxf(top, v);
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

    // ---- bounds ------------------------------------------------------------------------------------
    const float limit = kFade * temperature, scale = (float)kBins / limit;
    auto part_of = [&](float v) { const float d = top - v; return v == top ? 0 : (int)fminf(d * scale, (float)(kBins - 1)); };
    auto fades = [&](float v) { return v != top && !(top - v <= limit); };
    int lists = 0;

    // Adds up the CTAs' histograms and finds the last key's part: where the sum from the largest keys down (bins in the order given by `down`) reaches what is wanted.
    // `before`: the sum above the interval. False: it is not reached.
    auto find = [&](bool by_mass, u64 want, double share_of_mass, bool first_round, bool down, u64& before, int& part) -> bool {
        cluster.sync();  // all histograms are complete
        const int mine = kBins / ctas;
        for (int i = tid; i < mine; i += kThreads) {
            const int b = rank * mine + i;
            u64 sum = 0;
            for (int c = 0; c < ctas; ++c) sum += cluster.map_shared_rank(&sh, c)->hist[b];
            for (int c = 0; c < ctas; ++c) cluster.map_shared_rank(&sh, c)->merged[b] = sum;
        }
        cluster.sync();
        // two neighbouring parts a thread, from the largest keys down
        const int a = 2 * tid, b0 = down ? kBins - 1 - a : a, b1 = down ? b0 - 1 : a + 1;
        const u64 m0 = sh.merged[b0], m1 = sh.merged[b1];
        sh.hist[a] = sh.hist[a + 1] = 0;
        u64 scan = m0 + m1;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) { const u64 o = __shfl_up_sync(0xffffffffu, scan, off); if (lane >= off) scan += o; }
        if (lane == 31) sh.warp_sum[warp] = scan;
        if (tid == 0) sh.part = -1;
        __syncthreads();
        u64 total = 0;
        for (int w = 0; w < kWarps; ++w) { if (w < warp) scan += sh.warp_sum[w]; total += sh.warp_sum[w]; }
        if (by_mass && first_round) {
            share_of_mass = share_of_mass * (double)total;
            if (!(share_of_mass > 0.0)) share_of_mass = 0.5;  // at least one token: any weight reaches a half
            if (tid == 0) sh.total = __double_as_longlong(share_of_mass);
        }
        const u64 low = before + scan - m0 - m1, mid = low + m0, high = mid + m1;
        auto reached = [&](u64 s) { return by_mass ? (double)s >= share_of_mass : s >= want; };
        if (m0 && reached(mid) && !reached(low)) { sh.part = b0; sh.before = low; }
        if (m1 && reached(high) && !reached(mid)) { sh.part = b1; sh.before = mid; }
        __syncthreads();
        part = sh.part;
        if (part >= 0) before = sh.before;
        return part >= 0;
    };
    // The last key, in falling order, up to which the counts reach `want` or the weights the share top_p of all, among keys of at least `floor`
    auto reach = [&](bool by_mass, u64 want, u64 floor) -> u64 {
        const uint32_t floor_bits = (uint32_t)(floor >> 32);
        for (int i = begin + lane; i < end; i += 32) {
            const float v = at(i);
            if (fades(v) || ascending(v) < floor_bits || (floor && rank_key(v, first + i) < floor)) continue;
            const u64 add = by_mass ? mass_of(weight(v, top, temperature)) : 1;
            if (add) atomicAdd(&sh.hist[part_of(v)], add);
        }
        u64 before = 0;
        int part;
        double target = top_p;
        if (!find(by_mass, want, target, true, false, before, part)) return floor;
        if (by_mass) target = __longlong_as_double(sh.total);
        // the tokens of that part, or of an interval of keys in it, to the first CTA
        u64 base = 0;
        int shift = 64;
        while (true) {
            const int list = lists++ & 15;
            auto inside = [&](float v, u64 key) { return part_of(v) == part && key >= floor && key >= base && (shift == 64 || !((key - base) >> shift)); };
            for (int i = begin + lane; i < end; i += 32) {
                const float v = at(i);
                if (fades(v) || part_of(v) != part) continue;
                const u64 key = rank_key(v, first + i);
                if (!inside(v, key)) continue;
                const u64 mass = by_mass ? mass_of(weight(v, top, temperature)) : 1;
                if (!mass) continue;
                const uint32_t place = atomicAdd(&leader->listed[list], 1u);
                if (place < kList) { leader->list[place] = key; leader->list_mass[place] = mass; }
            }
            cluster.sync();
            const uint32_t n = leader->listed[list];
            if (n <= kList) {
                if (rank == 0) {
                    for (uint32_t i = tid; i < n; i += kThreads) {
                        const u64 key = sh.list[i], mass = sh.list_mass[i];
                        u64 above = before;
#pragma unroll 4
                        for (uint32_t j = 0; j < n; ++j) above += sh.list[j] > key ? sh.list_mass[j] : 0;
                        const bool reached = by_mass ? (double)(above + mass) >= target && !((double)above >= target) : above + mass >= want && above < want;
                        if (reached) sh.bound = key;
                    }
                }
                cluster.sync();
                if (tid == 0 && rank == 0) sh.listed[(list + 8) & 15] = 0;  // (eight lists on: nobody looks at that one any more)
                return leader->bound;
            }
            // more than fit: ten bits of the key further
            const int next = max(shift - 10, 0);
            for (int i = begin + lane; i < end; i += 32) {
                const float v = at(i);
                if (fades(v)) continue;
                const u64 key = rank_key(v, first + i);
                if (!inside(v, key)) continue;
                const u64 mass = by_mass ? mass_of(weight(v, top, temperature)) : 1;
                if (mass) atomicAdd(&sh.hist[(int)((key - base) >> next)], mass);
            }
            int sub = 0;
            find(by_mass, want, target, false, true, before, sub);
            if (tid == 0 && rank == 0) sh.listed[(list + 8) & 15] = 0;
            base += (u64)max(sub, 0) << next;
            shift = next;
        }
    };
    const bool nothing = top == -INFINITY;
    u64 bound = 0;
    if (!nothing && top_k < p.vocabulary) bound = reach(false, (u64)top_k, 0);
    if (!nothing && top_p < 1.0f) bound = reach(true, 0, bound);

    // ---- the draw -----------------------------------------------------------------------------------
    const uint32_t bound_bits = (uint32_t)(bound >> 32);
    auto kept_mass = [&](int i) -> u64 {
        const float v = at(i);
        if (ascending(v) < bound_bits || fades(v) || rank_key(v, first + i) < bound) return 0;
        const float e = weight(v, top, temperature);
        return e >= min_p || v == top ? mass_of(e) : 0;
    };
    u64 sum = 0, tokens = 0;
    if (!nothing)
        for (int i = begin + lane; i < end; i += 32) { const u64 w = kept_mass(i); sum += w; tokens += w != 0; }
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
    for (int c = 0; c < ctas; ++c) {
        const Shared* other = cluster.map_shared_rank(&sh, c);
        if (c < rank) ahead += other->sum;
        total += other->sum;
        all += other->count;
    }
    if (nothing) {
        if (rank == 0 && tid == 0) { p.token[row] = -1; if (p.probability) p.probability[row] = 0.0f; if (p.kept) p.kept[row] = 0; }
    } else {
        const double u = fmin(fmax((double)p.uniform[row], 0.0), 1.0);
        u64 want = (u64)(u * (double)total);
        if (want >= total) want = total - 1;
        for (int w = 0; w < warp; ++w) ahead += sh.warp_sum[w];
        if (ahead <= want && want < ahead + sh.warp_sum[warp]) {
            u64 run = ahead;
            for (int i0 = begin; i0 < end; i0 += 32) {
                const u64 w = i0 + lane < end ? kept_mass(i0 + lane) : 0;
                u64 scan = w;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) { const u64 o = __shfl_up_sync(0xffffffffu, scan, off); if (lane >= off) scan += o; }
                const uint32_t past = __ballot_sync(0xffffffffu, run + scan > want);
                if (past) {
                    if (lane == __ffs(past) - 1) {
                        p.token[row] = first + i0 + lane;
                        if (p.probability) p.probability[row] = (float)((double)w / (double)total);
                        if (p.kept) p.kept[row] = (int32_t)all;
                    }
                    break;
                }
                run += __shfl_sync(0xffffffffu, scan, 31);
            }
        }
    }
    cluster.sync();  // nobody leaves while its shared memory may be read
}

template <bool STAGED>
int launch_sample(const SampleParams& p, int rows, int ctas, cudaStream_t s) {
    static bool allowed = false;
    auto kernel = rq_sample_kernel<STAGED>;
    if (!allowed) {
        RQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        if (STAGED) RQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kShare * (int)sizeof(float)));
        allowed = true;
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
    // CTAs a row: as few as hold it, and more while the GPU has room and a share would still be some thousand logits
    int ctas = 1;
    while (ctas < kMostCtas && (vocabulary > (int64_t)ctas * kShare || ((int64_t)rows * ctas * 2 <= ctx->sm_count && vocabulary > (int64_t)ctas * 4096))) ctas *= 2;
    const int64_t unit = kThreads;  // a share is so many logits a warp, a whole number of 32
    SampleParams p = {logits, temperature, top_p, min_p, uniform, top_k, token, kept, probability, row_stride, (int)vocabulary, 0};
    p.share = (int)(((vocabulary + ctas - 1) / ctas + unit - 1) / unit * unit);
    if (p.share <= kShare) return launch_sample<true>(p, rows, ctas, (cudaStream_t)stream);
    return launch_sample<false>(p, rows, ctas, (cudaStream_t)stream);
}
