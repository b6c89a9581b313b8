// The next token of a row of logits, from one given random number.
//
// Weights are whole numbers, w = floor(2^40 exp((x - max) / T)), so that their sums are exact: which tokens top_k, top_p and min_p keep and
// which one the random number meets depend on no order of additions. Tokens are ranked by a 64-bit key, the logit's bits made
// ascending above the complement of the index: the kept tokens are those whose key is at least a bound, and the bound is found by
// refining an interval of keys, ten bits a round, from counts (top_k) or masses (top_p) of its 1024 parts.
#include "rq_serve.cuh"

using namespace rqserve;

namespace {

constexpr int kThreads = 1024, kBins = 1024;

struct SampleParams {
    const float *logits, *temperature, *top_p, *min_p, *uniform;
    const int32_t* top_k;
    int32_t *token, *kept;
    float* probability;
    int64_t stride;
    int vocabulary;
};

// NaN as -inf, -0 as +0
__device__ __forceinline__ float cleaned(float x) { return x != x ? -INFINITY : x + 0.0f; }
__device__ __forceinline__ uint64_t rank_key(float x, int index) {
    const uint32_t u = __float_as_uint(x);
    return (uint64_t)(u ^ (u >> 31 ? 0xffffffffu : 0x80000000u)) << 32 | (uint32_t)~index;
}
// the weight over 2^40; equal to the largest logit: one, also where that is +inf
__device__ __forceinline__ float weight(float x, float top, float temperature) {
    if (x == top) return 1.0f;
    return temperature > 0.0f ? expf((x - top) / temperature) : 0.0f;
}
__device__ __forceinline__ uint64_t mass_of(float e) { return (uint64_t)(e * 1099511627776.0f); }

struct Shared {
    unsigned long long mass[kBins];
    uint32_t count[kBins];
    unsigned long long warp_sum[32];
    uint64_t bound;
    unsigned long long before;
    int bin;
    float warp_top[32];
};

__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, Shared& sh, unsigned long long* inclusive = nullptr) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long scan = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) { const unsigned long long o = __shfl_up_sync(0xffffffffu, scan, off); if (lane >= off) scan += o; }
    __syncthreads();
    if (lane == 31) sh.warp_sum[warp] = scan;
    __syncthreads();
    unsigned long long total = 0;
    for (int w = 0; w < 32; ++w) { if (w == warp && inclusive) *inclusive = total + scan; total += sh.warp_sum[w]; }
    return total;
}

__global__ void __launch_bounds__(kThreads) rq_sample_kernel(SampleParams p) {
    __shared__ Shared sh;
    launch_dependents();
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.vocabulary;
    wait_for_previous();
    const float* x = p.logits + row * p.stride;
    const float temperature = p.temperature ? p.temperature[row] : 1.0f, top_p = p.top_p ? p.top_p[row] : 1.0f, min_p = p.min_p ? p.min_p[row] : 0.0f;
    const int top_k = !(temperature > 0.0f) ? 1 : (p.top_k && p.top_k[row] > 0 ? p.top_k[row] : n);
    float top = -INFINITY;
    for (int i = tid; i < n; i += kThreads) top = fmaxf(top, cleaned(x[i]));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if (lane == 0) sh.warp_top[warp] = top;
    __syncthreads();
    for (int w = 0; w < 32; ++w) top = fmaxf(top, sh.warp_top[w]);
    if (top == -INFINITY) {
        if (tid == 0) { p.token[row] = -1; if (p.probability) p.probability[row] = 0.0f; if (p.kept) p.kept[row] = 0; }
        return;
    }
    // The last key, in falling order, up to which the counts reach `want` or the masses `target`, among keys of at least `floor` with a weight
    auto reach = [&](bool by_mass, uint32_t want, double target, uint64_t floor) {
        uint64_t base = 0;
        int shift = 64;
        unsigned long long before = 0;  // count or mass above the interval
        while (shift > 0) {
            const int next = max(shift - 10, 0);
            for (int b = tid; b < kBins; b += kThreads) { sh.mass[b] = 0; sh.count[b] = 0; }
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                const float v = cleaned(x[i]);
                const uint64_t key = rank_key(v, i);
                if (key < floor || key < base || (shift < 64 && (key - base) >> shift)) continue;
                const uint64_t w = mass_of(weight(v, top, temperature));
                if (!w) continue;
                const int bin = (int)((key - base) >> next);
                atomicAdd(&sh.count[bin], 1u);
                atomicAdd(&sh.mass[bin], (unsigned long long)w);
            }
            __syncthreads();
            // bins from the largest keys down, one a thread
            const int bin = kBins - 1 - tid;
            const unsigned long long here = by_mass ? sh.mass[bin] : sh.count[bin];
            unsigned long long upto = 0;
            const unsigned long long total = block_sum(here, sh, &upto);
            if (tid == 0) sh.bin = -1;
            __syncthreads();
            const bool reached = by_mass ? (double)(before + upto) >= target : before + upto >= want;
            const bool earlier = by_mass ? (double)(before + upto - here) >= target : before + upto - here >= want;
            if (here && reached && !earlier) { sh.bin = bin; sh.before = before + upto - here; }
            __syncthreads();
            if (sh.bin < 0) { (void)total; return floor; }  // fewer than that: all of them
            before = sh.before;
            base += (uint64_t)sh.bin << next;
            shift = next;
            __syncthreads();
        }
        return base;
    };
    uint64_t bound = 0;
    if (top_k < n) bound = reach(false, (uint32_t)top_k, 0.0, 0);
    auto kept_mass = [&](int i, float v, bool with_min) -> uint64_t {
        if (rank_key(v, i) < bound) return 0;
        const float e = weight(v, top, temperature);
        return with_min && !(e >= min_p || v == top) ? 0 : mass_of(e);
    };
    if (top_p < 1.0f) {
        unsigned long long mine = 0;
        for (int i = tid; i < n; i += kThreads) mine += kept_mass(i, cleaned(x[i]), false);
        const double target = (double)top_p * (double)block_sum(mine, sh);
        bound = reach(true, 0, target > 0.0 ? target : 0.5, bound);  // at least one token: any positive mass reaches a half
    }
    // the running sum in index order: a thread takes neighbours
    const int each = (n + kThreads - 1) / kThreads, first = min(tid * each, n), last = min(first + each, n);
    unsigned long long mine = 0, upto = 0, counted = 0;
    for (int i = first; i < last; ++i) { const uint64_t w = kept_mass(i, cleaned(x[i]), true); mine += w; counted += w != 0; }
    const unsigned long long total = block_sum(mine, sh, &upto), count = block_sum(counted, sh);
    const double u = fmin(fmax((double)p.uniform[row], 0.0), 1.0);
    unsigned long long want = (unsigned long long)(u * (double)total);
    if (want >= total) want = total - 1;
    if (upto > want && upto - mine <= want) {
        unsigned long long run = upto - mine;
        for (int i = first; i < last; ++i) {
            const uint64_t w = kept_mass(i, cleaned(x[i]), true);
            run += w;
            if (run > want) {
                p.token[row] = i;
                if (p.probability) p.probability[row] = (float)((double)w / (double)total);
                if (p.kept) p.kept[row] = (int32_t)count;
                break;
            }
        }
    }
}

}  // namespace

extern "C" int rq_sample(rq_ctx* ctx, const float* logits, int64_t row_stride, int rows, int64_t vocabulary, const float* temperature, const int32_t* top_k, const float* top_p,
                         const float* min_p, const float* uniform, int32_t* token, float* probability, int32_t* kept, void* stream) {
    if (!ctx || !logits || !uniform || !token) return rq_fail(RQ_ERR_INVALID, "rq_sample: null argument");
    if (rows <= 0 || vocabulary <= 0 || (rows > 1 && row_stride < vocabulary)) return rq_fail(RQ_ERR_INVALID, "rq_sample: rows and vocabulary must be positive and row_stride at least vocabulary");
    if (vocabulary > RQ_MAX_VOCABULARY) return rq_fail(RQ_ERR_LIMIT, "rq_sample: %lld tokens; at most %d", (long long)vocabulary, RQ_MAX_VOCABULARY);
    DeviceGuard guard(ctx->device);
    SampleParams p = {logits, temperature, top_p, min_p, uniform, top_k, token, kept, probability, row_stride, (int)vocabulary};
    return launch(rq_sample_kernel, dim3((unsigned)rows), kThreads, 0, (cudaStream_t)stream, p);
}
