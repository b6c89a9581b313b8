// Log probabilities of given tokens, with entropy, rank and the likeliest alternatives, in one pass over the logits.
//
//   log p_t = (x_t - m) - log Z,  Z = sum_i e^(x_i - m);  H = log Z - sum_i e^(x_i - m) (x_i - m) / Z: two terms that are not negative, nothing cancels
//
// A row is dealt out over a cluster of up to sixteen CTAs, a contiguous share each, which go through it in rounds of sixteen logits a thread, the next round's on their way.
// A thread keeps a running maximum, the sum and the first moment against it, and how many of its logits lie ahead of the given token's (whose logit is read first).
// Alternatives: a CTA keeps a list of logits above a bound that at least `top` of those that it has seen reach. The first bound comes from the warps: the least of their
// k-th largest threads' largest logits, k = ceil(top / warps), which is reached by at least `top` logits and, where logits are in no order, by a few times as many. A list of
// more than twice `top` is cut down to the first `top` of it by comparison of all with all, and the bound is then the last of these: later logits have to be larger (equal ones
// come behind by their index). A round that would overflow the list is gone through again with the bound that 64 votes over the threads' largest find exactly, at most
// sixteen a thread over it. At the end the first CTA of the cluster joins the CTAs' sums in their order and their lists through distributed shared memory: the same bits on
// every run.
#include <cooperative_groups.h>

#include "rq_serve.cuh"

using namespace rqserve;
namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kQuads = 4, kEach = 4 * kQuads, kRound = kThreads * kEach;
constexpr int kList = 2048, kMostCtas = 16;
static_assert(kMostCtas * RQ_MAX_ALTERNATIVES <= kList && 2 * kEach * RQ_MAX_ALTERNATIVES <= kList, "lists");

typedef unsigned long long u64;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct LogprobParams {
    const float* logits;
    const int32_t* token;
    float *logprob, *entropy, *top_logprob;
    int32_t *rank, *top_token;
    int64_t stride;
    int vocabulary, top, share;  // quads a CTA
};

__device__ __forceinline__ uint32_t ascending(float x) { const uint32_t u = __float_as_uint(x); return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u); }
__device__ __forceinline__ float value_of(u64 key) { const uint32_t b = (uint32_t)(key >> 32); return __uint_as_float(b >> 31 ? b ^ 0x80000000u : ~b); }
// larger logits first, among equal ones lower indices (-0 is +0)
__device__ __forceinline__ u64 rank_key(float x, int index) { return (u64)ascending(x + 0.0f) << 32 | (uint32_t)~index; }
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// the least number above x; above the largest and +inf: none
__device__ __forceinline__ float above(float x) {
    const uint32_t u = __float_as_uint(x);
    return __uint_as_float((u << 1) == 0 ? 1u : (u >> 31 ? u - 1 : u + 1));
}

// the largest number below x (x >= -inf); below -inf: none, it is -inf
__device__ __forceinline__ float below(float x) {
    const uint32_t u = __float_as_uint(x);
    return x != x || x == -INFINITY ? -INFINITY : __uint_as_float((u << 1) == 0 ? 0x80000001u : (u >> 31 ? u + 1 : u - 1));
}

// A maximum, the sum of 2^d and of d 2^d over logits, d = (x - maximum) log2(e)
struct Sums {
    float top, sum, moment;
    __device__ __forceinline__ void move_to(float to) {  // to >= top
        const float d = top == -INFINITY ? 0.0f : fmaxf((top - to) * kLog2e, -200.0f), f = exp2_fast(d);
        moment = (moment + sum * d) * f;
        sum *= f;
        top = to;
    }
    __device__ __forceinline__ void add(Sums o) {
        const float to = fmaxf(top, o.top);
        move_to(to);
        o.move_to(to);
        sum += o.sum;
        moment += o.moment;
    }
};

struct Shared {
    u64 list[kList], best[RQ_MAX_ALTERNATIVES];
    Sums warp_sums[kWarps], sums;
    int warp_ahead[kWarps], ahead;
    uint32_t warp_bound[kWarps];
    int listed, found;  // entries of list; of best
};

// The first `top` of the n entries of the list, in order, to best; their number
__device__ __forceinline__ int keep_best(Shared& sh, int n, int top) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const u64 key = sh.list[i];
        int before = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) before += sh.list[j] > key;
        if (before < top) sh.best[before] = key;
    }
    return min(n, top);
}

template <bool ALTERNATIVES>
__global__ void __launch_bounds__(kThreads) rq_logprobs_kernel(LogprobParams p) {
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    launch_dependents();
    const float* x = p.logits + row * p.stride;
    // quads are counted from the 16-byte boundary at or before the row
    const int skew = (int)((uintptr_t)x >> 2 & 3), end = p.vocabulary + skew, quads = (end + 3) / 4;
    const int first = rank * p.share, last = min(first + p.share, quads);
    if (tid == 0) { sh.listed = 0; sh.found = 0; }
    wait_for_previous();
    const int token = p.token ? p.token[row] : -1;
    const bool has_token = token >= 0 && token < p.vocabulary;
    // A logit is ahead of the given token's where it reaches `equal`, by a lower index, or `larger`. (A token at -inf has all of lower index ahead of it, the ones that count as -inf
    // among them: these are added at the end.)
    const float mine = has_token ? fmaxf(__ldcg(x + token), -INFINITY) : INFINITY, larger = above(mine), equal = mine == -INFINITY ? NAN : mine;
    const int token_at = has_token ? token + skew : -1;
    if (ALTERNATIVES) __syncthreads();

    auto load = [&](int quad, float (&v)[kEach]) {
#pragma unroll
        for (int j = 0; j < kQuads; ++j) {
            const int at = 4 * (quad + j * kThreads);
            float4 a = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (quad + j * kThreads < last) {
                const float* from = x - skew + at;
                if (at >= skew && at + 4 <= end) {
                    a = __ldcs((const float4*)from);
                } else {
                    if (at >= skew && at < end) a.x = __ldcs(from);
                    if (at + 1 >= skew && at + 1 < end) a.y = __ldcs(from + 1);
                    if (at + 2 >= skew && at + 2 < end) a.z = __ldcs(from + 2);
                    if (at + 3 >= skew && at + 3 < end) a.w = __ldcs(from + 3);
                }
            }
            v[4 * j] = a.x; v[4 * j + 1] = a.y; v[4 * j + 2] = a.z; v[4 * j + 3] = a.w;
        }
    };

    Sums sums = {-INFINITY, 0.0f, 0.0f};
    int ahead = 0;
    float bound = -INFINITY;  // logits above it may be alternatives
    bool bounded = !ALTERNATIVES;
    float now[kEach], then[kEach];
    load(first + tid, then);
    for (int quad0 = first; quad0 < last; quad0 += kThreads * kQuads) {
        const int quad = quad0 + tid;
#pragma unroll
        for (int i = 0; i < kEach; ++i) now[i] = fmaxf(then[i], -INFINITY);  // (NaN counts as -inf)
        load(quad + kThreads * kQuads, then);
        float top = now[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i) top = fmaxf(top, now[i]);
        if (top > sums.top) sums.move_to(top);
        float sum = 0.0f, moment = 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const float d = fmaxf((now[i] - sums.top) * kLog2e, -200.0f), e = exp2_fast(d);  // (-inf: 2^-200 is none)
            sum += e;
            moment = fmaf(e, d, moment);
        }
        sums.sum += sum;
        sums.moment += moment;
#pragma unroll
        for (int j = 0; j < kQuads; ++j) {
            const int at = 4 * (quad + j * kThreads);
            if (at <= token_at && token_at <= at + 3) {
#pragma unroll
                for (int e = 0; e < 4; ++e) ahead += now[4 * j + e] >= (at + e < token_at ? equal : larger);
            } else {
                const float from = at < token_at ? equal : larger;
#pragma unroll
                for (int e = 0; e < 4; ++e) ahead += now[4 * j + e] >= from;
            }
        }
        if (ALTERNATIVES) {
            if (!bounded) {
                // the least of the warps' k-th largest of their threads' largest logits
                uint32_t key = ascending(top), kth = 0;
                for (int k = (p.top + kWarps - 1) / kWarps; k > 0; --k) {
                    kth = __reduce_max_sync(0xffffffffu, key);
                    const uint32_t who = __ballot_sync(0xffffffffu, key == kth);
                    if (lane == __ffs(who) - 1) key = 0;
                }
                if (lane == 0) sh.warp_bound[warp] = kth;
                __syncthreads();
                kth = sh.warp_bound[0];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) kth = min(kth, sh.warp_bound[w]);
                bound = below(value_of((u64)kth << 32));  // (logits that reach it are listed)
                bounded = true;
            }
            const int held = sh.listed;
            __syncthreads();  // (everybody has read it)
            auto list = [&](u64 least) {
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    if (now[i] > bound) {
                        const u64 key = rank_key(now[i], 4 * (quad + (i / 4) * kThreads) + i % 4 - skew);
                        if (key < least) continue;
                        const int at = atomicAdd(&sh.listed, 1);
                        if (at < kList) sh.list[at] = key;
                    }
                }
            };
            if (top > bound) list(0);
            __syncthreads();
            int n = sh.listed;
            if (n > kList) {
                // again, with a bound that at most `top` threads reach: the top-th of the threads' largest keys, bit by bit
                __syncthreads();
                if (tid == 0) sh.listed = held;
                u64 largest = 0;
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const u64 key = now[i] > bound ? rank_key(now[i], 4 * (quad + (i / 4) * kThreads) + i % 4 - skew) : 0;
                    largest = key > largest ? key : largest;
                }
                u64 least = 0;
                for (int bit = 63; bit >= 0; --bit)
                    if (__syncthreads_count(largest >= (least | 1ull << bit)) >= p.top) least |= 1ull << bit;
                list(least);
                __syncthreads();
                n = sh.listed;
            }
            if (n > 2 * p.top + 32) {
                keep_best(sh, n, p.top);
                __syncthreads();
                for (int i = tid; i < p.top; i += kThreads) sh.list[i] = sh.best[i];
                if (tid == 0) sh.listed = p.top;
                bound = value_of(sh.best[p.top - 1]);
                __syncthreads();
            }
        }
    }

    // ---- the CTA's sums and list -----------------------------------------------------------------------
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        Sums o;
        o.top = __shfl_xor_sync(0xffffffffu, sums.top, off);
        o.sum = __shfl_xor_sync(0xffffffffu, sums.sum, off);
        o.moment = __shfl_xor_sync(0xffffffffu, sums.moment, off);
        sums.add(o);
        ahead += __shfl_xor_sync(0xffffffffu, ahead, off);
    }
    if (lane == 0) { sh.warp_sums[warp] = sums; sh.warp_ahead[warp] = ahead; }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kWarps; ++w) { sums.add(sh.warp_sums[w]); ahead += sh.warp_ahead[w]; }
        sh.sums = sums;
        sh.ahead = ahead;
    }
    if (ALTERNATIVES) {
        const int n = keep_best(sh, sh.listed, p.top);
        if (tid == 0) sh.found = n;
    }
    if (ctas > 1) cluster.sync();
    else __syncthreads();
    if (rank == 0) {
        // ---- the row's -------------------------------------------------------------------------------
        sums = sh.sums;
        ahead = sh.ahead;
        for (int c = 1; c < ctas; ++c) {
            const Shared* other = cluster.map_shared_rank(&sh, c);
            sums.add(other->sums);
            ahead += other->ahead;
        }
        const bool nothing = sums.top == -INFINITY;
        const float log_sum = logf(sums.sum);
        if (tid == 0) {
            if (p.token) {
                if (p.logprob) p.logprob[row] = !has_token ? 0.0f : (nothing || mine == -INFINITY ? -INFINITY : (mine - sums.top) - log_sum);
                if (p.rank) p.rank[row] = has_token && !nothing ? ahead + (mine == -INFINITY ? token : 0) : -1;
            }
            if (p.entropy) p.entropy[row] = nothing ? 0.0f : log_sum - sums.moment / sums.sum * kLn2;
        }
        if (ALTERNATIVES) {
            int found = sh.found;
            if (ctas > 1) {
                // of the CTAs' lists, what is not below the last of a full one
                u64 least = 0;
                for (int c = 0; c < ctas; ++c) {
                    const Shared* other = cluster.map_shared_rank(&sh, c);
                    const u64 key = other->found == p.top ? other->best[p.top - 1] : 0;
                    least = key > least ? key : least;
                }
                __syncthreads();
                if (tid == 0) sh.listed = 0;
                __syncthreads();
                for (int i = tid; i < ctas * p.top; i += kThreads) {
                    const int c = i / p.top, at = i % p.top;
                    const Shared* other = cluster.map_shared_rank(&sh, c);
                    if (at >= other->found) continue;
                    const u64 key = other->best[at];
                    if (key >= least) sh.list[atomicAdd(&sh.listed, 1)] = key;
                }
                __syncthreads();
                found = keep_best(sh, sh.listed, p.top);
                __syncthreads();
            }
            for (int i = tid; i < p.top; i += kThreads) {
                const bool there = i < found;
                if (p.top_token) p.top_token[(int64_t)row * p.top + i] = there ? (int32_t)~(uint32_t)sh.best[i] : -1;
                if (p.top_logprob) p.top_logprob[(int64_t)row * p.top + i] = there ? (value_of(sh.best[i]) - sums.top) - log_sum : -INFINITY;
            }
        }
    }
    if (ctas > 1) cluster.sync();  // nobody leaves while its shared memory may be read
}

template <bool ALTERNATIVES>
int launch_logprobs(rq_ctx* ctx, const LogprobParams& p, int rows, int ctas, cudaStream_t s) {
    auto kernel = rq_logprobs_kernel<ALTERNATIVES>;
    static bool configured[64] = {};  // by device: the opt-in to clusters of sixteen
    if (ctx->device >= 64 || !configured[ctx->device]) {
        RQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        if (ctx->device < 64) configured[ctx->device] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * ctas));
    cfg.blockDim = dim3(kThreads);
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

extern "C" int rq_logprobs(rq_ctx* ctx, const float* logits, int64_t row_stride, int rows, int64_t vocabulary, const int32_t* token, float* logprob, float* entropy, int32_t* rank,
                           int top, int32_t* top_token, float* top_logprob, void* stream) {
    if (!ctx || !logits || (!token && (logprob || rank))) return rq_fail(RQ_ERR_INVALID, "rq_logprobs: null argument (logprob and rank are a token's)");
    if (rows <= 0 || vocabulary <= 0 || (rows > 1 && row_stride < vocabulary)) return rq_fail(RQ_ERR_INVALID, "rq_logprobs: rows and vocabulary must be positive and row_stride at least vocabulary");
    if (vocabulary > RQ_MAX_VOCABULARY) return rq_fail(RQ_ERR_LIMIT, "rq_logprobs: %lld tokens; at most %d", (long long)vocabulary, RQ_MAX_VOCABULARY);
    if (rows > (1 << 26)) return rq_fail(RQ_ERR_LIMIT, "rq_logprobs: %d rows; at most 2^26", rows);
    if (top < 0 || top > RQ_MAX_ALTERNATIVES) return rq_fail(RQ_ERR_LIMIT, "rq_logprobs: %d alternatives; from 0 to %d", top, RQ_MAX_ALTERNATIVES);
    if (top > 0 && !top_token && !top_logprob) return rq_fail(RQ_ERR_INVALID, "rq_logprobs: alternatives without a place for them");
    if (((uintptr_t)logits & 3) != 0) return rq_fail(RQ_ERR_INVALID, "rq_logprobs: logits must be 4-byte aligned");
    DeviceGuard guard(ctx->device);
    int ctas = 1;
    while (ctas < kMostCtas && (int64_t)rows * ctas * 2 <= 8 * ctx->sm_count && vocabulary > (int64_t)ctas * 2 * kRound) ctas *= 2;
    LogprobParams p = {logits, token, logprob, entropy, top_logprob, rank, top_token, row_stride, (int)vocabulary, top, 0};
    p.share = (int)(((vocabulary + 3 + 3) / 4 + ctas - 1) / ctas);  // (a row may begin three logits behind a boundary)
    return top > 0 ? launch_logprobs<true>(ctx, p, rows, ctas, (cudaStream_t)stream) : launch_logprobs<false>(ctx, p, rows, ctas, (cudaStream_t)stream);
}
