// Log probabilities of given tokens, with entropy, rank and the likeliest alternatives, in one pass over the logits.
//
//   log p_t = (x_t - m) - log Z,  Z = sum_i e^(x_i - m);  H = log Z - sum_i e^(x_i - m) (x_i - m) / Z: two terms that are not negative, nothing cancels
//
// A row is dealt out over a cluster of up to eight CTAs (few rows: sixteen), a contiguous share each, which stream through it: a thread keeps a running maximum, the sum and the
// first moment against it, and how many of its logits lie ahead of the given token's (whose logit is read beside the first ones). There is no barrier before the end of a share.
// Alternatives: each thread also leaves the largest logit of each of up to sixteen segments of its logits in shared memory. The `top`-th largest of the threads' largest logits (its
// upper sixteen bits, by a search of one warp) is a bound that at least `top` logits of the share reach, and the largest of the CTAs' bounds holds for the row. Segments that
// reach it are read again (from L2), and their logits that reach it, a few times `top` of the row's, go to the CTA's part of the first CTA's list, which puts them in order by
// comparison of all with all. Where equal or ordered logits overflow a part, the exact key of the `top`-th logit is found bit by bit, in 64 rounds over the row. What
// others need is written into their shared memory; a cluster meets twice.
// Sums are joined in a fixed order: the same bits on every run.
//
// Bound by bytes for many rows: 2039 x 32000 without alternatives 50 us, 5.2 TB/s, 0.79 of the measured copy (23 instructions a logit, one at a time, in place of nine: 55). For rows that a cluster
// each takes, by what comes behind the stream: 64 x 262144 with twenty alternatives 27.6 us, 13 to 16 of them the stream (CTAs of SMs that hold four, or three), then 1 for the sums, 1.5 for
// the bound, 1.5 for each meeting, 3 for the segments, 2 for the order; 2039 x 32000 with twenty 77. One row in a recorded sequence: of 32000 3.7 us, with twenty alternatives 8.4, of 262144
// with twenty 12.7. A list kept up to date in every round, with barriers: 60 us by sixteen CTAs a row, 34 by eight.
#include <cooperative_groups.h>

#include "rq_pairs.cuh"
#include "rq_serve.cuh"

using namespace rqserve;
namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kQuads = 4, kEach = 4 * kQuads, kRound = kThreads * kEach;
constexpr int kList = 2048, kMostCtas = 16, kSegments = 16;

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

// Sums of a warp's lanes, over lanes 0 .. n - 1 (a power of two) in lane 0, in a fixed order
__device__ __forceinline__ void add_lanes(Sums& sums, int& ahead, int n) {
    for (int off = n / 2; off > 0; off >>= 1) {
        Sums o;
        o.top = __shfl_down_sync(0xffffffffu, sums.top, off);
        o.sum = __shfl_down_sync(0xffffffffu, sums.sum, off);
        o.moment = __shfl_down_sync(0xffffffffu, sums.moment, off);
        sums.add(o);
        ahead += __shfl_down_sync(0xffffffffu, ahead, off);
    }
}

struct Shared {
    Sums warp_sums[kWarps];
    int warp_ahead[kWarps];
    // the first CTA's: of the CTAs
    Sums sums[kMostCtas];
    int ahead[kMostCtas];
    float row_top, log_sum;
};
struct Lists {
    union {
        float largest[kSegments][kThreads];  // of a thread's segments
        u64 kept[kList];                     // the first CTA's, at the end: all logits that reach the row's bound (of small shared memory, loads have the L1 cache to be on their way in)
    };
    uint32_t keys[kThreads];             // of the threads' largest logits
    int listed;
    // every CTA's: the CTAs' bounds, each reached by at least `top` logits of a share, and how many logits they have sent
    float bounds[kMostCtas];
    int sent[kMostCtas];
    // the first CTA's: the CTAs' logits that reach the row's bound, a part each, and the first of them
    u64 list[kList], best[RQ_MAX_ALTERNATIVES];
    int held;
    u64 warp_count[kWarps], count;
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

template <bool ALTERNATIVES>
__global__ void __launch_bounds__(kThreads) rq_logprobs_kernel(LogprobParams p) {
    __shared__ Shared sh;
    extern __shared__ __align__(16) unsigned char dynamic[];
    Lists& lists = *(Lists*)dynamic;  // (with alternatives)
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    launch_dependents();
    if (ctas > 1) cluster_arrive();  // (nobody writes to a CTA that has not begun)
    const float* x = p.logits + row * p.stride;
    // quads are counted from the 16-byte boundary at or before the row
    const int skew = (int)((uintptr_t)x >> 2 & 3), end = p.vocabulary + skew, quads = (end + 3) / 4;
    const int first = rank * p.share, last = min(first + p.share, quads);
    wait_for_previous();

    // sixteen logits of the round that begins at `quad0`: four quads, neighbours by thread; past the share's ends -inf
    const float* const row_at = x - skew;
    const int whole = min(last, end / 4);  // quads below lie inside, from the second one on (the first one too, where the row begins at a boundary)
    auto load = [&](int quad0, float (&v)[kEach]) {
        const float* from = row_at + 4 * (int64_t)(quad0 + tid);
        if ((quad0 > 0 || skew == 0) && quad0 + kThreads * kQuads <= whole) {
#pragma unroll
            for (int j = 0; j < kQuads; ++j) {
                const float4 a = __ldcg((const float4*)from + j * kThreads);
                v[4 * j] = a.x; v[4 * j + 1] = a.y; v[4 * j + 2] = a.z; v[4 * j + 3] = a.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int quad = quad0 + tid + i / 4 * kThreads, at = 4 * quad + i % 4;
                v[i] = quad < last && at >= skew && at < end ? __ldcg(from + 4 * (i / 4) * kThreads + i % 4) : -INFINITY;
            }
        }
    };
    auto key_of = [&](float v, int quad0, int i) { return rank_key(v, 4 * (quad0 + tid + (i / 4) * kThreads) + i % 4 - skew); };

    float v[kEach];
    load(first, v);
    const int token = p.token ? p.token[row] : -1;
    const bool has_token = token >= 0 && token < p.vocabulary;
    // A logit is ahead of the given token's where it reaches `equal`, by a lower index, or `larger`. (A token at -inf has all of lower index ahead of it, the ones that count as -inf
    // among them: these are added at the end.)
    const float mine = has_token ? fmaxf(__ldcg(x + token), -INFINITY) : INFINITY, larger = above(mine), equal = mine == -INFINITY ? NAN : mine;
    const int token_at = has_token ? token + skew : -1;

    // ---- the share -------------------------------------------------------------------------------------
    const int rounds = (p.share + kThreads * kQuads - 1) / (kThreads * kQuads), segment_rounds = (rounds + kSegments - 1) / kSegments;
    Sums sums = {-INFINITY, 0.0f, 0.0f};
    float segment_top = -INFINITY;
    int ahead = 0, left = segment_rounds, segment = 0;
    Pair sum = pair_of(0.0f, 0.0f), moment = sum;  // of the even logits, of the odd ones
    const Pair scale = pair_of(kLog2e, kLog2e);
    const bool ranked = p.rank != nullptr && has_token;
    for (int round = 0, quad0 = first; round < rounds; ++round, quad0 += kThreads * kQuads) {
        if (round) load(quad0, v);
        float top = v[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i) top = fmaxf(top, v[i]);
        if (top > sums.top) {
            // the sums against the new maximum: (m + s d) f, s f
            const float d = sums.top == -INFINITY ? 0.0f : fmaxf((sums.top - top) * kLog2e, -200.0f), f = exp2_fast(d);
            moment = pair_mul(pair_fma(sum, pair_of(d, d), moment), pair_of(f, f));
            sum = pair_mul(sum, pair_of(f, f));
            sums.top = top;
        }
        const Pair down = pair_of(-sums.top, -sums.top);
        Pair here = pair_of(0.0f, 0.0f), here_moment = here;
#pragma unroll
        for (int i = 0; i < kEach; i += 2) {
            Pair d = pair_mul(pair_add(pair_of(v[i], v[i + 1]), down), scale);
            const float a = fmaxf(pair_at(d, 0), -200.0f), b = fmaxf(pair_at(d, 1), -200.0f);  // (-inf and NaN: 2^-200 is none)
            const Pair e = pair_of(exp2_fast(a), exp2_fast(b));
            here = pair_add(here, e);
            here_moment = pair_fma(e, pair_of(a, b), here_moment);
        }
        sum = pair_add(sum, here);
        moment = pair_add(moment, here_moment);
        if (ranked && top >= mine) {  // (none of a round's is ahead otherwise, and of a token at -inf all above are)
#pragma unroll
            for (int j = 0; j < kQuads; ++j) {
                const int at = 4 * (quad0 + tid + j * kThreads);
                if (at <= token_at && token_at <= at + 3) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) ahead += v[4 * j + e] >= (at + e < token_at ? equal : larger);
                } else {
                    const float from = at < token_at ? equal : larger;
#pragma unroll
                    for (int e = 0; e < 4; ++e) ahead += v[4 * j + e] >= from;
                }
            }
        }
        if (ALTERNATIVES) {
            segment_top = fmaxf(segment_top, top);
            if (--left == 0) {
                lists.largest[segment++][tid] = segment_top;
                segment_top = -INFINITY;
                left = segment_rounds;
            }
        }
    }
    sums.sum = pair_at(sum, 0) + pair_at(sum, 1);
    sums.moment = pair_at(moment, 0) + pair_at(moment, 1);
    if (ALTERNATIVES) {
        if (left != segment_rounds) lists.largest[segment++][tid] = segment_top;
        lists.keys[tid] = ascending(sums.top + 0.0f);
        if (tid == 0) { lists.listed = 0; lists.held = 0; }
    }
    add_lanes(sums, ahead, 32);
    if (lane == 0) { sh.warp_sums[warp] = sums; sh.warp_ahead[warp] = ahead; }
    __syncthreads();
    if (ctas > 1) cluster_wait();
    Shared* const first_sh = ctas > 1 ? cluster.map_shared_rank(&sh, 0) : &sh;
    Lists* const first_lists = !ALTERNATIVES ? nullptr : (ctas > 1 ? cluster.map_shared_rank(&lists, 0) : &lists);
    if (warp == kWarps - 1) {
        sums = sh.warp_sums[lane % kWarps];
        ahead = sh.warp_ahead[lane % kWarps];
        add_lanes(sums, ahead, kWarps);
        if (lane == 0) { first_sh->sums[rank] = sums; first_sh->ahead[rank] = ahead; }
    }
    auto meet = [&]() {
        if (ctas > 1) { cluster_arrive(); cluster_wait(); }
        else __syncthreads();
    };
    const int part = kList / ctas;
    if (ALTERNATIVES) {
        if (warp == 0) {
            // the top-th of the threads' largest logits, by the upper sixteen bits of its place in their order
            uint32_t key[kThreads / 32], bound = 0;
#pragma unroll
            for (int i = 0; i < kThreads / 32; ++i) key[i] = lists.keys[32 * i + lane];
#pragma unroll 1
            for (int bit = 30; bit >= 16; bit -= 2) {  // two bits a step: how many reach each of three, ten bits a count
                const uint32_t step = 1u << bit;
                uint32_t count = 0;
#pragma unroll
                for (int i = 0; i < kThreads / 32; ++i) count += (key[i] >= bound + step ? 1u : 0u) + (key[i] >= bound + 2 * step ? 1u << 10 : 0u) + (key[i] >= bound + 3 * step ? 1u << 20 : 0u);
                count = __reduce_add_sync(0xffffffffu, count);
                if ((int)(count >> 20) >= p.top) bound += 3 * step;
                else if ((int)(count >> 10 & 1023) >= p.top) bound += 2 * step;
                else if ((int)(count & 1023) >= p.top) bound += step;
            }
            const float at = bound <= ascending(-INFINITY) ? -INFINITY : value_of((u64)bound << 32);
            if (lane < ctas) (ctas > 1 ? cluster.map_shared_rank(&lists, lane) : &lists)->bounds[rank] = at;
        }
    }
    meet();

    // ---- the row's -----------------------------------------------------------------------------------
    if (rank == 0 && warp == kWarps - 1) {
        if (ctas > 1) {
            sums = sh.sums[lane % ctas];
            ahead = sh.ahead[lane % ctas];
            add_lanes(sums, ahead, ctas);
        }
        if (lane == 0) {
            const bool nothing = sums.top == -INFINITY;
            const float log_sum = logf(sums.sum);
            if (p.token) {
                if (p.logprob) p.logprob[row] = !has_token ? 0.0f : (nothing || mine == -INFINITY ? -INFINITY : (mine - sums.top) - log_sum);
                if (p.rank) p.rank[row] = has_token && !nothing ? ahead + (mine == -INFINITY ? token : 0) : -1;
            }
            if (p.entropy) p.entropy[row] = nothing ? 0.0f : log_sum - sums.moment / sums.sum * kLn2;
            sh.row_top = sums.top;
            sh.log_sum = log_sum;
        }
        __syncwarp();
    }
    if (ALTERNATIVES) {
        // logits that reach the bound, and the key, to this CTA's part of the first one's list
        float bound = lists.bounds[0];
        for (int c = 1; c < ctas; ++c) bound = fmaxf(bound, lists.bounds[c]);
        auto send = [&](u64 least) {
            for (int n = 0; n < segment; ++n) {
                if (!(lists.largest[n][tid] >= bound)) continue;
                for (int round = n * segment_rounds; round < min((n + 1) * segment_rounds, rounds); ++round) {
                    const int quad0 = first + round * kThreads * kQuads;
                    load(quad0, v);
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {
                        if (v[i] >= bound && v[i] > -INFINITY) {
                            const u64 key = key_of(v[i], quad0, i);
                            if (key < least) continue;
                            const int at = atomicAdd(&lists.listed, 1);
                            if (at < part) first_lists->list[rank * part + at] = key;
                        }
                    }
                }
            }
            __syncthreads();
            if (tid < ctas) (ctas > 1 ? cluster.map_shared_rank(&lists, tid) : &lists)->sent[rank] = lists.listed;
        };
        send(0);
        meet();
        bool overflow = false;
        for (int c = 0; c < ctas; ++c) overflow = overflow || lists.sent[c] > part;
        if (overflow) {
            // too many that are equal to a bound or nearly: the key of the top-th logit, bit by bit, is one that exactly `top` reach
            u64 least = 0;
#pragma unroll 1
            for (int bit = 63; bit >= 0; --bit) {
                const u64 tried = least | 1ull << bit;
                int count = 0;
                for (int n = 0; n < segment; ++n) {
                    if (!(lists.largest[n][tid] >= bound)) continue;
                    for (int round = n * segment_rounds; round < min((n + 1) * segment_rounds, rounds); ++round) {
                        const int quad0 = first + round * kThreads * kQuads;
                        load(quad0, v);
#pragma unroll
                        for (int i = 0; i < kEach; ++i) count += v[i] >= bound && v[i] > -INFINITY && key_of(v[i], quad0, i) >= tried;
                    }
                }
                const int of_warp = __reduce_add_sync(0xffffffffu, count);
                if (lane == 0) lists.warp_count[warp] = of_warp;
                __syncthreads();
                if (tid == 0) {
                    u64 sum = 0;
                    for (int w = 0; w < kWarps; ++w) sum += lists.warp_count[w];
                    lists.count = sum;
                }
                meet();
                u64 sum = 0;
                for (int c = 0; c < ctas; ++c) sum += (ctas > 1 ? cluster.map_shared_rank(&lists, c) : &lists)->count;
                if (sum >= (u64)p.top) least = tried;
                meet();  // (counts have been read)
            }
            if (tid == 0) lists.listed = 0;
            __syncthreads();
            send(least);
            meet();
        }
        if (rank != 0) return;
        // all that is needed lies in the first CTA
        for (int c = warp; c < ctas; c += kWarps)
            for (int i = lane; i < lists.sent[c]; i += 32) lists.kept[atomicAdd(&lists.held, 1)] = lists.list[c * part + i];
        __syncthreads();
        const int n = lists.held, found = min(n, p.top);
        for (int i = tid; i < n; i += kThreads) {
            const u64 key = lists.kept[i];
            int before = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) before += lists.kept[j] > key;
            if (before < p.top) lists.best[before] = key;
        }
        __syncthreads();
        for (int i = tid; i < p.top; i += kThreads) {
            const bool there = i < found;
            if (p.top_token) p.top_token[(int64_t)row * p.top + i] = there ? (int32_t)~(uint32_t)lists.best[i] : -1;
            if (p.top_logprob) p.top_logprob[(int64_t)row * p.top + i] = there ? (value_of(lists.best[i]) - sh.row_top) - sh.log_sum : -INFINITY;
        }
    }
}

template <bool ALTERNATIVES>
int launch_logprobs(rq_ctx* ctx, const LogprobParams& p, int rows, int ctas, cudaStream_t s) {
    auto kernel = rq_logprobs_kernel<ALTERNATIVES>;
    static bool configured[64] = {};  // by device: the opt-ins to clusters of sixteen and to large shared memory
    if (ctx->device >= 64 || !configured[ctx->device]) {
        RQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        if (ALTERNATIVES) RQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Lists)));
        if (ctx->device < 64) configured[ctx->device] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = ALTERNATIVES ? sizeof(Lists) : 0;
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
    // CTAs a row: as many as the GPU holds at once (four an SM), of shares of two rounds and more; sixteen where every CTA has an SM to itself
    int ctas = 1;
    while (ctas < kMostCtas && (int64_t)rows * ctas * 2 <= (ctas == 8 ? 1 : 4) * ctx->sm_count && vocabulary > (int64_t)ctas * 2 * kRound) ctas *= 2;
    LogprobParams p = {logits, token, logprob, entropy, top_logprob, rank, top_token, row_stride, (int)vocabulary, top, 0};
    p.share = (int)(((vocabulary + 3 + 3) / 4 + ctas - 1) / ctas);  // (a row may begin three logits behind a boundary)
    return top > 0 ? launch_logprobs<true>(ctx, p, rows, ctas, (cudaStream_t)stream) : launch_logprobs<false>(ctx, p, rows, ctas, (cudaStream_t)stream);
}
