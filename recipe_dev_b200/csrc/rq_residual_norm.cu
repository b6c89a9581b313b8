// From one block of a layer to the next: the norm behind the block, its gate and scale, the residual sum, and the norm in front of the next block.
//
//   x' = x + r gate norm(delta),  y = norm(x'),  norm(v) = v / sqrt(mean(v^2) + epsilon) * gain
//
// A CTA takes a token and holds it in registers from its one reading to its last writing: two sums over the CTA, one barrier each, lie between them. Bound by bytes
// for a prompt, by the launch and the chain of a load and two sums for a few tokens. Sums of squares are held in fp32: of a thread's elements, of a warp by shuffles, of
// the warps by shuffles again, in every warp for itself; the order follows from the width alone, so that a token has the same bits in every call.
// 2039 tokens of 4096 with a gate for each element 30.5 us, 5.4 TB/s, 0.83 of the measured copy (one element in four a thread 34.5, sixteen elements a thread 35.4, eight with gates and
// gains loaded where they are used 32.5); 64 of 2560 7.9 us and one of 4096 7.6, which is what a call from Python takes (in a
// recorded sequence 3.0 and 2.1).
#include "rq_serve.cuh"

using namespace rqserve;

namespace {

struct JoinParams {
    const float *x, *delta, *delta_gain, *gate, *gain;
    float *x_out, *y;
    int64_t x_stride, delta_stride, gate_stride, out_stride, y_stride, n;
    int gate_elements;  // a gate's value an element (1), or one for the token (0)
    float scale, epsilon;
};

// Elements at .. at + 3 of a token, those past its n as zeros; WIDE: 16-byte accesses. KEEP: through the L1 cache, for what other tokens' CTAs read too.
template <bool WIDE, bool KEEP = false> __device__ __forceinline__ float4 load4(const float* p, int64_t at, int64_t n) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (WIDE) {
        if (at < n) v = KEEP ? *(const float4*)(p + at) : __ldcg((const float4*)(p + at));
    } else {
        if (at < n) v.x = KEEP ? p[at] : __ldcg(p + at);
        if (at + 1 < n) v.y = KEEP ? p[at + 1] : __ldcg(p + at + 1);
        if (at + 2 < n) v.z = KEEP ? p[at + 2] : __ldcg(p + at + 2);
        if (at + 3 < n) v.w = KEEP ? p[at + 3] : __ldcg(p + at + 3);
    }
    return v;
}
template <bool WIDE> __device__ __forceinline__ void store4(float* p, int64_t at, int64_t n, float4 v) {
    if (WIDE) {
        if (at < n) *(float4*)(p + at) = v;
    } else {
        if (at < n) p[at] = v.x;
        if (at + 1 < n) p[at + 1] = v.y;
        if (at + 2 < n) p[at + 2] = v.z;
        if (at + 3 < n) p[at + 3] = v.w;
    }
}
__device__ __forceinline__ float squares(float4 v, float sum) { return fmaf(v.w, v.w, fmaf(v.z, v.z, fmaf(v.y, v.y, fmaf(v.x, v.x, sum)))); }

// The CTA's sum, in every thread; `warps` is this sum's own
__device__ __forceinline__ float block_sum(float v, float* warps) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    if (lane == 0) warps[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < (int)(blockDim.x >> 5) ? warps[lane] : 0.0f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// HELD: four elements each that a thread holds; 0: rows beyond what a CTA holds, gone through again for each sum
template <int HELD, bool WIDE>
__global__ void __launch_bounds__(1024) rq_residual_norm_kernel(JoinParams p) {
    __shared__ float behind[32], ahead[32];
    launch_dependents();
    const int64_t t = blockIdx.x, first = 4 * (int64_t)threadIdx.x, step = 4 * (int64_t)blockDim.x;
    const float *x = p.x + t * p.x_stride, *delta = p.delta + t * p.delta_stride, *gate = p.gate + t * p.gate_stride;
    float *out = p.x_out + t * p.out_stride, *y = p.y + t * p.y_stride;
    wait_for_previous();
    const float one_gate = p.gate && !p.gate_elements ? __ldcg(gate) : 1.0f;
    float of_delta = 1.0f;
    // what is read of a gain or gate: ones where there is none
    auto ones_or = [&](const float* from, int64_t at) { return from ? load4<WIDE, true>(from, at, p.n) : make_float4(1.0f, 1.0f, 1.0f, 1.0f); };
    auto gate_of = [&](int64_t at) { return p.gate && p.gate_elements ? load4<WIDE>(gate, at, p.n) : make_float4(one_gate, one_gate, one_gate, one_gate); };
    // x' of four elements
    auto join = [&](float4 a, float4 d, float4 of_block, float4 g) {
        if (p.delta_gain) { d.x = d.x * of_delta * of_block.x; d.y = d.y * of_delta * of_block.y; d.z = d.z * of_delta * of_block.z; d.w = d.w * of_delta * of_block.w; }
        return make_float4(fmaf(p.scale, d.x * g.x, a.x), fmaf(p.scale, d.y * g.y, a.y), fmaf(p.scale, d.z * g.z, a.z), fmaf(p.scale, d.w * g.w, a.w));
    };
    auto normed = [&](float4 v, float f, float4 g) { return make_float4(v.x * f * g.x, v.y * f * g.y, v.z * f * g.z, v.w * f * g.w); };
    auto factor = [&](float sum) { return 1.0f / sqrtf(sum / (float)p.n + p.epsilon); };
    if (HELD) {
        constexpr int N = HELD ? HELD : 1;
        constexpr bool kAhead = N <= 2;  // gains and gates on their way with the rest (of four, registers do not hold them)
        float4 a[N], d[N], g[N], block_gain[N];
#pragma unroll
        for (int i = 0; i < N; ++i) { d[i] = load4<WIDE>(delta, first + i * step, p.n); a[i] = load4<WIDE>(x, first + i * step, p.n); }
        if (kAhead)
#pragma unroll
            for (int i = 0; i < N; ++i) { g[i] = gate_of(first + i * step); block_gain[i] = ones_or(p.delta_gain, first + i * step); }
        if (p.delta_gain) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) sum = squares(d[i], sum);
            of_delta = factor(block_sum(sum, behind));
        }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            a[i] = kAhead ? join(a[i], d[i], block_gain[i], g[i]) : join(a[i], d[i], ones_or(p.delta_gain, first + i * step), gate_of(first + i * step));
            store4<WIDE>(out, first + i * step, p.n, a[i]);
            sum = squares(a[i], sum);
        }
        if (kAhead)
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = ones_or(p.gain, first + i * step);
        const float f = factor(block_sum(sum, ahead));
#pragma unroll
        for (int i = 0; i < N; ++i) store4<WIDE>(y, first + i * step, p.n, normed(a[i], f, kAhead ? g[i] : ones_or(p.gain, first + i * step)));
    } else {
        if (p.delta_gain) {
            float sum = 0.0f;
#pragma unroll 4
            for (int64_t at = first; at < p.n; at += step) sum = squares(load4<WIDE>(delta, at, p.n), sum);
            of_delta = factor(block_sum(sum, behind));
        }
        float sum = 0.0f;
#pragma unroll 2
        for (int64_t at = first; at < p.n; at += step) {
            const float4 v = join(load4<WIDE>(x, at, p.n), load4<WIDE>(delta, at, p.n), ones_or(p.delta_gain, at), gate_of(at));
            store4<WIDE>(out, at, p.n, v);
            sum = squares(v, sum);
        }
        const float f = factor(block_sum(sum, ahead));
        // (a thread reads again what it wrote itself)
#pragma unroll 4
        for (int64_t at = first; at < p.n; at += step) store4<WIDE>(y, at, p.n, normed(load4<WIDE>(out, at, p.n), f, ones_or(p.gain, at)));
    }
}

template <int HELD>
int launch_join(const JoinParams& p, int tokens, unsigned threads, bool wide, cudaStream_t s) {
    return launch(wide ? rq_residual_norm_kernel<HELD, true> : rq_residual_norm_kernel<HELD, false>, dim3((unsigned)tokens), threads, 0, s, p);
}

}  // namespace

extern "C" int rq_residual_norm(rq_ctx* ctx, const float* x, int64_t x_t_stride, const float* delta, int64_t delta_t_stride, int64_t n, int tokens, const float* delta_gain,
                                const float* gate, int64_t gate_k_stride, int64_t gate_t_stride, float residual_scale, const float* gain, float epsilon, float* x_out,
                                int64_t x_out_t_stride, float* y, int64_t y_t_stride, void* stream) {
    if (!ctx || !x || !delta || !x_out || !y) return rq_fail(RQ_ERR_INVALID, "rq_residual_norm: null argument");
    if (n <= 0 || tokens <= 0 || n > (int64_t)1 << 31) return rq_fail(RQ_ERR_INVALID, "rq_residual_norm: n (up to 2^31) and tokens must be positive");
    if (tokens > 1 && (x_t_stride < n || delta_t_stride < n || x_out_t_stride < n || y_t_stride < n)) return rq_fail(RQ_ERR_INVALID, "rq_residual_norm: token strides must be at least n");
    if (gate && ((gate_k_stride != 0 && gate_k_stride != 1) || gate_t_stride < 0)) return rq_fail(RQ_ERR_INVALID, "rq_residual_norm: gate_k_stride must be 0 or 1 and gate_t_stride not negative");
    if (!(epsilon >= 0.0f)) return rq_fail(RQ_ERR_INVALID, "rq_residual_norm: epsilon must be non-negative");
    DeviceGuard guard(ctx->device);
    JoinParams p = {x, delta, delta_gain, gate, gain, x_out, y, x_t_stride, delta_t_stride, gate ? gate_t_stride : 0, x_out_t_stride, y_t_stride, n, (int)gate_k_stride, residual_scale, epsilon};
    const bool elements = gate && gate_k_stride;
    const bool wide = (((uintptr_t)x | (uintptr_t)delta | (uintptr_t)delta_gain | (uintptr_t)gain | (uintptr_t)x_out | (uintptr_t)y | (elements ? (uintptr_t)gate : 0)) & 15) == 0 && n % 4 == 0 &&
                      (tokens == 1 || ((x_t_stride | delta_t_stride | x_out_t_stride | y_t_stride | (elements ? gate_t_stride : 0)) & 3) == 0);
    const int64_t quads = (n + 3) / 4;
    auto threads = [&](int held) { return (unsigned)((quads + 32 * held - 1) / (32 * held) * 32); };
    cudaStream_t s = (cudaStream_t)stream;
    if (quads <= 2 * 1024) return launch_join<2>(p, tokens, threads(2), wide, s);
    if (quads <= 4 * 1024) return launch_join<4>(p, tokens, threads(4), wide, s);
    return launch_join<0>(p, tokens, 1024, wide, s);
}
