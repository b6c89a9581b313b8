// What the kernels of rq_attention share: parameters, the 16-bit parts of fp32 numbers, and how a batch's keys are dealt out.
#pragma once
#include "rq_serve.cuh"

namespace rqattn {

struct AttentionParams {
    const float* q;
    float* y;
    const uint16_t *k, *v;
    const int32_t *block_table, *starts, *lengths;
    float* partial;      // sums of rows whose keys several CTAs share
    uint32_t* arrived;   // per CTA (the tensor-core kernel: and warp of rows): how many have left their part of the rows that begin there; zero between calls
    int64_t q_stride, y_stride, table_stride, head_stride, pages;
    uint32_t page_bytes, line_bytes;
    int tokens, requests, q_heads, kv_heads, table_width, page_shift, window;
    int few;  // requests of at most so many rows a key head are the rows kernel's, the others the tensor-core kernel's
    float scale;
    int wide;  // q and y allow accesses of 16 bytes (1), of 32 (2)
    int* error_flag;
    unsigned long long wait_ns;
};
// A cache of codes: the scales of each position's head
struct CodesParams : AttentionParams {
    const float *k_scale, *v_scale;
    int64_t scale_page, scale_head, scale_line;
    float scale_size;  // scale * log2(e) = scale_size * 2^scale_exponent, 1 <= scale_size <= 2
    int scale_exponent;
};

// What the work area holds: sums of rows for each CTA's first and last item (the tensor-core kernel: two tiles of 128 rows of 128 elements and their
// bases and sums of weights), then the counts.
constexpr int kTensorCtas = 148, kRowCtas = 148 * 4;
constexpr size_t kTensorPartial = (size_t)kTensorCtas * 2 * 2 * 128 * (128 + 2), kRowPartial = (size_t)kRowCtas * 2 * 16 * (256 + 2);  // floats
constexpr size_t kCounts = kTensorCtas * 2 * 4 > kRowCtas ? kTensorCtas * 2 * 4 : kRowCtas;
constexpr size_t kPartialBytes = sizeof(float) * (kTensorPartial > kRowPartial ? kTensorPartial : kRowPartial);

// Rows by the hundred (rq_attention_tc.cu); one_tile: at most 128 rows a request and key head. RQ_ERR_UNSUPPORTED (no error text) = a cache that it does not
// serve: 256 elements a head, pages of fewer than eight positions, strides of zero.
int launch_tensor(rq_ctx* ctx, const CodesParams& p, const rq_kv_cache& cache, bool one_tile, cudaStream_t s);

// Rows by the few over a cache of codes (rq_attention_int8.cu); two: sixteen rows at a time
int launch_rows_int8(rq_ctx* ctx, const CodesParams& p, const rq_kv_cache& cache, bool two, cudaStream_t s);

constexpr float kLog2e = 1.4426950408889634f;
// Weights are 2^(s - max + kRaise): an f16 part below 2^-14 loses bits, raised by 2^12 that is a weight of 2^-26 of the row's largest. bf16 has fp32's exponents: its
// parts need none of it, and values near the end of its range leave sums no room for it.
template <int TYPE> constexpr float kRaise = TYPE == RQ_KV_F16 ? 12.0f : 0.0f;

#ifdef __CUDACC__
// How many of a request's new tokens the call has queries for: a batch may be longer than the call
__device__ __forceinline__ int tokens_here(const AttentionParams& p, int start, int next) { return start < 0 ? 0 : max(min(next, p.tokens) - start, 0); }

__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// Codes of a cache as f16 numbers, exactly: with the sign bit turned over a code is c + 128, as the low byte under 0x64 that is 1024 + c + 128. FIRST, SECOND: which bytes
// of the word.
__device__ __forceinline__ uint32_t turn_codes(uint32_t word) { return word ^ 0x80808080u; }
template <int FIRST, int SECOND> __device__ __forceinline__ uint32_t widen_codes(uint32_t turned) {
    const uint32_t w = __byte_perm(turned, 0x64646464u, FIRST | 4 << 4 | SECOND << 8 | 4 << 12);
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0x64806480u));
    return r;
}

// A value's scale takes part in the row's base (the largest of score + log2 of the scale), by its exponent, so that weights times scales stay within f16's range whatever the
// scales are; one that is no number takes no part
__device__ __forceinline__ float exponent_of(float scale) {
    const int e = (int)(__float_as_uint(scale) >> 23 & 0xff);
    return __uint_as_float(0x4b000000u | (uint32_t)(e == 255 ? 127 : min(max(e, 127 - 80), 127 + 90))) - (8388608.0f + 127.0f);
}

// two fp32 numbers as a pair of 16-bit ones (the first in the low half), and what the pair leaves of them
template <int TYPE> __device__ __forceinline__ uint32_t pair_of(float a, float b) {
    uint32_t w;
    if (TYPE == RQ_KV_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    return w;
}
template <int TYPE> __device__ __forceinline__ uint32_t take_pair(float& a, float& b) {
    const uint32_t w = pair_of<TYPE>(a, b);
    a -= rqserve::to_float<TYPE>((uint16_t)w);
    b -= rqserve::to_float<TYPE>((uint16_t)(w >> 16));
    return w;
}

// Queries over an f16 cache: a row is multiplied by a power of two that brings its largest element to 2 or more (at best to 2^14 .. 2^15), so that its parts keep their 22
// bits whatever the row's size (an f16 number below 2^-14 loses bits, one above 65504 is none), and the scores' factor makes up for it. `largest`: the bits
// of that element without its sign; rows of zeros and below 2^-112 stay below, those that are not finite are none afterwards either.
__device__ __forceinline__ int raise_of(uint32_t largest) { return min(141 - (int)(largest >> 23), 126); }  // from -114
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// Over codes: a row's scores are sums of codes times its queries, raised, times a key's scale and scale_size * 2^exponent. So that no product in between is past fp32's range where
// the score is not, the power of two is taken in two parts, 2^first with the sum (a number of 1 to 2^45) before it meets the key's scale, the rest with scale_size after that: with
// 2^80 at most 2^125 meets a scale, and what the rest would raise stays below the score itself; from 2^-126 the sum stays a normal number.
struct PowerParts {
    float first, rest;
};
__device__ __forceinline__ PowerParts power_parts(float size, int exponent) {
    const int first = min(max(exponent, -126), 80);
    return {power_of_two(first), size * power_of_two(min(max(exponent - first, -126), 126))};
}
constexpr int kUsualRaise = 7;  // right for rows whose largest element is 2^-6 .. 2^9
// What scores are multiplied by to be exponents of two: positive and finite, so that masked scores stay -inf and scores of zero stay zero
__device__ __forceinline__ float factor_of(float scale, int raise) { return fminf(fmaxf(scale * power_of_two(-raise) * kLog2e, 1.2e-38f), 3e38f); }
#endif

}  // namespace rqattn
