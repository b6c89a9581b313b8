// Shared by the kernels of a serving step (plan, rotation and cache, attention, the next token): launches, the cache's checks,
// 16-bit conversions and where a batch's requests begin.
#pragma once
#include <cuda_bf16.h>

#include "rq_internal.cuh"

namespace rqserve {

// The cache's description as a caller hands it over: RQ_OK, or the status and text of what is wrong with it.
int check_cache(const char* who, const rq_kv_cache* c);

// A launch that may begin before the kernel in front of it has ended: every kernel here waits (griddepcontrol.wait) in all threads
// before it touches global memory.
template <typename... Params, typename... Args>
int launch(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    RQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    return RQ_OK;
}

#ifdef __CUDACC__
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <int TYPE> __device__ __forceinline__ float to_float(uint16_t v) { return TYPE == RQ_KV_F16 ? __half2float(__ushort_as_half(v)) : __uint_as_float((uint32_t)v << 16); }
template <int TYPE> __device__ __forceinline__ uint16_t from_float(float v) { return TYPE == RQ_KV_F16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v)); }

// The last index r of the ascending table starts[0 .. n] with starts[r] <= t (t >= starts[0])
__device__ __forceinline__ int owner_of(const int32_t* starts, int n, int t) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (starts[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
#endif

}  // namespace rqserve
