// The plan of a serving step: page tables, slot map and token positions from the requests' lengths, in one launch.
//
// Whole numbers only: with held_r = ceil(cached_r / page), need_r = ceil((cached_r + fresh_r) / page) - held_r and B_r, S_r the sums of need and
// fresh over the requests before r, the page of request r's column c >= held_r is free_pages[B_r + c - held_r], and token t belongs
// to the last r with S_r <= t. What bounds it is one launch and its chain of dependent loads (lengths, free pages): every CTA adds up all
// requests' lengths for itself (at most 4096, 32 bytes a thread and round) rather than wait for another launch to have done so.
#include "rq_serve.cuh"

using namespace rqserve;

namespace {

constexpr int kThreads = 256;

struct PlanParams {
    const int32_t *cached, *fresh, *free_pages;
    int32_t *block_table, *starts, *lengths, *slots, *positions, *owners, *status;
    int64_t table_stride;
    int requests, table_width, free_count, max_tokens, page_shift;
};

constexpr int64_t kMost = 0x7fffffff;

// Inclusive sum over the CTA's threads of two numbers at once
__device__ __forceinline__ longlong2 block_sums(longlong2 v, longlong2* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int64_t a = __shfl_up_sync(0xffffffffu, v.x, off), b = __shfl_up_sync(0xffffffffu, v.y, off);
        if (lane >= off) { v.x += a; v.y += b; }
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    for (int w = 0; w < warp; ++w) { v.x += warp_sums[w].x; v.y += warp_sums[w].y; }
    __syncthreads();
    return v;
}

__global__ void __launch_bounds__(kThreads) rq_batch_plan_kernel(PlanParams p) {
    extern __shared__ int32_t table[];  // starts [requests + 1] | pages before [requests + 1] | cached [requests]
    __shared__ longlong2 warp_sums[kThreads / 32];
    __shared__ unsigned long long lacking;
    launch_dependents();
    int32_t *starts = table, *before = table + p.requests + 1, *cached = before + p.requests + 1;
    const int page = 1 << p.page_shift, tid = threadIdx.x;
    // (of up to 2^31 - 1 positions: an unsigned sum does not wrap)
    auto pages_of = [&](int positions) { return (int)(((uint32_t)positions + (uint32_t)(page - 1)) >> p.page_shift); };
    wait_for_previous();
    longlong2 carry = make_longlong2(0, 0);  // sums in 64 bits, kept up to 2^31 - 1: whatever the lengths are, starts ascend and every index below lies inside its array
    int64_t too_wide = 0;
    if (tid == 0) { starts[0] = 0; before[0] = 0; lacking = 0; }
    for (int r0 = 0; r0 < p.requests; r0 += kThreads) {
        const int r = r0 + tid;
        int have = 0, more = 0, need = 0;
        if (r < p.requests) {
            have = max(p.cached[r], 0);
            more = max(p.fresh[r], 0);
            const int64_t all = ((int64_t)have + more + page - 1) >> p.page_shift;
            const int held = pages_of(have);
            need = max((int)min(all, (int64_t)p.table_width) - held, 0);
            too_wide += all - held - need;
            cached[r] = have;
            if (blockIdx.x == 0) p.lengths[r] = (int)min((int64_t)have + more, kMost);
        }
        longlong2 sum = block_sums(make_longlong2(more, need), warp_sums);
        sum.x = min(sum.x + carry.x, (long long)kMost);
        sum.y = min(sum.y + carry.y, (long long)kMost);
        if (r < p.requests) {
            starts[r + 1] = (int)sum.x;
            before[r + 1] = (int)sum.y;
            if (blockIdx.x == 0) p.starts[r + 1] = (int)sum.x;
        }
        __syncthreads();
        const int last = min(r0 + kThreads, p.requests);
        carry = make_longlong2(starts[last], before[last]);
    }
    const int tokens = (int)carry.x, pages = (int)carry.y;
    if (blockIdx.x == 0) {
        if (too_wide) atomicAdd(&lacking, (unsigned long long)too_wide);  // whole numbers: any order gives the same
        __syncthreads();
        if (tid == 0) {
            p.starts[0] = 0;
            p.status[0] = tokens;
            p.status[1] = min(pages, p.free_count);
            p.status[2] = (int)min((int64_t)max(pages - p.free_count, 0) + (int64_t)lacking, kMost);
        }
    }
    const int64_t first = (int64_t)blockIdx.x * kThreads + tid, step = (int64_t)gridDim.x * kThreads;
    for (int64_t n = first; n < pages; n += step) {
        const int i = (int)n, r = owner_of(before, p.requests, i);
        const int column = pages_of(cached[r]) + i - before[r];
        p.block_table[(int64_t)r * p.table_stride + column] = i < p.free_count ? p.free_pages[i] : -1;
    }
    for (int64_t t = first; t < p.max_tokens; t += step) {
        int slot = -1, position = 0, owner = -1;
        if (t < tokens) {
            owner = owner_of(starts, p.requests, (int)t);
            const int64_t at = (int64_t)cached[owner] + t - starts[owner];
            position = (int)min(at, kMost);
            const int column = position >> p.page_shift, held = pages_of(cached[owner]);
            int entry = -1;
            if (at <= kMost && column < p.table_width) {
                const int64_t i = (int64_t)before[owner] + column - held;  // a new page: from the list, its entry may not be written yet
                entry = column < held ? p.block_table[(int64_t)owner * p.table_stride + column] : (i < p.free_count ? p.free_pages[i] : -1);
            }
            // (an entry that names no page of any cache must not come out as a position of another one's)
            const int64_t place = ((int64_t)entry << p.page_shift) + (position & (page - 1));
            if (entry >= 0 && place <= kMost) slot = (int)place;
        }
        p.slots[t] = slot;
        p.positions[t] = position;
        p.owners[t] = owner;
    }
}

}  // namespace

int rqserve::check_cache(const char* who, const rq_kv_cache* c) {
    if (!c || !c->k || !c->v) return rq_fail(RQ_ERR_INVALID, "%s: null cache", who);
    if (c->type != RQ_KV_F16 && c->type != RQ_KV_BF16 && c->type != RQ_KV_INT8) return rq_fail(RQ_ERR_INVALID, "%s: cache type %d is none of F16(0), BF16(1) and INT8(2)", who, c->type);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return rq_fail(RQ_ERR_UNSUPPORTED, "%s: head_dim=%d is not 64, 128 or 256", who, c->head_dim);
    if (c->heads <= 0 || c->pages <= 0) return rq_fail(RQ_ERR_INVALID, "%s: the cache's heads and pages must be positive", who);
    if (c->page_size <= 0 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)))
        return rq_fail(RQ_ERR_INVALID, "%s: page_size=%d is not a power of two up to 4096", who, c->page_size);
    if (c->pages >= ((int64_t)1 << 31) / c->page_size) return rq_fail(RQ_ERR_LIMIT, "%s: %lld pages of %d positions are 2^31 positions or more", who, (long long)c->pages, c->page_size);
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return rq_fail(RQ_ERR_INVALID, "%s: the cache's pointers must be 16-byte aligned", who);
    if (c->page_stride < 0 || c->head_stride < 0 || c->line_stride < 0 || (c->page_stride | c->head_stride | c->line_stride) & 7)
        return rq_fail(RQ_ERR_INVALID, "%s: the cache's strides must be non-negative multiples of 8 elements", who);
    if (c->type == RQ_KV_INT8) {
        if (!c->k_scale || !c->v_scale || (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3)) return rq_fail(RQ_ERR_INVALID, "%s: an INT8 cache needs 4-byte aligned k_scale and v_scale", who);
        if ((c->page_stride | c->head_stride | c->line_stride) & 15) return rq_fail(RQ_ERR_INVALID, "%s: an INT8 cache's strides must be multiples of 16 elements", who);
        if (c->scale_page_stride < 0 || c->scale_head_stride < 0 || c->scale_line_stride < 0 || c->scale_page_stride >= (int64_t)1 << 31 || c->scale_line_stride >= (int64_t)1 << 31)
            return rq_fail(RQ_ERR_LIMIT, "%s: the scales' strides must not be negative, those of pages and lines below 2^31", who);
    }
    if (c->page_stride >= (int64_t)1 << 31 || c->line_stride >= (int64_t)1 << 31) return rq_fail(RQ_ERR_LIMIT, "%s: the cache's page and line strides must be below 2^31 elements", who);
    return RQ_OK;
}

extern "C" int rq_batch_plan(rq_ctx* ctx, const int32_t* cached, const int32_t* fresh, int requests, int page_size, int32_t* block_table, int64_t table_stride,
                             int table_width, const int32_t* free_pages, int free_count, int32_t* starts, int32_t* lengths, int32_t* slots, int32_t* positions,
                             int32_t* owners, int max_tokens, int32_t* status, void* stream) {
    if (!ctx || !cached || !fresh || !block_table || !starts || !lengths || !slots || !positions || !owners || !status || (!free_pages && free_count > 0))
        return rq_fail(RQ_ERR_INVALID, "rq_batch_plan: null argument");
    if (requests <= 0 || table_width <= 0 || table_stride < table_width || free_count < 0 || max_tokens <= 0)
        return rq_fail(RQ_ERR_INVALID, "rq_batch_plan: requests, table_width and max_tokens must be positive, free_count not negative and table_stride at least table_width");
    if (page_size <= 0 || page_size > 4096 || (page_size & (page_size - 1))) return rq_fail(RQ_ERR_INVALID, "rq_batch_plan: page_size=%d is not a power of two up to 4096", page_size);
    if (requests > RQ_MAX_REQUESTS) return rq_fail(RQ_ERR_LIMIT, "rq_batch_plan: %d requests; at most %d", requests, RQ_MAX_REQUESTS);
    DeviceGuard guard(ctx->device);
    PlanParams p = {cached, fresh, free_pages, block_table, starts, lengths, slots, positions, owners, status, table_stride, requests, table_width, free_count, max_tokens, 0};
    while (1 << p.page_shift < page_size) ++p.page_shift;
    const int64_t ctas = ((int64_t)max_tokens + kThreads - 1) / kThreads;
    const unsigned grid = (unsigned)(ctas < ctx->sm_count ? ctas : ctx->sm_count);
    const size_t smem = sizeof(int32_t) * (3 * (size_t)requests + 2);
    // (48 KB without asking are for it and the kernel's static shared memory together)
    if (smem > 47 * 1024) RQ_CUDA(cudaFuncSetAttribute(rq_batch_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    return launch(rq_batch_plan_kernel, dim3(grid), kThreads, smem, (cudaStream_t)stream, p);
}
