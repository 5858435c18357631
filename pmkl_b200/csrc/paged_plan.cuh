// paged_plan.cuh -- pages, block table and slot map of a step's new tokens
// from the requests' lengths.
//
// Everything follows from two running sums over the requests: of the new
// tokens (where a request's tokens begin) and of the pages that they need
// (which of the free pages they get).  Every CTA forms both sums for itself,
// kThreads requests at a time with the totals carried along, so that no CTA
// waits for another and one launch does all of it; it then writes its share:
// the slots of its range of tokens, found by a search in the sums (held in
// shared memory), and the table rows and lengths of every gridDim-th request.
// A slot in a new page takes the page from the free list, not from the table
// row that another CTA may be writing.
#pragma once

#include "paged_common.cuh"

namespace pmkl_b200 {
namespace paged {

constexpr int kPlanThreads = 256;

struct PlanArgs {
    const int *cached, *fresh;  // lengths: in the cache, new
    int *table;
    long long table_stride;
    const int *free_blocks, *free_count;
    int free_capacity, batch, max_blocks, block;
    long long max_tokens, tokens_per_cta;
    int *seq_lens, *query_starts;
    long long *slots;
    int *free_out, *status;
};

// Inclusive sums over the block of two values, by warp shuffles.
__device__ __forceinline__ void block_scan2(long long &a, long long &b, long long (&wa)[kPlanThreads / 32],
                                            long long (&wb)[kPlanThreads / 32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) a += x, b += y;
    }
    __syncthreads();  // the sums of the round before have been read
    if (lane == 31) wa[warp] = a, wb[warp] = b;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w)
        if (w < warp) a += wa[w], b += wb[w];
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanArgs p) {
    __shared__ long long wa[kPlanThreads / 32], wb[kPlanThreads / 32];
    __shared__ long long s_end[kPlanThreads];    // tokens up to and with this request
    __shared__ long long s_taken[kPlanThreads];  // pages taken before this request
    __shared__ int s_cached[kPlanThreads], s_first[kPlanThreads];
    __shared__ bool s_ok[kPlanThreads];
    __shared__ long long s_total[2];
    const int tid = threadIdx.x;
    int count = *p.free_count;
    count = count < 0 ? 0 : (count > p.free_capacity ? p.free_capacity : count);
    const long long t_begin = blockIdx.x * p.tokens_per_cta;
    const long long t_end = min(p.max_tokens, t_begin + p.tokens_per_cta);
    long long tokens_before = 0, pages_before = 0, granted = 0;

    for (int r0 = 0; r0 < p.batch; r0 += kPlanThreads) {
        const int r = r0 + tid;
        const bool real = r < p.batch;
        const int c = real ? max(0, p.cached[r]) : 0, n = real ? max(0, p.fresh[r]) : 0;
        const long long total = static_cast<long long>(c) + n;
        const long long first = (static_cast<long long>(c) + p.block - 1) / p.block;
        const long long last = (total + p.block - 1) / p.block;
        // Two sums: tokens first, since whether a request's tokens fit decides
        // whether its pages count.
        long long end = n, unused = 0;
        block_scan2(end, unused, wa, wb);
        end += tokens_before;
        const bool past = end > p.max_tokens, wide = last > p.max_blocks;
        const long long need = (real && !past && !wide) ? last - first : 0;
        long long taken = need, got = 0;
        block_scan2(taken, got, wa, wb);
        taken += pages_before;
        const bool none_left = need > 0 && taken > count;
        const bool ok = real && !past && !wide && !none_left;
        __syncthreads();
        s_end[tid] = end;
        s_taken[tid] = taken - need;
        s_cached[tid] = c;
        s_first[tid] = static_cast<int>(first < p.max_blocks ? first : p.max_blocks);
        s_ok[tid] = ok;
        if (tid == kPlanThreads - 1) s_total[0] = end, s_total[1] = taken;
        // Granted pages: the sums of granted requests that need some are a
        // prefix, so the largest is what is gone.
        if (ok && need > 0 && taken > granted) granted = taken;
        if (real && r % gridDim.x == blockIdx.x) {
            p.seq_lens[r] = static_cast<int>(ok ? total : c);
            p.status[r] = past ? PMKL_PLAN_NO_TOKENS
                               : (wide ? PMKL_PLAN_NO_COLUMNS : (none_left ? PMKL_PLAN_NO_BLOCKS : PMKL_PLAN_OK));
            p.query_starts[r + 1] = static_cast<int>(end < 0x7FFFFFFFLL ? end : 0x7FFFFFFFLL);
            if (r == 0) p.query_starts[0] = 0;
        }
        __syncthreads();
        // Table rows of this CTA's requests, a warp each.
        const int here = min(kPlanThreads, p.batch - r0);
        const int skip = (static_cast<int>(blockIdx.x) - r0 % static_cast<int>(gridDim.x) + static_cast<int>(gridDim.x)) %
                         static_cast<int>(gridDim.x);
        for (long long i = skip + static_cast<long long>(tid >> 5) * gridDim.x; i < here;
             i += static_cast<long long>(kPlanThreads / 32) * gridDim.x) {
            if (!s_ok[i]) continue;
            const long long req_end = s_end[i], req_begin = i ? s_end[i - 1] : tokens_before;
            const long long f = s_first[i];
            const long long l = (s_cached[i] + (req_end - req_begin) + p.block - 1) / p.block;
            for (long long j = f + (tid & 31); j < l; j += 32)
                p.table[(r0 + i) * p.table_stride + j] = p.free_blocks[count - 1 - s_taken[i] - (j - f)];
        }
        // Slots of this CTA's tokens that belong to these requests.
        const long long lo = max(t_begin, tokens_before), hi = min(t_end, s_total[0]);
        for (long long t = lo + tid; t < hi; t += kPlanThreads) {
            int a = 0, b = here - 1;  // the first request whose end is past t
            while (a < b) {
                const int m = (a + b) >> 1;
                if (s_end[m] > t)
                    b = m;
                else
                    a = m + 1;
            }
            long long slot = -1;
            if (s_ok[a]) {
                const long long place = s_cached[a] + (t - (a ? s_end[a - 1] : tokens_before));
                const long long j = place / p.block;
                const int page = j < s_first[a] ? p.table[(r0 + a) * p.table_stride + j]
                                                : p.free_blocks[count - 1 - s_taken[a] - (j - s_first[a])];
                slot = static_cast<long long>(page) * p.block + (place - j * p.block);
            }
            p.slots[t] = slot;
        }
        tokens_before = s_total[0];
        pages_before = s_total[1];
        __syncthreads();  // the sums have been read
    }
    for (long long t = max(t_begin, tokens_before) + tid; t < t_end; t += kPlanThreads) p.slots[t] = -1;

    if (blockIdx.x == 0) {
        if (p.batch == 0 && tid == 0) p.query_starts[0] = 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) granted = max(granted, __shfl_xor_sync(0xffffffffu, granted, o));
        if ((tid & 31) == 0) wa[tid >> 5] = granted;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kPlanThreads / 32; ++w) granted = max(granted, wa[w]);
            *p.free_out = count - static_cast<int>(granted);
        }
    }
}

}  // namespace paged
}  // namespace pmkl_b200
