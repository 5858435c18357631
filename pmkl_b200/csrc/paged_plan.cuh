// paged_plan.cuh -- pages, block table and slot map of a step's new tokens
// from the requests' lengths.
//
// Everything follows from two running sums over the requests: of the new
// tokens (where a request's tokens begin) and of the pages that they need
// (which of the free pages they get).  Every CTA forms both sums for itself,
// one or four requests a thread at a time with the totals carried along, so that no CTA waits for another and one launch does all of it; it
// then writes its share: the slots of its range of tokens, found by a search in
// the sums (held in shared memory), and the table rows and lengths of every
// gridDim-th request.  A slot in a new page takes the page from the free list,
// not from the table row that another CTA may be writing.
//
// Bound by latency: a launch, two block sums and a search.  B200, device time:
// 4.0 us for 16 requests of one token, 6.8 us for 1024 requests and 66 Ki tokens
// (13.5 us with one request a thread in four rounds; four a thread cost the small
// case 1.3 us, hence both forms).
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

// Sum over the threads before this one; `total` gets the block's.
__device__ __forceinline__ long long block_before(long long v, long long (&w)[kPlanThreads / 32], long long &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // the sums of the round before have been read
    if (lane == 31) w[warp] = x;
    __syncthreads();
    x -= v;
    total = 0;
#pragma unroll
    for (int i = 0; i < kPlanThreads / 32; ++i) {
        if (i < warp) x += w[i];
        total += w[i];
    }
    return x;
}

// Pages of n rows (32-bit division: n is below 2^32).
__device__ __forceinline__ unsigned pages_of(unsigned n, unsigned block) { return n ? (n - 1) / block + 1 : 0; }

// EACH requests a thread: one up to kPlanThreads requests, four beyond.
template <int EACH>
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanArgs p) {
    constexpr int kPlanEach = EACH, kPlanRequests = kPlanThreads * EACH;
    __shared__ long long w_sum[kPlanThreads / 32];
    __shared__ long long s_end[kPlanRequests];  // tokens up to and with this request
    __shared__ int s_taken[kPlanRequests];      // pages taken before this request, -1: left out
    __shared__ unsigned s_cached[kPlanRequests], s_first[kPlanRequests];
    const int tid = threadIdx.x, grid = static_cast<int>(gridDim.x), cta = static_cast<int>(blockIdx.x);
    int count = *p.free_count;
    const long long t_begin = cta * p.tokens_per_cta;
    const long long t_end = min(p.max_tokens, t_begin + p.tokens_per_cta);
    long long tokens_before = 0, pages_before = 0, granted = 0;
    const unsigned block = static_cast<unsigned>(p.block);

    for (int r0 = 0; r0 < p.batch; r0 += kPlanRequests) {
        const int r1 = r0 + tid * kPlanEach;
        unsigned c[kPlanEach], n[kPlanEach];
        long long mine = 0, total_tokens, total_pages;
#pragma unroll
        for (int i = 0; i < kPlanEach; ++i) {
            const bool real = r1 + i < p.batch;
            c[i] = real ? max(0, p.cached[r1 + i]) : 0;
            n[i] = real ? max(0, p.fresh[r1 + i]) : 0;
            mine += n[i];
        }
        count = count < 0 ? 0 : (count > p.free_capacity ? p.free_capacity : count);
        // Tokens first, since whether a request's tokens fit decides whether its pages count.
        long long end = tokens_before + block_before(mine, w_sum, total_tokens);
        unsigned first[kPlanEach], need[kPlanEach];
        int why[kPlanEach];
        mine = 0;
#pragma unroll
        for (int i = 0; i < kPlanEach; ++i) {
            end += n[i];
            first[i] = pages_of(c[i], block);
            const unsigned last = pages_of(c[i] + n[i], block);
            // (a length past 31 bits fits no table either)
            const bool wide = last > static_cast<unsigned>(p.max_blocks) || c[i] + n[i] > 0x7FFFFFFFu;
            why[i] = end > p.max_tokens ? PMKL_PLAN_NO_TOKENS : (wide ? PMKL_PLAN_NO_COLUMNS : PMKL_PLAN_OK);
            need[i] = why[i] == PMKL_PLAN_OK ? last - first[i] : 0;
            mine += need[i];
            s_end[r1 - r0 + i] = end;
            s_cached[r1 - r0 + i] = c[i];
            s_first[r1 - r0 + i] = first[i];
            if (r1 + i < p.batch && (r1 + i) % grid == cta) {
                p.query_starts[r1 + i + 1] = static_cast<int>(min(end, 0x7FFFFFFFLL));
                if (r1 + i == 0) p.query_starts[0] = 0;
            }
        }
        long long taken = pages_before + block_before(mine, w_sum, total_pages);
#pragma unroll
        for (int i = 0; i < kPlanEach; ++i) {
            taken += need[i];
            if (need[i] > 0 && taken > count) why[i] = PMKL_PLAN_NO_BLOCKS;
            const bool ok = why[i] == PMKL_PLAN_OK;
            // The sums of the requests that get pages are a prefix, so the largest is what is gone.
            if (ok && need[i] > 0) granted = max(granted, taken);
            s_taken[r1 - r0 + i] = ok ? static_cast<int>(min(taken, static_cast<long long>(count)) - need[i]) : -1;
            if (ok && need[i] == 0) s_taken[r1 - r0 + i] = 0;
            if (r1 + i < p.batch && (r1 + i) % grid == cta) {
                p.seq_lens[r1 + i] = static_cast<int>(ok ? c[i] + n[i] : c[i]);
                p.status[r1 + i] = why[i];
            }
        }
        __syncthreads();
        // Table rows of this CTA's requests, a warp each.
        const int here = min(kPlanRequests, p.batch - r0);
        const int skip = (cta - r0 % grid + grid) % grid;
        for (long long i = skip + static_cast<long long>(tid >> 5) * grid; i < here;
             i += static_cast<long long>(kPlanThreads / 32) * grid) {
            if (s_taken[i] < 0) continue;
            const long long begin = i ? s_end[i - 1] : tokens_before;
            const unsigned f = s_first[i], l = pages_of(s_cached[i] + static_cast<unsigned>(s_end[i] - begin), block);
            for (unsigned j = f + (tid & 31); j < l; j += 32)
                p.table[(r0 + i) * p.table_stride + j] = p.free_blocks[count - 1 - s_taken[i] - static_cast<int>(j - f)];
        }
        // Slots of this CTA's tokens that belong to these requests.
        const long long lo = max(t_begin, tokens_before), hi = min(t_end, tokens_before + total_tokens);
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
            if (s_taken[a] >= 0) {
                const unsigned place = s_cached[a] + static_cast<unsigned>(t - (a ? s_end[a - 1] : tokens_before));
                const unsigned j = place / block;
                const int page = j < s_first[a] ? p.table[(r0 + a) * p.table_stride + j]
                                                : p.free_blocks[count - 1 - s_taken[a] - static_cast<int>(j - s_first[a])];
                slot = static_cast<long long>(page) * p.block + (place - j * block);
            }
            p.slots[t] = slot;
        }
        tokens_before += total_tokens;
        pages_before += total_pages;
        __syncthreads();  // the sums have been read
    }
    for (long long t = max(t_begin, tokens_before) + tid; t < t_end; t += kPlanThreads) p.slots[t] = -1;

    if (cta == 0) {
        if (p.batch == 0) {
            if (tid == 0) p.query_starts[0] = 0;
            count = count < 0 ? 0 : (count > p.free_capacity ? p.free_capacity : count);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) granted = max(granted, __shfl_xor_sync(0xffffffffu, granted, o));
        if ((tid & 31) == 0) w_sum[tid >> 5] = granted;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kPlanThreads / 32; ++w) granted = max(granted, w_sum[w]);
            *p.free_out = count - static_cast<int>(granted);
        }
    }
}

}  // namespace paged
}  // namespace pmkl_b200
