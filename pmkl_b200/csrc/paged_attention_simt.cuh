// paged_attention_simt.cuh -- attention over the paged 8-bit cache on the CUDA
// cores: any dtype, head size 1..256, any block size.
//
// One CTA per query row and head; its warps take 32-key tiles in turn, each
// with a running maximum and sum of its own (lane j scores key j of the tile,
// each lane sums every 32nd output column), and join at the end through
// shared memory.  fp32 throughout.  The general path: head sizes other than
// 64 and 128, pages whose rows are no multiple of 16.
#pragma once

#include "paged_common.cuh"

namespace pmkl_b200 {
namespace paged {

struct AttnArgs {
    const void *q;
    void *o;
    long long q_st[2], o_st[2];  // (token, head)
    CacheView k, v;
    const int *table;
    long long table_stride;
    const int *seq_lens, *query_starts;
    float *lse;
    int tokens, batch, H, Hkv, D, num_blocks, block, max_blocks, causal;
    int max_q;  // rows of a request that launches are sized for; a request may have more
    float scale;
};

// Rows and keys of request b, kept within the tensors whatever the device
// arrays hold.
struct Request {
    int first, rows, keys;  // first row of q, rows, rows in the cache
    int shift;              // row i sees keys j <= i + shift
};

__host__ __device__ __forceinline__ Request request_of(const AttnArgs &p, int b) {
    Request r;
    int begin = b, end = b + 1;
    if (p.query_starts) {
        begin = min(max(p.query_starts[b], 0), p.tokens);
        end = min(max(p.query_starts[b + 1], begin), p.tokens);
    }
    // Room above, so that key positions rounded up to a tile stay 32-bit.
    const long long cap = min(static_cast<long long>(p.max_blocks) * p.block, 0x7FFFFFFFLL - 4096);
    const int len = max(0, p.seq_lens[b]);
    r.first = begin;
    r.rows = end - begin;
    r.keys = static_cast<int>(len < cap ? len : cap);
    r.shift = r.keys - r.rows;
    return r;
}

// Keys that row i of the request sees.
__host__ __device__ __forceinline__ int visible(const AttnArgs &p, const Request &r, int i) {
    return p.causal ? min(r.keys, max(0, i + r.shift + 1)) : r.keys;
}

// Rows of q that belong to no request, before the first and behind the last: o =
// 0, lse = -inf.  Called by the whole grid (128 threads and more a CTA).
template <typename T>
__device__ __forceinline__ void clear_unused(const AttnArgs &p) {
    if (!p.query_starts) return;
    const int first = min(max(p.query_starts[0], 0), p.tokens);
    const int used = min(max(p.query_starts[p.batch], first), p.tokens);
    const long long n = static_cast<long long>(first + p.tokens - used) * p.H;
    for (long long i = blockIdx.x; i < n; i += gridDim.x) {
        const long long h = i % p.H;
        long long t = i / p.H;
        if (t >= first) t += used - first;
        T *o = static_cast<T *>(p.o) + t * p.o_st[0] + h * p.o_st[1];
        for (int d = threadIdx.x; d < p.D; d += blockDim.x) o[d] = Elem<T>::from_float(0.f);
        if (p.lse && threadIdx.x == 0) p.lse[t * p.H + h] = -INFINITY;
    }
}

// The scale of a page of values within its documented range.
__device__ __forceinline__ float value_scale(float s) {
    return fminf(fmaxf(s, 5.421010862427522e-20f), 1.8446744073709552e19f);  // 2^-64, 2^64
}

// The scale of a page of keys: no smaller than what paged_append writes, so that
// its product with a row's factor is not 0 (below).
__device__ __forceinline__ float key_scale(float s) {
    return s < 5.421010862427522e-20f ? 5.421010862427522e-20f : s;  // 2^-64; NaN stays
}

// Query rows are held in fp16 over a power of two 2^e, and a score is the raw
// product times the row's factor (2^e * c, c the score scale in log2 units) and
// the page's key scale.  Returns the e that brings the row's largest value to
// 2^7 .. 2^8, or, for rows so small (0 among them) that the factor would fall below 2^-85, the e
// that keeps it there: times a key scale it is then never 0 in fp32, and -inf
// in masked places stays -inf.  Such a row loses 2^-25 * 2^-85 of its values,
// 2^-30 in a score over the largest keys.
__device__ __forceinline__ int query_exponent(float amax, float c) {
    const int least = max(-100, 127 - 85 - static_cast<int>(__float_as_uint(c) >> 23));
    return min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127 - 7, least), 126);
}

// The rare path of the kernels whose products would spread a NaN value as 0 *
// NaN: sets in `cols` (a bit a column) the columns that hold NaN in the rows
// [key, end) of request row `table`, K/V head h.
__device__ __forceinline__ void mark_nan(const AttnArgs &p, const int *table, int h, int key, int end, uint32_t *cols) {
#pragma unroll 1
    for (; key < end; ++key) {
        const int col = key / p.block, page = table[col];
        if (page < 0 || page >= p.num_blocks) continue;
        const uint8_t *v = p.v.base + page * p.v.s[0] + h * p.v.s[1] + (key - col * p.block) * p.v.s[2];
#pragma unroll 1
        for (int d = 0; d < p.D; ++d)
            if ((v[d] & 0x7F) == 0x7F) atomicOr(&cols[d >> 5], 1u << (d & 31));
    }
}

// Bit 7 of each byte that is an e4m3 NaN (0x7F with either sign).
__device__ __forceinline__ uint32_t nan_bits(uint32_t four) {
    return ((four & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}
__device__ __forceinline__ uint32_t without_nan(uint32_t four) {
    const uint32_t n = nan_bits(four);
    return four & ~(n | (n - (n >> 7)));
}

constexpr int kSimtThreads = 128;
constexpr int kSimtCols = 8;  // output columns a lane, head size up to 256

template <typename T>
__global__ void __launch_bounds__(kSimtThreads) paged_attention_simt_kernel(const AttnArgs p) {
    constexpr int kWarps = kSimtThreads / 32;
    __shared__ float qs[256];
    __shared__ float part[kWarps][256];
    __shared__ float ms[kWarps], ls[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    clear_unused<T>(p);
    const long long units = static_cast<long long>(p.batch) * p.max_q * p.H;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
        const int h = static_cast<int>(u % p.H);
        const long long bi = u / p.H;
        const int b = static_cast<int>(bi / p.max_q);
        const Request r = request_of(p, b);
        const int hk = h / (p.H / p.Hkv);
        for (long long row = bi % p.max_q; row < r.rows; row += p.max_q) {
            const int i = static_cast<int>(row);
            const int keys = visible(p, r, i);
            const T *q = static_cast<const T *>(p.q) + (r.first + i) * p.q_st[0] + h * p.q_st[1];
            __syncthreads();  // the row before has been read
            for (int d = threadIdx.x; d < p.D; d += kSimtThreads) qs[d] = Elem<T>::to_float(q[d]) * p.scale;
            __syncthreads();
            float m = -INFINITY, l = 0.f, acc[kSimtCols] = {};
            for (long long j0 = warp * 32; j0 < keys; j0 += kWarps * 32) {
                const long long j = j0 + lane;
                float s = -INFINITY, vs = 0.f;
                long long vrow = 0;
                bool there = j < keys;
                if (there) {
                    const int page = p.table[b * p.table_stride + j / p.block];
                    there = page >= 0 && page < p.num_blocks;
                    if (there) {
                        const long long at_row = j % p.block;
                        const uint8_t *k = p.k.base + page * p.k.s[0] + hk * p.k.s[1] + at_row * p.k.s[2];
                        float dot = 0.f;
                        for (int d = 0; d < p.D; ++d) dot = fmaf(qs[d], e4m3_to_float(k[d]), dot);
                        const long long at = static_cast<long long>(page) * p.Hkv + hk;
                        s = dot * key_scale(p.k.scale[at]);
                        vs = value_scale(p.v.scale[at]);
                        vrow = page * p.v.s[0] + hk * p.v.s[1] + at_row * p.v.s[2];
                    }
                }
                float top = s;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                top = fmaxf(top, m);
                const float base = top == -INFINITY ? 0.f : top;
                const float fix = expf(m - base);
                const float e = there ? expf(s - base) : 0.f;
                float sum = e;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                m = top;
                l = l * fix + sum;
#pragma unroll
                for (int c = 0; c < kSimtCols; ++c) acc[c] *= fix;
                const float w = e * vs;
                const unsigned int mine = __ballot_sync(0xffffffffu, there);
                for (int x = 0; x < 32; ++x) {
                    const float wx = __shfl_sync(0xffffffffu, w, x);
                    const long long at = __shfl_sync(0xffffffffu, vrow, x);
                    if (!((mine >> x) & 1u)) continue;  // a row that is not there may hold anything
#pragma unroll
                    for (int c = 0; c < kSimtCols; ++c) {
                        const int d = c * 32 + lane;
                        if (d < p.D) acc[c] = fmaf(wx, e4m3_to_float(p.v.base[at + d]), acc[c]);
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < kSimtCols; ++c) part[warp][c * 32 + lane] = acc[c];
            if (lane == 0) ms[warp] = m, ls[warp] = l;
            __syncthreads();
            float top = ms[0];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) top = fmaxf(top, ms[w]);
            const float base = top == -INFINITY ? 0.f : top;
            float sum = 0.f, f[kWarps];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                f[w] = expf(ms[w] - base);
                sum += f[w] * ls[w];
            }
            // A sum of 0 is a row without keys; a NaN goes through to the output.
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            T *o = static_cast<T *>(p.o) + (r.first + i) * p.o_st[0] + h * p.o_st[1];
            for (int d = threadIdx.x; d < p.D; d += kSimtThreads) {
                float x = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) x = fmaf(f[w], part[w][d], x);
                o[d] = Elem<T>::from_float(x * inv);
            }
            if (p.lse && threadIdx.x == 0)
                p.lse[static_cast<long long>(r.first + i) * p.H + h] = sum == 0.f ? -INFINITY : base + logf(sum);
        }
    }
}

}  // namespace paged
}  // namespace pmkl_b200
