// paged_append.cuh -- new keys and values into the paged cache, as 8-bit
// floats with one power-of-two scale a page and head.
//
// A run of tokens that fill neighbouring rows of one page shares one scale,
// which needs the largest value of the whole run (and the page's scale, where
// the page holds rows already) before the first value is rounded.  One warp
// takes one run of one head, of keys or of values: it finds the run's length,
// then its largest value, then the scale, rounds the page's older rows again
// where the scale grew, and writes the new ones.
#pragma once

#include "paged_common.cuh"

namespace pmkl_b200 {
namespace paged {

constexpr int kAppendThreads = 128;

struct AppendArgs {
    const void *x[2];        // new keys, new values
    long long x_st[2][2];    // their (token, head) strides
    CacheView cache[2];
    const long long *slots;
    int tokens, kv_heads, hidden, block;
    long long num_slots;
};

// The finite magnitude of x; 0 where it has none.
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.f;
}

template <typename T>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendArgs p) {
    const int lane = threadIdx.x & 31;
    const long long units = static_cast<long long>(p.tokens) * p.kv_heads * 2;
    const long long warps = static_cast<long long>(gridDim.x) * (kAppendThreads / 32);
    for (long long u = static_cast<long long>(blockIdx.x) * (kAppendThreads / 32) + (threadIdx.x >> 5); u < units;
         u += warps) {
        const int t = static_cast<int>(u / (p.kv_heads * 2)), hv = static_cast<int>(u % (p.kv_heads * 2));
        const int h = hv >> 1, side = hv & 1;
        const long long slot = p.slots[t];
        if (slot < 0 || slot >= p.num_slots) continue;
        const long long page = slot / p.block;
        const int row = static_cast<int>(slot - page * p.block);
        if (row > 0 && t > 0 && p.slots[t - 1] == slot - 1) continue;  // inside a run
        int n = 1;
        while (row + n < p.block && t + n < p.tokens && p.slots[t + n] == slot + n) ++n;

        const T *x = static_cast<const T *>(p.x[side]) + t * p.x_st[side][0] + h * p.x_st[side][1];
        const long long x_row = p.x_st[side][0];
        const CacheView &c = p.cache[side];
        uint8_t *dst = c.base + page * c.s[0] + h * c.s[1];
        float *scale = c.scale + page * p.kv_heads + h;

        float amax = 0.f;
        for (int i = 0; i < n; ++i)
            for (int d = lane; d < p.hidden; d += 32) amax = fmaxf(amax, finite_abs(Elem<T>::to_float(x[i * x_row + d])));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        float s = exp2_int(scale_exponent(amax));
        if (row > 0) {
            const float held = *scale;
            if (held >= s) {
                s = held;
            } else {
                const float ratio = held / s;
                for (int i = 0; i < row; ++i)
                    for (int d = lane; d < p.hidden; d += 32) {
                        uint8_t *at = dst + i * c.s[2] + d;
                        *at = float_to_e4m3(e4m3_to_float(*at) * ratio);
                    }
            }
        }
        __syncwarp();
        if (lane == 0) *scale = s;
        const float inv = 1.f / s;
        for (int i = 0; i < n; ++i)
            for (int d = lane; d < p.hidden; d += 32)
                dst[(row + i) * c.s[2] + d] = float_to_e4m3(Elem<T>::to_float(x[i * x_row + d]) * inv);
    }
}

// The same for rows of 16-byte vectors, kept in registers between the search
// for the largest value and the rounding, so that each value is read once.
//
// A CTA takes `span` neighbouring tokens of one head.  It lists the runs that
// begin there (a run may end in the next span), and its warps take them, keys
// and values apart, WPU warps a run: as many as it takes to hold a page's rows
// (16 bytes a lane and vector, NV vectors a lane); where a page is larger, the
// rows beyond are read again, from L2.  CTAs of neighbouring heads run side by
// side, so that a token's whole row is read at about one time.
//
// Bound by HBM: 16 x 4096 tokens, 32 heads of 128, bf16 (1.61 GB): 288 us on a
// B200, 5.59 TB/s, 0.85 of the measured copy bandwidth (435 us with the maxima
// taken element by element).  8 ragged chunks, 16 heads of 64, fp16 (22 MB): 8.0
// us; one token for each of 16 requests: 3.3 us, a launch and three dependent loads.
constexpr int kSpanMax = 32;

// The largest magnitude of 16-byte vectors, kept as the elements are: fp32, or
// two 16-bit maxima side by side (one instruction for two elements).  NaN is
// passed over; an infinity stays, and the caller then looks again by element.
template <typename T>
struct Largest;
template <>
struct Largest<float> {
    float m = 0.f;
    __device__ __forceinline__ void add(const uint4 &u) {
        m = fmaxf(fmaxf(fmaxf(m, fabsf(__uint_as_float(u.x))), fabsf(__uint_as_float(u.y))),
                  fmaxf(fabsf(__uint_as_float(u.z)), fabsf(__uint_as_float(u.w))));
    }
    __device__ __forceinline__ float get() const { return m; }
};
template <>
struct Largest<__half> {
    __half2 m = __float2half2_rn(0.f);
    __device__ __forceinline__ static __half2 mag(uint32_t w) {
        w &= 0x7FFF7FFFu;
        return *reinterpret_cast<const __half2 *>(&w);
    }
    __device__ __forceinline__ void add(const uint4 &u) {
        m = __hmax2(__hmax2(m, __hmax2(mag(u.x), mag(u.y))), __hmax2(mag(u.z), mag(u.w)));
    }
    __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};
template <>
struct Largest<__nv_bfloat16> {
    __nv_bfloat162 m = __float2bfloat162_rn(0.f);
    __device__ __forceinline__ static __nv_bfloat162 mag(uint32_t w) {
        w &= 0x7FFF7FFFu;
        return *reinterpret_cast<const __nv_bfloat162 *>(&w);
    }
    __device__ __forceinline__ void add(const uint4 &u) {
        m = __hmax2(__hmax2(m, __hmax2(mag(u.x), mag(u.y))), __hmax2(mag(u.z), mag(u.w)));
    }
    __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};

// The largest finite magnitude of a vector, element by element.
template <typename T>
__device__ __forceinline__ float vec_amax(const uint4 &u) {
    const T *e = reinterpret_cast<const T *>(&u);
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 16 / static_cast<int>(sizeof(T)); ++i) a = fmaxf(a, finite_abs(Elem<T>::to_float(e[i])));
    return a;
}

// The two elements of a word as fp32.
template <typename T>
__device__ __forceinline__ float2 word_floats(uint32_t w);
template <>
__device__ __forceinline__ float2 word_floats<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <>
__device__ __forceinline__ float2 word_floats<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

// A vector's elements times `inv` as 8-bit floats.
template <typename T>
__device__ __forceinline__ void vec_store(uint8_t *dst, const uint4 &u, float inv) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<uint32_t *>(dst) = pack_e4m3(__uint_as_float(u.x) * inv, __uint_as_float(u.y) * inv,
                                                       __uint_as_float(u.z) * inv, __uint_as_float(u.w) * inv);
    } else {
        const float2 a = word_floats<T>(u.x), b = word_floats<T>(u.y), c = word_floats<T>(u.z), d = word_floats<T>(u.w);
        *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_e4m3(a.x * inv, a.y * inv, b.x * inv, b.y * inv),
                                                     pack_e4m3(c.x * inv, c.y * inv, d.x * inv, d.y * inv));
    }
}

template <typename T, int WPU, int NV>
__global__ void __launch_bounds__(kAppendThreads) paged_append_vec_kernel(const AppendArgs p, int span) {
    constexpr int kWarps = kAppendThreads / 32, kUnits = kWarps / WPU, kElems = 16 / sizeof(T);
    __shared__ int s_lead[kSpanMax];
    __shared__ int s_count;
    __shared__ float s_max[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int h = blockIdx.x % p.kv_heads;
    const int t0 = blockIdx.x / p.kv_heads * span;
    if (warp == 0) {
        const int t = t0 + lane;
        bool lead = false;
        if (lane < span && t < p.tokens) {
            const long long slot = p.slots[t];
            lead = slot >= 0 && slot < p.num_slots && (t == 0 || slot % p.block == 0 || p.slots[t - 1] != slot - 1);
        }
        const unsigned int leads = __ballot_sync(0xffffffffu, lead);
        if (lead) s_lead[__popc(leads & ((1u << lane) - 1))] = t;
        if (lane == 0) s_count = __popc(leads);
    }
    __syncthreads();
    const int units = s_count * 2;
    // Lanes: one vector of a row each, as many rows at a time as fit the unit's lanes.
    const int per_row = p.hidden / kElems, rows_w = 32 / per_row;
    const int my_row = lane / per_row, col = (lane - my_row * per_row) * kElems;
    const bool active = my_row < rows_w;
    const int sub = warp % WPU, row_first = sub * rows_w + my_row, row_step = rows_w * WPU;
    for (int u0 = 0; u0 < units; u0 += kUnits) {
        const int u = u0 + warp / WPU;
        const bool real = u < units;
        const int t = real ? s_lead[u >> 1] : t0, side = u & 1;
        const long long slot = real ? p.slots[t] : 0;
        const long long page = slot / p.block;
        const int row = static_cast<int>(slot - page * p.block);
        const CacheView &c = p.cache[side];
        float *scale = c.scale + page * p.kv_heads + h;
        float held = 0.f;
        if (real && row > 0) held = *scale;
        int n = real ? 1 : 0;
        if (real) {
            const int most = min(p.block - row, p.tokens - t);
            for (bool all = true; all && n < most; ) {
                const int i = n + lane;
                const bool in = i < most && p.slots[t + i] == slot + i;
                const unsigned int out = __ballot_sync(0xffffffffu, !in);
                n += out ? __ffs(out) - 1 : 32;
                all = out == 0;
            }
        }
        const T *x = static_cast<const T *>(p.x[side]) + t * p.x_st[side][0] + h * p.x_st[side][1] + col;
        const long long x_row = p.x_st[side][0];
        uint8_t *dst = c.base + page * c.s[0] + h * c.s[1] + col;

        uint4 v[NV];
        Largest<T> largest;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int i = row_first + k * row_step;
            v[k] = make_uint4(0, 0, 0, 0);
            if (active && i < n) v[k] = *reinterpret_cast<const uint4 *>(x + i * x_row);
        }
        for (int i = row_first + NV * row_step; active && i < n; i += row_step)
            largest.add(*reinterpret_cast<const uint4 *>(x + i * x_row));
#pragma unroll
        for (int k = 0; k < NV; ++k) largest.add(v[k]);
        float amax = largest.get();
        if (__any_sync(0xffffffffu, !(amax <= 3.402823466e38f))) {
            // Infinities: the finite elements alone count.
            amax = 0.f;
#pragma unroll 1
            for (int i = row_first; active && i < n; i += row_step)
                amax = fmaxf(amax, vec_amax<T>(*reinterpret_cast<const uint4 *>(x + i * x_row)));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if constexpr (WPU > 1) {
            if (lane == 0) s_max[warp] = amax;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WPU; ++w) amax = fmaxf(amax, s_max[warp - sub + w]);
            __syncthreads();
        }
        if (!real) continue;
        float s = exp2_int(scale_exponent(amax));
        if (row > 0) {
            if (held >= s) {
                s = held;
            } else {
                const float ratio = held / s;
                for (int i = row_first; active && i < row; i += row_step) {
                    uint8_t *at = dst + i * c.s[2];
                    uint32_t *w = reinterpret_cast<uint32_t *>(at);
#pragma unroll
                    for (int k = 0; k < static_cast<int>(4 / sizeof(T)); ++k) {
                        const uint32_t b = w[k];
                        w[k] = pack_e4m3(e4m3_to_float(b & 255u) * ratio, e4m3_to_float(b >> 8 & 255u) * ratio,
                                         e4m3_to_float(b >> 16 & 255u) * ratio, e4m3_to_float(b >> 24) * ratio);
                    }
                }
            }
        }
        if (sub == 0 && lane == 0) *scale = s;
        const float inv = 1.f / s;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int i = row_first + k * row_step;
            if (active && i < n) vec_store<T>(dst + (row + i) * c.s[2], v[k], inv);
        }
        for (int i = row_first + NV * row_step; active && i < n; i += row_step)
            vec_store<T>(dst + (row + i) * c.s[2], *reinterpret_cast<const uint4 *>(x + i * x_row), inv);
    }
}

}  // namespace paged
}  // namespace pmkl_b200
