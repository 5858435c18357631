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

}  // namespace paged
}  // namespace pmkl_b200
