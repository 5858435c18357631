// paged_common.cuh -- what the operators of the paged 8-bit cache share: the
// cache's layout and lengths as the kernels see them, and the conversions
// between its 8-bit floats (e4m3) and fp32.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace pmkl_b200 {
namespace paged {

// Scales are powers of two in this range.
constexpr int kMinScaleExp = -64, kMaxScaleExp = 64;

// One side (keys or values) of the cache: 8-bit elements at block * s[0] +
// head * s[1] + row * s[2] + col, 64-bit offsets.
struct CacheView {
    uint8_t *base;
    long long s[3];
    float *scale;  // [num_blocks][kv_heads]
};

__device__ __forceinline__ float e4m3_to_float(uint8_t b) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}

// To the nearest, ties to even, beyond 448 as 448, NaN stays NaN.
__device__ __forceinline__ uint8_t float_to_e4m3(float x) {
    return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

// Exponent of the smallest power of two s with amax <= 448 s (448 = 1.75 *
// 2^8), within the scales' range; amax finite and not negative.
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return e < kMinScaleExp ? kMinScaleExp : (e > kMaxScaleExp ? kMaxScaleExp : e);
}

__device__ __forceinline__ float exp2_int(int e) {  // -126 <= e <= 127
    return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

}  // namespace paged
}  // namespace pmkl_b200
