// Arithmetic shared by the read-out kernels: element conversions, the 8-bit
// block format, and block-wide sums.
#pragma once

#include <cfloat>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "readout.h"

namespace engram {

// Storage types by ElementType.  e4m3 is read as its byte.
template <uint32_t TYPE> struct Element;
template <> struct Element<kBf16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float get(T v) { return __bfloat162float(v); }
    static __device__ __forceinline__ T put(float v) { return __float2bfloat16_rn(v); }
    static constexpr float kLargest = 3.38953139e38f;
};
template <> struct Element<kFp16> {
    using T = __half;
    static __device__ __forceinline__ float get(T v) { return __half2float(v); }
    static __device__ __forceinline__ T put(float v) { return __float2half_rn(v); }
    static constexpr float kLargest = 65504.f;
};
template <> struct Element<kFp32> {
    using T = float;
    static __device__ __forceinline__ float get(T v) { return v; }
    static __device__ __forceinline__ T put(float v) { return v; }
    static constexpr float kLargest = FLT_MAX;
};
template <> struct Element<kE4m3> {
    using T = uint8_t;
    static __device__ __forceinline__ float get(T v) {
        return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)));
    }
};

// A parameter vector's element; its type is uniform over the launch.
__device__ __forceinline__ float load_param(const void *ptr, uint32_t type, int64_t at) {
    if (type == kBf16)
        return __bfloat162float(static_cast<const __nv_bfloat16 *>(ptr)[at]);
    if (type == kFp16)
        return __half2float(static_cast<const __half *>(ptr)[at]);
    return static_cast<const float *>(ptr)[at];
}

__device__ __forceinline__ void store_param(void *ptr, uint32_t type, int64_t at, float v) {
    if (type == kBf16)
        static_cast<__nv_bfloat16 *>(ptr)[at] = __float2bfloat16_rn(v);
    else if (type == kFp16)
        static_cast<__half *>(ptr)[at] = __float2half_rn(v);
    else
        static_cast<float *>(ptr)[at] = v;
}

// The 8-bit block format.  A block's scale is the least 2^k with
// max|v| <= 448 * 2^k over its finite values (448 = 1.75 * 2^8 is e4m3's
// largest; k is at least -126 so that 2^k and 2^-k are normal), or 1 for a
// block of zeros.  Dividing by a power of two is exact, so a code is the one
// rounding of v, at most 2^-4 of |v| off (e4m3's normal range, 2^-6 to 448 of
// the scale), and scale * code is exact in bf16.  A power of two costs no
// relative precision against amax / 448: it only shifts where the subnormal
// range begins by at most one bit.  Infinities and NaN are stored as NaN, and
// leave the other values of their block as they are.
__device__ __forceinline__ float finite_abs(float v) {
    const float a = fabsf(v);
    return a <= FLT_MAX ? a : 0.f;
}

__device__ __forceinline__ int block_exponent(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    const int k = int(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return amax == 0.f ? 0 : max(k, -126);
}

__device__ __forceinline__ float exp2_int(int k) { return __uint_as_float(uint32_t(k + 127) << 23); }

// Two codes (the first in the low byte) of values already divided by the scale.
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
    // The conversion saturates infinities; here they have to stay visible.
    const float nan = __uint_as_float(0x7FFFFFFFu);
    a = fabsf(a) <= FLT_MAX ? a : nan;
    b = fabsf(b) <= FLT_MAX ? b : nan;
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float2 from_e4m3x2(uint32_t two) {
    return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(two), __NV_E4M3)));
}

template <int LANES = 32> __device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2)
        v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
    return v;
}

// Sums of two values over the block, in every thread.  `shared` holds two
// floats per warp; a barrier ends the call's use of it.
__device__ __forceinline__ float2 block_sum2(float a, float b, float2 *shared) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        a += __shfl_xor_sync(0xFFFFFFFFu, a, d);
        b += __shfl_xor_sync(0xFFFFFFFFu, b, d);
    }
    const uint32_t warps = blockDim.x / 32;
    if (threadIdx.x % 32 == 0)
        shared[threadIdx.x / 32] = make_float2(a, b);
    __syncthreads();
    float2 total = make_float2(0.f, 0.f);
    for (uint32_t w = 0; w < warps; ++w) {
        total.x += shared[w].x;
        total.y += shared[w].y;
    }
    __syncthreads();
    return total;
}

} // namespace engram
