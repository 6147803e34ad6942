// Arithmetic shared by the read-out kernels: element conversions, the 8-bit
// block format, and block-wide sums.
#pragma once

#include <cfloat>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "ptx.cuh"
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

// Sums of two values over the warp, in every lane.
__device__ __forceinline__ float2 lanes_sum2(float a, float b) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        a += __shfl_xor_sync(0xFFFFFFFFu, a, d);
        b += __shfl_xor_sync(0xFFFFFFFFu, b, d);
    }
    return make_float2(a, b);
}

// Sums of two values over the block, in every thread.  `shared` holds one
// float2 per warp and must not be the one of the block's previous call: one
// barrier then suffices, since every thread has read that one by then.
__device__ __forceinline__ float2 block_sum2(float a, float b, float2 *shared) {
    const float2 own = lanes_sum2(a, b);
    const uint32_t warps = blockDim.x / 32;
    if (threadIdx.x % 32 == 0)
        shared[threadIdx.x / 32] = own;
    __syncthreads();
    float2 total = make_float2(0.f, 0.f);
    for (uint32_t w = 0; w < warps; ++w) {
        total.x += shared[w].x;
        total.y += shared[w].y;
    }
    return total;
}

// Eight adjacent values as they lie in memory: 16 bytes of a 16-bit type, 32
// of fp32, 8 of codes.  Rows are streamed past L1; parameters stay in it.
template <uint32_t TYPE> struct Raw8 {
    Vec16 v;
    static constexpr int kBytes = 16;
};
template <> struct Raw8<kFp32> {
    Vec16 v, v2;
    static constexpr int kBytes = 32;
};
template <> struct Raw8<kE4m3> {
    uint2 v;
    static constexpr int kBytes = 8;
};

template <uint32_t TYPE> __device__ __forceinline__ Raw8<TYPE> load_row8(const void *ptr) {
    Raw8<TYPE> r;
    if constexpr (TYPE == kE4m3) {
        asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.v.x), "=r"(r.v.y) : "l"(ptr));
    } else {
        r.v = ld_nc_na_v4(ptr);
        if constexpr (TYPE == kFp32)
            r.v2 = ld_nc_na_v4(static_cast<const uint8_t *>(ptr) + 16);
    }
    return r;
}

__device__ __forceinline__ float2 from_bf16x2(uint32_t two) {
    return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xFFFF0000u));
}
__device__ __forceinline__ float2 from_fp16x2(uint32_t two) { return __half22float2(*reinterpret_cast<__half2 *>(&two)); }

template <uint32_t TYPE> __device__ __forceinline__ void unpack8(const Raw8<TYPE> &r, float (&x)[8]) {
    if constexpr (TYPE == kFp32) {
        const uint32_t w[8] = {r.v.x, r.v.y, r.v.z, r.v.w, r.v2.x, r.v2.y, r.v2.z, r.v2.w};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            x[e] = __uint_as_float(w[e]);
    } else if constexpr (TYPE == kE4m3) {
        const uint32_t w[4] = {r.v.x & 0xFFFFu, r.v.x >> 16, r.v.y & 0xFFFFu, r.v.y >> 16};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = from_e4m3x2(w[e]);
            x[2 * e] = f.x;
            x[2 * e + 1] = f.y;
        }
    } else {
        const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = TYPE == kBf16 ? from_bf16x2(w[e]) : from_fp16x2(w[e]);
            x[2 * e] = f.x;
            x[2 * e + 1] = f.y;
        }
    }
}

__device__ __forceinline__ uint32_t to_bf16x2(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

template <uint32_t TYPE> __device__ __forceinline__ void store_row8(void *ptr, const float (&x)[8]) {
    if constexpr (TYPE == kFp32) {
        st_na_v4(ptr, Vec16{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])});
        st_na_v4(static_cast<uint8_t *>(ptr) + 16,
                 Vec16{__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7])});
    } else {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (TYPE == kBf16) {
                w[e] = to_bf16x2(x[2 * e], x[2 * e + 1]);
            } else {
                const __half2 h = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
                w[e] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        st_na_v4(ptr, Vec16{w[0], w[1], w[2], w[3]});
    }
}

// Eight codes of values already divided by their scale.
__device__ __forceinline__ uint2 to_e4m3x8(const float (&x)[8], float down) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        w[e] = to_e4m3x2(x[2 * e] * down, x[2 * e + 1] * down);
    return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

// Eight adjacent parameters (16-byte aligned); their type is uniform over the launch.
__device__ __forceinline__ void load_param8(const void *ptr, uint32_t type, uint32_t at, float (&x)[8]) {
    if (type == kFp32) {
        const float4 *q = reinterpret_cast<const float4 *>(static_cast<const float *>(ptr) + at);
        const float4 a = __ldg(q), b = __ldg(q + 1);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(ptr) + at));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = type == kBf16 ? from_bf16x2(w[e]) : from_fp16x2(w[e]);
            x[2 * e] = f.x;
            x[2 * e + 1] = f.y;
        }
    }
}

inline bool on_boundary(const void *ptr, uint32_t bytes) { return reinterpret_cast<uintptr_t>(ptr) % bytes == 0; }

inline __host__ __device__ constexpr uint32_t element_bytes(uint32_t type) { return type == kFp32 ? 4 : type == kE4m3 ? 1 : 2; }

} // namespace engram
