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

struct BlockScale {
    float up, down;  // 2^k and 2^-k
};

__device__ __forceinline__ BlockScale block_scale(float amax) {
    // 2^k's bits: amax's exponent less 8, one more where its fraction is above .75
    // (the addition then carries into the exponent).
    const int bits = int((__float_as_uint(amax) + 0x1FFFFFu) & 0x7F800000u) - (8 << 23);
    const uint32_t up = amax == 0.f ? 127u << 23 : uint32_t(max(bits, 1 << 23));
    return {__uint_as_float(up), __uint_as_float((254u << 23) - up)};
}

// The code of a value already divided by its scale.
__device__ __forceinline__ uint8_t to_e4m3(float v) {
    // The conversion saturates infinities; here they have to stay visible.
    return __nv_cvt_float_to_fp8(fabsf(v) <= FLT_MAX ? v : __uint_as_float(0x7FFFFFFFu), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float2 from_e4m3x2(uint32_t two) {
    return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(two), __NV_E4M3)));
}

// The largest magnitude of three, NaN passed by.
__device__ __forceinline__ float largest3(float a, float b, float c) {
    float r;
    asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <int LANES = 32> __device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2)
        v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
    return v;
}

// Sum of one value over the warp, in every lane.
__device__ __forceinline__ float lanes_sum(float a) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2)
        a += __shfl_xor_sync(0xFFFFFFFFu, a, d);
    return a;
}

// Sums of two values over the warp: of a in lanes 0-15, of b in lanes 16-31.
// The first step swaps halves, so two sums cost five shuffles and not ten.
__device__ __forceinline__ float lanes_sum_halves(float a, float b) {
    const bool upper = threadIdx.x & 16;
    float v = upper ? b : a;
    v += __shfl_xor_sync(0xFFFFFFFFu, upper ? a : b, 16);
#pragma unroll
    for (int d = 8; d > 0; d /= 2)
        v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    return v;
}

// Sums of two values over the warp, in every lane.
__device__ __forceinline__ float2 lanes_sum2(float a, float b) {
    const float v = lanes_sum_halves(a, b), w = __shfl_xor_sync(0xFFFFFFFFu, v, 16);
    return threadIdx.x & 16 ? make_float2(w, v) : make_float2(v, w);
}

// Sums over a block of at most 16 warps, in every thread.  `shared` must not be
// the one of the block's previous call: one barrier then suffices, since every
// thread has read that one by then.  Entries past the block's warps are zero
// (clear_sums), so the warps' sums are joined by one load and four shuffles,
// whatever their number.
struct WarpSums {
    float of[2][16];
};

__device__ __forceinline__ void clear_sums(WarpSums &shared) {
    for (uint32_t i = threadIdx.x; i < 32; i += blockDim.x)
        shared.of[i / 16][i % 16] = 0.f;
}

__device__ __forceinline__ float2 block_sum2(float a, float b, WarpSums &shared) {
    const uint32_t lane = threadIdx.x % 32;
    float v = lanes_sum_halves(a, b);
    if (lane % 16 == 0)
        shared.of[lane / 16][threadIdx.x / 32] = v;
    __syncthreads();
    v = shared.of[lane / 16][lane % 16];
#pragma unroll
    for (int d = 8; d > 0; d /= 2)
        v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    const float w = __shfl_xor_sync(0xFFFFFFFFu, v, 16);
    return lane & 16 ? make_float2(w, v) : make_float2(v, w);
}

__device__ __forceinline__ float block_sum(float a, WarpSums &shared) {
    const uint32_t lane = threadIdx.x % 32;
    a = lanes_sum(a);
    if (lane == 0)
        shared.of[0][threadIdx.x / 32] = a;
    __syncthreads();
    a = shared.of[0][lane % 16];
#pragma unroll
    for (int d = 8; d > 0; d /= 2)
        a += __shfl_xor_sync(0xFFFFFFFFu, a, d);
    return a;
}

// The same for blocks of up to T threads, more than 16 warps by pairs in lanes.
template <int T> struct RowSums : WarpSums {
    __device__ __forceinline__ void clear() { clear_sums(*this); }
    __device__ __forceinline__ float sum(float a) { return block_sum(a, *this); }
    __device__ __forceinline__ float2 sum2(float a, float b) { return block_sum2(a, b, *this); }
};
struct WideSums {
    float2 of[32];
    __device__ __forceinline__ void clear() {}
    __device__ __forceinline__ float sum(float a) { return sum2(a, 0.f).x; }
    __device__ __forceinline__ float2 sum2(float a, float b) {
        const uint32_t lane = threadIdx.x % 32;
        const float2 own = lanes_sum2(a, b);
        if (lane == 0)
            of[threadIdx.x / 32] = own;
        __syncthreads();
        const float2 v = lane < blockDim.x / 32 ? of[lane] : make_float2(0.f, 0.f);
        return lanes_sum2(v.x, v.y);
    }
};
template <> struct RowSums<768> : WideSums {};
template <> struct RowSums<1024> : WideSums {};

// Eight adjacent values as they lie in memory: 16 bytes of a 16-bit type, 32
// of fp32, 8 of codes.
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

// Two fp32 values in one register pair, and two operations in one instruction
// (sm_100).  The kernels over rows take half to 60% of the issue slots, so fewer
// instructions count beside memory.  A pair stays one 64-bit value from its unpacking to its rounding:
// taken apart between operations it costs moves.
struct Pair {
    uint64_t v;
};
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ Pair pair(float2 f) { return pair(f.x, f.y); }
__device__ __forceinline__ Pair both(float f) { return pair(f, f); }
__device__ __forceinline__ float2 parts(Pair p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p.v));
    return r;
}
__device__ __forceinline__ float total(Pair p) {
    const float2 f = parts(p);
    return f.x + f.y;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

__device__ __forceinline__ float2 from_bf16x2(uint32_t two) {
    return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xFFFF0000u));
}
__device__ __forceinline__ float2 from_fp16x2(uint32_t two) { return __half22float2(*reinterpret_cast<__half2 *>(&two)); }
__device__ __forceinline__ uint32_t to_bf16x2(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t to_fp16x2(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

template <uint32_t TYPE> __device__ __forceinline__ void unpack8(const Raw8<TYPE> &r, Pair (&x)[4]) {
    if constexpr (TYPE == kFp32) {
        x[0] = pair(__uint_as_float(r.v.x), __uint_as_float(r.v.y));
        x[1] = pair(__uint_as_float(r.v.z), __uint_as_float(r.v.w));
        x[2] = pair(__uint_as_float(r.v2.x), __uint_as_float(r.v2.y));
        x[3] = pair(__uint_as_float(r.v2.z), __uint_as_float(r.v2.w));
    } else if constexpr (TYPE == kE4m3) {
        x[0] = pair(from_e4m3x2(r.v.x & 0xFFFFu));
        x[1] = pair(from_e4m3x2(r.v.x >> 16));
        x[2] = pair(from_e4m3x2(r.v.y & 0xFFFFu));
        x[3] = pair(from_e4m3x2(r.v.y >> 16));
    } else {
        const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            x[e] = pair(TYPE == kBf16 ? from_bf16x2(w[e]) : from_fp16x2(w[e]));
    }
}

template <uint32_t TYPE> __device__ __forceinline__ void store_row8(void *ptr, const Pair (&x)[4]) {
    if constexpr (TYPE == kFp32) {
        Vec32 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w.v[2 * e] = __float_as_uint(parts(x[e]).x);
            w.v[2 * e + 1] = __float_as_uint(parts(x[e]).y);
        }
        st_v8(ptr, w);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = TYPE == kBf16 ? to_bf16x2(parts(x[e]).x, parts(x[e]).y) : to_fp16x2(parts(x[e]).x, parts(x[e]).y);
        st_na_v4(ptr, Vec16{w[0], w[1], w[2], w[3]});
    }
}

// Eight codes of values that are finite or NaN, divided by their scale.
__device__ __forceinline__ uint2 to_e4m3x8(const Pair (&x)[4], float down) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        w[e] = __nv_cvt_float2_to_fp8x2(parts(mul2(x[e], both(down))), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

// Eight adjacent parameters (on a 16-byte boundary, fp32 on a 32-byte one), kept in L1.
template <uint32_t TYPE> __device__ __forceinline__ void load_param8(const uint8_t *ptr, Pair (&x)[4]) {
    Raw8<TYPE> r;
    if constexpr (TYPE == kFp32) {
        asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r.v.x), "=r"(r.v.y), "=r"(r.v.z), "=r"(r.v.w), "=r"(r.v2.x), "=r"(r.v2.y), "=r"(r.v2.z),
                       "=r"(r.v2.w)
                     : "l"(ptr));
    } else {
        const uint4 a = __ldg(reinterpret_cast<const uint4 *>(ptr));
        r.v = Vec16{a.x, a.y, a.z, a.w};
    }
    unpack8<TYPE>(r, x);
}

// Eight values from shared memory.
template <uint32_t TYPE> __device__ __forceinline__ void load_shared8(uint32_t at, Pair (&x)[4]) {
    Raw8<TYPE> r;
    if constexpr (TYPE == kE4m3) {
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.v.x), "=r"(r.v.y) : "r"(at));
    } else {
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r.v.x), "=r"(r.v.y), "=r"(r.v.z), "=r"(r.v.w)
                     : "r"(at));
        if constexpr (TYPE == kFp32)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(r.v2.x), "=r"(r.v2.y), "=r"(r.v2.z), "=r"(r.v2.w)
                         : "r"(at + 16));
    }
    unpack8<TYPE>(r, x);
}

// A kernel that only needs the one before it in its stream for a part of its
// work starts while that one ends: the earlier one says when (all its blocks
// have called start_next or ended), the later one waits for its end and its
// memory where it needs them.
__device__ __forceinline__ void start_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <class... Params, class... Args>
cudaError_t launch_overlapped(void (*kernel)(Params...), dim3 grid, uint32_t threads, uint32_t shared, cudaStream_t stream,
                              const Args &...args) {
    cudaLaunchAttribute overlap{};
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    config.attrs = &overlap;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

inline bool on_boundary(const void *ptr, uint32_t bytes) { return reinterpret_cast<uintptr_t>(ptr) % bytes == 0; }

inline __host__ __device__ constexpr uint32_t element_bytes(uint32_t type) { return type == kFp32 ? 4 : type == kE4m3 ? 1 : 2; }

} // namespace engram
