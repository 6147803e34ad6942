// Activations to 8 bits and back (sm_100a): e4m3 codes with one power-of-two
// scale per row and 128 columns (the format is described in rowmath.cuh).
#include "readout.h"
#include "rowmath.cuh"

namespace engram {

namespace {

constexpr int kThreads = 256;

// One warp per block of 128 columns: any width, stride and alignment.
template <uint32_t TYPE>
__global__ void __launch_bounds__(kThreads) save_any(const __grid_constant__ SaveFp8Params p) {
    const uint32_t lane = threadIdx.x % 32;
    const uint32_t blocks = (p.width + kCheckpointBlock - 1) / kCheckpointBlock;
    const int64_t total = p.rows * blocks, stride = int64_t(gridDim.x) * (kThreads / 32);
    for (int64_t at = int64_t(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32; at < total; at += stride) {
        const int64_t r = at / blocks;
        const uint32_t blk = uint32_t(at - r * blocks);
        const auto *x = static_cast<const typename Element<TYPE>::T *>(p.x) + r * p.x_stride;
        float v[4], amax = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t c = blk * kCheckpointBlock + i * 32 + lane;
            v[i] = c < p.width ? Element<TYPE>::get(x[c]) : 0.f;
            amax = fmaxf(amax, finite_abs(v[i]));
        }
        const int k = block_exponent(lanes_max(amax));
        const float down = exp2_int(-k);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t c = blk * kCheckpointBlock + i * 32 + lane;
            if (c < p.width)
                p.codes[r * p.codes_stride + c] = uint8_t(to_e4m3x2(v[i] * down, 0.f));
        }
        if (lane == 0)
            p.scales[at] = exp2_int(k);
    }
}

// A finite code's value that its type cannot hold (a block's largest value may
// have been rounded up past it) becomes the type's largest.
template <uint32_t TYPE> __device__ __forceinline__ float held(float v, float code) {
    const float most = Element<TYPE>::kLargest;
    return isnan(code) ? code : fminf(fmaxf(v, -most), most);
}

template <uint32_t TYPE>
__global__ void __launch_bounds__(kThreads) restore_any(const __grid_constant__ RestoreFp8Params p) {
    const uint32_t lane = threadIdx.x % 32;
    const uint32_t blocks = (p.width + kCheckpointBlock - 1) / kCheckpointBlock;
    const int64_t total = p.rows * blocks, stride = int64_t(gridDim.x) * (kThreads / 32);
    for (int64_t at = int64_t(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32; at < total; at += stride) {
        const int64_t r = at / blocks;
        const uint32_t blk = uint32_t(at - r * blocks);
        const float scale = p.scales[r * p.scale_row_stride + blk * p.scale_col_stride];
        auto *x = static_cast<typename Element<TYPE>::T *>(p.x) + r * p.width;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t c = blk * kCheckpointBlock + i * 32 + lane;
            if (c < p.width) {
                const float code = Element<kE4m3>::get(p.codes[r * p.codes_stride + c]);
                x[c] = Element<TYPE>::put(held<TYPE>(code * scale, code));
            }
        }
    }
}

uint32_t grid_of(int64_t rows, uint32_t width, int num_sms) {
    const int64_t blocks = (width + kCheckpointBlock - 1) / kCheckpointBlock;
    const int64_t need = (rows * blocks + kThreads / 32 - 1) / (kThreads / 32);
    return uint32_t(need < int64_t(num_sms) * 8 ? need : int64_t(num_sms) * 8);
}

} // namespace

cudaError_t launch_save_fp8(const SaveFp8Params &p, int num_sms, cudaStream_t stream) {
    const uint32_t grid = grid_of(p.rows, p.width, num_sms);
    if (p.type == kBf16)
        save_any<kBf16><<<grid, kThreads, 0, stream>>>(p);
    else if (p.type == kFp16)
        save_any<kFp16><<<grid, kThreads, 0, stream>>>(p);
    else
        save_any<kFp32><<<grid, kThreads, 0, stream>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_restore_fp8(const RestoreFp8Params &p, int num_sms, cudaStream_t stream) {
    const uint32_t grid = grid_of(p.rows, p.width, num_sms);
    if (p.type == kBf16)
        restore_any<kBf16><<<grid, kThreads, 0, stream>>>(p);
    else if (p.type == kFp16)
        restore_any<kFp16><<<grid, kThreads, 0, stream>>>(p);
    else
        restore_any<kFp32><<<grid, kThreads, 0, stream>>>(p);
    return cudaGetLastError();
}

} // namespace engram
