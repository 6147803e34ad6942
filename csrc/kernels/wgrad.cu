// A projection's weight and bias gradients from the 8-bit checkpoint of its
// input (sm_100a).
//
// dW[o][k] = sum_m dy[m][o] X[m][k] with X the checkpoint's rows.  Where the
// projection's input was X w + b (a norm's affine part), the same checkpoint
// serves: dW[o][k] = w[k] G[o][k] + b[k] s[o], G = dy^T X and s[o] = sum_m
// dy[m][o], which is also the bias gradient.
#include "readout.h"
#include "rowmath.cuh"

namespace engram {

namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64, kDepth = 16;

// Column sums of dy over one part of the rows.
template <uint32_t TYPE>
__global__ void __launch_bounds__(kThreads) dy_sums_part(const __grid_constant__ WeightGradParams p) {
    __shared__ float s_sum[kThreads / 32][32];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, o = blockIdx.x * 32 + lane;
    const int64_t share = (p.rows + p.parts - 1) / p.parts;
    const int64_t first = int64_t(blockIdx.y) * share, last = min(first + share, p.rows);
    float sum = 0.f;
    if (o < p.out)
        for (int64_t r = first + warp; r < last; r += kThreads / 32)
            sum += Element<TYPE>::get(static_cast<const typename Element<TYPE>::T *>(p.dy)[r * p.dy_stride + o]);
    s_sum[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && o < p.out) {
#pragma unroll
        for (int w = 1; w < kThreads / 32; ++w)
            sum += s_sum[w][lane];
        p.partial[int64_t(blockIdx.y) * p.out + o] = sum;
    }
}

__global__ void __launch_bounds__(kThreads) dy_sums_join(const __grid_constant__ WeightGradParams p) {
    const uint32_t o = blockIdx.x * kThreads + threadIdx.x;
    if (o >= p.out)
        return;
    float sum = 0.f;
    for (uint32_t part = 0; part < p.parts; ++part)
        sum += p.partial[int64_t(part) * p.out + o];
    p.dy_sums[o] = sum;
    if (p.dbias != nullptr)
        store_param(p.dbias, p.out_type, o, sum);
}

// 64 x 64 outputs per block, 16 rows at a time through shared memory.
template <uint32_t TYPE>
__global__ void __launch_bounds__(kThreads) weight_grad_any(const __grid_constant__ WeightGradParams p) {
    __shared__ float s_dy[kDepth][kTile], s_x[kDepth][kTile];
    const uint32_t o0 = blockIdx.y * kTile, k0 = blockIdx.x * kTile;
    const uint32_t ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    float acc[4][4] = {};
    for (int64_t m0 = 0; m0 < p.rows; m0 += kDepth) {
        for (uint32_t i = threadIdx.x; i < kDepth * kTile; i += kThreads) {
            const uint32_t d = i / kTile, c = i % kTile;
            const int64_t m = m0 + d;
            float a = 0.f, b = 0.f;
            if (m < p.rows && o0 + c < p.out)
                a = Element<TYPE>::get(static_cast<const typename Element<TYPE>::T *>(p.dy)[m * p.dy_stride + o0 + c]);
            if (m < p.rows && k0 + c < p.width)
                b = Element<kE4m3>::get(p.codes[m * p.codes_stride + k0 + c]) *
                    p.scales[m * p.scale_row_stride + (k0 + c) / kCheckpointBlock * p.scale_col_stride];
            s_dy[d][c] = a;
            s_x[d][c] = b;
        }
        __syncthreads();
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            float a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = s_dy[d][ty * 4 + i];
                b[i] = s_x[d][tx * 4 + i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] += a[i] * b[j];
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t o = o0 + ty * 4 + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t k = k0 + tx * 4 + j;
            if (o >= p.out || k >= p.width)
                continue;
            float v = acc[i][j];
            if (p.norm_weight != nullptr)
                v *= load_param(p.norm_weight, p.param_type, k);
            if (p.norm_bias != nullptr)
                v += load_param(p.norm_bias, p.param_type, k) * p.dy_sums[o];
            store_param(p.dweight, p.out_type, int64_t(o) * p.width + k, v);
        }
    }
}

template <uint32_t TYPE> void weight_grad(const WeightGradParams &p, cudaStream_t stream) {
    if (p.dy_sums != nullptr) {
        dy_sums_part<TYPE><<<dim3((p.out + 31) / 32, p.parts), kThreads, 0, stream>>>(p);
        dy_sums_join<<<(p.out + kThreads - 1) / kThreads, kThreads, 0, stream>>>(p);
    }
    weight_grad_any<TYPE><<<dim3((p.width + kTile - 1) / kTile, (p.out + kTile - 1) / kTile), kThreads, 0, stream>>>(p);
}

} // namespace

uint32_t weight_grad_parts(const WeightGradParams &p, int num_sms) {
    const int64_t want = int64_t(num_sms) * 4 * 32 / p.out + 1, most = (p.rows + 31) / 32;
    return uint32_t(want < most ? want : most);
}

cudaError_t launch_weight_grad(const WeightGradParams &p, int, cudaStream_t stream) {
    if (p.type == kBf16)
        weight_grad<kBf16>(p, stream);
    else if (p.type == kFp16)
        weight_grad<kFp16>(p, stream);
    else
        weight_grad<kFp32>(p, stream);
    return cudaGetLastError();
}

} // namespace engram
