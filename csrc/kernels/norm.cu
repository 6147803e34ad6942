// Layer norm over rows, forward and backward (sm_100a).
//
// Forward, per row: mean = sum x / N, r = 1 / sqrt(sum (x - mean)^2 / N + eps),
// h = (x - mean) r, y = h w + b.  Backward, with g = dy w: dx = r (g - mean(g) -
// h mean(g h)); per column: dw = sum dy h, db = sum dy.  All sums are fp32.
// The variance is the corrected two-pass form: with d = x - m for the first
// pass's mean m, sum d (zero but for m's rounding) corrects both mean and
// variance, so a large common offset of a row costs no digits.
#include "readout.h"
#include "rowmath.cuh"

namespace engram {

namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;

// One element of a forward row as fp32.
template <uint32_t IN> struct RowReader {
    const typename Element<IN>::T *row;
    __device__ RowReader(const NormForwardParams &p, int64_t r)
        : row(static_cast<const typename Element<IN>::T *>(p.x) + r * p.x_stride) {}
    __device__ __forceinline__ float operator()(uint32_t c) const { return Element<IN>::get(row[c]); }
};
template <> struct RowReader<kE4m3> {
    const uint8_t *row;
    const float *scales;
    int64_t col_stride;
    uint32_t hidden, packs, block;
    __device__ RowReader(const NormForwardParams &p, int64_t r)
        : row(static_cast<const uint8_t *>(p.x) + r * p.x_stride), scales(p.scales + r * p.scale_row_stride),
          col_stride(p.scale_col_stride), hidden(p.hidden), packs(p.packs), block(p.block) {}
    __device__ __forceinline__ float operator()(uint32_t c) const {
        const uint32_t pack = c / hidden * packs + c % hidden / block;
        return Element<kE4m3>::get(row[c]) * scales[pack * col_stride];
    }
};

// Any width, stride and alignment: one block per row, which it reads three
// times (twice from cache).
template <uint32_t IN, uint32_t OUT>
__global__ void __launch_bounds__(kRowThreads) norm_forward_any(const __grid_constant__ NormForwardParams p) {
    __shared__ float2 s_sum[kRowWarps];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const float inv = 1.f / float(p.width);
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const RowReader<IN> x(p, r);
        float a = 0.f, b = 0.f;
        for (uint32_t c = threadIdx.x; c < p.width; c += kRowThreads)
            a += x(c);
        float mean = block_sum2(a, 0.f, s_sum).x * inv;
        a = 0.f;
        for (uint32_t c = threadIdx.x; c < p.width; c += kRowThreads) {
            const float d = x(c) - mean;
            a += d;
            b += d * d;
        }
        const float2 sums = block_sum2(a, b, s_sum);
        const float shift = sums.x * inv;
        const float rstd = 1.f / sqrtf(fmaxf(sums.y * inv - shift * shift, 0.f) + p.eps);
        mean += shift;
        if (threadIdx.x == 0) {
            if (p.keep == kKeepStats)
                p.mean[r] = mean;
            if (p.keep != kKeepNothing)
                p.rstd[r] = rstd;
        }
        auto *y = static_cast<typename Element<OUT>::T *>(p.y) + r * p.width;
        const uint32_t blocks = (p.width + kCheckpointBlock - 1) / kCheckpointBlock;
        for (uint32_t blk = warp; blk < blocks; blk += kRowWarps) {
            float h[4], amax = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t c = blk * kCheckpointBlock + i * 32 + lane;
                h[i] = 0.f;
                if (c < p.width) {
                    h[i] = (x(c) - mean) * rstd;
                    amax = fmaxf(amax, finite_abs(h[i]));
                    float v = h[i];
                    if (p.weight != nullptr)
                        v *= load_param(p.weight, p.param_type, c);
                    if (p.bias != nullptr)
                        v += load_param(p.bias, p.param_type, c);
                    y[c] = Element<OUT>::put(v);
                }
            }
            if (p.keep == kKeepFp8) {
                const int k = block_exponent(lanes_max(amax));
                const float down = exp2_int(-k);
                uint8_t *codes = p.codes + r * p.codes_stride;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t c = blk * kCheckpointBlock + i * 32 + lane;
                    if (c < p.width)
                        codes[c] = uint8_t(to_e4m3x2(h[i] * down, 0.f));
                }
                if (lane == 0)
                    p.code_scales[r * blocks + blk] = exp2_int(k);
            }
        }
    }
}

// A normalised value of the backward pass.
template <uint32_t X> __device__ __forceinline__ float kept_value(const NormBackwardParams &p, int64_t r, uint32_t c) {
    if (X == kE4m3)
        return Element<kE4m3>::get(p.codes[r * p.codes_stride + c]) *
               p.code_scales[r * p.code_scales_stride + c / kCheckpointBlock * p.scale_col_stride];
    else
        return (Element<X>::get(static_cast<const typename Element<X>::T *>(p.x)[r * p.x_stride + c]) - p.mean[r]) *
               p.rstd[r];
}

template <uint32_t X, uint32_t DY>
__global__ void __launch_bounds__(kRowThreads) norm_backward_rows_any(const __grid_constant__ NormBackwardParams p) {
    __shared__ float2 s_sum[kRowWarps];
    const float inv = 1.f / float(p.width);
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const auto *dy = static_cast<const typename Element<DY>::T *>(p.dy) + r * p.dy_stride;
        auto *dx = static_cast<typename Element<DY>::T *>(p.dx) + r * p.width;
        float a = 0.f, b = 0.f;
        for (uint32_t c = threadIdx.x; c < p.width; c += kRowThreads) {
            float g = Element<DY>::get(dy[c]);
            if (p.weight != nullptr)
                g *= load_param(p.weight, p.param_type, c);
            a += g;
            b += g * kept_value<X>(p, r, c);
        }
        const float2 sums = block_sum2(a, b, s_sum);
        const float c1 = sums.x * inv, c2 = sums.y * inv, rstd = p.rstd[r];
        for (uint32_t c = threadIdx.x; c < p.width; c += kRowThreads) {
            float g = Element<DY>::get(dy[c]);
            if (p.weight != nullptr)
                g *= load_param(p.weight, p.param_type, c);
            dx[c] = Element<DY>::put(rstd * (g - c1 - kept_value<X>(p, r, c) * c2));
        }
    }
}

// Column sums of dy and dy h over one part of the rows: a block takes 32
// columns, its warps take every eighth row of the part.
template <uint32_t X, uint32_t DY>
__global__ void __launch_bounds__(kRowThreads) norm_backward_columns_any(const __grid_constant__ NormBackwardParams p) {
    __shared__ float s_w[kRowWarps][32], s_b[kRowWarps][32];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t c = blockIdx.x * 32 + lane;
    const int64_t share = (p.rows + p.parts - 1) / p.parts;
    const int64_t first = int64_t(blockIdx.y) * share, last = min(first + share, p.rows);
    float dw = 0.f, db = 0.f;
    if (c < p.width)
        for (int64_t r = first + warp; r < last; r += kRowWarps) {
            const float g = Element<DY>::get(static_cast<const typename Element<DY>::T *>(p.dy)[r * p.dy_stride + c]);
            db += g;
            dw += g * kept_value<X>(p, r, c);
        }
    s_w[warp][lane] = dw;
    s_b[warp][lane] = db;
    __syncthreads();
    if (warp == 0 && c < p.width) {
#pragma unroll
        for (int w = 1; w < kRowWarps; ++w) {
            dw += s_w[w][lane];
            db += s_b[w][lane];
        }
        p.partial[int64_t(blockIdx.y) * p.width + c] = dw;
        p.partial[int64_t(p.parts + blockIdx.y) * p.width + c] = db;
    }
}

// Joins the parts in order, so the sums do not depend on which block came first.
__global__ void __launch_bounds__(kRowThreads) norm_backward_join(const __grid_constant__ NormBackwardParams p) {
    const uint32_t c = blockIdx.x * kRowThreads + threadIdx.x;
    if (c >= p.width)
        return;
    const float *partial = p.partial + int64_t(blockIdx.y) * p.parts * p.width + c;
    float sum = 0.f;
    for (uint32_t part = 0; part < p.parts; ++part)
        sum += partial[int64_t(part) * p.width];
    store_param(blockIdx.y == 0 ? p.dweight : p.dbias, p.param_type, c, sum);
}

uint32_t row_grid(int64_t rows, int num_sms) {
    return uint32_t(rows < int64_t(num_sms) * 8 ? rows : int64_t(num_sms) * 8);
}

template <uint32_t IN, uint32_t OUT> void forward(const NormForwardParams &p, int num_sms, cudaStream_t stream) {
    norm_forward_any<IN, OUT><<<row_grid(p.rows, num_sms), kRowThreads, 0, stream>>>(p);
}

template <uint32_t X, uint32_t DY> void backward(const NormBackwardParams &p, int num_sms, cudaStream_t stream) {
    if (p.dx != nullptr)
        norm_backward_rows_any<X, DY><<<row_grid(p.rows, num_sms), kRowThreads, 0, stream>>>(p);
    if (p.dweight == nullptr)
        return;
    norm_backward_columns_any<X, DY><<<dim3((p.width + 31) / 32, p.parts), kRowThreads, 0, stream>>>(p);
    norm_backward_join<<<dim3((p.width + kRowThreads - 1) / kRowThreads, 2), kRowThreads, 0, stream>>>(p);
}

} // namespace

cudaError_t launch_norm_forward(const NormForwardParams &p, int num_sms, cudaStream_t stream) {
    if (p.in_type == kBf16)
        forward<kBf16, kBf16>(p, num_sms, stream);
    else if (p.in_type == kFp16)
        forward<kFp16, kFp16>(p, num_sms, stream);
    else if (p.in_type == kFp32)
        forward<kFp32, kFp32>(p, num_sms, stream);
    else if (p.out_type == kBf16)
        forward<kE4m3, kBf16>(p, num_sms, stream);
    else if (p.out_type == kFp16)
        forward<kE4m3, kFp16>(p, num_sms, stream);
    else
        forward<kE4m3, kFp32>(p, num_sms, stream);
    return cudaGetLastError();
}

uint32_t norm_backward_parts(const NormBackwardParams &p, int num_sms) {
    const int64_t want = int64_t(num_sms) * 4 * 32 / p.width + 1, most = (p.rows + 31) / 32;
    return uint32_t(want < most ? want : most);
}

cudaError_t launch_norm_backward(const NormBackwardParams &p, int num_sms, cudaStream_t stream) {
    const bool fp8 = p.keep == kKeepFp8;
    if (p.dy_type == kBf16)
        fp8 ? backward<kE4m3, kBf16>(p, num_sms, stream) : backward<kBf16, kBf16>(p, num_sms, stream);
    else if (p.dy_type == kFp16)
        fp8 ? backward<kE4m3, kFp16>(p, num_sms, stream) : backward<kFp16, kFp16>(p, num_sms, stream);
    else
        fp8 ? backward<kE4m3, kFp32>(p, num_sms, stream) : backward<kFp32, kFp32>(p, num_sms, stream);
    return cudaGetLastError();
}

} // namespace engram
