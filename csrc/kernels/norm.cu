// Layer norm over rows, forward and backward (sm_100a).
//
// Forward, per row: mean = sum x / N, r = 1 / sqrt(sum (x - mean)^2 / N + eps),
// h = (x - mean) r, y = h w + b.  Backward, with g = dy w: dx = r (g - mean(g) -
// h mean(g h)); per column: dw = sum dy h, db = sum dy.  All sums are fp32.
// The variance is the corrected two-pass form: with d = x - m for the first
// pass's mean m, sum d (zero but for m's rounding) corrects both mean and
// variance, so a large common offset of a row costs no digits.
#include <algorithm>

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
    __shared__ float2 s_sum[2][kRowWarps];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const float inv = 1.f / float(p.width);
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const RowReader<IN> x(p, r);
        float a = 0.f, b = 0.f;
        for (uint32_t c = threadIdx.x; c < p.width; c += kRowThreads)
            a += x(c);
        float mean = block_sum2(a, 0.f, s_sum[0]).x * inv;
        a = 0.f;
        for (uint32_t c = threadIdx.x; c < p.width; c += kRowThreads) {
            const float d = x(c) - mean;
            a += d;
            b += d * d;
        }
        const float2 sums = block_sum2(a, b, s_sum[1]);
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

// A row of whole 8-value chunks on vector boundaries, held in registers: one
// pass over memory.  Chunk c of a row is thread c % T's, T the block (or, for
// rows of at most 32 V chunks, each warp, which then has a row of its own).
// Sixteen lanes hold a checkpoint block, so its largest value takes four
// shuffles.
template <uint32_t IN, uint32_t OUT, int V>
__global__ void __launch_bounds__(1024) norm_forward_row(const __grid_constant__ NormForwardParams p, bool warp_rows) {
    __shared__ float2 s_sum[2][32];
    const uint32_t lane = threadIdx.x % 32, chunks = p.width / 8;
    const uint32_t t = warp_rows ? lane : threadIdx.x, stride = warp_rows ? 32 : blockDim.x;
    const int64_t r = warp_rows ? int64_t(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32 : int64_t(blockIdx.x);
    if (r >= p.rows)
        return;  // a whole warp of a block of warp rows
    const float inv = 1.f / float(p.width);
    const uint8_t *row = static_cast<const uint8_t *>(p.x) + r * p.x_stride * int64_t(sizeof(typename Element<IN>::T));
    float x[V][8];
    Raw8<IN> raw[V];
    float scale[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const uint32_t c = t + i * stride;
        scale[i] = 1.f;
        if (c < chunks) {
            raw[i] = load_row8<IN>(row + c * Raw8<IN>::kBytes);
            if constexpr (IN == kE4m3) {
                const uint32_t entry = c * 8 / p.hidden, column = c * 8 - entry * p.hidden;
                scale[i] = __ldg(p.scales + r * p.scale_row_stride +
                                 (entry * p.packs + column / p.block) * p.scale_col_stride);
            }
        }
    }
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (t + i * stride < chunks) {
            unpack8<IN>(raw[i], x[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if constexpr (IN == kE4m3)
                    x[i][e] *= scale[i];
                a += x[i][e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[i][e] = 0.f;
        }
    }
    float mean = (warp_rows ? lanes_sum2(a, 0.f) : block_sum2(a, 0.f, s_sum[0])).x * inv;
    a = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (t + i * stride < chunks) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = x[i][e] - mean;
                a += d;
                b += d * d;
            }
        }
    const float2 sums = warp_rows ? lanes_sum2(a, b) : block_sum2(a, b, s_sum[1]);
    const float shift = sums.x * inv;
    const float rstd = 1.f / sqrtf(fmaxf(sums.y * inv - shift * shift, 0.f) + p.eps);
    mean += shift;
    if (t == 0) {
        if (p.keep == kKeepStats)
            p.mean[r] = mean;
        if (p.keep != kKeepNothing)
            p.rstd[r] = rstd;
    }
    uint8_t *y = static_cast<uint8_t *>(p.y) + r * p.width * int64_t(sizeof(typename Element<OUT>::T));
    const uint32_t blocks = (p.width + kCheckpointBlock - 1) / kCheckpointBlock;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const uint32_t c = t + i * stride;
        const bool there = c < chunks;
        float amax = 0.f;
        if (there) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[i][e] = (x[i][e] - mean) * rstd;
                amax = fmaxf(amax, finite_abs(x[i][e]));
                v[e] = x[i][e];
            }
            if (p.weight != nullptr) {
                float w[8];
                load_param8(p.weight, p.param_type, c * 8, w);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] *= w[e];
            }
            if (p.bias != nullptr) {
                float w[8];
                load_param8(p.bias, p.param_type, c * 8, w);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] += w[e];
            }
            store_row8<OUT>(y + c * Raw8<OUT>::kBytes, v);
        }
        if (p.keep == kKeepFp8) {
            const int k = block_exponent(lanes_max<16>(amax));
            if (there) {
                *reinterpret_cast<uint2 *>(p.codes + r * p.codes_stride + c * 8) = to_e4m3x8(x[i], exp2_int(-k));
                if (lane % 16 == 0)
                    p.code_scales[r * blocks + c / 16] = exp2_int(k);
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
    __shared__ float2 s_sum[2][kRowWarps];
    const float inv = 1.f / float(p.width);
    uint32_t turn = 0;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x, turn ^= 1) {
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
        const float2 sums = block_sum2(a, b, s_sum[turn]);
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

// Joins the parts in order, so the sums do not depend on which block came
// first: a block takes 32 columns, its warps every 16th part.
constexpr int kJoinWarps = 16;
__global__ void __launch_bounds__(kJoinWarps * 32) norm_backward_join(const __grid_constant__ NormBackwardParams p) {
    __shared__ float s_sum[kJoinWarps][32];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, c = blockIdx.x * 32 + lane;
    const float *partial = p.partial + int64_t(blockIdx.y) * p.parts * p.width + c;
    float sum = 0.f;
    if (c < p.width)
#pragma unroll 4
        for (uint32_t part = warp; part < p.parts; part += kJoinWarps)
            sum += __ldg(partial + int64_t(part) * p.width);
    s_sum[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < p.width) {
#pragma unroll
        for (int w = 1; w < kJoinWarps; ++w)
            sum += s_sum[w][lane];
        store_param(blockIdx.y == 0 ? p.dweight : p.dbias, p.param_type, c, sum);
    }
}

// Rows of whole chunks (as in norm_forward_row), dx and the column sums in one
// pass over memory.  A block stays and takes every gridDim-th row (or warp
// row), so a thread owns the same columns in all of them: its sums for dweight
// and dbias stay in registers, and each block leaves one part of them.  What a
// thread needs of the rows to come it copies itself into its own slots of
// shared memory, DEPTH - 1 rows ahead, so no barrier guards the copies.
template <uint32_t X, uint32_t DY, int V> struct BackwardSlots {
    static constexpr int kDepth = DY == kFp32 ? 2 : 3;
    static constexpr int kChunk = Raw8<DY>::kBytes + Raw8<X>::kBytes + (X == kE4m3 ? 4 : 0);  // bytes per thread
    static constexpr int kThread = kDepth * V * kChunk;
};

template <uint32_t TYPE> __device__ __forceinline__ void copy_row8(void *slot, uint32_t slot_stride, const uint8_t *src) {
    if constexpr (TYPE == kE4m3) {
        cp_async_8(slot, src);
    } else {
        cp_async_16(slot, src);
        if constexpr (TYPE == kFp32)
            cp_async_16(static_cast<uint8_t *>(slot) + slot_stride, src + 16);
    }
}

template <uint32_t TYPE> __device__ __forceinline__ void slot_row8(const void *slot, uint32_t slot_stride, float (&x)[8]) {
    Raw8<TYPE> r;
    if constexpr (TYPE == kE4m3) {
        r.v = *static_cast<const uint2 *>(slot);
    } else {
        r.v = ld_shared_v4(slot);
        if constexpr (TYPE == kFp32)
            r.v2 = ld_shared_v4(static_cast<const uint8_t *>(slot) + slot_stride);
    }
    unpack8<TYPE>(r, x);
}

template <uint32_t X, uint32_t DY, int V>
__global__ void __launch_bounds__(512) norm_backward_row(const __grid_constant__ NormBackwardParams p, bool warp_rows) {
    using Slots = BackwardSlots<X, DY, V>;
    constexpr int kDepth = Slots::kDepth;
    extern __shared__ __align__(16) uint8_t s_slots[];
    __shared__ float2 s_sum[2][16];
    const uint32_t lane = threadIdx.x % 32, threads = blockDim.x, chunks = p.width / 8;
    const uint32_t t = warp_rows ? lane : threadIdx.x, stride = warp_rows ? 32 : threads;
    const int64_t first = warp_rows ? int64_t(blockIdx.x) * (threads / 32) + threadIdx.x / 32 : int64_t(blockIdx.x);
    const int64_t step = warp_rows ? int64_t(gridDim.x) * (threads / 32) : int64_t(gridDim.x);
    const float inv = 1.f / float(p.width);
    // Slots: per depth and chunk, 16-byte (codes: 8) pieces side by side over the
    // threads, then the scales.
    const uint32_t piece = threads * 16;
    uint8_t *dy_slots = s_slots, *x_slots = dy_slots + kDepth * V * threads * Raw8<DY>::kBytes;
    float *scale_slots = reinterpret_cast<float *>(x_slots + kDepth * V * threads * Raw8<X>::kBytes);
    auto dy_slot = [&](int d, int i) { return dy_slots + (d * V + i) * threads * Raw8<DY>::kBytes + threadIdx.x * 16; };
    auto x_slot = [&](int d, int i) {
        return x_slots + (d * V + i) * threads * Raw8<X>::kBytes + threadIdx.x * (X == kE4m3 ? 8 : 16);
    };
    auto scale_slot = [&](int d, int i) { return scale_slots + (d * V + i) * threads + threadIdx.x; };

    auto copy = [&](int64_t r, int d) {
        if (r < p.rows) {
            const uint8_t *dy = static_cast<const uint8_t *>(p.dy) + r * p.dy_stride * int64_t(element_bytes(DY));
            const uint8_t *x = X == kE4m3 ? p.codes + r * p.codes_stride
                                          : static_cast<const uint8_t *>(p.x) + r * p.x_stride * int64_t(element_bytes(X));
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const uint32_t c = t + i * stride;
                if (c < chunks) {
                    copy_row8<DY>(dy_slot(d, i), piece, dy + c * Raw8<DY>::kBytes);
                    copy_row8<X>(x_slot(d, i), piece, x + c * Raw8<X>::kBytes);
                    if constexpr (X == kE4m3)
                        cp_async_4(scale_slot(d, i), p.code_scales + r * p.code_scales_stride + c / 16 * p.scale_col_stride);
                }
            }
        }
        cp_async_commit();
    };

    float dw[V][8], db[V][8], w[V][8];
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dw[i][e] = db[i][e] = 0.f;
            w[i][e] = 1.f;
        }
        if (p.weight != nullptr && t + i * stride < chunks)
            load_param8(p.weight, p.param_type, (t + i * stride) * 8, w[i]);
    }
#pragma unroll
    for (int d = 0; d < kDepth - 1; ++d)
        copy(first + d * step, d);
    int slot = 0, turn = 0;
    float rstd = 0.f, mean = 0.f;
    if (first < p.rows) {
        rstd = __ldg(p.rstd + first);
        if (X != kE4m3)
            mean = __ldg(p.mean + first);
    }
    for (int64_t r = first; r < p.rows; r += step, turn ^= 1) {
        cp_async_wait<kDepth - 2>();
        const float r_rstd = rstd, r_mean = mean;
        if (r + step < p.rows) {
            rstd = __ldg(p.rstd + r + step);
            if (X != kE4m3)
                mean = __ldg(p.mean + r + step);
        }
        // The normalised value is x * up + shift.
        auto values = [&](int i, float (&g)[8], float (&h)[8]) {
            slot_row8<DY>(dy_slot(slot, i), piece, g);
            slot_row8<X>(x_slot(slot, i), piece, h);
            const float up = X == kE4m3 ? *scale_slot(slot, i) : r_rstd;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                h[e] = X == kE4m3 ? h[e] * up : (h[e] - r_mean) * up;
        };
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (t + i * stride < chunks) {
                float g[8], h[8];
                values(i, g, h);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    dw[i][e] += g[e] * h[e];
                    db[i][e] += g[e];
                    const float gw = g[e] * w[i][e];
                    a += gw;
                    b += gw * h[e];
                }
            }
        const float2 sums = warp_rows ? lanes_sum2(a, b) : block_sum2(a, b, s_sum[turn]);
        if (p.dx != nullptr) {
            const float c1 = sums.x * inv, c2 = sums.y * inv;
            uint8_t *dx = static_cast<uint8_t *>(p.dx) + r * p.width * int64_t(element_bytes(DY));
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (t + i * stride < chunks) {
                    float g[8], h[8];
                    values(i, g, h);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        g[e] = r_rstd * (g[e] * w[i][e] - c1 - h[e] * c2);
                    store_row8<DY>(dx + (t + i * stride) * Raw8<DY>::kBytes, g);
                }
        }
        // This row's slots were read by this thread alone, so they can be refilled
        // without a barrier once kDepth - 1 others are ahead of them.
        const int refill = slot == 0 ? kDepth - 1 : slot - 1;
        copy(r + (kDepth - 1) * step, refill);
        slot = slot + 1 == kDepth ? 0 : slot + 1;
    }
    if (p.dweight == nullptr)
        return;
    float *part[2] = {p.partial + int64_t(blockIdx.x) * p.width, p.partial + int64_t(p.parts + blockIdx.x) * p.width};
    if (!warp_rows) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (const uint32_t c = t + i * stride; c < chunks) {
                store_row8<kFp32>(part[0] + c * 8, dw[i]);
                store_row8<kFp32>(part[1] + c * 8, db[i]);
            }
        return;
    }
    // Warp rows: the block's warps hold sums of the same columns.
    cp_async_wait<0>();
    float *sums = reinterpret_cast<float *>(s_slots);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (const uint32_t c = t + i * stride; c < chunks) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    sums[threadIdx.x / 32 * p.width + c * 8 + e] = which == 0 ? dw[i][e] : db[i][e];
            }
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < p.width; c += threads) {
            float sum = 0.f;
            for (uint32_t g = 0; g < threads / 32; ++g)
                sum += sums[g * p.width + c];
            part[which][c] = sum;
        }
    }
}

uint32_t row_grid(int64_t rows, int num_sms) {
    return uint32_t(rows < int64_t(num_sms) * 8 ? rows : int64_t(num_sms) * 8);
}

// Whether norm_forward_row's vector accesses are on their boundaries.
bool whole_chunks(const NormForwardParams &p) {
    const uint32_t in = p.in_type == kE4m3 ? 8 : 16;
    if (p.width % 8 != 0 || p.width > 8 * 4 * 1024 || !on_boundary(p.x, in) ||
        p.x_stride * element_bytes(p.in_type) % in != 0 || !on_boundary(p.weight, 16) || !on_boundary(p.bias, 16))
        return false;
    return p.in_type != kE4m3 || (p.hidden % 8 == 0 && p.block % 8 == 0);
}

template <uint32_t IN, uint32_t OUT, int V>
void forward_row(const NormForwardParams &p, cudaStream_t stream) {
    const uint32_t chunks = p.width / 8;
    const bool warp_rows = chunks <= 32 * V;
    const uint32_t threads = warp_rows ? 128 : ((chunks + V - 1) / V + 31) / 32 * 32;
    const int64_t grid = warp_rows ? (p.rows + 3) / 4 : p.rows;
    norm_forward_row<IN, OUT, V><<<uint32_t(grid), threads, 0, stream>>>(p, warp_rows);
}

template <uint32_t IN, uint32_t OUT> void forward(const NormForwardParams &p, int num_sms, cudaStream_t stream) {
    if (whole_chunks(p)) {
        const uint32_t chunks = p.width / 8;
        // By the width alone, so a row's bits do not depend on its batch.
        if (chunks <= 32)
            forward_row<IN, OUT, 1>(p, stream);
        else if (chunks <= 64)
            forward_row<IN, OUT, 2>(p, stream);
        else
            forward_row<IN, OUT, 4>(p, stream);
        return;
    }
    norm_forward_any<IN, OUT><<<row_grid(p.rows, num_sms), kRowThreads, 0, stream>>>(p);
}

// How norm_backward_row takes a call; threads == 0: it cannot, and the kernels
// for any width, stride and alignment do.
struct BackwardPlan {
    uint32_t threads, grid, shared;
    int vectors;
    bool warp_rows;
};

BackwardPlan backward_plan(const NormBackwardParams &p, int num_sms) {
    BackwardPlan plan{};
    const bool fp8 = p.keep == kKeepFp8;
    const uint32_t dy_bytes = element_bytes(p.dy_type), x_bytes = fp8 ? 1 : dy_bytes, x_boundary = fp8 ? 8 : 16;
    const void *x = fp8 ? static_cast<const void *>(p.codes) : p.x;
    const int64_t x_stride = fp8 ? p.codes_stride : p.x_stride;
    if (p.width % 8 != 0 || !on_boundary(p.dy, 16) || p.dy_stride * dy_bytes % 16 != 0 || !on_boundary(x, x_boundary) ||
        x_stride * x_bytes % x_boundary != 0 || !on_boundary(p.weight, 16))
        return plan;
    const uint32_t chunks = p.width / 8;
    plan.vectors = chunks <= 32 ? 1 : chunks <= 64 ? 2 : 4;
    plan.warp_rows = chunks <= 32u * plan.vectors;
    const uint32_t threads = plan.warp_rows ? 256 : ((chunks + plan.vectors - 1) / plan.vectors + 31) / 32 * 32;
    const uint32_t depth = p.dy_type == kFp32 ? 2 : 3;
    plan.shared = threads * plan.vectors * depth * (8 * (dy_bytes + x_bytes) + (fp8 ? 4 : 0));
    if (plan.warp_rows)
        plan.shared = std::max(plan.shared, threads / 32 * p.width * 4);
    if (threads > 512 || plan.shared > 200 * 1024)
        return plan;
    plan.threads = threads;
    const int64_t groups = plan.warp_rows ? (p.rows + threads / 32 - 1) / (threads / 32) : p.rows;
    const uint32_t resident = std::max(1u, std::min({228u * 1024 / (plan.shared + 2048), 65536u / (threads * 128), 8u}));
    plan.grid = uint32_t(std::min<int64_t>(groups, int64_t(num_sms) * resident));
    return plan;
}

template <uint32_t X, uint32_t DY, int V>
cudaError_t backward_row(const NormBackwardParams &p, const BackwardPlan &plan, cudaStream_t stream) {
    const cudaError_t rc =
        cudaFuncSetAttribute(norm_backward_row<X, DY, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (rc == cudaSuccess)
        norm_backward_row<X, DY, V><<<plan.grid, plan.threads, plan.shared, stream>>>(p, plan.warp_rows);
    return rc;
}

template <uint32_t X, uint32_t DY>
cudaError_t backward(const NormBackwardParams &p, int num_sms, cudaStream_t stream) {
    const BackwardPlan plan = backward_plan(p, num_sms);
    cudaError_t rc = cudaSuccess;
    if (plan.threads != 0) {
        rc = plan.vectors == 1   ? backward_row<X, DY, 1>(p, plan, stream)
             : plan.vectors == 2 ? backward_row<X, DY, 2>(p, plan, stream)
                                 : backward_row<X, DY, 4>(p, plan, stream);
    } else {
        if (p.dx != nullptr)
            norm_backward_rows_any<X, DY><<<row_grid(p.rows, num_sms), kRowThreads, 0, stream>>>(p);
        if (p.dweight != nullptr)
            norm_backward_columns_any<X, DY><<<dim3((p.width + 31) / 32, p.parts), kRowThreads, 0, stream>>>(p);
    }
    if (rc == cudaSuccess && p.dweight != nullptr)
        norm_backward_join<<<dim3((p.width + 31) / 32, 2), kJoinWarps * 32, 0, stream>>>(p);
    return rc;
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
    const BackwardPlan plan = backward_plan(p, num_sms);
    if (plan.threads != 0)
        return plan.grid;
    const int64_t want = int64_t(num_sms) * 4 * 32 / p.width + 1, most = (p.rows + 31) / 32;
    return uint32_t(want < most ? want : most);
}

cudaError_t launch_norm_backward(const NormBackwardParams &p, int num_sms, cudaStream_t stream) {
    const bool fp8 = p.keep == kKeepFp8;
    cudaError_t rc;
    if (p.dy_type == kBf16)
        rc = fp8 ? backward<kE4m3, kBf16>(p, num_sms, stream) : backward<kBf16, kBf16>(p, num_sms, stream);
    else if (p.dy_type == kFp16)
        rc = fp8 ? backward<kE4m3, kFp16>(p, num_sms, stream) : backward<kFp16, kFp16>(p, num_sms, stream);
    else
        rc = fp8 ? backward<kE4m3, kFp32>(p, num_sms, stream) : backward<kFp32, kFp32>(p, num_sms, stream);
    return rc == cudaSuccess ? cudaGetLastError() : rc;
}

} // namespace engram
