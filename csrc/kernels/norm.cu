// Layer norm over rows, forward and backward (sm_100a).
//
// Forward, per row: mean = sum x / N, r = 1 / sqrt(sum (x - mean)^2 / N + eps),
// h = (x - mean) r, y = h w + b.  Backward, with g = dy w: dx = r (g - mean(g) -
// h mean(g h)); per column: dw = sum dy h, db = sum dy.  All sums are fp32.
// The variance is the corrected two-pass form: with d = x - m for the first
// pass's mean m, sum d (zero but for m's rounding) corrects both mean and
// variance, so a large common offset of a row costs no digits as long as m and
// the correction are taken off one after the other: their sum rounds.
#include <algorithm>

#include "readout.h"
#include "rowmath.cuh"
#include "tensor.cuh"

namespace engram {

namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;

// A row's mean m + shift for the backward pass: the sum rounded to fp32, and
// what that rounding left (exactly).  With the rounded sum alone, dweight of fp32
// rows at 4096 + N(0, 1) was 1.2e-4 of its norm off.
__device__ __forceinline__ void keep_mean(const NormForwardParams &p, int64_t r, float m, float shift) {
    const float mean = m + shift, second = mean - m;
    p.mean[r] = mean;
    p.shift[r] = (m - (mean - second)) + (shift - second);
}

// 1 / sqrt(variance + eps).  The variance may round to below zero, and is NaN
// where it and its correction overflow fp32: then rstd is NaN as well (fmaxf
// would make it that of a row without variance).
__device__ __forceinline__ float row_rstd(float variance, float eps) {
    return 1.f / sqrtf((variance < 0.f ? 0.f : variance) + eps);
}

// The scale of a block of normalised values.  Where rstd is infinite (a variance
// that underflowed, and no eps) or NaN, none of a row's values is finite: scale
// 1, and 2^-k as NaN makes every code NaN, where the conversion would saturate.
__device__ __forceinline__ BlockScale kept_scale(float amax, float rstd) {
    const BlockScale s = block_scale(rstd <= FLT_MAX ? amax : 0.f);
    return {s.up, fmaf(rstd, 0.f, s.down)};
}

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
// times (twice from cache).  What takes it: rows past 16384 columns, and codes
// whose rows, entries or scale blocks are not whole vectors.  4096 x 20001 bf16:
// 325 us, 1.0 TB/s.
template <uint32_t IN, uint32_t OUT>
__global__ void __launch_bounds__(kRowThreads) norm_forward_any(const __grid_constant__ NormForwardParams p) {
    __shared__ WarpSums s_sum[2];
    clear_sums(s_sum[0]);
    clear_sums(s_sum[1]);
    __syncthreads();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const float inv = 1.f / float(p.width);
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const RowReader<IN> x(p, r);
        float a = 0.f, b = 0.f;
        for (uint32_t c = threadIdx.x; c < p.width; c += kRowThreads)
            a += x(c);
        float mean = block_sum(a, s_sum[0]) * inv;
        a = 0.f;
        for (uint32_t c = threadIdx.x; c < p.width; c += kRowThreads) {
            const float d = x(c) - mean;
            a += d;
            b += d * d;
        }
        const float2 sums = block_sum2(a, b, s_sum[1]);
        const float shift = sums.x * inv;
        const float rstd = row_rstd(sums.y * inv - shift * shift, p.eps);
        if (threadIdx.x == 0) {
            if (p.keep == kKeepStats)
                keep_mean(p, r, mean, shift);
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
                    h[i] = (x(c) - mean - shift) * rstd;
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
                const BlockScale scale = kept_scale(lanes_max(amax), rstd);
                uint8_t *codes = p.codes + r * p.codes_stride;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t c = blk * kCheckpointBlock + i * 32 + lane;
                    if (c < p.width)
                        codes[c] = to_e4m3(h[i] * scale.down);
                }
                if (lane == 0)
                    p.code_scales[r * blocks + blk] = scale.up;
            }
        }
    }
}

// Rows of whole 8-value chunks on vector boundaries.  A warp holds 32 V adjacent
// chunks of its row, lane l those with l = c % 32, so all of a thread's offsets
// are constants; FULL: every thread has V of them.  A row takes a block of
// warps or, with at most 32 V chunks, one warp of a block.  Blocks stay and
// take every gridDim-th row (warp row).  One thread copies the rows to come
// into a ring in shared memory by bulk copies (per-thread copies of 4 and 8
// bytes kept the load/store unit busy two thirds of the time).
constexpr int ring_depth(uint32_t type) { return type == kFp32 ? 2 : 3; }
constexpr uint64_t kWaitNs = 2000000000ull;  // far above any legal wait
constexpr int kMaxWarps = 16;

struct RowShare {
    uint32_t row, step, chunk, group;  // first row, rows to the next, first chunk, ring
    bool leader;                       // issues its ring's copies
    __device__ __forceinline__ RowShare(bool warp_rows, int vectors) {
        const uint32_t warp = threadIdx.x / 32, warps = blockDim.x / 32;
        row = warp_rows ? blockIdx.x * warps + warp : blockIdx.x;
        step = warp_rows ? gridDim.x * warps : gridDim.x;
        chunk = threadIdx.x % 32 + (warp_rows ? 0 : warp * 32 * vectors);
        group = warp_rows ? warp : 0;
        leader = warp_rows ? threadIdx.x % 32 == 0 : threadIdx.x == 0;
    }
};

// A wait that ran out: reported, and the ring's other copies may still land
// before the block goes.
__device__ __forceinline__ void give_up(uint64_t *full, int depth, uint32_t slot, uint32_t phase, bool leader, uint32_t *fault) {
    st_release_sys_u32(fault, kPipelineTimeout);
    if (leader)
        for (uint32_t d = 0; d < uint32_t(depth); ++d)
            mbar_wait_often(&full[d], d >= slot ? phase : phase ^ 1, kWaitNs);
}

// The row is read once and held in registers between the two sums and the
// output.  Sixteen lanes hold a checkpoint block, so its largest value takes
// four shuffles.  Four chunks per thread: with two, the two sums (a barrier and
// ten shuffles each) were shared by half as many values.  8192 x 12288 bf16 with
// 8 bits kept: 102 us, 4.9 TB/s; 4096 x 6144 bf16: 24.8 us, 4.1 TB/s; from e4m3
// rows 26.1 us, 2.9 TB/s (33.1 kept).  Bound by latency at few warps: 80 registers
// allow 24 per SM, and with them issue slots are free 41% of the time while warps
// wait for loads from L1 and shared memory (37% of their time), for the latency of
// the instruction before (17%) and at barriers (8%).  64 registers and 30
// warps spilled and were 4-8% slower.
template <uint32_t IN, uint32_t OUT, uint32_t PARAM, int V, bool FULL, bool FP8, int T>
__global__ void __launch_bounds__(T, T > 384 ? 1 : 768 / T)
    norm_forward_row(const __grid_constant__ NormForwardParams p, bool warp_rows) {
    constexpr int kDepth = ring_depth(IN);
    extern __shared__ __align__(16) uint8_t s_ring[];
    __shared__ WarpSums s_sum[2];
    __shared__ uint64_t s_full[kMaxWarps][kDepth];
    const RowShare share(warp_rows, V);
    clear_sums(s_sum[0]);
    clear_sums(s_sum[1]);
    if (share.leader) {
        for (int d = 0; d < kDepth; ++d)
            mbar_init(&s_full[share.group][d], 1);
        fence_mbar_init();
    }
    __syncthreads();
    const uint32_t chunks = p.width / 8, rows = uint32_t(p.rows), lane = threadIdx.x % 32;
    const float inv = 1.f / float(p.width);
    const uint32_t row_bytes = chunks * Raw8<IN>::kBytes;
    uint8_t *ring = s_ring + share.group * kDepth * row_bytes;
    const uint32_t x_slot = smem_addr(ring) + share.chunk * Raw8<IN>::kBytes;
    const auto there = [&](int i) { return FULL || share.chunk + i * 32 < chunks; };

    const int64_t x_step = share.step * p.x_stride * int64_t(element_bytes(IN));
    const uint8_t *x_at = static_cast<const uint8_t *>(p.x) + share.row * p.x_stride * int64_t(element_bytes(IN));
    uint32_t copied = share.row;
    auto copy = [&](uint32_t slot) {  // the leader's
        if (copied < rows) {
            mbar_arrive_expect_tx(&s_full[share.group][slot], row_bytes);
            bulk_load(ring + slot * row_bytes, x_at, row_bytes, &s_full[share.group][slot]);
        }
        copied += share.step;
        x_at += x_step;
    };
    if (share.leader)
        for (int d = 0; d < kDepth; ++d)
            copy(d);
    const float *scale_at = IN == kE4m3 ? p.scales + share.row * p.scale_row_stride : nullptr;
    uint32_t pack[V];
    float next_scale[V];
    auto load_scales = [&] {
#pragma unroll
        for (int i = 0; i < V; ++i)
            next_scale[i] = there(i) ? __ldg(scale_at + pack[i] * p.scale_col_stride) : 0.f;
        scale_at += share.step * p.scale_row_stride;
    };
    if constexpr (IN == kE4m3) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const uint32_t column = (share.chunk + i * 32) * 8, entry = column / p.hidden;
            pack[i] = entry * p.packs + (column - entry * p.hidden) / p.block;
        }
        if (share.row < rows)
            load_scales();
    }
    uint32_t slot = 0, phase = 0;
    uint8_t *y_at = static_cast<uint8_t *>(p.y) + int64_t(share.row) * p.width * element_bytes(OUT) + share.chunk * Raw8<OUT>::kBytes;
    const int64_t y_step = int64_t(share.step) * p.width * element_bytes(OUT);
    const uint8_t *w_at = static_cast<const uint8_t *>(p.weight) + share.chunk * Raw8<PARAM>::kBytes;
    const uint8_t *b_at = static_cast<const uint8_t *>(p.bias) + share.chunk * Raw8<PARAM>::kBytes;
    const uint32_t blocks = (p.width + kCheckpointBlock - 1) / kCheckpointBlock;
    uint8_t *code_at = p.codes + share.row * p.codes_stride + share.chunk * 8;
    float *code_scale_at = p.code_scales + int64_t(share.row) * blocks + share.chunk / 16;
    const bool affine = p.weight != nullptr, shifted = p.bias != nullptr;
    for (uint32_t r = share.row; r < rows; r += share.step) {
        if (!mbar_wait_often(&s_full[share.group][slot], phase, kWaitNs)) {
            give_up(s_full[share.group], kDepth, slot, phase, share.leader, p.fault);
            return;
        }
        Pair x[V][4];
        Pair a = both(0.f), b = both(0.f);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (there(i)) {
                load_shared8<IN>(x_slot + slot * row_bytes + i * 32 * Raw8<IN>::kBytes, x[i]);
                if constexpr (IN == kE4m3) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x[i][e] = mul2(x[i][e], both(next_scale[i]));
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    a = add2(a, x[i][e]);
            }
        if constexpr (IN == kE4m3)
            if (r + share.step < rows)
                load_scales();
        // Every thread of the row has read its slot when the first sum is there.
        const float mean = (warp_rows ? lanes_sum(total(a)) : block_sum(total(a), s_sum[0])) * inv;
        if (share.leader)
            copy(slot);
        slot = slot + 1 == kDepth ? 0 : slot + 1;
        phase ^= slot == 0 ? 1 : 0;
        const Pair minus_mean = both(-mean);
        a = both(0.f);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (there(i)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[i][e] = add2(x[i][e], minus_mean);
                    a = add2(a, x[i][e]);
                    b = fma2(x[i][e], x[i][e], b);
                }
            }
        const float2 sums = warp_rows ? lanes_sum2(total(a), total(b)) : block_sum2(total(a), total(b), s_sum[1]);
        const float shift = sums.x * inv;
        const float rstd = row_rstd(sums.y * inv - shift * shift, p.eps);
        if (share.leader && p.keep != kKeepNothing) {
            if (p.keep == kKeepStats)
                keep_mean(p, r, mean, shift);
            p.rstd[r] = rstd;
        }
        const Pair minus_shift = both(-shift), up = both(rstd);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float amax = 0.f;
            if (there(i)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // Finite, or in none of a row: an infinity makes the mean NaN or infinite, and rstd
                    // may be infinite.
                    x[i][e] = mul2(add2(x[i][e], minus_shift), up);
                    if constexpr (FP8)
                        amax = largest3(amax, parts(x[i][e]).x, parts(x[i][e]).y);
                }
                if (affine) {
                    Pair v[4], w[4];
                    load_param8<PARAM>(w_at + i * 32 * Raw8<PARAM>::kBytes, w);
                    if (shifted) {
                        load_param8<PARAM>(b_at + i * 32 * Raw8<PARAM>::kBytes, v);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            v[e] = fma2(x[i][e], w[e], v[e]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            v[e] = mul2(x[i][e], w[e]);
                    }
                    store_row8<OUT>(y_at + i * 32 * Raw8<OUT>::kBytes, v);
                } else {
                    store_row8<OUT>(y_at + i * 32 * Raw8<OUT>::kBytes, x[i]);
                }
            }
            if constexpr (FP8) {
                const BlockScale unit = kept_scale(lanes_max<16>(amax), rstd);
                if (there(i)) {
                    *reinterpret_cast<uint2 *>(code_at + i * 256) = to_e4m3x8(x[i], unit.down);
                    if (lane % 16 == 0)
                        code_scale_at[i * 2] = unit.up;
                }
            }
        }
        y_at += y_step;
        if constexpr (FP8) {
            code_at += share.step * p.codes_stride;
            code_scale_at += int64_t(share.step) * blocks;
        }
    }
}

// Rows of 16- and 32-bit values of any width up to 16384 and any alignment, one
// read: as above with single values for chunks, so every access is one element
// (64 or 128 bytes of a warp together).  E is a multiple of four: a warp's
// columns are whole checkpoint blocks.  4096 x 4097 bf16: 43 us, 1.5 TB/s, 8
// bits kept 60 us: an access moves one element, and a thread's sixteen spill 70-90
// bytes of 64 registers where codes are kept (with eight elements per thread the
// sums' share made it a third slower; reading the row three times 45% slower).
template <uint32_t IN, uint32_t PARAM, int E, bool FP8, int T0>
__global__ void __launch_bounds__(T0, 1024 / T0)
    norm_forward_elements(const __grid_constant__ NormForwardParams p, bool warp_rows) {
    using T = typename Element<IN>::T;
    using W = typename Element<PARAM>::T;
    __shared__ RowSums<T0> s_sum[2];
    const RowShare share(warp_rows, E);
    s_sum[0].clear();
    s_sum[1].clear();
    __syncthreads();
    const uint32_t lane = threadIdx.x % 32, rows = uint32_t(p.rows), c0 = share.chunk;
    const float inv = 1.f / float(p.width);
    const uint32_t blocks = (p.width + kCheckpointBlock - 1) / kCheckpointBlock;
    const W *weight = static_cast<const W *>(p.weight), *bias = static_cast<const W *>(p.bias);
    const bool whole = c0 - lane + 32 * E <= p.width;  // this warp's columns all exist
    for (uint32_t r = share.row; r < rows; r += share.step) {
        const T *row = static_cast<const T *>(p.x) + r * p.x_stride;
        T *y = static_cast<T *>(p.y) + int64_t(r) * p.width + c0;
        float x[E], a = 0.f, b = 0.f;
        T raw[E];
        // All in flight: no branch guards a single load.
        if (whole) {
#pragma unroll
            for (int j = 0; j < E; ++j)
                raw[j] = row[c0 + j * 32];
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j)
                raw[j] = row[min(c0 + j * 32, p.width - 1)];
        }
#pragma unroll
        for (int j = 0; j < E; ++j) {
            x[j] = whole || c0 + j * 32 < p.width ? Element<IN>::get(raw[j]) : 0.f;
            a += x[j];
        }
        const float mean = (warp_rows ? lanes_sum(a) : s_sum[0].sum(a)) * inv;
        a = 0.f;
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (whole || c0 + j * 32 < p.width) {
                x[j] -= mean;
                a += x[j];
                b += x[j] * x[j];
            }
        const float2 sums = warp_rows ? lanes_sum2(a, b) : s_sum[1].sum2(a, b);
        const float shift = sums.x * inv;
        const float rstd = row_rstd(sums.y * inv - shift * shift, p.eps);
        if (share.leader && p.keep != kKeepNothing) {
            if (p.keep == kKeepStats)
                keep_mean(p, r, mean, shift);
            p.rstd[r] = rstd;
        }
        float v[E];
#pragma unroll
        for (int j = 0; j < E; ++j) {
            x[j] = whole || c0 + j * 32 < p.width ? (x[j] - shift) * rstd : 0.f;
            v[j] = x[j];
        }
        if (weight != nullptr)
#pragma unroll
            for (int j = 0; j < E; ++j)
                v[j] *= Element<PARAM>::get(__ldg(weight + (whole ? c0 + j * 32 : min(c0 + j * 32, p.width - 1))));
        if (bias != nullptr)
#pragma unroll
            for (int j = 0; j < E; ++j)
                v[j] += Element<PARAM>::get(__ldg(bias + (whole ? c0 + j * 32 : min(c0 + j * 32, p.width - 1))));
        if (whole) {
#pragma unroll
            for (int j = 0; j < E; ++j)
                y[j * 32] = Element<IN>::put(v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (c0 + j * 32 < p.width)
                    y[j * 32] = Element<IN>::put(v[j]);
        }
        if constexpr (FP8) {
            uint8_t *codes = p.codes + r * p.codes_stride + c0;
#pragma unroll
            for (int q = 0; q < E / 4; ++q) {
                const float *h = x + q * 4;
                const BlockScale unit =
                    kept_scale(lanes_max(largest3(largest3(0.f, h[0], h[1]), h[2], h[3])), rstd);
                const uint32_t c = c0 - lane + q * kCheckpointBlock;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j * 32 + lane < p.width)
                        codes[(q * 4 + j) * 32] = to_e4m3(h[j] * unit.down);
                if (lane == 0 && c < p.width)
                    p.code_scales[int64_t(r) * blocks + c / kCheckpointBlock] = unit.up;
            }
        }
    }
}

// What a row's normalised values take beside its elements (exact rows).
struct RowStats {
    float mean = 0.f, shift = 0.f, rstd = 0.f;
    __device__ __forceinline__ RowStats(const NormBackwardParams &p, int64_t r) {
        if (p.keep != kKeepStats)
            return;
        mean = p.mean[r];
        shift = p.shift != nullptr ? p.shift[r] : 0.f;
        rstd = p.rstd[r];
    }
};

// A normalised value of the backward pass.
template <uint32_t X>
__device__ __forceinline__ float kept_value(const NormBackwardParams &p, int64_t r, uint32_t c, const RowStats &row) {
    if (X == kE4m3)
        return Element<kE4m3>::get(p.codes[r * p.codes_stride + c]) *
               p.code_scales[r * p.code_scales_stride + c / kCheckpointBlock * p.scale_col_stride];
    else
        return (Element<X>::get(static_cast<const typename Element<X>::T *>(p.x)[r * p.x_stride + c]) - row.mean -
                row.shift) *
               row.rstd;
}

template <uint32_t X, uint32_t DY>
__global__ void __launch_bounds__(kRowThreads) norm_backward_rows_any(const __grid_constant__ NormBackwardParams p) {
    __shared__ WarpSums s_sum[2];
    clear_sums(s_sum[0]);
    clear_sums(s_sum[1]);
    __syncthreads();
    const float inv = 1.f / float(p.width);
    uint32_t turn = 0;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x, turn ^= 1) {
        const auto *dy = static_cast<const typename Element<DY>::T *>(p.dy) + r * p.dy_stride;
        auto *dx = static_cast<typename Element<DY>::T *>(p.dx) + r * p.width;
        const RowStats row(p, r);
        float a = 0.f, b = 0.f;
        for (uint32_t c = threadIdx.x; c < p.width; c += kRowThreads) {
            float g = Element<DY>::get(dy[c]);
            if (p.weight != nullptr)
                g *= load_param(p.weight, p.param_type, c);
            a += g;
            b += g * kept_value<X>(p, r, c, row);
        }
        const float2 sums = block_sum2(a, b, s_sum[turn]);
        const float c1 = sums.x * inv, c2 = sums.y * inv, rstd = p.rstd[r];
        for (uint32_t c = threadIdx.x; c < p.width; c += kRowThreads) {
            float g = Element<DY>::get(dy[c]);
            if (p.weight != nullptr)
                g *= load_param(p.weight, p.param_type, c);
            dx[c] = Element<DY>::put(rstd * (g - c1 - kept_value<X>(p, r, c, row) * c2));
        }
    }
}

// Past 12288 columns of what norm_backward_row does not take: dx by a block per
// row, then column sums of dy and dy h over one part of the rows: a block takes
// 32 columns, its warps every eighth row of the part.  4096 x 20001 bf16 exact: 646
// us, 0.76 TB/s (rows are read three times).
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
            dw += g * kept_value<X>(p, r, c, RowStats(p, r));
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
    wait_for_previous();
    if (c < p.width)
#pragma unroll 8
        for (uint32_t part = warp; part < p.parts; part += kJoinWarps)
            sum += partial[int64_t(part) * p.width];
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
// pass over memory.  A thread owns the same columns in all rows of its block:
// its sums for dweight and dbias stay in registers, and each block leaves one
// part of them.  A ring slot holds dy's row, then the kept one, each with room
// for a chunk in every place; what no chunk fills is zero and adds nothing.
// Both passes over a row read it from the ring: holding it in registers beside
// the sums left one block per SM.  8192 x 12288 from 8 bits: 99 us, 5.1 TB/s
// (0.78 of a copy's rate); 4096 x 6144 bf16 exact: 35 us, 4.3 TB/s, 4-5 us of
// them the join of the parts.  Bound by latency at few warps: 154-168 registers
// leave 12 per SM at widths of 6144 and 12288, 7 to 9 between 6152 and 9216 (4096
// rows from 8 bits: 6144 34.7 us, 7168 45.4, 8192 46.4, 9216 53.6), and issue slots
// are free half of the time.  Past 12288 columns 512 threads of 128 registers spill
// 90-150 bytes.
template <uint32_t X, uint32_t DY, uint32_t PARAM, int V, int T>
__global__ void __launch_bounds__(T) norm_backward_row(const __grid_constant__ NormBackwardParams p, bool warp_rows) {
    constexpr int kDepth = ring_depth(DY);
    extern __shared__ __align__(16) uint8_t s_ring[];
    __shared__ WarpSums s_sum[2];
    __shared__ uint64_t s_full[kMaxWarps][kDepth];
    const RowShare share(warp_rows, V);
    clear_sums(s_sum[0]);
    clear_sums(s_sum[1]);
    if (share.leader) {
        for (int d = 0; d < kDepth; ++d)
            mbar_init(&s_full[share.group][d], 1);
        fence_mbar_init();
    }
    const uint32_t chunks = p.width / 8, rows = uint32_t(p.rows);
    const float inv = 1.f / float(p.width);
    const uint32_t places = (warp_rows ? 32 : blockDim.x) * V;
    const uint32_t x_offset = places * Raw8<DY>::kBytes, slot_bytes = places * (Raw8<DY>::kBytes + Raw8<X>::kBytes);
    const uint32_t groups = warp_rows ? blockDim.x / 32 : 1;
    for (uint32_t at = threadIdx.x * 16; at < groups * kDepth * slot_bytes; at += blockDim.x * 16)
        *reinterpret_cast<uint4 *>(s_ring + at) = make_uint4(0, 0, 0, 0);
    fence_async_shared();
    __syncthreads();
    uint8_t *ring = s_ring + share.group * kDepth * slot_bytes;
    const uint32_t dy_slot = smem_addr(ring) + share.chunk * Raw8<DY>::kBytes;
    const uint32_t x_slot = smem_addr(ring) + x_offset + share.chunk * Raw8<X>::kBytes;
    const auto there = [&](int i) { return share.chunk + i * 32 < chunks; };

    const uint8_t *dy_at = static_cast<const uint8_t *>(p.dy) + share.row * p.dy_stride * int64_t(element_bytes(DY));
    const uint8_t *x_at = X == kE4m3 ? p.codes + share.row * p.codes_stride
                                     : static_cast<const uint8_t *>(p.x) + share.row * p.x_stride * int64_t(element_bytes(X));
    const int64_t dy_step = share.step * p.dy_stride * int64_t(element_bytes(DY));
    const int64_t x_step = X == kE4m3 ? share.step * p.codes_stride : share.step * p.x_stride * int64_t(element_bytes(X));
    const uint32_t dy_bytes = chunks * Raw8<DY>::kBytes, x_bytes = chunks * Raw8<X>::kBytes;
    uint32_t copied = share.row;
    auto copy = [&](uint32_t slot) {  // the leader's
        if (copied < rows) {
            uint64_t *full = &s_full[share.group][slot];
            mbar_arrive_expect_tx(full, dy_bytes + x_bytes);
            bulk_load(ring + slot * slot_bytes, dy_at, dy_bytes, full);
            bulk_load(ring + slot * slot_bytes + x_offset, x_at, x_bytes, full);
        }
        copied += share.step;
        dy_at += dy_step;
        x_at += x_step;
    };
    if (share.leader)
        for (int d = 0; d < kDepth - 1; ++d)
            copy(d);

    Pair dw[V][4], db[V][4], w[V][4];
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            dw[i][e] = db[i][e] = both(0.f);
            w[i][e] = both(1.f);
        }
        if (p.weight != nullptr && there(i))
            load_param8<PARAM>(static_cast<const uint8_t *>(p.weight) + (share.chunk + i * 32) * Raw8<PARAM>::kBytes, w[i]);
    }
    const float *scale_at =
        X == kE4m3 ? p.code_scales + share.row * p.code_scales_stride + share.chunk / 16 * p.scale_col_stride : nullptr;
    float next_rstd = 0.f, next_mean = 0.f, next_shift = 0.f, next_scale[V];
    auto load_stats = [&](uint32_t r) {
        next_rstd = __ldg(p.rstd + r);
        if constexpr (X == kE4m3) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                next_scale[i] = there(i) ? __ldg(scale_at + i * 2 * p.scale_col_stride) : 0.f;
            scale_at += share.step * p.code_scales_stride;
        } else {
            next_mean = __ldg(p.mean + r);
            if (p.shift != nullptr)
                next_shift = __ldg(p.shift + r);
        }
    };
    if (share.row < rows)
        load_stats(share.row);
    uint32_t slot = 0, phase = 0, turn = 0, refill = kDepth - 1;
    uint8_t *dx_at = static_cast<uint8_t *>(p.dx) + int64_t(share.row) * p.width * element_bytes(DY) + share.chunk * Raw8<DY>::kBytes;
    const int64_t dx_step = int64_t(share.step) * p.width * element_bytes(DY);
    for (uint32_t r = share.row; r < rows; r += share.step, turn ^= 1) {
        const float rstd = next_rstd;
        const Pair minus_mean = both(-next_mean), minus_shift = both(-next_shift);
        float scale[V];
        if constexpr (X == kE4m3) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                scale[i] = next_scale[i];
        }
        if (r + share.step < rows)
            load_stats(r + share.step);
        if (!mbar_wait_often(&s_full[share.group][slot], phase, kWaitNs)) {
            give_up(s_full[share.group], kDepth, slot, phase, share.leader, p.fault);
            return;
        }
        auto values = [&](int i, Pair (&g)[4], Pair (&h)[4]) {
            load_shared8<DY>(dy_slot + slot * slot_bytes + i * 32 * Raw8<DY>::kBytes, g);
            load_shared8<X>(x_slot + slot * slot_bytes + i * 32 * Raw8<X>::kBytes, h);
            const Pair up = both(X == kE4m3 ? scale[i] : rstd);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                h[e] = mul2(X == kE4m3 ? h[e] : add2(add2(h[e], minus_mean), minus_shift), up);
        };
        Pair a = both(0.f), b = both(0.f);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            Pair g[4], h[4];
            values(i, g, h);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                dw[i][e] = fma2(g[e], h[e], dw[i][e]);
                db[i][e] = add2(db[i][e], g[e]);
                g[e] = mul2(g[e], w[i][e]);
                a = add2(a, g[e]);
                b = fma2(g[e], h[e], b);
            }
        }
        const float2 sums = warp_rows ? lanes_sum2(total(a), total(b)) : block_sum2(total(a), total(b), s_sum[turn]);
        // Past the sum every thread is done with the row before this one.
        if (share.leader)
            copy(refill);
        if (p.dx != nullptr) {
            const Pair c1 = both(-sums.x * inv), c2 = both(-sums.y * inv), up = both(rstd);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (there(i)) {
                    Pair g[4], h[4];
                    values(i, g, h);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        g[e] = mul2(fma2(h[e], c2, fma2(g[e], w[i][e], c1)), up);
                    store_row8<DY>(dx_at + i * 32 * Raw8<DY>::kBytes, g);
                }
            dx_at += dx_step;
        }
        refill = slot;
        slot = slot + 1 == kDepth ? 0 : slot + 1;
        phase ^= slot == 0 ? 1 : 0;
    }
    if (p.dweight == nullptr)
        return;
    start_next();
    float *part[2] = {p.partial + int64_t(blockIdx.x) * p.width, p.partial + int64_t(p.parts + blockIdx.x) * p.width};
    if (!warp_rows) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (const uint32_t c = share.chunk + i * 32; c < chunks) {
                store_row8<kFp32>(part[0] + c * 8, dw[i]);
                store_row8<kFp32>(part[1] + c * 8, db[i]);
            }
        return;
    }
    // Warp rows: the block's warps hold sums of the same columns.
    float *sums = reinterpret_cast<float *>(s_ring);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (const uint32_t c = share.chunk + i * 32; c < chunks) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *reinterpret_cast<float2 *>(sums + threadIdx.x / 32 * p.width + c * 8 + e * 2) =
                        parts(which == 0 ? dw[i][e] : db[i][e]);
            }
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < p.width; c += blockDim.x) {
            float sum = 0.f;
            for (uint32_t g = 0; g < blockDim.x / 32; ++g)
                sum += sums[g * p.width + c];
            part[which][c] = sum;
        }
    }
}

// The same for rows of up to 12288 columns of any alignment, by single elements.
// 4096 x 4097 bf16: 62 us, 1.6 TB/s (two passes over the rows took 111 us); a
// branch around each load made it 83 us, from 8 bits 192 us.  Bound by the number
// of accesses, and by spills: 8-36 bytes of 64 registers up to 4096 columns, 240-370
// of 80 past 8192 (8192 x 11111 from 8 bits 286 us, 1.6 TB/s).
template <uint32_t X, uint32_t DY, uint32_t PARAM, int E, int T>
__global__ void __launch_bounds__(T, E == 8 ? 2 : 1) norm_backward_elements(const __grid_constant__ NormBackwardParams p, bool warp_rows) {
    using D = typename Element<DY>::T;
    using K = typename Element<X>::T;
    using W = typename Element<PARAM>::T;
    __shared__ RowSums<T> s_sum[2];
    __shared__ float s_part[8][32 * E];
    const RowShare share(warp_rows, E);
    s_sum[0].clear();
    s_sum[1].clear();
    __syncthreads();
    const uint32_t rows = uint32_t(p.rows), c0 = share.chunk;
    const float inv = 1.f / float(p.width);
    const uint32_t last = p.width - 1;
    float dw[E] = {}, db[E] = {}, w[E];
#pragma unroll
    for (int j = 0; j < E; ++j)
        w[j] = p.weight == nullptr ? 1.f : Element<PARAM>::get(static_cast<const W *>(p.weight)[min(c0 + j * 32, last)]);
    uint32_t turn = 0;
    for (uint32_t r = share.row; r < rows; r += share.step, turn ^= 1) {
        const D *dy = static_cast<const D *>(p.dy) + r * p.dy_stride;
        const K *kept = X == kE4m3 ? reinterpret_cast<const K *>(p.codes) + r * p.codes_stride
                                   : static_cast<const K *>(p.x) + r * p.x_stride;
        D *dx = static_cast<D *>(p.dx) + int64_t(r) * p.width + c0;
        const float rstd = __ldg(p.rstd + r), mean = X == kE4m3 ? 0.f : __ldg(p.mean + r);
        const float shift = X == kE4m3 || p.shift == nullptr ? 0.f : __ldg(p.shift + r);
        D raw_g[E];
        K raw_h[E];
        float scale[E / 4];
#pragma unroll
        for (int j = 0; j < E; ++j) {  // all in flight: no branch guards a load
            const uint32_t c = min(c0 + j * 32, last);
            raw_g[j] = dy[c];
            raw_h[j] = kept[c];
        }
        if constexpr (X == kE4m3) {
            const float *scales = p.code_scales + r * p.code_scales_stride;
#pragma unroll
            for (int q = 0; q < E / 4; ++q)
                scale[q] = scales[min(c0 + q * kCheckpointBlock, last) / kCheckpointBlock * p.scale_col_stride];
        }
        float g[E], h[E], a = 0.f, b = 0.f;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const bool there = c0 + j * 32 < p.width;
            g[j] = there ? Element<DY>::get(raw_g[j]) : 0.f;
            h[j] = X == kE4m3 ? Element<X>::get(raw_h[j]) * scale[j / 4] : (Element<X>::get(raw_h[j]) - mean - shift) * rstd;
            h[j] = there ? h[j] : 0.f;
            dw[j] += g[j] * h[j];
            db[j] += g[j];
            g[j] *= w[j];
            a += g[j];
            b += g[j] * h[j];
        }
        const float2 sums = warp_rows ? lanes_sum2(a, b) : s_sum[turn].sum2(a, b);
        if (p.dx != nullptr) {
            const float c1 = sums.x * inv, c2 = sums.y * inv;
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (c0 + j * 32 < p.width)
                    dx[j * 32] = Element<DY>::put(rstd * (g[j] - c1 - h[j] * c2));
        }
    }
    if (p.dweight == nullptr)
        return;
    start_next();
    float *part[2] = {p.partial + int64_t(blockIdx.x) * p.width, p.partial + int64_t(p.parts + blockIdx.x) * p.width};
    if (!warp_rows) {
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (const uint32_t c = c0 + j * 32; c < p.width) {
                part[0][c] = dw[j];
                part[1][c] = db[j];
            }
        return;
    }
    // Warp rows: the block's warps hold sums of the same columns.
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < E; ++j)
            s_part[threadIdx.x / 32][c0 + j * 32] = which == 0 ? dw[j] : db[j];
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < p.width; c += blockDim.x) {
            float sum = 0.f;
            for (uint32_t w = 0; w < blockDim.x / 32; ++w)
                sum += s_part[w][c];
            part[which][c] = sum;
        }
    }
}

uint32_t row_grid(int64_t rows, int num_sms) {
    return uint32_t(rows < int64_t(num_sms) * 8 ? rows : int64_t(num_sms) * 8);
}

// Whether norm_forward_row's copies and vectors are on their boundaries.
bool whole_chunks(const NormForwardParams &p) {
    const uint32_t size = element_bytes(p.in_type), param = 8 * element_bytes(p.param_type);
    if (p.width % 8 != 0 || p.width > 8 * 4 * 512 || p.width * size % 16 != 0 || !on_boundary(p.x, 16) ||
        p.x_stride * size % 16 != 0 || !on_boundary(p.weight, param) || !on_boundary(p.bias, param))
        return false;
    return p.in_type != kE4m3 || (p.hidden % 8 == 0 && p.block % 8 == 0);
}

// Blocks of a row kernel that fit an SM at once.
uint32_t resident(uint32_t threads, uint32_t registers, uint32_t shared) {
    return std::max(1u, std::min({65536 / (threads * registers), 226 * 1024 / (shared + 1280), 2048 / threads, 16u}));
}

template <uint32_t IN, uint32_t OUT, uint32_t PARAM, int V, bool FULL, int T>
cudaError_t forward_row(const NormForwardParams &p, int num_sms, cudaStream_t stream) {
    const uint32_t chunks = p.width / 8;
    const bool warp_rows = chunks <= 32 * V;
    const uint32_t threads = warp_rows ? 128 : (chunks + 32 * V - 1) / (32 * V) * 32;
    const uint32_t shared = (warp_rows ? 4 : 1) * ring_depth(IN) * p.width * element_bytes(IN);
    const int64_t groups = warp_rows ? (p.rows + 3) / 4 : p.rows;
    const uint32_t grid = uint32_t(std::min<int64_t>(groups, int64_t(num_sms) * resident(threads, T > 384 ? 128 : 80, shared)));
    const auto kernel = p.keep == kKeepFp8 ? norm_forward_row<IN, OUT, PARAM, V, FULL, true, T>
                                           : norm_forward_row<IN, OUT, PARAM, V, FULL, false, T>;
    if (shared > 40 * 1024)
        if (const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(shared));
            rc != cudaSuccess)
            return rc;
    kernel<<<grid, threads, shared, stream>>>(p, warp_rows);
    return cudaSuccess;
}

template <uint32_t IN, uint32_t OUT, uint32_t PARAM>
cudaError_t forward_rows(const NormForwardParams &p, int num_sms, cudaStream_t stream) {
    // By the width alone (and whole_chunks, by alignment), never by the number of rows:
    // a row's bits do not depend on its batch.
    const uint32_t chunks = p.width / 8;
    return chunks <= 32        ? forward_row<IN, OUT, PARAM, 1, false, 128>(p, num_sms, stream)
           : chunks <= 64      ? forward_row<IN, OUT, PARAM, 2, false, 128>(p, num_sms, stream)
           : chunks > 1536     ? forward_row<IN, OUT, PARAM, 4, false, 512>(p, num_sms, stream)
           : chunks % 128 == 0 ? forward_row<IN, OUT, PARAM, 4, true, 384>(p, num_sms, stream)
                               : forward_row<IN, OUT, PARAM, 4, false, 384>(p, num_sms, stream);
}

template <uint32_t IN, uint32_t PARAM, int E, int T>
void forward_elements(const NormForwardParams &p, int num_sms, cudaStream_t stream) {
    const bool warp_rows = p.width <= 32 * E;
    const uint32_t threads = warp_rows ? 128 : (p.width + 32 * E - 1) / (32 * E) * 32;
    const int64_t groups = warp_rows ? (p.rows + 3) / 4 : p.rows;
    const uint32_t grid = uint32_t(std::min<int64_t>(groups, int64_t(num_sms) * resident(threads, 64, 0)));
    if (p.keep == kKeepFp8)
        norm_forward_elements<IN, PARAM, E, true, T><<<grid, threads, 0, stream>>>(p, warp_rows);
    else
        norm_forward_elements<IN, PARAM, E, false, T><<<grid, threads, 0, stream>>>(p, warp_rows);
}

template <uint32_t IN, uint32_t PARAM> void forward_elements(const NormForwardParams &p, int num_sms, cudaStream_t stream) {
    if (p.width <= 256)
        forward_elements<IN, PARAM, 8, 512>(p, num_sms, stream);
    else if (p.width <= 8192)
        forward_elements<IN, PARAM, 16, 512>(p, num_sms, stream);
    else
        forward_elements<IN, PARAM, 16, 1024>(p, num_sms, stream);
}

template <uint32_t IN, uint32_t OUT>
cudaError_t forward(const NormForwardParams &p, int num_sms, cudaStream_t stream) {
    if (IN != kE4m3 && !whole_chunks(p) && p.width <= 16 * 1024) {
        constexpr uint32_t kIn = IN == kE4m3 ? OUT : IN;
        if (p.param_type == kFp32)
            forward_elements<kIn, kFp32>(p, num_sms, stream);
        else
            forward_elements<kIn, kIn>(p, num_sms, stream);
        return cudaGetLastError();
    }
    if (!whole_chunks(p)) {
        norm_forward_any<IN, OUT><<<row_grid(p.rows, num_sms), kRowThreads, 0, stream>>>(p);
        return cudaGetLastError();
    }
    const cudaError_t rc = OUT != kFp32 && p.weight != nullptr && p.param_type == kFp32
                               ? forward_rows<IN, OUT, kFp32>(p, num_sms, stream)
                               : forward_rows<IN, OUT, OUT>(p, num_sms, stream);
    return rc == cudaSuccess ? cudaGetLastError() : rc;
}

// How norm_backward_row takes a call, or norm_backward_elements (`elements` per
// thread); threads == 0: neither can, and the kernels for any width do.
struct BackwardPlan {
    uint32_t threads, grid, shared;
    int vectors, elements;
    bool warp_rows;
};

BackwardPlan backward_plan(const NormBackwardParams &p, int num_sms) {
    BackwardPlan plan{};
    const bool fp8 = p.keep == kKeepFp8;
    const uint32_t dy_bytes = element_bytes(p.dy_type), x_bytes = fp8 ? 1 : dy_bytes, chunks = p.width / 8;
    const void *x = fp8 ? static_cast<const void *>(p.codes) : p.x;
    const int64_t x_stride = fp8 ? p.codes_stride : p.x_stride;
    plan.vectors = chunks <= 32 ? 1 : chunks <= 64 ? 2 : 4;
    plan.warp_rows = chunks <= 32u * plan.vectors;
    plan.threads = plan.warp_rows ? 256 : (chunks + 32 * plan.vectors - 1) / (32 * plan.vectors) * 32;
    plan.shared = plan.threads * plan.vectors * ring_depth(p.dy_type) * 8 * (dy_bytes + x_bytes);
    if (plan.warp_rows)
        plan.shared = std::max(plan.shared, plan.threads / 32 * p.width * 4);
    uint32_t registers = plan.vectors == 4 && plan.threads <= 384 ? 168 : 128;
    const bool boundaries = p.width % 8 == 0 && on_boundary(p.dy, 16) && p.dy_stride * dy_bytes % 16 == 0 &&
                            on_boundary(x, 16) && x_stride * x_bytes % 16 == 0 && p.width * x_bytes % 16 == 0 &&
                            on_boundary(p.weight, p.param_type == kFp32 ? 32 : 16);
    if (!boundaries || plan.threads > 512 || plan.shared > 200 * 1024) {
        if (p.width > 12288)
            return BackwardPlan{};
        plan.elements = p.width > 4096 || (p.width > 256 && p.width <= 512) ? 16 : 8;  // 512: a warp holds a row
        plan.warp_rows = p.width <= 32u * plan.elements;
        plan.threads = plan.warp_rows ? 256 : (p.width + 32 * plan.elements - 1) / (32 * plan.elements) * 32;
        plan.shared = 0;
        registers = plan.elements == 8 ? 64 : plan.threads <= 512 ? 128 : 84;
    }
    const int64_t groups = plan.warp_rows ? (p.rows + plan.threads / 32 - 1) / (plan.threads / 32) : p.rows;
    // Each block leaves a part of the column sums: eight rows for each where there
    // are enough, or the parts would be as much to move and add up as the rows.
    const int64_t most = p.dweight == nullptr ? groups : std::max<int64_t>(2 * num_sms, groups / 8);
    plan.grid = uint32_t(std::min({groups, most, int64_t(num_sms) * resident(plan.threads, registers, plan.shared)}));
    return plan;
}

template <uint32_t X, uint32_t DY, uint32_t PARAM, int V, int T>
cudaError_t backward_row(const NormBackwardParams &p, const BackwardPlan &plan, cudaStream_t stream) {
    const auto kernel = norm_backward_row<X, DY, PARAM, V, T>;
    if (plan.shared > 40 * 1024)
        if (const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(plan.shared));
            rc != cudaSuccess)
            return rc;
    kernel<<<plan.grid, plan.threads, plan.shared, stream>>>(p, plan.warp_rows);
    return cudaSuccess;
}

template <uint32_t X, uint32_t DY, uint32_t PARAM>
cudaError_t backward_rows(const NormBackwardParams &p, const BackwardPlan &plan, cudaStream_t stream) {
    if (plan.elements == 8)
        norm_backward_elements<X, DY, PARAM, 8, 512><<<plan.grid, plan.threads, 0, stream>>>(p, plan.warp_rows);
    else if (plan.elements == 16 && plan.threads <= 512)
        norm_backward_elements<X, DY, PARAM, 16, 512><<<plan.grid, plan.threads, 0, stream>>>(p, plan.warp_rows);
    else if (plan.elements == 16)
        norm_backward_elements<X, DY, PARAM, 16, 768><<<plan.grid, plan.threads, 0, stream>>>(p, plan.warp_rows);
    if (plan.elements != 0)
        return cudaSuccess;
    return plan.vectors == 1    ? backward_row<X, DY, PARAM, 1, 256>(p, plan, stream)
           : plan.vectors == 2  ? backward_row<X, DY, PARAM, 2, 256>(p, plan, stream)
           : plan.threads > 384 ? backward_row<X, DY, PARAM, 4, 512>(p, plan, stream)
                                : backward_row<X, DY, PARAM, 4, 384>(p, plan, stream);
}

template <uint32_t X, uint32_t DY>
cudaError_t backward(const NormBackwardParams &p, int num_sms, cudaStream_t stream) {
    const BackwardPlan plan = backward_plan(p, num_sms);
    cudaError_t rc = cudaSuccess;
    if (plan.threads != 0) {
        if (DY != kFp32 && p.weight != nullptr && p.param_type == kFp32)
            rc = backward_rows<X, DY, kFp32>(p, plan, stream);
        else
            rc = backward_rows<X, DY, DY>(p, plan, stream);
    } else {
        if (p.dx != nullptr)
            norm_backward_rows_any<X, DY><<<row_grid(p.rows, num_sms), kRowThreads, 0, stream>>>(p);
        if (p.dweight != nullptr)
            norm_backward_columns_any<X, DY><<<dim3((p.width + 31) / 32, p.parts), kRowThreads, 0, stream>>>(p);
    }
    if (rc == cudaSuccess && p.dweight != nullptr)
        rc = launch_overlapped(norm_backward_join, dim3((p.width + 31) / 32, 2), kJoinWarps * 32, 0, stream, p);
    return rc;
}

} // namespace

cudaError_t launch_norm_forward(const NormForwardParams &p, int num_sms, cudaStream_t stream) {
    if (p.in_type == kBf16)
        return forward<kBf16, kBf16>(p, num_sms, stream);
    if (p.in_type == kFp16)
        return forward<kFp16, kFp16>(p, num_sms, stream);
    if (p.in_type == kFp32)
        return forward<kFp32, kFp32>(p, num_sms, stream);
    if (p.out_type == kBf16)
        return forward<kE4m3, kBf16>(p, num_sms, stream);
    if (p.out_type == kFp16)
        return forward<kE4m3, kFp16>(p, num_sms, stream);
    return forward<kE4m3, kFp32>(p, num_sms, stream);
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
