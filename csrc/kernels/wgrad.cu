// A projection's weight and bias gradients from the 8-bit checkpoint of its
// input (sm_100a, tcgen05).
//
// dW[o][k] = sum_m dy[m][o] X[m][k] with X the checkpoint's rows.  Where the
// projection's input was X w + b (a norm's affine part), the same checkpoint
// serves: dW[o][k] = w[k] G[o][k] + b[k] s[o], G = dy^T X and s[o] = sum_m
// dy[m][o], which is also the bias gradient.
//
// X is decoded to bf16 on its way into shared memory, which is exact: a code
// has four significant bits and its scale is a power of two.  dy is bf16, or a
// sum of bf16 terms that hold every bit of it down to 2^-133 (two for fp16, three
// for fp32), one more pass over the rows for each.  So all products are exact and only
// the fp32 accumulation rounds.  The tensor core cuts what it adds rather than
// rounding it, an error that goes with the accumulator's size and the number of
// additions: the smallest terms go first, while the accumulator is small (512
// rows of fp32 are 1.5e-7 of the result's norm off, with the largest term first
// they were 2.5e-6), and an accumulator takes a limited number of rows before it
// is rounded into the sum of its like (most_steps), so that the error does not
// grow with the rows.
#include <algorithm>

#include "../driver.h"
#include "readout.h"
#include "rowmath.cuh"
#include "tensor.cuh"

namespace engram {

namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------- column sums of dy
// Sums over one part of the rows: a lane takes W adjacent columns (one vector
// of 16-byte rows, or one column), the block's warps every eighth row.  The
// product's kernel adds the parts up.
template <uint32_t TYPE, int W>
__global__ void __launch_bounds__(kThreads) dy_sums_part(const __grid_constant__ WeightGradParams p) {
    __shared__ float s_sum[kThreads / 32][32 * W];
    using T = typename Element<TYPE>::T;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, o = blockIdx.x * 32 * W + lane * W;
    const int64_t share = (p.rows + p.sum_rows - 1) / p.sum_rows;
    const int64_t first = int64_t(blockIdx.y) * share, last = min(first + share, p.rows);
    float sum[W] = {};
    start_next();
    if (o < p.out)
#pragma unroll 8
        for (int64_t r = first + warp; r < last; r += kThreads / 32) {
            const T *dy = static_cast<const T *>(p.dy) + r * p.dy_stride + o;
            if constexpr (W == 1) {
                sum[0] += Element<TYPE>::get(*dy);
            } else {
                T v[W];
                *reinterpret_cast<uint4 *>(v) = __ldg(reinterpret_cast<const uint4 *>(dy));
#pragma unroll
                for (int e = 0; e < W; ++e)
                    sum[e] += Element<TYPE>::get(v[e]);
            }
        }
#pragma unroll
    for (int e = 0; e < W; ++e)
        s_sum[warp][lane * W + e] = sum[e];
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < 32 * W; c += kThreads) {
        float total = 0.f;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w)
            total += s_sum[w][c];
        if (blockIdx.x * 32 * W + c < p.out)
            p.sum_parts[int64_t(blockIdx.y) * p.out + blockIdx.x * 32 * W + c] = total;
    }
}

// ---------------------------------------------------------------- dy as bf16 terms
// Each term is the rest's leading eight bits, cut (not rounded, which could
// carry beyond bf16's range), so the rest is exact; a non-finite value is all
// in the first.  With one term this lays bf16 rows out on 16-byte boundaries.
// A thread takes four adjacent columns (by one load where VECTOR).
template <uint32_t TYPE, bool VECTOR>
__global__ void __launch_bounds__(kThreads) split_dy(const __grid_constant__ WeightGradParams p) {
    using T = typename Element<TYPE>::T;
    const uint32_t o = (blockIdx.x * 64 + threadIdx.x % 64) * 4;
    if (o >= p.out)
        return;
    for (int64_t r = int64_t(blockIdx.y) * 4 + threadIdx.x / 64; r < p.rows; r += int64_t(gridDim.y) * 4) {
        const T *dy = static_cast<const T *>(p.dy) + r * p.dy_stride;
        T raw[4];
        if constexpr (VECTOR && sizeof(T) == 4)
            *reinterpret_cast<uint4 *>(raw) = __ldg(reinterpret_cast<const uint4 *>(dy + o));
        else if constexpr (VECTOR)
            *reinterpret_cast<uint2 *>(raw) = __ldg(reinterpret_cast<const uint2 *>(dy + o));
        else
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                raw[e] = dy[min(o + e, p.out - 1)];
        float rest[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            rest[e] = Element<TYPE>::get(raw[e]);
        for (uint32_t plane = 0; plane < p.planes; ++plane) {
            uint32_t bits[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                bits[e] = isnan(rest[e]) ? 0x7FC00000u : __float_as_uint(rest[e]) & 0xFFFF0000u;
                rest[e] = fabsf(rest[e]) <= FLT_MAX ? rest[e] - __uint_as_float(bits[e]) : 0.f;
            }
            // plane_stride is a multiple of eight: there is room for all four.
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.dy_planes) + (int64_t(plane) * p.rows + r) * p.plane_stride + o) =
                make_uint2(bits[0] >> 16 | bits[1], bits[2] >> 16 | bits[3]);
        }
    }
}

// ---------------------------------------------------------------- the product
constexpr uint32_t kSteps = 64;              // rows per stage
constexpr int64_t kPartBytes = 512 << 20;    // workspace for parts of the rows

// Stages of the rows that one accumulator takes, four additions each.  What the
// cuts of its additions take grows with their number, 7e-9 of the result's norm
// for each: 3.7e-6 for 8192 rows.  A 16-bit result loses 1.7e-3 to its rounding
// anyway; an fp32 one of 16-bit gradients goes by 4096 rows, of fp32 gradients by
// 2048, 6.5e-7 whatever their number (8192 x 12288 to 2048: 970 us, 906 in one
// accumulator for each term).
uint32_t most_steps(uint32_t dy_type, uint32_t out_type) { return out_type != kFp32 ? 128 : dy_type != kFp32 ? 64 : 32; }
constexpr int kLoadStages = 4, kOperandStages = 3;
constexpr uint32_t kDyChunk = kSteps * 128;  // 64 columns of dy (bf16)
constexpr uint32_t kCodeChunk = kSteps * 64; // 64 columns of codes
// A block's share of a pair's stage: 2 x 128 outputs, 128 columns.
constexpr uint32_t kDyBytes = 4 * kDyChunk, kCodeBytes = 2 * kCodeChunk, kOperandBytes = 2 * kDyChunk;
constexpr uint32_t kRingBytes = kLoadStages * (kDyBytes + kCodeBytes) + kOperandStages * kOperandBytes;
constexpr uint32_t kSharedBytes = kRingBytes + 1024;  // + alignment of the swizzled tiles
constexpr int kDecodeWarps = 8, kLoadWarp = 8, kScaleWarp = 9, kMmaWarp = 10, kSumWarp = 11, kTensorThreads = 12 * 32;
constexpr uint32_t kBlocks = 2;              // 128-column blocks that a block's share touches at most
constexpr uint32_t kTmemColumns = 512;
constexpr uint32_t kBoxBytes = 32 * 128;     // an epilogue box: 32 rows x 32 columns
constexpr int kBoxes = 3;                    // of each warp
constexpr uint64_t kWaitNs = 2000000000ull;  // far above any legal wait

// How a row's 128-column block is decoded.  Four codes s eeee mmm become four
// bf16 values by moving their bits to s 0000eeee mmm0000, the code's value
// times 2^-120 (subnormal codes included), and one multiplication by scale *
// 2^120: exact where the scale is a power of two up to 2^7.  Any other scale
// (and a NaN code, whose bits would read as 480) takes a conversion by way of
// fp32, rounded once.
struct Decoder {
    uint32_t factor;  // scale * 2^120 as two bf16, 0: by way of fp32
    float scale;
};
__device__ __forceinline__ Decoder decoder_of(float scale) {
    const uint32_t bits = __float_as_uint(scale);
    const bool simple = (bits & 0x7FFFFFu) == 0 && bits >= 1u << 23 && bits <= (127u + 7) << 23;
    return {simple ? __byte_perm(bits + (120u << 23), 0, 0x3232) : 0, scale};
}

// Words of a 16-code unit in which some byte is a NaN code have a bit of 0x80808080 set.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t codes) { return (codes & 0x7F7F7F7Fu) + 0x01010101u; }

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Codes 0 and 2 of a word, then 1 and 3: pairs that lie sixteen bits apart need
// no byte moves.  The columns of the product are put back in order where they
// leave TMEM (store_tile).
__device__ __forceinline__ void decode4(uint32_t codes, uint32_t factor, uint32_t &even, uint32_t &odd) {
    const uint32_t up = codes << 8;
    even = mul_bf16x2((up & 0x80008000u) | (up >> 4 & 0x07F007F0u), factor);
    odd = mul_bf16x2((codes & 0x80008000u) | (codes >> 4 & 0x07F007F0u), factor);
}
__device__ __forceinline__ void decode4_by_fp32(uint32_t codes, float scale, uint32_t &even, uint32_t &odd) {
    const float2 a = from_e4m3x2(codes & 0xFFFFu), b = from_e4m3x2(codes >> 16);
    even = to_bf16x2(a.x * scale, b.x * scale);
    odd = to_bf16x2(a.y * scale, b.y * scale);
}

struct Shared {
    uint64_t loaded[kLoadStages], load_free[kLoadStages];
    uint64_t decoded[kOperandStages], operand_free[kOperandStages];
    uint64_t done;
    uint32_t tmem;
    uint32_t failed;
    Decoder decoders[kLoadStages][kBlocks][kSteps];
    float row_sums[2 * 128];                   // of dy, for this block's outputs
    alignas(16) float weight[256], bias[256];  // the folded norm's, for the pair's columns
};

__device__ __forceinline__ Vec16 load_shared16(uint32_t at) {
    Vec16 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ uint2 load_shared8(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}
__device__ __forceinline__ void store_shared16(uint32_t at, const Vec16 &v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// A block's accumulators to memory, folding the norm in where no parts are to be
// joined first.  A warp takes 32 rows x 32 columns at a time (TMEM gives a lane
// a row) by way of boxes in its part of the ring, which is free by then: tiled
// stores where rows are on 16-byte boundaries, else row by row.
template <uint32_t TYPE>
__device__ __forceinline__ void store_tile(const WeightGradParams &p, const CUtensorMap *map, const Shared &s, uint32_t tmem,
                                           uint8_t *boxes, uint32_t o0, uint32_t k0, uint32_t slot) {
    constexpr uint32_t kSize = element_bytes(TYPE), kRow = 32 * kSize;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, columns = min(p.tile_k, p.width - k0);
    const uint32_t half = p.halves == 2 ? warp / 4 : 0, row0 = warp % 4 * 32;
    const uint32_t o_first = o0 + half * 256 + row0;
    if (o_first >= p.out)
        return;
    const bool weighted = p.parts == 1 && p.norm_weight != nullptr, shifted = p.parts == 1 && p.norm_bias != nullptr;
    const float row_sum = shifted ? s.row_sums[half * 128 + row0 + lane] : 0.f;
    int box = 0;
    for (uint32_t c0 = p.halves == 2 ? 0 : warp / 4 * 32; c0 < columns; c0 += p.halves == 2 ? 32 : 64) {
        uint32_t v[32];
        tmem_load32(tmem + (row0 << 16) + half * 256 + c0, v);
        if (lane == 0)
            bulk_wait_read<kBoxes - 1>();  // this box has been stored
        __syncwarp();
        tmem_wait_loads();
        uint8_t *at = boxes + box * kBoxBytes;
        float x[32];
#pragma unroll
        for (int c = 0; c < 32; ++c)  // accumulators are in the decoders' order: columns 0, 2, 1, 3
            x[c] = __uint_as_float(v[c % 4 == 1 ? c + 1 : c % 4 == 2 ? c - 1 : c]);
        if (weighted) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float4 w = *reinterpret_cast<const float4 *>(s.weight + c0 + q * 4);
                x[q * 4] *= w.x, x[q * 4 + 1] *= w.y, x[q * 4 + 2] *= w.z, x[q * 4 + 3] *= w.w;
            }
        }
        if (shifted) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float4 b = *reinterpret_cast<const float4 *>(s.bias + c0 + q * 4);
                x[q * 4] += b.x * row_sum, x[q * 4 + 1] += b.y * row_sum;
                x[q * 4 + 2] += b.z * row_sum, x[q * 4 + 3] += b.w * row_sum;
            }
        }
        // Rows of 64 or 128 bytes with the stores' swizzle of that width.
#pragma unroll
        for (uint32_t q = 0; q < kRow / 16; ++q) {
            uint4 w;
            if constexpr (TYPE == kFp32)
                w = make_uint4(__float_as_uint(x[q * 4]), __float_as_uint(x[q * 4 + 1]), __float_as_uint(x[q * 4 + 2]),
                               __float_as_uint(x[q * 4 + 3]));
            else if constexpr (TYPE == kBf16)
                w = make_uint4(to_bf16x2(x[q * 8], x[q * 8 + 1]), to_bf16x2(x[q * 8 + 2], x[q * 8 + 3]),
                               to_bf16x2(x[q * 8 + 4], x[q * 8 + 5]), to_bf16x2(x[q * 8 + 6], x[q * 8 + 7]));
            else
                w = make_uint4(to_fp16x2(x[q * 8], x[q * 8 + 1]), to_fp16x2(x[q * 8 + 2], x[q * 8 + 3]),
                               to_fp16x2(x[q * 8 + 4], x[q * 8 + 5]), to_fp16x2(x[q * 8 + 6], x[q * 8 + 7]));
            const uint32_t swizzled = TYPE == kFp32 ? q ^ (lane & 7) : q ^ (lane >> 1 & 3);
            *reinterpret_cast<uint4 *>(at + lane * kRow + swizzled * 16) = w;
        }
        if (p.boxes) {
            fence_async_shared();
            __syncwarp();
            if (lane == 0) {
                tensor_store_3d(map, int(k0 + c0), int(o_first), int(slot), at);
                bulk_commit();
            }
            box = box + 1 == kBoxes ? 0 : box + 1;
        } else {
            __syncwarp();
            using T = typename Element<TYPE>::T;
            T *out = p.parts == 1 ? static_cast<T *>(p.dweight)
                                  : reinterpret_cast<T *>(p.dw_parts + int64_t(slot) * p.out * p.width);
            const uint32_t o_rows = min(32u, p.out - o_first), chunk = lane * kSize / 16;
            if (c0 + lane < columns)
#pragma unroll 8
                for (uint32_t r = 0; r < o_rows; ++r) {
                    const uint32_t swizzled = TYPE == kFp32 ? chunk ^ (r & 7) : chunk ^ (r >> 1 & 3);
                    out[int64_t(o_first + r) * p.width + k0 + c0 + lane] =
                        *reinterpret_cast<const T *>(at + r * kRow + swizzled * 16 + lane * kSize % 16);
                }
            __syncwarp();
        }
    }
    if (lane == 0)
        bulk_wait_read<0>();
}

// A pair of blocks: halves x 256 outputs by tile_k columns over one part of the
// rows, by 256 x n x 16 MMAs on both SMs.  Each block brings its 128 rows of a
// half's dy and decodes half of the columns; the tensor cores read the other
// half from the other block, and each decoded value is used 512 times.  With
// one SM on its own (256 x 256 outputs) shared memory was the bound: 192 KB
// moved through it per 1024 cycles of MMAs against 128 KB here.
//
// Warp 8 copies tiles of dy and codes into a ring of four stages; warps 0-7
// decode a stage's codes into one of three operand buffers, by the factors
// that warp 9 makes of its scales; the leader's warp 10 issues the MMAs of a
// stage for both halves; warp 11 adds up the column sums of dy meanwhile.
// Accumulators fill TMEM (2 x 256 columns).
//
// 8192 x 12288 to 2048 bf16: 291 us, 1417 TFLOP/s (0.85 of the measured cuBLAS
// burst; the library's product of the same size with bf16 rows at hand takes 265
// us, and restoring them first 58 us more); 4096 x 6144 to 2048 with a norm folded
// in: 106 us, 970 TFLOP/s: its 128 tiles are 1.7 rounds of the 74 pairs.  A round
// costs ~8 us outside its MMAs (fill, epilogue), and a stage of 64 rows 1370 cycles
// for 896 of MMAs at 224 columns, the tile chosen for 8192 x 12288 to 2048.
__global__ void __cluster_dims__(2) __launch_bounds__(kTensorThreads, 1)
    weight_grad_tensor(const __grid_constant__ WeightGradParams p, const __grid_constant__ CUtensorMap dy_map,
                       const __grid_constant__ CUtensorMap code_map, const __grid_constant__ CUtensorMap out_map) {
    extern __shared__ uint8_t s_raw[];
    __shared__ Shared s;
    uint8_t *ring = s_raw + ((1024u - (smem_addr(s_raw) & 1023u)) & 1023u);
    uint8_t *dy_tiles = ring, *code_tiles = ring + kLoadStages * kDyBytes,
            *operands = code_tiles + kLoadStages * kCodeBytes;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, rank = cluster_rank();
    const uint32_t tile = blockIdx.x / 2, share = p.tile_k / 2;
    const uint32_t o0 = tile % p.tiles_o * (p.halves * 256) + rank * 128;  // half h: o0 + h * 256
    const uint32_t tile_k0 = tile / p.tiles_o % p.tiles_k * p.tile_k;
    const uint32_t k0 = tile_k0 + rank * share;                            // this block's columns to decode
    const uint32_t place = tile / (p.tiles_o * p.tiles_k), part = p.first_part + place, slot = p.first_slot + place;
    const uint32_t plane_steps = uint32_t((p.rows + kSteps - 1) / kSteps);
    // A part's rows, once for each term of dy, the smallest term first.
    const uint32_t first = part * p.part_steps, row_steps = min(p.part_steps, plane_steps - first);
    const uint32_t steps = row_steps * p.planes;
    const uint32_t columns = k0 < p.width ? min(share, p.width - k0) : 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kLoadStages; ++i) {
            mbar_init(&s.loaded[i], 2);  // the copies and the decoders
            mbar_init(&s.load_free[i], kDecodeWarps + 1);
        }
        for (int i = 0; i < kOperandStages; ++i) {
            mbar_init(&s.decoded[i], 2 * kDecodeWarps);
            mbar_init(&s.operand_free[i], 1);
        }
        mbar_init(&s.done, 1);
        s.failed = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp)
        tmem_alloc(&s.tmem, kTmemColumns);
    tensor_fence_before();
    __syncthreads();
    cluster_sync();  // the other block's barriers are there
    tensor_fence_after();
    const uint32_t tmem = s.tmem;

    bool ok = true;
    if (warp == kLoadWarp) {
        if (lane == 0) {
            prefetch_tensor_map(&dy_map);
            prefetch_tensor_map(&code_map);
            uint32_t dy_chunks = 0;
            for (uint32_t c = 0; c < p.halves * 2; ++c)
                dy_chunks += o0 + c / 2 * 256 + c % 2 * 64 < p.out;  // the first ones: outputs ascend
            const uint32_t code_chunks = (columns + 63) / 64;
            uint32_t i = 0;
            for (; ok && i < steps; ++i) {
                const uint32_t at = i % kLoadStages;
                ok = mbar_wait_often(&s.load_free[at], (i / kLoadStages & 1) ^ 1, kWaitNs);
                if (!ok)
                    break;
                const int m = int((first + i % row_steps) * kSteps), plane = int(p.planes - 1 - i / row_steps);
                mbar_arrive_expect_tx(&s.loaded[at], dy_chunks * kDyChunk + code_chunks * kCodeChunk);
                for (uint32_t c = 0; c < dy_chunks; ++c)
                    tensor_load_3d(dy_tiles + at * kDyBytes + c * kDyChunk, &dy_map, int(o0 + c / 2 * 256 + c % 2 * 64), m,
                                   plane, &s.loaded[at]);
                for (uint32_t c = 0; c < code_chunks; ++c)
                    tensor_load_3d(code_tiles + at * kCodeBytes + c * kCodeChunk, &code_map, int(k0 + c * 64), m, 0,
                                   &s.loaded[at]);
            }
            if (!ok)  // let the copies in flight land before the block goes
                for (uint32_t j = i > kLoadStages ? i - kLoadStages : 0; j < i; ++j)
                    mbar_wait_often(&s.loaded[j % kLoadStages], j / kLoadStages & 1, kWaitNs);
        }
    } else if (warp == kMmaWarp) {
        if (rank == 0 && lane == 0) {
            const uint32_t shape = mma_shape_bf16(p.tile_k);
            uint32_t at = 0, to = 0, phase = 0;
            for (uint32_t i = 0; i < steps; ++i) {
                // Both blocks' decoders have seen their dy tiles land too.
                ok = mbar_wait_often(&s.decoded[to], phase, kWaitNs);
                if (!ok)
                    break;
                tensor_fence_after();
                for (uint32_t half = 0; half < p.halves; ++half)
#pragma unroll
                    for (uint32_t j = 0; j < kSteps / 16; ++j)
                        mma_bf16(tmem + half * 256,
                                 mma_operand(dy_tiles + at * kDyBytes + half * 2 * kDyChunk + j * 2048, kDyChunk, 1024),
                                 mma_operand(operands + to * kOperandBytes + j * 2048, kDyChunk, 1024), shape,
                                 (i | j) != 0);
                mma_commit(&s.load_free[at]);
                mma_commit(&s.operand_free[to]);
                at = at + 1 == kLoadStages ? 0 : at + 1;
                to = to + 1 == kOperandStages ? 0 : to + 1;
                phase ^= to == 0 ? 1 : 0;
            }
            mma_commit(&s.done);
        }
    } else if (warp == kScaleWarp) {
        // Lane l: rows l and l + 32 of a stage.  Loads are kAhead stages ahead: one
        // stage ahead, their latency was the time of a stage.
        constexpr uint32_t kAhead = 8;
        const uint32_t block0 = k0 / kCheckpointBlock;
        const uint32_t blocks = columns == 0 ? 0 : (k0 + columns - 1) / kCheckpointBlock - block0 + 1;
        const float *scales = p.scales + block0 * p.scale_col_stride;
        float next[kAhead][2][kBlocks];
        auto load = [&](uint32_t i, float (&to)[2][kBlocks]) {
            const int64_t m = int64_t(first + i % row_steps) * kSteps + lane;
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                for (uint32_t b = 0; b < kBlocks; ++b)
                    to[h][b] = i < steps && m + h * 32 < p.rows && b < blocks
                                   ? __ldg(scales + (m + h * 32) * p.scale_row_stride + b * p.scale_col_stride)
                                   : 1.f;
        };
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a)
            load(a, next[a]);
        for (uint32_t i0 = 0; ok && i0 < steps; i0 += kAhead)
#pragma unroll
            for (uint32_t a = 0; a < kAhead; ++a) {
                const uint32_t i = i0 + a, at = i % kLoadStages;
                if (i >= steps)
                    break;
                ok = mbar_wait_often(&s.load_free[at], (i / kLoadStages & 1) ^ 1, kWaitNs);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok)
                    break;
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                    for (uint32_t b = 0; b < kBlocks; ++b)
                        s.decoders[at][b][lane + h * 32] = decoder_of(next[a][h][b]);
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&s.loaded[at]);
                load(i + kAhead, next[a]);
            }
    } else if (warp == kSumWarp) {
        const bool weighted = p.parts == 1 && p.norm_weight != nullptr, shifted = p.parts == 1 && p.norm_bias != nullptr;
        for (uint32_t c = lane; c < p.tile_k; c += 32) {
            const bool there = tile_k0 + c < p.width;
            s.weight[c] = weighted && there ? load_param(p.norm_weight, p.param_type, tile_k0 + c) : 0.f;
            s.bias[c] = shifted && there ? load_param(p.norm_bias, p.param_type, tile_k0 + c) : 0.f;
        }
        const bool told = tile_k0 == 0 && part == 0;  // to the join and the bias
        wait_for_previous();  // the sums' parts; nothing else here needs them
        if (p.dy_sums != nullptr && (shifted || told)) {
            // A lane's eight outputs together: their loads are in flight at once.
            float sum[8] = {};
            uint32_t o[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                o[j] = o0 + j / 4 * 256 + j % 4 * 32 + lane;
                if (j / 4 >= p.halves)
                    o[j] = p.out;
            }
#pragma unroll 4
            for (uint32_t r = 0; r < p.sum_rows; ++r)
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j)
                    if (o[j] < p.out)
                        sum[j] += p.sum_parts[int64_t(r) * p.out + o[j]];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                s.row_sums[j * 32 + lane] = sum[j];
                if (told && o[j] < p.out) {
                    p.dy_sums[o[j]] = sum[j];
                    if (p.dbias != nullptr)
                        store_param(p.dbias, p.out_type, o[j], sum[j]);
                }
            }
        }
    } else {
        // A warp takes 32 rows and every fourth 16-byte unit of them: eight lanes
        // of one shared-memory phase are eight rows of one unit, which both
        // swizzles spread over all banks.  Nothing but the stage changes from
        // one to the next.
        constexpr int kUnits = 2;
        const uint32_t row = warp % 2 * 32 + lane, units = (columns + 15) / 16;
        uint32_t from[kUnits], to_low[kUnits], to_high[kUnits], decoder[kUnits];
#pragma unroll
        for (uint32_t j = 0; j < kUnits; ++j) {
            const uint32_t u = warp / 2 + j * 4, chunk = u % 4 * 2;
            from[j] = smem_addr(code_tiles) + u / 4 * kCodeChunk + row * 64 + ((u % 4 ^ (row >> 1 & 3)) << 4);
            to_low[j] = smem_addr(operands) + u / 4 * kDyChunk + row * 128 + ((chunk ^ (row & 7)) << 4);
            to_high[j] = smem_addr(operands) + u / 4 * kDyChunk + row * 128 + ((chunk + 1 ^ (row & 7)) << 4);
            const uint32_t b = (k0 + u * 16) / kCheckpointBlock - k0 / kCheckpointBlock;
            decoder[j] = smem_addr(&s.decoders[0][min(b, kBlocks - 1)][row]);
        }
        const uint32_t leader = leader_barrier(&s.decoded[0]);
        uint32_t at = 0, load_phase = 0, to = 0, operand_phase = 1;
        for (uint32_t i = 0; i < steps; ++i) {
            ok = mbar_wait_often(&s.loaded[at], load_phase, kWaitNs);
            Vec16 v[kUnits];
            uint2 d[kUnits];
#pragma unroll
            for (uint32_t j = 0; j < kUnits; ++j)
                if (warp / 2 + j * 4 < units) {
                    v[j] = load_shared16(from[j] + at * kCodeBytes);
                    d[j] = load_shared8(decoder[j] + at * uint32_t(sizeof(s.decoders[0])));
                }
            ok = ok && mbar_wait_often(&s.operand_free[to], operand_phase, kWaitNs);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok)
                break;
#pragma unroll
            for (uint32_t j = 0; j < kUnits; ++j)
                if (warp / 2 + j * 4 < units) {
                    const uint32_t nan = (nan_bytes(v[j].x) | nan_bytes(v[j].y) | nan_bytes(v[j].z) | nan_bytes(v[j].w)) & 0x80808080u;
                    Vec16 x, y;
                    if (d[j].x != 0 && nan == 0) {
                        decode4(v[j].x, d[j].x, x.x, x.y);
                        decode4(v[j].y, d[j].x, x.z, x.w);
                        decode4(v[j].z, d[j].x, y.x, y.y);
                        decode4(v[j].w, d[j].x, y.z, y.w);
                    } else {
                        const float scale = __uint_as_float(d[j].y);
                        decode4_by_fp32(v[j].x, scale, x.x, x.y);
                        decode4_by_fp32(v[j].y, scale, x.z, x.w);
                        decode4_by_fp32(v[j].z, scale, y.x, y.y);
                        decode4_by_fp32(v[j].w, scale, y.z, y.w);
                    }
                    store_shared16(to_low[j] + to * kOperandBytes, x);
                    store_shared16(to_high[j] + to * kOperandBytes, y);
                }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive_leader(leader + to * 8);
                mbar_arrive(&s.load_free[at]);
            }
            at = at + 1 == kLoadStages ? 0 : at + 1;
            load_phase ^= at == 0 ? 1 : 0;
            to = to + 1 == kOperandStages ? 0 : to + 1;
            operand_phase ^= to == 0 ? 1 : 0;
        }
    }
    if (!ok)
        s.failed = 1;
    __syncthreads();
    if (warp < kDecodeWarps) {
        ok = mbar_wait_often(&s.done, 0, kWaitNs);
        ok = __all_sync(0xFFFFFFFFu, ok) && s.failed == 0;
        tensor_fence_after();
        if (ok) {
            uint8_t *boxes = ring + warp * (kBoxes * kBoxBytes);
            const uint32_t type = p.parts == 1 ? p.out_type : uint32_t(kFp32);
            if (type == kBf16)
                store_tile<kBf16>(p, &out_map, s, tmem, boxes, o0, tile_k0, slot);
            else if (type == kFp16)
                store_tile<kFp16>(p, &out_map, s, tmem, boxes, o0, tile_k0, slot);
            else
                store_tile<kFp32>(p, &out_map, s, tmem, boxes, o0, tile_k0, slot);
        }
        tensor_fence_before();
        if (!ok && lane == 0)
            st_release_sys_u32(p.fault, kPipelineTimeout);
    }
    __syncthreads();
    cluster_sync();  // neither block goes while the other may reach into it
    if (warp == kMmaWarp) {
        tensor_fence_after();
        tmem_free(tmem, kTmemColumns);
        if (lane == 0 && s.failed != 0)
            st_release_sys_u32(p.fault, kPipelineTimeout);
    }
}

// Adds the parts of the rows in order, and folds the norm in with the last.  A
// thread takes four adjacent columns of every gridDim.y-th output (by one load
// and store where VECTOR).
template <bool VECTOR> __global__ void __launch_bounds__(kThreads) weight_grad_join(const __grid_constant__ WeightGradParams p) {
    const uint32_t k = (blockIdx.x * kThreads + threadIdx.x) * 4;
    if (k >= p.width)
        return;
    const int64_t total = int64_t(p.out) * p.width;
    float w[4], b[4];
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
        w[e] = p.last && p.norm_weight != nullptr && k + e < p.width ? load_param(p.norm_weight, p.param_type, k + e) : 1.f;
        b[e] = p.last && p.norm_bias != nullptr && k + e < p.width ? load_param(p.norm_bias, p.param_type, k + e) : 0.f;
    }
    for (uint32_t o = blockIdx.y; o < p.out; o += gridDim.y) {
        const int64_t at = int64_t(o) * p.width + k;
        float v[4] = {};
#pragma unroll 4
        for (uint32_t slot = 0; slot < p.joined; ++slot) {
            const float *part = p.dw_parts + slot * total + at;
            if constexpr (VECTOR) {
                const float4 q = *reinterpret_cast<const float4 *>(part);
                v[0] += q.x, v[1] += q.y, v[2] += q.z, v[3] += q.w;
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    if (k + e < p.width)
                        v[e] += part[e];
            }
        }
        if (p.last) {
            const float sum = p.norm_bias != nullptr ? p.dy_sums[o] : 0.f;
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                if (p.norm_weight != nullptr)
                    v[e] = __fmul_rn(v[e], w[e]);
                if (p.norm_bias != nullptr)
                    v[e] = __fmaf_rn(b[e], sum, v[e]);
            }
        }
        const uint32_t type = p.last ? p.out_type : uint32_t(kFp32);
        void *to = p.last ? p.dweight : p.dw_parts;
        if (VECTOR && type == kFp32)
            *reinterpret_cast<float4 *>(static_cast<float *>(to) + at) = make_float4(v[0], v[1], v[2], v[3]);
        else if (VECTOR)
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(to) + at) =
                type == kBf16 ? make_uint2(to_bf16x2(v[0], v[1]), to_bf16x2(v[2], v[3]))
                              : make_uint2(to_fp16x2(v[0], v[1]), to_fp16x2(v[2], v[3]));
        else
            for (uint32_t e = 0; e < 4 && k + e < p.width; ++e)
                store_param(to, type, at + e, v[e]);
    }
}

// [planes][rows][columns] in boxes; what lies outside reads as zero.
CUtensorMap tile_map(CUtensorMapDataType type, const void *base, uint64_t columns, uint64_t rows, uint64_t planes,
                     uint64_t row_bytes, uint32_t box_columns, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
    CUtensorMap map;
    const cuuint64_t dims[3] = {columns, rows, planes}, strides[2] = {row_bytes, row_bytes * rows};
    const cuuint32_t box[3] = {box_columns, box_rows, 1}, steps[3] = {1, 1, 1};
    check_cu(driver().TensorMapEncodeTiled(&map, type, 3, const_cast<void *>(base), dims, strides, box, steps,
                                           CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE),
             "encode tensor map");
    return map;
}

template <uint32_t TYPE> void dy_passes(const WeightGradParams &p, cudaStream_t stream) {
    constexpr int kVector = 16 / element_bytes(TYPE);
    if (p.dy_planes != nullptr) {
        const dim3 grid((p.out + 255) / 256, uint32_t(std::min<int64_t>((p.rows + 3) / 4, 4096)));
        if (on_boundary(p.dy, 16) && p.dy_stride % 4 == 0 && p.out % 4 == 0)
            split_dy<TYPE, true><<<grid, kThreads, 0, stream>>>(p);
        else
            split_dy<TYPE, false><<<grid, kThreads, 0, stream>>>(p);
    }
    // Last, so that the product overlaps this alone.
    if (p.dy_sums != nullptr) {
        if (on_boundary(p.dy, 16) && p.dy_stride % kVector == 0 && p.out % kVector == 0)
            dy_sums_part<TYPE, kVector>
                <<<dim3((p.out + 32 * kVector - 1) / (32 * kVector), p.sum_rows), kThreads, 0, stream>>>(p);
        else
            dy_sums_part<TYPE, 1><<<dim3((p.out + 31) / 32, p.sum_rows), kThreads, 0, stream>>>(p);
    }
}

} // namespace

void plan_weight_grad(WeightGradParams &p, int num_sms) {
    // Few parts for the product's sum warp to add up; 16 rows each at least.
    p.sum_rows = uint32_t(std::min<int64_t>((p.rows + 15) / 16, 32));
    p.planes = p.type == kBf16 ? 1 : p.type == kFp16 ? 2 : 3;
    p.halves = p.out > 256 ? 2 : 1;
    p.tiles_o = (p.out + p.halves * 256 - 1) / (p.halves * 256);
    const int64_t steps = (p.rows + kSteps - 1) / kSteps, pairs = num_sms / 2;
    // Cycles of one pair: a stage is bound by its MMAs (256 x 16 x n takes n / 2)
    // or by shared memory (128 bytes a cycle: dy in and out, codes in and out,
    // operands in, and out for each half); the epilogue moves ~12 values a cycle
    // and block.  Splitting the rows costs a pass over the parts at ~3.5 KB a cycle.
    double best = 1e300;
    const int64_t limit = most_steps(p.type, p.out_type), fewest = (steps + limit - 1) / limit;
    const int64_t most = std::max(fewest, std::min<int64_t>(steps, 64));
    for (uint32_t tile = 32; tile <= 256; tile += 32) {
        const uint32_t tiles_k = (p.width + tile - 1) / tile;
        const int64_t tiles = int64_t(p.tiles_o) * tiles_k;
        for (int64_t parts = fewest; parts <= most; parts = parts < 8 ? parts + 1 : parts * 2) {
            const int64_t part_steps = (steps + parts - 1) / parts, used = (steps + part_steps - 1) / part_steps;
            const double waves = double((tiles * used + pairs - 1) / pairs);
            const double stage = std::max({2.0 * p.halves * tile, 256.0 * p.halves + (1 + p.halves / 2.) * tile, 400.});
            const double block = 5000 + part_steps * p.planes * stage + p.halves * 128.0 * tile / 12;
            const double join = used > 1 ? 3000 + 8.0 * used * p.out * p.width / 3500 : 0;
            const double cost = waves * block + join;
            if (cost < best * 0.999) {
                best = cost;
                p.tile_k = tile;
                p.tiles_k = tiles_k;
                p.parts = uint32_t(used);
                p.part_steps = uint32_t(part_steps);
            }
        }
    }
    const int64_t room = kPartBytes / (4 * int64_t(p.out) * p.width);
    p.slots = uint32_t(std::min<int64_t>(p.parts, std::max<int64_t>(2, room)));
}

cudaError_t launch_weight_grad(const WeightGradParams &p, cudaStream_t stream) {
    if (p.type == kBf16)
        dy_passes<kBf16>(p, stream);
    else if (p.type == kFp16)
        dy_passes<kFp16>(p, stream);
    else
        dy_passes<kFp32>(p, stream);
    const bool split = p.dy_planes != nullptr;
    const CUtensorMap dy_map =
        tile_map(CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, split ? p.dy_planes : p.dy, p.out, p.rows, p.planes,
                 uint64_t(split ? p.plane_stride : p.dy_stride) * 2, 64, kSteps, CU_TENSOR_MAP_SWIZZLE_128B);
    const CUtensorMap code_map = tile_map(CU_TENSOR_MAP_DATA_TYPE_UINT8, p.codes, p.width, p.rows, 1,
                                          uint64_t(p.codes_stride), 64, kSteps, CU_TENSOR_MAP_SWIZZLE_64B);
    const uint32_t type = p.parts == 1 ? p.out_type : uint32_t(kFp32);
    WeightGradParams q = p;
    q.boxes = p.width * element_bytes(type) % 16 == 0;
    CUtensorMap out_map = code_map;  // not used without boxes
    if (q.boxes)
        out_map = tile_map(type == kBf16   ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                           : type == kFp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                           : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                           p.parts == 1 ? p.dweight : p.dw_parts, p.width, p.out, p.slots,
                           uint64_t(p.width) * element_bytes(type), 32, 32,
                           type == kFp32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
    cudaError_t rc = cudaFuncSetAttribute(weight_grad_tensor, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedBytes);
    if (rc != cudaSuccess)
        return rc;
    for (uint32_t first = 0; first < p.parts;) {
        q.first_part = first;
        q.first_slot = first == 0 ? 0 : 1;
        const uint32_t count = std::min(p.parts - first, p.slots - q.first_slot);
        const dim3 grid(2 * p.tiles_o * p.tiles_k * count);
        if (first == 0 && p.dy_sums != nullptr) {
            rc = launch_overlapped(weight_grad_tensor, grid, kTensorThreads, kSharedBytes, stream, q, dy_map, code_map, out_map);
            if (rc != cudaSuccess)
                return rc;
        } else {
            weight_grad_tensor<<<grid, kTensorThreads, kSharedBytes, stream>>>(q, dy_map, code_map, out_map);
        }
        first += count;
        q.joined = q.first_slot + count;
        q.last = first == p.parts;
        if (p.parts > 1) {
            // Blocks enough to fill the GPU, or one for each output.
            const uint32_t across = (p.width + 4 * kThreads - 1) / (4 * kThreads);
            const dim3 blocks(across, std::max(1u, std::min({p.out, 148 * 16 / across + 1, 65535u})));
            if (p.width % 4 == 0)
                weight_grad_join<true><<<blocks, kThreads, 0, stream>>>(q);
            else
                weight_grad_join<false><<<blocks, kThreads, 0, stream>>>(q);
        }
    }
    return cudaGetLastError();
}

} // namespace engram
