// Activations to 8 bits and back (sm_100a): e4m3 codes with one power-of-two
// scale per row and 128 columns (the format is described in rowmath.cuh).
// Both directions are one pass over memory and bound by it.
#include <algorithm>

#include "readout.h"
#include "rowmath.cuh"

namespace engram {

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // pieces of work whose loads a warp has in flight together

// A warp's pieces of all rows, `piece` columns each, `across` of them in a row:
// every gridful-th, kUnroll at a time.
struct Pieces {
    int64_t at, stride, total;
    uint32_t across;
    __device__ __forceinline__ Pieces(int64_t rows, uint32_t width, uint32_t piece)
        : at(int64_t(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32), stride(int64_t(gridDim.x) * (kThreads / 32)),
          across((width + piece - 1) / piece) {
        total = rows * across;
    }
    __device__ __forceinline__ void next() { at += stride * kUnroll; }
    // Row and place in the row of the j-th.
    __device__ __forceinline__ bool place(int j, int64_t &row, uint32_t &part) const {
        const int64_t i = at + j * stride;
        if (total <= 0x7FFFFFFFll) {
            row = uint32_t(i) / across;
            part = uint32_t(i) - uint32_t(row) * across;
        } else {
            row = i / across;
            part = uint32_t(i - row * across);
        }
        return i < total;
    }
};

// Sixteen values from 16-byte boundaries.
template <uint32_t TYPE> struct Sixteen {
    Raw8<TYPE> low, high;
};

template <uint32_t TYPE> __device__ __forceinline__ Raw8<TYPE> load_values8(const uint8_t *at) {
    Raw8<TYPE> r;
    r.v = ld_nc_na_v4(at);
    if constexpr (TYPE == kFp32)
        r.v2 = ld_nc_na_v4(at + 16);
    return r;
}

// Rows of whole 16-column chunks on 16-byte boundaries: a lane turns 16 values
// into one 16-byte store of codes; eight lanes hold a block.  8192 x 12288 bf16:
// 53.2 us, 5.7 TB/s (0.86 of a copy's rate; 49.8 us without the call before it);
// one value per lane and load took 157 us.
template <uint32_t TYPE>
__global__ void __launch_bounds__(kThreads) save_chunks(const __grid_constant__ SaveFp8Params p) {
    const uint32_t lane = threadIdx.x % 32, blocks = (p.width + kCheckpointBlock - 1) / kCheckpointBlock;
    for (Pieces q(p.rows, p.width, 512); q.at < q.total; q.next()) {
        Sixteen<TYPE> raw[kUnroll];
        int64_t row[kUnroll];
        uint32_t column[kUnroll];
        bool there[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            there[j] = q.place(j, row[j], column[j]);
            column[j] = column[j] * 512 + lane * 16;
            there[j] = there[j] && column[j] < p.width;
            if (there[j]) {
                const uint8_t *x = static_cast<const uint8_t *>(p.x) +
                                   (row[j] * p.x_stride + column[j]) * int64_t(element_bytes(TYPE));
                raw[j].low = load_values8<TYPE>(x);
                raw[j].high = load_values8<TYPE>(x + 8 * element_bytes(TYPE));
            }
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            Pair v[2][4];
            float amax = 0.f;
            if (there[j]) {
                unpack8<TYPE>(raw[j].low, v[0]);
                unpack8<TYPE>(raw[j].high, v[1]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 f = parts(v[e / 4][e % 4]);
                    amax = largest3(amax, f.x, f.y);
                }
            }
            // fmaxf passes NaN by; only an infinity hides the finite values' largest.
            if (__any_sync(0xFFFFFFFFu, amax > FLT_MAX)) {
                amax = 0.f;
                if (there[j])
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float2 f = parts(v[e / 4][e % 4]);
                        amax = fmaxf(amax, fmaxf(finite_abs(f.x), finite_abs(f.y)));
                        // The conversion saturates infinities, and they have to stay visible.
                        f.x = fabsf(f.x) <= FLT_MAX ? f.x : __uint_as_float(0x7FFFFFFFu);
                        f.y = fabsf(f.y) <= FLT_MAX ? f.y : __uint_as_float(0x7FFFFFFFu);
                        v[e / 4][e % 4] = pair(f);
                    }
            }
            const BlockScale scale = block_scale(lanes_max<8>(amax));
            if (there[j]) {
                const uint2 low = to_e4m3x8(v[0], scale.down), high = to_e4m3x8(v[1], scale.down);
                st_na_v4(p.codes + row[j] * p.codes_stride + column[j], Vec16{low.x, low.y, high.x, high.y});
                if (lane % 8 == 0)
                    p.scales[row[j] * blocks + column[j] / kCheckpointBlock] = scale.up;
            }
        }
    }
}

// Any width, stride and alignment: a warp takes blocks of 128 columns, a lane
// four adjacent ones, whose codes leave in one store (rows of codes start on
// 16-byte boundaries).  4096 x 4097 bf16: 33 us, 1.5 TB/s, bound by the number of
// loads (one element each).
template <uint32_t TYPE>
__global__ void __launch_bounds__(kThreads) save_any(const __grid_constant__ SaveFp8Params p) {
    const uint32_t lane = threadIdx.x % 32;
    for (Pieces q(p.rows, p.width, kCheckpointBlock); q.at < q.total; q.next()) {
        typename Element<TYPE>::T raw[kUnroll][4];
        int64_t row[kUnroll];
        uint32_t block[kUnroll];
        bool there[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            there[j] = q.place(j, row[j], block[j]);
            const uint32_t c = block[j] * kCheckpointBlock + lane * 4;
            const auto *x = static_cast<const typename Element<TYPE>::T *>(p.x) + min(row[j], p.rows - 1) * p.x_stride;
#pragma unroll
            for (int i = 0; i < 4; ++i)  // all in flight: no branch guards a load
                raw[j][i] = x[min(c + i, p.width - 1)];
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const uint32_t c = block[j] * kCheckpointBlock + lane * 4;
            float v[4], amax = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = c + i < p.width ? Element<TYPE>::get(raw[j][i]) : 0.f;
                amax = fmaxf(amax, finite_abs(v[i]));
            }
            const BlockScale scale = block_scale(lanes_max(amax));
            if (!there[j] || c >= p.width)
                continue;
            uint32_t codes = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                codes |= uint32_t(to_e4m3(v[i] * scale.down)) << (8 * i);
            uint8_t *to = p.codes + row[j] * p.codes_stride + c;
            if (c + 4 <= p.width)
                *reinterpret_cast<uint32_t *>(to) = codes;
            else
                for (uint32_t i = 0; c + i < p.width; ++i)
                    to[i] = uint8_t(codes >> (8 * i));
            if (lane == 0)
                p.scales[row[j] * q.across + block[j]] = scale.up;
        }
    }
}

// A finite code's value that its type cannot hold (a block's largest value may
// have been rounded up past it) becomes the type's largest.  An infinite scale,
// which no save writes, makes infinities and not finite values.
template <uint32_t TYPE> __device__ __forceinline__ float held(float v, float scale) {
    const float most = Element<TYPE>::kLargest;
    return isnan(v) || isinf(scale) ? v : fminf(fmaxf(v, -most), most);
}

// The way back: 8192 x 12288 to bf16 in 57.8 us, 5.2 TB/s (two thirds of what it
// moves are stores, 32 bytes per lane; as 16-byte stores they took 72 us).
template <uint32_t TYPE>
__global__ void __launch_bounds__(kThreads) restore_chunks(const __grid_constant__ RestoreFp8Params p) {
    const uint32_t lane = threadIdx.x % 32;
    for (Pieces q(p.rows, p.width, 512); q.at < q.total; q.next()) {
        Vec16 raw[kUnroll];
        float scale[kUnroll];
        int64_t row[kUnroll];
        uint32_t column[kUnroll];
        bool there[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            there[j] = q.place(j, row[j], column[j]);
            column[j] = column[j] * 512 + lane * 16;
            there[j] = there[j] && column[j] < p.width;
            if (there[j]) {
                raw[j] = ld_nc_na_v4(p.codes + row[j] * p.codes_stride + column[j]);
                scale[j] = __ldg(p.scales + row[j] * p.scale_row_stride + column[j] / kCheckpointBlock * p.scale_col_stride);
            }
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j)
            if (there[j]) {
                uint8_t *x = static_cast<uint8_t *>(p.x) + (row[j] * p.width + column[j]) * int64_t(element_bytes(TYPE));
                // Only a scale of 2^7 and more can carry a code past fp16, of 2^119 past the others.
                const bool far = scale[j] >= (TYPE == kFp16 ? 128.f : 6.6e35f);
                Pair v[2][4];
                unpack8<kE4m3>(Raw8<kE4m3>{make_uint2(raw[j].x, raw[j].y)}, v[0]);
                unpack8<kE4m3>(Raw8<kE4m3>{make_uint2(raw[j].z, raw[j].w)}, v[1]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    Pair &f = v[e / 4][e % 4];
                    f = mul2(f, both(scale[j]));
                    if (far)
                        f = pair(held<TYPE>(parts(f).x, scale[j]), held<TYPE>(parts(f).y, scale[j]));
                }
                if constexpr (TYPE == kFp32) {
                    store_row8<TYPE>(x, v[0]);
                    store_row8<TYPE>(x + 32, v[1]);
                } else {
                    Vec32 w;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 f = parts(v[e / 4][e % 4]);
                        w.v[e] = TYPE == kBf16 ? to_bf16x2(f.x, f.y) : to_fp16x2(f.x, f.y);
                    }
                    st_v8(x, w);
                }
            }
    }
}

// Any width, stride and alignment, by bytes and elements: 4096 x 4097 to bf16 29 us,
// 1.7 TB/s.
template <uint32_t TYPE>
__global__ void __launch_bounds__(kThreads) restore_any(const __grid_constant__ RestoreFp8Params p) {
    const uint32_t lane = threadIdx.x % 32;
    for (Pieces q(p.rows, p.width, kCheckpointBlock); q.at < q.total; q.next()) {
        uint8_t code[kUnroll][4];
        float scale[kUnroll];
        int64_t row[kUnroll];
        uint32_t block[kUnroll];
        bool there[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            there[j] = q.place(j, row[j], block[j]);
            const int64_t r = min(row[j], p.rows - 1);
            scale[j] = __ldg(p.scales + r * p.scale_row_stride + block[j] * p.scale_col_stride);
#pragma unroll
            for (int i = 0; i < 4; ++i)  // all in flight: no branch guards a load
                code[j][i] = p.codes[r * p.codes_stride + min(block[j] * kCheckpointBlock + i * 32 + lane, p.width - 1)];
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            auto *x = static_cast<typename Element<TYPE>::T *>(p.x) + row[j] * p.width;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t c = block[j] * kCheckpointBlock + i * 32 + lane;
                if (there[j] && c < p.width)
                    x[c] = Element<TYPE>::put(held<TYPE>(Element<kE4m3>::get(code[j][i]) * scale[j], scale[j]));
            }
        }
    }
}

// Six blocks of 256 threads per SM keep their loads in flight.
uint32_t grid_of(int64_t rows, uint32_t width, uint32_t piece, int num_sms) {
    const int64_t pieces = rows * ((width + piece - 1) / piece);
    return uint32_t(std::min<int64_t>((pieces + kThreads / 32 - 1) / (kThreads / 32), int64_t(num_sms) * 6));
}

template <uint32_t TYPE> void save(const SaveFp8Params &p, int num_sms, cudaStream_t stream) {
    if (p.width % 16 == 0 && on_boundary(p.x, 16) && p.x_stride * element_bytes(TYPE) % 16 == 0)
        save_chunks<TYPE><<<grid_of(p.rows, p.width, 512, num_sms), kThreads, 0, stream>>>(p);
    else
        save_any<TYPE><<<grid_of(p.rows, p.width, kCheckpointBlock, num_sms), kThreads, 0, stream>>>(p);
}

template <uint32_t TYPE> void restore(const RestoreFp8Params &p, int num_sms, cudaStream_t stream) {
    if (p.width % 16 == 0 && on_boundary(p.codes, 16) && p.codes_stride % 16 == 0)
        restore_chunks<TYPE><<<grid_of(p.rows, p.width, 512, num_sms), kThreads, 0, stream>>>(p);
    else
        restore_any<TYPE><<<grid_of(p.rows, p.width, kCheckpointBlock, num_sms), kThreads, 0, stream>>>(p);
}

} // namespace

cudaError_t launch_save_fp8(const SaveFp8Params &p, int num_sms, cudaStream_t stream) {
    p.type == kBf16   ? save<kBf16>(p, num_sms, stream)
    : p.type == kFp16 ? save<kFp16>(p, num_sms, stream)
                      : save<kFp32>(p, num_sms, stream);
    return cudaGetLastError();
}

cudaError_t launch_restore_fp8(const RestoreFp8Params &p, int num_sms, cudaStream_t stream) {
    p.type == kBf16   ? restore<kBf16>(p, num_sms, stream)
    : p.type == kFp16 ? restore<kFp16>(p, num_sms, stream)
                      : restore<kFp32>(p, num_sms, stream);
    return cudaGetLastError();
}

} // namespace engram
