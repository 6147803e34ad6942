// Launch parameters of the read-out kernels: layer norm over looked-up rows,
// 8-bit activation checkpoints, and the backward passes that read them.
// Plain structs passed by value, like params.h.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace engram {

// Element types of the read-out operators.
enum ElementType : uint32_t { kBf16 = 0, kFp16 = 1, kFp32 = 2, kE4m3 = 3 };

// Columns that share one scale in a checkpoint.
constexpr uint32_t kCheckpointBlock = 128;

// What a forward norm keeps for its backward pass.
enum KeepMode : uint32_t {
    kKeepNothing = 0,
    kKeepStats = 1,  // mean (in two parts) and rstd; the caller keeps the rows
    kKeepFp8 = 2,    // rstd and the normalised rows in 8 bits
};

// y = (x - mean) * rstd * weight + bias per row.  `x` is 16- or 32-bit rows or,
// with `scales`, the e4m3 codes of a lookup: entries of `hidden` columns, each
// with `packs` scales of `block` columns, in either of fetch()'s layouts.
struct NormForwardParams {
    const void *x;
    const float *scales;     // nullptr: none
    const void *weight;      // nullptr: no affine part
    const void *bias;        // nullptr: none
    void *y;
    float *mean, *shift;     // [rows], kKeepStats: the mean is their sum, shift what mean's rounding left
    float *rstd;             // [rows], with either
    uint8_t *codes;          // kKeepFp8: [rows][codes_stride]
    float *code_scales;      // kKeepFp8: [rows][ceil(width / 128)]
    uint32_t *fault;         // host-mapped: set when a wait ran out
    int64_t rows, x_stride, codes_stride, scale_row_stride, scale_col_stride;
    uint32_t width, hidden, packs, block;
    uint32_t in_type, out_type, param_type, keep;
    float eps;
};

// dx, and per-column sums for dweight and dbias.  The normalised rows come from
// `x`, `mean`, `shift` and `rstd` (kKeepStats; x as above) or from `codes` and
// `code_scales` (kKeepFp8).
struct NormBackwardParams {
    const void *dy;
    const void *x;
    const float *mean, *shift, *rstd;  // shift nullptr: zeros
    const uint8_t *codes;
    const float *code_scales;
    const void *weight;      // nullptr: no affine part
    void *dx;                // nullptr: not wanted
    void *dweight, *dbias;   // nullptr: not wanted (both or neither)
    float *partial;          // [2][parts][width] of dweight and dbias sums
    uint32_t *fault;         // host-mapped: set when a wait ran out
    int64_t rows, dy_stride, x_stride, codes_stride, code_scales_stride, scale_col_stride;
    uint32_t width, parts;
    uint32_t dy_type, param_type, keep;
};

struct SaveFp8Params {
    const void *x;
    uint8_t *codes;
    float *scales;           // [rows][ceil(width / 128)]
    int64_t rows, x_stride, codes_stride;
    uint32_t width, type;
};

struct RestoreFp8Params {
    const uint8_t *codes;
    const float *scales;
    void *x;                 // [rows][width]
    int64_t rows, codes_stride, scale_row_stride, scale_col_stride;
    uint32_t width, type;
};

// dweight[o][k] = sum over rows of dy[row][o] * X[row][k], X the rows of an
// 8-bit checkpoint; with a norm folded in, X * norm_weight + norm_bias.
// Code rows start on 16-byte boundaries, and so do those of a bf16 dy without
// dy_planes.
struct WeightGradParams {
    const void *dy;
    const uint8_t *codes;
    const float *scales;
    const void *norm_weight, *norm_bias;  // nullptr: not folded
    void *dweight, *dbias;                // dbias nullptr: not wanted
    float *dy_sums;                       // [out] fp32 column sums of dy; nullptr: not needed
    float *sum_parts;                     // [sum_rows][out], what dy_sums adds up
    void *dy_planes;                      // [planes][rows][plane_stride] bf16; nullptr: dy itself serves
    float *dw_parts;                      // [slots][out][width], parts > 1
    uint32_t *fault;                      // host-mapped: set when a wait ran out
    int64_t rows, dy_stride, codes_stride, scale_row_stride, scale_col_stride, plane_stride;
    uint32_t width, out, type, param_type, out_type, sum_rows;
    // The plan (plan_weight_grad): dy as `planes` bf16 terms; pairs of blocks for
    // `halves` x 256 outputs by tile_k columns; the rows in `parts` of `part_steps` x 64,
    // each with all terms of its rows.
    uint32_t planes, halves, tile_k, tiles_k, tiles_o, parts, part_steps;
    // At most `slots` parts at a time; of later launches slot 0 holds the sum of the
    // parts before.  A launch's parts start at first_part, in first_slot, and its
    // join adds up `joined` slots, into dweight with the last.
    uint32_t slots, first_part, first_slot, joined, last;
    uint32_t boxes;  // results leave by tiled stores
};

cudaError_t launch_norm_forward(const NormForwardParams &p, int num_sms, cudaStream_t stream);
// Parts of the column sums that launch_norm_backward wants workspace for.
uint32_t norm_backward_parts(const NormBackwardParams &p, int num_sms);
cudaError_t launch_norm_backward(const NormBackwardParams &p, int num_sms, cudaStream_t stream);
cudaError_t launch_save_fp8(const SaveFp8Params &p, int num_sms, cudaStream_t stream);
cudaError_t launch_restore_fp8(const RestoreFp8Params &p, int num_sms, cudaStream_t stream);
// Fills in the plan and sum_rows from rows, width, out and type.
void plan_weight_grad(WeightGradParams &p, int num_sms);
cudaError_t launch_weight_grad(const WeightGradParams &p, cudaStream_t stream);

} // namespace engram
