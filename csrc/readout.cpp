// Read-out operators of the extension: layer norm over looked-up rows, 8-bit
// activation checkpoints, and a projection's gradients from such a checkpoint.
// Arguments are checked here (ValueError, before any device is touched);
// everything runs on the current stream of the inputs' device, and outputs and
// workspaces come from torch's allocator, so calls can be captured into graphs.
#include <ATen/TracerMode.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/stl.h>
#include <torch/extension.h>

#include <array>
#include <atomic>
#include <cstring>
#include <mutex>
#include <optional>
#include <utility>

#include "bindings.h"
#include "driver.h"
#include "kernels/readout.h"

namespace py = pybind11;

namespace engram {

namespace {

using at::ScalarType;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

void need(bool ok, const char *what) {
    if (!ok)
        throw py::value_error(what);
}

// A trace (torch.jit.trace) does not see these calls and would keep their results
// as constants.  `recorded`: the caller is an autograd function, which a trace
// records as a whole (a graph of the dispatcher's calls, make_fx, does not).
void need_untraced(bool recorded) {
    using Modes = c10::impl::TorchDispatchModeTLS;
    check(!Modes::any_modes_set() || !Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
          "a graph of the dispatcher's calls would keep this call's result as a constant");
    check(recorded || !at::tracer::impl::is_dispatch_enabled(),
          "a trace would keep this call's result as a constant; trace layer_norm, linear or norm_linear");
}

bool is_wide(ScalarType t) {
    return t == ScalarType::BFloat16 || t == ScalarType::Half || t == ScalarType::Float;
}

uint32_t element_type(ScalarType t) {
    return t == ScalarType::BFloat16 ? kBf16 : t == ScalarType::Half ? kFp16 : t == ScalarType::Float ? kFp32 : kE4m3;
}

// [rows, width] with adjacent columns; rows may be strided (0: repeated).
void need_rows(const Tensor &t, const char *what) {
    need(t.dim() == 2 && t.size(1) >= 1 && t.size(1) <= (1 << 30) && t.size(0) <= 0x7FFFFFFF &&
             (t.stride(1) == 1 || t.size(1) == 1) && t.stride(0) >= 0,
         what);
}

// Per-column parameters of a norm: [width], 16-bit like the rows or fp32.
void need_params(const OptTensor &weight, const OptTensor &bias, int64_t width, ScalarType rows_type) {
    need(!bias || weight, "a bias needs a weight");
    if (!weight)
        return;
    need(weight->dim() == 1 && weight->size(0) == width && weight->is_contiguous(), "weight must be contiguous [width]");
    need(weight->scalar_type() == rows_type || weight->scalar_type() == ScalarType::Float,
         "weight must have the rows' type or float32");
    if (bias)
        need(bias->dim() == 1 && bias->size(0) == width && bias->is_contiguous() &&
                 bias->scalar_type() == weight->scalar_type(),
             "bias must be contiguous [width] of the weight's type");
}

// A checkpoint's codes [rows, width] and scales [rows, ceil(width / 128)].
void need_checkpoint(const Tensor &codes, const Tensor &scales) {
    need_rows(codes, "codes must be [rows, width] with adjacent columns");
    need(codes.scalar_type() == ScalarType::Float8_e4m3fn, "codes must be float8_e4m3fn");
    need(scales.dim() == 2 && scales.scalar_type() == ScalarType::Float && scales.size(0) == codes.size(0) &&
             scales.size(1) == (codes.size(1) + kCheckpointBlock - 1) / kCheckpointBlock,
         "scales must be float32 [rows, ceil(width / 128)]");
}

// A tensor whose values lie in memory of its own, all of it there.  Fake and
// functionalised tensors, masked ones and freed storages (a sharded parameter's
// between its uses) have null pointers; a negated view's values are not what lies
// in its memory.
void need_plain(const Tensor &t) {
    need(t.layout() == at::kStrided && t.has_storage() && !t.is_neg() && !t._is_zerotensor(),
         "tensors must be plain, with their values in memory");
    if (t.numel() == 0)
        return;
    int64_t last = t.storage_offset();
    for (int64_t d = 0; d < t.dim(); ++d)
        last += (t.size(d) - 1) * t.stride(d);
    const uintptr_t at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
    need(size_t(last + 1) * t.element_size() <= t.storage().nbytes() && at != 0 && at % t.element_size() == 0,
         "tensors must be plain, with their values in memory");
}

// The device all of these are on, which has to be a GPU.  Results carry no tangent
// of forward-mode differentiation, so arguments may not either (`recorded`: an
// autograd function's do, and torch raises for it).
int need_device(const Tensor &first, std::initializer_list<const OptTensor *> others, bool recorded = false) {
    const auto check_one = [recorded](const Tensor &t) {
        need_plain(t);
        need(recorded || !t._fw_grad(0).defined(), "the call would lose its arguments' tangents");
    };
    check_one(first);
    for (const OptTensor *t : others)
        if (*t)
            check_one(**t);
    need(first.is_cuda(), "tensors must be on a GPU");
    for (const OptTensor *t : others)
        need(!*t || (*t)->device() == first.device(), "tensors must be on one GPU");
    return first.get_device();
}

int sm_count(int device) { return at::cuda::getDeviceProperties(device)->multiProcessorCount; }

void *data(const OptTensor &t) { return t ? t->data_ptr() : nullptr; }

// New tensors, past the dispatcher (half of a small call's time was spent in it).
Tensor empty(at::IntArrayRef size, ScalarType dtype, const Tensor &like) {
    return at::detail::empty_cuda(size, dtype, like.device(), std::nullopt);
}

// Row `at` of a new tensor [.., width] as a tensor of its own.
Tensor row_of(const Tensor &all, int64_t at) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
    impl->set_storage_offset(at * all.size(1));
    impl->set_sizes_contiguous({all.size(1)});
    return Tensor(std::move(impl));
}

// Code rows start on 16-byte boundaries, so every kernel can read them in vectors.
Tensor empty_codes(const Tensor &like, int64_t rows, int64_t width) {
    return at::detail::empty_strided_cuda({rows, width}, {(width + 15) / 16 * 16, 1}, ScalarType::Float8_e4m3fn,
                                          like.device());
}

Tensor empty_scales(const Tensor &like, int64_t rows, int64_t width) {
    return empty({rows, (width + kCheckpointBlock - 1) / kCheckpointBlock}, ScalarType::Float, like);
}

// Rows that start on 16-byte boundaries, one after the other.
bool on_16_bytes(const Tensor &t, int64_t size) {
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && t.stride(0) * size % 16 == 0 &&
           t.stride(0) >= t.size(1);
}

// One host-mapped word per device that a kernel sets when one of its bounded
// waits ran out (its results are then not to be used).
uint32_t *fault_word(int device) {
    static std::array<std::atomic<uint32_t *>, 64> words{};
    static std::mutex mutex;
    check(device >= 0 && device < int(words.size()), "device index out of range");
    uint32_t *word = words[device].load(std::memory_order_acquire);
    if (word != nullptr)
        return word;
    std::lock_guard<std::mutex> lock(mutex);
    word = words[device].load(std::memory_order_relaxed);
    if (word == nullptr) {
        // Allowed while a graph is captured: the allocation is no part of it.
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        check_cuda(cudaThreadExchangeStreamCaptureMode(&mode), "capture mode");
        void *fresh = nullptr;
        const cudaError_t rc = cudaHostAlloc(&fresh, 64, cudaHostAllocMapped | cudaHostAllocPortable);
        cudaThreadExchangeStreamCaptureMode(&mode);
        check_cuda(rc, "allocate fault word");
        std::memset(fresh, 0, 64);
        word = static_cast<uint32_t *>(fresh);
        words[device].store(word, std::memory_order_release);
    }
    return word;
}

// The word, read before every launch without synchronising: a set one refuses
// all further calls.  Replays of captured calls do not come here (check_readout).
uint32_t *healthy_word(int device) {
    uint32_t *word = fault_word(device);
    check(*static_cast<const volatile uint32_t *>(word) == 0,
          "an earlier read-out kernel on this GPU gave up waiting for its own copies; its results are invalid");
    return word;
}

// (y, codes | None, scales | None, mean | None, rstd | None, shift | None)
py::tuple norm_forward(const Tensor &x, const OptTensor &weight, const OptTensor &bias, double eps,
                       const OptTensor &scales, std::optional<int64_t> hidden, int64_t block,
                       std::optional<ScalarType> dtype, uint32_t keep, bool recorded) {
    need_untraced(recorded);
    need_rows(x, "rows must be [tokens, width] with adjacent columns");
    const int64_t rows = x.size(0), width = x.size(1);
    const bool fp8 = x.scalar_type() == ScalarType::Float8_e4m3fn;
    need(fp8 || is_wide(x.scalar_type()), "rows must be bfloat16, float16, float32 or float8_e4m3fn");
    const ScalarType out = fp8 ? dtype.value_or(ScalarType::BFloat16) : x.scalar_type();
    need(is_wide(out), "dtype must be bfloat16, float16 or float32");
    need(fp8 || !dtype || *dtype == out, "dtype can be chosen for float8_e4m3fn rows only");
    need(fp8 == scales.has_value(), "float8_e4m3fn rows need scales, other rows take none");
    need(eps >= 0, "eps must not be negative");
    need(keep <= kKeepFp8 && !(fp8 && keep == kKeepStats), "float8_e4m3fn rows are kept as \"fp8\" only");
    NormForwardParams p{};
    p.hidden = uint32_t(hidden.value_or(width));
    if (fp8) {
        const int64_t h = hidden.value_or(width);
        need(h >= 1 && h <= width && width % h == 0, "hidden must divide the width");
        need(block >= 1 && block <= (1 << 30), "block must be positive");
        const int64_t packs = (h + block - 1) / block;
        need(scales->dim() == 2 && scales->scalar_type() == ScalarType::Float && scales->size(0) == rows &&
                 scales->size(1) == width / h * packs,
             "scales must be float32 [tokens, width / hidden * ceil(hidden / block)]");
        p.scales = static_cast<const float *>(scales->data_ptr());
        p.scale_row_stride = scales->stride(0);
        p.scale_col_stride = scales->stride(1);
        p.packs = uint32_t(packs);
        p.block = uint32_t(block);
    } else {
        need(!hidden, "hidden describes the scales of float8_e4m3fn rows");
    }
    need_params(weight, bias, width, out);
    const int device = need_device(x, {&weight, &bias, &scales}, recorded);
    c10::cuda::CUDAGuard guard(device);
    const Tensor y = empty({rows, width}, out, x);
    OptTensor codes, code_scales, mean, rstd, shift;
    if (keep == kKeepStats) {
        // One allocation for the three (each takes as long as a check of all arguments).
        const Tensor stats = empty({3, rows}, ScalarType::Float, x);
        mean = row_of(stats, 0);
        shift = row_of(stats, 1);
        rstd = row_of(stats, 2);
    }
    if (keep == kKeepFp8) {
        rstd = empty({rows}, ScalarType::Float, x);
        codes = empty_codes(x, rows, width);
        code_scales = empty_scales(x, rows, width);
    }
    if (rows > 0) {
        p.x = x.data_ptr();
        p.weight = data(weight);
        p.bias = data(bias);
        p.y = y.data_ptr();
        p.mean = static_cast<float *>(data(mean));
        p.shift = static_cast<float *>(data(shift));
        p.rstd = static_cast<float *>(data(rstd));
        p.codes = static_cast<uint8_t *>(data(codes));
        p.code_scales = static_cast<float *>(data(code_scales));
        p.rows = rows;
        p.x_stride = x.stride(0);
        p.codes_stride = codes ? codes->stride(0) : 0;
        p.width = uint32_t(width);
        p.in_type = element_type(x.scalar_type());
        p.out_type = element_type(out);
        p.param_type = weight ? element_type(weight->scalar_type()) : 0;
        p.keep = keep;
        p.eps = float(eps);
        p.fault = healthy_word(device);
        check_cuda(launch_norm_forward(p, sm_count(device), at::cuda::getCurrentCUDAStream(device).stream()),
                   "launch layer norm");
    }
    return py::make_tuple(y, codes, code_scales, mean, rstd, shift);
}

// (dx | None, dweight | None, dbias | None).  Kept rows: (x, mean, rstd, shift | None) or (codes, scales, rstd).
py::tuple norm_backward(const Tensor &dy, const Tensor &kept, const OptTensor &scales, const OptTensor &mean,
                        const Tensor &rstd, const OptTensor &weight, bool want_dx, bool want_params,
                        const OptTensor &shift) {
    need_untraced(false);
    need_rows(dy, "dy must be [tokens, width] with adjacent columns");
    need(is_wide(dy.scalar_type()), "dy must be bfloat16, float16 or float32");
    const int64_t rows = dy.size(0), width = dy.size(1);
    const bool fp8 = scales.has_value();
    need(kept.dim() == 2 && kept.size(0) == rows && kept.size(1) == width, "dy must have the shape of the kept rows");
    if (fp8) {
        need_checkpoint(kept, *scales);
    } else {
        need_rows(kept, "rows must be [tokens, width] with adjacent columns");
        need(kept.scalar_type() == dy.scalar_type(), "dy must have the rows' type");
        need(mean && mean->dim() == 1 && mean->size(0) == rows && mean->scalar_type() == ScalarType::Float &&
                 mean->is_contiguous(),
             "mean must be contiguous float32 [tokens]");
        need(!shift || (shift->dim() == 1 && shift->size(0) == rows && shift->scalar_type() == ScalarType::Float &&
                        shift->is_contiguous()),
             "shift must be contiguous float32 [tokens]");
    }
    need(rstd.dim() == 1 && rstd.size(0) == rows && rstd.scalar_type() == ScalarType::Float && rstd.is_contiguous(),
         "rstd must be contiguous float32 [tokens]");
    need_params(weight, std::nullopt, width, dy.scalar_type());
    const OptTensor kept_opt = kept, rstd_opt = rstd;
    const int device = need_device(dy, {&kept_opt, &scales, &mean, &rstd_opt, &weight, &shift});
    c10::cuda::CUDAGuard guard(device);
    OptTensor dx, dweight, dbias, partial;
    if (want_dx)
        dx = empty({rows, width}, dy.scalar_type(), dy);
    const bool params = want_params && weight.has_value();
    if (params) {
        dweight = empty({width}, weight->scalar_type(), dy);
        dbias = empty({width}, weight->scalar_type(), dy);
    }
    if (rows == 0) {
        if (params) {
            dweight->zero_();
            dbias->zero_();
        }
        return py::make_tuple(dx, dweight, dbias);
    }
    NormBackwardParams p{};
    p.dy = dy.data_ptr();
    p.rstd = static_cast<const float *>(rstd.data_ptr());
    if (fp8) {
        p.codes = static_cast<const uint8_t *>(kept.data_ptr());
        p.code_scales = static_cast<const float *>(scales->data_ptr());
        p.codes_stride = kept.stride(0);
        p.code_scales_stride = scales->stride(0);
        p.scale_col_stride = scales->stride(1);
    } else {
        p.x = kept.data_ptr();
        p.x_stride = kept.stride(0);
        p.mean = static_cast<const float *>(mean->data_ptr());
        p.shift = static_cast<const float *>(data(shift));
    }
    p.weight = data(weight);
    p.dx = data(dx);
    p.dweight = data(dweight);
    p.dbias = data(dbias);
    p.rows = rows;
    p.dy_stride = dy.stride(0);
    p.width = uint32_t(width);
    p.dy_type = element_type(dy.scalar_type());
    p.param_type = weight ? element_type(weight->scalar_type()) : 0;
    p.keep = fp8 ? kKeepFp8 : kKeepStats;
    p.fault = healthy_word(device);
    const int sms = sm_count(device);
    if (params) {
        p.parts = norm_backward_parts(p, sms);
        partial = empty({2, int64_t(p.parts), width}, ScalarType::Float, dy);
        p.partial = static_cast<float *>(partial->data_ptr());
    }
    check_cuda(launch_norm_backward(p, sms, at::cuda::getCurrentCUDAStream(device).stream()),
               "launch layer norm backward");
    return py::make_tuple(dx, dweight, dbias);
}

py::tuple save_fp8(const Tensor &x, bool recorded) {
    need_untraced(recorded);
    need_rows(x, "activations must be [rows, width] with adjacent columns");
    need(is_wide(x.scalar_type()), "activations must be bfloat16, float16 or float32");
    const int device = need_device(x, {}, recorded);
    c10::cuda::CUDAGuard guard(device);
    const int64_t rows = x.size(0), width = x.size(1);
    const Tensor codes = empty_codes(x, rows, width), scales = empty_scales(x, rows, width);
    if (rows > 0) {
        healthy_word(device);
        SaveFp8Params p{};
        p.x = x.data_ptr();
        p.codes = static_cast<uint8_t *>(codes.data_ptr());
        p.scales = static_cast<float *>(scales.data_ptr());
        p.rows = rows;
        p.x_stride = x.stride(0);
        p.codes_stride = codes.stride(0);
        p.width = uint32_t(width);
        p.type = element_type(x.scalar_type());
        check_cuda(launch_save_fp8(p, sm_count(device), at::cuda::getCurrentCUDAStream(device).stream()),
                   "launch 8-bit save");
    }
    return py::make_tuple(codes, scales);
}

Tensor restore_fp8(const Tensor &codes, const Tensor &scales, ScalarType dtype) {
    need_untraced(false);
    need_checkpoint(codes, scales);
    need(is_wide(dtype), "dtype must be bfloat16, float16 or float32");
    const OptTensor scales_opt = scales;
    const int device = need_device(codes, {&scales_opt});
    c10::cuda::CUDAGuard guard(device);
    const int64_t rows = codes.size(0), width = codes.size(1);
    const Tensor x = empty({rows, width}, dtype, codes);
    if (rows > 0) {
        healthy_word(device);
        RestoreFp8Params p{};
        p.codes = static_cast<const uint8_t *>(codes.data_ptr());
        p.scales = static_cast<const float *>(scales.data_ptr());
        p.x = x.data_ptr();
        p.rows = rows;
        p.codes_stride = codes.stride(0);
        p.scale_row_stride = scales.stride(0);
        p.scale_col_stride = scales.stride(1);
        p.width = uint32_t(width);
        p.type = element_type(dtype);
        check_cuda(launch_restore_fp8(p, sm_count(device), at::cuda::getCurrentCUDAStream(device).stream()),
                   "launch 8-bit restore");
    }
    return x;
}

// (dweight [out, width], dbias [out] | None)
py::tuple fp8_weight_grad(const Tensor &dy, const Tensor &codes, const Tensor &scales, const OptTensor &norm_weight,
                          const OptTensor &norm_bias, std::optional<ScalarType> dtype, bool want_bias) {
    need_untraced(false);
    need_rows(dy, "dy must be [rows, out] with adjacent columns");
    need(is_wide(dy.scalar_type()), "dy must be bfloat16, float16 or float32");
    need_checkpoint(codes, scales);
    need(dy.size(0) == codes.size(0), "dy and codes must have the same rows");
    const ScalarType result = dtype.value_or(dy.scalar_type());
    need(result == dy.scalar_type() || result == ScalarType::Float, "dtype must be dy's type or float32");
    const int64_t rows = dy.size(0), out = dy.size(1), width = codes.size(1);
    need_params(norm_weight, norm_bias, width, dy.scalar_type());
    const OptTensor codes_opt = codes, scales_opt = scales;
    const int device = need_device(dy, {&codes_opt, &scales_opt, &norm_weight, &norm_bias});
    c10::cuda::CUDAGuard guard(device);
    const Tensor dweight = empty({out, width}, result, dy);
    OptTensor dbias, sums;
    if (want_bias)
        dbias = empty({out}, result, dy);
    if (rows == 0) {
        dweight.zero_();
        if (dbias)
            dbias->zero_();
        return py::make_tuple(dweight, dbias);
    }
    uint32_t *fault = healthy_word(device);
    // Tiled copies want rows on 16-byte boundaries; others are copied first.
    Tensor rows_codes = codes;
    if (!on_16_bytes(codes, 1)) {
        rows_codes = empty_codes(codes, rows, width);
        rows_codes.copy_(codes);
    }
    WeightGradParams p{};
    p.dy = dy.data_ptr();
    p.codes = static_cast<const uint8_t *>(rows_codes.data_ptr());
    p.scales = static_cast<const float *>(scales.data_ptr());
    p.norm_weight = data(norm_weight);
    p.norm_bias = data(norm_bias);
    p.dweight = dweight.data_ptr();
    p.dbias = data(dbias);
    p.fault = fault;
    p.rows = rows;
    p.dy_stride = dy.stride(0);
    p.codes_stride = rows_codes.stride(0);
    p.scale_row_stride = scales.stride(0);
    p.scale_col_stride = scales.stride(1);
    p.width = uint32_t(width);
    p.out = uint32_t(out);
    p.type = element_type(dy.scalar_type());
    p.param_type = norm_weight ? element_type(norm_weight->scalar_type()) : 0;
    p.out_type = element_type(result);
    plan_weight_grad(p, sm_count(device));
    OptTensor planes, dw_parts;
    if (want_bias || norm_bias) {
        sums = empty({int64_t(p.sum_rows) + 1, out}, ScalarType::Float, dy);
        p.dy_sums = static_cast<float *>(sums->data_ptr());
        p.sum_parts = p.dy_sums + out;
    }
    if (p.planes > 1 || !on_16_bytes(dy, 2)) {
        p.plane_stride = (out + 7) / 8 * 8;
        planes = empty({int64_t(p.planes), rows, p.plane_stride}, ScalarType::BFloat16, dy);
        p.dy_planes = planes->data_ptr();
    }
    if (p.parts > 1) {
        dw_parts = empty({int64_t(p.slots), out, width}, ScalarType::Float, dy);
        p.dw_parts = static_cast<float *>(dw_parts->data_ptr());
    }
    check_cuda(launch_weight_grad(p, at::cuda::getCurrentCUDAStream(device).stream()), "launch weight gradient");
    return py::make_tuple(dweight, dbias);
}

} // namespace

void bind_readout(py::module_ &m) {
    m.def("norm_forward", &norm_forward, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"),
          py::arg("scales"), py::arg("hidden"), py::arg("block"), py::arg("dtype"), py::arg("keep"),
          py::arg("recorded") = false);
    m.def("norm_backward", &norm_backward, py::arg("dy"), py::arg("kept"), py::arg("scales"), py::arg("mean"),
          py::arg("rstd"), py::arg("weight"), py::arg("want_dx"), py::arg("want_params"), py::arg("shift"));
    m.def(
        "check_readout", [](int device) { healthy_word(device); }, py::arg("device"),
        "Raise if a read-out kernel on this GPU gave up waiting.");
    m.def(
        "debug_readout_fault",
        [](int device, uint32_t code) { return std::exchange(*static_cast<volatile uint32_t *>(fault_word(device)), code); },
        py::arg("device"), py::arg("code"), "Replace a device's fault word (tests of how a given-up wait is reported).");
    m.def("save_fp8", &save_fp8, py::arg("x"), py::arg("recorded") = false);
    m.def("restore_fp8", &restore_fp8, py::arg("codes"), py::arg("scales"), py::arg("dtype"));
    m.def("fp8_weight_grad", &fp8_weight_grad, py::arg("dy"), py::arg("codes"), py::arg("scales"),
          py::arg("norm_weight"), py::arg("norm_bias"), py::arg("dtype"), py::arg("want_bias"));
}

} // namespace engram
