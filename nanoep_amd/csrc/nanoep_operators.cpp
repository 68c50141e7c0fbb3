// The host side of the expert layer's operators: argument checks, outputs, the caller's stream, one call of the
// C ABI each.  Everything runs on the current stream of the inputs' device, and outputs come from that stream's
// pool; a caller whose inputs were made on another stream orders the two as for any torch operator.

#include "nanoep_operators_host.h"

#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>

#include <initializer_list>
#include <optional>
#include <sstream>
#include <tuple>

#include "nanoep_hip.h"

namespace nanoep {
namespace {

using Device = c10::Device;
using DeviceGuard = c10::hip::HIPGuardMasqueradingAsCUDA;

constexpr int64_t kScaleBlock = 128;

template <class... Parts>
[[noreturn]] void refuse(const Parts&... parts) {
    std::ostringstream text;
    (text << ... << parts);
    throw py::value_error(text.str());
}

void check(int status, const char* what) {
    TORCH_CHECK(status == NANOEP_OK, "nanoep ", what, " failed: ", nanoep_status_string(status), " ", nanoep_last_hip_error());
}

void* current_stream(const Device& device) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index()).stream(); }

torch::Tensor make(at::IntArrayRef sizes, at::ScalarType dtype, const Device& device) {
    const auto& context = at::globalContext();
    if (C10_UNLIKELY(context.deterministicAlgorithms() && context.deterministicFillUninitializedMemory()))
        return torch::empty(sizes, torch::TensorOptions().dtype(dtype).device(device));
    return torch::Tensor(at::detail::empty_cuda(sizes, dtype, device, std::nullopt));
}

// Rows of another type within a tensor of records, made without the dispatcher; a view for autograd's version counter.
torch::Tensor rows_within(const torch::Tensor& base, at::ScalarType dtype, int64_t offset, int64_t rows, int64_t columns, int64_t row_stride) {
    auto part = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(base.storage()), base.key_set(),
                                                         c10::scalarTypeToTypeMeta(dtype));
    auto* impl = part.unsafeGetTensorImpl();
    const int64_t sizes[] = {rows, columns}, strides[] = {row_stride, 1};
    impl->set_sizes_and_strides(sizes, strides, offset);
    if (!base.is_inference())
        impl->set_version_counter(base.unsafeGetTensorImpl()->version_counter());
    return part;
}

void require_gpu(const torch::Tensor& tensor, const char* what, const char* name) {
    if (!tensor.is_cuda())
        refuse(what, " ", name, " must be a CUDA tensor");
}

void require(const torch::Tensor& tensor, const Device& device, at::ScalarType dtype, std::initializer_list<int64_t> sizes, const char* what,
             const char* name) {
    bool fits = tensor.device() == device && tensor.scalar_type() == dtype && tensor.dim() == static_cast<int64_t>(sizes.size()) &&
                tensor.is_contiguous();
    int64_t d = 0;
    for (const int64_t size : sizes)
        fits = fits && tensor.size(d++) == size;
    if (!fits) {
        std::ostringstream shape;
        d = 0;
        for (const int64_t size : sizes)
            shape << (d++ ? ", " : "") << size;
        refuse(what, " ", name, " must be contiguous ", c10::toString(dtype), " of shape [", shape.str(), "] on ", device.str());
    }
}

// Kernels move 16 bytes at a time; a view may start anywhere.
void require_aligned(const torch::Tensor& tensor, const char* what, const char* name) {
    if (reinterpret_cast<uintptr_t>(tensor.data_ptr()) % 16 != 0)
        refuse(what, " ", name, " must start at a multiple of 16 bytes");
}

// Forward mode goes by the tensors alone: torch.no_grad() leaves it on.
void require_no_tangent(const char* what, std::initializer_list<const torch::Tensor*> tensors) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode())
        return;
    for (const torch::Tensor* tensor : tensors)
        TORCH_CHECK(tensor == nullptr || !tensor->_fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative");
}

void require_no_gradient(const char* what, std::initializer_list<const torch::Tensor*> tensors) {
    require_no_tangent(what, tensors);
    if (!at::GradMode::is_enabled())
        return;
    for (const torch::Tensor* tensor : tensors)
        TORCH_CHECK(tensor == nullptr || !tensor->requires_grad(), what, " has no gradient: call it under torch.no_grad() or detach its inputs");
}

const void* pointer_of(const std::optional<torch::Tensor>& tensor) { return tensor.has_value() ? tensor->data_ptr() : nullptr; }

struct Records {
    torch::Tensor payload, values, scales;
};

Records make_records(int64_t rows, int64_t columns, const Device& device) {
    const int64_t bytes = nanoep_fp8_record_bytes(columns);
    Records made;
    made.payload = make({rows, bytes / 2}, at::kBFloat16, device);
    made.values = rows_within(made.payload, at::kFloat8_e4m3fn, 0, rows, columns, bytes);
    made.scales = rows_within(made.payload, at::kFloat, columns / 4, rows, (columns + kScaleBlock - 1) / kScaleBlock, bytes / 4);
    return made;
}

using NormOutputs = std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, std::optional<torch::Tensor>, std::optional<torch::Tensor>>;

NormOutputs rms_norm_fp8(const torch::Tensor& x, const torch::Tensor& gamma, const std::optional<torch::Tensor>& residual, double eps,
                         bool normalized) {
    const char* what = "rms_norm_fp8";
    require_gpu(x, what, "x");
    if (x.dim() != 2)
        refuse(what, " x must be [tokens, hidden]");
    const Device device = x.device();
    const int64_t tokens = x.size(0), hidden = x.size(1);
    if (hidden <= 0 || hidden % 16 != 0 || hidden > 65536)
        refuse(what, " hidden must be a positive multiple of 16 and at most 65536");
    if (!(eps >= 0.0))
        refuse(what, " eps must not be negative");
    require(x, device, at::kBFloat16, {tokens, hidden}, what, "x");
    require(gamma, device, at::kBFloat16, {hidden}, what, "gamma");
    require_aligned(x, what, "x");
    require_aligned(gamma, what, "gamma");
    if (residual.has_value()) {
        require(*residual, device, at::kBFloat16, {tokens, hidden}, what, "residual");
        require_aligned(*residual, what, "residual");
    }
    require_no_gradient(what, {&x, &gamma, residual.has_value() ? &*residual : nullptr});
    const DeviceGuard guard(device);
    Records rows = make_records(tokens, hidden, device);
    std::optional<torch::Tensor> sum, plain;
    if (residual.has_value())
        sum = make({tokens, hidden}, at::kBFloat16, device);
    if (normalized)
        plain = make({tokens, hidden}, at::kBFloat16, device);
    check(nanoep_rms_norm_fp8(x.data_ptr(), pointer_of(residual), gamma.data_ptr(), tokens, static_cast<int>(hidden), static_cast<float>(eps),
                              rows.payload.data_ptr(), const_cast<void*>(pointer_of(sum)), const_cast<void*>(pointer_of(plain)),
                              current_stream(device)),
          what);
    return {rows.payload, rows.values, rows.scales, sum, plain};
}

struct ProductArguments {
    int64_t rows, inner, columns, experts;
    const int64_t* offsets;
    const int64_t* counts;
};

ProductArguments require_product(const char* what, const torch::Tensor& values, const torch::Tensor& scales, const torch::Tensor& weight,
                                 const torch::Tensor& weight_scales, const std::optional<torch::Tensor>& expert_offsets,
                                 const std::optional<torch::Tensor>& expert_counts, int64_t column_multiple) {
    require_gpu(values, what, "values");
    const Device device = values.device();
    if (values.dim() != 2 || values.scalar_type() != at::kFloat8_e4m3fn || (values.numel() > 0 && values.stride(1) != 1))
        refuse(what, " values must be float8_e4m3fn [rows, inner] with neighbouring columns");
    const int64_t rows = values.size(0), inner = values.size(1);
    if (inner <= 0 || inner % 16 != 0 || inner > (1 << 24))
        refuse(what, " inner must be a positive multiple of 16 and at most 2^24");
    if (rows > 0x7fffffff)
        refuse(what, " takes fewer than 2^31 rows");
    const int64_t groups = (inner + kScaleBlock - 1) / kScaleBlock;
    if (rows > 1 && (values.stride(0) < inner || values.stride(0) % 16 != 0))
        refuse(what, " values must have rows a multiple of 16 bytes apart");
    if (scales.device() != device || scales.dim() != 2 || scales.scalar_type() != at::kFloat || scales.size(0) != rows ||
        scales.size(1) != groups || (rows > 0 && groups > 1 && scales.stride(1) != 1) || (rows > 1 && scales.stride(0) < groups))
        refuse(what, " scales must be float32 [rows, ceil(inner / 128)] with neighbouring columns, on the values' device");
    if (weight.dim() != 3)
        refuse(what, " weight must be [experts, columns, inner]");
    const int64_t experts = weight.size(0), columns = weight.size(1);
    if (experts <= 0 || experts >= (1 << 30) || columns <= 0 || columns % column_multiple != 0 || columns > (1 << 24))
        refuse(what, " weight must have at least one expert and a positive multiple of ", column_multiple, " columns, at most 2^24");
    require(weight, device, at::kFloat8_e4m3fn, {experts, columns, inner}, what, "weight");
    require(weight_scales, device, at::kFloat, {experts, (columns + kScaleBlock - 1) / kScaleBlock, groups}, what, "weight scales");
    require_aligned(values, what, "values");
    require_aligned(weight, what, "weight");
    if (expert_offsets.has_value() != expert_counts.has_value())
        refuse(what, " takes expert_offsets and expert_counts together");
    if (expert_offsets.has_value()) {
        require(*expert_offsets, device, at::kLong, {experts + 1}, what, "expert_offsets");
        require(*expert_counts, device, at::kLong, {experts}, what, "expert_counts");
    } else if (experts != 1) {
        refuse(what, " without expert_offsets takes the weight of one expert");
    }
    return {rows, inner, columns, experts, static_cast<const int64_t*>(pointer_of(expert_offsets)),
            static_cast<const int64_t*>(pointer_of(expert_counts))};
}

// A single row's stride says nothing.
int64_t row_stride(const torch::Tensor& tensor, int64_t least, int64_t multiple) {
    if (tensor.size(0) > 1)
        return tensor.stride(0);
    return (least + multiple - 1) / multiple * multiple;
}

torch::Tensor experts_linear(const torch::Tensor& values, const torch::Tensor& scales, const torch::Tensor& weight,
                             const torch::Tensor& weight_scales, const std::optional<torch::Tensor>& expert_offsets,
                             const std::optional<torch::Tensor>& expert_counts) {
    const char* what = "experts_linear";
    const ProductArguments p = require_product(what, values, scales, weight, weight_scales, expert_offsets, expert_counts, 8);
    require_no_gradient(what, {&values, &scales, &weight, &weight_scales});
    const Device device = values.device();
    const DeviceGuard guard(device);
    torch::Tensor out = make({p.rows, p.columns}, at::kBFloat16, device);
    check(nanoep_experts_linear(values.data_ptr(), row_stride(values, p.inner, 16), static_cast<const float*>(scales.data_ptr()),
                                row_stride(scales, scales.size(1), 1), weight.data_ptr(), static_cast<const float*>(weight_scales.data_ptr()),
                                p.offsets, p.counts, p.rows, p.experts, static_cast<int>(p.inner), static_cast<int>(p.columns), out.data_ptr(),
                                current_stream(device)),
          what);
    return out;
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> experts_gated(const torch::Tensor& values, const torch::Tensor& scales,
                                                                      const torch::Tensor& weight, const torch::Tensor& weight_scales,
                                                                      const std::optional<torch::Tensor>& expert_offsets,
                                                                      const std::optional<torch::Tensor>& expert_counts) {
    const char* what = "experts_gated";
    const ProductArguments p = require_product(what, values, scales, weight, weight_scales, expert_offsets, expert_counts, 32);
    require_no_gradient(what, {&values, &scales, &weight, &weight_scales});
    const Device device = values.device();
    const DeviceGuard guard(device);
    Records rows = make_records(p.rows, p.columns / 2, device);
    const int64_t value_stride = row_stride(values, p.inner, 16), scale_stride = row_stride(scales, scales.size(1), 1);
    const size_t bytes = nanoep_experts_gated_workspace_bytes(p.rows, p.experts, static_cast<int>(p.inner), static_cast<int>(p.columns),
                                                              value_stride, scale_stride);
    torch::Tensor workspace;
    if (bytes > 0)
        workspace = make({static_cast<int64_t>(bytes)}, at::kByte, device);
    check(nanoep_experts_gated(values.data_ptr(), value_stride, static_cast<const float*>(scales.data_ptr()), scale_stride, weight.data_ptr(), static_cast<const float*>(weight_scales.data_ptr()),
                               p.offsets, p.counts, p.rows, p.experts, static_cast<int>(p.inner), static_cast<int>(p.columns),
                               rows.payload.data_ptr(), bytes > 0 ? workspace.data_ptr() : nullptr, bytes, current_stream(device)),
          what);
    return {rows.payload, rows.values, rows.scales};
}

struct WeightedArguments {
    int64_t tokens, topk, hidden;
};

WeightedArguments require_weighted(const char* what, const torch::Tensor& y, const torch::Tensor& token_slots, const torch::Tensor& weights) {
    require_gpu(y, what, "y");
    const Device device = y.device();
    if (y.dim() != 2 || token_slots.dim() != 2)
        refuse(what, " y must be [rows, hidden] and token_slots [tokens, topk]");
    const int64_t hidden = y.size(1), tokens = token_slots.size(0), topk = token_slots.size(1);
    if (hidden <= 0 || hidden % 8 != 0 || hidden > (1 << 24))
        refuse(what, " hidden must be a positive multiple of 8 and at most 2^24");
    if (topk < 1 || topk > 32)
        refuse(what, " takes 1 to 32 choices a token");
    if (y.size(0) > 0x7fffffff || tokens > 0x7fffffff / 32)
        refuse(what, " takes fewer than 2^31 rows and 2^26 tokens");
    require(y, device, at::kBFloat16, {y.size(0), hidden}, what, "y");
    require(token_slots, device, at::kInt, {tokens, topk}, what, "token_slots");
    require(weights, device, at::kFloat, {tokens, topk}, what, "weights");
    require_aligned(y, what, "y");
    return {tokens, topk, hidden};
}

// The experts of a layout, 0 without one.
int64_t require_layout(const char* what, const Device& device, const std::optional<torch::Tensor>& expert_offsets,
                       const std::optional<torch::Tensor>& expert_counts) {
    if (expert_offsets.has_value() != expert_counts.has_value())
        refuse(what, " takes expert_offsets and expert_counts together");
    if (!expert_counts.has_value())
        return 0;
    const int64_t experts = expert_counts->numel();
    if (experts <= 0 || experts >= (1 << 30))
        refuse(what, " expert_counts must name at least one expert");
    require(*expert_counts, device, at::kLong, {experts}, what, "expert_counts");
    require(*expert_offsets, device, at::kLong, {experts + 1}, what, "expert_offsets");
    return experts;
}

// (the layout is for the gradient; what is wrong with it is said here)
torch::Tensor combine_weighted(const torch::Tensor& y, const torch::Tensor& token_slots, const torch::Tensor& weights,
                               const std::optional<torch::Tensor>& bias, const std::optional<torch::Tensor>& expert_offsets,
                               const std::optional<torch::Tensor>& expert_counts) {
    const char* what = "combine_weighted";
    const WeightedArguments a = require_weighted(what, y, token_slots, weights);
    const Device device = y.device();
    require_layout(what, device, expert_offsets, expert_counts);
    if (bias.has_value()) {
        require(*bias, device, at::kBFloat16, {a.tokens, a.hidden}, what, "bias");
        require_aligned(*bias, what, "bias");
    }
    require_no_tangent(what, {&y, &weights, bias.has_value() ? &*bias : nullptr});
    const DeviceGuard guard(device);
    torch::Tensor out = make({a.tokens, a.hidden}, at::kBFloat16, device);
    check(nanoep_combine_weighted(y.data_ptr(), y.size(0), static_cast<const int32_t*>(token_slots.data_ptr()),
                                  static_cast<const float*>(weights.data_ptr()), pointer_of(bias), a.tokens, static_cast<int>(a.hidden),
                                  static_cast<int>(a.topk), out.data_ptr(), current_stream(device)),
          what);
    return out;
}

std::tuple<torch::Tensor, torch::Tensor> combine_weighted_backward(const torch::Tensor& grad, const torch::Tensor& y,
                                                                   const torch::Tensor& token_slots, const torch::Tensor& weights,
                                                                   const std::optional<torch::Tensor>& expert_offsets,
                                                                   const std::optional<torch::Tensor>& expert_counts) {
    const char* what = "combine_weighted_backward";
    const WeightedArguments a = require_weighted(what, y, token_slots, weights);
    const Device device = y.device();
    require(grad, device, at::kBFloat16, {a.tokens, a.hidden}, what, "grad");
    require_aligned(grad, what, "grad");
    const int64_t experts = require_layout(what, device, expert_offsets, expert_counts);
    require_no_gradient(what, {&grad, &y, &weights});
    const DeviceGuard guard(device);
    torch::Tensor grad_y = make({y.size(0), a.hidden}, at::kBFloat16, device);
    torch::Tensor grad_weights = make({a.tokens, a.topk}, at::kFloat, device);
    check(nanoep_combine_weighted_backward(grad.data_ptr(), y.data_ptr(), y.size(0), static_cast<const int32_t*>(token_slots.data_ptr()),
                                           static_cast<const float*>(weights.data_ptr()),
                                           static_cast<const int64_t*>(pointer_of(expert_offsets)),
                                           static_cast<const int64_t*>(pointer_of(expert_counts)), experts, a.tokens,
                                           static_cast<int>(a.hidden), static_cast<int>(a.topk), grad_y.data_ptr(),
                                           static_cast<float*>(grad_weights.data_ptr()), current_stream(device)),
          what);
    return {grad_y, grad_weights};
}

}  // namespace

void bind_operators(py::module_& module) {
    module.def("rms_norm_fp8", &rms_norm_fp8, py::arg("x"), py::arg("gamma"), py::arg("residual"), py::arg("eps"), py::arg("normalized"),
               py::call_guard<py::gil_scoped_release>());
    module.def("experts_linear", &experts_linear, py::arg("values"), py::arg("scales"), py::arg("weight"), py::arg("weight_scales"),
               py::arg("expert_offsets"), py::arg("expert_counts"), py::call_guard<py::gil_scoped_release>());
    module.def("experts_gated", &experts_gated, py::arg("values"), py::arg("scales"), py::arg("weight"), py::arg("weight_scales"),
               py::arg("expert_offsets"), py::arg("expert_counts"), py::call_guard<py::gil_scoped_release>());
    module.def("combine_weighted", &combine_weighted, py::arg("y"), py::arg("token_slots"), py::arg("weights"), py::arg("bias"),
               py::arg("expert_offsets"), py::arg("expert_counts"), py::call_guard<py::gil_scoped_release>());
    module.def("combine_weighted_backward", &combine_weighted_backward, py::arg("grad"), py::arg("y"), py::arg("token_slots"),
               py::arg("weights"), py::arg("expert_offsets"), py::arg("expert_counts"), py::call_guard<py::gil_scoped_release>());
}

}  // namespace nanoep
