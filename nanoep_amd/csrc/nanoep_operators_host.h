// What the hosts of the operators (nanoep_operators.cpp, nanoep_entry.cpp) share, and what nanoep_torch.cpp, which makes the module,
// needs of them.
#ifndef NANOEP_OPERATORS_HOST_H_
#define NANOEP_OPERATORS_HOST_H_

#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <torch/extension.h>

#include <initializer_list>
#include <optional>
#include <sstream>

#include "nanoep_hip.h"

namespace py = pybind11;

namespace nanoep {

// Adds the expert layer's operators, and those of its entry, to the module.
void bind_operators(py::module_& module);
void bind_entry(py::module_& module);

namespace host {

using Device = c10::Device;
using DeviceGuard = c10::hip::HIPGuardMasqueradingAsCUDA;

template <class... Parts>
[[noreturn]] void refuse(const Parts&... parts) {
    std::ostringstream text;
    (text << ... << parts);
    throw py::value_error(text.str());
}

inline void check(int status, const char* what) {
    TORCH_CHECK(status == NANOEP_OK, "nanoep ", what, " failed: ", nanoep_status_string(status), " ", nanoep_last_hip_error());
}

inline void* current_stream(const Device& device) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index()).stream(); }

inline torch::Tensor make(at::IntArrayRef sizes, at::ScalarType dtype, const Device& device) {
    const auto& context = at::globalContext();
    if (C10_UNLIKELY(context.deterministicAlgorithms() && context.deterministicFillUninitializedMemory()))
        return torch::empty(sizes, torch::TensorOptions().dtype(dtype).device(device));
    return torch::Tensor(at::detail::empty_cuda(sizes, dtype, device, std::nullopt));
}

inline void require_gpu(const torch::Tensor& tensor, const char* what, const char* name) {
    if (!tensor.is_cuda())
        refuse(what, " ", name, " must be a CUDA tensor");
}

inline void require(const torch::Tensor& tensor, const Device& device, at::ScalarType dtype, std::initializer_list<int64_t> sizes, const char* what,
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
inline void require_aligned(const torch::Tensor& tensor, const char* what, const char* name) {
    if (reinterpret_cast<uintptr_t>(tensor.data_ptr()) % 16 != 0)
        refuse(what, " ", name, " must start at a multiple of 16 bytes");
}

// Forward mode goes by the tensors alone: torch.no_grad() leaves it on.
inline void require_no_tangent(const char* what, std::initializer_list<const torch::Tensor*> tensors) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode())
        return;
    for (const torch::Tensor* tensor : tensors)
        TORCH_CHECK(tensor == nullptr || !tensor->_fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative");
}

inline void require_no_gradient(const char* what, std::initializer_list<const torch::Tensor*> tensors) {
    require_no_tangent(what, tensors);
    if (!at::GradMode::is_enabled())
        return;
    for (const torch::Tensor* tensor : tensors)
        TORCH_CHECK(tensor == nullptr || !tensor->requires_grad(), what, " has no gradient: call it under torch.no_grad() or detach its inputs");
}

inline const void* pointer_of(const std::optional<torch::Tensor>& tensor) { return tensor.has_value() ? tensor->data_ptr() : nullptr; }

}  // namespace host
}  // namespace nanoep

#endif  // NANOEP_OPERATORS_HOST_H_
