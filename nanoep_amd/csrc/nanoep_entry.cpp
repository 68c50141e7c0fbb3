// The host side of what is at an expert layer's entry (norms, router, balance loss) and of its gradients: argument checks, outputs,
// workspaces, the caller's stream, one call of the C ABI each, as nanoep_operators.cpp has it for the operators behind them.

#include "nanoep_operators_host.h"

#include <tuple>

namespace nanoep {

using namespace host;

namespace {

using MaybeTensor = std::optional<torch::Tensor>;

const torch::Tensor* given(const MaybeTensor& tensor) { return tensor.has_value() ? &*tensor : nullptr; }

int type_of(at::ScalarType type) { return type == at::kFloat ? NANOEP_FP32 : NANOEP_BF16; }

bool known_type(at::ScalarType type) { return type == at::kBFloat16 || type == at::kFloat; }

void* address(const MaybeTensor& tensor) { return tensor.has_value() ? tensor->data_ptr() : nullptr; }

// ------------------------------------------------------------------ norms

struct NormArguments {
    int64_t tokens, hidden;
    at::ScalarType rows, parameters;
};

// rows [tokens, hidden] and gamma.
NormArguments require_norm(const char* what, const torch::Tensor& rows, const char* name, const torch::Tensor& gamma) {
    require_gpu(rows, what, name);
    if (rows.dim() != 2 || !known_type(rows.scalar_type()))
        refuse(what, " ", name, " must be bfloat16 or float32 [tokens, hidden]");
    const int64_t tokens = rows.size(0), hidden = rows.size(1);
    if (hidden <= 0 || hidden % 8 != 0 || hidden > 16384)
        refuse(what, " hidden must be a positive multiple of 8 and at most 16384");
    if (tokens > 0x7fffffff)
        refuse(what, " takes fewer than 2^31 tokens");
    if (gamma.scalar_type() != rows.scalar_type() && gamma.scalar_type() != at::kFloat)
        refuse(what, " gamma must have the type of ", name, " or be float32");
    require(rows, rows.device(), rows.scalar_type(), {tokens, hidden}, what, name);
    require(gamma, rows.device(), gamma.scalar_type(), {hidden}, what, "gamma");
    require_aligned(rows, what, name);
    require_aligned(gamma, what, "gamma");
    return {tokens, hidden, rows.scalar_type(), gamma.scalar_type()};
}

void require_rows(const char* what, const torch::Tensor& tensor, const NormArguments& a, const Device& device, const char* name) {
    require(tensor, device, a.rows, {a.tokens, a.hidden}, what, name);
    require_aligned(tensor, what, name);
}

// normalized, total (with a residual), mean (of a layer norm), rstd.
std::tuple<torch::Tensor, MaybeTensor, MaybeTensor, torch::Tensor> norm(const char* what, const torch::Tensor& x, const torch::Tensor& gamma,
                                                                        const MaybeTensor& beta, const MaybeTensor& residual, double eps,
                                                                        bool centred) {
    const NormArguments a = require_norm(what, x, "x", gamma);
    const Device device = x.device();
    if (!(eps >= 0.0))
        refuse(what, " eps must not be negative");
    if (beta.has_value()) {
        require(*beta, device, a.parameters, {a.hidden}, what, "beta");
        require_aligned(*beta, what, "beta");
    }
    if (residual.has_value())
        require_rows(what, *residual, a, device, "residual");
    require_no_tangent(what, {&x, &gamma, given(beta), given(residual)});
    const DeviceGuard guard(device);
    torch::Tensor normalized = make({a.tokens, a.hidden}, a.rows, device), rstd = make({a.tokens}, at::kFloat, device);
    MaybeTensor total, mean;
    if (residual.has_value())
        total = make({a.tokens, a.hidden}, a.rows, device);
    if (centred)
        mean = make({a.tokens}, at::kFloat, device);
    check(nanoep_layer_norm(x.data_ptr(), pointer_of(residual), gamma.data_ptr(), pointer_of(beta), a.tokens, static_cast<int>(a.hidden),
                            static_cast<float>(eps), type_of(a.rows), type_of(a.parameters), address(total), normalized.data_ptr(),
                            static_cast<float*>(address(mean)), static_cast<float*>(rstd.data_ptr()), current_stream(device)),
          what);
    return {normalized, total, mean, rstd};
}

auto layer_norm(const torch::Tensor& x, const torch::Tensor& gamma, const MaybeTensor& beta, const MaybeTensor& residual, double eps) {
    return norm("layer_norm", x, gamma, beta, residual, eps, true);
}

auto rms_norm(const torch::Tensor& x, const torch::Tensor& gamma, const MaybeTensor& residual, double eps) {
    return norm("rms_norm", x, gamma, std::nullopt, residual, eps, false);
}

// grad_x, grad_gamma, grad_beta.
std::tuple<MaybeTensor, MaybeTensor, MaybeTensor> norm_backward(const char* what, const torch::Tensor& grad, const torch::Tensor& total,
                                                                const torch::Tensor& gamma, const MaybeTensor& mean, const torch::Tensor& rstd,
                                                                const MaybeTensor& grad_residual, bool input, bool parameters) {
    const NormArguments a = require_norm(what, total, "total", gamma);
    const Device device = total.device();
    require_rows(what, grad, a, device, "grad");
    if (mean.has_value())
        require(*mean, device, at::kFloat, {a.tokens}, what, "mean");
    require(rstd, device, at::kFloat, {a.tokens}, what, "rstd");
    if (grad_residual.has_value())
        require_rows(what, *grad_residual, a, device, "grad_residual");
    if (!input && !parameters)
        refuse(what, " is asked for no gradient");
    require_no_gradient(what, {&grad, &total, &gamma, given(mean), &rstd, given(grad_residual)});
    const DeviceGuard guard(device);
    MaybeTensor grad_x, grad_gamma, grad_beta;
    torch::Tensor workspace;
    size_t bytes = 0;
    if (input)
        grad_x = make({a.tokens, a.hidden}, a.rows, device);
    if (parameters) {
        grad_gamma = make({a.hidden}, a.parameters, device);
        if (mean.has_value())
            grad_beta = make({a.hidden}, a.parameters, device);
        bytes = nanoep_layer_norm_backward_workspace_bytes(a.tokens, static_cast<int>(a.hidden), type_of(a.rows));
        if (bytes > 0)
            workspace = make({static_cast<int64_t>(bytes)}, at::kByte, device);
    }
    check(nanoep_layer_norm_backward(grad.data_ptr(), total.data_ptr(), gamma.data_ptr(), static_cast<const float*>(pointer_of(mean)),
                                     static_cast<const float*>(rstd.data_ptr()), pointer_of(grad_residual), a.tokens, static_cast<int>(a.hidden),
                                     type_of(a.rows), type_of(a.parameters), address(grad_x), address(grad_gamma), address(grad_beta),
                                     bytes > 0 ? workspace.data_ptr() : nullptr, bytes, current_stream(device)),
          what);
    return {grad_x, grad_gamma, grad_beta};
}

auto layer_norm_backward(const torch::Tensor& grad, const torch::Tensor& total, const torch::Tensor& gamma, const torch::Tensor& mean,
                         const torch::Tensor& rstd, const MaybeTensor& grad_residual, bool input, bool parameters) {
    return norm_backward("layer_norm_backward", grad, total, gamma, mean, rstd, grad_residual, input, parameters);
}

auto rms_norm_backward(const torch::Tensor& grad, const torch::Tensor& total, const torch::Tensor& gamma, const torch::Tensor& rstd,
                       const MaybeTensor& grad_residual, bool input, bool parameters) {
    return norm_backward("rms_norm_backward", grad, total, gamma, std::nullopt, rstd, grad_residual, input, parameters);
}

// ------------------------------------------------------------------ router

struct RouterArguments {
    int64_t tokens, stride;
    int experts, type;
};

RouterArguments require_logits(const char* what, const torch::Tensor& logits) {
    require_gpu(logits, what, "logits");
    if (logits.dim() != 2 || !known_type(logits.scalar_type()))
        refuse(what, " logits must be bfloat16 or float32 [tokens, experts]");
    const int64_t tokens = logits.size(0), experts = logits.size(1);
    if (experts < 1 || experts > 4096)
        refuse(what, " takes 1 to 4096 experts");
    if (tokens > 0x7fffffff / 32)
        refuse(what, " takes fewer than 2^26 tokens");
    const int64_t stride = tokens > 1 ? logits.stride(0) : experts;  // (a single row's says nothing)
    if (tokens > 0 && ((experts > 1 && logits.stride(1) != 1) || stride < experts || stride > int64_t{1} << 31))
        refuse(what, " logits must have neighbouring experts, and tokens that do not overlap and are at most 2^31 elements apart");
    return {tokens, tokens > 0 ? stride : experts, static_cast<int>(experts), type_of(logits.scalar_type())};
}

int require_topk(const char* what, int64_t topk) {
    if (topk < 1 || topk > 32)
        refuse(what, " takes 1 to 32 choices a token");
    return static_cast<int>(topk);
}

int require_ids(const char* what, const torch::Tensor& ids, const RouterArguments& a, const Device& device) {
    if (ids.dim() != 2)
        refuse(what, " ids must be [tokens, topk]");
    const int topk = require_topk(what, ids.size(1));
    require(ids, device, at::kLong, {a.tokens, ids.size(1)}, what, "ids");
    return topk;
}

std::tuple<torch::Tensor, torch::Tensor> route_topk(const torch::Tensor& logits, int64_t topk, int scoring, const MaybeTensor& bias,
                                                    const MaybeTensor& mask, int64_t groups, int64_t topk_groups, bool normalize, double scale) {
    const char* what = "route_topk";
    const RouterArguments a = require_logits(what, logits);
    const Device device = logits.device();
    require_topk(what, topk);
    if (topk > a.experts)
        refuse(what, " topk must not exceed the experts");
    if (groups < 1 || groups > 64 || a.experts % groups != 0)
        refuse(what, " groups must be 1 to 64 and divide the experts evenly");
    if (topk_groups < 1 || topk_groups > groups || topk > topk_groups * (a.experts / groups))
        refuse(what, " topk_groups must be 1 to groups, with at least topk experts in them");
    if (bias.has_value())
        require(*bias, device, at::kFloat, {a.experts}, what, "bias");
    if (mask.has_value())
        require(*mask, device, at::kBool, {a.tokens}, what, "mask");
    require_no_tangent(what, {&logits, given(bias)});
    const DeviceGuard guard(device);
    torch::Tensor ids = make({a.tokens, topk}, at::kLong, device), weights = make({a.tokens, topk}, at::kFloat, device);
    check(nanoep_route_topk(logits.data_ptr(), a.stride, a.type, static_cast<const float*>(pointer_of(bias)),
                            static_cast<const uint8_t*>(pointer_of(mask)), a.tokens, a.experts, static_cast<int>(topk), static_cast<int>(groups),
                            static_cast<int>(topk_groups), scoring, normalize ? 1 : 0, static_cast<float>(scale),
                            static_cast<int64_t*>(ids.data_ptr()), static_cast<float*>(weights.data_ptr()), current_stream(device)),
          what);
    return {ids, weights};
}

torch::Tensor route_topk_backward(const torch::Tensor& grad, const torch::Tensor& logits, const torch::Tensor& ids, int scoring, bool normalize,
                                  double scale) {
    const char* what = "route_topk_backward";
    const RouterArguments a = require_logits(what, logits);
    const Device device = logits.device();
    const int topk = require_ids(what, ids, a, device);
    require(grad, device, at::kFloat, {a.tokens, ids.size(1)}, what, "grad");
    require_no_gradient(what, {&grad, &logits});
    const DeviceGuard guard(device);
    torch::Tensor grad_logits = make({a.tokens, a.experts}, logits.scalar_type(), device);
    check(nanoep_route_topk_backward(static_cast<const float*>(grad.data_ptr()), logits.data_ptr(), a.stride, a.type,
                                     static_cast<const int64_t*>(ids.data_ptr()), a.tokens, a.experts, topk, scoring, normalize ? 1 : 0,
                                     static_cast<float>(scale), grad_logits.data_ptr(), current_stream(device)),
          what);
    return grad_logits;
}

// ------------------------------------------------------------------ balance

int64_t require_sequences(const char* what, const MaybeTensor& offsets, const Device& device) {
    if (!offsets.has_value())
        return 1;
    const int64_t entries = offsets->numel();
    if (entries < 2 || entries > 0x7fffffff)
        refuse(what, " sequence_offsets must name at least one sequence and fewer than 2^31");
    require(*offsets, device, at::kLong, {entries}, what, "sequence_offsets");
    return entries - 1;
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> balance_loss(const torch::Tensor& logits, const torch::Tensor& ids, int scoring,
                                                                     const MaybeTensor& sequence_offsets) {
    const char* what = "balance_loss";
    const RouterArguments a = require_logits(what, logits);
    const Device device = logits.device();
    const int topk = require_ids(what, ids, a, device);
    const int64_t sequences = require_sequences(what, sequence_offsets, device);
    require_no_tangent(what, {&logits});
    const DeviceGuard guard(device);
    torch::Tensor loss, counts, tokens, workspace;
    if (sequence_offsets.has_value()) {
        loss = make({sequences}, at::kFloat, device);
        counts = make({sequences, a.experts}, at::kLong, device);
        tokens = make({sequences}, at::kLong, device);
    } else {
        loss = make({}, at::kFloat, device);
        counts = make({a.experts}, at::kLong, device);
        tokens = make({}, at::kLong, device);
    }
    const size_t bytes = nanoep_balance_loss_workspace_bytes(a.tokens, a.experts, topk, sequences);
    if (bytes > 0)
        workspace = make({static_cast<int64_t>(bytes)}, at::kByte, device);
    check(nanoep_balance_loss(logits.data_ptr(), a.stride, a.type, static_cast<const int64_t*>(ids.data_ptr()),
                              static_cast<const int64_t*>(pointer_of(sequence_offsets)), a.tokens, a.experts, topk, sequences, scoring,
                              static_cast<float*>(loss.data_ptr()), static_cast<int64_t*>(counts.data_ptr()),
                              static_cast<int64_t*>(tokens.data_ptr()), bytes > 0 ? workspace.data_ptr() : nullptr, bytes, current_stream(device)),
          what);
    return {loss, counts, tokens};
}

torch::Tensor balance_loss_backward(const torch::Tensor& grad, const torch::Tensor& logits, const torch::Tensor& ids, const torch::Tensor& counts,
                                    const torch::Tensor& tokens, int scoring, const MaybeTensor& sequence_offsets) {
    const char* what = "balance_loss_backward";
    const RouterArguments a = require_logits(what, logits);
    const Device device = logits.device();
    const int topk = require_ids(what, ids, a, device);
    const int64_t sequences = require_sequences(what, sequence_offsets, device);
    if (sequence_offsets.has_value()) {
        require(grad, device, at::kFloat, {sequences}, what, "grad");
        require(counts, device, at::kLong, {sequences, a.experts}, what, "counts");
        require(tokens, device, at::kLong, {sequences}, what, "tokens");
    } else {
        require(grad, device, at::kFloat, {}, what, "grad");
        require(counts, device, at::kLong, {a.experts}, what, "counts");
        require(tokens, device, at::kLong, {}, what, "tokens");
    }
    require_no_gradient(what, {&grad, &logits});
    const DeviceGuard guard(device);
    torch::Tensor grad_logits = make({a.tokens, a.experts}, logits.scalar_type(), device);
    check(nanoep_balance_loss_backward(static_cast<const float*>(grad.data_ptr()), logits.data_ptr(), a.stride, a.type,
                                       static_cast<const int64_t*>(ids.data_ptr()), static_cast<const int64_t*>(counts.data_ptr()),
                                       static_cast<const int64_t*>(tokens.data_ptr()), static_cast<const int64_t*>(pointer_of(sequence_offsets)),
                                       a.tokens, a.experts, topk, sequences, scoring, grad_logits.data_ptr(), current_stream(device)),
          what);
    return grad_logits;
}

}  // namespace

void bind_entry(py::module_& module) {
    const auto unlocked = py::call_guard<py::gil_scoped_release>();
    module.def("layer_norm", &layer_norm, py::arg("x"), py::arg("gamma"), py::arg("beta"), py::arg("residual"), py::arg("eps"), unlocked);
    module.def("rms_norm", &rms_norm, py::arg("x"), py::arg("gamma"), py::arg("residual"), py::arg("eps"), unlocked);
    module.def("layer_norm_backward", &layer_norm_backward, py::arg("grad"), py::arg("total"), py::arg("gamma"), py::arg("mean"), py::arg("rstd"),
               py::arg("grad_residual"), py::arg("input"), py::arg("parameters"), unlocked);
    module.def("rms_norm_backward", &rms_norm_backward, py::arg("grad"), py::arg("total"), py::arg("gamma"), py::arg("rstd"),
               py::arg("grad_residual"), py::arg("input"), py::arg("parameters"), unlocked);
    module.def("route_topk", &route_topk, py::arg("logits"), py::arg("topk"), py::arg("scoring"), py::arg("bias"), py::arg("mask"), py::arg("groups"),
               py::arg("topk_groups"), py::arg("normalize"), py::arg("scale"), unlocked);
    module.def("route_topk_backward", &route_topk_backward, py::arg("grad"), py::arg("logits"), py::arg("ids"), py::arg("scoring"),
               py::arg("normalize"), py::arg("scale"), unlocked);
    module.def("balance_loss", &balance_loss, py::arg("logits"), py::arg("ids"), py::arg("scoring"), py::arg("sequence_offsets"), unlocked);
    module.def("balance_loss_backward", &balance_loss_backward, py::arg("grad"), py::arg("logits"), py::arg("ids"), py::arg("counts"),
               py::arg("tokens"), py::arg("scoring"), py::arg("sequence_offsets"), unlocked);
}

}  // namespace nanoep
