// What the torch bindings share: the kernel library's entry points, launches on
// a tensor's device and current stream, argument checks, and the rules of
// differentiation (reverse mode, first order).
#pragma once

#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <cmath>
#include <mutex>
#include <string>
#include <tuple>
#include <vector>

#include "koemi_b200.h"

namespace koemi_torch {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptionalTensor = std::optional<Tensor>;

// ------------------------------------------------------------ the library

struct Library {
    decltype(&koemi_last_error) last_error;
    decltype(&koemi_device_init) device_init;
    decltype(&koemi_dense_gated_recurrence_forward) gated_forward;
    decltype(&koemi_dense_gated_recurrence_backward) gated_backward;
    decltype(&koemi_moe_route_learned_workspace) route_workspace;
    decltype(&koemi_moe_route_learned_forward) route_forward;
    decltype(&koemi_moe_route_learned_backward) route_backward;
    decltype(&koemi_think_policy_loss_workspace) policy_workspace;
    decltype(&koemi_think_policy_loss_forward) policy_forward;
    decltype(&koemi_think_policy_loss_backward) policy_backward;
    decltype(&koemi_think_policy_loss_scale) policy_scale;
    decltype(&koemi_core_clip_gradients_workspace) clip_workspace;
    decltype(&koemi_core_clip_gradients) clip;
    decltype(&koemi_core_layer_norm_forward) norm_forward;
    decltype(&koemi_core_layer_norm_backward_workspace) norm_workspace;
    decltype(&koemi_core_layer_norm_backward) norm_backward;
    decltype(&koemi_core_dropout) dropout;
    decltype(&koemi_dense_gated_feed_forward_kept) block_kept;
    decltype(&koemi_dense_gated_feed_forward_workspace) block_workspace;
    decltype(&koemi_dense_gated_feed_forward_forward) block_forward;
    decltype(&koemi_dense_gated_feed_forward_backward) block_backward;
};

const Library &lib();  // refuses until koemi_torch_open has run

inline void check(const char *function, int status) {
    if (status == KOEMI_OK) return;
    char message[1024];
    lib().last_error(message, sizeof(message));
    TORCH_CHECK(false, function, " failed with status ", status, ": ", message);
}

// Makes a tensor's device current, its per-device state initialised, and
// names its current stream.
struct Launch {
    c10::cuda::CUDAGuard guard;
    void *stream;
    explicit Launch(const Tensor &t) : guard(t.device()) {
        static std::once_flag initialised[64];
        const int device = t.device().index();
        TORCH_CHECK(device >= 0 && device < 64, "device index ", device, " is out of range");
        std::call_once(initialised[device], [device] { check("koemi_device_init", lib().device_init(device)); });
        stream = c10::cuda::getCurrentCUDAStream(device).stream();
    }
};

inline int code_of(const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return KOEMI_F32;
        case at::kHalf: return KOEMI_F16;
        case at::kBFloat16: return KOEMI_BF16;
        default: TORCH_CHECK_VALUE(false, "unsupported dtype ", t.scalar_type());
    }
}

template <typename T>
T *address(const Tensor &t) {
    return static_cast<T *>(t.data_ptr());
}
template <typename T>
T *address(const OptionalTensor &t) {
    return t.has_value() && t->defined() ? static_cast<T *>(t->data_ptr()) : nullptr;
}
inline Tensor f32(const Tensor &like, at::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kFloat)); }
inline OptionalTensor given(const Tensor &t) { return t.defined() ? OptionalTensor(t) : OptionalTensor(); }
inline OptionalTensor dense(const Tensor &t) { return t.defined() ? OptionalTensor(t.contiguous()) : OptionalTensor(); }

inline bool differentiates(const Tensor &t) { return t.defined() && t.requires_grad(); }
inline bool differentiates(const OptionalTensor &t) { return t.has_value() && differentiates(*t); }

// A node whose gradients go to `inputs`, in their order.
template <typename NodeType, typename... Inputs>
std::shared_ptr<NodeType> node_of(const Inputs &...inputs) {
    std::shared_ptr<NodeType> node(new NodeType(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
    return node;
}

// The fronts explain a refusal in their own error types; these are what the
// kernels rely on, whoever calls.
inline bool one_of_ours(const Tensor &t) {
    const auto type = t.scalar_type();
    return t.is_cuda() && (type == at::kFloat || type == at::kHalf || type == at::kBFloat16);
}
inline void require(const char *name, const Tensor &t, at::IntArrayRef shape, at::ScalarType type, const Tensor &on) {
    TORCH_CHECK_VALUE(t.scalar_type() == type && t.sizes() == shape && t.device() == on.device() && t.is_contiguous(), name,
                      " must be contiguous ", type, " of shape ", shape, " on ", on.device(), ", got ", t.scalar_type(), " of ",
                      t.sizes(), " on ", t.device());
}
inline void require(const char *name, const OptionalTensor &t, at::IntArrayRef shape, at::ScalarType type, const Tensor &on) {
    if (t.has_value() && t->defined()) require(name, *t, shape, type, on);
}
inline OptionalTensor dense(const OptionalTensor &t) { return t.has_value() && t->defined() ? OptionalTensor(t->contiguous()) : OptionalTensor(); }

// For the ops that a node calls: nothing of them is recorded. torch.func.grad
// runs every backward with gradients enabled, and what is outside it may record
// the calls: there they stay visible, and refuse to be differentiated.
struct BelowAutograd {
    std::optional<at::AutoDispatchBelowADInplaceOrView> below;
    static bool transformed() { return c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode); }
    BelowAutograd() {
        if (!transformed()) below.emplace();
    }
};
inline void first_order_only() {
    TORCH_CHECK(!at::GradMode::is_enabled() || BelowAutograd::transformed(),
                "the training operators are differentiable to first order only (create_graph=True)");
}

// There is no forward-mode derivative: an input that carries a tangent is
// refused, or the result would pass for a constant.
inline bool has_tangent(const Tensor &t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
inline bool has_tangent(const OptionalTensor &t) { return t.has_value() && has_tangent(*t); }
// Asked only while there is a level of tangents: a list of hundreds of views
// costs microseconds.
inline bool forward_mode() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
template <typename... Inputs>
void reverse_mode_only(const Inputs &...inputs) {
    TORCH_CHECK_NOT_IMPLEMENTED(!forward_mode() || !(has_tangent(inputs) || ...), "the training operators have no forward-mode derivative");
}

// --------------------------------------------------------------- strided rows

struct Rows {
    int64_t rows, vocab, inner, outer_stride, inner_stride;
    // [N, V] or [B, T, V] logits whose last dimension is contiguous
    explicit Rows(const Tensor &logits) : vocab(logits.size(-1)) {
        const bool batched = logits.dim() == 3;
        rows = batched ? logits.size(0) * logits.size(1) : logits.size(0);
        inner = std::max<int64_t>(batched ? logits.size(1) : rows, 1);
        outer_stride = batched ? logits.stride(0) : 0;
        inner_stride = batched ? logits.stride(1) : logits.stride(0);
    }
};

// Logits with the last dimension contiguous, the others as they are.
inline Tensor readable(const Tensor &logits) {
    return logits.dim() > 0 && logits.size(-1) > 1 && logits.stride(-1) != 1 ? logits.contiguous() : logits;
}

#define KOEMI_OP(name, signature) \
    static auto name = c10::Dispatcher::singleton().findSchemaOrThrow("koemi_b200::" #name, "").typed<signature>()

}  // namespace koemi_torch
