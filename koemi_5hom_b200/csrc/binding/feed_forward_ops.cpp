// PyTorch operators of a feed-forward sub-layer over the C ABI of
// libkoemi_b200.so: layer norm and dropout, with their autograd nodes (see
// training_ops.cpp for why they are C++).
#include "binding.h"

using namespace koemi_torch;

namespace {

// ---------------------------------------------------------------- layer norm

struct NormShape {
    Rows rows;
    int weight_code;
    NormShape(const Tensor &values, const Tensor &weight, const OptionalTensor &bias) : rows(values), weight_code(code_of(weight)) {
        require("weight", weight, {values.size(-1)}, weight.scalar_type(), values);
        require("bias", bias, {values.size(-1)}, weight.scalar_type(), values);
        TORCH_CHECK_VALUE(weight.scalar_type() == values.scalar_type() || weight.scalar_type() == at::kFloat,
                          "weight must have the values' dtype or float32");
    }
};

void check_norm(const Tensor &values) {
    TORCH_CHECK_VALUE(one_of_ours(values) && (values.dim() == 2 || values.dim() == 3) && values.size(-1) > 0 &&
                          (values.size(-1) == 1 || values.stride(-1) == 1),
                      "values must be [rows, width] or [batch, length, width] in f32, bf16 or f16 on a CUDA device");
}

Tensor norm_forward(const Tensor &values, const Tensor &weight, const OptionalTensor &bias, double eps, Tensor *stats) {
    check_norm(values);
    const NormShape shape(values, weight, bias);
    TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite(static_cast<float>(eps)), "eps must be finite and non-negative");
    const Launch launch(values);
    Tensor out = at::empty(values.sizes(), values.options());
    if (stats != nullptr) *stats = f32(values, {2, shape.rows.rows});
    check("koemi_core_layer_norm_forward",
          lib().norm_forward(address<void>(values), shape.rows.rows, shape.rows.vocab, shape.rows.inner, shape.rows.outer_stride,
                             shape.rows.inner_stride, address<void>(weight), address<void>(bias), shape.weight_code,
                             address<void>(out), stats != nullptr ? address<float>(*stats) : nullptr, static_cast<float>(eps),
                             code_of(values), launch.stream));
    return out;
}

Tensor layer_norm_cuda(const Tensor &values, const Tensor &weight, const OptionalTensor &bias, double eps) {
    return norm_forward(readable(values), weight.contiguous(), dense(bias), eps, nullptr);
}

std::tuple<Tensor, Tensor> layer_norm_keep_cuda(const Tensor &values, const Tensor &weight, const OptionalTensor &bias, double eps) {
    Tensor stats;
    Tensor out = norm_forward(values, weight, bias, eps, &stats);
    return {out, stats};
}

// Gradients of the values, the weight and the bias; one that is not wanted is empty.
std::tuple<Tensor, Tensor, Tensor> layer_norm_backward_cuda(const Tensor &values, const Tensor &weight, const Tensor &stats,
                                                            const Tensor &grad, std::array<bool, 3> wanted) {
    check_norm(values);
    const NormShape shape(values, weight, OptionalTensor());
    require("stats", stats, {2, shape.rows.rows}, at::kFloat, values);
    require("grad", grad, values.sizes(), values.scalar_type(), values);
    const Launch launch(values);
    auto result = [&](bool want, at::IntArrayRef sizes, const Tensor &like) {
        return want ? at::empty(sizes, like.options()) : at::empty({0}, like.options());
    };
    Tensor grad_values = result(wanted[0], values.sizes(), values), grad_weight = result(wanted[1], weight.sizes(), weight);
    Tensor grad_bias = result(wanted[2], weight.sizes(), weight), workspace;
    const int64_t size = wanted[1] || wanted[2] ? static_cast<int64_t>(lib().norm_workspace(shape.rows.rows, shape.rows.vocab)) : 0;
    if (size > 0) workspace = at::empty({size}, values.options().dtype(at::kByte));
    check("koemi_core_layer_norm_backward",
          lib().norm_backward(address<void>(values), shape.rows.rows, shape.rows.vocab, shape.rows.inner, shape.rows.outer_stride,
                              shape.rows.inner_stride, address<void>(weight), shape.weight_code, address<float>(stats),
                              address<void>(grad), wanted[0] ? address<void>(grad_values) : nullptr,
                              wanted[1] ? address<void>(grad_weight) : nullptr, wanted[2] ? address<void>(grad_bias) : nullptr,
                              code_of(values), size > 0 ? address<void>(workspace) : nullptr, size, launch.stream));
    return {grad_values, grad_weight, grad_bias};
}

struct LayerNormBackward final : torch::autograd::Node {
    SavedVariable values, weight, stats;
    variable_list apply(variable_list &&grads) override {
        first_order_only();
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list result(3);
        if (!grads[0].defined()) return result;
        const Tensor values_ = values.unpack(), weight_ = weight.unpack(), stats_ = stats.unpack();
        const BelowAutograd below;
        KOEMI_OP(layer_norm_backward, decltype(layer_norm_backward_cuda));
        const std::array<bool, 3> wanted = {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2)};
        auto [grad_values, grad_weight, grad_bias] = layer_norm_backward.call(values_, weight_, stats_, grads[0].contiguous(), wanted);
        if (wanted[0]) result[0] = grad_values;
        if (wanted[1]) result[1] = grad_weight;
        if (wanted[2]) result[2] = grad_bias;
        return result;
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable *saved : {&values, &weight, &stats}) saved->reset_data();
    }
    std::string name() const override { return "LayerNormBackward"; }
};

Tensor layer_norm_autograd(const Tensor &values_, const Tensor &weight_, const OptionalTensor &bias_, double eps) {
    const Tensor values = readable(values_), weight = weight_.contiguous();  // differentiably
    const OptionalTensor bias = dense(bias_);
    reverse_mode_only(values, weight, bias);
    if (at::GradMode::is_enabled() && (differentiates(values) || differentiates(weight) || differentiates(bias))) {
        auto node = node_of<LayerNormBackward>(values, weight, bias.value_or(Tensor()));
        Tensor out, stats;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            KOEMI_OP(layer_norm_keep, decltype(layer_norm_keep_cuda));
            std::tie(out, stats) = layer_norm_keep.call(values, weight, bias, eps);
        }
        node->values = SavedVariable(values, false);
        node->weight = SavedVariable(weight, false);
        node->stats = SavedVariable(stats, false);
        torch::autograd::set_history(out, node);
        return out;
    }
    at::AutoDispatchBelowADInplaceOrView below;
    KOEMI_OP(layer_norm, decltype(layer_norm_cuda));
    return layer_norm.call(values, weight, bias, eps);
}

// ------------------------------------------------------------------- dropout

Tensor dropout_cuda(const Tensor &values_, const OptionalTensor &residual_, const OptionalTensor &step, int64_t dropped, int64_t seed,
                    int64_t site, int64_t step_number) {
    TORCH_CHECK_VALUE(one_of_ours(values_), "values must be f32, bf16 or f16 on a CUDA device");
    TORCH_CHECK_VALUE(0 <= dropped && dropped <= 65536, "dropped must be in [0, 65536]");
    const Tensor values = values_.contiguous();
    const OptionalTensor residual = dense(residual_);
    require("residual", residual, values.sizes(), values.scalar_type(), values);
    require("step", step, {}, at::kLong, values);
    const Launch launch(values);
    Tensor out = at::empty(values.sizes(), values.options());
    check("koemi_core_dropout",
          lib().dropout(address<void>(values), address<void>(residual), address<void>(out), values.numel(), dropped,
                        static_cast<uint64_t>(seed), static_cast<uint64_t>(site), static_cast<uint64_t>(step_number),
                        address<int64_t>(step), code_of(values), launch.stream));
    return out;
}

// Linear in both inputs: the gradient is the operator on the gradient, which
// is recorded where a further order is asked for.
struct DropoutBackward final : torch::autograd::Node {
    SavedVariable step;
    bool has_step = false;
    int64_t dropped = 0, seed = 0, site = 0, step_number = 0;
    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list result(2);
        if (!grads[0].defined()) return result;
        KOEMI_OP(dropout, decltype(dropout_cuda));
        if (task_should_compute_output(0)) {
            const OptionalTensor step_ = has_step ? OptionalTensor(step.unpack()) : OptionalTensor();
            result[0] = dropout.call(grads[0], OptionalTensor(), step_, dropped, seed, site, step_number);
        }
        if (task_should_compute_output(1)) result[1] = grads[0];
        return result;
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        step.reset_data();
    }
    std::string name() const override { return "DropoutBackward"; }
};

Tensor dropout_autograd(const Tensor &values, const OptionalTensor &residual, const OptionalTensor &step, int64_t dropped, int64_t seed,
                        int64_t site, int64_t step_number) {
    reverse_mode_only(values, residual);
    const bool record = at::GradMode::is_enabled() && (differentiates(values) || differentiates(residual));
    Tensor out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        KOEMI_OP(dropout, decltype(dropout_cuda));
        out = dropout.call(values, residual, step, dropped, seed, site, step_number);
    }
    if (record) {
        auto node = node_of<DropoutBackward>(values, residual.value_or(Tensor()));
        node->has_step = step.has_value() && step->defined();
        if (node->has_step) node->step = SavedVariable(*step, false);
        node->dropped = dropped;
        node->seed = seed;
        node->site = site;
        node->step_number = step_number;
        torch::autograd::set_history(out, node);
    }
    return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(koemi_b200, m) {
    m.def("layer_norm(Tensor values, Tensor weight, Tensor? bias, float eps) -> Tensor");
    m.def("layer_norm_keep(Tensor values, Tensor weight, Tensor? bias, float eps) -> (Tensor, Tensor)");
    m.def("layer_norm_backward(Tensor values, Tensor weight, Tensor stats, Tensor grad, bool[3] wanted) -> (Tensor, Tensor, Tensor)");
    m.def("dropout(Tensor values, Tensor? residual, Tensor? step, int dropped, int seed, int site, int step_number) -> Tensor");
}

TORCH_LIBRARY_IMPL(koemi_b200, CUDA, m) {
    m.impl("layer_norm", layer_norm_cuda);
    m.impl("layer_norm_keep", layer_norm_keep_cuda);
    m.impl("layer_norm_backward", layer_norm_backward_cuda);
    m.impl("dropout", dropout_cuda);
}

TORCH_LIBRARY_IMPL(koemi_b200, Autograd, m) {
    m.impl("layer_norm", layer_norm_autograd);
    m.impl("dropout", dropout_autograd);
    for (const char *inner : {"layer_norm_keep", "layer_norm_backward"}) m.impl(inner, torch::autograd::autogradNotImplementedFallback());
}
