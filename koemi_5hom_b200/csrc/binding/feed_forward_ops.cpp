// PyTorch operators of a feed-forward sub-layer over the C ABI of
// libkoemi_b200.so: layer norm, dropout and the gated block, with their autograd
// nodes (see training_ops.cpp for why they are C++).
#include <algorithm>
#include <array>

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

// The operator without a residual, under a name of its own: a batch of gradients
// of one call has that call's mask, so vmap may call this once for each.
Tensor dropout_gradient_cuda(const Tensor &grad, const OptionalTensor &step, int64_t dropped, int64_t seed, int64_t site, int64_t step_number) {
    return dropout_cuda(grad, OptionalTensor(), step, dropped, seed, site, step_number);
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
        KOEMI_OP(dropout_gradient, decltype(dropout_gradient_cuda));
        if (task_should_compute_output(0)) {
            const OptionalTensor step_ = has_step ? OptionalTensor(step.unpack()) : OptionalTensor();
            result[0] = dropout_gradient.call(grads[0], step_, dropped, seed, site, step_number);
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

// `out` recorded as dropout of `values` onto `residual`, where one of them is differentiated.
Tensor dropped_out(Tensor out, const Tensor &values, const OptionalTensor &residual, const OptionalTensor &step, int64_t dropped, int64_t seed,
                   int64_t site, int64_t step_number) {
    if (!at::GradMode::is_enabled() || !(differentiates(values) || differentiates(residual))) return out;
    auto node = node_of<DropoutBackward>(values, residual.value_or(Tensor()));
    node->has_step = step.has_value() && step->defined();
    if (node->has_step) node->step = SavedVariable(*step, false);
    node->dropped = dropped;
    node->seed = seed;
    node->site = site;
    node->step_number = step_number;
    torch::autograd::set_history(out, node);
    return out;
}

Tensor dropout_autograd(const Tensor &values, const OptionalTensor &residual, const OptionalTensor &step, int64_t dropped, int64_t seed,
                        int64_t site, int64_t step_number) {
    reverse_mode_only(values, residual);
    Tensor out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        KOEMI_OP(dropout, decltype(dropout_cuda));
        out = dropout.call(values, residual, step, dropped, seed, site, step_number);
    }
    return dropped_out(out, values, residual, step, dropped, seed, site, step_number);
}

Tensor dropout_gradient_autograd(const Tensor &grad, const OptionalTensor &step, int64_t dropped, int64_t seed, int64_t site, int64_t step_number) {
    reverse_mode_only(grad);
    Tensor out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        KOEMI_OP(dropout_gradient, decltype(dropout_gradient_cuda));
        out = dropout_gradient.call(grad, step, dropped, seed, site, step_number);
    }
    return dropped_out(out, grad, OptionalTensor(), step, dropped, seed, site, step_number);
}

// vmap would call the operator once a sample, each time with the same positions and so the same mask.
Tensor dropout_batched(const Tensor &, const OptionalTensor &, const OptionalTensor &, int64_t, int64_t, int64_t, int64_t) {
    TORCH_CHECK_NOT_IMPLEMENTED(false, "dropout has no vmap rule: every sample would get the same mask; call it on the whole batch");
}

// ------------------------------------------------------------ the gated block

// The weights and biases of a call, in the order of its gradients after the values'.
struct BlockShape {
    int64_t rows, width, hidden, out, stride;
    BlockShape(const Tensor &values, const Tensor &gate_weight, const Tensor &value_weight, const Tensor &output_weight,
               const OptionalTensor &gate_bias, const OptionalTensor &value_bias, const OptionalTensor &output_bias) {
        TORCH_CHECK_VALUE(one_of_ours(values) && values.dim() == 2 && values.size(1) > 0 && readable_rows(values),
                          "values must be [rows, width] in f32, bf16 or f16 on a CUDA device");
        TORCH_CHECK_VALUE(gate_weight.dim() == 2 && gate_weight.size(0) > 0 && output_weight.dim() == 2 && output_weight.size(0) > 0,
                          "weights must be matrices with rows");
        rows = values.size(0);
        width = values.size(1);
        hidden = gate_weight.size(0);
        out = output_weight.size(0);
        stride = rows > 1 ? values.stride(0) : width;
        const auto type = values.scalar_type();
        require("gate_weight", gate_weight, {hidden, width}, type, values);
        require("value_weight", value_weight, {hidden, width}, type, values);
        require("output_weight", output_weight, {out, hidden}, type, values);
        require("gate_bias", gate_bias, {hidden}, type, values);
        require("value_bias", value_bias, {hidden}, type, values);
        require("output_bias", output_bias, {out}, type, values);
    }
    // Rows that do not overlap, their entries contiguous.
    static bool readable_rows(const Tensor &values) {
        return (values.size(1) == 1 || values.stride(1) == 1) && (values.size(0) <= 1 || values.stride(0) >= values.size(1));
    }
};

Tensor rows_of(const Tensor &values) { return BlockShape::readable_rows(values) ? values : values.contiguous(); }

Tensor bytes_of(const Tensor &like, size_t size) {
    return at::empty({static_cast<int64_t>(std::max<size_t>(size, 256))}, like.options().dtype(at::kByte));
}

// Whether the kernels read these as they lie, as far as starts and the values' stride go.
int aligned_pass(int64_t stride, std::initializer_list<const Tensor *> operands) {
    bool aligned = stride % 8 == 0;
    for (const Tensor *t : operands) aligned = aligned && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0;
    return aligned ? KOEMI_FEED_FORWARD_ALIGNED : 0;
}

Tensor block_forward(const Tensor &values, const Tensor &gate_weight, const Tensor &value_weight, const Tensor &output_weight,
                     const OptionalTensor &gate_bias, const OptionalTensor &value_bias, const OptionalTensor &output_bias, Tensor *kept) {
    const BlockShape s(values, gate_weight, value_weight, output_weight, gate_bias, value_bias, output_bias);
    const Launch launch(values);
    const int code = code_of(values);
    Tensor out = at::empty({s.rows, s.out}, values.options());
    if (kept != nullptr) *kept = bytes_of(values, lib().block_kept(s.rows, s.hidden, code));
    const int pass = aligned_pass(s.stride, {&values, &gate_weight, &value_weight, &output_weight}) | (kept != nullptr ? KOEMI_FEED_FORWARD_KEEPS : 0);
    Tensor workspace = bytes_of(values, lib().block_workspace(s.rows, s.width, s.hidden, s.out, code, pass));
    check("koemi_dense_gated_feed_forward_forward",
          lib().block_forward(address<void>(values), s.stride, address<void>(gate_weight), address<void>(value_weight),
                              address<void>(output_weight), address<void>(gate_bias), address<void>(value_bias),
                              address<void>(output_bias), address<void>(out), kept != nullptr ? address<void>(*kept) : nullptr,
                              kept != nullptr ? kept->numel() : 0, s.rows, s.width, s.hidden, s.out, code, address<void>(workspace),
                              workspace.numel(), launch.stream));
    return out;
}

Tensor gated_feed_forward_cuda(const Tensor &values_, const Tensor &gate_weight, const Tensor &value_weight, const Tensor &output_weight,
                               const OptionalTensor &gate_bias, const OptionalTensor &value_bias, const OptionalTensor &output_bias) {
    TORCH_CHECK_VALUE(values_.dim() > 0 && output_weight.dim() == 2 && values_.size(-1) > 0, "values must be [..., width], weights matrices");
    const Tensor values = values_.dim() == 2 ? values_ : values_.reshape({values_.numel() / values_.size(-1), values_.size(-1)});
    Tensor out = block_forward(rows_of(values), gate_weight.contiguous(), value_weight.contiguous(), output_weight.contiguous(),
                               dense(gate_bias), dense(value_bias), dense(output_bias), nullptr);
    if (values_.dim() == 2) return out;
    auto sizes = values_.sizes().vec();
    sizes.back() = out.size(1);
    return out.view(sizes);
}

std::tuple<Tensor, Tensor> gated_feed_forward_keep_cuda(const Tensor &values, const Tensor &gate_weight, const Tensor &value_weight,
                                                        const Tensor &output_weight, const OptionalTensor &gate_bias,
                                                        const OptionalTensor &value_bias, const OptionalTensor &output_bias) {
    Tensor kept;
    Tensor out = block_forward(values, gate_weight, value_weight, output_weight, gate_bias, value_bias, output_bias, &kept);
    return {out, kept};
}

// Gradients of values, gate_weight, value_weight, output_weight and the three
// biases, bit k of `wanted` for the k-th; one that is not wanted is empty. A
// tuple: vmap, which calls this once a sample, takes no list.
using BlockGradients = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;
BlockGradients gated_feed_forward_backward_cuda(const Tensor &values, const Tensor &gate_weight, const Tensor &value_weight,
                                                     const Tensor &output_weight, const Tensor &kept, const Tensor &grad, int64_t wanted) {
    const OptionalTensor none;
    const BlockShape s(values, gate_weight, value_weight, output_weight, none, none, none);
    const Launch launch(values);
    const int code = code_of(values);
    require("grad", grad, {s.rows, s.out}, values.scalar_type(), values);
    TORCH_CHECK_VALUE(kept.scalar_type() == at::kByte && kept.is_contiguous() && kept.device() == values.device() &&
                          kept.numel() >= static_cast<int64_t>(lib().block_kept(s.rows, s.hidden, code)),
                      "kept is not what the forward of these values returned");
    const std::vector<int64_t> sizes[] = {{s.rows, s.width}, {s.hidden, s.width}, {s.hidden, s.width}, {s.out, s.hidden}, {s.hidden}, {s.hidden}, {s.out}};
    std::array<Tensor, 7> grads;
    void *p[7];
    for (int k = 0; k < 7; ++k) {
        const bool want = wanted >> k & 1;
        grads[k] = want ? at::empty(sizes[k], values.options()) : at::empty({0}, values.options());
        p[k] = want ? address<void>(grads[k]) : nullptr;
    }
    const int pass = aligned_pass(s.stride, {&values, &gate_weight, &value_weight, &output_weight, &grad}) | KOEMI_FEED_FORWARD_BACKWARD;
    Tensor workspace = bytes_of(values, lib().block_workspace(s.rows, s.width, s.hidden, s.out, code, pass));
    check("koemi_dense_gated_feed_forward_backward",
          lib().block_backward(address<void>(values), s.stride, address<void>(gate_weight), address<void>(value_weight),
                               address<void>(output_weight), address<void>(kept), kept.numel(), address<void>(grad), p[0], p[1], p[2],
                               p[3], p[4], p[5], p[6], s.rows, s.width, s.hidden, s.out, code, address<void>(workspace),
                               workspace.numel(), launch.stream));
    return std::tuple_cat(grads);
}

struct GatedFeedForwardBackward final : torch::autograd::Node {
    SavedVariable values, gate_weight, value_weight, output_weight, kept;
    variable_list apply(variable_list &&grads) override {
        first_order_only();
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list result(7);
        if (!grads[0].defined()) return result;
        const Tensor values_ = values.unpack(), gate = gate_weight.unpack(), value = value_weight.unpack(), output = output_weight.unpack();
        const Tensor kept_ = kept.unpack();
        const BelowAutograd below;
        int64_t wanted = 0;
        for (int k = 0; k < 7; ++k) wanted |= static_cast<int64_t>(task_should_compute_output(k)) << k;
        KOEMI_OP(gated_feed_forward_backward, decltype(gated_feed_forward_backward_cuda));
        std::array<Tensor, 7> found;
        std::tie(found[0], found[1], found[2], found[3], found[4], found[5], found[6]) =
            gated_feed_forward_backward.call(values_, gate, value, output, kept_, grads[0].contiguous(), wanted);
        for (int k = 0; k < 7; ++k) {
            if (wanted >> k & 1) result[k] = found[k];
        }
        return result;
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable *saved : {&values, &gate_weight, &value_weight, &output_weight, &kept}) saved->reset_data();
    }
    std::string name() const override { return "GatedFeedForwardBackward"; }
};

Tensor gated_feed_forward_autograd(const Tensor &values_, const Tensor &gate_weight_, const Tensor &value_weight_, const Tensor &output_weight_,
                                   const OptionalTensor &gate_bias_, const OptionalTensor &value_bias_, const OptionalTensor &output_bias_) {
    reverse_mode_only(values_, gate_weight_, value_weight_, output_weight_, gate_bias_, value_bias_, output_bias_);
    if (!(at::GradMode::is_enabled() && (differentiates(values_) || differentiates(gate_weight_) || differentiates(value_weight_) ||
                                         differentiates(output_weight_) || differentiates(gate_bias_) || differentiates(value_bias_) ||
                                         differentiates(output_bias_)))) {
        at::AutoDispatchBelowADInplaceOrView below;
        KOEMI_OP(gated_feed_forward, decltype(gated_feed_forward_cuda));
        return gated_feed_forward.call(values_, gate_weight_, value_weight_, output_weight_, gate_bias_, value_bias_, output_bias_);
    }
    TORCH_CHECK_VALUE(values_.dim() > 0 && output_weight_.dim() == 2 && values_.size(-1) > 0, "values must be [..., width], weights matrices");
    // differentiably
    const Tensor values = rows_of(values_.dim() == 2 ? values_ : values_.reshape({values_.numel() / values_.size(-1), values_.size(-1)}));
    const Tensor gate_weight = gate_weight_.contiguous(), value_weight = value_weight_.contiguous(), output_weight = output_weight_.contiguous();
    const OptionalTensor gate_bias = dense(gate_bias_), value_bias = dense(value_bias_), output_bias = dense(output_bias_);
    auto node = node_of<GatedFeedForwardBackward>(values, gate_weight, value_weight, output_weight, gate_bias.value_or(Tensor()),
                                                  value_bias.value_or(Tensor()), output_bias.value_or(Tensor()));
    Tensor out, kept;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        KOEMI_OP(gated_feed_forward_keep, decltype(gated_feed_forward_keep_cuda));
        std::tie(out, kept) = gated_feed_forward_keep.call(values, gate_weight, value_weight, output_weight, gate_bias, value_bias, output_bias);
    }
    node->values = SavedVariable(values, false);
    node->gate_weight = SavedVariable(gate_weight, false);
    node->value_weight = SavedVariable(value_weight, false);
    node->output_weight = SavedVariable(output_weight, false);
    node->kept = SavedVariable(kept, false);
    torch::autograd::set_history(out, node);
    if (values_.dim() == 2) return out;
    auto sizes = values_.sizes().vec();
    sizes.back() = out.size(1);
    return out.view(sizes);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(koemi_b200, m) {
    m.def("layer_norm(Tensor values, Tensor weight, Tensor? bias, float eps) -> Tensor");
    m.def("layer_norm_keep(Tensor values, Tensor weight, Tensor? bias, float eps) -> (Tensor, Tensor)");
    m.def("layer_norm_backward(Tensor values, Tensor weight, Tensor stats, Tensor grad, bool[3] wanted) -> (Tensor, Tensor, Tensor)");
    m.def("dropout(Tensor values, Tensor? residual, Tensor? step, int dropped, int seed, int site, int step_number) -> Tensor");
    m.def("dropout_gradient(Tensor grad, Tensor? step, int dropped, int seed, int site, int step_number) -> Tensor");
    m.def("gated_feed_forward(Tensor values, Tensor gate_weight, Tensor value_weight, Tensor output_weight, Tensor? gate_bias, Tensor? value_bias, Tensor? output_bias) -> Tensor");
    m.def("gated_feed_forward_keep(Tensor values, Tensor gate_weight, Tensor value_weight, Tensor output_weight, Tensor? gate_bias, Tensor? value_bias, Tensor? output_bias) -> (Tensor, Tensor)");
    m.def("gated_feed_forward_backward(Tensor values, Tensor gate_weight, Tensor value_weight, Tensor output_weight, Tensor kept, Tensor grad, int wanted) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(koemi_b200, CUDA, m) {
    m.impl("layer_norm", layer_norm_cuda);
    m.impl("layer_norm_keep", layer_norm_keep_cuda);
    m.impl("layer_norm_backward", layer_norm_backward_cuda);
    m.impl("dropout", dropout_cuda);
    m.impl("dropout_gradient", dropout_gradient_cuda);
    m.impl("gated_feed_forward", gated_feed_forward_cuda);
    m.impl("gated_feed_forward_keep", gated_feed_forward_keep_cuda);
    m.impl("gated_feed_forward_backward", gated_feed_forward_backward_cuda);
}

TORCH_LIBRARY_IMPL(koemi_b200, FuncTorchBatched, m) { m.impl("dropout", dropout_batched); }

TORCH_LIBRARY_IMPL(koemi_b200, Autograd, m) {
    m.impl("layer_norm", layer_norm_autograd);
    m.impl("dropout", dropout_autograd);
    m.impl("dropout_gradient", dropout_gradient_autograd);
    m.impl("gated_feed_forward", gated_feed_forward_autograd);
    for (const char *inner : {"layer_norm_keep", "layer_norm_backward", "gated_feed_forward_keep", "gated_feed_forward_backward"}) {
        m.impl(inner, torch::autograd::autogradNotImplementedFallback());
    }
}
