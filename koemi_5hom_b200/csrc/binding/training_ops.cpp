// PyTorch operators of a training step over the C ABI of libkoemi_b200.so:
// dispatcher schemas, CUDA implementations and autograd formulas.
//
// They are C++ because their backward passes run on autograd's device thread,
// where a Python function waits for the interpreter: a forward and backward of
// an 8 x 257 policy loss took 142 us of host time with Python autograd functions
// and ctypes calls (kernels: 10 us) and takes 67 us; a C++ op of torch takes 50.
// The clipping of gradients is called directly with its Python lists: through
// the dispatcher, which copies a list of tensors twice, 2 x 144 tensors took 48
// us where the kernels take 10. The autograd nodes are plain ones, as torch's
// own ops have, with what the backward needs in fields.
// Nothing here computes: every op checks what the kernels rely on (3 to 5 us
// less than in Python, where only a refusal is explained), allocates from the
// caching allocator and calls one entry point on the current stream.
#include "binding.h"

namespace koemi_torch {

static Library library;
static bool opened = false;

const Library &lib() {
    TORCH_CHECK(opened, "libkoemi_b200 is not open");
    return library;
}

}  // namespace koemi_torch

using namespace koemi_torch;

namespace {

// ----------------------------------------------------- the gated recurrence

constexpr int64_t kSegment = 128;  // positions between two carries

void check_recurrence(const Tensor &projections, const OptionalTensor &valid, const OptionalTensor &restart) {
    TORCH_CHECK_VALUE(one_of_ours(projections) && projections.dim() == 3 && projections.size(2) % 2 == 0 && projections.is_contiguous(),
                      "projections must be contiguous [batch, length, 2 * features] in f32, bf16 or f16 on a CUDA device");
    const int64_t shape[] = {projections.size(0), projections.size(1)};
    require("valid", valid, shape, at::kBool, projections);
    require("restart", restart, shape, at::kBool, projections);
}

void check_forward(const Tensor &projections, const OptionalTensor &initial, const OptionalTensor &valid,
                   const OptionalTensor &restart, double low, double high) {
    check_recurrence(projections, valid, restart);
    require("initial", initial, {projections.size(0), projections.size(2) / 2}, at::kFloat, projections);
    const float lo = static_cast<float>(low), hi = static_cast<float>(high);  // as the kernels have them
    TORCH_CHECK_VALUE(0.0f < lo && low <= high && hi < 1.0f, "retention bounds must satisfy 0 < minimum <= maximum < 1 in fp32");
}

std::tuple<Tensor, Tensor, Tensor> gated_forward(const Tensor &projections, const OptionalTensor &initial,
                                                 const OptionalTensor &valid, const OptionalTensor &restart, double low,
                                                 double high, bool keep) {
    check_forward(projections, initial, valid, restart, low, high);
    TORCH_CHECK_VALUE(projections.size(1) > 0, "projections must hold a position");
    const Launch launch(projections);
    const int64_t batch = projections.size(0), length = projections.size(1), features = projections.size(2) / 2;
    Tensor states = at::empty({batch, length, features}, projections.options());
    Tensor final_state = f32(projections, {batch, features});
    Tensor carries;
    if (keep) carries = f32(projections, {batch, (length + kSegment - 1) / kSegment, features});
    check("koemi_dense_gated_recurrence_forward",
          lib().gated_forward(address<void>(projections), address<float>(initial), address<uint8_t>(valid), address<uint8_t>(restart),
                              address<void>(states), address<float>(final_state), keep ? address<float>(carries) : nullptr, batch,
                              length, features, static_cast<float>(low), static_cast<float>(high), code_of(projections),
                              launch.stream));
    return {states, final_state, carries};
}

// No position: no states, and the state as it was (differentiably, above the CUDA key).
std::tuple<Tensor, Tensor> no_positions(const Tensor &projections, const OptionalTensor &initial) {
    const int64_t features = projections.size(2) / 2;
    return {projections.slice(2, 0, features).contiguous(),
            initial.has_value() && initial->defined() ? initial->clone() : at::zeros({projections.size(0), features}, projections.options().dtype(at::kFloat))};
}

std::tuple<Tensor, Tensor> gated_recurrence_cuda(const Tensor &projections, const OptionalTensor &initial,
                                                 const OptionalTensor &valid, const OptionalTensor &restart, double low,
                                                 double high) {
    if (projections.dim() == 3 && projections.size(1) == 0) {
        check_forward(projections.contiguous(), dense(initial), dense(valid), dense(restart), low, high);
        return no_positions(projections, initial);
    }
    auto [states, final_state, carries] =
        gated_forward(projections.contiguous(), dense(initial), dense(valid), dense(restart), low, high, false);
    return {states, final_state};
}

std::tuple<Tensor, Tensor, Tensor> gated_recurrence_keep_cuda(const Tensor &projections, const OptionalTensor &initial,
                                                              const OptionalTensor &valid, const OptionalTensor &restart,
                                                              double low, double high) {
    return gated_forward(projections, initial, valid, restart, low, high, true);
}

std::tuple<Tensor, Tensor> gated_recurrence_backward_cuda(const Tensor &projections, const OptionalTensor &valid,
                                                          const OptionalTensor &restart, const Tensor &carries,
                                                          const OptionalTensor &grad_states,
                                                          const OptionalTensor &grad_final, double low, double high) {
    check_recurrence(projections, valid, restart);
    TORCH_CHECK_VALUE(projections.size(1) > 0, "projections must hold a position");
    const Launch launch(projections);
    const int64_t batch = projections.size(0), length = projections.size(1), features = projections.size(2) / 2;
    require("carries", carries, {batch, (length + kSegment - 1) / kSegment, features}, at::kFloat, projections);
    require("grad_states", grad_states, {batch, length, features}, projections.scalar_type(), projections);
    require("grad_final", grad_final, {batch, features}, at::kFloat, projections);
    Tensor grad_projections = at::empty_like(projections), grad_initial = f32(projections, {batch, features});
    check("koemi_dense_gated_recurrence_backward",
          lib().gated_backward(address<void>(projections), address<uint8_t>(valid), address<uint8_t>(restart), address<float>(carries),
                               address<void>(grad_states), address<float>(grad_final), address<void>(grad_projections),
                               address<float>(grad_initial), batch, length, features, static_cast<float>(low),
                               static_cast<float>(high), code_of(projections), launch.stream));
    return {grad_projections, grad_initial};
}

// The nodes unpack what they saved above the autograd keys: under activation
// checkpointing that runs the forward again, which has to be recorded.
struct GatedRecurrenceBackward final : torch::autograd::Node {
    SavedVariable projections, valid, restart, carries;
    double low = 0, high = 0;
    variable_list apply(variable_list &&grads) override {
        first_order_only();
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list result(2);
        if (!grads[0].defined() && !grads[1].defined()) return result;
        const Tensor projections_ = projections.unpack(), valid_ = valid.unpack(), restart_ = restart.unpack();
        const Tensor carries_ = carries.unpack();
        const BelowAutograd below;
        KOEMI_OP(gated_recurrence_backward, decltype(gated_recurrence_backward_cuda));
        auto [grad_projections, grad_initial] = gated_recurrence_backward.call(
            projections_, given(valid_), given(restart_), carries_, dense(grads[0]), dense(grads[1]), low, high);
        if (task_should_compute_output(0)) result[0] = grad_projections;
        if (task_should_compute_output(1)) result[1] = grad_initial;
        return result;
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable *saved : {&projections, &valid, &restart, &carries}) saved->reset_data();
    }
    std::string name() const override { return "GatedRecurrenceBackward"; }
};

std::tuple<Tensor, Tensor> gated_recurrence_autograd(const Tensor &projections_, const OptionalTensor &initial_,
                                                     const OptionalTensor &valid_, const OptionalTensor &restart_,
                                                     double low, double high) {
    const Tensor projections = projections_.contiguous();  // differentiably
    const OptionalTensor initial = dense(initial_), valid = dense(valid_), restart = dense(restart_);
    if (projections.dim() == 3 && projections.size(1) == 0) {
        check_forward(projections, initial, valid, restart, low, high);
        return no_positions(projections, initial);
    }
    reverse_mode_only(projections, initial);
    if (at::GradMode::is_enabled() && (differentiates(projections) || differentiates(initial))) {
        auto node = node_of<GatedRecurrenceBackward>(projections, initial);
        Tensor states, final_state, carries;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            KOEMI_OP(gated_recurrence_keep, decltype(gated_recurrence_keep_cuda));
            std::tie(states, final_state, carries) = gated_recurrence_keep.call(projections, initial, valid, restart, low, high);
        }
        node->projections = SavedVariable(projections, false);
        node->valid = SavedVariable(valid, false);
        node->restart = SavedVariable(restart, false);
        node->carries = SavedVariable(carries, false);
        node->low = low;
        node->high = high;
        torch::autograd::set_history({states, final_state}, node);
        return {states, final_state};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    KOEMI_OP(gated_recurrence, decltype(gated_recurrence_cuda));
    return gated_recurrence.call(projections, initial, valid, restart, low, high);
}

// ---------------------------------------------------------- the learned route

using Route = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

// ids, weights, counts, balance loss, and the loss's slope per probability
Route route_learned_keep_cuda(const Tensor &logits, const OptionalTensor &valid, int64_t top_k, bool renormalize) {
    TORCH_CHECK_VALUE(one_of_ours(logits) && logits.dim() == 2 && logits.is_contiguous(),
                      "logits must be contiguous [tokens, experts] in f32, bf16 or f16 on a CUDA device");
    const int64_t tokens = logits.size(0), experts = logits.size(1);
    require("valid", valid, {tokens}, at::kBool, logits);
    TORCH_CHECK_VALUE(1 <= top_k && top_k <= experts, "top_k must be in [1, experts]");
    const Launch launch(logits);
    const auto ints = logits.options().dtype(at::kLong);
    Tensor ids = at::empty({tokens, top_k}, ints), weights = f32(logits, {tokens, top_k});
    Tensor counts = at::empty({experts}, ints), balance = f32(logits, {}), slope = f32(logits, {experts});
    const int64_t size = static_cast<int64_t>(lib().route_workspace(tokens, experts));
    Tensor workspace = at::empty({size}, logits.options().dtype(at::kByte));
    check("koemi_moe_route_learned_forward",
          lib().route_forward(address<void>(logits), address<uint8_t>(valid), address<int64_t>(ids), address<float>(weights),
                              address<int64_t>(counts), address<float>(balance), address<float>(slope), tokens, experts, top_k,
                              renormalize, code_of(logits), address<void>(workspace), size, launch.stream));
    return {ids, weights, counts, balance, slope};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> route_learned_cuda(const Tensor &logits, const OptionalTensor &valid,
                                                              int64_t top_k, bool renormalize) {
    auto [ids, weights, counts, balance, slope] = route_learned_keep_cuda(logits.contiguous(), dense(valid), top_k, renormalize);
    return {ids, weights, counts, balance};
}

Tensor route_learned_backward_cuda(const Tensor &logits, const Tensor &ids, const Tensor &weights, const Tensor &slope,
                                   const OptionalTensor &grad_weights, const OptionalTensor &grad_balance,
                                   bool renormalize) {
    TORCH_CHECK_VALUE(one_of_ours(logits) && logits.dim() == 2 && logits.is_contiguous() && ids.dim() == 2,
                      "logits must be contiguous [tokens, experts] in f32, bf16 or f16 on a CUDA device");
    const int64_t pairs[] = {logits.size(0), ids.size(1)};
    require("ids", ids, pairs, at::kLong, logits);
    require("weights", weights, pairs, at::kFloat, logits);
    require("slope", slope, {logits.size(1)}, at::kFloat, logits);
    require("grad_weights", grad_weights, pairs, at::kFloat, logits);
    require("grad_balance", grad_balance, {}, at::kFloat, logits);
    const Launch launch(logits);
    Tensor grad = at::empty_like(logits);
    check("koemi_moe_route_learned_backward",
          lib().route_backward(address<void>(logits), address<int64_t>(ids), address<float>(weights), address<float>(grad_weights),
                               address<float>(grad_balance), address<float>(slope), address<void>(grad), logits.size(0),
                               logits.size(1), ids.size(1), renormalize, code_of(logits), launch.stream));
    return grad;
}

struct RouteLearnedBackward final : torch::autograd::Node {
    SavedVariable logits, ids, weights, slope;
    bool renormalize = false;
    variable_list apply(variable_list &&grads) override {
        first_order_only();
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list result(1);
        if (!grads[0].defined() && !grads[1].defined()) return result;
        const Tensor logits_ = logits.unpack(), ids_ = ids.unpack(), weights_ = weights.unpack(shared_from_this());
        const Tensor slope_ = slope.unpack();
        const BelowAutograd below;
        KOEMI_OP(route_learned_backward, decltype(route_learned_backward_cuda));
        result[0] = route_learned_backward.call(logits_, ids_, weights_, slope_, dense(grads[0]), dense(grads[1]), renormalize);
        return result;
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable *saved : {&logits, &ids, &weights, &slope}) saved->reset_data();
    }
    std::string name() const override { return "RouteLearnedBackward"; }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> route_learned_autograd(const Tensor &logits_, const OptionalTensor &valid_,
                                                                  int64_t top_k, bool renormalize) {
    const Tensor logits = logits_.contiguous();
    const OptionalTensor valid = dense(valid_);
    reverse_mode_only(logits);
    if (at::GradMode::is_enabled() && differentiates(logits)) {
        auto node = node_of<RouteLearnedBackward>(logits);
        Tensor ids, weights, counts, balance, slope;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            KOEMI_OP(route_learned_keep, decltype(route_learned_keep_cuda));
            std::tie(ids, weights, counts, balance, slope) = route_learned_keep.call(logits, valid, top_k, renormalize);
        }
        node->logits = SavedVariable(logits, false);
        node->ids = SavedVariable(ids, false);
        node->slope = SavedVariable(slope, false);
        node->renormalize = renormalize;
        torch::autograd::set_history({weights, balance}, node);
        node->weights = SavedVariable(weights, true);  // an output of the node itself
        return {ids, weights, counts, balance};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    KOEMI_OP(route_learned, decltype(route_learned_cuda));
    return route_learned.call(logits, valid, top_k, renormalize);
}

// ------------------------------------------------------------ the policy loss

void check_policy(const Tensor &logits, const Tensor &targets, const OptionalTensor &valid) {
    TORCH_CHECK_VALUE(one_of_ours(logits) && (logits.dim() == 2 || logits.dim() == 3) && logits.size(-1) > 0 &&
                          (logits.size(-1) == 1 || logits.stride(-1) == 1),
                      "logits must be [rows, vocabulary] or [batch, length, vocabulary] in f32, bf16 or f16 on a CUDA device");
    const auto shape = logits.sizes().slice(0, logits.dim() - 1);
    require("targets", targets, shape, at::kLong, logits);
    require("valid", valid, shape, at::kBool, logits);
}

// loss, kl, log-probs, (maxima | sums | slopes), gradient (undefined unless wanted)
Route policy_forward(const Tensor &logits, const Tensor &targets, const Tensor &old, const Tensor &advantages,
                     const OptionalTensor &reference, const OptionalTensor &valid, double clip_low, double clip_high,
                     double kl_weight, bool with_gradient) {
    check_policy(logits, targets, valid);
    require("old", old, targets.sizes(), at::kFloat, logits);
    require("advantages", advantages, targets.sizes(), at::kFloat, logits);
    require("reference", reference, targets.sizes(), at::kFloat, logits);
    TORCH_CHECK_VALUE(clip_low >= 0.0 && clip_high >= 0.0 && std::isfinite(static_cast<float>(kl_weight)) &&
                          (kl_weight == 0.0 || (reference.has_value() && reference->defined())),
                      "clip widths must be non-negative, kl_weight finite and, without reference, zero");
    const Launch launch(logits);
    const Rows shape(logits);
    Tensor loss = f32(logits, {}), kl = f32(logits, {}), log_probs = f32(logits, targets.sizes());
    Tensor kept = f32(logits, {3, shape.rows}), gradient;
    if (with_gradient) gradient = at::empty(logits.sizes(), logits.options());
    const int64_t size = static_cast<int64_t>(lib().policy_workspace());
    Tensor workspace = at::empty({size}, logits.options().dtype(at::kByte));
    check("koemi_think_policy_loss_forward",
          lib().policy_forward(address<void>(logits), shape.rows, shape.vocab, shape.inner, shape.outer_stride,
                               shape.inner_stride, address<int64_t>(targets), address<float>(old), address<float>(advantages),
                               address<float>(reference), address<uint8_t>(valid), static_cast<float>(clip_low),
                               static_cast<float>(clip_high), static_cast<float>(kl_weight), address<float>(loss),
                               address<float>(kl), address<float>(log_probs), address<float>(kept), address<float>(kept) + 2 * shape.rows,
                               with_gradient ? address<void>(gradient) : nullptr, code_of(logits) | KOEMI_POLICY_SUMS, address<void>(workspace), size,
                               launch.stream));
    return {loss, kl, log_probs, kept, gradient};
}

std::tuple<Tensor, Tensor, Tensor> policy_loss_cuda(const Tensor &logits, const Tensor &targets, const Tensor &old,
                                                    const Tensor &advantages, const OptionalTensor &reference,
                                                    const OptionalTensor &valid, double clip_low, double clip_high,
                                                    double kl_weight) {
    auto [loss, kl, log_probs, kept, gradient] =
        policy_forward(readable(logits), targets.contiguous(), old.contiguous(), advantages.contiguous(), dense(reference),
                       dense(valid), clip_low, clip_high, kl_weight, false);
    return {loss, kl, log_probs};
}

Route policy_loss_keep_cuda(const Tensor &logits, const Tensor &targets, const Tensor &old, const Tensor &advantages,
                            const OptionalTensor &reference, const OptionalTensor &valid, double clip_low,
                            double clip_high, double kl_weight) {
    Route out = policy_forward(logits, targets, old, advantages, reference, valid, clip_low, clip_high, kl_weight,
                               logits.scalar_type() != at::kHalf);
    if (!std::get<4>(out).defined()) std::get<4>(out) = at::empty({0}, logits.options());
    return out;
}

// Into `grad`; held: it holds the gradient for a factor of one.
void policy_backward(const Tensor &logits, const Tensor &targets, const OptionalTensor &valid, const Tensor &kept,
                     const Tensor &grad_loss, const Tensor &grad, bool held) {
    const Rows shape(logits);
    require("kept", kept, {3, shape.rows}, at::kFloat, logits);
    require("grad_loss", grad_loss, {}, at::kFloat, logits);
    const Launch launch(logits);
    check("koemi_think_policy_loss_backward",
          lib().policy_backward(address<void>(logits), shape.rows, shape.vocab, shape.inner, shape.outer_stride,
                                shape.inner_stride, address<int64_t>(targets), address<uint8_t>(valid), address<float>(kept),
                                address<float>(kept) + 2 * shape.rows, address<float>(grad_loss), address<void>(grad),
                                code_of(logits) | KOEMI_POLICY_SUMS | (held ? KOEMI_POLICY_HELD : 0), launch.stream));
}

Tensor policy_loss_backward_cuda(const Tensor &logits, const Tensor &targets, const OptionalTensor &valid,
                                 const Tensor &kept, const Tensor &grad_loss) {
    check_policy(logits, targets, valid);
    Tensor grad = at::empty(logits.sizes(), logits.options());
    policy_backward(logits, targets, valid, kept, grad_loss, grad, false);
    return grad;
}

void policy_loss_rescale_cuda(const Tensor &gradient, const Tensor &logits, const Tensor &targets, const OptionalTensor &valid,
                              const Tensor &kept, const Tensor &factor) {
    check_policy(logits, targets, valid);
    require("gradient", gradient, logits.sizes(), logits.scalar_type(), logits);
    policy_backward(logits, targets, valid, kept, factor, gradient, true);
}

void policy_loss_scale_cuda(const Tensor &gradient, const Tensor &factor) {
    TORCH_CHECK_VALUE(one_of_ours(gradient) && gradient.is_contiguous(), "gradient must be contiguous f32, bf16 or f16 on a CUDA device");
    require("factor", factor, {}, at::kFloat, gradient);
    const Launch launch(gradient);
    check("koemi_think_policy_loss_scale", lib().policy_scale(address<void>(gradient), gradient.numel(), address<float>(factor),
                                                              code_of(gradient), launch.stream));
}

struct PolicyLossBackward final : torch::autograd::Node {
    SavedVariable logits, targets, valid, kept;
    Tensor gradient;  // of the forward's pass, until it is handed out
    variable_list apply(variable_list &&grads) override {
        first_order_only();
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list result(1);
        if (!grads[0].defined()) return result;
        const Tensor logits_ = logits.unpack(), targets_ = targets.unpack(), valid_ = valid.unpack(), kept_ = kept.unpack();
        const BelowAutograd below;
        const Tensor factor = grads[0].contiguous();
        if (!gradient.defined()) {  // f16, and another backward through a retained graph: from the logits
            KOEMI_OP(policy_loss_backward, decltype(policy_loss_backward_cuda));
            result[0] = policy_loss_backward.call(logits_, targets_, given(valid_), kept_, factor);
            return result;
        }
        result[0] = std::move(gradient);
        gradient = Tensor();
        if (logits_.scalar_type() == at::kFloat) {  // a product more costs 2^-24
            KOEMI_OP(policy_loss_scale, decltype(policy_loss_scale_cuda));
            policy_loss_scale.call(result[0], factor);
        } else {
            KOEMI_OP(policy_loss_rescale, decltype(policy_loss_rescale_cuda));
            policy_loss_rescale.call(result[0], logits_, targets_, given(valid_), kept_, factor);
        }
        return result;
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable *saved : {&logits, &targets, &valid, &kept}) saved->reset_data();
        gradient = Tensor();
    }
    std::string name() const override { return "PolicyLossBackward"; }
};

std::tuple<Tensor, Tensor, Tensor> policy_loss_autograd(const Tensor &logits_, const Tensor &targets_, const Tensor &old_,
                                                        const Tensor &advantages_, const OptionalTensor &reference_,
                                                        const OptionalTensor &valid_, double clip_low, double clip_high,
                                                        double kl_weight) {
    const Tensor logits = readable(logits_), targets = targets_.contiguous();
    const Tensor old = old_.contiguous(), advantages = advantages_.contiguous();
    const OptionalTensor reference = dense(reference_), valid = dense(valid_);
    reverse_mode_only(logits, old, advantages, reference);
    if (at::GradMode::is_enabled() && differentiates(logits)) {
        auto node = node_of<PolicyLossBackward>(logits);
        Tensor loss, kl, log_probs, kept, gradient;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            KOEMI_OP(policy_loss_keep, decltype(policy_loss_keep_cuda));
            std::tie(loss, kl, log_probs, kept, gradient) = policy_loss_keep.call(
                logits, targets, old, advantages, reference, valid, clip_low, clip_high, kl_weight);
        }
        node->logits = SavedVariable(logits, false);
        node->targets = SavedVariable(targets, false);
        node->valid = SavedVariable(valid, false);
        node->kept = SavedVariable(kept, false);
        if (logits.scalar_type() != at::kHalf) node->gradient = gradient;
        torch::autograd::set_history(loss, node);
        return {loss, kl, log_probs};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    KOEMI_OP(policy_loss, decltype(policy_loss_cuda));
    return policy_loss.call(logits, targets, old, advantages, reference, valid, clip_low, clip_high, kl_weight);
}

// ---------------------------------------------------- the clipping of gradients

// A Python list of tensors as the C entry takes it. Borrows the list's tensors.
struct Table {
    std::vector<const Tensor *> tensors;
    std::vector<uint64_t> addresses;
    std::vector<int64_t> elements;
    std::vector<int32_t> codes;
    Table(PyObject *list, const char *name) {
        TORCH_CHECK_TYPE(PyList_Check(list), name, " must be a list");
        const Py_ssize_t count = PyList_GET_SIZE(list);
        TORCH_CHECK_VALUE(count > 0, name, " must not be empty");
        tensors.reserve(count);
        addresses.reserve(count);
        const bool tangents = forward_mode();
        elements.reserve(count);
        codes.reserve(count);
        for (Py_ssize_t i = 0; i < count; ++i) {
            PyObject *item = PyList_GET_ITEM(list, i);
            TORCH_CHECK_TYPE(THPVariable_Check(item), name, " must be torch.Tensors");
            const Tensor &t = THPVariable_Unpack(item);
            TORCH_CHECK_VALUE(t.is_cuda() && t.device() == (i == 0 ? t : *tensors[0]).device(), name, " must be on one CUDA device");
            TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.is_contiguous(), name, " must be contiguous");
            const auto type = t.scalar_type();
            TORCH_CHECK_VALUE(type == at::kFloat || type == at::kHalf || type == at::kBFloat16, name,
                              " must use float32, float16 or bfloat16; found ", type);
            if (tangents) reverse_mode_only(t);
            tensors.push_back(&t);
            addresses.push_back(reinterpret_cast<uint64_t>(t.data_ptr()));
            elements.push_back(t.numel());
            codes.push_back(code_of(t));
        }
    }
};

// outputs: the gradients' own table, another, or NULL (the norm only).
Tensor clip(const Table &gradients, const Table *outputs, double max_norm) {
    const Tensor &like = *gradients.tensors[0];
    if (outputs != nullptr && outputs != &gradients) {
        TORCH_CHECK_VALUE(gradients.elements == outputs->elements && gradients.codes == outputs->codes &&
                              outputs->tensors[0]->device() == like.device(),
                          "out must match gradients in sizes, dtypes and device");
    }
    const Launch launch(like);
    const int64_t count = static_cast<int64_t>(gradients.elements.size());
    Tensor norm = f32(like, {});
    const int64_t size = static_cast<int64_t>(lib().clip_workspace(gradients.elements.data(), count));
    Tensor workspace = at::empty({size}, like.options().dtype(at::kByte));
    check("koemi_core_clip_gradients",
          lib().clip(gradients.addresses.data(), outputs == nullptr ? nullptr : outputs->addresses.data(),
                     gradients.elements.data(), gradients.codes.data(), count, static_cast<float>(max_norm),
                     address<float>(norm), address<void>(workspace), size, launch.stream));
    if (outputs != nullptr) {
        for (const Tensor *t : outputs->tensors) {
            if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
        }
    }
    return norm;
}

}  // namespace

// Takes the entry points from the library at `path`; a message, or NULL.
extern "C" __attribute__((visibility("default"))) const char *koemi_torch_open(const char *path) {
    static std::string message;
    void *handle = dlopen(path, RTLD_NOW | RTLD_LOCAL);
    if (handle == nullptr) {
        message = dlerror();
        return message.c_str();
    }
    auto take = [&](auto &function, const char *name) {
        function = reinterpret_cast<std::decay_t<decltype(function)>>(dlsym(handle, name));
        if (function == nullptr && message.empty()) message = std::string(path) + " does not export " + name;
    };
    message.clear();
    take(library.last_error, "koemi_last_error");
    take(library.device_init, "koemi_device_init");
    take(library.gated_forward, "koemi_dense_gated_recurrence_forward");
    take(library.gated_backward, "koemi_dense_gated_recurrence_backward");
    take(library.route_workspace, "koemi_moe_route_learned_workspace");
    take(library.route_forward, "koemi_moe_route_learned_forward");
    take(library.route_backward, "koemi_moe_route_learned_backward");
    take(library.policy_workspace, "koemi_think_policy_loss_workspace");
    take(library.policy_forward, "koemi_think_policy_loss_forward");
    take(library.policy_backward, "koemi_think_policy_loss_backward");
    take(library.policy_scale, "koemi_think_policy_loss_scale");
    take(library.clip_workspace, "koemi_core_clip_gradients_workspace");
    take(library.clip, "koemi_core_clip_gradients");
    take(library.norm_forward, "koemi_core_layer_norm_forward");
    take(library.norm_workspace, "koemi_core_layer_norm_backward_workspace");
    take(library.norm_backward, "koemi_core_layer_norm_backward");
    take(library.dropout, "koemi_core_dropout");
    take(library.block_kept, "koemi_dense_gated_feed_forward_kept");
    take(library.block_workspace, "koemi_dense_gated_feed_forward_workspace");
    take(library.block_forward, "koemi_dense_gated_feed_forward_forward");
    take(library.block_backward, "koemi_dense_gated_feed_forward_backward");
    opened = message.empty();
    return opened ? nullptr : message.c_str();
}

// The norm of a list of gradients, after scaling them into `out`: a list, the
// same list, or None (the norm only). NULL with a Python exception set where a
// tensor breaks a rule.
extern "C" __attribute__((visibility("default"))) PyObject *koemi_torch_clip_gradients(PyObject *gradients, PyObject *out,
                                                                                       double max_norm) {
    try {
        at::AutoDispatchBelowADInplaceOrView below;
        const Table table(gradients, "gradients");
        if (out == Py_None) return THPVariable_Wrap(clip(table, nullptr, max_norm));
        if (out == gradients) return THPVariable_Wrap(clip(table, &table, max_norm));
        const Table target(out, "out");
        return THPVariable_Wrap(clip(table, &target, max_norm));
    } catch (const c10::TypeError &error) {
        PyErr_SetString(PyExc_TypeError, error.what_without_backtrace());
    } catch (const c10::ValueError &error) {
        PyErr_SetString(PyExc_ValueError, error.what_without_backtrace());
    } catch (const c10::Error &error) {
        PyErr_SetString(PyExc_RuntimeError, error.what_without_backtrace());
    } catch (const std::exception &error) {
        PyErr_SetString(PyExc_RuntimeError, error.what());
    }
    return nullptr;
}

TORCH_LIBRARY_FRAGMENT(koemi_b200, m) {
    m.def("gated_recurrence(Tensor projections, Tensor? initial, Tensor? valid, Tensor? restart, float low, float high) -> (Tensor, Tensor)");
    m.def("gated_recurrence_keep(Tensor projections, Tensor? initial, Tensor? valid, Tensor? restart, float low, float high) -> (Tensor, Tensor, Tensor)");
    m.def("gated_recurrence_backward(Tensor projections, Tensor? valid, Tensor? restart, Tensor carries, Tensor? grad_states, Tensor? grad_final, float low, float high) -> (Tensor, Tensor)");
    m.def("route_learned(Tensor logits, Tensor? valid, int top_k, bool renormalize) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("route_learned_keep(Tensor logits, Tensor? valid, int top_k, bool renormalize) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("route_learned_backward(Tensor logits, Tensor ids, Tensor weights, Tensor slope, Tensor? grad_weights, Tensor? grad_balance, bool renormalize) -> Tensor");
    m.def("policy_loss(Tensor logits, Tensor targets, Tensor old, Tensor advantages, Tensor? reference, Tensor? valid, float clip_low, float clip_high, float kl_weight) -> (Tensor, Tensor, Tensor)");
    m.def("policy_loss_keep(Tensor logits, Tensor targets, Tensor old, Tensor advantages, Tensor? reference, Tensor? valid, float clip_low, float clip_high, float kl_weight) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("policy_loss_backward(Tensor logits, Tensor targets, Tensor? valid, Tensor kept, Tensor grad_loss) -> Tensor");
    m.def("policy_loss_scale(Tensor(a!) gradient, Tensor factor) -> ()");
    m.def("policy_loss_rescale(Tensor(a!) gradient, Tensor logits, Tensor targets, Tensor? valid, Tensor kept, Tensor factor) -> ()");
}

TORCH_LIBRARY_IMPL(koemi_b200, CUDA, m) {
    m.impl("gated_recurrence", gated_recurrence_cuda);
    m.impl("gated_recurrence_keep", gated_recurrence_keep_cuda);
    m.impl("gated_recurrence_backward", gated_recurrence_backward_cuda);
    m.impl("route_learned", route_learned_cuda);
    m.impl("route_learned_keep", route_learned_keep_cuda);
    m.impl("route_learned_backward", route_learned_backward_cuda);
    m.impl("policy_loss", policy_loss_cuda);
    m.impl("policy_loss_keep", policy_loss_keep_cuda);
    m.impl("policy_loss_backward", policy_loss_backward_cuda);
    m.impl("policy_loss_scale", policy_loss_scale_cuda);
    m.impl("policy_loss_rescale", policy_loss_rescale_cuda);
}

TORCH_LIBRARY_IMPL(koemi_b200, Autograd, m) {
    m.impl("gated_recurrence", gated_recurrence_autograd);
    m.impl("route_learned", route_learned_autograd);
    m.impl("policy_loss", policy_loss_autograd);
    // reached with gradients to record under torch.func alone, an order or a level further out
    for (const char *inner : {"gated_recurrence_keep", "gated_recurrence_backward", "route_learned_keep", "route_learned_backward",
                              "policy_loss_keep", "policy_loss_backward", "policy_loss_scale", "policy_loss_rescale"}) {
        m.impl(inner, torch::autograd::autogradNotImplementedFallback());
    }
}
