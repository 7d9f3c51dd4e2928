// Dense front: gated linear recurrence from raw projections, forward and
// backward.
//
//   s = sigmoid(p), a = lo + (hi - lo) s, k = tanh(c)
//   h_t = a_t h' + (1 - a_t) k_t,  h' = 0 at a restart, else h_{t-1}
//   (an invalid position keeps the state: h_t = h')
//
// projections are [batch, length, 2 F] (p | c), states [batch, length, F];
// the running state is fp32. The forward can leave the state before every
// 64th position in `carries`, from which the backward recomputes the states
// it needs instead of reading them:
//
//   adj_t = g_t + a_{t+1} adj_{t+1} (no term across a restart)
//   dp_t = adj_t (h' - k_t) (hi - lo) s (1 - s)
//   dc_t = adj_t (1 - a_t) (1 - k_t^2),  d_initial = a_0 adj_0
//
// One thread walks one (batch, feature) lane.
#include "common.cuh"

namespace koemi {
namespace {

constexpr int kSegment = 64;  // positions between two carries

struct Gate {
    float s, a, k;
};

__device__ __forceinline__ Gate gate_of(float p, float c, float lo, float hi) {
    Gate g;
    g.s = sigmoidf_(p);
    g.a = lo + (hi - lo) * g.s;
    g.k = tanhf(c);
    return g;
}

struct GatedShape {
    int64_t batch, length, features, segments;
    float lo, hi;
    const uint8_t *valid, *restart;
};

template <typename T>
__global__ void gated_forward_lane_kernel(GatedShape shape, const T *__restrict__ projections,
                                          const float *__restrict__ initial, T *__restrict__ states,
                                          float *__restrict__ final_state, float *__restrict__ carries) {
    const int64_t lane = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (lane >= shape.batch * shape.features) return;
    const int64_t b = lane / shape.features, f = lane - b * shape.features;
    float h = initial != nullptr ? initial[lane] : 0.0f;
    for (int64_t t = 0; t < shape.length; ++t) {
        const int64_t row = b * shape.length + t;
        if (carries != nullptr && t % kSegment == 0) carries[(b * shape.segments + t / kSegment) * shape.features + f] = h;
        if (shape.restart != nullptr && shape.restart[row]) h = 0.0f;
        if (shape.valid == nullptr || shape.valid[row]) {
            const Gate g = gate_of(to_acc(projections[row * 2 * shape.features + f]),
                                   to_acc(projections[row * 2 * shape.features + shape.features + f]), shape.lo, shape.hi);
            h = fmaf(g.a, h, (1.0f - g.a) * g.k);
        }
        states[row * shape.features + f] = from_acc<T>(h);
    }
    final_state[lane] = h;
}

template <typename T>
__global__ void gated_backward_lane_kernel(GatedShape shape, const T *__restrict__ projections,
                                           const float *__restrict__ carries, const T *__restrict__ grad_states,
                                           const float *__restrict__ grad_final, T *__restrict__ grad_projections,
                                           float *__restrict__ grad_initial) {
    const int64_t lane = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (lane >= shape.batch * shape.features) return;
    const int64_t b = lane / shape.features, f = lane - b * shape.features;
    float incoming = grad_final != nullptr ? grad_final[lane] : 0.0f;
    for (int64_t segment = shape.segments - 1; segment >= 0; --segment) {
        const int64_t first = segment * kSegment;
        const int count = static_cast<int>(shape.length - first < kSegment ? shape.length - first : kSegment);
        float before[kSegment];
        float h = carries[(b * shape.segments + segment) * shape.features + f];
        for (int j = 0; j < count; ++j) {
            const int64_t row = b * shape.length + first + j;
            if (shape.restart != nullptr && shape.restart[row]) h = 0.0f;
            before[j] = h;
            if (shape.valid == nullptr || shape.valid[row]) {
                const Gate g = gate_of(to_acc(projections[row * 2 * shape.features + f]),
                                       to_acc(projections[row * 2 * shape.features + shape.features + f]), shape.lo, shape.hi);
                h = fmaf(g.a, h, (1.0f - g.a) * g.k);
            }
        }
        for (int j = count - 1; j >= 0; --j) {
            const int64_t row = b * shape.length + first + j;
            const float adjoint = incoming + (grad_states != nullptr ? to_acc(grad_states[row * shape.features + f]) : 0.0f);
            float dp = 0.0f, dc = 0.0f;
            incoming = adjoint;
            if (shape.valid == nullptr || shape.valid[row]) {
                const Gate g = gate_of(to_acc(projections[row * 2 * shape.features + f]),
                                       to_acc(projections[row * 2 * shape.features + shape.features + f]), shape.lo, shape.hi);
                dp = adjoint * (before[j] - g.k) * ((shape.hi - shape.lo) * g.s * (1.0f - g.s));
                dc = adjoint * (1.0f - g.a) * (1.0f - g.k * g.k);
                incoming = g.a * adjoint;
            }
            if (shape.restart != nullptr && shape.restart[row]) incoming = 0.0f;
            grad_projections[row * 2 * shape.features + f] = from_acc<T>(dp);
            grad_projections[row * 2 * shape.features + shape.features + f] = from_acc<T>(dc);
        }
    }
    if (grad_initial != nullptr) grad_initial[lane] = incoming;
}

template <typename T>
int gated_forward(const GatedShape &shape, const void *projections, const float *initial, void *states,
                  float *final_state, float *carries, cudaStream_t stream) {
    const unsigned blocks = static_cast<unsigned>(ceil_div(shape.batch * shape.features, 128));
    gated_forward_lane_kernel<T><<<blocks, 128, 0, stream>>>(shape, static_cast<const T *>(projections), initial,
                                                             static_cast<T *>(states), final_state, carries);
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

template <typename T>
int gated_backward(const GatedShape &shape, const void *projections, const float *carries, const void *grad_states,
                   const float *grad_final, void *grad_projections, float *grad_initial, cudaStream_t stream) {
    const unsigned blocks = static_cast<unsigned>(ceil_div(shape.batch * shape.features, 128));
    gated_backward_lane_kernel<T><<<blocks, 128, 0, stream>>>(shape, static_cast<const T *>(projections), carries,
                                                              static_cast<const T *>(grad_states), grad_final,
                                                              static_cast<T *>(grad_projections), grad_initial);
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

int check_gated(const GatedShape &shape) {
    if (shape.batch < 0 || shape.length < 0 || shape.features < 0) {
        return fail(KOEMI_ERR_INVALID, "recurrence sizes must be non-negative");
    }
    if (!(shape.lo > 0.0f && shape.lo <= shape.hi && shape.hi < 1.0f)) {
        return fail(KOEMI_ERR_INVALID, "retention bounds must satisfy 0 < minimum <= maximum < 1");
    }
    constexpr int64_t kMost = int64_t(1) << 30;
    if (shape.batch > kMost || shape.length > kMost || shape.features > kMost ||
        (shape.features > 0 && shape.batch > (int64_t(1) << 36) / shape.features)) {
        return fail(KOEMI_ERR_INVALID, "recurrence tensor is too large");
    }
    return KOEMI_OK;
}

}  // namespace
}  // namespace koemi

using namespace koemi;

extern "C" int koemi_dense_gated_recurrence_forward(const void *projections, const float *initial,
                                                    const uint8_t *valid, const uint8_t *restart, void *states,
                                                    float *final_state, float *carries, int64_t batch, int64_t length,
                                                    int64_t features, float minimum_retention,
                                                    float maximum_retention, int dtype, void *stream) {
    clear_error();
    const GatedShape shape{batch, length, features, ceil_div(length, kSegment), minimum_retention, maximum_retention, valid, restart};
    const int rc = check_gated(shape);
    if (rc != KOEMI_OK) return rc;
    if (batch == 0 || length == 0 || features == 0) return KOEMI_OK;
    if (projections == nullptr || states == nullptr || final_state == nullptr) {
        return fail(KOEMI_ERR_INVALID, "projections, states and final_state must be non-NULL");
    }
    cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case KOEMI_F32: return gated_forward<float>(shape, projections, initial, states, final_state, carries, s);
        case KOEMI_F16: return gated_forward<__half>(shape, projections, initial, states, final_state, carries, s);
        case KOEMI_BF16: return gated_forward<__nv_bfloat16>(shape, projections, initial, states, final_state, carries, s);
        default: return fail(KOEMI_ERR_INVALID, "unsupported recurrence dtype %d", dtype);
    }
}

extern "C" int koemi_dense_gated_recurrence_backward(const void *projections, const uint8_t *valid,
                                                     const uint8_t *restart, const float *carries,
                                                     const void *grad_states, const float *grad_final,
                                                     void *grad_projections, float *grad_initial, int64_t batch,
                                                     int64_t length, int64_t features, float minimum_retention,
                                                     float maximum_retention, int dtype, void *stream) {
    clear_error();
    const GatedShape shape{batch, length, features, ceil_div(length, kSegment), minimum_retention, maximum_retention, valid, restart};
    const int rc = check_gated(shape);
    if (rc != KOEMI_OK) return rc;
    if (batch == 0 || length == 0 || features == 0) return KOEMI_OK;
    if (projections == nullptr || carries == nullptr || grad_projections == nullptr) {
        return fail(KOEMI_ERR_INVALID, "projections, carries and grad_projections must be non-NULL");
    }
    cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case KOEMI_F32: return gated_backward<float>(shape, projections, carries, grad_states, grad_final, grad_projections, grad_initial, s);
        case KOEMI_F16: return gated_backward<__half>(shape, projections, carries, grad_states, grad_final, grad_projections, grad_initial, s);
        case KOEMI_BF16: return gated_backward<__nv_bfloat16>(shape, projections, carries, grad_states, grad_final, grad_projections, grad_initial, s);
        default: return fail(KOEMI_ERR_INVALID, "unsupported recurrence dtype %d", dtype);
    }
}
