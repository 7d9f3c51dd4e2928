// MoE front: the learned route of a training step -- softmax over the gate's
// logits, top-k, per-expert counts, the balance loss -- and its gradient.
//
//   p = softmax(l);  i_1..i_k the k largest logits (ties: lowest id)
//   w_j = p_{i_j}, divided by their sum S under renormalisation
//   balance = E sum_e importance_e load_e, importance_e = sum_t p_te / N,
//   load_e = counts_e / sum counts (no gradient through the counts)
//   dl = p (dp - sum p dp),  dp_e = dw'_j (e = i_j) + dbalance E load_e / N,
//   dw' = dw, or (dw - sum dw w) / S under renormalisation
//
// Rows that are not valid, or whose logits are all -inf, take no part: ids
// -1, weights 0, gradient 0. A NaN logit is never preferred, and its row's
// probabilities are NaN. One warp works on one row at a time; a CTA adds its
// rows' probabilities up in a fixed order and leaves one partial row, and a
// second kernel adds the partial rows, so equal inputs give equal bits.
#include "common.cuh"

namespace koemi {
namespace {

constexpr int kRouteWarps = 8;
constexpr int kRouteBlocks = 296;

struct RouteShape {
    int64_t tokens, experts, top_k;
    bool renormalize;
    const uint8_t *valid;
};

__device__ __forceinline__ float selectable(float v) { return isnan(v) ? -INFINITY : v; }

struct RowSoftmax {
    float max, sum;
    bool live;
};

template <typename T>
__device__ RowSoftmax row_softmax(const T *row, int64_t experts, bool valid) {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY;
    bool nan = false;
    for (int64_t e = lane; e < experts; e += 32) {
        const float v = to_acc(row[e]);
        nan |= isnan(v);
        m = fmaxf(m, v);
    }
    m = warp_max(m);
    nan = __any_sync(0xffffffffu, nan);
    float sum = 0.0f;
    for (int64_t e = lane; e < experts; e += 32) sum += expf(to_acc(row[e]) - m);
    sum = warp_sum(sum);
    return RowSoftmax{m, sum, valid && (nan || m != -INFINITY)};
}

template <typename T>
__global__ void route_forward_kernel(RouteShape shape, const T *__restrict__ logits, int64_t *__restrict__ ids,
                                     float *__restrict__ weights, float *__restrict__ partial_mass,
                                     int32_t *__restrict__ partial_counts, int32_t *__restrict__ partial_live) {
    extern __shared__ float mass[];  // [warps][experts], then counts [experts]
    int32_t *counts = reinterpret_cast<int32_t *>(mass + kRouteWarps * shape.experts);
    __shared__ int32_t live_rows;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t i = threadIdx.x; i < (kRouteWarps + 1) * shape.experts; i += blockDim.x) mass[i] = 0.0f;
    if (threadIdx.x == 0) live_rows = 0;
    __syncthreads();
    for (int64_t t = int64_t(blockIdx.x) * kRouteWarps + warp; t < shape.tokens; t += int64_t(gridDim.x) * kRouteWarps) {
        const T *row = logits + t * shape.experts;
        const RowSoftmax soft = row_softmax(row, shape.experts, shape.valid == nullptr || shape.valid[t] != 0);
        if (!soft.live) {
            for (int64_t k = lane; k < shape.top_k; k += 32) {
                ids[t * shape.top_k + k] = -1;
                weights[t * shape.top_k + k] = 0.0f;
            }
            continue;
        }
        for (int64_t e = lane; e < shape.experts; e += 32) {
            mass[warp * shape.experts + e] += expf(to_acc(row[e]) - soft.max) / soft.sum;
        }
        float last = INFINITY, chosen = 0.0f;
        int64_t last_id = -1;
        for (int64_t k = 0; k < shape.top_k; ++k) {
            float best = -INFINITY;
            int64_t best_id = INT64_MAX;
            for (int64_t e = lane; e < shape.experts; e += 32) {
                const float v = selectable(to_acc(row[e]));
                const bool after = v < last || (v == last && e > last_id);
                if (after && (best_id == INT64_MAX || v > best)) best = v, best_id = e;
            }
#pragma unroll
            for (int offset = 16; offset > 0; offset >>= 1) {
                const float v = __shfl_xor_sync(0xffffffffu, best, offset);
                const int64_t id = __shfl_xor_sync(0xffffffffu, best_id, offset);
                if (v > best || (v == best && id < best_id)) best = v, best_id = id;
            }
            last = best;
            last_id = best_id;
            const float p = expf(to_acc(row[best_id]) - soft.max) / soft.sum;
            chosen += p;
            if (lane == 0) {
                ids[t * shape.top_k + k] = best_id;
                weights[t * shape.top_k + k] = p;
                atomicAdd(&counts[best_id], 1);
            }
        }
        if (lane == 0) {
            atomicAdd(&live_rows, 1);
            if (shape.renormalize) {
                for (int64_t k = 0; k < shape.top_k; ++k) weights[t * shape.top_k + k] /= chosen;
            }
        }
    }
    __syncthreads();
    for (int64_t e = threadIdx.x; e < shape.experts; e += blockDim.x) {
        float sum = 0.0f;
        for (int w = 0; w < kRouteWarps; ++w) sum += mass[w * shape.experts + e];
        partial_mass[blockIdx.x * shape.experts + e] = sum;
        partial_counts[blockIdx.x * shape.experts + e] = counts[e];
    }
    if (threadIdx.x == 0) partial_live[blockIdx.x] = live_rows;
}

__global__ void route_finish_kernel(const float *__restrict__ partial_mass, const int32_t *__restrict__ partial_counts,
                                    const int32_t *__restrict__ partial_live, int64_t blocks, int64_t experts,
                                    int64_t top_k, int64_t *__restrict__ counts, float *__restrict__ balance,
                                    float *__restrict__ slope) {
    __shared__ float sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t live = 0;
    for (int64_t b = 0; b < blocks; ++b) live += partial_live[b];
    const float n = static_cast<float>(live > 0 ? live : 1);
    const float scale = static_cast<float>(experts) / n / (n * static_cast<float>(top_k));
    float total = 0.0f;
    for (int64_t e = threadIdx.x; e < experts; e += blockDim.x) {
        double mass = 0.0;
        int64_t count = 0;
        for (int64_t b = 0; b < blocks; ++b) {
            mass += partial_mass[b * experts + e];
            count += partial_counts[b * experts + e];
        }
        counts[e] = count;
        slope[e] = scale * static_cast<float>(count);
        total += static_cast<float>(mass) * slope[e];
    }
    total = warp_sum(total);
    if (lane == 0) sums[warp] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
        float all = 0.0f;
        for (unsigned w = 0; w < blockDim.x / 32; ++w) all += sums[w];
        *balance = all;
    }
}

template <typename T>
__global__ void route_backward_kernel(RouteShape shape, const T *__restrict__ logits, const int64_t *__restrict__ ids,
                                      const float *__restrict__ weights, const float *__restrict__ grad_weights,
                                      const float *__restrict__ grad_balance, const float *__restrict__ slope,
                                      T *__restrict__ grad_logits) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float db = grad_balance != nullptr ? *grad_balance : 0.0f;
    for (int64_t t = int64_t(blockIdx.x) * kRouteWarps + warp; t < shape.tokens; t += int64_t(gridDim.x) * kRouteWarps) {
        const T *row = logits + t * shape.experts;
        T *out = grad_logits + t * shape.experts;
        const int64_t *chosen = ids + t * shape.top_k;
        if (chosen[0] < 0) {
            for (int64_t e = lane; e < shape.experts; e += 32) out[e] = from_acc<T>(0.0f);
            continue;
        }
        const RowSoftmax soft = row_softmax(row, shape.experts, true);
        float total = 1.0f, mean = 0.0f;
        if (shape.renormalize) {
            total = 0.0f;
            for (int64_t k = 0; k < shape.top_k; ++k) {
                total += expf(to_acc(row[chosen[k]]) - soft.max) / soft.sum;
                if (grad_weights != nullptr) mean += grad_weights[t * shape.top_k + k] * weights[t * shape.top_k + k];
            }
        }
        float dot = 0.0f;
        for (int64_t e = lane; e < shape.experts; e += 32) {
            float dp = db * slope[e];
            if (grad_weights != nullptr) {
                for (int64_t k = 0; k < shape.top_k; ++k) {
                    if (chosen[k] == e) dp += (grad_weights[t * shape.top_k + k] - mean) / total;
                }
            }
            dot += expf(to_acc(row[e]) - soft.max) / soft.sum * dp;
        }
        dot = warp_sum(dot);
        for (int64_t e = lane; e < shape.experts; e += 32) {
            float dp = db * slope[e];
            if (grad_weights != nullptr) {
                for (int64_t k = 0; k < shape.top_k; ++k) {
                    if (chosen[k] == e) dp += (grad_weights[t * shape.top_k + k] - mean) / total;
                }
            }
            out[e] = from_acc<T>(expf(to_acc(row[e]) - soft.max) / soft.sum * (dp - dot));
        }
    }
}

int64_t route_blocks(int64_t tokens) {
    const int64_t blocks = ceil_div(tokens, kRouteWarps);
    return blocks < kRouteBlocks ? (blocks > 0 ? blocks : 1) : kRouteBlocks;
}

int check_route(const RouteShape &shape) {
    if (shape.tokens < 0 || shape.tokens > (int64_t(1) << 31)) return fail(KOEMI_ERR_INVALID, "tokens must be in [0, 2^31]");
    if (shape.experts < 1 || shape.experts > 4096) return fail(KOEMI_ERR_INVALID, "expert_count must be in [1, 4096]");
    if (shape.top_k < 1 || shape.top_k > shape.experts || shape.top_k > 256) {
        return fail(KOEMI_ERR_INVALID, "top_k must be in [1, min(expert_count, 256)]");
    }
    return KOEMI_OK;
}

template <typename T>
int route_forward(const RouteShape &shape, const void *logits, int64_t *ids, float *weights, int64_t *counts,
                  float *balance, float *slope, void *workspace, cudaStream_t stream) {
    const int64_t blocks = route_blocks(shape.tokens);
    float *mass = static_cast<float *>(workspace);
    int32_t *partial_counts = reinterpret_cast<int32_t *>(mass + blocks * shape.experts);
    int32_t *live = partial_counts + blocks * shape.experts;
    const size_t smem = (kRouteWarps + 1) * shape.experts * sizeof(float);
    auto kernel = route_forward_kernel<T>;
    KOEMI_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    kernel<<<static_cast<unsigned>(blocks), kRouteWarps * 32, smem, stream>>>(
        shape, static_cast<const T *>(logits), ids, weights, mass, partial_counts, live);
    KOEMI_LAUNCH_CHECK();
    route_finish_kernel<<<1, 512, 0, stream>>>(mass, partial_counts, live, blocks, shape.experts, shape.top_k, counts,
                                               balance, slope);
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

template <typename T>
int route_backward(const RouteShape &shape, const void *logits, const int64_t *ids, const float *weights,
                   const float *grad_weights, const float *grad_balance, const float *slope, void *grad_logits,
                   cudaStream_t stream) {
    route_backward_kernel<T><<<static_cast<unsigned>(route_blocks(shape.tokens)), kRouteWarps * 32, 0, stream>>>(
        shape, static_cast<const T *>(logits), ids, weights, grad_weights, grad_balance, slope,
        static_cast<T *>(grad_logits));
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

}  // namespace
}  // namespace koemi

using namespace koemi;

extern "C" size_t koemi_moe_route_learned_workspace(int64_t tokens, int64_t expert_count) {
    if (tokens < 0 || expert_count < 1) return 0;
    const int64_t blocks = route_blocks(tokens);
    return static_cast<size_t>(blocks * (2 * expert_count + 1)) * 4;
}

extern "C" int koemi_moe_route_learned_forward(const void *logits, const uint8_t *valid, int64_t *expert_ids,
                                               float *weights, int64_t *counts, float *balance, float *slope,
                                               int64_t tokens, int64_t expert_count, int64_t top_k, int renormalize,
                                               int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    const RouteShape shape{tokens, expert_count, top_k, renormalize != 0, valid};
    const int rc = check_route(shape);
    if (rc != KOEMI_OK) return rc;
    if (counts == nullptr || balance == nullptr || slope == nullptr || workspace == nullptr ||
        (tokens > 0 && (logits == nullptr || expert_ids == nullptr || weights == nullptr))) {
        return fail(KOEMI_ERR_INVALID, "route tensors and workspace must be non-NULL");
    }
    if (workspace_bytes < koemi_moe_route_learned_workspace(tokens, expert_count)) {
        return fail(KOEMI_ERR_WORKSPACE, "the route's workspace is smaller than koemi_moe_route_learned_workspace()");
    }
    cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case KOEMI_F32: return route_forward<float>(shape, logits, expert_ids, weights, counts, balance, slope, workspace, s);
        case KOEMI_F16: return route_forward<__half>(shape, logits, expert_ids, weights, counts, balance, slope, workspace, s);
        case KOEMI_BF16: return route_forward<__nv_bfloat16>(shape, logits, expert_ids, weights, counts, balance, slope, workspace, s);
        default: return fail(KOEMI_ERR_INVALID, "unsupported route dtype %d", dtype);
    }
}

extern "C" int koemi_moe_route_learned_backward(const void *logits, const int64_t *expert_ids, const float *weights,
                                                const float *grad_weights, const float *grad_balance,
                                                const float *slope, void *grad_logits, int64_t tokens,
                                                int64_t expert_count, int64_t top_k, int renormalize, int dtype,
                                                void *stream) {
    clear_error();
    const RouteShape shape{tokens, expert_count, top_k, renormalize != 0, nullptr};
    const int rc = check_route(shape);
    if (rc != KOEMI_OK) return rc;
    if (tokens == 0) return KOEMI_OK;
    if (logits == nullptr || expert_ids == nullptr || weights == nullptr || slope == nullptr || grad_logits == nullptr) {
        return fail(KOEMI_ERR_INVALID, "route backward tensors must be non-NULL");
    }
    cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case KOEMI_F32: return route_backward<float>(shape, logits, expert_ids, weights, grad_weights, grad_balance, slope, grad_logits, s);
        case KOEMI_F16: return route_backward<__half>(shape, logits, expert_ids, weights, grad_weights, grad_balance, slope, grad_logits, s);
        case KOEMI_BF16: return route_backward<__nv_bfloat16>(shape, logits, expert_ids, weights, grad_weights, grad_balance, slope, grad_logits, s);
        default: return fail(KOEMI_ERR_INVALID, "unsupported route dtype %d", dtype);
    }
}
