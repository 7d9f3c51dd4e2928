// Think front: clipped policy loss with a KL term over vocabulary logits,
// forward and gradient.
//
//   lp = l[target] - lse(l),  r = exp(lp - old),  d = ref - lp
//   loss_t = -min(r A, clip(r, 1 - cl, 1 + ch) A) + beta (exp(d) - d - 1)
//   loss = sum over valid rows / N,  kl = sum (exp(d) - d - 1) / N
//   dloss/dlp = (-r A where the unclipped term is the smaller) + beta (1 - exp(d)),
//   dlogits = dloss/dlp (onehot - softmax(l)) / N
//
// Rows that are not valid read nothing of their logits, give log-prob 0 and
// gradient 0. A target outside [0, vocab) makes its row's log-prob NaN.
// A CTA takes whole rows; per-CTA sums are added in a fixed order by a second
// kernel, so equal inputs give equal bits.
#include "vec.cuh"

namespace koemi {
namespace {

constexpr int kPolicyThreads = 256;
constexpr int kPolicyBlocks = 592;

// Row r of the logits starts at (r / inner) * outer_stride + (r % inner) *
// inner_stride elements.
struct PolicyRows {
    int64_t rows, vocab, inner, outer_stride, inner_stride;
    __device__ int64_t start(int64_t row) const {
        return (row / inner) * outer_stride + (row % inner) * inner_stride;
    }
};

struct PolicyTerms {
    const int64_t *targets;
    const float *old, *advantages, *reference;  // reference may be NULL: no KL term
    const uint8_t *valid;                       // may be NULL: every row
    float clip_low, clip_high, beta;
};

__device__ __forceinline__ float block_max(float v, float *scratch) {
    v = warp_max(v);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[0];
    for (unsigned w = 1; w < blockDim.x / 32; ++w) v = fmaxf(v, scratch[w]);
    __syncthreads();
    return v;
}
__device__ __forceinline__ float block_sum(float v, float *scratch) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    for (unsigned w = 0; w < blockDim.x / 32; ++w) v += scratch[w];
    __syncthreads();
    return v;
}

// Loss, KL and d loss / d log-prob of one row.
__device__ __forceinline__ void policy_terms(const PolicyTerms &terms, int64_t row, float lp, float &loss, float &kl,
                                             float &slope) {
    const float a = terms.advantages[row];
    const float r = expf(lp - terms.old[row]);
    const float free = r * a;
    const float clipped = fminf(fmaxf(r, 1.0f - terms.clip_low), 1.0f + terms.clip_high) * a;
    const bool take = free <= clipped;
    loss = -(take ? free : clipped);
    slope = take ? -free : 0.0f;
    kl = 0.0f;
    if (terms.reference != nullptr) {
        const float d = terms.reference[row] - lp;
        const float e = expm1f(d);
        kl = e - d;
        loss += terms.beta * kl;
        slope -= terms.beta * e;
    }
    if (isnan(free) || isnan(clipped)) loss = slope = NAN;
}

__global__ void policy_count_kernel(const uint8_t *__restrict__ valid, int64_t rows, float *__restrict__ inverse) {
    __shared__ int32_t sums[32];
    int32_t count = 0;
    for (int64_t i = threadIdx.x; i < rows; i += blockDim.x) count += valid == nullptr || valid[i] != 0;
    count = __reduce_add_sync(0xffffffffu, count);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = count;
    __syncthreads();
    if (threadIdx.x == 0) {
        int64_t all = 0;
        for (unsigned w = 0; w < blockDim.x / 32; ++w) all += sums[w];
        *inverse = 1.0f / static_cast<float>(all > 0 ? all : 1);
    }
}

template <typename T>
__global__ __launch_bounds__(kPolicyThreads) void policy_forward_kernel(
    PolicyRows shape, PolicyTerms terms, const T *__restrict__ logits, const float *__restrict__ inverse,
    float *__restrict__ log_probs, float *__restrict__ lse_out, float *__restrict__ slope_out,
    T *__restrict__ grad_logits, float2 *__restrict__ partials) {
    __shared__ float scratch[kPolicyThreads / 32];
    const float scale = *inverse;
    float loss_sum = 0.0f, kl_sum = 0.0f;
    for (int64_t row = blockIdx.x; row < shape.rows; row += gridDim.x) {
        const T *in = logits + shape.start(row);
        T *out = grad_logits == nullptr ? nullptr : grad_logits + row * shape.vocab;
        if (terms.valid != nullptr && terms.valid[row] == 0) {
            if (out != nullptr) {
                for (int64_t v = threadIdx.x; v < shape.vocab; v += blockDim.x) out[v] = from_acc<T>(0.0f);
            }
            if (threadIdx.x == 0) log_probs[row] = lse_out[row] = slope_out[row] = 0.0f;
            continue;
        }
        float m = -INFINITY;
        for (int64_t v = threadIdx.x; v < shape.vocab; v += blockDim.x) m = fmaxf(m, to_acc(in[v]));
        m = block_max(m, scratch);
        float sum = 0.0f;
        for (int64_t v = threadIdx.x; v < shape.vocab; v += blockDim.x) sum += expf(to_acc(in[v]) - m);
        sum = block_sum(sum, scratch);
        const float lse = m + logf(sum);
        const int64_t target = terms.targets[row];
        const float lp = target >= 0 && target < shape.vocab ? to_acc(in[target]) - lse : NAN;
        float loss, kl, slope;
        policy_terms(terms, row, lp, loss, kl, slope);
        loss_sum += loss;
        kl_sum += kl;
        slope *= scale;
        if (threadIdx.x == 0) {
            log_probs[row] = lp;
            lse_out[row] = lse;
            slope_out[row] = slope;
        }
        if (out != nullptr) {
            for (int64_t v = threadIdx.x; v < shape.vocab; v += blockDim.x) {
                out[v] = from_acc<T>(slope * ((v == target ? 1.0f : 0.0f) - expf(to_acc(in[v]) - lse)));
            }
        }
    }
    if (threadIdx.x == 0) partials[blockIdx.x] = make_float2(loss_sum, kl_sum);
}

__global__ void policy_finish_kernel(const float2 *__restrict__ partials, int64_t count,
                                     const float *__restrict__ inverse, float *__restrict__ loss,
                                     float *__restrict__ kl) {
    double l = 0.0, k = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += 32) {
        l += partials[i].x;
        k += partials[i].y;
    }
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, offset);
        k += __shfl_xor_sync(0xffffffffu, k, offset);
    }
    if (threadIdx.x == 0) {
        *loss = static_cast<float>(l * *inverse);
        *kl = static_cast<float>(k * *inverse);
    }
}

template <typename T>
__global__ __launch_bounds__(kPolicyThreads) void policy_backward_kernel(
    PolicyRows shape, const T *__restrict__ logits, const int64_t *__restrict__ targets,
    const uint8_t *__restrict__ valid, const float *__restrict__ lse, const float *__restrict__ slopes,
    const float *__restrict__ grad_loss, T *__restrict__ grad_logits) {
    const float scale = *grad_loss;
    for (int64_t row = blockIdx.x; row < shape.rows; row += gridDim.x) {
        const T *in = logits + shape.start(row);
        T *out = grad_logits + row * shape.vocab;
        const bool live = valid == nullptr || valid[row] != 0;
        const float slope = slopes[row] * scale, z = lse[row];
        const int64_t target = targets[row];
        for (int64_t v = threadIdx.x; v < shape.vocab; v += blockDim.x) {
            const float g = live ? slope * ((v == target ? 1.0f : 0.0f) - expf(to_acc(in[v]) - z)) : 0.0f;
            out[v] = from_acc<T>(g);
        }
    }
}

// grad *= *factor, unless the factor is one.
template <typename T>
__global__ void policy_scale_kernel(T *__restrict__ grad, int64_t count, const float *__restrict__ factor) {
    const float f = *factor;
    if (f == 1.0f) return;
    for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < count; i += int64_t(gridDim.x) * blockDim.x) {
        grad[i] = from_acc<T>(to_acc(grad[i]) * f);
    }
}

unsigned policy_blocks(int64_t rows) {
    return static_cast<unsigned>(rows < kPolicyBlocks ? (rows > 0 ? rows : 1) : kPolicyBlocks);
}

int check_policy(const PolicyRows &shape) {
    if (shape.rows < 0 || shape.rows > (int64_t(1) << 31)) return fail(KOEMI_ERR_INVALID, "rows must be in [0, 2^31]");
    if (shape.vocab < 1 || shape.vocab > (int64_t(1) << 30)) return fail(KOEMI_ERR_INVALID, "vocab must be in [1, 2^30]");
    if (shape.inner < 1) return fail(KOEMI_ERR_INVALID, "inner_rows must be positive");
    return KOEMI_OK;
}

template <typename T>
int policy_forward(const PolicyRows &shape, const PolicyTerms &terms, const void *logits, float *loss, float *kl,
                   float *log_probs, float *lse, float *slopes, void *grad_logits, void *workspace,
                   cudaStream_t stream) {
    float *inverse = static_cast<float *>(workspace);
    float2 *partials = reinterpret_cast<float2 *>(static_cast<unsigned char *>(workspace) + 256);
    policy_count_kernel<<<1, 1024, 0, stream>>>(terms.valid, shape.rows, inverse);
    KOEMI_LAUNCH_CHECK();
    const unsigned blocks = policy_blocks(shape.rows);
    policy_forward_kernel<T><<<blocks, kPolicyThreads, 0, stream>>>(shape, terms, static_cast<const T *>(logits), inverse,
                                                                    log_probs, lse, slopes,
                                                                    static_cast<T *>(grad_logits), partials);
    KOEMI_LAUNCH_CHECK();
    policy_finish_kernel<<<1, 32, 0, stream>>>(partials, blocks, inverse, loss, kl);
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

template <typename T>
int policy_backward(const PolicyRows &shape, const void *logits, const int64_t *targets, const uint8_t *valid,
                    const float *lse, const float *slopes, const float *grad_loss, void *grad_logits,
                    cudaStream_t stream) {
    policy_backward_kernel<T><<<policy_blocks(shape.rows), kPolicyThreads, 0, stream>>>(
        shape, static_cast<const T *>(logits), targets, valid, lse, slopes, grad_loss, static_cast<T *>(grad_logits));
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

template <typename T>
int policy_scale(void *grad, int64_t count, const float *factor, cudaStream_t stream) {
    const int64_t blocks = ceil_div(count, 256);
    policy_scale_kernel<T><<<static_cast<unsigned>(blocks < 1184 ? blocks : 1184), 256, 0, stream>>>(
        static_cast<T *>(grad), count, factor);
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

}  // namespace
}  // namespace koemi

using namespace koemi;

extern "C" size_t koemi_think_policy_loss_workspace(void) { return 256 + kPolicyBlocks * sizeof(float2); }

extern "C" int koemi_think_policy_loss_forward(const void *logits, int64_t rows, int64_t vocab, int64_t inner_rows,
                                               int64_t outer_stride, int64_t inner_stride, const int64_t *targets,
                                               const float *old_log_probs, const float *advantages,
                                               const float *reference_log_probs, const uint8_t *valid, float clip_low,
                                               float clip_high, float kl_weight, float *loss, float *kl,
                                               float *log_probs, float *lse, float *slopes, void *grad_logits,
                                               int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    const PolicyRows shape{rows, vocab, inner_rows, outer_stride, inner_stride};
    const int rc = check_policy(shape);
    if (rc != KOEMI_OK) return rc;
    if (!(clip_low >= 0.0f && clip_high >= 0.0f)) return fail(KOEMI_ERR_INVALID, "clip widths must be non-negative");
    if (loss == nullptr || kl == nullptr || workspace == nullptr ||
        (rows > 0 && (logits == nullptr || targets == nullptr || old_log_probs == nullptr || advantages == nullptr ||
                      log_probs == nullptr || lse == nullptr || slopes == nullptr))) {
        return fail(KOEMI_ERR_INVALID, "policy loss tensors and workspace must be non-NULL");
    }
    if (workspace_bytes < koemi_think_policy_loss_workspace()) {
        return fail(KOEMI_ERR_WORKSPACE, "the policy loss's workspace is smaller than koemi_think_policy_loss_workspace()");
    }
    const PolicyTerms terms{targets, old_log_probs, advantages, reference_log_probs, valid, clip_low, clip_high, kl_weight};
    cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case KOEMI_F32: return policy_forward<float>(shape, terms, logits, loss, kl, log_probs, lse, slopes, grad_logits, workspace, s);
        case KOEMI_F16: return policy_forward<__half>(shape, terms, logits, loss, kl, log_probs, lse, slopes, grad_logits, workspace, s);
        case KOEMI_BF16: return policy_forward<__nv_bfloat16>(shape, terms, logits, loss, kl, log_probs, lse, slopes, grad_logits, workspace, s);
        default: return fail(KOEMI_ERR_INVALID, "unsupported policy loss dtype %d", dtype);
    }
}

extern "C" int koemi_think_policy_loss_backward(const void *logits, int64_t rows, int64_t vocab, int64_t inner_rows,
                                                int64_t outer_stride, int64_t inner_stride, const int64_t *targets,
                                                const uint8_t *valid, const float *lse, const float *slopes,
                                                const float *grad_loss, void *grad_logits, int dtype, void *stream) {
    clear_error();
    const PolicyRows shape{rows, vocab, inner_rows, outer_stride, inner_stride};
    const int rc = check_policy(shape);
    if (rc != KOEMI_OK) return rc;
    if (rows == 0) return KOEMI_OK;
    if (logits == nullptr || targets == nullptr || lse == nullptr || slopes == nullptr || grad_loss == nullptr ||
        grad_logits == nullptr) {
        return fail(KOEMI_ERR_INVALID, "policy loss backward tensors must be non-NULL");
    }
    cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case KOEMI_F32: return policy_backward<float>(shape, logits, targets, valid, lse, slopes, grad_loss, grad_logits, s);
        case KOEMI_F16: return policy_backward<__half>(shape, logits, targets, valid, lse, slopes, grad_loss, grad_logits, s);
        case KOEMI_BF16: return policy_backward<__nv_bfloat16>(shape, logits, targets, valid, lse, slopes, grad_loss, grad_logits, s);
        default: return fail(KOEMI_ERR_INVALID, "unsupported policy loss dtype %d", dtype);
    }
}

extern "C" int koemi_think_policy_loss_scale(void *grad_logits, int64_t count, const float *factor, int dtype,
                                             void *stream) {
    clear_error();
    if (count < 0) return fail(KOEMI_ERR_INVALID, "count must be non-negative");
    if (count == 0) return KOEMI_OK;
    if (grad_logits == nullptr || factor == nullptr) return fail(KOEMI_ERR_INVALID, "grad_logits and factor must be non-NULL");
    cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case KOEMI_F32: return policy_scale<float>(grad_logits, count, factor, s);
        case KOEMI_F16: return policy_scale<__half>(grad_logits, count, factor, s);
        case KOEMI_BF16: return policy_scale<__nv_bfloat16>(grad_logits, count, factor, s);
        default: return fail(KOEMI_ERR_INVALID, "unsupported policy loss dtype %d", dtype);
    }
}
