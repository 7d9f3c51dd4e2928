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
// probabilities are NaN. A CTA adds its rows' probabilities up in a fixed order
// and leaves one partial row, and a second kernel adds the partial rows, so
// equal inputs give equal bits.
//
// Up to 256 experts a row is held in registers by a group of 8, 16 or 32
// lanes, element e in lane e % lanes: every logit is loaded once, and a warp
// works on 1 to 4 rows. Wider rows are walked from memory by one warp
// (route_*_wide_kernel).
//
// A row is a chain of reductions and its bytes are few: 32768 tokens of 64
// fp32 logits, top-2, take 11.8 us (8.4 MB, 1.3 us of copy bandwidth), the
// second kernel 6.5 us and the gradient 7.1 us (16.8 MB, 2.6 us); 256 tokens
// 3.5 and 2.8 us, the latency of two launches.
#include <type_traits>

#include "common.cuh"

namespace koemi {
namespace {

constexpr int kRouteWarps = 16;  // 32 warps per SM: a row is a chain of reductions
constexpr int kWideWarps = 8;    // each has a row of sums in shared memory
constexpr int kRouteBlocks = 296;
constexpr int kMostExperts = 4096;

struct RouteShape {
    int64_t tokens, experts, top_k;
    bool renormalize;
    const uint8_t *valid;
};

__device__ __forceinline__ float selectable(float v) { return isnan(v) ? -INFINITY : v; }

// Where the results over all rows go.
struct RouteTotals {
    int64_t *counts;
    float *balance, *slope;
};
// d balance / d probability of any row: E counts_e / (N sum counts), all rows
// that take part having top_k pairs.
__device__ __forceinline__ float balance_slope(int64_t experts, int64_t top_k, int64_t live, int64_t count) {
    const float n = static_cast<float>(live > 0 ? live : 1);
    return static_cast<float>(experts) / n / (n * static_cast<float>(top_k)) * static_cast<float>(count);
}

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
__global__ void route_forward_wide_kernel(RouteShape shape, const T *__restrict__ logits, int64_t *__restrict__ ids,
                                     float *__restrict__ weights, float *__restrict__ partial_mass,
                                     int32_t *__restrict__ partial_counts, int32_t *__restrict__ partial_live) {
    extern __shared__ float mass[];  // [warps][experts], then counts [experts]
    int32_t *counts = reinterpret_cast<int32_t *>(mass + kWideWarps * shape.experts);
    __shared__ int32_t live_rows;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t i = threadIdx.x; i < (kWideWarps + 1) * shape.experts; i += blockDim.x) mass[i] = 0.0f;
    if (threadIdx.x == 0) live_rows = 0;
    __syncthreads();
    for (int64_t t = int64_t(blockIdx.x) * kWideWarps + warp; t < shape.tokens; t += int64_t(gridDim.x) * kWideWarps) {
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
        for (int w = 0; w < kWideWarps; ++w) sum += mass[w * shape.experts + e];
        partial_mass[blockIdx.x * shape.experts + e] = sum;
        partial_counts[blockIdx.x * shape.experts + e] = counts[e];
    }
    if (threadIdx.x == 0) partial_live[blockIdx.x] = live_rows;
}

// Adds the partial rows: `parts` threads per expert take every parts-th block,
// then one adds the parts, always in the same order.
constexpr int kFinishThreads = 1024;
__global__ __launch_bounds__(kFinishThreads) void route_finish_kernel(
    const float *__restrict__ partial_mass, const int32_t *__restrict__ partial_counts,
    const int32_t *__restrict__ partial_live, int blocks, int experts, int64_t top_k, int64_t *__restrict__ counts,
    float *__restrict__ balance, float *__restrict__ slope) {
    __shared__ double masses[kFinishThreads];
    __shared__ int64_t pairs[kFinishThreads];
    __shared__ int64_t live_sums[kFinishThreads / 32];
    __shared__ float sums[kFinishThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int live = 0;
    for (int b = threadIdx.x; b < blocks; b += kFinishThreads) live += partial_live[b];
    live = __reduce_add_sync(0xffffffffu, live);
    if (lane == 0) live_sums[warp] = live;
    const int width = experts < kFinishThreads ? experts : kFinishThreads, parts = kFinishThreads / width;
    const int part = threadIdx.x / width, column = threadIdx.x - part * width;
    float total = 0.0f;
    for (int first = 0; first < experts; first += width) {
        const int e = first + column;
        double mass = 0.0;
        int64_t count = 0;
        if (part < parts && e < experts) {
#pragma unroll 4
            for (int b = part; b < blocks; b += parts) {
                mass += partial_mass[int64_t(b) * experts + e];
                count += partial_counts[int64_t(b) * experts + e];
            }
        }
        masses[threadIdx.x] = mass;
        pairs[threadIdx.x] = count;
        __syncthreads();
        if (part == 0 && e < experts) {
            int64_t all = 0;
            for (int w = 0; w < kFinishThreads / 32; ++w) all += live_sums[w];
            for (int i = 1; i < parts; ++i) {
                mass += masses[i * width + column];
                count += pairs[i * width + column];
            }
            const float s = balance_slope(experts, top_k, all, count);
            counts[e] = count;
            slope[e] = s;
            total += static_cast<float>(mass) * s;
        }
        __syncthreads();
    }
    total = warp_sum(total);
    if (lane == 0) sums[warp] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
        float all = 0.0f;
        for (int w = 0; w < kFinishThreads / 32; ++w) all += sums[w];
        *balance = all;
    }
}

// ------------------------------------------------------- rows in registers

// e^(v - max): the difference is exact to half a unit, ex2.approx to 2 units.
__device__ __forceinline__ float exp_from(float v, float max) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"((v - max) * 1.4426950408889634f));
    return r;
}
template <int kLanes>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int offset = kLanes / 2; offset > 0; offset >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, offset));
    return v;
}
template <int kLanes>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int offset = kLanes / 2; offset > 0; offset >>= 1) v += __shfl_xor_sync(0xffffffffu, v, offset);
    return v;
}
// The value's order as an integer; a NaN ranks with -inf. 0: no candidate.
__device__ __forceinline__ uint32_t rank_key(float v) {
    const uint32_t bits = __float_as_uint(selectable(v) + 0.0f);  // -0 becomes +0
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// One row of a group: the lane's logits become exponentials; -inf beyond the row.
template <typename T, int kLanes, int kPer>
__device__ __forceinline__ RowSoftmax load_row(const T *row, int experts, int at, bool take, float (&logit)[kPer],
                                               float (&e)[kPer]) {
    float m = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int id = at + j * kLanes;
        logit[j] = take && id < experts ? to_acc(row[id]) : -INFINITY;
        nan |= isnan(logit[j]);
        m = fmaxf(m, logit[j]);
    }
    m = group_max<kLanes>(m);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        e[j] = exp_from(logit[j], m);
        sum += at + j * kLanes < experts ? e[j] : 0.0f;
    }
    sum = group_sum<kLanes>(sum);
    const bool any_nan = group_max<kLanes>(nan ? 1.0f : 0.0f) != 0.0f;  // the maximum passes NaNs over
    return RowSoftmax{m, sum, take && (m != -INFINITY || any_nan)};
}

template <typename T, int kLanes, int kPer>
__global__ __launch_bounds__(kRouteWarps * 32, 2) void route_forward_kernel(
    RouteShape shape, const T *__restrict__ logits, int64_t *__restrict__ ids, float *__restrict__ weights,
    float *__restrict__ partial_mass, int32_t *__restrict__ partial_counts, int32_t *__restrict__ partial_live,
    RouteTotals totals) {
    constexpr int kGroups = kRouteWarps * 32 / kLanes, kWidth = kLanes * kPer;
    __shared__ float mass[kRouteWarps][kWidth];
    __shared__ int32_t counts[kWidth];
    __shared__ int32_t live_rows;
    const int at = threadIdx.x % kLanes, group = threadIdx.x / kLanes, warp = threadIdx.x >> 5;
    // the lanes of this group: the reductions of a warp's groups are apart
    const uint32_t members = kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1) << (threadIdx.x % 32 / kLanes * kLanes);
    const int experts = static_cast<int>(shape.experts), top_k = static_cast<int>(shape.top_k);
    for (int i = threadIdx.x; i < kWidth; i += blockDim.x) counts[i] = 0;
    if (threadIdx.x == 0) live_rows = 0;
    __syncthreads();
    float summed[kPer] = {};
    int live = 0;
    // every group of a warp takes the same number of turns: the shuffles are the warp's
    for (int64_t first = int64_t(blockIdx.x) * kGroups; first < shape.tokens; first += int64_t(gridDim.x) * kGroups) {
        const int64_t t = first + group;
        const bool take = t < shape.tokens && (shape.valid == nullptr || shape.valid[t] != 0);
        float logit[kPer], e[kPer];
        const RowSoftmax soft = load_row<T, kLanes, kPer>(logits + t * shape.experts, experts, at, take, logit, e);
        const float inverse = 1.0f / soft.sum;
        uint32_t keys[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int id = at + j * kLanes;
            keys[j] = id < experts ? rank_key(logit[j]) : 0;
            if (soft.live && id < experts) summed[j] += e[j] * inverse;
        }
        live += soft.live && at == 0;
        // Choice k stays in lane k % lanes, slot k / lanes, until all are known.
        float chosen = 0.0f, weight[kPer] = {};
        int choice[kPer] = {};
        for (int k = 0; k < top_k; ++k) {
            uint32_t best = keys[0];
#pragma unroll
            for (int j = 1; j < kPer; ++j) best = keys[j] > best ? keys[j] : best;
            best = __reduce_max_sync(members, best);
            uint32_t id = 0xffffffffu;  // the lowest that has it
#pragma unroll
            for (int j = kPer - 1; j >= 0; --j) id = keys[j] == best ? at + j * kLanes : id;
            id = __reduce_min_sync(members, id);
#pragma unroll
            for (int j = 0; j < kPer; ++j) keys[j] = static_cast<uint32_t>(at + j * kLanes) == id ? 0 : keys[j];
            const float p = exp_from(value_of(best), soft.max) * inverse;
            chosen += p;
            if (k < kLanes) {
                weight[0] = k == at ? p : weight[0];
                choice[0] = k == at ? static_cast<int>(id) : choice[0];
            } else {
#pragma unroll
                for (int j = 1; j < kPer; ++j) {
                    weight[j] = k == at + j * kLanes ? p : weight[j];
                    choice[j] = k == at + j * kLanes ? static_cast<int>(id) : choice[j];
                }
            }
        }
        if (t < shape.tokens) {
            const float share = shape.renormalize ? 1.0f / chosen : 1.0f;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const int k = at + j * kLanes;
                if (k >= top_k) continue;
                ids[t * top_k + k] = soft.live ? choice[j] : -1;
                weights[t * top_k + k] = soft.live ? weight[j] * share : 0.0f;
                if (soft.live) atomicAdd(&counts[choice[j]], 1);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        // the warp's groups, then the CTA's warps
#pragma unroll
        for (int offset = kLanes; offset < 32; offset <<= 1) summed[j] += __shfl_xor_sync(0xffffffffu, summed[j], offset);
        if ((threadIdx.x & 31) < kLanes) mass[warp][at + j * kLanes] = summed[j];
    }
    if (live > 0) atomicAdd(&live_rows, live);
    __syncthreads();
    float total = 0.0f;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kRouteWarps; ++w) sum += mass[w][e];
        if (gridDim.x > 1) {
            partial_mass[int64_t(blockIdx.x) * experts + e] = sum;
            partial_counts[int64_t(blockIdx.x) * experts + e] = counts[e];
        } else {  // all rows are this CTA's: no second kernel
            const float slope = balance_slope(experts, top_k, live_rows, counts[e]);
            totals.counts[e] = counts[e];
            totals.slope[e] = slope;
            total = fmaf(sum, slope, total);
        }
    }
    if (gridDim.x > 1) {
        if (threadIdx.x == 0) partial_live[blockIdx.x] = live_rows;
        return;
    }
    __shared__ float sums[kRouteWarps];
    total = warp_sum(total);
    if (threadIdx.x % 32 == 0) sums[warp] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kRouteWarps; ++w) total += sums[w];
        *totals.balance = total;
    }
}

template <typename T, int kLanes, int kPer>
__global__ __launch_bounds__(kRouteWarps * 32, 2) void route_backward_kernel(
    RouteShape shape, const T *__restrict__ logits, const int64_t *__restrict__ ids, const float *__restrict__ weights,
    const float *__restrict__ grad_weights, const float *__restrict__ grad_balance, const float *__restrict__ slope,
    T *__restrict__ grad_logits) {
    constexpr int kGroups = kRouteWarps * 32 / kLanes;
    const int at = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    const int experts = static_cast<int>(shape.experts), top_k = static_cast<int>(shape.top_k);
    const float db = grad_balance != nullptr ? *grad_balance : 0.0f;
    float base[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) base[j] = at + j * kLanes < experts ? db * slope[at + j * kLanes] : 0.0f;
    for (int64_t first = int64_t(blockIdx.x) * kGroups; first < shape.tokens; first += int64_t(gridDim.x) * kGroups) {
        const int64_t t = first + group;
        const int64_t *chosen = ids + t * top_k;
        const bool live = t < shape.tokens && chosen[0] >= 0;
        float logit[kPer], e[kPer];
        const RowSoftmax soft = load_row<T, kLanes, kPer>(logits + t * shape.experts, experts, at, live, logit, e);
        const float inverse = 1.0f / soft.sum;
        float dp[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            e[j] *= inverse;
            dp[j] = base[j];
        }
        if (live && grad_weights != nullptr) {
            const float *gw = grad_weights + t * top_k;
            float mean = 0.0f, scale = 1.0f;
            if (shape.renormalize) {
                // a weight is its probability over their sum; the largest weight's probability gives the sum
                for (int k = 0; k < top_k; ++k) mean = fmaf(gw[k], weights[t * top_k + k], mean);
                scale = weights[t * top_k] / (exp_from(to_acc(logits[t * shape.experts + chosen[0]]), soft.max) * inverse);
            }
            for (int k = 0; k < top_k; ++k) {
                const int id = static_cast<int>(chosen[k]);
                const float g = (gw[k] - mean) * scale;
#pragma unroll
                for (int j = 0; j < kPer; ++j) dp[j] += id == at + j * kLanes ? g : 0.0f;
            }
        }
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < kPer; ++j) dot += at + j * kLanes < experts ? e[j] * dp[j] : 0.0f;
        dot = group_sum<kLanes>(dot);
        if (t < shape.tokens) {
            T *out = grad_logits + t * shape.experts;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                if (at + j * kLanes < experts) out[at + j * kLanes] = from_acc<T>(live ? e[j] * (dp[j] - dot) : 0.0f);
            }
        }
    }
}

// ------------------------------------------------------------ wider rows

template <typename T>
__global__ void route_backward_wide_kernel(RouteShape shape, const T *__restrict__ logits, const int64_t *__restrict__ ids,
                                      const float *__restrict__ weights, const float *__restrict__ grad_weights,
                                      const float *__restrict__ grad_balance, const float *__restrict__ slope,
                                      T *__restrict__ grad_logits) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float db = grad_balance != nullptr ? *grad_balance : 0.0f;
    for (int64_t t = int64_t(blockIdx.x) * kWideWarps + warp; t < shape.tokens; t += int64_t(gridDim.x) * kWideWarps) {
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

// Rows a CTA takes in one turn: a warp each, or a group of lanes each.
int rows_per_turn(int64_t experts) {
    return experts <= 32 ? kRouteWarps * 4 : experts <= 64 ? kRouteWarps * 2 : experts <= 256 ? kRouteWarps : kWideWarps;
}
// Up to kSoloTurns turns one CTA takes all rows, and finishes: a launch less. A
// turn takes 1.5 us, as much as the second launch; 8 turns (256 tokens of 64
// experts) were faster for a host that launches one call after the other, 16.4
// for 18.9 us, and slower on the device, 14.6 for 7.0 us, which counts in a graph.
constexpr int64_t kSoloTurns = 2;
int64_t route_blocks(int64_t tokens, int64_t experts) {
    const int64_t blocks = ceil_div(tokens, rows_per_turn(experts));
    if (experts <= 256 && blocks <= kSoloTurns) return 1;
    return blocks < kRouteBlocks ? (blocks > 0 ? blocks : 1) : kRouteBlocks;
}

// Calls go(lanes, per) with the register layout of `experts`, or returns false.
template <typename F>
bool with_layout(int64_t experts, F &&go) {
    if (experts <= 32) return go(std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{}), true;
    if (experts <= 64) return go(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{}), true;
    if (experts <= 128) return go(std::integral_constant<int, 32>{}, std::integral_constant<int, 4>{}), true;
    if (experts <= 256) return go(std::integral_constant<int, 32>{}, std::integral_constant<int, 8>{}), true;
    return false;
}

int check_route(const RouteShape &shape) {
    if (shape.tokens < 0 || shape.tokens > (int64_t(1) << 31)) return fail(KOEMI_ERR_INVALID, "tokens must be in [0, 2^31]");
    if (shape.experts < 1 || shape.experts > kMostExperts) return fail(KOEMI_ERR_INVALID, "expert_count must be in [1, 4096]");
    if (shape.top_k < 1 || shape.top_k > shape.experts || shape.top_k > 256) {
        return fail(KOEMI_ERR_INVALID, "top_k must be in [1, min(expert_count, 256)]");
    }
    return KOEMI_OK;
}

template <typename T>
int route_forward(const RouteShape &shape, const void *logits, int64_t *ids, float *weights, int64_t *counts,
                  float *balance, float *slope, void *workspace, cudaStream_t stream) {
    const int64_t blocks = route_blocks(shape.tokens, shape.experts);
    float *mass = static_cast<float *>(workspace);
    int32_t *partial_counts = reinterpret_cast<int32_t *>(mass + blocks * shape.experts);
    int32_t *live = partial_counts + blocks * shape.experts;
    const T *in = static_cast<const T *>(logits);
    const unsigned grid = static_cast<unsigned>(blocks);
    const bool narrow = with_layout(shape.experts, [&](auto lanes, auto per) {
        route_forward_kernel<T, lanes.value, per.value><<<grid, kRouteWarps * 32, 0, stream>>>(
            shape, in, ids, weights, mass, partial_counts, live, RouteTotals{counts, balance, slope});
    });
    if (!narrow) {
        const size_t per_expert = (kWideWarps + 1) * sizeof(float), smem = per_expert * shape.experts;
        auto kernel = route_forward_wide_kernel<T>;
        // the most that any call wants, not this one's: another thread's launch may stand between the two calls
        KOEMI_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(per_expert * kMostExperts)));
        kernel<<<grid, kWideWarps * 32, smem, stream>>>(shape, in, ids, weights, mass, partial_counts, live);
    }
    KOEMI_LAUNCH_CHECK();
    if (narrow && blocks == 1) return KOEMI_OK;
    route_finish_kernel<<<1, kFinishThreads, 0, stream>>>(mass, partial_counts, live, static_cast<int>(blocks),
                                                          static_cast<int>(shape.experts), shape.top_k, counts, balance,
                                                          slope);
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

template <typename T>
int route_backward(const RouteShape &shape, const void *logits, const int64_t *ids, const float *weights,
                   const float *grad_weights, const float *grad_balance, const float *slope, void *grad_logits,
                   cudaStream_t stream) {
    const T *in = static_cast<const T *>(logits);
    T *out = static_cast<T *>(grad_logits);
    // enough CTAs for a turn each, up to two per SM
    const int64_t turns = ceil_div(shape.tokens, rows_per_turn(shape.experts));
    const unsigned grid = static_cast<unsigned>(turns < kRouteBlocks ? turns : kRouteBlocks);
    const bool narrow = with_layout(shape.experts, [&](auto lanes, auto per) {
        route_backward_kernel<T, lanes.value, per.value><<<grid, kRouteWarps * 32, 0, stream>>>(
            shape, in, ids, weights, grad_weights, grad_balance, slope, out);
    });
    if (!narrow) {
        route_backward_wide_kernel<T><<<grid, kWideWarps * 32, 0, stream>>>(shape, in, ids, weights, grad_weights,
                                                                             grad_balance, slope, out);
    }
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

}  // namespace
}  // namespace koemi

using namespace koemi;

extern "C" size_t koemi_moe_route_learned_workspace(int64_t tokens, int64_t expert_count) {
    if (tokens < 0 || expert_count < 1) return 0;
    const int64_t blocks = route_blocks(tokens, expert_count);
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
