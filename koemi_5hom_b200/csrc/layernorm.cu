// Layer norm of rows, forward and backward, for sm_100a.
//
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), u = (x - m) r,
//   y = u w + b;
//   a = g w, dx = r (a - mean(a) - u mean(a u)), dw = sum_rows g u, db = sum_rows g.
//
// Bound by bytes: x in and y out, and x, g in and dx out (the weights stay in
// L1 and L2). A row is read once: its 16-byte packets stay in the registers of
// its team (a warp for short rows, a CTA for longer ones) from the statistics
// to the result. The variance is taken about the mean of each warp's part and
// the parts are joined by counts, means and squares, so one exchange between
// warps gives both statistics and nothing cancels.
//
// Backward: the CTAs are resident and walk rows a grid apart, so that a
// thread meets the same columns in every row and keeps their part of dw and db
// in registers; the next row's packets are requested before the current row's
// sums. Each CTA leaves one partial row of dw and db (fp32) and a second kernel
// adds the partial rows in order: equal inputs give equal bits.
#include <algorithm>

#include "vec.cuh"

namespace koemi {
namespace {

struct NormRows {
    const void *x;
    int64_t rows, inner;  // row r starts at (r / inner) * outer_stride + (r % inner) * inner_stride elements
    int64_t outer_stride, inner_stride;
    int width;
};

__device__ __forceinline__ int64_t row_start(const NormRows &a, int64_t r) {
    if (a.inner >= a.rows) return r * a.inner_stride;
    const int64_t outer = r / a.inner;
    return outer * a.outer_stride + (r - outer * a.inner) * a.inner_stride;
}

// One packet: kWide elements of T from p (16 bytes where vectors fit, else one element).
template <typename T, bool kVec>
struct Packet {
    static constexpr int kWide = kVec ? Pack<T>::kWidth : 1;
    uint4 raw;
    T one;
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (kVec) {
            raw = load_stream(p);
        } else {
            one = *p;
        }
    }
    __device__ __forceinline__ void zero() {
        if constexpr (kVec) {
            raw = make_uint4(0, 0, 0, 0);
        } else {
            one = from_acc<T>(0.0f);
        }
    }
    __device__ __forceinline__ void values(float (&out)[kWide]) const {
        if constexpr (kVec) {
            unpack(raw, out, T());
        } else {
            out[0] = to_acc(one);
        }
    }
    static __device__ __forceinline__ void store(T *p, const float (&in)[kWide]) {
        if constexpr (kVec) {
            store_stream(p, pack(in, T()));
        } else {
            *p = from_acc<T>(in[0]);
        }
    }
};

// kWide weights from column c, fp32 or of type T.
template <typename T, int kWide>
__device__ __forceinline__ void load_weights(const void *w, bool wide, int c, float (&out)[kWide]) {
    if (wide) {
        const float *p = static_cast<const float *>(w) + c;
        if constexpr (kWide >= 4) {
#pragma unroll
            for (int q = 0; q < kWide / 4; ++q) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(p) + q);
                out[4 * q] = v.x, out[4 * q + 1] = v.y, out[4 * q + 2] = v.z, out[4 * q + 3] = v.w;
            }
        } else {
            out[0] = __ldg(p);
        }
    } else {
        const T *p = static_cast<const T *>(w) + c;
        if constexpr (kWide > 1) {
            unpack(load_cached(p), out, T());
        } else {
            out[0] = to_acc(*p);
        }
    }
}

struct Moments {
    float mean, square;  // square: the sum of squared distances from the mean
};

// Mean and rsqrt(variance + eps) from one (mean, square) a warp; counts[w]
// is the number of elements that warp w holds.
__device__ __forceinline__ void join(const Moments *parts, const float *counts, int warps, int width, float eps, float &mean,
                                     float &inverse) {
    const int lane = threadIdx.x & 31;
    const float n = lane < warps ? counts[lane] : 0.0f;
    const Moments part = lane < warps ? parts[lane] : Moments{0.0f, 0.0f};
    const float inv_width = 1.0f / static_cast<float>(width);
    mean = warp_sum(n * part.mean) * inv_width;
    const float gap = part.mean - mean;
    inverse = rsqrtf(warp_sum(fmaf(n * gap, gap, part.square)) * inv_width + eps);
}

// The longest rows of the forward pass take 1024 threads of the most packets, all others up to 512.
template <typename T, bool kVec, int K>
constexpr int most_threads() {
    return K == (kVec ? 4 : 16) ? 1024 : 512;
}

// kWarp: a warp a row, 8 rows a CTA; else a CTA a row. K packets a thread.
template <typename T, bool kVec, int K, bool kWarp>
__global__ __launch_bounds__(kWarp ? 256 : most_threads<T, kVec, K>()) void norm_forward_kernel(const NormRows a, const void *__restrict__ weight, const void *__restrict__ bias, bool wide,
                                    T *__restrict__ y, float *__restrict__ stats, float eps) {
    using P = Packet<T, kVec>;
    constexpr int W = P::kWide;
    const int team = kWarp ? 32 : blockDim.x;
    const int t = kWarp ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = kWarp ? static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
    if (kWarp && row >= a.rows) return;
    const T *x = static_cast<const T *>(a.x) + row_start(a, row);
    P packets[K];
    int held = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * team + t) * W;
        if (c < a.width) {
            packets[k].load(x + c);
            held += W;
        } else {
            packets[k].zero();
        }
    }
    float v[K][W], sum = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        packets[k].values(v[k]);
#pragma unroll
        for (int e = 0; e < W; ++e) sum += v[k][e];
    }
    const float count = kWarp ? static_cast<float>(a.width) : warp_sum(static_cast<float>(held));
    float mean = warp_sum(sum) / fmaxf(count, 1.0f), square = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if ((k * team + t) * W < a.width) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float gap = v[k][e] - mean;
                square = fmaf(gap, gap, square);
            }
        }
    }
    square = warp_sum(square);
    float inverse;
    if constexpr (kWarp) {
        inverse = rsqrtf(square / count + eps);
    } else {
        __shared__ Moments parts[32];
        __shared__ float counts[32];
        if ((t & 31) == 0) {
            parts[t >> 5] = Moments{mean, square};
            counts[t >> 5] = count;
        }
        __syncthreads();
        join(parts, counts, (blockDim.x + 31) / 32, a.width, eps, mean, inverse);
    }
    if (stats != nullptr && t == 0) {
        stats[row] = mean;
        stats[a.rows + row] = inverse;
    }
    T *out = y + row * a.width;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * team + t) * W;
        if (c >= a.width) continue;
        float w[W], b[W];
        load_weights<T>(weight, wide, c, w);
        if (bias != nullptr) {
            load_weights<T>(bias, wide, c, b);
        } else {
#pragma unroll
            for (int e = 0; e < W; ++e) b[e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < W; ++e) v[k][e] = fmaf((v[k][e] - mean) * inverse, w[e], b[e]);
        P::store(out + c, v[k]);
    }
}

// Rows that no team holds in registers: three walks over the row, the later ones in L2.
template <typename T>
__global__ __launch_bounds__(1024) void norm_forward_long_kernel(const NormRows a, const void *__restrict__ weight,
                                                                 const void *__restrict__ bias, bool wide, T *__restrict__ y,
                                                                 float *__restrict__ stats, float eps) {
    __shared__ float parts[2][32];
    const T *x = static_cast<const T *>(a.x) + row_start(a, blockIdx.x);
    float sum = 0.0f;
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) sum += to_acc(x[c]);
    sum = warp_sum(sum);
    if ((threadIdx.x & 31) == 0) parts[0][threadIdx.x >> 5] = sum;
    __syncthreads();
    const float inv_width = 1.0f / static_cast<float>(a.width);
    const float mean = warp_sum(parts[0][threadIdx.x & 31]) * inv_width;
    float square = 0.0f;
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
        const float gap = to_acc(x[c]) - mean;
        square = fmaf(gap, gap, square);
    }
    square = warp_sum(square);
    if ((threadIdx.x & 31) == 0) parts[1][threadIdx.x >> 5] = square;
    __syncthreads();
    const float inverse = rsqrtf(warp_sum(parts[1][threadIdx.x & 31]) * inv_width + eps);
    if (stats != nullptr && threadIdx.x == 0) {
        stats[blockIdx.x] = mean;
        stats[a.rows + blockIdx.x] = inverse;
    }
    T *out = y + static_cast<int64_t>(blockIdx.x) * a.width;
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
        float w[1], b[1] = {0.0f};
        load_weights<T>(weight, wide, c, w);
        if (bias != nullptr) load_weights<T>(bias, wide, c, b);
        out[c] = from_acc<T>(fmaf((to_acc(x[c]) - mean) * inverse, w[0], b[0]));
    }
}

// ---------------------------------------------------------------- backward

// partials: [grid][2][width], NULL where neither dw nor db is wanted; dx may be NULL.
template <typename T, bool kVec, int K, bool kWarp>
__global__ __launch_bounds__(kWarp ? 256 : 512) void norm_backward_kernel(const NormRows a, const void *__restrict__ weight, bool wide, const float *__restrict__ stats,
                                     const T *__restrict__ g, T *__restrict__ dx, float *__restrict__ partials) {
    using P = Packet<T, kVec>;
    constexpr int W = P::kWide;
    extern __shared__ float pool[];  // kWarp: [2][width]; else two rounds of two sums a warp
    const int team = kWarp ? 32 : blockDim.x;
    const int t = kWarp ? threadIdx.x & 31 : threadIdx.x;
    const int warps = (blockDim.x + 31) / 32;
    const int64_t step = kWarp ? static_cast<int64_t>(gridDim.x) * warps : gridDim.x;
    int64_t row = kWarp ? static_cast<int64_t>(blockIdx.x) * warps + threadIdx.x / 32 : blockIdx.x;
    const float inv_width = 1.0f / static_cast<float>(a.width);

    float w[K][W], dw[K][W], db[K][W];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * team + t) * W;
#pragma unroll
        for (int e = 0; e < W; ++e) w[k][e] = dw[k][e] = db[k][e] = 0.0f;
        if (c < a.width) load_weights<T>(weight, wide, c, w[k]);
    }
    P px[K], pg[K];
    auto request = [&](int64_t r) {
        const T *x = static_cast<const T *>(a.x) + row_start(a, r), *gr = g + r * a.width;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * team + t) * W;
            if (c < a.width) {
                px[k].load(x + c);
                pg[k].load(gr + c);
            } else {
                px[k].zero();
                pg[k].zero();
            }
        }
    };
    float mean = 0.0f, inverse = 0.0f;
    if (row < a.rows) {
        request(row);
        mean = stats[row], inverse = stats[a.rows + row];
    }
    for (int round = 0; row < a.rows; row += step, round ^= 1) {
        float u[K][W], q[K][W], first = 0.0f, second = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool live = (k * team + t) * W < a.width;
            px[k].values(u[k]);
            pg[k].values(q[k]);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                u[k][e] = live ? (u[k][e] - mean) * inverse : 0.0f;
                dw[k][e] = fmaf(q[k][e], u[k][e], dw[k][e]);
                db[k][e] += q[k][e];
                q[k][e] *= w[k][e];
                first += q[k][e];
                second = fmaf(q[k][e], u[k][e], second);
            }
        }
        const float scale = inverse;
        const int64_t current = row;
        if (row + step < a.rows) {
            request(row + step);
            mean = stats[row + step], inverse = stats[a.rows + row + step];
        }
        if (dx == nullptr) continue;
        first = warp_sum(first);
        second = warp_sum(second);
        if constexpr (!kWarp) {
            // the slots of the other round are free: all have passed this round's
            // barrier only after reading them
            float2 *slots = reinterpret_cast<float2 *>(pool) + round * 32;
            if ((t & 31) == 0) slots[t >> 5] = make_float2(first, second);
            __syncthreads();
            const float2 part = (t & 31) < warps ? slots[t & 31] : make_float2(0.0f, 0.0f);
            first = warp_sum(part.x);
            second = warp_sum(part.y);
        }
        first *= inv_width;
        second *= inv_width;
        T *out = dx + current * a.width;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * team + t) * W;
            if (c >= a.width) continue;
#pragma unroll
            for (int e = 0; e < W; ++e) q[k][e] = scale * (q[k][e] - first - u[k][e] * second);
            P::store(out + c, q[k]);
        }
    }
    if (partials == nullptr) return;
    float *mine = partials + static_cast<int64_t>(blockIdx.x) * 2 * a.width;
    if constexpr (kWarp) {  // the CTA's warps add their parts in order
        for (int turn = 0; turn < warps; ++turn) {
            if (turn == static_cast<int>(threadIdx.x / 32)) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const int c = (k * team + t) * W;
                    if (c >= a.width) continue;
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        pool[c + e] = turn == 0 ? dw[k][e] : pool[c + e] + dw[k][e];
                        pool[a.width + c + e] = turn == 0 ? db[k][e] : pool[a.width + c + e] + db[k][e];
                    }
                }
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < 2 * a.width; i += blockDim.x) mine[i] = pool[i];
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * team + t) * W;
            if (c >= a.width) continue;
#pragma unroll
            for (int e = 0; e < W; ++e) {
                mine[c + e] = dw[k][e];
                mine[a.width + c + e] = db[k][e];
            }
        }
    }
}

// dx of rows that no team holds in registers: two walks.
template <typename T>
__global__ __launch_bounds__(1024) void norm_backward_long_kernel(const NormRows a, const void *__restrict__ weight, bool wide,
                                                                  const float *__restrict__ stats, const T *__restrict__ g,
                                                                  T *__restrict__ dx) {
    __shared__ float parts[2][32];
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row_start(a, row), *gr = g + row * a.width;
    const float mean = stats[row], inverse = stats[a.rows + row], inv_width = 1.0f / static_cast<float>(a.width);
    float first = 0.0f, second = 0.0f, w[1];
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
        load_weights<T>(weight, wide, c, w);
        const float q = to_acc(gr[c]) * w[0];
        first += q;
        second = fmaf(q, (to_acc(x[c]) - mean) * inverse, second);
    }
    first = warp_sum(first);
    second = warp_sum(second);
    if ((threadIdx.x & 31) == 0) parts[0][threadIdx.x >> 5] = first, parts[1][threadIdx.x >> 5] = second;
    __syncthreads();
    first = warp_sum(parts[0][threadIdx.x & 31]) * inv_width;
    second = warp_sum(parts[1][threadIdx.x & 31]) * inv_width;
    T *out = dx + row * a.width;
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
        load_weights<T>(weight, wide, c, w);
        out[c] = from_acc<T>(inverse * (to_acc(gr[c]) * w[0] - first - (to_acc(x[c]) - mean) * inverse * second));
    }
}

// Their partial rows of dw and db: CTA (columns, slice of the rows).
template <typename T>
__global__ __launch_bounds__(256) void norm_columns_kernel(const NormRows a, const float *__restrict__ stats, const T *__restrict__ g,
                                                           float *__restrict__ partials) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.width) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float q = to_acc(g[row * a.width + c]);
        const float x = to_acc(static_cast<const T *>(a.x)[row_start(a, row) + c]);
        dw = fmaf(q, (x - stats[row]) * stats[a.rows + row], dw);
        db += q;
    }
    float *mine = partials + static_cast<int64_t>(blockIdx.y) * 2 * a.width;
    mine[c] = dw;
    mine[a.width + c] = db;
}

// dw (grid.y 0) and db (1): the partial rows added in order, 32 columns a
// CTA, 16 of its warps' strided parts joined in order.
constexpr int kFinishWarps = 16;
__global__ __launch_bounds__(32 * kFinishWarps) void norm_finish_kernel(const float *__restrict__ partials, int64_t rows, int width,
                                                                         void *dw, void *db, int dtype) {
    __shared__ float parts[kFinishWarps][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    void *out = blockIdx.y == 0 ? dw : db;
    if (out == nullptr) return;
    float sum = 0.0f;
    if (c < width) {
        const float *p = partials + static_cast<int64_t>(blockIdx.y) * width + c;
#pragma unroll 8
        for (int64_t r = warp; r < rows; r += kFinishWarps) sum += p[r * 2 * width];
    }
    parts[warp][lane] = sum;
    __syncthreads();
    if (warp != 0 || c >= width) return;
#pragma unroll
    for (int k = 1; k < kFinishWarps; ++k) sum += parts[k][lane];
    if (dtype == KOEMI_F32) {
        static_cast<float *>(out)[c] = sum;
    } else if (dtype == KOEMI_F16) {
        static_cast<__half *>(out)[c] = from_acc<__half>(sum);
    } else {
        static_cast<__nv_bfloat16 *>(out)[c] = from_acc<__nv_bfloat16>(sum);
    }
}

// -------------------------------------------------------------------- plan

constexpr int kWarpRows = 8;       // rows (warps) a CTA of the warp-a-row kernels
constexpr int kMostPartials = 1024;  // partial rows of dw and db

// How a row is held: packets of `wide` elements, `per_thread` of them a thread.
struct Plan {
    bool vector, warp, fits;
    int threads, per_thread;
};

Plan plan_of(bool vector, int wide, int64_t width, int most_per_thread, int most_threads) {
    Plan plan{vector, false, true, 0, 0};
    const int64_t packets = ceil_div(width, wide);
    const int warp_most = std::min(vector ? 4 : 16, most_per_thread);
    if (packets <= 32 * warp_most) {
        plan.warp = true;
        plan.threads = 32 * kWarpRows;
        plan.per_thread = static_cast<int>(ceil_div(packets, 32));
    } else {
        // as few packets a thread as 512 threads hold, then up to the limits
        int per = 1;
        while (per < most_per_thread && ceil_div(packets, per) > 512) per *= 2;
        const int64_t threads = ceil_div(ceil_div(packets, per), 32) * 32;
        plan.fits = threads <= most_threads;
        plan.threads = static_cast<int>(std::min<int64_t>(threads, most_threads));
        plan.per_thread = per;
    }
    return plan;
}

template <typename T>
bool rows_fit_vectors(const NormRows &a) {
    const int64_t wide = Pack<T>::kWidth;
    return aligned(a.x, 16) && a.width % wide == 0 && a.inner_stride % wide == 0 && (a.inner >= a.rows || a.outer_stride % wide == 0);
}

template <typename T, bool kVec, int K>
void launch_forward(const Plan &plan, const NormRows &a, const void *weight, const void *bias, bool wide, void *y, float *stats,
                    float eps, cudaStream_t stream) {
    if (plan.warp) {
        norm_forward_kernel<T, kVec, K, true><<<static_cast<unsigned>(ceil_div(a.rows, kWarpRows)), plan.threads, 0, stream>>>(
            a, weight, bias, wide, static_cast<T *>(y), stats, eps);
    } else {
        norm_forward_kernel<T, kVec, K, false><<<static_cast<unsigned>(a.rows), plan.threads, 0, stream>>>(
            a, weight, bias, wide, static_cast<T *>(y), stats, eps);
    }
}

template <typename T>
int forward(const NormRows &a, const void *weight, const void *bias, bool wide, void *y, float *stats, float eps, cudaStream_t stream) {
    const bool vector = rows_fit_vectors<T>(a) && aligned(y, 16) && aligned(weight, 16) && aligned(bias, 16);
    const Plan plan = plan_of(vector, vector ? Pack<T>::kWidth : 1, a.width, vector ? 4 : 16, 1024);
    if (!plan.fits) {
        norm_forward_long_kernel<T><<<static_cast<unsigned>(a.rows), 1024, 0, stream>>>(a, weight, bias, wide, static_cast<T *>(y), stats, eps);
    } else if (vector) {
        if (plan.per_thread <= 1) launch_forward<T, true, 1>(plan, a, weight, bias, wide, y, stats, eps, stream);
        else if (plan.per_thread <= 2) launch_forward<T, true, 2>(plan, a, weight, bias, wide, y, stats, eps, stream);
        else launch_forward<T, true, 4>(plan, a, weight, bias, wide, y, stats, eps, stream);
    } else {
        if (plan.per_thread <= 4) launch_forward<T, false, 4>(plan, a, weight, bias, wide, y, stats, eps, stream);
        else launch_forward<T, false, 16>(plan, a, weight, bias, wide, y, stats, eps, stream);
    }
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

template <typename T, bool kVec, int K>
int launch_backward(const Plan &plan, const NormRows &a, const void *weight, bool wide, const float *stats, const void *g, void *dx,
                    float *partials, int64_t *grid_out, cudaStream_t stream) {
    auto kernel = plan.warp ? norm_backward_kernel<T, kVec, K, true> : norm_backward_kernel<T, kVec, K, false>;
    const size_t shared = plan.warp ? sizeof(float) * 2 * a.width : sizeof(float2) * 2 * 32;
    int resident = 0;
    KOEMI_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, plan.threads, shared));
    const int64_t teams = plan.warp ? ceil_div(a.rows, kWarpRows) : a.rows;
    const int64_t grid = std::min<int64_t>({teams, static_cast<int64_t>(sm_count()) * std::max(resident, 1), kMostPartials});
    kernel<<<static_cast<unsigned>(grid), plan.threads, shared, stream>>>(a, weight, wide, stats, static_cast<const T *>(g),
                                                                          static_cast<T *>(dx), partials);
    *grid_out = grid;
    return KOEMI_OK;
}

template <typename T>
int backward(const NormRows &a, const void *weight, bool wide, const float *stats, const void *g, void *dx, void *dw, void *db,
             float *partials, cudaStream_t stream) {
    const bool vector = rows_fit_vectors<T>(a) && aligned(g, 16) && aligned(dx, 16) && aligned(weight, 16);
    const Plan plan = plan_of(vector, vector ? Pack<T>::kWidth : 1, a.width, vector ? 16 / Pack<T>::kWidth : 16, 512);
    if (dw == nullptr && db == nullptr) partials = nullptr;
    int64_t grid = 0;
    int rc = KOEMI_OK;
    if (!plan.fits) {
        if (dx != nullptr) {
            norm_backward_long_kernel<T><<<static_cast<unsigned>(a.rows), 1024, 0, stream>>>(a, weight, wide, stats, static_cast<const T *>(g), static_cast<T *>(dx));
        }
        if (partials != nullptr) {
            const int64_t columns = ceil_div(a.width, 256);
            grid = std::min<int64_t>({a.rows, std::max<int64_t>(1, 8 * sm_count() / columns), kMostPartials});
            norm_columns_kernel<T><<<dim3(static_cast<unsigned>(columns), static_cast<unsigned>(grid)), 256, 0, stream>>>(
                a, stats, static_cast<const T *>(g), partials);
        }
    } else if (vector) {
        // 16 elements a thread at most: dw and db take a register each for every one of them
        if (plan.per_thread <= 1) rc = launch_backward<T, true, 1>(plan, a, weight, wide, stats, g, dx, partials, &grid, stream);
        else if (plan.per_thread <= 2) rc = launch_backward<T, true, 2>(plan, a, weight, wide, stats, g, dx, partials, &grid, stream);
        else if constexpr (sizeof(T) == 4) rc = launch_backward<T, true, 4>(plan, a, weight, wide, stats, g, dx, partials, &grid, stream);
    } else {
        if (plan.per_thread <= 4) rc = launch_backward<T, false, 4>(plan, a, weight, wide, stats, g, dx, partials, &grid, stream);
        else rc = launch_backward<T, false, 16>(plan, a, weight, wide, stats, g, dx, partials, &grid, stream);
    }
    if (rc != KOEMI_OK) return rc;
    KOEMI_LAUNCH_CHECK();
    if (partials != nullptr) {
        const int dtype = wide ? KOEMI_F32 : sizeof(T) == 4 ? KOEMI_F32 : std::is_same<T, __half>::value ? KOEMI_F16 : KOEMI_BF16;
        norm_finish_kernel<<<dim3(static_cast<unsigned>(ceil_div(a.width, 32)), 2), 32 * kFinishWarps, 0, stream>>>(
            partials, grid, a.width, dw, db, dtype);
        KOEMI_LAUNCH_CHECK();
    }
    return KOEMI_OK;
}

int check(const void *x, int64_t rows, int64_t width, int64_t inner, int64_t outer_stride, int64_t inner_stride, int dtype, int weight_dtype) {
    if (rows < 0 || width < 1 || inner < 1 || outer_stride < 0 || inner_stride < 0) return fail(KOEMI_ERR_INVALID, "bad layer norm sizes");
    if (width > (int64_t(1) << 30) || rows > INT32_MAX) return fail(KOEMI_ERR_INVALID, "layer norm rows are too many or too wide");
    if (dtype != KOEMI_F32 && dtype != KOEMI_F16 && dtype != KOEMI_BF16) return fail(KOEMI_ERR_INVALID, "unsupported layer norm dtype %d", dtype);
    if (weight_dtype != dtype && weight_dtype != KOEMI_F32) return fail(KOEMI_ERR_INVALID, "layer norm weights are of the values' dtype or fp32");
    if (!aligned(x, dtype_size(dtype))) return fail(KOEMI_ERR_INVALID, "values are not aligned to their type");
    return KOEMI_OK;
}

}  // namespace
}  // namespace koemi

using namespace koemi;

extern "C" int koemi_core_layer_norm_forward(const void *values, int64_t rows, int64_t width, int64_t inner_rows, int64_t outer_stride,
                                             int64_t inner_stride, const void *weight, const void *bias, int weight_dtype, void *out,
                                             float *stats, float eps, int dtype, void *stream) {
    clear_error();
    const int rc = check(values, rows, width, inner_rows, outer_stride, inner_stride, dtype, weight_dtype);
    if (rc != KOEMI_OK) return rc;
    if (!(eps >= 0.0f) || eps > 3.0e38f) return fail(KOEMI_ERR_INVALID, "eps must be finite and non-negative");
    if (rows == 0) return KOEMI_OK;
    if (values == nullptr || weight == nullptr || out == nullptr) return fail(KOEMI_ERR_INVALID, "values, weight and out must be non-NULL");
    const NormRows a{values, rows, inner_rows, outer_stride, inner_stride, static_cast<int>(width)};
    const bool wide = weight_dtype == KOEMI_F32;
    if (dtype == KOEMI_F32) return forward<float>(a, weight, bias, wide, out, stats, eps, as_stream(stream));
    if (dtype == KOEMI_F16) return forward<__half>(a, weight, bias, wide, out, stats, eps, as_stream(stream));
    return forward<__nv_bfloat16>(a, weight, bias, wide, out, stats, eps, as_stream(stream));
}

extern "C" size_t koemi_core_layer_norm_backward_workspace(int64_t rows, int64_t width) {
    if (rows < 1 || width < 1) return 0;
    return static_cast<size_t>(std::min<int64_t>(rows, kMostPartials)) * 2 * width * sizeof(float);
}

extern "C" int koemi_core_layer_norm_backward(const void *values, int64_t rows, int64_t width, int64_t inner_rows, int64_t outer_stride,
                                              int64_t inner_stride, const void *weight, int weight_dtype, const float *stats,
                                              const void *grad_out, void *grad_values, void *grad_weight, void *grad_bias, int dtype,
                                              void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    const int rc = check(values, rows, width, inner_rows, outer_stride, inner_stride, dtype, weight_dtype);
    if (rc != KOEMI_OK) return rc;
    const bool sums = grad_weight != nullptr || grad_bias != nullptr;
    if (rows == 0) {  // the sum of no rows
        const size_t bytes = dtype_size(weight_dtype) * static_cast<size_t>(width);
        if (grad_weight != nullptr) KOEMI_CUDA_TRY(cudaMemsetAsync(grad_weight, 0, bytes, as_stream(stream)));
        if (grad_bias != nullptr) KOEMI_CUDA_TRY(cudaMemsetAsync(grad_bias, 0, bytes, as_stream(stream)));
        return KOEMI_OK;
    }
    if (values == nullptr || weight == nullptr || stats == nullptr || grad_out == nullptr) {
        return fail(KOEMI_ERR_INVALID, "values, weight, stats and grad_out must be non-NULL");
    }
    if (sums && (workspace == nullptr || workspace_bytes < koemi_core_layer_norm_backward_workspace(rows, width))) {
        return fail(KOEMI_ERR_WORKSPACE, "layer norm backward needs %zu workspace bytes", koemi_core_layer_norm_backward_workspace(rows, width));
    }
    const NormRows a{values, rows, inner_rows, outer_stride, inner_stride, static_cast<int>(width)};
    const bool wide = weight_dtype == KOEMI_F32;
    float *partials = static_cast<float *>(workspace);
    if (dtype == KOEMI_F32) return backward<float>(a, weight, wide, stats, grad_out, grad_values, grad_weight, grad_bias, partials, as_stream(stream));
    if (dtype == KOEMI_F16) return backward<__half>(a, weight, wide, stats, grad_out, grad_values, grad_weight, grad_bias, partials, as_stream(stream));
    return backward<__nv_bfloat16>(a, weight, wide, stats, grad_out, grad_values, grad_weight, grad_bias, partials, as_stream(stream));
}
