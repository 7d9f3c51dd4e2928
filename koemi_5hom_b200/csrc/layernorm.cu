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
//
// Measured, forward and backward: 32768 x 2048 bf16 51 and 90 us (0.81 and 0.69 of
// the copy rate), 2048 x 16384 fp32 48 and 84 (0.86 and 0.75), 10007 x 1021 fp16,
// whose rows no 16-byte load fits, 25 and 41.
#include <algorithm>

#include "vec.cuh"

namespace koemi {
namespace {

struct NormRows {
    const void *x;
    int64_t rows, inner;  // row r starts at (r / inner) * outer_stride + (r % inner) * inner_stride elements
    int64_t outer_stride, inner_stride;
    int width;
    int lanes;  // of a warp that share a row, where no CTA does (a power of two)
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

// A thread's packets of a row; p: the row, or NULL behind the last. The next
// row is asked for as soon as this one's values are taken. (Rings of three and
// four rows in shared memory by cp.async were slower: 32768 x 2048 bf16 67 for
// 64 us forward, 115 for 95 backward.)
template <typename T, bool kVec, int K>
struct RowPackets {
    Packet<T, kVec> packets[K];
    __device__ __forceinline__ void request(const T *p, int team, int t, int width) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * team + t) * Packet<T, kVec>::kWide;
            if (p != nullptr && c < width) {
                packets[k].load(p + c);
            } else {
                packets[k].zero();
            }
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

// Pairs of fp32 values (vec.cuh): these kernels are bound by issue slots before
// they are bound by bytes.
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// A thread's K packets of W elements as pairs.
template <int W, int N>
__device__ __forceinline__ void to_pairs(const float (&in)[W], int k, float2 (&out)[N]) {
#pragma unroll
    for (int e = 0; e < W; ++e) {
        const int i = k * W + e;
        if (i % 2 == 0) out[i / 2].x = in[e]; else out[i / 2].y = in[e];
    }
}
template <int W, int N>
__device__ __forceinline__ void from_pairs(const float2 (&in)[N], int k, float (&out)[W]) {
#pragma unroll
    for (int e = 0; e < W; ++e) {
        const int i = k * W + e;
        out[e] = i % 2 == 0 ? in[i / 2].x : in[i / 2].y;
    }
}

struct Moments {
    float mean, square;  // square: the sum of squared distances from the mean
};

// The sum over lanes that differ in the bits below `span` (a power of two).
__device__ __forceinline__ float span_sum(float v, int span) {
    for (int offset = span >> 1; offset > 0; offset >>= 1) v += __shfl_xor_sync(0xffffffffu, v, offset);
    return v;
}

// Mean and rsqrt(variance + eps) from one (mean, square) a warp; counts[w]
// is the number of elements that warp w holds, zero behind the last up to `span`.
__device__ __forceinline__ void join(const Moments *parts, const float *counts, int warps, int span, float inv_width, float eps,
                                     float &mean, float &inverse) {
    const int w = threadIdx.x & (span - 1);
    const float n = counts[w];
    const Moments part = w < warps ? parts[w] : Moments{0.0f, 0.0f};
    mean = span_sum(n * part.mean, span) * inv_width;
    const float gap = part.mean - mean;
    inverse = rsqrtf(span_sum(fmaf(n * gap, gap, part.square), span) * inv_width + eps);
}

// Two sums over a warp for little more than one: the halves of the warp take
// one each. a's is in lanes 0 to 15, b's in the others.
__device__ __forceinline__ float half_sums(float a, float b) {
    const bool upper = threadIdx.x & 16;
    float mine = upper ? b : a;
    mine += __shfl_xor_sync(0xffffffffu, upper ? a : b, 16);
    return span_sum(mine, 16);
}

__host__ __device__ __forceinline__ int span_of(int warps) {
    int span = 1;
    while (span < warps) span *= 2;
    return span;
}

// kWarp: 8 warps a CTA, a row for every `lanes` lanes; else a CTA a row. K packets a thread.
template <typename T, bool kVec, int K, bool kWarp>
__global__ __launch_bounds__(kWarp ? 256 : 512) void norm_forward_kernel(const NormRows a, const void *__restrict__ weight,
                                                                                             const void *__restrict__ bias, bool wide,
                                                                                             T *__restrict__ y, float *__restrict__ stats, float eps) {
    using P = Packet<T, kVec>;
    constexpr int W = P::kWide;
    __shared__ Moments parts[kWarp ? 1 : 2][32];
    __shared__ float counts[32];
    const int team = kWarp ? a.lanes : blockDim.x;
    const int t = kWarp ? threadIdx.x & (team - 1) : threadIdx.x;
    const int warps = blockDim.x / 32, teams = kWarp ? blockDim.x / team : 1;
    const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
    // the team's row, and that of its warp's first team: a warp's lanes leave the loop together
    int64_t row = static_cast<int64_t>(blockIdx.x) * teams + (kWarp ? threadIdx.x / team : 0);
    int64_t lead = static_cast<int64_t>(blockIdx.x) * teams + (kWarp ? (threadIdx.x & ~31) / team : 0);
    RowPackets<T, kVec, K> next;
    auto request = [&](int64_t at) {
        next.request(at < a.rows ? static_cast<const T *>(a.x) + row_start(a, at) : nullptr, team, t, a.width);
    };
    request(row);
    constexpr bool kHeld = K * W <= (kVec ? 16 : 8);  // the weights' columns stay in registers, too
    constexpr int N = K * W / 2;
    float2 w[kHeld ? N : 1], b[kHeld ? N : 1];
    float count = static_cast<float>(a.width);
    auto weights_of = [&](int c, float (&wk)[W], float (&bk)[W]) {
#pragma unroll
        for (int e = 0; e < W; ++e) wk[e] = bk[e] = 0.0f;
        if (c < a.width) {
            load_weights<T>(weight, wide, c, wk);
            if (bias != nullptr) load_weights<T>(bias, wide, c, bk);
        }
    };
    if constexpr (kHeld) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float wk[W], bk[W];
            weights_of((k * team + t) * W, wk, bk);
            to_pairs(wk, k, w);
            to_pairs(bk, k, b);
        }
    }
    if constexpr (!kWarp) {
        int held = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) held += (k * team + t) * W < a.width ? W : 0;
        count = warp_sum(static_cast<float>(held));
        if (t < 32) counts[t] = 0.0f;
        __syncthreads();
        if ((t & 31) == 0) counts[t >> 5] = count;
    }
    const int span = span_of(warps);
    const float inv_count = 1.0f / fmaxf(count, 1.0f), inv_width = 1.0f / static_cast<float>(a.width);
    for (int round = 0; lead < a.rows; lead += step, row += step, round ^= 1) {
        float2 v[N], sum = both(0.0f), square = both(0.0f);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float x[W];
            next.packets[k].values(x);
            to_pairs(x, k, v);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) sum = add2(sum, v[i]);
        if (lead + step < a.rows) request(row + step);
        float mean = (kWarp ? span_sum(sum.x + sum.y, team) : warp_sum(sum.x + sum.y)) * inv_count;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float2 gap = add2(v[i], both(-mean));
            if (((2 * i / W) * team + t) * W >= a.width) gap.x = 0.0f;
            if (((2 * i + 1) / W * team + t) * W >= a.width) gap.y = 0.0f;
            square = fma2(gap, gap, square);
        }
        float inverse = kWarp ? span_sum(square.x + square.y, team) : warp_sum(square.x + square.y);
        if constexpr (kWarp) {
            inverse = rsqrtf(inverse * inv_width + eps);
        } else {
            // the other round's slots are free: all have passed this round's barrier only after reading them
            if ((t & 31) == 0) parts[round][t >> 5] = Moments{mean, inverse};
            __syncthreads();
            join(parts[round], counts, warps, span, inv_width, eps, mean, inverse);
        }
        if (kWarp && row >= a.rows) continue;
        if (stats != nullptr && t == 0) {
            stats[row] = mean;
            stats[a.rows + row] = inverse;
        }
        T *out = y + row * a.width;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = mul2(add2(v[i], both(-mean)), both(inverse));
        if constexpr (kHeld) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = fma2(v[i], w[i], b[i]);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * team + t) * W;
            if (c >= a.width) continue;
            float o[W];
            from_pairs(v, k, o);
            if constexpr (!kHeld) {
                float wk[W], bk[W];
                weights_of(c, wk, bk);
#pragma unroll
                for (int e = 0; e < W; ++e) o[e] = fmaf(o[e], wk[e], bk[e]);
            }
            P::store(out + c, o);
        }
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
__global__ __launch_bounds__(kWarp ? 256 : 512) void norm_backward_kernel(const NormRows a, const void *__restrict__ weight, bool wide,
                                                                          const float *__restrict__ stats, const T *__restrict__ g,
                                                                          T *__restrict__ dx, float *__restrict__ partials) {
    using P = Packet<T, kVec>;
    constexpr int W = P::kWide;
    extern __shared__ float pool[];  // kWarp: [2][width]
    __shared__ float slots[kWarp ? 1 : 2][32];  // a round's first sums, then its second
    const int team = kWarp ? a.lanes : blockDim.x;
    const int t = kWarp ? threadIdx.x & (team - 1) : threadIdx.x;
    const int warps = blockDim.x / 32, teams = kWarp ? blockDim.x / team : 1;
    const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
    int64_t row = static_cast<int64_t>(blockIdx.x) * teams + (kWarp ? threadIdx.x / team : 0);
    int64_t lead = static_cast<int64_t>(blockIdx.x) * teams + (kWarp ? (threadIdx.x & ~31) / team : 0);
    const float inv_width = 1.0f / static_cast<float>(a.width);
    const int span = span_of(warps);
    pdl_trigger();

    RowPackets<T, kVec, K> next_x, next_g;
    float next_mean = 0.0f, next_inverse = 0.0f;
    auto request = [&](int64_t at) {
        const bool live = at < a.rows;
        next_x.request(live ? static_cast<const T *>(a.x) + row_start(a, at) : nullptr, team, t, a.width);
        next_g.request(live ? g + at * a.width : nullptr, team, t, a.width);
        next_mean = live ? stats[at] : 0.0f;
        next_inverse = live ? stats[a.rows + at] : 0.0f;
    };
    request(row);
    constexpr int N = K * W / 2;
    float2 w[N], dw[N], db[N];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * team + t) * W;
        float wk[W];
#pragma unroll
        for (int e = 0; e < W; ++e) wk[e] = 0.0f;
        if (c < a.width) load_weights<T>(weight, wide, c, wk);
        to_pairs(wk, k, w);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) dw[i] = db[i] = both(0.0f);
    for (int round = 0; lead < a.rows; lead += step, row += step, round ^= 1) {
        float2 u[N], q[N], firsts = both(0.0f), seconds = both(0.0f);
        const float mean = next_mean, inverse = next_inverse;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float x[W], y[W];
            next_x.packets[k].values(x);
            next_g.packets[k].values(y);
            to_pairs(x, k, u);
            to_pairs(y, k, q);
        }
        // columns and rows behind the last have g = 0 and w = 0: whatever finite u is there, nothing of it counts
#pragma unroll
        for (int i = 0; i < N; ++i) {
            u[i] = mul2(add2(u[i], both(-mean)), both(inverse));
            dw[i] = fma2(q[i], u[i], dw[i]);
            db[i] = add2(db[i], q[i]);
            q[i] = mul2(q[i], w[i]);
            firsts = add2(firsts, q[i]);
            seconds = fma2(q[i], u[i], seconds);
        }
        // A large constant row's mean over sqrt(eps) is infinite, and 0 times it NaN: the sum over its own columns only.
        // (Their mean taken as 0 in every row cost rows by element 96 bytes of spills.)
        if (isinf(mean * inverse)) {
            seconds = both(0.0f);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (((2 * i / W) * team + t) * W < a.width) seconds.x = fmaf(q[i].x, u[i].x, seconds.x);
                if (((2 * i + 1) / W * team + t) * W < a.width) seconds.y = fmaf(q[i].y, u[i].y, seconds.y);
            }
        }
        float first = firsts.x + firsts.y, second = seconds.x + seconds.y;
        if (lead + step < a.rows) request(row + step);
        if (dx == nullptr) continue;
        if (kWarp && team < 32) {
            first = span_sum(first, team);
            second = span_sum(second, team);
        } else {
            float sums = half_sums(first, second);
            if constexpr (!kWarp) {
                // the slots of the other round are free: all have passed this
                // round's barrier only after reading them
                if ((t & 15) == 0) slots[round][(t & 16) + (t >> 5)] = sums;
                __syncthreads();
                const int w = t & (span - 1);  // at most 16 warps
                sums = span_sum(w < warps ? slots[round][(t & 16) + w] : 0.0f, span);
            }
            first = __shfl_sync(0xffffffffu, sums, 0);
            second = __shfl_sync(0xffffffffu, sums, 16);
        }
        if (kWarp && row >= a.rows) continue;
        first *= inv_width;
        second *= inv_width;
        T *out = dx + row * a.width;
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = mul2(both(inverse), fma2(u[i], both(-second), add2(q[i], both(-first))));
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * team + t) * W;
            if (c >= a.width) continue;
            float o[W];
            from_pairs(q, k, o);
            P::store(out + c, o);
        }
    }
    if (partials == nullptr) return;
    float *mine = partials + static_cast<int64_t>(blockIdx.x) * 2 * a.width;
    float *const to = kWarp ? pool : mine;
    if (kWarp) {  // the teams of a warp first
        for (int offset = team; offset < 32; offset <<= 1) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                dw[i].x += __shfl_xor_sync(0xffffffffu, dw[i].x, offset);
                dw[i].y += __shfl_xor_sync(0xffffffffu, dw[i].y, offset);
                db[i].x += __shfl_xor_sync(0xffffffffu, db[i].x, offset);
                db[i].y += __shfl_xor_sync(0xffffffffu, db[i].y, offset);
            }
        }
    }
    for (int turn = 0; turn < (kWarp ? warps : 1); ++turn) {  // then the CTA's warps, in order
        if (!kWarp || (turn == static_cast<int>(threadIdx.x / 32) && (threadIdx.x & 31) < team)) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = (k * team + t) * W;
                if (c >= a.width) continue;
                float one[W], other[W];
                from_pairs(dw, k, one);
                from_pairs(db, k, other);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    to[c + e] = turn == 0 ? one[e] : to[c + e] + one[e];
                    to[a.width + c + e] = turn == 0 ? other[e] : to[a.width + c + e] + other[e];
                }
            }
        }
        if (kWarp) __syncthreads();
    }
    if constexpr (kWarp) {
        for (int i = threadIdx.x; i < 2 * a.width; i += blockDim.x) mine[i] = pool[i];
    }
}

// Wide rows: 1024 threads, one CTA an SM, dw and db of all columns in its
// shared memory (a register each would be 64 a thread). A row is asked into L2
// while the one before it is worked on.
template <typename T, int K>
__global__ __launch_bounds__(1024) void norm_backward_wide_kernel(const NormRows a, const void *__restrict__ weight, bool wide,
                                                                  const float *__restrict__ stats, const T *__restrict__ g,
                                                                  T *__restrict__ dx, float *__restrict__ partials) {
    constexpr int W = Pack<T>::kWidth;
    extern __shared__ float4 sums[];  // [dw | db][width / 4]
    __shared__ float2 slots[2][32];
    pdl_trigger();
    const int t = threadIdx.x, quads = a.width / 4;
    const float inv_width = 1.0f / static_cast<float>(a.width);
    if (partials != nullptr) {
        for (int i = t; i < 2 * quads; i += 1024) sums[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        __syncthreads();
    }
    for (int64_t row = blockIdx.x, round = 0; row < a.rows; row += gridDim.x, round ^= 1) {
        const T *x = static_cast<const T *>(a.x) + row_start(a, row), *gr = g + row * a.width;
        const float mean = stats[row], inverse = stats[a.rows + row];
        uint4 px[K], pg[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * 1024 + t) * W;
            px[k] = pg[k] = make_uint4(0, 0, 0, 0);
            if (c < a.width) px[k] = load_stream(x + c), pg[k] = load_stream(gr + c);
        }
        if (row + gridDim.x < a.rows) {
            const T *nx = static_cast<const T *>(a.x) + row_start(a, row + gridDim.x), *ng = gr + static_cast<int64_t>(gridDim.x) * a.width;
            constexpr int kLine = 128 / sizeof(T);
            for (int c = t * kLine; c < a.width; c += 1024 * kLine) {
                asm volatile("prefetch.global.L2 [%0];" ::"l"(nx + c));
                asm volatile("prefetch.global.L2 [%0];" ::"l"(ng + c));
            }
        }
        float first = 0.0f, second = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * 1024 + t) * W;
            if (c >= a.width) continue;
            float u[W], q[W], w[W];
            unpack(px[k], u, T());
            unpack(pg[k], q, T());
            load_weights<T>(weight, wide, c, w);
#pragma unroll
            for (int e = 0; e < W; ++e) u[e] = (u[e] - mean) * inverse;
            if (partials != nullptr) {
#pragma unroll
                for (int e = 0; e < W; e += 4) {
                    float4 dw = sums[(c + e) / 4], db = sums[quads + (c + e) / 4];
                    dw.x = fmaf(q[e], u[e], dw.x), dw.y = fmaf(q[e + 1], u[e + 1], dw.y);
                    dw.z = fmaf(q[e + 2], u[e + 2], dw.z), dw.w = fmaf(q[e + 3], u[e + 3], dw.w);
                    db.x += q[e], db.y += q[e + 1], db.z += q[e + 2], db.w += q[e + 3];
                    sums[(c + e) / 4] = dw;
                    sums[quads + (c + e) / 4] = db;
                }
            }
#pragma unroll
            for (int e = 0; e < W; ++e) {
                first = fmaf(q[e], w[e], first);
                second = fmaf(q[e] * w[e], u[e], second);
            }
        }
        if (dx == nullptr) continue;
        first = warp_sum(first);
        second = warp_sum(second);
        if ((t & 31) == 0) slots[round][t >> 5] = make_float2(first, second);
        __syncthreads();
        const float2 part = slots[round][t & 31];
        first = warp_sum(part.x) * inv_width;
        second = warp_sum(part.y) * inv_width;
        T *out = dx + row * a.width;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * 1024 + t) * W;
            if (c >= a.width) continue;
            float u[W], q[W], w[W];
            unpack(px[k], u, T());
            unpack(pg[k], q, T());
            load_weights<T>(weight, wide, c, w);
#pragma unroll
            for (int e = 0; e < W; ++e) q[e] = inverse * (q[e] * w[e] - first - (u[e] - mean) * inverse * second);
            store_stream(out + c, pack(q, T()));
        }
    }
    if (partials == nullptr) return;
    __syncthreads();
    float4 *mine = reinterpret_cast<float4 *>(partials + static_cast<int64_t>(blockIdx.x) * 2 * a.width);
    for (int i = t; i < 2 * quads; i += 1024) mine[i] = sums[i];
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
__global__ __launch_bounds__(32 * kFinishWarps) void norm_finish_kernel(const float *partials, int64_t rows, int width,
                                                                         void *dw, void *db, int dtype) {
    __shared__ float parts[kFinishWarps][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    void *out = blockIdx.y == 0 ? dw : db;
    if (out == nullptr) return;
    pdl_wait();
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

constexpr int kTeamThreads = 256;  // a CTA of the kernels whose rows are shared by lanes
constexpr int kMostPartials = 1024;  // partial rows of dw and db
constexpr size_t kMostShared = 224 * 1024;

// CTAs of a backward launch, each of which leaves a partial row. A thread holds at most 16 columns in 64 registers and
// more, so an SM holds no more than 1024 threads' worth of rows.
int64_t most_partials(int64_t rows, int64_t width) {
    return std::min<int64_t>({rows, kMostPartials, sm_count() * std::max<int64_t>(1, 16 * 1024 / width)});
}

// How a row is held: packets of `wide` elements, `per_thread` of them a thread.
struct Plan {
    bool warp, fits;
    int threads, per_thread, lanes;
    int64_t teams_of(int64_t rows) const { return warp ? ceil_div(rows, kTeamThreads / lanes) : rows; }  // CTAs of one row a team
};

// Many rows are bound by instructions, of which a row's sums are a warp's worth
// whatever it holds, so they get few threads with many elements each: `good`
// packets a thread, up to 32 lanes a row and else CTAs, and more only where 512 threads need
// them (32768 x 2048 bf16 forward: 52 us with two packets and their weights in
// registers, 64 with one, 66 with two and the weights from L1, 68 with eight in
// a warp; 524288 x 128: 88 with a warp a row). Few rows are bound by latency and get a packet a thread.
Plan plan_of(bool vector, int wide, int64_t rows, int64_t width, int warp_good, int good, int most) {
    Plan plan{false, true, 0, 0, 32};
    const int64_t packets = ceil_div(width, wide);
    const bool few = vector && rows < 8 * sm_count();
    if (!vector && packets <= 128) warp_good = 4;
    if (few) warp_good = good = 1;
    if (packets <= 32 * warp_good) {
        plan.warp = true;
        plan.threads = kTeamThreads;
        plan.per_thread = warp_good;
        plan.lanes = span_of(static_cast<int>(ceil_div(packets, warp_good)));
        return plan;
    }
    int per = good;
    while (per < most && ceil_div(packets, per) > 512) per *= 2;
    const int64_t threads = ceil_div(ceil_div(packets, per), 32) * 32;
    plan.fits = threads <= 512;
    plan.threads = static_cast<int>(std::min<int64_t>(threads, 512));
    plan.per_thread = per;
    return plan;
}

template <typename T>
bool rows_fit_vectors(const NormRows &a) {
    const int64_t wide = Pack<T>::kWidth;
    return aligned(a.x, 16) && a.width % wide == 0 && a.inner_stride % wide == 0 && (a.inner >= a.rows || a.outer_stride % wide == 0);
}

// CTAs of `kernel` that the GPU holds at once.
template <typename Kernel>
int64_t resident_of(Kernel kernel, int threads, size_t shared) {
    int per_sm = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, shared) != cudaSuccess) cudaGetLastError();
    return static_cast<int64_t>(sm_count()) * std::max(per_sm, 1);
}

template <typename T, bool kVec, int K, bool kWarp>
int launch_forward(const Plan &plan, NormRows a, const void *weight, const void *bias, bool wide, void *y, float *stats,
                   float eps, cudaStream_t stream) {
    auto kernel = norm_forward_kernel<T, kVec, K, kWarp>;
    a.lanes = plan.lanes;
    const int64_t teams = plan.teams_of(a.rows);
    const int64_t grid = std::min(teams, resident_of(kernel, plan.threads, 0));
    kernel<<<static_cast<unsigned>(grid), plan.threads, 0, stream>>>(a, weight, bias, wide, static_cast<T *>(y), stats, eps);
    return KOEMI_OK;
}

template <typename T, bool kVec, int K>
int forward_of(const Plan &plan, const NormRows &a, const void *weight, const void *bias, bool wide, void *y, float *stats, float eps,
               cudaStream_t stream) {
    return plan.warp ? launch_forward<T, kVec, K, true>(plan, a, weight, bias, wide, y, stats, eps, stream)
                     : launch_forward<T, kVec, K, false>(plan, a, weight, bias, wide, y, stats, eps, stream);
}

template <typename T>
int forward(const NormRows &a, const void *weight, const void *bias, bool wide, void *y, float *stats, float eps, cudaStream_t stream) {
    const bool vector = rows_fit_vectors<T>(a) && aligned(y, 16) && aligned(weight, 16) && aligned(bias, 16);
    constexpr int kGood = 16 / Pack<T>::kWidth;  // with their weights: 48 registers
    const Plan plan = plan_of(vector, vector ? Pack<T>::kWidth : 1, a.rows, a.width, vector ? kGood : 16, vector ? kGood : 16, vector ? 8 : 16);
    int rc = KOEMI_OK;
    if (!plan.fits) {
        norm_forward_long_kernel<T><<<static_cast<unsigned>(a.rows), 1024, 0, stream>>>(a, weight, bias, wide, static_cast<T *>(y), stats, eps);
    } else if (vector) {
        if (plan.per_thread <= 1) rc = forward_of<T, true, 1>(plan, a, weight, bias, wide, y, stats, eps, stream);
        else if (plan.per_thread <= 2) rc = forward_of<T, true, 2>(plan, a, weight, bias, wide, y, stats, eps, stream);
        else if (plan.per_thread <= 4) rc = forward_of<T, true, 4>(plan, a, weight, bias, wide, y, stats, eps, stream);
        else rc = launch_forward<T, true, 8, false>(plan, a, weight, bias, wide, y, stats, eps, stream);
    } else {
        if (plan.per_thread <= 4) rc = forward_of<T, false, 4>(plan, a, weight, bias, wide, y, stats, eps, stream);
        else rc = forward_of<T, false, 16>(plan, a, weight, bias, wide, y, stats, eps, stream);
    }
    if (rc != KOEMI_OK) return rc;
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

template <typename T, bool kVec, int K, bool kWarp>
int launch_backward(const Plan &plan, NormRows a, const void *weight, bool wide, const float *stats, const void *g, void *dx,
                    float *partials, int64_t *grid, cudaStream_t stream) {
    auto kernel = norm_backward_kernel<T, kVec, K, kWarp>;
    a.lanes = plan.lanes;
    const size_t shared = kWarp ? sizeof(float) * 2 * a.width : 0;
    const int64_t teams = plan.teams_of(a.rows);
    *grid = std::min<int64_t>({teams, resident_of(kernel, plan.threads, shared), most_partials(a.rows, a.width)});
    kernel<<<static_cast<unsigned>(*grid), plan.threads, shared, stream>>>(a, weight, wide, stats, static_cast<const T *>(g),
                                                                           static_cast<T *>(dx), partials);
    return KOEMI_OK;
}

// *grid: the number of partial rows.
template <typename T, bool kVec, int K>
int backward_of(const Plan &plan, const NormRows &a, const void *weight, bool wide, const float *stats, const void *g, void *dx,
                float *partials, int64_t *grid, cudaStream_t stream) {
    return plan.warp ? launch_backward<T, kVec, K, true>(plan, a, weight, wide, stats, g, dx, partials, grid, stream)
                     : launch_backward<T, kVec, K, false>(plan, a, weight, wide, stats, g, dx, partials, grid, stream);
}

template <typename T, int K>
int backward_wide(const NormRows &a, const void *weight, bool wide, const float *stats, const void *g, void *dx, float *partials,
                  int64_t *grid, cudaStream_t stream) {
    auto kernel = norm_backward_wide_kernel<T, K>;
    KOEMI_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostShared)));
    *grid = std::min<int64_t>(sm_count(), most_partials(a.rows, a.width));
    kernel<<<static_cast<unsigned>(*grid), 1024, partials != nullptr ? sizeof(float) * 2 * a.width : 0, stream>>>(
        a, weight, wide, stats, static_cast<const T *>(g), static_cast<T *>(dx), partials);
    return KOEMI_OK;
}

template <typename T>
int backward(const NormRows &a, const void *weight, bool wide, const float *stats, const void *g, void *dx, void *dw, void *db,
             float *partials, cudaStream_t stream) {
    const bool vector = rows_fit_vectors<T>(a) && aligned(g, 16) && aligned(dx, 16) && aligned(weight, 16);
    constexpr int kMost = 16 / Pack<T>::kWidth;  // 16 elements a thread: dw and db take a register each for every one
    const Plan plan = plan_of(vector, vector ? Pack<T>::kWidth : 1, a.rows, a.width, vector ? 2 : 16, vector ? kMost : 16, vector ? kMost : 16);
    if (dw == nullptr && db == nullptr) partials = nullptr;
    int64_t grid = 0;
    int rc = KOEMI_OK;
    const int64_t packets = ceil_div(a.width, Pack<T>::kWidth);
    if (!plan.fits && vector && packets <= 4096 && sizeof(float) * 2 * a.width <= kMostShared) {
        rc = packets <= 2048 ? backward_wide<T, 2>(a, weight, wide, stats, g, dx, partials, &grid, stream)
                             : backward_wide<T, 4>(a, weight, wide, stats, g, dx, partials, &grid, stream);
    } else if (!plan.fits) {
        if (dx != nullptr) {
            norm_backward_long_kernel<T><<<static_cast<unsigned>(a.rows), 1024, 0, stream>>>(a, weight, wide, stats, static_cast<const T *>(g), static_cast<T *>(dx));
        }
        if (partials != nullptr) {
            const int64_t columns = ceil_div(a.width, 256);
            grid = std::min<int64_t>(std::max<int64_t>(1, 8 * sm_count() / columns), most_partials(a.rows, a.width));
            norm_columns_kernel<T><<<dim3(static_cast<unsigned>(columns), static_cast<unsigned>(grid)), 256, 0, stream>>>(
                a, stats, static_cast<const T *>(g), partials);
        }
    } else if (vector) {
        if (plan.per_thread <= 1) rc = backward_of<T, true, 1>(plan, a, weight, wide, stats, g, dx, partials, &grid, stream);
        else if (plan.per_thread <= 2) rc = backward_of<T, true, 2>(plan, a, weight, wide, stats, g, dx, partials, &grid, stream);
        else if constexpr (sizeof(T) == 4) rc = backward_of<T, true, 4>(plan, a, weight, wide, stats, g, dx, partials, &grid, stream);
    } else {
        if (plan.per_thread <= 4) rc = backward_of<T, false, 4>(plan, a, weight, wide, stats, g, dx, partials, &grid, stream);
        else rc = backward_of<T, false, 16>(plan, a, weight, wide, stats, g, dx, partials, &grid, stream);
    }
    if (rc != KOEMI_OK) return rc;
    KOEMI_LAUNCH_CHECK();
    if (partials != nullptr) {
        const int dtype = wide ? KOEMI_F32 : sizeof(T) == 4 ? KOEMI_F32 : std::is_same<T, __half>::value ? KOEMI_F16 : KOEMI_BF16;
        KOEMI_CUDA_TRY(launch_programmatic(true, norm_finish_kernel, dim3(static_cast<unsigned>(ceil_div(a.width, 32)), 2), dim3(32 * kFinishWarps), 0,
                                           stream, dim3(1, 1, 1), partials, grid, a.width, dw, db, dtype));
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

int misaligned() { return fail(KOEMI_ERR_INVALID, "layer norm's pointers must be aligned to their types"); }

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
    if (!aligned(out, dtype_size(dtype)) || !aligned({weight, bias}, dtype_size(weight_dtype)) || !aligned(stats, 4)) return misaligned();
    const NormRows a{values, rows, inner_rows, outer_stride, inner_stride, static_cast<int>(width), 32};
    const bool wide = weight_dtype == KOEMI_F32;
    if (dtype == KOEMI_F32) return forward<float>(a, weight, bias, wide, out, stats, eps, as_stream(stream));
    if (dtype == KOEMI_F16) return forward<__half>(a, weight, bias, wide, out, stats, eps, as_stream(stream));
    return forward<__nv_bfloat16>(a, weight, bias, wide, out, stats, eps, as_stream(stream));
}

extern "C" size_t koemi_core_layer_norm_backward_workspace(int64_t rows, int64_t width) {
    if (rows < 1 || width < 1) return 0;
    return static_cast<size_t>(most_partials(rows, width)) * 2 * width * sizeof(float);
}

extern "C" int koemi_core_layer_norm_backward(const void *values, int64_t rows, int64_t width, int64_t inner_rows, int64_t outer_stride,
                                              int64_t inner_stride, const void *weight, int weight_dtype, const float *stats,
                                              const void *grad_out, void *grad_values, void *grad_weight, void *grad_bias, int dtype,
                                              void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    const int rc = check(values, rows, width, inner_rows, outer_stride, inner_stride, dtype, weight_dtype);
    if (rc != KOEMI_OK) return rc;
    const bool sums = grad_weight != nullptr || grad_bias != nullptr;
    if (!aligned({grad_out, grad_values}, dtype_size(dtype)) || !aligned({weight, grad_weight, grad_bias}, dtype_size(weight_dtype)) ||
        !aligned(stats, 4)) {
        return misaligned();
    }
    if (rows == 0) {  // the sum of no rows
        const size_t bytes = dtype_size(weight_dtype) * static_cast<size_t>(width);
        if (grad_weight != nullptr) KOEMI_CUDA_TRY(cudaMemsetAsync(grad_weight, 0, bytes, as_stream(stream)));
        if (grad_bias != nullptr) KOEMI_CUDA_TRY(cudaMemsetAsync(grad_bias, 0, bytes, as_stream(stream)));
        return KOEMI_OK;
    }
    if (values == nullptr || weight == nullptr || stats == nullptr || grad_out == nullptr) {
        return fail(KOEMI_ERR_INVALID, "values, weight, stats and grad_out must be non-NULL");
    }
    if (sums && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < koemi_core_layer_norm_backward_workspace(rows, width))) {
        return fail(KOEMI_ERR_WORKSPACE, "layer norm backward needs %zu workspace bytes from a multiple of 16",
                    koemi_core_layer_norm_backward_workspace(rows, width));
    }
    const NormRows a{values, rows, inner_rows, outer_stride, inner_stride, static_cast<int>(width), 32};
    const bool wide = weight_dtype == KOEMI_F32;
    float *partials = static_cast<float *>(workspace);
    if (dtype == KOEMI_F32) return backward<float>(a, weight, wide, stats, grad_out, grad_values, grad_weight, grad_bias, partials, as_stream(stream));
    if (dtype == KOEMI_F16) return backward<__half>(a, weight, wide, stats, grad_out, grad_values, grad_weight, grad_bias, partials, as_stream(stream));
    return backward<__nv_bfloat16>(a, weight, wide, stats, grad_out, grad_values, grad_weight, grad_bias, partials, as_stream(stream));
}
