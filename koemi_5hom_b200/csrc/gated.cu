// Dense front: gated linear recurrence from raw projections, forward and
// backward.
//
//   s = sigmoid(p), a = lo + (hi - lo) s, k = tanh(c)
//   h_t = a_t h' + (1 - a_t) k_t,  h' = 0 at a restart, else h_{t-1}
//   (an invalid position keeps the state: h_t = h')
//
// projections are [batch, length, 2 F] (p | c), states [batch, length, F];
// the running state is fp32. The forward can leave the state before every
// 128th position in `carries`, from which the backward recomputes the states
// it needs on chip instead of reading them:
//
//   adj_t = g_t + x_t,  x_{t-1} = a_t adj_t (0 at a restart)
//   dp_t = adj_t (h' - k_t) (hi - lo) s (1 - s)
//   dc_t = adj_t (1 - a_t) (1 - k_t^2),  d_initial = x_{-1}
//
// Every step is an affine map of the state (forward) or of x (backward), so a
// tile of 128 positions x 32 features composes into one map per feature. A
// CTA takes a tile: each half warp holds 8 neighbouring rows in registers, a
// lane two features, and leaves its rows' map in shared memory; one warp, a
// thread per feature, then walks these maps from the carry and leaves each
// half warp the value its rows start from. A chain (one batch row, 32
// features) is walked by a cluster of 1 to 8 CTAs, a wave of as many
// neighbouring tiles at a time: the walking warps store their tiles' maps
// into each other's shared memory and fold the maps of the tiles in front of
// theirs onto the carry. Nothing is exchanged through global memory, no CTA
// waits for one outside its cluster, and the order of every sum is fixed, so
// equal inputs give equal bits.
//
// Every byte is read and written once; the time is the arithmetic's and the
// walk's beside HBM's. Batch x length x features, microseconds forward and
// backward, and the fraction of the device's copy bandwidth:
//   16 x 4096 x 1184 bf16   106, 0.67   168, 0.71   (places of the GPU filled)
//   8 x 4096 x 1024 fp32     69, 0.90   111, 0.92   (half the arithmetic per byte)
//   8 x 4096 x 1024 bf16     63, 0.49    86, 0.60   (256 chains: 3 or 4 CTAs an SM)
//   1 x 32768 x 2048 bf16   125, 0.49   189, 0.54   (64 chains, in clusters of 8 and of 4)
//   256 x 128 x 2048 bf16   108, 0.57   178, 0.58   (one tile a chain)
// In the first case the schedulers issue in about six tenths of their cycles and
// the special-function units are busy for half; the rest is waits at the tile's
// barriers. Tiles of 64 x 64, of four warps with 16 rows each or of 16 with
// four, three or four stages, and three CTAs per SM backward were slower. With
// plain remote stores and cluster barriers, whose release waits for global
// stores, and arithmetic on single floats, 8 x 4096 x 1024 bf16 with masks took
// 177 us forward; it takes 66.
#include "common.cuh"

namespace koemi {
namespace {

constexpr int kSegment = 128;  // positions of a tile, and between two carries
constexpr int kTileFeatures = 32;
constexpr int kWarps = 8;
constexpr int kTileThreads = kWarps * 32;
constexpr int kBlocks = 2 * kWarps;             // half warps of a CTA
constexpr int kRows = kSegment / kBlocks;       // rows of a half warp
constexpr int kMaxCluster = 8;
// CTAs per SM that the kernels are compiled for and the launches planned with:
// forward four of 64 registers in 16 bits, and in fp32 three, which is what 74
// KB of shared memory each let in. fp32 planned with two instead took 45 for 43 us at 64 x 128 x 2048 with
// masks and as long elsewhere; compiled for two, 47 there and 124 for 131 at
// 64 x 1024 x 1024 without masks.
template <typename T>
constexpr int forward_resident() {
    return sizeof(T) == 2 ? 4 : 3;
}
constexpr int kBackwardResident = 2;
constexpr int kShortLength = 16;  // up to here one thread walks a lane

struct GatedShape {
    int64_t batch, length, features, segments;
    float lo, hi;
    const uint8_t *valid, *restart;
};

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float ex2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// s and k of one element. With yp = 1 + e^-p and yc = 1 + e^2c, s = 1 / yp and
// k = 1 - 2 / yc share one reciprocal, of yp yc; the exponents stop at 40,
// where both have reached their limits in fp32, so that the product stays
// finite. Both are good to a few 2^-24 of 1, which near 0 is not good enough
// for k, as small as c there, and would make something of a c of 0. fp32
// inputs take tanh's series up to |c| = 1/4 (good to 2^-24 of k); 16-bit inputs
// below 2^-8 are their own tanh to 2^-17, and above the 2^-24s are 2^-14 of k
// at most, a part of the inputs' own rounding (8 x 4096 x 1024 bf16 173 to 175
// us a pass, 1 x 32768 x 2048 312 to 320).
constexpr float kOwnTanh = 0.00390625f;
template <typename T>
__device__ __forceinline__ void gate_of(float p, float c, float &s, float &k) {
    constexpr float kLog2e = 1.4426950408889634f;
    const float yp = 1.0f + ex2_approx(min_nan(-kLog2e * p, 40.0f * kLog2e));
    const float yc = 1.0f + ex2_approx(min_nan(2.0f * kLog2e * c, 40.0f * kLog2e));
    const float r = rcp_approx(yp * yc);
    s = r * yc;
    k = fmaf(-2.0f, r * yp, 1.0f);
    if constexpr (sizeof(T) == 4) {
        const float z = c * c;
        float series = fmaf(z, 62.0f / 2835.0f, -17.0f / 315.0f);
        series = fmaf(z, series, 2.0f / 15.0f);
        series = fmaf(z, series, -1.0f / 3.0f);
        if (z < 0.0625f) k = fmaf(c * z, series, c);
    } else if (fabsf(c) < kOwnTanh) {
        k = c;
    }
}

// -------------------------------------------------------- short sequences

// One thread walks one (batch, feature) lane. At most kShortLength positions,
// so that a walk costs about as many dependent steps as a tile's; T = 1 is
// the decode step.
template <typename T>
__global__ void gated_forward_lane_kernel(GatedShape shape, const T *__restrict__ projections,
                                          const float *__restrict__ initial, T *__restrict__ states,
                                          float *__restrict__ final_state, float *__restrict__ carries) {
    const int64_t lane = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (lane >= shape.batch * shape.features) return;
    const int64_t b = lane / shape.features, f = lane - b * shape.features;
    float h = initial != nullptr ? initial[lane] : 0.0f;
    if (carries != nullptr) carries[lane] = h;
    for (int64_t t = 0; t < shape.length; ++t) {
        const int64_t row = b * shape.length + t;
        if (shape.restart != nullptr && shape.restart[row]) h = 0.0f;
        if (shape.valid == nullptr || shape.valid[row]) {
            float s, k;
            gate_of<T>(to_acc(projections[row * 2 * shape.features + f]),
                       to_acc(projections[row * 2 * shape.features + shape.features + f]), s, k);
            const float a = fmaf(shape.hi - shape.lo, s, shape.lo);
            h = fmaf(a, h, fmaf(-a, k, k));
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
    const float span = shape.hi - shape.lo;
    float s[kShortLength], k[kShortLength], before[kShortLength];
    uint32_t live = 0, cut = 0;
    float h = carries[lane];
#pragma unroll
    for (int t = 0; t < kShortLength; ++t) {
        if (t >= shape.length) continue;
        const int64_t row = b * shape.length + t;
        if (shape.restart != nullptr && shape.restart[row]) {
            cut |= 1u << t;
            h = 0.0f;
        }
        before[t] = h;
        if (shape.valid == nullptr || shape.valid[row]) {
            live |= 1u << t;
            gate_of<T>(to_acc(projections[row * 2 * shape.features + f]),
                       to_acc(projections[row * 2 * shape.features + shape.features + f]), s[t], k[t]);
            const float a = fmaf(span, s[t], shape.lo);
            h = fmaf(a, h, fmaf(-a, k[t], k[t]));
        }
    }
    float x = grad_final != nullptr ? grad_final[lane] : 0.0f;
#pragma unroll
    for (int t = kShortLength - 1; t >= 0; --t) {
        if (t >= shape.length) continue;
        const int64_t row = b * shape.length + t;
        const float adjoint = x + (grad_states != nullptr ? to_acc(grad_states[row * shape.features + f]) : 0.0f);
        float dp = 0.0f, dc = 0.0f;
        x = adjoint;
        if (live >> t & 1u) {
            // the gate's slope from s: read back from a it would lose digits under narrow bounds, and be 0 / 0 under equal ones
            const float a = fmaf(span, s[t], shape.lo);
            dp = adjoint * (before[t] - k[t]) * (span * s[t] * (1.0f - s[t]));
            dc = adjoint * (1.0f - a) * fmaf(-k[t], k[t], 1.0f);
            x = a * adjoint;
        }
        if (cut >> t & 1u) x = 0.0f;
        grad_projections[row * 2 * shape.features + f] = from_acc<T>(dp);
        grad_projections[row * 2 * shape.features + shape.features + f] = from_acc<T>(dc);
    }
    if (grad_initial != nullptr) grad_initial[lane] = x;
}

// ------------------------------------------------------------------ tiles

// Two features at once: Blackwell's packed fp32 instructions issue once for
// both, and the tile kernels are bound by issue slots next to HBM.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, c, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 r, a, b, c;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 r, a, b;\n\t"
        "mov.b64 {%0, %1}, r;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 r, a, b;\n\t"
        "mov.b64 {%0, %1}, r;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return fma2(b, both(-1.0f), a); }

// s and k of gate_of for two features; p and c are already clamped (p >= -40,
// c <= 20).
template <typename T>
__device__ __forceinline__ void gates_of(float2 p, float2 c, float2 &s, float2 &k) {
    constexpr float kLog2e = 1.4426950408889634f;
    const float2 ep = mul2(p, both(-kLog2e)), ec = mul2(c, both(2.0f * kLog2e));
    const float2 yp = add2(make_float2(ex2_approx(ep.x), ex2_approx(ep.y)), both(1.0f));
    const float2 yc = add2(make_float2(ex2_approx(ec.x), ex2_approx(ec.y)), both(1.0f));
    const float2 product = mul2(yp, yc);
    const float2 r = make_float2(rcp_approx(product.x), rcp_approx(product.y));
    s = mul2(r, yc);
    k = fma2(mul2(r, yp), both(-2.0f), both(1.0f));
    if constexpr (sizeof(T) == 4) {
        const float2 z = mul2(c, c);
        float2 series = fma2(z, both(62.0f / 2835.0f), both(-17.0f / 315.0f));
        series = fma2(z, series, both(2.0f / 15.0f));
        series = fma2(z, series, both(-1.0f / 3.0f));
        series = fma2(mul2(c, z), series, c);
        if (z.x < 0.0625f) k.x = series.x;
        if (z.y < 0.0625f) k.y = series.y;
    } else {
        if (fabsf(c.x) < kOwnTanh) k.x = c.x;
        if (fabsf(c.y) < kOwnTanh) k.y = c.y;
    }
}

// Two features of a projection row in shared memory, clamped from below (p)
// or above (c); a NaN stays.
template <bool kBelow>
__device__ __forceinline__ float2 load_clamped(const __nv_bfloat16 *at) {
    const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162 *>(at);
    return __bfloat1622float2(kBelow ? __hmax2_nan(v, __float2bfloat162_rn(-40.0f)) : __hmin2_nan(v, __float2bfloat162_rn(20.0f)));
}
template <bool kBelow>
__device__ __forceinline__ float2 load_clamped(const __half *at) {
    const __half2 v = *reinterpret_cast<const __half2 *>(at);
    return __half22float2(kBelow ? __hmax2_nan(v, __float2half2_rn(-40.0f)) : __hmin2_nan(v, __float2half2_rn(20.0f)));
}
template <bool kBelow>
__device__ __forceinline__ float2 clamped(float2 v) {
    return kBelow ? make_float2(max_nan(v.x, -40.0f), max_nan(v.y, -40.0f)) : make_float2(min_nan(v.x, 20.0f), min_nan(v.y, 20.0f));
}
template <bool kBelow>
__device__ __forceinline__ float2 load_clamped(const float *at) {
    return clamped<kBelow>(*reinterpret_cast<const float2 *>(at));
}

__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Stores 8 bytes into CTA `rank`'s copy of `local` and counts them on its copy
// of `bar`. Unlike a plain remote store and a barrier it needs no release,
// which would wait for the warp's global stores.
__device__ __forceinline__ void store_to_rank(float2 *local, uint64_t *bar, int rank, float2 v) {
    asm volatile(
        "{\n\t.reg .b32 a, b;\n\tmapa.shared::cluster.u32 a, %0, %2;\n\tmapa.shared::cluster.u32 b, %1, %2;\n\t"
        "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [a], {%3, %4}, [b];\n\t}" ::"r"(smem_addr(local)),
        "r"(smem_addr(bar)), "r"(rank), "f"(v.x), "f"(v.y)
        : "memory");
}

template <typename T>
struct GatedMapType;
template <>
struct GatedMapType<__nv_bfloat16> {
    static constexpr CUtensorMapDataType value = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
};
template <>
struct GatedMapType<__half> {
    static constexpr CUtensorMapDataType value = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
};
template <>
struct GatedMapType<float> {
    static constexpr CUtensorMapDataType value = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
};

__device__ __forceinline__ float2 load_two(const __nv_bfloat16 *p) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(p));
}
__device__ __forceinline__ float2 load_two(const __half *p) {
    return __half22float2(*reinterpret_cast<const __half2 *>(p));
}
__device__ __forceinline__ float2 load_two(const float *p) { return *reinterpret_cast<const float2 *>(p); }
__device__ __forceinline__ void store_two(__nv_bfloat16 *p, float2 v) {
    *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(v.x, v.y);
}
__device__ __forceinline__ void store_two(__half *p, float2 v) {
    *reinterpret_cast<__half2 *>(p) = __floats2half2_rn(v.x, v.y);
}
__device__ __forceinline__ void store_two(float *p, float2 v) { *reinterpret_cast<float2 *>(p) = v; }

// Where a lane's two features are; lanes 16 to 31 hold the same features of
// other rows. TMA tiles: features 2 l and 2 l + 1 (one 4- or 8-byte access;
// the width is a multiple of 4 features at least). Without TMA: l and l + 16,
// single elements, so that accesses stay contiguous at any alignment.
template <bool kTma>
struct LaneFeatures {
    int64_t x;
    bool x_in, y_in;
    __device__ LaneFeatures(int64_t first, int lane, int64_t features) {
        x = first + (kTma ? 2 * (lane & 15) : lane & 15);
        x_in = x < features;
        y_in = x + (kTma ? 1 : 16) < features;
    }
    // `row` points at feature x of a row
    template <typename T>
    __device__ __forceinline__ float2 load(const T *row) const {
        return make_float2(x_in ? to_acc(row[0]) : 0.0f, y_in ? to_acc(row[kTma ? 1 : 16]) : 0.0f);
    }
    template <typename T>
    __device__ __forceinline__ void store(T *row, float2 v) const {
        if (kTma) {
            if (x_in) store_two(row, v);
        } else {
            if (x_in) row[0] = from_acc<T>(v.x);
            if (y_in) row[16] = from_acc<T>(v.y);
        }
    }
};

// The tile feature at place i of a row of the shared maps (places 2 l and 2 l + 1
// are lane l's).
template <bool kTma>
__device__ __forceinline__ int walked_feature(int i) {
    return kTma ? i : (i >> 1) + 16 * (i & 1);
}

// Which of a half warp's rows are inside the sequence, which of those are
// valid, and which restart (bits); plain: all of the warp's rows are ordinary.
struct RowFlags {
    uint32_t live, cut;
    int rows_in;
    bool plain;
};
template <bool kMasks>
__device__ __forceinline__ RowFlags row_flags(const GatedShape &shape, int64_t batch, int segment, int warp, int lane) {
    constexpr uint32_t kAll = (1u << kRows) - 1;
    RowFlags f;
    const int t0 = segment * kSegment + warp * 2 * kRows, half = lane >> 4;
    const int left = static_cast<int>(shape.length) - t0;
    const int mine = left - half * kRows;
    f.rows_in = mine >= kRows ? kRows : mine > 0 ? mine : 0;
    if (kMasks) {
        const bool in = lane < 2 * kRows && lane < left;
        const int64_t row = batch * shape.length + t0 + lane;
        const uint32_t live = __ballot_sync(0xffffffffu, in && (shape.valid == nullptr || shape.valid[row] != 0));
        const uint32_t cut = __ballot_sync(0xffffffffu, in && shape.restart != nullptr && shape.restart[row] != 0);
        f.plain = live == (kAll << kRows | kAll) && cut == 0;
        f.live = live >> half * kRows & kAll;
        f.cut = cut >> half * kRows & kAll;
    } else {
        f.plain = left >= 2 * kRows;
        f.live = (1u << f.rows_in) - 1;
        f.cut = 0;
    }
    return f;
}

constexpr float kSmallest = 1.4e-45f;  // keeps a product of positive factors positive: 0 would undo an infinity

// A map v -> m v + n. A restart among its rows makes n the result, whatever v
// holds (a NaN, say): m is then 0, and only there.
template <bool kMasks>
__device__ __forceinline__ float apply(float m, float n, float v) {
    const float r = fmaf(m, v, n);
    return kMasks && m == 0.0f ? n : r;
}
// m of a map put in front of one with m of `next`
template <bool kMasks>
__device__ __forceinline__ float chain(float m, float next) {
    return kMasks && (m == 0.0f || next == 0.0f) ? 0.0f : fmaxf(m * next, kSmallest);
}

constexpr int kLoader = kTileThreads - 32;  // the thread that issues the loads: not in the walking warp
template <typename T>
constexpr int backward_stages() {
    return sizeof(T) == 2 ? 3 : 2;
}

// The chains of a cluster: `count` neighbouring ones from `first` on, each
// `waves` waves long; item i of a CTA is wave i % waves of chain first + i /
// waves.
struct Walk {
    int64_t first, feature_tiles;
    int count, waves, cluster, rank;
    __device__ Walk(const GatedShape &shape, int64_t tiles, int cluster_, int per) : feature_tiles(tiles), cluster(cluster_) {
        rank = static_cast<int>(blockIdx.x % cluster);
        first = int64_t(blockIdx.x / cluster) * per;
        const int64_t left = shape.batch * feature_tiles - first;
        count = left < per ? static_cast<int>(left) : per;
        waves = (static_cast<int>(shape.segments) + cluster - 1) / cluster;
    }
    __device__ __forceinline__ int64_t batch(int chain) const { return (first + chain) / feature_tiles; }
    __device__ __forceinline__ int64_t feature(int chain) const { return (first + chain) % feature_tiles * kTileFeatures; }
};

// Shared memory of a tile kernel: kStages stages of kArrays boxes; per half
// warp and feature the rows' map (kMaps values) and the start values
// (kStarts); the cluster's maps of two waves; the barriers.
template <typename T, int kArrays, int kStages, int kMaps, int kStarts>
struct TileMemory {
    static constexpr int kBox = kSegment * kTileFeatures;
    static constexpr uint32_t kStageBytes = kArrays * kBox * sizeof(T);
    static constexpr int kPlane = kBlocks * kTileFeatures;
    T *stages;
    uint64_t *full;  // [kStages]
    uint64_t *met;   // [2]
    int *issued;     // items whose loads are on their way or done: the loading thread's
    float *maps;     // [kMaps][kBlocks][32]
    float *starts;   // [kStarts][kBlocks][32]
    float2 *tiles;   // [2][CTAs of the cluster][32]
    __device__ explicit TileMemory(unsigned char *raw) {
        stages = reinterpret_cast<T *>(raw);
        full = reinterpret_cast<uint64_t *>(raw + size_t(kStages) * kStageBytes);
        met = full + 4;
        issued = reinterpret_cast<int *>(met + 2);
        maps = reinterpret_cast<float *>(met + 4);
        starts = maps + kMaps * kPlane;
        tiles = reinterpret_cast<float2 *>(starts + kStarts * kPlane);
    }
    static size_t bytes(int cluster_size) {
        return size_t(kStages) * kStageBytes + 64 + (kMaps + kStarts) * kPlane * sizeof(float) +
               (cluster_size > 1 ? 2 * size_t(cluster_size) * kTileFeatures * sizeof(float2) : 0);
    }
};

// The map of a whole tile, by the walking warp (a thread per feature), in row
// order or from the last row.
template <bool kMasks, bool kBackward>
__device__ __forceinline__ float2 tile_map_of(const float *mm, const float *nn) {
    float tm = 1.0f, tn = 0.0f;
#pragma unroll 8
    for (int i = 0; i < kBlocks; ++i) {
        const int block = kBackward ? kBlocks - 1 - i : i;
        const float m = mm[block * kTileFeatures], n = nn[block * kTileFeatures];
        tm = chain<kMasks>(tm, m);
        tn = apply<kMasks>(m, n, tn);
    }
    return make_float2(tm, tn);
}

// The walking warp of a cluster's CTA gives its tile's map to every CTA, waits
// for everyone's and folds them onto `carry` in tile order (or from the last
// tile). Returns the value its own tile starts from. The maps of two items
// have places of their own: a CTA has received every map of item i + 1 only
// when all have left item i.
template <bool kMasks, bool kBackward, typename Memory>
__device__ __forceinline__ float meet(Memory &memory, int item, int cluster, int rank, float2 mine, float &carry,
                                      bool &dead, int *status) {
    const int lane = threadIdx.x, parity = item & 1;
    uint64_t *bar = &memory.met[parity];
    float2 *tiles = memory.tiles + parity * cluster * kTileFeatures + lane;
    if (dead) return carry;  // nor sends any more: the others give up too
    if (lane == 0) mbar_arrive_expect_tx(bar, cluster * kTileFeatures * sizeof(float2));
    for (int r = 0; r < cluster; ++r) store_to_rank(tiles + rank * kTileFeatures, bar, r, mine);
    dead = !mbar_wait_bounded<true>(bar, static_cast<uint32_t>(item >> 1) & 1, status);
    float start = carry;
    for (int i = 0; i < cluster; ++i) {
        const int r = kBackward ? cluster - 1 - i : i;
        if (r == rank) start = carry;
        const float2 v = tiles[r * kTileFeatures];
        carry = apply<kMasks>(v.x, v.y, carry);
    }
    return start;
}

// The end of a tile kernel. After a wait that gave up, the loading thread waits
// (again with a limit) for the copies that it has issued, `*issued` items of
// them, an item a stage; and no CTA of a cluster ends while another may store
// into it.
template <int kStages>
__device__ __forceinline__ void leave(uint64_t *full, const int *issued, int cluster, bool dead, int *status) {
    if constexpr (kStages > 0) {
        if (threadIdx.x == kLoader && dead) {
            for (int s = 0; s < kStages; ++s) {
                const int phases = (*issued + kStages - 1 - s) / kStages;
                if (phases > 0) mbar_wait_bounded(&full[s], static_cast<uint32_t>(phases - 1) & 1, status);
            }
        }
    }
    if (cluster > 1) cluster_sync();
}

template <typename T, bool kTma, bool kMasks>
__global__ __launch_bounds__(kTileThreads, forward_resident<T>()) void gated_forward_tile_kernel(
    const __grid_constant__ CUtensorMap map, GatedShape shape, int64_t feature_tiles, int cluster, int per,
    const T *__restrict__ projections, const float *__restrict__ initial, T *__restrict__ states,
    float *__restrict__ final_state, float *__restrict__ carries, int *status) {
    constexpr int kStages = kTma ? 2 : 0;
    using Memory = TileMemory<T, 2, kStages, 2, 1>;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Memory memory(smem_raw);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, block = 2 * warp + (lane >> 4);
    const Walk walk(shape, feature_tiles, cluster, per);
    const int rank = walk.rank, segments = static_cast<int>(shape.segments), items = walk.count * walk.waves;
    const float2 span = both(shape.hi - shape.lo), lo = both(shape.lo);
    const float2 fall = both(shape.lo - shape.hi), top = both(1.0f - shape.lo);  // 1 - a = top + fall s

    auto issue = [&](int item) {
        const int chain = item / walk.waves, segment = (item - chain * walk.waves) * cluster + rank;
        uint64_t *bar = &memory.full[item & 1];
        *memory.issued = item + 1;
        if (segment >= segments) {  // no tile in the chain's last wave: an empty phase
            mbar_arrive(bar);
            return;
        }
        T *box = memory.stages + (item & 1) * 2 * Memory::kBox;
        mbar_arrive_expect_tx(bar, Memory::kStageBytes);
        const int32_t f = static_cast<int32_t>(walk.feature(chain)), batch = static_cast<int32_t>(walk.batch(chain));
        tma_load_3d(box, &map, bar, f, segment * kSegment, batch);
        tma_load_3d(box + Memory::kBox, &map, bar, static_cast<int32_t>(shape.features) + f, segment * kSegment, batch);
    };
    bool dead = false;  // a wait gave up: go on without waiting or loading
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(&memory.full[s], 1);
            mbar_init(&memory.met[s], 1);
        }
        fence_barrier_init();
        if (kTma) prefetch_tensor_map(&map);
    }
    __syncthreads();
    if (kTma && threadIdx.x == kLoader) {
        for (int i = 0; i < items && i < kStages; ++i) issue(i);
    }
    if (cluster > 1) cluster_sync();  // every CTA's barriers are ready before one stores into another

    int item = 0;
    for (int chain = 0; chain < walk.count; ++chain) {
        const int64_t batch = walk.batch(chain), f0 = walk.feature(chain);
        const LaneFeatures<kTma> features(f0, lane, shape.features);
        const int64_t first_row = batch * shape.length + int64_t(rank) * kSegment + block * kRows;
        const T *in = projections + first_row * 2 * shape.features + features.x;
        T *out = states + first_row * shape.features + features.x;
        // the walking warp's feature and state
        const int64_t walked = f0 + walked_feature<kTma>(lane);
        const bool walks = warp == 0, walks_in = walks && walked < shape.features;
        float carry = walks_in && initial != nullptr ? initial[batch * shape.features + walked] : 0.0f;
        RowFlags next_flags = row_flags<kMasks>(shape, batch, rank, warp, lane);
        for (int segment = rank; segment - rank < segments; segment += cluster, ++item) {
            const RowFlags flags = next_flags;
            next_flags = row_flags<kMasks>(shape, batch, segment + cluster, warp, lane);

            if (kTma && !dead) dead = !mbar_wait_bounded(&memory.full[item & 1], static_cast<uint32_t>(item >> 1) & 1, status);
            float2 a[kRows], b[kRows];
            float2 m = both(1.0f), n = both(0.0f);
            const T *box = memory.stages + (item & 1) * 2 * Memory::kBox + block * kRows * kTileFeatures + 2 * (lane & 15);
            auto gates = [&](int j) {
                float2 p, c, s, k;
                if (kTma) {
                    p = load_clamped<true>(box + j * kTileFeatures);
                    c = load_clamped<false>(box + Memory::kBox + j * kTileFeatures);
                } else {
                    p = clamped<true>(features.load(in + j * 2 * shape.features));
                    c = clamped<false>(features.load(in + j * 2 * shape.features + shape.features));
                }
                gates_of<T>(p, c, s, k);
                a[j] = fma2(span, s, lo);
                b[j] = mul2(fma2(fall, s, top), k);
            };
            if (flags.plain) {
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    gates(j);
                    m = mul2(m, a[j]);
                    n = fma2(a[j], n, b[j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    a[j] = both(1.0f);
                    b[j] = both(0.0f);
                    if (flags.cut >> j & 1u) n = both(0.0f);
                    if (flags.live >> j & 1u) gates(j);
                    m = mul2(m, a[j]);
                    n = fma2(a[j], n, b[j]);
                }
            }
            m = flags.cut != 0 ? both(0.0f) : make_float2(fmaxf(m.x, kSmallest), fmaxf(m.y, kSmallest));
            const int at = block * kTileFeatures + 2 * (lane & 15);
            *reinterpret_cast<float2 *>(memory.maps + at) = m;
            *reinterpret_cast<float2 *>(memory.maps + Memory::kPlane + at) = n;
            __syncthreads();
            if (kTma && threadIdx.x == kLoader && !dead && item + kStages < items) issue(item + kStages);

            if (walks) {
                const float *mm = memory.maps + lane, *nn = mm + Memory::kPlane;
                float start = carry;
                if (cluster > 1) {
                    start = meet<kMasks, false>(memory, item, cluster, rank, tile_map_of<kMasks, false>(mm, nn), carry, dead, status);
                }
                if (carries != nullptr && walks_in && segment < segments) {
                    carries[(batch * shape.segments + segment) * shape.features + walked] = start;
                }
                float mr[kBlocks / 2], nr[kBlocks / 2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int i = 0; i < kBlocks / 2; ++i) {
                        mr[i] = mm[(half * (kBlocks / 2) + i) * kTileFeatures];
                        nr[i] = nn[(half * (kBlocks / 2) + i) * kTileFeatures];
                    }
#pragma unroll
                    for (int i = 0; i < kBlocks / 2; ++i) {
                        memory.starts[(half * (kBlocks / 2) + i) * kTileFeatures + lane] = start;
                        start = apply<kMasks>(mr[i], nr[i], start);
                    }
                }
                if (cluster == 1) carry = start;
            }
            __syncthreads();

            float2 h = *reinterpret_cast<const float2 *>(memory.starts + at);
            T *row = out;
            if (flags.plain) {
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    h = fma2(a[j], h, b[j]);
                    features.store(row, h);
                    row += shape.features;
                }
            } else {
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    if (flags.cut >> j & 1u) h = both(0.0f);
                    h = fma2(a[j], h, b[j]);
                    if (j < flags.rows_in) features.store(row, h);
                    row += shape.features;
                }
            }
            in += int64_t(cluster) * kSegment * 2 * shape.features;
            out += int64_t(cluster) * kSegment * shape.features;
        }
        if (rank == 0 && walks_in) final_state[batch * shape.features + walked] = carry;
    }
    leave<kStages>(memory.full, memory.issued, cluster, dead, status);
}

// The waves run from the end. Per row a lane keeps a, k and u = (h' - k)(hi -
// lo) s (1 - s) in registers, h' recomputed from the tile's carry; g stays in
// its stage until the row's gradients are stored.
template <typename T, bool kTma, bool kMasks>
__global__ __launch_bounds__(kTileThreads, kBackwardResident) void gated_backward_tile_kernel(
    const __grid_constant__ CUtensorMap map, const __grid_constant__ CUtensorMap grad_map, GatedShape shape,
    int64_t feature_tiles, int cluster, int per, const T *__restrict__ projections, const float *__restrict__ carries,
    const T *__restrict__ grad_states, const float *__restrict__ grad_final, T *__restrict__ grad_projections,
    float *__restrict__ grad_initial, int *status) {
    constexpr int kStages = kTma ? backward_stages<T>() : 0;
    using Memory = TileMemory<T, 3, kStages, 3, 2>;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Memory memory(smem_raw);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, block = 2 * warp + (lane >> 4);
    const Walk walk(shape, feature_tiles, cluster, per);
    const int rank = walk.rank, segments = static_cast<int>(shape.segments), items = walk.count * walk.waves;
    const float2 span = both(shape.hi - shape.lo), lo = both(shape.lo);
    const bool have_grad = grad_states != nullptr;

    auto issue = [&](int item) {
        const int chain = item / walk.waves, segment = (walk.waves - 1 - (item - chain * walk.waves)) * cluster + rank;
        const int stage = item % (kStages > 0 ? kStages : 1);
        uint64_t *bar = &memory.full[stage];
        *memory.issued = item + 1;
        if (segment >= segments) {  // no tile in the chain's last wave: an empty phase
            mbar_arrive(bar);
            return;
        }
        T *box = memory.stages + stage * 3 * Memory::kBox;
        mbar_arrive_expect_tx(bar, have_grad ? Memory::kStageBytes : Memory::kStageBytes / 3 * 2);
        const int32_t t = segment * kSegment, f = static_cast<int32_t>(walk.feature(chain));
        const int32_t batch = static_cast<int32_t>(walk.batch(chain));
        tma_load_3d(box, &map, bar, f, t, batch);
        tma_load_3d(box + Memory::kBox, &map, bar, static_cast<int32_t>(shape.features) + f, t, batch);
        if (have_grad) tma_load_3d(box + 2 * Memory::kBox, &grad_map, bar, f, t, batch);
    };
    bool dead = false;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(&memory.full[s], 1);
        for (int s = 0; s < 2; ++s) mbar_init(&memory.met[s], 1);
        fence_barrier_init();
        if (kTma) prefetch_tensor_map(&map);
        if (kTma && have_grad) prefetch_tensor_map(&grad_map);
    }
    __syncthreads();
    if (kTma && threadIdx.x == kLoader) {
        for (int i = 0; i < items && i < kStages; ++i) issue(i);
    }
    if (cluster > 1) cluster_sync();

    int item = 0;
    for (int chain = 0; chain < walk.count; ++chain) {
        const int64_t batch = walk.batch(chain), f0 = walk.feature(chain);
        const LaneFeatures<kTma> features(f0, lane, shape.features);
        const int last = (walk.waves - 1) * cluster + rank;
        const int64_t first_row = batch * shape.length + int64_t(last) * kSegment;
        const T *in = projections + first_row * 2 * shape.features;
        const T *grad_in = grad_states + first_row * shape.features;
        T *grad_out = grad_projections + first_row * 2 * shape.features;
        const uint32_t width = static_cast<uint32_t>(shape.features);
        const uint32_t two_at = block * kRows * 2 * width + static_cast<uint32_t>(features.x);
        const uint32_t one_at = block * kRows * width + static_cast<uint32_t>(features.x);
        const int64_t walked = f0 + walked_feature<kTma>(lane);
        const bool walks = warp == 0, walks_in = walks && walked < shape.features;
        float x = walks_in && grad_final != nullptr ? grad_final[batch * shape.features + walked] : 0.0f;
        RowFlags next_flags = row_flags<kMasks>(shape, batch, last, warp, lane);
        for (int segment = last; segment >= 0; segment -= cluster, ++item) {
            float before = 0.0f;  // the state before this tile
            if (walks_in && segment < segments) before = carries[(batch * shape.segments + segment) * shape.features + walked];
            const RowFlags flags = next_flags;
            if (segment >= cluster) next_flags = row_flags<kMasks>(shape, batch, segment - cluster, warp, lane);
            const int stage = item % (kStages > 0 ? kStages : 1);
            if (kTma && !dead) {
                dead = !mbar_wait_bounded(&memory.full[stage], static_cast<uint32_t>(item / (kStages > 0 ? kStages : 1)) & 1, status);
            }
            const T *box = memory.stages + stage * 3 * Memory::kBox + block * kRows * kTileFeatures + 2 * (lane & 15);
            auto load_grad = [&](int j) {
                if (!have_grad) return both(0.0f);
                return kTma ? load_two(box + 2 * Memory::kBox + j * kTileFeatures) : features.load(grad_in + (one_at + j * width));
            };

            float2 a[kRows], k[kRows], u[kRows];  // u: (hi - lo) s (1 - s), then times h' - k
            float2 m = both(1.0f), n = both(0.0f), back = both(0.0f);
            auto gates = [&](int j) {
                float2 p, c, s;
                if (kTma) {
                    p = load_clamped<true>(box + j * kTileFeatures);
                    c = load_clamped<false>(box + Memory::kBox + j * kTileFeatures);
                } else {
                    p = clamped<true>(features.load(in + (two_at + j * 2 * width)));
                    c = clamped<false>(features.load(in + (two_at + j * 2 * width + width)));
                }
                gates_of<T>(p, c, s, k[j]);
                a[j] = fma2(span, s, lo);
                u[j] = mul2(mul2(span, s), sub2(both(1.0f), s));
            };
            if (flags.plain) {
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    gates(j);
                    m = mul2(m, a[j]);
                    n = fma2(a[j], sub2(n, k[j]), k[j]);
                }
#pragma unroll
                for (int j = kRows - 1; j >= 0; --j) back = mul2(a[j], add2(back, load_grad(j)));
            } else {
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    a[j] = both(1.0f);
                    k[j] = u[j] = both(0.0f);
                    if (flags.cut >> j & 1u) n = both(0.0f);
                    if (flags.live >> j & 1u) {
                        gates(j);
                        m = mul2(m, a[j]);
                        n = fma2(a[j], sub2(n, k[j]), k[j]);
                    }
                }
#pragma unroll
                for (int j = kRows - 1; j >= 0; --j) {
                    if (j < flags.rows_in) back = mul2(a[j], add2(back, load_grad(j)));
                    if (flags.cut >> j & 1u) back = both(0.0f);
                }
            }
            m = flags.cut != 0 ? both(0.0f) : make_float2(fmaxf(m.x, kSmallest), fmaxf(m.y, kSmallest));
            const int at = block * kTileFeatures + 2 * (lane & 15);
            *reinterpret_cast<float2 *>(memory.maps + at) = m;
            *reinterpret_cast<float2 *>(memory.maps + Memory::kPlane + at) = n;
            *reinterpret_cast<float2 *>(memory.maps + 2 * Memory::kPlane + at) = back;
            __syncthreads();
            // every warp is done with the previous item's stage
            if (kTma && threadIdx.x == kLoader && !dead && item > 0 && item - 1 + kStages < items) issue(item - 1 + kStages);

            if (walks) {
                const float *mm = memory.maps + lane, *nn = mm + Memory::kPlane, *gg = nn + Memory::kPlane;
                float *h_at = memory.starts + lane, *x_at = h_at + Memory::kPlane;
                float start = x;
                if (cluster > 1) {
                    start = meet<kMasks, true>(memory, item, cluster, rank, tile_map_of<kMasks, true>(mm, gg), x, dead, status);
                }
                float mr[kBlocks], vr[kBlocks];
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) {
                    mr[i] = mm[i * kTileFeatures];
                    vr[i] = nn[i * kTileFeatures];
                }
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) {
                    h_at[i * kTileFeatures] = before;
                    before = apply<kMasks>(mr[i], vr[i], before);
                }
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) vr[i] = gg[i * kTileFeatures];
#pragma unroll
                for (int i = kBlocks - 1; i >= 0; --i) {
                    x_at[i * kTileFeatures] = start;
                    start = apply<kMasks>(mr[i], vr[i], start);
                }
                if (cluster == 1) x = start;
            }
            __syncthreads();

            float2 h = *reinterpret_cast<const float2 *>(memory.starts + at);
            float2 from = *reinterpret_cast<const float2 *>(memory.starts + Memory::kPlane + at);
            auto state_through = [&](int j) {  // u times h' - k, and the state behind row j
                const float2 gap = sub2(h, k[j]);
                u[j] = mul2(gap, u[j]);
                h = fma2(a[j], gap, k[j]);
            };
            auto gradients = [&](int j, float2 &dp, float2 &dc) {  // of row j, and x in front of it
                const float2 adjoint = add2(from, load_grad(j));
                dp = mul2(adjoint, u[j]);
                dc = mul2(adjoint, mul2(sub2(both(1.0f), a[j]), sub2(both(1.0f), mul2(k[j], k[j]))));
                from = mul2(a[j], adjoint);
            };
            if (flags.plain) {
#pragma unroll
                for (int j = 0; j < kRows; ++j) state_through(j);
                T *row = grad_out + (two_at + (kRows - 1) * 2 * width);
#pragma unroll
                for (int j = kRows - 1; j >= 0; --j) {
                    float2 dp, dc;
                    gradients(j, dp, dc);
                    features.store(row + width, dc);
                    features.store(row, dp);
                    row -= 2 * shape.features;
                }
            } else {
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    if (flags.cut >> j & 1u) h = both(0.0f);
                    state_through(j);
                }
#pragma unroll
                for (int j = kRows - 1; j >= 0; --j) {
                    if (j >= flags.rows_in) continue;
                    float2 dp, dc;
                    gradients(j, dp, dc);
                    if (!(flags.live >> j & 1u)) dp = dc = both(0.0f);
                    if (flags.cut >> j & 1u) from = both(0.0f);
                    features.store(grad_out + (two_at + j * 2 * width), dp);
                    features.store(grad_out + (two_at + j * 2 * width + width), dc);
                }
            }
            in -= int64_t(cluster) * kSegment * 2 * shape.features;
            grad_in -= int64_t(cluster) * kSegment * shape.features;
            grad_out -= int64_t(cluster) * kSegment * 2 * shape.features;
        }
        if (grad_initial != nullptr && rank == 0 && walks_in) grad_initial[batch * shape.features + walked] = x;
    }
    leave<kStages>(memory.full, memory.issued, cluster, dead, status);
}

// A tensor map over [batch, length, width] in boxes of one tile.
template <typename T>
int tile_map(CUtensorMap *map, const void *base, int64_t batch, int64_t length, int64_t width) {
    const uint64_t es = sizeof(T);
    const uint64_t dims[3] = {static_cast<uint64_t>(width), static_cast<uint64_t>(length), static_cast<uint64_t>(batch)};
    const uint64_t strides[2] = {width * es, length * width * es};
    const uint32_t box[3] = {kTileFeatures, kSegment, 1};
    return encode_tensor_map(map, GatedMapType<T>::value, 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Whether TMA can address the rows: F elements are a multiple of 16 bytes (the
// candidates start F elements into a row) and the bases are aligned.
template <typename T>
bool tma_rows(const GatedShape &shape, const void *projections, const void *grad, const void *out) {
    return (shape.features * sizeof(T)) % 16 == 0 && aligned(projections, 16) && aligned(grad, 16) && aligned(out, 16);
}

// CTAs per chain: as many as the GPU holds at once (`resident` CTAs per SM), up
// to `most` and to the number of tiles. Clusters of 4 fill 19/20 of the places
// (a cluster stays within a group of SMs): 148 chains of 8192 positions took 75
// us in twos and 81 us in fours that needed every place. Clusters of 8, past
// which nothing hides a long chain's latency, may overflow: 74 chains of 32768
// positions took 158 us in eights and 177 us in fours.
int cluster_size(const GatedShape &shape, int64_t chains, int resident, int most) {
    const int64_t places = int64_t(resident) * sm_count();
    int cluster = 1;
    while (cluster < most && 2 * cluster <= shape.segments) {
        const int wider = 2 * cluster;
        if (chains * wider > (wider == 4 ? places * 19 / 20 : places)) break;
        cluster = wider;
    }
    return cluster;
}

// Neighbouring chains a cluster walks one after the other: up to kItems tiles
// per CTA, as long as the GPU's places are taken kRounds times over (with
// fewer rounds the last, partly filled one costs more than a CTA's first load
// and setup do).
int chains_per_cluster(const GatedShape &shape, int64_t chains, int cluster, int resident) {
    constexpr int64_t kItems = 8, kRounds = 4;
    const int64_t waves = ceil_div(shape.segments, cluster), places = ceil_div(int64_t(resident) * sm_count(), cluster);
    int64_t per = kItems / waves;
    if (per > chains / (kRounds * places)) per = chains / (kRounds * places);
    return per < 1 ? 1 : static_cast<int>(per);
}

template <typename... KernelArgs, typename... Args>
int launch_tiles(void (*kernel)(KernelArgs...), int64_t clusters, int cluster, size_t smem, size_t most_smem, cudaStream_t stream,
                 Args &&...args) {
    if (clusters * cluster >= (int64_t(1) << 31)) return fail(KOEMI_ERR_UNSUPPORTED, "the recurrence has too many lanes");
    // the most that any call wants, not this one's: another thread's launch may stand between the two calls
    KOEMI_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most_smem)));
    KOEMI_CUDA_TRY(launch_programmatic(false, kernel, dim3(static_cast<unsigned>(clusters * cluster)), dim3(kTileThreads), smem,
                                       stream, dim3(cluster, 1, 1), std::forward<Args>(args)...));
    return KOEMI_OK;
}

template <typename T>
int gated_forward(const GatedShape &shape, const void *projections, const float *initial, void *states,
                  float *final_state, float *carries, cudaStream_t stream) {
    const T *in = static_cast<const T *>(projections);
    T *out = static_cast<T *>(states);
    if (shape.length <= kShortLength) {
        const unsigned blocks = static_cast<unsigned>(ceil_div(shape.batch * shape.features, 128));
        gated_forward_lane_kernel<T><<<blocks, 128, 0, stream>>>(shape, in, initial, out, final_state, carries);
        KOEMI_LAUNCH_CHECK();
        return KOEMI_OK;
    }
    const int64_t feature_tiles = ceil_div(shape.features, kTileFeatures);
    const int64_t chains = shape.batch * feature_tiles;
    const int cluster = cluster_size(shape, chains, forward_resident<T>(), kMaxCluster);
    const int per = chains_per_cluster(shape, chains, cluster, forward_resident<T>());
    const bool masks = shape.valid != nullptr || shape.restart != nullptr;
    int *status = device_status_word();
    CUtensorMap map{};
    auto go = [&](auto kernel, bool tma) {
        auto bytes = tma ? TileMemory<T, 2, 2, 2, 1>::bytes : TileMemory<T, 2, 0, 2, 1>::bytes;
        return launch_tiles(kernel, ceil_div(chains, per), cluster, bytes(cluster), bytes(kMaxCluster), stream, map, shape,
                            feature_tiles, cluster, per, in, initial, out, final_state, carries, status);
    };
    if (tma_rows<T>(shape, projections, nullptr, states)) {
        const int rc = tile_map<T>(&map, projections, shape.batch, shape.length, 2 * shape.features);
        if (rc != KOEMI_OK) return rc;
        return masks ? go(gated_forward_tile_kernel<T, true, true>, true) : go(gated_forward_tile_kernel<T, true, false>, true);
    }
    return masks ? go(gated_forward_tile_kernel<T, false, true>, false) : go(gated_forward_tile_kernel<T, false, false>, false);
}

template <typename T>
int gated_backward(const GatedShape &shape, const void *projections, const float *carries, const void *grad_states,
                   const float *grad_final, void *grad_projections, float *grad_initial, cudaStream_t stream) {
    const T *in = static_cast<const T *>(projections);
    const T *grad = static_cast<const T *>(grad_states);
    T *out = static_cast<T *>(grad_projections);
    if (shape.length <= kShortLength) {
        const unsigned blocks = static_cast<unsigned>(ceil_div(shape.batch * shape.features, 128));
        gated_backward_lane_kernel<T><<<blocks, 128, 0, stream>>>(shape, in, carries, grad, grad_final, out, grad_initial);
        KOEMI_LAUNCH_CHECK();
        return KOEMI_OK;
    }
    const int64_t feature_tiles = ceil_div(shape.features, kTileFeatures);
    const int64_t chains = shape.batch * feature_tiles;
    const int cluster = cluster_size(shape, chains, kBackwardResident, kMaxCluster);
    const int per = chains_per_cluster(shape, chains, cluster, kBackwardResident);
    const bool masks = shape.valid != nullptr || shape.restart != nullptr;
    int *status = device_status_word();
    CUtensorMap map{}, grad_map{};
    auto go = [&](auto kernel, bool tma) {
        auto bytes = tma ? TileMemory<T, 3, backward_stages<T>(), 3, 2>::bytes : TileMemory<T, 3, 0, 3, 2>::bytes;
        return launch_tiles(kernel, ceil_div(chains, per), cluster, bytes(cluster), bytes(kMaxCluster), stream, map, grad_map,
                            shape, feature_tiles, cluster, per, in, carries, grad, grad_final, out, grad_initial, status);
    };
    if (tma_rows<T>(shape, projections, grad_states, grad_projections)) {
        int rc = tile_map<T>(&map, projections, shape.batch, shape.length, 2 * shape.features);
        if (rc == KOEMI_OK && grad != nullptr) rc = tile_map<T>(&grad_map, grad_states, shape.batch, shape.length, shape.features);
        if (rc != KOEMI_OK) return rc;
        return masks ? go(gated_backward_tile_kernel<T, true, true>, true) : go(gated_backward_tile_kernel<T, true, false>, true);
    }
    return masks ? go(gated_backward_tile_kernel<T, false, true>, false) : go(gated_backward_tile_kernel<T, false, false>, false);
}

int check_gated(const GatedShape &shape) {
    if (shape.batch < 0 || shape.length < 0 || shape.features < 0) {
        return fail(KOEMI_ERR_INVALID, "recurrence sizes must be non-negative");
    }
    if (!(shape.lo > 0.0f && shape.lo <= shape.hi && shape.hi < 1.0f)) {
        return fail(KOEMI_ERR_INVALID, "retention bounds must satisfy 0 < minimum <= maximum < 1");
    }
    // a tile's places are counted in 32 bits: 128 rows of 2 F elements
    constexpr int64_t kMost = int64_t(1) << 30, kWidest = int64_t(1) << 22;
    if (shape.batch > kMost || shape.length > kMost || shape.features > kWidest ||
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
