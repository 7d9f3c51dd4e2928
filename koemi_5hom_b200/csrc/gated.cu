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
// it needs on chip instead of reading them:
//
//   adj_t = g_t + x_t,  x_{t-1} = a_t adj_t (0 at a restart)
//   dp_t = adj_t (h' - k_t) (hi - lo) s (1 - s)
//   dc_t = adj_t (1 - a_t) (1 - k_t^2),  d_initial = x_{-1}
//
// Every step is an affine map of the state (forward) or of x (backward), so a
// tile of 64 positions x 64 features composes into one map per feature. A CTA
// of 8 warps takes a tile: warp w holds rows [8 w, 8 w + 8) in registers, a
// lane two features; the warps' maps meet in shared memory. A chain (one
// batch row, 64 features) is walked by a cluster of 1 to 8 CTAs, a wave of as
// many neighbouring tiles at a time: every CTA stores its tile's map into the
// other CTAs' shared memory, and one cluster barrier later each folds the
// maps in front of its tile onto the carry and replays its rows. Nothing is
// exchanged through global memory, no CTA waits for one outside its cluster,
// and the order of every sum is fixed, so equal inputs give equal bits.
#include "common.cuh"

namespace koemi {
namespace {

constexpr int kSegment = 64;  // positions of a tile, and between two carries
constexpr int kTileFeatures = 64;
constexpr int kTileWarps = 8;
constexpr int kTileThreads = kTileWarps * 32;
constexpr int kTileRows = kSegment / kTileWarps;
constexpr int kMaxCluster = 8;
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

// a and k of one element. With yp = 1 + e^-p and yc = 1 + e^2c, s = 1 / yp and
// k = 1 - 2 / yc share one reciprocal, of yp yc; the exponents stop at 40,
// where both have reached their limits in fp32, so that the product stays
// finite. Both are good to a few 2^-24 of 1. For 16-bit inputs that is far
// below the inputs' own rounding; fp32 inputs near 0 take tanh's series
// instead (good to 2^-24 of k up to |c| = 1/4), since k is as small as c there.
template <typename T>
__device__ __forceinline__ void gate_of(float p, float c, float lo, float span, float &a, float &k) {
    constexpr float kLog2e = 1.4426950408889634f;
    const float yp = 1.0f + ex2_approx(min_nan(-kLog2e * p, 40.0f * kLog2e));
    const float yc = 1.0f + ex2_approx(min_nan(2.0f * kLog2e * c, 40.0f * kLog2e));
    const float r = rcp_approx(yp * yc);
    a = fmaf(span, r * yc, lo);
    k = fmaf(-2.0f, r * yp, 1.0f);
    if constexpr (sizeof(T) == 4) {
        const float z = c * c;
        float series = fmaf(z, 62.0f / 2835.0f, -17.0f / 315.0f);
        series = fmaf(z, series, 2.0f / 15.0f);
        series = fmaf(z, series, -1.0f / 3.0f);
        if (z < 0.0625f) k = fmaf(c * z, series, c);
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
            float a, k;
            gate_of<T>(to_acc(projections[row * 2 * shape.features + f]),
                       to_acc(projections[row * 2 * shape.features + shape.features + f]), shape.lo,
                       shape.hi - shape.lo, a, k);
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
    float a[kShortLength], k[kShortLength], before[kShortLength];
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
                       to_acc(projections[row * 2 * shape.features + shape.features + f]), shape.lo, span, a[t], k[t]);
            h = fmaf(a[t], h, fmaf(-a[t], k[t], k[t]));
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
            dp = adjoint * (before[t] - k[t]) * ((a[t] - shape.lo) * (shape.hi - a[t]) / span);
            dc = adjoint * (1.0f - a[t]) * fmaf(-k[t], k[t], 1.0f);
            x = a[t] * adjoint;
        }
        if (cut >> t & 1u) x = 0.0f;
        grad_projections[row * 2 * shape.features + f] = from_acc<T>(dp);
        grad_projections[row * 2 * shape.features + shape.features + f] = from_acc<T>(dc);
    }
    if (grad_initial != nullptr) grad_initial[lane] = x;
}

// ------------------------------------------------------------------ tiles

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void store_remote(void *local, uint32_t rank, float4 v) {
    uint32_t address;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(address) : "r"(smem_addr(local)), "r"(rank));
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(address), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                 : "memory");
}

// A map v -> m v + n of two features, {m.x, m.y, n.x, n.y}. m is exactly 0
// only where a restart drops v, and then v is not multiplied (it may be a
// NaN); a product that underflows stays at the smallest positive number.
__device__ __forceinline__ float apply(float m, float n, float v) { return m == 0.0f ? n : fmaf(m, v, n); }
__device__ __forceinline__ float chain(float m, float n) {
    return m == 0.0f || n == 0.0f ? 0.0f : fmaxf(m * n, 1.4e-45f);
}
// first, then second
__device__ __forceinline__ float4 compose(float4 first, float4 second) {
    return make_float4(chain(second.x, first.x), chain(second.y, first.y), apply(second.x, second.z, first.z),
                       apply(second.y, second.w, first.w));
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

// Where a lane's two features are. TMA tiles: features 2 l and 2 l + 1 (one
// 4- or 8-byte access, the width is a multiple of 8 bytes at least). Without
// TMA: l and l + 32, single elements, so that a warp's accesses stay
// contiguous at any alignment.
template <bool kTma>
struct LaneFeatures {
    int64_t x, y;
    bool x_in, y_in;
    __device__ LaneFeatures(int64_t first, int lane, int64_t features) {
        x = first + (kTma ? 2 * lane : lane);
        y = kTma ? x + 1 : x + 32;
        x_in = x < features;
        y_in = y < features;
    }
    template <typename T>
    __device__ __forceinline__ float2 load(const T *row) const {
        if (kTma) return x_in ? load_two(row + x) : make_float2(0.0f, 0.0f);
        return make_float2(x_in ? to_acc(row[x]) : 0.0f, y_in ? to_acc(row[y]) : 0.0f);
    }
    template <typename T>
    __device__ __forceinline__ void store(T *row, float2 v) const {
        if (kTma) {
            if (x_in) store_two(row + x, v);
        } else {
            if (x_in) row[x] = from_acc<T>(v.x);
            if (y_in) row[y] = from_acc<T>(v.y);
        }
    }
    // fp32 side arrays, whose base has its own alignment
    __device__ __forceinline__ float2 load_side(const float *row) const {
        return make_float2(x_in ? row[x] : 0.0f, y_in ? row[y] : 0.0f);
    }
    __device__ __forceinline__ void store_side(float *row, float2 v) const {
        if (x_in) row[x] = v.x;
        if (y_in) row[y] = v.y;
    }
};

// Which of a warp's rows are inside the sequence and valid, and which restart.
struct RowFlags {
    uint32_t live, cut;
};
template <bool kMasks>
__device__ __forceinline__ RowFlags row_flags(const GatedShape &shape, int64_t batch, int64_t t0, int lane) {
    RowFlags f;
    if (kMasks) {
        const int64_t t = t0 + lane;
        const bool in = lane < kTileRows && t < shape.length;
        const int64_t row = batch * shape.length + t;
        f.live = __ballot_sync(0xffffffffu, in && (shape.valid == nullptr || shape.valid[row] != 0));
        f.cut = __ballot_sync(0xffffffffu, in && shape.restart != nullptr && shape.restart[row] != 0);
    } else {
        const int64_t left = shape.length - t0;
        f.live = left >= kTileRows ? (1u << kTileRows) - 1 : left <= 0 ? 0u : (1u << left) - 1;
        f.cut = 0;
    }
    return f;
}

// Shared memory of a tile kernel: kStages stages of kArrays boxes, then the
// warps' maps of two waves, the cluster's maps of two waves, the barriers.
template <typename T, int kArrays, int kStages>
struct TileMemory {
    static constexpr int kBox = kSegment * kTileFeatures;
    static constexpr uint32_t kStageBytes = kArrays * kBox * sizeof(T);
    T *stages;
    float4 *warps;    // [2][kTileWarps][32]
    float2 *extra;    // [2][kTileWarps][32], the backward's third value
    float4 *cluster;  // [2][kMaxCluster][32]
    uint64_t *full;   // [kStages]
    __device__ explicit TileMemory(unsigned char *raw) {
        stages = reinterpret_cast<T *>(raw);
        warps = reinterpret_cast<float4 *>(raw + size_t(kStages) * kStageBytes);
        cluster = warps + 2 * kTileWarps * 32;
        extra = reinterpret_cast<float2 *>(cluster + 2 * kMaxCluster * 32);
        full = reinterpret_cast<uint64_t *>(extra + 2 * kTileWarps * 32);
    }
    static size_t bytes(bool tma) {
        return (tma ? size_t(kStages) * kStageBytes : 0) + 2 * (kTileWarps + kMaxCluster) * 32 * sizeof(float4) +
               2 * kTileWarps * 32 * sizeof(float2) + kStages * sizeof(uint64_t);
    }
};

template <typename T>
constexpr int forward_stages() {
    return sizeof(T) == 2 ? 3 : 2;
}

template <typename T, bool kTma, bool kMasks>
__global__ __launch_bounds__(kTileThreads, 3) void gated_forward_tile_kernel(
    const __grid_constant__ CUtensorMap map, GatedShape shape, int64_t feature_tiles, int cluster,
    const T *__restrict__ projections, const float *__restrict__ initial, T *__restrict__ states,
    float *__restrict__ final_state, float *__restrict__ carries, int *status) {
    constexpr int kStages = kTma ? forward_stages<T>() : 0;
    using Memory = TileMemory<T, 2, kStages>;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Memory memory(smem_raw);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = static_cast<int>(blockIdx.x % cluster);
    const int64_t chain_index = blockIdx.x / cluster;
    const int64_t batch = chain_index / feature_tiles;
    const int64_t f0 = (chain_index - batch * feature_tiles) * kTileFeatures;
    const int64_t waves = (shape.segments + cluster - 1) / cluster;
    const LaneFeatures<kTma> features(f0, lane, shape.features);
    const float span = shape.hi - shape.lo;
    const T *in = projections + batch * shape.length * 2 * shape.features;
    T *out = states + batch * shape.length * shape.features;

    auto issue = [&](int64_t wave) {
        const int64_t segment = wave * cluster + rank;
        if (segment >= shape.segments) return;
        const int stage = static_cast<int>(wave % (kStages > 0 ? kStages : 1));
        T *box = memory.stages + size_t(stage) * 2 * Memory::kBox;
        mbar_arrive_expect_tx(&memory.full[stage], Memory::kStageBytes);
        const int32_t t = static_cast<int32_t>(segment * kSegment), f = static_cast<int32_t>(f0);
        tma_load_3d(box, &map, &memory.full[stage], f, t, static_cast<int32_t>(batch));
        tma_load_3d(box + Memory::kBox, &map, &memory.full[stage], static_cast<int32_t>(shape.features) + f, t,
                    static_cast<int32_t>(batch));
    };
    bool dead = false;  // a load never arrived: go on without waiting or loading
    if (kTma) {
        if (threadIdx.x == 0) {
            for (int s = 0; s < kStages; ++s) mbar_init(&memory.full[s], 1);
            fence_barrier_init();
            prefetch_tensor_map(&map);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int64_t w = 0; w < waves && w < kStages; ++w) issue(w);
        }
    }
    if (cluster > 1) cluster_sync();  // every CTA of the cluster runs before one stores into another

    float2 carry = initial != nullptr ? features.load_side(initial + batch * shape.features) : make_float2(0.0f, 0.0f);
    RowFlags next_flags = row_flags<kMasks>(shape, batch, int64_t(rank) * kSegment + warp * kTileRows, lane);
    for (int64_t wave = 0; wave < waves; ++wave) {
        const int64_t segment = wave * cluster + rank;
        const int64_t t0 = segment * kSegment + warp * kTileRows;
        const int parity = static_cast<int>(wave & 1);
        const RowFlags flags = next_flags;
        next_flags = row_flags<kMasks>(shape, batch, t0 + int64_t(cluster) * kSegment, lane);
        const bool plain = flags.live == (1u << kTileRows) - 1 && flags.cut == 0;

        float2 a[kTileRows], b[kTileRows];
        if (kTma && segment < shape.segments && !dead) {
            const int stage = static_cast<int>(wave % (kStages > 0 ? kStages : 1));
            dead = !mbar_wait_bounded(&memory.full[stage], static_cast<uint32_t>(wave / (kStages > 0 ? kStages : 1)) & 1, status);
        }
        {
            const int stage = static_cast<int>(wave % (kStages > 0 ? kStages : 1));
            const T *box = memory.stages + size_t(stage) * 2 * Memory::kBox + warp * kTileRows * kTileFeatures + 2 * lane;
#pragma unroll
            for (int j = 0; j < kTileRows; ++j) {
                float2 p, c;
                if (kTma) {
                    p = load_two(box + j * kTileFeatures);
                    c = load_two(box + Memory::kBox + j * kTileFeatures);
                } else {
                    p = c = make_float2(0.0f, 0.0f);
                    if (t0 + j < shape.length) {
                        p = features.load(in + (t0 + j) * 2 * shape.features);
                        c = features.load(in + (t0 + j) * 2 * shape.features + shape.features);
                    }
                }
                float kx, ky;
                gate_of<T>(p.x, c.x, shape.lo, span, a[j].x, kx);
                gate_of<T>(p.y, c.y, shape.lo, span, a[j].y, ky);
                b[j] = make_float2(fmaf(-a[j].x, kx, kx), fmaf(-a[j].y, ky, ky));
            }
        }
        float4 rows = make_float4(1.0f, 1.0f, 0.0f, 0.0f);
        if (plain) {
#pragma unroll
            for (int j = 0; j < kTileRows; ++j) {
                rows.x *= a[j].x;
                rows.y *= a[j].y;
                rows.z = fmaf(a[j].x, rows.z, b[j].x);
                rows.w = fmaf(a[j].y, rows.w, b[j].y);
            }
            rows.x = fmaxf(rows.x, 1.4e-45f);
            rows.y = fmaxf(rows.y, 1.4e-45f);
        } else {
#pragma unroll
            for (int j = 0; j < kTileRows; ++j) {
                if (!(flags.live >> j & 1u)) {
                    a[j] = make_float2(1.0f, 1.0f);
                    b[j] = make_float2(0.0f, 0.0f);
                }
                if (flags.cut >> j & 1u) a[j] = make_float2(0.0f, 0.0f);
                rows = compose(rows, make_float4(a[j].x, a[j].y, b[j].x, b[j].y));
            }
        }
        float4 *warps = memory.warps + parity * kTileWarps * 32 + lane;
        warps[warp * 32] = rows;
        __syncthreads();
        if (kTma && threadIdx.x == 0 && !dead && wave + kStages < waves) issue(wave + kStages);

        if (cluster > 1) {
            float4 *tiles = memory.cluster + parity * kMaxCluster * 32 + lane;
            if (warp < cluster) {
                float4 total = warps[0];
#pragma unroll
                for (int w = 1; w < kTileWarps; ++w) total = compose(total, warps[w * 32]);
                store_remote(tiles + rank * 32, static_cast<uint32_t>(warp), total);
            }
            cluster_sync();
            float2 h = carry;
            for (int r = 0; r < cluster; ++r) {
                if (r == rank) carry = h;  // from here on: the state before this tile
                const float4 m = tiles[r * 32];
                h = make_float2(apply(m.x, m.z, h.x), apply(m.y, m.w, h.y));
            }
            // h: the state after the wave; carry: before this tile
            const float2 after = h;
            h = carry;
            if (carries != nullptr && warp == 0 && segment < shape.segments) {
                features.store_side(carries + (batch * shape.segments + segment) * shape.features, h);
            }
            for (int w = 0; w < warp; ++w) {
                const float4 m = warps[w * 32];
                h = make_float2(apply(m.x, m.z, h.x), apply(m.y, m.w, h.y));
            }
            carry = h;
#pragma unroll
            for (int j = 0; j < kTileRows; ++j) {
                if (plain) {
                    carry = make_float2(fmaf(a[j].x, carry.x, b[j].x), fmaf(a[j].y, carry.y, b[j].y));
                } else {
                    carry = make_float2(apply(a[j].x, b[j].x, carry.x), apply(a[j].y, b[j].y, carry.y));
                }
                if (t0 + j < shape.length) features.store(out + (t0 + j) * shape.features, carry);
            }
            carry = after;
        } else {
            if (carries != nullptr && warp == 0) {
                features.store_side(carries + (batch * shape.segments + segment) * shape.features, carry);
            }
            float2 h = carry;
#pragma unroll
            for (int w = 0; w < kTileWarps; ++w) {
                if (w == warp) h = carry;
                const float4 m = warps[w * 32];
                carry = make_float2(apply(m.x, m.z, carry.x), apply(m.y, m.w, carry.y));
            }
#pragma unroll
            for (int j = 0; j < kTileRows; ++j) {
                if (plain) {
                    h = make_float2(fmaf(a[j].x, h.x, b[j].x), fmaf(a[j].y, h.y, b[j].y));
                } else {
                    h = make_float2(apply(a[j].x, b[j].x, h.x), apply(a[j].y, b[j].y, h.y));
                }
                if (t0 + j < shape.length) features.store(out + (t0 + j) * shape.features, h);
            }
        }
    }
    if (rank == 0 && warp == 0) features.store_side(final_state + batch * shape.features, carry);
}

template <typename T>
constexpr int backward_stages() {
    return 2;
}

// The waves run from the end. A row's rolling values: a, k (registers), the
// state before it (recomputed from the segment's carry and the warps' maps)
// and g; x comes from the right.
template <typename T, bool kTma, bool kMasks>
__global__ __launch_bounds__(kTileThreads, 2) void gated_backward_tile_kernel(
    const __grid_constant__ CUtensorMap map, const __grid_constant__ CUtensorMap grad_map, GatedShape shape,
    int64_t feature_tiles, int cluster, const T *__restrict__ projections, const float *__restrict__ carries,
    const T *__restrict__ grad_states, const float *__restrict__ grad_final, T *__restrict__ grad_projections,
    float *__restrict__ grad_initial, int *status) {
    constexpr int kStages = kTma ? backward_stages<T>() : 0;
    using Memory = TileMemory<T, 3, kStages>;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Memory memory(smem_raw);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = static_cast<int>(blockIdx.x % cluster);
    const int64_t chain_index = blockIdx.x / cluster;
    const int64_t batch = chain_index / feature_tiles;
    const int64_t f0 = (chain_index - batch * feature_tiles) * kTileFeatures;
    const int64_t waves = (shape.segments + cluster - 1) / cluster;
    const LaneFeatures<kTma> features(f0, lane, shape.features);
    const float span = shape.hi - shape.lo, inverse_span = 1.0f / span;
    const T *in = projections + batch * shape.length * 2 * shape.features;
    const T *grad_in = grad_states == nullptr ? nullptr : grad_states + batch * shape.length * shape.features;
    T *grad_out = grad_projections + batch * shape.length * 2 * shape.features;

    // step i is wave waves - 1 - i
    auto issue = [&](int64_t step) {
        const int64_t segment = (waves - 1 - step) * cluster + rank;
        if (segment >= shape.segments) return;
        const int stage = static_cast<int>(step % (kStages > 0 ? kStages : 1));
        T *box = memory.stages + size_t(stage) * 3 * Memory::kBox;
        const uint32_t bytes = grad_in == nullptr ? Memory::kStageBytes / 3 * 2 : Memory::kStageBytes;
        mbar_arrive_expect_tx(&memory.full[stage], bytes);
        const int32_t t = static_cast<int32_t>(segment * kSegment), f = static_cast<int32_t>(f0);
        tma_load_3d(box, &map, &memory.full[stage], f, t, static_cast<int32_t>(batch));
        tma_load_3d(box + Memory::kBox, &map, &memory.full[stage], static_cast<int32_t>(shape.features) + f, t,
                    static_cast<int32_t>(batch));
        if (grad_in != nullptr) {
            tma_load_3d(box + 2 * Memory::kBox, &grad_map, &memory.full[stage], f, t, static_cast<int32_t>(batch));
        }
    };
    // A stage's phase counts the loads it has had: a rank without a tile in
    // the last wave skips that one.
    const int64_t skipped = (waves - 1) * cluster + rank >= shape.segments ? 1 : 0;
    bool dead = false;
    if (kTma) {
        if (threadIdx.x == 0) {
            for (int s = 0; s < kStages; ++s) mbar_init(&memory.full[s], 1);
            fence_barrier_init();
            prefetch_tensor_map(&map);
            if (grad_in != nullptr) prefetch_tensor_map(&grad_map);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int64_t i = 0; i < waves && i < kStages; ++i) issue(i);
        }
    }
    if (cluster > 1) cluster_sync();

    float2 x = grad_final != nullptr ? features.load_side(grad_final + batch * shape.features) : make_float2(0.0f, 0.0f);
    for (int64_t step = 0; step < waves; ++step) {
        const int64_t segment = (waves - 1 - step) * cluster + rank;
        const int64_t t0 = segment * kSegment + warp * kTileRows;
        const int parity = static_cast<int>(step & 1);
        const bool have = segment < shape.segments;
        const float2 carry = have ? features.load_side(carries + (batch * shape.segments + segment) * shape.features)
                                  : make_float2(0.0f, 0.0f);
        const RowFlags flags = row_flags<kMasks>(shape, batch, t0, lane);
        const bool plain = flags.live == (1u << kTileRows) - 1 && flags.cut == 0;
        const int stage = static_cast<int>(step % (kStages > 0 ? kStages : 1));
        if (kTma && have && !dead) {
            const int64_t use = step / (kStages > 0 ? kStages : 1) - (stage == 0 ? skipped : 0);
            dead = !mbar_wait_bounded(&memory.full[stage], static_cast<uint32_t>(use) & 1, status);
        }
        const T *box = memory.stages + size_t(stage) * 3 * Memory::kBox + warp * kTileRows * kTileFeatures + 2 * lane;

        float2 a[kTileRows], k[kTileRows], g[kTileRows];
        float4 rows = make_float4(1.0f, 1.0f, 0.0f, 0.0f);
        float2 back = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < kTileRows; ++j) {
            float2 p, c;
            if (kTma) {
                p = load_two(box + j * kTileFeatures);
                c = load_two(box + Memory::kBox + j * kTileFeatures);
                g[j] = grad_in != nullptr ? load_two(box + 2 * Memory::kBox + j * kTileFeatures) : make_float2(0.0f, 0.0f);
            } else {
                p = c = g[j] = make_float2(0.0f, 0.0f);
                if (t0 + j < shape.length) {
                    p = features.load(in + (t0 + j) * 2 * shape.features);
                    c = features.load(in + (t0 + j) * 2 * shape.features + shape.features);
                    if (grad_in != nullptr) g[j] = features.load(grad_in + (t0 + j) * shape.features);
                }
            }
            gate_of<T>(p.x, c.x, shape.lo, span, a[j].x, k[j].x);
            gate_of<T>(p.y, c.y, shape.lo, span, a[j].y, k[j].y);
        }
        if (plain) {
#pragma unroll
            for (int j = 0; j < kTileRows; ++j) {
                rows.x *= a[j].x;
                rows.y *= a[j].y;
                rows.z = fmaf(a[j].x, rows.z, fmaf(-a[j].x, k[j].x, k[j].x));
                rows.w = fmaf(a[j].y, rows.w, fmaf(-a[j].y, k[j].y, k[j].y));
            }
#pragma unroll
            for (int j = kTileRows - 1; j >= 0; --j) back = make_float2(a[j].x * (back.x + g[j].x), a[j].y * (back.y + g[j].y));
            rows.x = fmaxf(rows.x, 1.4e-45f);
            rows.y = fmaxf(rows.y, 1.4e-45f);
        } else {
#pragma unroll
            for (int j = 0; j < kTileRows; ++j) {
                if (!(flags.live >> j & 1u)) {
                    a[j] = make_float2(1.0f, 1.0f);
                    k[j] = make_float2(0.0f, 0.0f);
                    if (t0 + j >= shape.length) g[j] = make_float2(0.0f, 0.0f);
                }
                const bool cut = flags.cut >> j & 1u;
                rows = compose(rows, make_float4(cut ? 0.0f : a[j].x, cut ? 0.0f : a[j].y, fmaf(-a[j].x, k[j].x, k[j].x),
                                                 fmaf(-a[j].y, k[j].y, k[j].y)));
            }
#pragma unroll
            for (int j = kTileRows - 1; j >= 0; --j) {
                back = flags.cut >> j & 1u ? make_float2(0.0f, 0.0f)
                                           : make_float2(a[j].x * (back.x + g[j].x), a[j].y * (back.y + g[j].y));
            }
        }
        float4 *warps = memory.warps + parity * kTileWarps * 32 + lane;
        float2 *backs = memory.extra + parity * kTileWarps * 32 + lane;
        warps[warp * 32] = rows;
        backs[warp * 32] = back;
        __syncthreads();
        if (kTma && threadIdx.x == 0 && !dead && step + kStages < waves) issue(step + kStages);

        // the state before this warp's rows
        float2 h = carry;
        for (int w = 0; w < warp; ++w) {
            const float4 m = warps[w * 32];
            h = make_float2(apply(m.x, m.z, h.x), apply(m.y, m.w, h.y));
        }
        // x after this warp's rows, and x before the whole wave
        float2 from = x;
        if (cluster > 1) {
            float4 *tiles = memory.cluster + parity * kMaxCluster * 32 + lane;
            if (warp < cluster) {
                float4 total = make_float4(1.0f, 1.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = kTileWarps - 1; w >= 0; --w) {
                    const float4 m = warps[w * 32];
                    const float2 n = backs[w * 32];
                    total = compose(total, make_float4(m.x, m.y, n.x, n.y));
                }
                store_remote(tiles + rank * 32, static_cast<uint32_t>(warp), total);
            }
            cluster_sync();
            for (int r = cluster - 1; r >= 0; --r) {
                if (r == rank) from = x;
                const float4 m = tiles[r * 32];
                x = make_float2(apply(m.x, m.z, x.x), apply(m.y, m.w, x.y));
            }
            for (int w = kTileWarps - 1; w > warp; --w) {
                const float4 m = warps[w * 32];
                const float2 n = backs[w * 32];
                from = make_float2(apply(m.x, n.x, from.x), apply(m.y, n.y, from.y));
            }
        } else {
#pragma unroll
            for (int w = kTileWarps - 1; w >= 0; --w) {
                if (w == warp) from = x;
                const float4 m = warps[w * 32];
                const float2 n = backs[w * 32];
                x = make_float2(apply(m.x, n.x, x.x), apply(m.y, n.y, x.y));
            }
        }
        // Replay: u = (h' - k)(hi - lo) s (1 - s), with (hi - lo) s (1 - s) =
        // (a - lo)(hi - a) / (hi - lo).
        float2 u[kTileRows];
#pragma unroll
        for (int j = 0; j < kTileRows; ++j) {
            if (!plain && (flags.cut >> j & 1u)) h = make_float2(0.0f, 0.0f);
            const float wx = (a[j].x - shape.lo) * (shape.hi - a[j].x) * inverse_span;
            const float wy = (a[j].y - shape.lo) * (shape.hi - a[j].y) * inverse_span;
            u[j] = make_float2((h.x - k[j].x) * wx, (h.y - k[j].y) * wy);
            h = make_float2(fmaf(a[j].x, h.x - k[j].x, k[j].x), fmaf(a[j].y, h.y - k[j].y, k[j].y));
        }
#pragma unroll
        for (int j = kTileRows - 1; j >= 0; --j) {
            const float2 adjoint = make_float2(from.x + g[j].x, from.y + g[j].y);
            float2 dp = make_float2(adjoint.x * u[j].x, adjoint.y * u[j].y);
            float2 dc = make_float2(adjoint.x * ((1.0f - a[j].x) * fmaf(-k[j].x, k[j].x, 1.0f)),
                                    adjoint.y * ((1.0f - a[j].y) * fmaf(-k[j].y, k[j].y, 1.0f)));
            from = make_float2(a[j].x * adjoint.x, a[j].y * adjoint.y);
            if (!plain) {
                if (!(flags.live >> j & 1u)) dp = dc = make_float2(0.0f, 0.0f);
                if (flags.cut >> j & 1u) from = make_float2(0.0f, 0.0f);
            }
            if (t0 + j < shape.length) {
                features.store(grad_out + (t0 + j) * 2 * shape.features, dp);
                features.store(grad_out + (t0 + j) * 2 * shape.features + shape.features, dc);
            }
        }
    }
    if (grad_initial != nullptr && rank == 0 && warp == 0) features.store_side(grad_initial + batch * shape.features, x);
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

// CTAs per chain: as many as fill the GPU (`resident` CTAs per SM), up to 8
// and to the number of tiles.
int cluster_size(const GatedShape &shape, int64_t chains, int resident) {
    int cluster = 1;
    while (cluster < kMaxCluster && chains * cluster < int64_t(resident) * sm_count() && 2 * cluster <= shape.segments) cluster *= 2;
    return cluster;
}

template <typename... KernelArgs, typename... Args>
int launch_tiles(void (*kernel)(KernelArgs...), int64_t chains, int cluster, size_t smem, cudaStream_t stream, Args &&...args) {
    if (chains * cluster >= (int64_t(1) << 31)) return fail(KOEMI_ERR_UNSUPPORTED, "the recurrence has too many lanes");
    KOEMI_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    KOEMI_CUDA_TRY(launch_programmatic(false, kernel, dim3(static_cast<unsigned>(chains * cluster)), dim3(kTileThreads), smem,
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
    const int cluster = cluster_size(shape, chains, 3);
    const bool masks = shape.valid != nullptr || shape.restart != nullptr;
    int *status = device_status_word();
    CUtensorMap map{};
    auto go = [&](auto kernel, bool tma) {
        return launch_tiles(kernel, chains, cluster, TileMemory<T, 2, forward_stages<T>()>::bytes(tma), stream, map, shape,
                            feature_tiles, cluster, in, initial, out, final_state, carries, status);
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
    const int cluster = cluster_size(shape, chains, 2);
    const bool masks = shape.valid != nullptr || shape.restart != nullptr;
    int *status = device_status_word();
    CUtensorMap map{}, grad_map{};
    auto go = [&](auto kernel, bool tma) {
        return launch_tiles(kernel, chains, cluster, TileMemory<T, 3, backward_stages<T>()>::bytes(tma), stream, map, grad_map,
                            shape, feature_tiles, cluster, in, carries, grad, grad_final, out, grad_initial, status);
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
