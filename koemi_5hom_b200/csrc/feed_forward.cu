// The gated feed-forward block, forward and backward, on tcgen05 tensor cores:
//
//   p = x Wg^T + bg, q = x Wv^T + bv, h = silu(p) q, y = h Wo^T + bo;
//   dh = dy Wo, dq = dh silu(p), dp = dh q s (1 + p (1 - s)), s = sigmoid(p),
//   dx = dp Wg + dq Wv, dWg = dp^T x, dWv = dq^T x, dWo = dy^T h, and the
//   biases' gradients are the column sums of dp, dq and dy.
//
// One matrix product kernel with three epilogues:
//   kGate   p and q of the same hidden units side by side in one accumulator,
//           h from both (and p, q for the backward): both projections, the
//           activation and the product in one pass over x;
//   kInner  dh, and from it, p and q, dp and dq (dh is never stored);
//   kOut    the plain product, with a bias or without.
// Its operands are row-major matrices of 16-bit values read by TMA, each with K
// along its rows (K-major) or down its columns (MN-major): the transposed
// products of the backward need no transposed copy.
//
// fp32 values are split into three bf16 parts (8 bits each, together the 24 of
// fp32), x = x0 + x1 + x2 with |x1| <= 2^-9 |x0|, |x2| <= 2^-18 |x0|, and a
// product is the six part products that matter, added up smallest first in the
// same fp32 accumulator: x0 y2, x2 y0, x1 y1, x0 y1, x1 y0, x0 y0. What is left
// out is below 2^-26 of |x y|. Six bf16 products run several times faster than
// fp32 FMAs. 16-bit operands whose rows TMA cannot describe (a width that is no
// multiple of 8, a start off 16 bytes) are copied to padded rows first.
//
// In 16 bits h, p, q, dp and dq are rounded to the type between two products
// (h, dp and dq because the tensor cores take no wider operand, p and q because
// their 32 bits would cost the backward twice the bytes); all sums are fp32.
#include <algorithm>

#include "umma.cuh"
#include "vec.cuh"

namespace koemi {
namespace {

constexpr int kBM = 128;  // accumulator rows of a CTA
constexpr int kBK = 64;   // K of a stage: 128 bytes of 16-bit values, the swizzle's span
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = (2 + kEpilogueWarps) * 32;
constexpr uint32_t kABytes = kBM * kBK * 2;
constexpr uint32_t kRingBytes = 192 * 1024;
constexpr int kMaxStages = 8;
// The tensor cores cut off what an fp32 accumulator cannot hold, which 256
// instructions in a row turn into 2e-6 of the result. Where that is too much,
// for fp32 values, the accumulators are added up in registers, rounded to
// nearest, every kPass K blocks (32 instructions).
constexpr int kPass = 8;
constexpr uint32_t kTmemColumns = 512;
constexpr size_t kSmemBytes = 1024 + kRingBytes + 256;
static_assert((2 * kMaxStages + 4) * 8 + 8 <= 256, "barrier area");

enum Epilogue : int { kGate = 0, kInner = 1, kOut = 2 };

// The tensor cores' operand type for values of type T.
template <typename T>
struct Operand16 {
    using type = T;
    static constexpr int kParts = 1;
};
template <>
struct Operand16<float> {
    using type = __nv_bfloat16;
    static constexpr int kParts = 3;
};

// Where an epilogue stores a 16-bit matrix of kParts parts.
struct Parts {
    void *base;
    int64_t ld, part_stride;  // elements
};

struct GemmArgs {
    CUtensorMap a[2], b[2];  // a segment's operands; kGate: b[0] and b[1] are the gate's and the value's weights
    int segments;            // D = sum over segments of A B
    int k_blocks[2];         // K blocks of a segment
    int pairs;               // part products: 1 or 6
    int a_mn, b_mn;          // MN-major operands
    int64_t m, n;            // rows and columns of the result (kGate: hidden units)
    int m_tiles, n_tiles, splits, band;
    int total_k, k_per_split;
    const void *bias0, *bias1;
    void *out;               // kOut
    int64_t ld_out;
    Parts first, second;     // kGate: first = h; kInner: first = dp, second = dq
    void *p, *q;             // kGate: written (NULL: not wanted); kInner: read
    int64_t ld_pq;
    float *partials;         // splits > 1: raw accumulators [split][gate | value][m][ld_partial]
    int64_t ld_partial;
    int *status;
    uint32_t idesc;
};

// ------------------------------------------------------------------- PTX

__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The address that `local` has in the first CTA of the pair.
__device__ __forceinline__ uint32_t in_leader(uint32_t local) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(local));
    return remote;
}

__device__ __forceinline__ void arrive_leader(uint64_t *bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_leader(smem_addr(bar))) : "memory");
}

template <int kCtas>
__device__ __forceinline__ void load_box(void *dst, const CUtensorMap *map, uint32_t bar, int32_t c0, int32_t c1, int32_t c2) {
    if constexpr (kCtas == 1) {
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_addr(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
            : "memory");
    } else {  // the bytes count on the leader's barrier
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_addr(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
            : "memory");
    }
}

template <int kCtas>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (kCtas == 1) {
        umma_f16(d, a, b, idesc, accumulate);
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
    }
}

// Arrives on the barrier (of both CTAs of a pair) when the MMAs so far are done.
template <int kCtas>
__device__ __forceinline__ void commit(uint64_t *bar) {
    if constexpr (kCtas == 1) {
        umma_commit(bar);
    } else {
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
            "h"(static_cast<uint16_t>(3))
            : "memory");
    }
}

template <bool kCluster>
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, volatile int *abort, int *status) {
    for (uint32_t spin = 0; spin < kWaitSpinLimit; ++spin) {
        if (mbar_try_wait<kCluster>(bar, parity)) return true;
        if ((spin & 255) == 255 && *abort) return false;
    }
    *abort = 1;
    if (status != nullptr) atomicExch(status, KOEMI_ERR_TIMEOUT);
    return false;
}

// -------------------------------------------------------------- scheduling

struct Tile {
    int m, n, split, k_begin, k_end;
};

// Bands of `band` row tiles, columns walked inside a band: the tiles that run
// together share their operands' tiles in L2.
__device__ __forceinline__ Tile tile_at(const GemmArgs &a, int t) {
    Tile tile;
    const int per_split = a.m_tiles * a.n_tiles;
    tile.split = t / per_split;
    t -= tile.split * per_split;
    const int per_band = a.band * a.n_tiles;
    const int band = t / per_band, inside = t - band * per_band;
    const int rows = min(a.band, a.m_tiles - band * a.band);
    tile.n = inside / rows;
    tile.m = band * a.band + (inside - tile.n * rows);
    tile.k_begin = tile.split * a.k_per_split;
    tile.k_end = min(a.total_k, tile.k_begin + a.k_per_split);
    return tile;
}

// K block `kb` of all: its segment, the parts of A and B, and its block there.
struct Block {
    int segment, a_part, b_part, k;
};
__device__ __forceinline__ Block block_at(const GemmArgs &a, int kb) {
    Block b;
    const int first = a.pairs * a.k_blocks[0];
    b.segment = kb >= first;
    if (b.segment) kb -= first;
    const int pair = kb / a.k_blocks[b.segment];
    b.k = kb - pair * a.k_blocks[b.segment];
    // the six pairs of parts, smallest products first: (0 2) (2 0) (1 1) (0 1) (1 0) (0 0)
    b.a_part = a.pairs == 1 ? 0 : (0x021010 >> (4 * (5 - pair))) & 3;
    b.b_part = a.pairs == 1 ? 0 : (0x201100 >> (4 * (5 - pair))) & 3;
    return b;
}

// ---------------------------------------------------------------- epilogues

// kWide values from column c of a row-major matrix, zeros from `left` on.
template <int kWide, typename T>
__device__ __forceinline__ void load_values(const T *src, int64_t left, float (&out)[kWide]) {
    constexpr int W = Pack<T>::kWidth;
    if (left >= kWide && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
#pragma unroll
        for (int q = 0; q < kWide / W; ++q) {
            float part[W];
            unpack(load_cached(src + q * W), part, T());
#pragma unroll
            for (int e = 0; e < W; ++e) out[q * W + e] = part[e];
        }
    } else {
#pragma unroll
        for (int j = 0; j < kWide; ++j) out[j] = j < left ? to_acc(src[j]) : 0.0f;
    }
}

template <int kWide, typename T>
__device__ __forceinline__ void store_values(T *dst, int64_t left, const float (&in)[kWide]) {
    constexpr int W = Pack<T>::kWidth;
    if (left >= kWide && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
        for (int q = 0; q < kWide / W; ++q) {
            float part[W];
#pragma unroll
            for (int e = 0; e < W; ++e) part[e] = in[q * W + e];
            store_stream(dst + q * W, pack(part, T()));
        }
    } else {
#pragma unroll
        for (int j = 0; j < kWide; ++j) {
            if (j < left) dst[j] = from_acc<T>(in[j]);
        }
    }
}

// The three bf16 parts of a value.
__device__ __forceinline__ void split(float v, float &a, float &b, float &c) {
    a = __bfloat162float(__float2bfloat16_rn(v));
    const float rest = v - a;
    b = __bfloat162float(__float2bfloat16_rn(rest));
    c = rest - b;
}

template <int kWide, typename T>
__device__ __forceinline__ void store_parts(const Parts &to, int64_t row, int64_t column, int64_t left, const float (&in)[kWide]) {
    using E = typename Operand16<T>::type;
    E *dst = static_cast<E *>(to.base) + row * to.ld + column;
    if constexpr (Operand16<T>::kParts == 1) {
        store_values<kWide>(dst, left, in);
    } else {
        float a[kWide], b[kWide], c[kWide];
#pragma unroll
        for (int j = 0; j < kWide; ++j) split(in[j], a[j], b[j], c[j]);
        store_values<kWide>(dst, left, a);
        store_values<kWide>(dst + to.part_stride, left, b);
        store_values<kWide>(dst + 2 * to.part_stride, left, c);
    }
}

// 16-bit results leave room for the fast exponential and quotient (relative error about 1e-6).
template <typename T>
__device__ __forceinline__ float sigmoid_of(float p) {
    if constexpr (sizeof(T) == 4) {
        return 1.0f / (1.0f + expf(-p));
    } else {
        return __fdividef(1.0f, 1.0f + __expf(-p));
    }
}

// kGate on kWide hidden units of one row: p and q without their biases.
template <int kWide, typename T>
__device__ __forceinline__ void finish_gate(const GemmArgs &a, int64_t row, int64_t column, bool live, float (&p)[kWide], float (&q)[kWide]) {
    const int64_t left = a.n - column;
    if (!live || left <= 0) return;
    if (a.bias0 != nullptr) {
        float b[kWide];
        load_values<kWide>(static_cast<const T *>(a.bias0) + column, left, b);
#pragma unroll
        for (int j = 0; j < kWide; ++j) p[j] += b[j];
    }
    if (a.bias1 != nullptr) {
        float b[kWide];
        load_values<kWide>(static_cast<const T *>(a.bias1) + column, left, b);
#pragma unroll
        for (int j = 0; j < kWide; ++j) q[j] += b[j];
    }
    if (a.p != nullptr) {
        store_values<kWide>(static_cast<T *>(a.p) + row * a.ld_pq + column, left, p);
        store_values<kWide>(static_cast<T *>(a.q) + row * a.ld_pq + column, left, q);
    }
#pragma unroll
    for (int j = 0; j < kWide; ++j) q[j] *= p[j] * sigmoid_of<T>(p[j]);
    store_parts<kWide, T>(a.first, row, column, left, q);
}

// kInner on kWide hidden units of one row of dh.
template <int kWide, typename T>
__device__ __forceinline__ void finish_inner(const GemmArgs &a, int64_t row, int64_t column, bool live, float (&dh)[kWide]) {
    const int64_t left = a.n - column;
    if (!live || left <= 0) return;
    float p[kWide], q[kWide];
    load_values<kWide>(static_cast<const T *>(a.p) + row * a.ld_pq + column, left, p);
    load_values<kWide>(static_cast<const T *>(a.q) + row * a.ld_pq + column, left, q);
#pragma unroll
    for (int j = 0; j < kWide; ++j) {
        const float s = sigmoid_of<T>(p[j]);
        q[j] *= dh[j] * (s * fmaf(p[j], 1.0f - s, 1.0f));
        p[j] *= s * dh[j];
    }
    store_parts<kWide, T>(a.first, row, column, left, q);
    store_parts<kWide, T>(a.second, row, column, left, p);
}

template <int kWide, typename T>
__device__ __forceinline__ void finish_out(const GemmArgs &a, int64_t row, int64_t column, bool live, float (&y)[kWide]) {
    const int64_t left = a.n - column;
    if (!live || left <= 0) return;
    if (a.bias0 != nullptr) {
        float b[kWide];
        load_values<kWide>(static_cast<const T *>(a.bias0) + column, left, b);
#pragma unroll
        for (int j = 0; j < kWide; ++j) y[j] += b[j];
    }
    store_values<kWide>(static_cast<T *>(a.out) + row * a.ld_out + column, left, y);
}

// ------------------------------------------------------------------- kernel
//
// Warp 0 loads, warp 1 multiplies, eight warps finish tiles: two per quarter of
// the accumulator's lanes, each on half of its columns. Two accumulators, so a
// tile is finished while the next is multiplied. kCtas = 2: a pair of CTAs
// computes 256 rows with one instruction; each loads its 128 rows of A and half
// of B's columns, so an SM reads a third fewer bytes per product than with a
// 128 x 256 tile of its own. Every wait is bounded; one that gives up raises the
// CTA's abort flag and the status word, and all roles leave.
template <typename T, int kEpilogue, int kTileN, int kCtas>
__global__ __launch_bounds__(kThreads, 1) void gemm_kernel(const __grid_constant__ GemmArgs args) {
    constexpr uint32_t kBBytes = static_cast<uint32_t>(kTileN / kCtas) * kBK * 2;
    constexpr uint32_t kStage = kABytes + kBBytes;
    constexpr int kStages = kRingBytes / kStage < kMaxStages ? kRingBytes / kStage : kMaxStages;
    constexpr int kUnits = kEpilogue == kGate ? kTileN / 2 : kTileN;  // result columns of a tile
    constexpr bool kPasses = sizeof(T) == 4;
    static_assert(!kPasses || kTileN <= 128, "an epilogue thread holds 64 sums");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    uint64_t *full = reinterpret_cast<uint64_t *>(ring + kRingBytes);
    uint64_t *empty = full + kMaxStages;
    uint64_t *acc_full = empty + kMaxStages;
    uint64_t *acc_empty = acc_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = kCtas == 1 ? 0 : static_cast<int>(cta_rank());
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], kEpilogueWarps * kCtas);
        }
        *abort = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        if constexpr (kCtas == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(kTmemColumns));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(kTmemColumns));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (kCtas == 2) cluster_sync();  // the pair's barriers are set up
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int tiles = args.m_tiles * args.n_tiles * args.splits;
    const int first_tile = blockIdx.x / kCtas, step = gridDim.x / kCtas;

    if (warp == 0) {
        if (lane == 0) {
            for (int s = 0; s < args.segments; ++s) {
                prefetch_tensor_map(&args.a[s]);
                prefetch_tensor_map(&args.b[s]);
            }
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = first_tile; t < tiles && ok; t += step) {
                const Tile tile = tile_at(args, t);
                const int32_t row = (tile.m * kCtas + rank) * kBM;
                for (int kb = tile.k_begin; kb < tile.k_end; ++kb) {
                    ok = wait<kCtas == 2>(&empty[stage], phase ^ 1, abort, args.status);
                    if (!ok) break;
                    const Block block = block_at(args, kb);
                    const CUtensorMap *ma = &args.a[block.segment], *mb = &args.b[block.segment];
                    uint8_t *to_a = ring + stage * kStage, *to_b = to_a + kABytes;
                    const uint32_t bar = kCtas == 1 ? smem_addr(&full[stage]) : in_leader(smem_addr(&full[stage]));
                    if (rank == 0) mbar_arrive_expect_tx(&full[stage], kStage * kCtas);
                    const int32_t k = block.k * kBK;
                    if (args.a_mn) {
                        load_box<kCtas>(to_a, ma, bar, row, k, block.a_part);
                        load_box<kCtas>(to_a + kABytes / 2, ma, bar, row + 64, k, block.a_part);
                    } else {
                        load_box<kCtas>(to_a, ma, bar, k, row, block.a_part);
                    }
                    if constexpr (kEpilogue == kGate) {  // K-major: the units' gate rows, then their value rows
                        const int32_t unit = tile.n * kUnits;
                        if constexpr (kCtas == 1) {
                            load_box<1>(to_b, &args.b[0], bar, k, unit, block.b_part);
                            load_box<1>(to_b + kBBytes / 2, &args.b[1], bar, k, unit, block.b_part);
                        } else {
                            load_box<2>(to_b, &args.b[rank], bar, k, unit, block.b_part);
                        }
                    } else {
                        const int32_t column = tile.n * kTileN + rank * (kTileN / kCtas);
                        if (args.b_mn) {
#pragma unroll
                            for (int c = 0; c < kTileN / kCtas / 64; ++c) {
                                load_box<kCtas>(to_b + c * 8192, mb, bar, column + 64 * c, k, block.b_part);
                            }
                        } else {
                            load_box<kCtas>(to_b, mb, bar, k, column, block.b_part);
                        }
                    }
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            if (*abort && rank == 0) {  // copies still under way land before the CTA ends
                for (int s = 0; s < kStages; ++s) {
                    for (uint32_t spin = 0; spin < (1u << 16) && !mbar_try_wait<kCtas == 2>(&full[s], s < stage ? phase : phase ^ 1); ++spin) {
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            auto full_accumulator = [&] {
                commit<kCtas>(&acc_full[acc]);
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1;
                }
            };
            for (int t = first_tile; t < tiles && ok; t += step) {
                const Tile tile = tile_at(args, t);
                uint32_t d = 0;
                for (int kb = tile.k_begin; kb < tile.k_end; ++kb) {
                    const bool fresh = kb == tile.k_begin || (kPasses && (kb - tile.k_begin) % kPass == 0);
                    if (fresh) {
                        if (kb > tile.k_begin) full_accumulator();
                        ok = wait<kCtas == 2>(&acc_empty[acc], acc_phase ^ 1, abort, args.status);
                        if (!ok) break;
                        tc_fence_after();
                        d = tmem + static_cast<uint32_t>(acc * kTileN);
                    }
                    ok = wait<kCtas == 2>(&full[stage], phase, abort, args.status);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t at_a = smem_addr(ring + stage * kStage), at_b = at_a + kABytes;
                    const uint64_t da = args.a_mn ? sw128_mnmajor_desc(at_a) : sw128_kmajor_desc(at_a);
                    const uint64_t db = args.b_mn ? sw128_mnmajor_desc(at_b) : sw128_kmajor_desc(at_b);
                    // 16 of K: 16 rows of 128 bytes, or 32 bytes of every row (addresses count 16 bytes)
                    const uint64_t step_a = args.a_mn ? 2048 >> 4 : 32 >> 4, step_b = args.b_mn ? 2048 >> 4 : 32 >> 4;
#pragma unroll
                    for (int k = 0; k < kBK / 16; ++k) {
                        mma<kCtas>(d, da + k * step_a, db + k * step_b, args.idesc, !fresh || k > 0);
                    }
                    commit<kCtas>(&empty[stage]);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (ok) full_accumulator();
            }
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, part = (warp - 2) >> 2;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        auto release = [&] {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (kCtas == 1) {
                    mbar_arrive(&acc_empty[acc]);
                } else {
                    arrive_leader(&acc_empty[acc]);
                }
            }
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1;
            }
        };
        for (int t = first_tile; t < tiles && ok; t += step) {
            const Tile tile = tile_at(args, t);
            const int64_t row = static_cast<int64_t>(tile.m * kCtas + rank) * kBM + quarter * 32 + lane;
            const bool live = row < args.m;
            const int64_t first_column = static_cast<int64_t>(tile.n) * kUnits;
            constexpr int kChunks = kUnits / 32, kSides = kEpilogue == kGate ? 2 : 1;
            // 32 columns of one row (kGate: of p and of q)
            auto finish = [&](int c, float (&v)[kSides][32]) {
                const int64_t column = first_column + c * 32;
                if (args.splits > 1) {
                    if (!live || column >= args.n) return;
                    float *dst = args.partials + (kSides * tile.split * args.m + row) * args.ld_partial + column;
#pragma unroll
                    for (int k = 0; k < kSides; ++k) store_values<32>(dst + k * args.m * args.ld_partial, args.n - column, v[k]);
                } else if constexpr (kEpilogue == kGate) {
                    finish_gate<32, T>(args, row, column, live, v[0], v[1]);
                } else if constexpr (kEpilogue == kInner) {
                    finish_inner<32, T>(args, row, column, live, v[0]);
                } else {
                    finish_out<32, T>(args, row, column, live, v[0]);
                }
            };
            if constexpr (kPasses) {
                constexpr int kMine = (kChunks + 1) / 2;
                float sum[kMine][kSides][32];
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
#pragma unroll
                    for (int k = 0; k < kSides; ++k) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) sum[i][k][j] = 0.0f;
                    }
                }
                for (int kb = tile.k_begin; kb < tile.k_end; kb += kPass) {
                    ok = wait<kCtas == 2>(&acc_full[acc], acc_phase, abort, args.status);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t from = tmem + lanes + static_cast<uint32_t>(acc * kTileN);
#pragma unroll
                    for (int i = 0; i < kMine; ++i) {
                        const int c = part + 2 * i;
                        if (c >= kChunks) continue;
#pragma unroll
                        for (int k = 0; k < kSides; ++k) {
                            uint32_t raw[32];
                            KOEMI_TMEM_LD32(from + k * kUnits + c * 32, raw);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; ++j) sum[i][k][j] += __uint_as_float(raw[j]);
                        }
                    }
                    release();
                }
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    if (part + 2 * i < kChunks) finish(part + 2 * i, sum[i]);
                }
            } else {
                ok = wait<kCtas == 2>(&acc_full[acc], acc_phase, abort, args.status);
                if (!ok) break;
                tc_fence_after();
                const uint32_t from = tmem + lanes + static_cast<uint32_t>(acc * kTileN);
#pragma unroll 1
                for (int c = part; c < kChunks; c += 2) {
                    uint32_t raw[kSides][32];
                    float v[kSides][32];
#pragma unroll
                    for (int k = 0; k < kSides; ++k) KOEMI_TMEM_LD32(from + k * kUnits + c * 32, raw[k]);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < kSides; ++k) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[k][j] = __uint_as_float(raw[k][j]);
                    }
                    finish(c, v);
                }
                release();
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (kCtas == 2) cluster_sync();  // no arrival reaches a CTA that has ended
    if (warp == 1) {
        tc_fence_after();
        if constexpr (kCtas == 1) {
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
        } else {
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
        }
    }
}

// The splits' accumulators added in order, then the epilogue: 8 columns a thread.
template <typename T, int kEpilogue>
__global__ __launch_bounds__(256) void join_kernel(const __grid_constant__ GemmArgs args) {
    const int64_t groups = (args.n + 7) / 8;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= groups * args.m) return;
    const int64_t row = i / groups, column = (i - row * groups) * 8;
    constexpr int kSides = kEpilogue == kGate ? 2 : 1;
    const int64_t side = args.m * args.ld_partial;
    const float *src = args.partials + row * args.ld_partial + column;
    float sum[kSides][8] = {};
    for (int s = 0; s < args.splits; ++s, src += kSides * side) {
#pragma unroll
        for (int k = 0; k < kSides; ++k) {
            float v[8];
            load_values<8>(src + k * side, 8, v);  // ld_partial is a multiple of 8
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[k][e] += v[e];
        }
    }
    if constexpr (kEpilogue == kGate) {
        finish_gate<8, T>(args, row, column, true, sum[0], sum[1]);
    } else if constexpr (kEpilogue == kInner) {
        finish_inner<8, T>(args, row, column, true, sum[0]);
    } else {
        finish_out<8, T>(args, row, column, true, sum[0]);
    }
}

// ------------------------------------------------------------ packed operands

struct PackJob {
    const void *src;
    int64_t rows, columns, ld;
    Parts to;
};
constexpr int kMaxJobs = 5;
struct PackArgs {
    PackJob jobs[kMaxJobs];
};

// Row-major matrices copied (fp32: split) to rows of a multiple of 8 columns, zeros behind the last. grid.y: the matrix.
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(const __grid_constant__ PackArgs args) {
    const PackJob &job = args.jobs[blockIdx.y];
    const int64_t groups = job.to.ld / 8, count = groups * job.rows;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = i / groups, column = (i - row * groups) * 8;
        float v[8];
        load_values<8>(static_cast<const T *>(job.src) + row * job.ld + column, job.columns - column, v);
        store_parts<8, T>(job.to, row, column, 8, v);
    }
}

// -------------------------------------------------------------- column sums

struct SumJob {
    const void *src;
    int64_t columns, ld, part_stride;
    int parts;   // 0: values of type T
    void *out;
};
struct SumArgs {
    SumJob jobs[3];
    int64_t rows, chunk;  // rows of a chunk
    int chunks;
    float *partials;      // [job][chunk][most columns]
    int64_t ld;
};

// grid (columns / 32, chunks, jobs): 32 columns, the chunk's rows over 8 warps.
template <typename T>
__global__ __launch_bounds__(256) void column_sums_kernel(const __grid_constant__ SumArgs args) {
    using E = typename Operand16<T>::type;
    __shared__ float parts[8][33];
    const SumJob &job = args.jobs[blockIdx.z];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t column = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    if (job.out == nullptr || static_cast<int64_t>(blockIdx.x) * 32 >= job.columns) return;
    const int64_t begin = blockIdx.y * args.chunk, end = min(args.rows, begin + args.chunk);
    float sum = 0.0f;
    if (column < job.columns) {
        if (job.parts == 0) {
            const T *src = static_cast<const T *>(job.src) + column;
#pragma unroll 4
            for (int64_t r = begin + warp; r < end; r += 8) sum += to_acc(src[r * job.ld]);
        } else {
            const E *src = static_cast<const E *>(job.src) + column;
#pragma unroll 4
            for (int64_t r = begin + warp; r < end; r += 8) {
                float v = to_acc(src[r * job.ld]);
                if (job.parts == 3) v += to_acc(src[r * job.ld + job.part_stride]) + to_acc(src[r * job.ld + 2 * job.part_stride]);
                sum += v;
            }
        }
    }
    parts[warp][lane] = sum;
    __syncthreads();
    if (warp != 0 || column >= job.columns) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) sum += parts[w][lane];
    args.partials[(blockIdx.z * args.chunks + blockIdx.y) * args.ld + column] = sum;
}

template <typename T>
__global__ __launch_bounds__(128) void column_totals_kernel(const __grid_constant__ SumArgs args) {
    const SumJob &job = args.jobs[blockIdx.y];
    const int64_t column = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
    if (job.out == nullptr || column >= job.columns) return;
    const float *src = args.partials + blockIdx.y * args.chunks * args.ld + column;
    float sum = 0.0f;
#pragma unroll 8
    for (int c = 0; c < args.chunks; ++c) sum += src[c * args.ld];
    static_cast<T *>(job.out)[column] = from_acc<T>(sum);
}

// --------------------------------------------------------------------- host

// A row-major 16-bit operand as TMA reads it.
struct Matrix {
    const void *base;
    int64_t rows, columns, ld, part_stride;
    int parts;
};

int64_t round8(int64_t v) { return (v + 7) / 8 * 8; }
size_t round256(size_t v) { return (v + 255) & ~size_t(255); }

int encode(CUtensorMap *map, const Matrix &matrix, bool half, bool mn_major, int box_rows) {
    const CUtensorMapDataType type = half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const uint64_t dims[3] = {static_cast<uint64_t>(matrix.columns), static_cast<uint64_t>(matrix.rows), static_cast<uint64_t>(matrix.parts)};
    const uint64_t part = static_cast<uint64_t>(matrix.parts > 1 ? matrix.part_stride : matrix.ld) * 2;
    const uint64_t strides[2] = {static_cast<uint64_t>(matrix.ld) * 2, part};
    const uint32_t box[3] = {64, mn_major ? 64u : static_cast<uint32_t>(box_rows), 1};
    return encode_tensor_map(map, type, 3, matrix.base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// How a product is cut: tile columns, CTAs a tile, parts of K.
struct Cut {
    int tile_n, ctas, splits;
};

// The cheapest of the cuts by clocks: an SM takes about 52 bytes a clock from
// L2 (measured with all SMs loading: 128 x 256 tiles 51, 128 x 128 tiles 53),
// which is what a K block of every shape but a pair's 256 x 256 waits for; a
// launch adds about 6500 for its first loads and its last epilogue; parts of K
// add a kernel and their accumulators' way through L2.
Cut cut_of(int64_t m, int64_t n, int total_k, bool gate, int parts, int sms) {
    Cut best{128, 1, 1};
    double least = 1e30;
    const struct { int tile_n, ctas; } shapes[] = {{256, 2}, {128, 2}, {256, 1}, {128, 1}, {64, 1}};
    for (const auto &shape : shapes) {
        if (parts > 1 && shape.tile_n > 128) continue;  // the sums of the passes have to fit registers
        if (shape.ctas == 2 && m <= kBM) continue;
        const double clocks = std::max(shape.tile_n * 2.0, (kBM + shape.tile_n / shape.ctas) * kBK * 2 / 52.0);
        const int64_t units = gate ? shape.tile_n / 2 : shape.tile_n;
        const int64_t tiles = ceil_div(m, kBM * shape.ctas) * ceil_div(n, units), places = std::max(1, sms / shape.ctas);
        for (int splits = 1; splits <= 64 && splits <= total_k; splits += splits < 8 ? 1 : splits / 4) {
            const int per = static_cast<int>(ceil_div(total_k, splits));
            if (ceil_div(total_k, per) != splits) continue;  // every part has blocks
            const double waves = static_cast<double>(ceil_div(tiles * splits, places));
            double cost = waves * per * clocks + 6500;
            if (splits > 1) cost += 6000 + (gate ? 2.0 : 1.0) * static_cast<double>(m) * static_cast<double>(n) * (splits + 1) * 4 / 2500;
            if (cost < least) least = cost, best = Cut{shape.tile_n, shape.ctas, splits};
        }
    }
    return best;
}

size_t partial_bytes(const Cut &cut, int64_t m, int64_t n, bool gate) {
    return cut.splits == 1 ? 0 : static_cast<size_t>(cut.splits) * (gate ? 2 : 1) * m * round8(n) * sizeof(float);
}

template <typename T, int kEpilogue, int kTileN, int kCtas>
int launch_shape(const GemmArgs &args, cudaStream_t stream) {
    auto kernel = gemm_kernel<T, kEpilogue, kTileN, kCtas>;
    KOEMI_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemBytes)));
    const int64_t tiles = static_cast<int64_t>(args.m_tiles) * args.n_tiles * args.splits;
    if (tiles > INT32_MAX) return fail(KOEMI_ERR_INVALID, "feed-forward sizes are too large");
    const int64_t grid = std::min<int64_t>(tiles, sm_count() / kCtas) * kCtas;
    KOEMI_CUDA_TRY(launch_programmatic(false, kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), kSmemBytes, stream, dim3(kCtas, 1, 1), args));
    return KOEMI_OK;
}

// One product: A and B of up to two segments (kGate: one A, B the two weights).
struct Product {
    Matrix a[2], b[2];
    int segments;
    bool a_mn, b_mn;
    int64_t m, n;
};

int total_k_of(const Product &p, bool gate) {
    const int pairs = p.a[0].parts == 3 ? 6 : 1;
    int64_t blocks = 0;
    for (int s = 0; s < (gate ? 1 : p.segments); ++s) blocks += ceil_div(p.a_mn ? p.a[s].rows : p.a[s].columns, kBK);
    return static_cast<int>(blocks * pairs);
}

template <typename T, int kEpilogue>
int multiply(const Product &p, GemmArgs args, float *partials, cudaStream_t stream) {
    constexpr bool gate = kEpilogue == kGate;
    const bool half = std::is_same<typename Operand16<T>::type, __half>::value;
    const int total_k = total_k_of(p, gate);
    const Cut cut = cut_of(p.m, p.n, total_k, gate, p.a[0].parts, sm_count());
    args.segments = gate ? 2 : p.segments;
    args.pairs = p.a[0].parts == 3 ? 6 : 1;
    args.a_mn = p.a_mn;
    args.b_mn = p.b_mn;
    args.m = p.m;
    args.n = p.n;
    args.m_tiles = static_cast<int>(ceil_div(p.m, kBM * cut.ctas));
    args.n_tiles = static_cast<int>(ceil_div(p.n, gate ? cut.tile_n / 2 : cut.tile_n));
    args.splits = cut.splits;
    args.band = std::max(1, 16 / cut.ctas);
    args.total_k = total_k;
    args.k_per_split = static_cast<int>(ceil_div(total_k, cut.splits));
    args.partials = partials;
    args.ld_partial = round8(p.n);
    args.status = device_status_word();
    args.idesc = 1u << 4 | (half ? 0u : 1u << 7 | 1u << 10) | (p.a_mn ? 1u << 15 : 0u) | (p.b_mn ? 1u << 16 : 0u) |
                 static_cast<uint32_t>(cut.tile_n >> 3) << 17 | static_cast<uint32_t>(kBM * cut.ctas >> 4) << 24;
    for (int s = 0; s < 2; ++s) {
        const Matrix &a = p.a[gate || s >= p.segments ? 0 : s], &b = p.b[gate || s < p.segments ? s : 0];
        args.k_blocks[s] = static_cast<int>(ceil_div(p.a_mn ? a.rows : a.columns, kBK));
        int rc = encode(&args.a[s], a, half, p.a_mn, kBM);
        if (rc == KOEMI_OK) rc = encode(&args.b[s], b, half, p.b_mn, gate ? cut.tile_n / 2 : cut.tile_n / cut.ctas);
        if (rc != KOEMI_OK) return rc;
    }
    int rc = KOEMI_OK;
    if (cut.tile_n == 64) {
        rc = launch_shape<T, kEpilogue, 64, 1>(args, stream);
    } else if (cut.tile_n == 128) {
        rc = cut.ctas == 2 ? launch_shape<T, kEpilogue, 128, 2>(args, stream) : launch_shape<T, kEpilogue, 128, 1>(args, stream);
    } else if constexpr (sizeof(T) == 2) {
        rc = cut.ctas == 2 ? launch_shape<T, kEpilogue, 256, 2>(args, stream) : launch_shape<T, kEpilogue, 256, 1>(args, stream);
    }
    if (rc != KOEMI_OK) return rc;
    if (cut.splits > 1) {
        const int64_t threads = (args.n + 7) / 8 * args.m;
        join_kernel<T, kEpilogue><<<static_cast<unsigned>(ceil_div(threads, 256)), 256, 0, stream>>>(args);
        KOEMI_LAUNCH_CHECK();
    }
    return KOEMI_OK;
}

// Hands out 256-byte aligned parts of a workspace; without one it only counts.
struct Pool {
    char *base;
    size_t used = 0;
    void *take(size_t bytes) {
        void *p = base == nullptr ? nullptr : base + used;
        used += round256(bytes);
        return p;
    }
};

struct Problem {
    const void *x, *wg, *wv, *wo, *bg, *bv, *bo;
    int64_t rows, width, hidden, out_width, ld_x;
    int dtype;
};

int parts_of(int dtype) { return dtype == KOEMI_F32 ? 3 : 1; }

// What the backward needs of the forward: h (in parts), p and q.
struct Kept {
    Parts h;
    void *p, *q;
    int64_t ld;
};

Kept kept_of(Pool &pool, int64_t rows, int64_t hidden, int dtype, bool with_pq) {
    Kept kept{};
    kept.ld = round8(hidden);
    const size_t count = static_cast<size_t>(rows) * kept.ld;
    kept.h = Parts{pool.take(count * 2 * parts_of(dtype)), kept.ld, rows * kept.ld};
    if (with_pq) {
        kept.p = pool.take(count * dtype_size(dtype));
        kept.q = pool.take(count * dtype_size(dtype));
    }
    return kept;
}

// `src` as an operand: itself where TMA reads it, else a packed copy, noted in `jobs`. With counting, the
// base is unknown: it asks for room as if the copy were made.
Matrix operand(Pool &pool, const void *src, int64_t rows, int64_t columns, int64_t ld, int dtype, PackArgs &jobs, int &count) {
    if (dtype != KOEMI_F32 && pool.base != nullptr && ld % 8 == 0 && aligned(src, 16)) return Matrix{src, rows, columns, ld, 0, 1};
    const int64_t padded = round8(columns);
    const Parts to{pool.take(static_cast<size_t>(rows) * padded * 2 * parts_of(dtype)), padded, rows * padded};
    jobs.jobs[count++] = PackJob{src, rows, columns, ld, to};
    return Matrix{to.base, rows, columns, padded, to.part_stride, parts_of(dtype)};
}

Matrix matrix_of(const Parts &parts, int64_t rows, int64_t columns, int dtype) {
    return Matrix{parts.base, rows, columns, parts.ld, parts.part_stride, parts_of(dtype)};
}

template <typename T>
int pack_all(const PackArgs &jobs, int count, cudaStream_t stream) {
    if (count == 0) return KOEMI_OK;
    int64_t most = 1;
    for (int j = 0; j < count; ++j) most = std::max(most, jobs.jobs[j].rows * jobs.jobs[j].to.ld / 8);
    const int64_t blocks = std::min<int64_t>(ceil_div(most, 256), 16 * sm_count());
    pack_kernel<T><<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(count)), 256, 0, stream>>>(jobs);
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

struct ForwardPlan {
    Matrix x, wg, wv, wo;
    Kept kept;
    PackArgs jobs;
    int job_count;
    Product gate, out;
    float *partials;
};

// pool: the workspace; kept_base: the buffer that the backward will read, or NULL.
void plan_forward(ForwardPlan &plan, const Problem &q, Pool &pool, char *kept_base, bool keep) {
    plan.job_count = 0;
    plan.x = operand(pool, q.x, q.rows, q.width, q.ld_x, q.dtype, plan.jobs, plan.job_count);
    plan.wg = operand(pool, q.wg, q.hidden, q.width, q.width, q.dtype, plan.jobs, plan.job_count);
    plan.wv = operand(pool, q.wv, q.hidden, q.width, q.width, q.dtype, plan.jobs, plan.job_count);
    plan.wo = operand(pool, q.wo, q.out_width, q.hidden, q.hidden, q.dtype, plan.jobs, plan.job_count);
    Pool kept_pool{kept_base};
    plan.kept = keep ? kept_of(kept_pool, q.rows, q.hidden, q.dtype, true) : kept_of(pool, q.rows, q.hidden, q.dtype, false);
    plan.gate = Product{{plan.x, {}}, {plan.wg, plan.wv}, 1, false, false, q.rows, q.hidden};
    plan.out = Product{{matrix_of(plan.kept.h, q.rows, q.hidden, q.dtype), {}}, {plan.wo, {}}, 1, false, false, q.rows, q.out_width};
    const int sms = sm_count();
    const size_t first = partial_bytes(cut_of(q.rows, q.hidden, total_k_of(plan.gate, true), true, parts_of(q.dtype), sms), q.rows, q.hidden, true);
    const size_t second = partial_bytes(cut_of(q.rows, q.out_width, total_k_of(plan.out, false), false, parts_of(q.dtype), sms), q.rows, q.out_width, false);
    plan.partials = static_cast<float *>(pool.take(std::max(first, second)));
}

template <typename T>
int forward(const Problem &q, void *y, void *kept, void *workspace, cudaStream_t stream) {
    ForwardPlan plan{};
    Pool pool{static_cast<char *>(workspace)};
    plan_forward(plan, q, pool, static_cast<char *>(kept), kept != nullptr);
    int rc = pack_all<T>(plan.jobs, plan.job_count, stream);
    if (rc != KOEMI_OK) return rc;
    GemmArgs gate{};
    gate.bias0 = q.bg;
    gate.bias1 = q.bv;
    gate.first = plan.kept.h;
    gate.p = plan.kept.p;
    gate.q = plan.kept.q;
    gate.ld_pq = plan.kept.ld;
    rc = multiply<T, kGate>(plan.gate, gate, plan.partials, stream);
    if (rc != KOEMI_OK) return rc;
    GemmArgs out{};
    out.bias0 = q.bo;
    out.out = y;
    out.ld_out = q.out_width;
    return multiply<T, kOut>(plan.out, out, plan.partials, stream);
}

struct Gradients {
    const void *dy;
    void *dx, *dwg, *dwv, *dwo, *dbg, *dbv, *dbo;
};

struct BackwardPlan {
    Matrix x, wg, wv, wo, dy;
    Kept kept;
    Parts dp, dq;
    PackArgs jobs;
    int job_count;
    Product inner, values, gate_weight, value_weight, output_weight;
    SumArgs sums;
    float *partials;
};

void plan_backward(BackwardPlan &plan, const Problem &q, const Gradients &g, Pool &pool, char *kept_base) {
    plan.job_count = 0;
    Pool kept_pool{kept_base};
    plan.kept = kept_of(kept_pool, q.rows, q.hidden, q.dtype, true);
    plan.dy = operand(pool, g.dy, q.rows, q.out_width, q.out_width, q.dtype, plan.jobs, plan.job_count);
    plan.x = operand(pool, q.x, q.rows, q.width, q.ld_x, q.dtype, plan.jobs, plan.job_count);
    plan.wg = operand(pool, q.wg, q.hidden, q.width, q.width, q.dtype, plan.jobs, plan.job_count);
    plan.wv = operand(pool, q.wv, q.hidden, q.width, q.width, q.dtype, plan.jobs, plan.job_count);
    plan.wo = operand(pool, q.wo, q.out_width, q.hidden, q.hidden, q.dtype, plan.jobs, plan.job_count);
    const int64_t ld = round8(q.hidden);
    const size_t bytes = static_cast<size_t>(q.rows) * ld * 2 * parts_of(q.dtype);
    plan.dp = Parts{pool.take(bytes), ld, q.rows * ld};
    plan.dq = Parts{pool.take(bytes), ld, q.rows * ld};
    const Matrix dp = matrix_of(plan.dp, q.rows, q.hidden, q.dtype), dq = matrix_of(plan.dq, q.rows, q.hidden, q.dtype);
    plan.inner = Product{{plan.dy, {}}, {plan.wo, {}}, 1, false, true, q.rows, q.hidden};
    plan.values = Product{{dp, dq}, {plan.wg, plan.wv}, 2, false, true, q.rows, q.width};
    plan.gate_weight = Product{{dp, {}}, {plan.x, {}}, 1, true, true, q.hidden, q.width};
    plan.value_weight = Product{{dq, {}}, {plan.x, {}}, 1, true, true, q.hidden, q.width};
    plan.output_weight = Product{{plan.dy, {}}, {matrix_of(plan.kept.h, q.rows, q.hidden, q.dtype), {}}, 1, true, true, q.out_width, q.hidden};
    const int sms = sm_count();
    size_t most = 0;
    for (const Product *p : {&plan.inner, &plan.values, &plan.gate_weight, &plan.value_weight, &plan.output_weight}) {
        most = std::max(most, partial_bytes(cut_of(p->m, p->n, total_k_of(*p, false), false, parts_of(q.dtype), sms), p->m, p->n, false));
    }
    plan.partials = static_cast<float *>(pool.take(most));
    const int64_t columns = std::max(q.hidden, q.out_width);
    plan.sums.rows = q.rows;
    plan.sums.chunks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ceil_div(q.rows, 64), 16 * sms / ceil_div(columns, 32))));
    plan.sums.chunk = ceil_div(q.rows, plan.sums.chunks);
    plan.sums.ld = columns;
    plan.sums.partials = static_cast<float *>(pool.take(static_cast<size_t>(3) * plan.sums.chunks * columns * sizeof(float)));
    const int parts = parts_of(q.dtype);
    plan.sums.jobs[0] = SumJob{plan.dp.base, q.hidden, ld, plan.dp.part_stride, parts, g.dbg};
    plan.sums.jobs[1] = SumJob{plan.dq.base, q.hidden, ld, plan.dq.part_stride, parts, g.dbv};
    plan.sums.jobs[2] = SumJob{g.dy, q.out_width, q.out_width, 0, 0, g.dbo};
}

template <typename T>
int backward(const Problem &q, const Gradients &g, const void *kept, void *workspace, cudaStream_t stream) {
    BackwardPlan plan{};
    Pool pool{static_cast<char *>(workspace)};
    plan_backward(plan, q, g, pool, static_cast<char *>(const_cast<void *>(kept)));
    int rc = pack_all<T>(plan.jobs, plan.job_count, stream);
    if (rc != KOEMI_OK) return rc;
    auto plain = [&](const Product &product, void *out) -> int {
        if (out == nullptr) return KOEMI_OK;
        GemmArgs args{};
        args.out = out;
        args.ld_out = product.n;
        return multiply<T, kOut>(product, args, plan.partials, stream);
    };
    if (g.dx != nullptr || g.dwg != nullptr || g.dwv != nullptr || g.dbg != nullptr || g.dbv != nullptr) {
        GemmArgs inner{};
        inner.first = plan.dp;
        inner.second = plan.dq;
        inner.p = plan.kept.p;
        inner.q = plan.kept.q;
        inner.ld_pq = plan.kept.ld;
        rc = multiply<T, kInner>(plan.inner, inner, plan.partials, stream);
    }
    if (rc == KOEMI_OK) rc = plain(plan.values, g.dx);
    if (rc == KOEMI_OK) rc = plain(plan.gate_weight, g.dwg);
    if (rc == KOEMI_OK) rc = plain(plan.value_weight, g.dwv);
    if (rc == KOEMI_OK) rc = plain(plan.output_weight, g.dwo);
    if (rc != KOEMI_OK) return rc;
    if (g.dbg != nullptr || g.dbv != nullptr || g.dbo != nullptr) {
        const unsigned columns = static_cast<unsigned>(plan.sums.ld);
        column_sums_kernel<T><<<dim3((columns + 31) / 32, plan.sums.chunks, 3), 256, 0, stream>>>(plan.sums);
        column_totals_kernel<T><<<dim3((columns + 127) / 128, 3), 128, 0, stream>>>(plan.sums);
        KOEMI_LAUNCH_CHECK();
    }
    return KOEMI_OK;
}

int check(int64_t rows, int64_t width, int64_t hidden, int64_t out_width, int dtype) {
    if (rows < 0 || width < 1 || hidden < 1 || out_width < 1) return fail(KOEMI_ERR_INVALID, "bad feed-forward sizes");
    const int64_t most = int64_t(1) << 30;
    if (rows > most || width > (1 << 24) || hidden > (1 << 24) || out_width > (1 << 24)) return fail(KOEMI_ERR_INVALID, "feed-forward sizes are too large");
    if (dtype != KOEMI_F32 && dtype != KOEMI_F16 && dtype != KOEMI_BF16) return fail(KOEMI_ERR_INVALID, "unsupported feed-forward dtype %d", dtype);
    return KOEMI_OK;
}

}  // namespace
}  // namespace koemi

using namespace koemi;

extern "C" size_t koemi_dense_gated_feed_forward_kept(int64_t rows, int64_t hidden_width, int dtype) {
    if (rows < 1 || hidden_width < 1 || dtype_size(dtype) == 0) return 0;
    Pool pool{nullptr};
    kept_of(pool, rows, hidden_width, dtype, true);
    return pool.used;
}

extern "C" size_t koemi_dense_gated_feed_forward_workspace(int64_t rows, int64_t width, int64_t hidden_width, int64_t out_width,
                                                           int dtype, int backward) {
    if (rows < 1 || check(rows, width, hidden_width, out_width, dtype) != KOEMI_OK) return 0;
    const Problem q{nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, rows, width, hidden_width, out_width, width, dtype};
    Pool pool{nullptr};
    if (backward) {
        BackwardPlan plan{};
        plan_backward(plan, q, Gradients{}, pool, nullptr);
    } else {
        ForwardPlan plan{};
        plan_forward(plan, q, pool, nullptr, false);
    }
    return pool.used;
}

extern "C" int koemi_dense_gated_feed_forward_forward(const void *values, int64_t value_stride, const void *gate_weight,
                                                      const void *value_weight, const void *output_weight, const void *gate_bias,
                                                      const void *value_bias, const void *output_bias, void *out, void *kept,
                                                      size_t kept_bytes, int64_t rows, int64_t width, int64_t hidden_width,
                                                      int64_t out_width, int dtype, void *workspace, size_t workspace_bytes,
                                                      void *stream) {
    clear_error();
    const int rc = check(rows, width, hidden_width, out_width, dtype);
    if (rc != KOEMI_OK) return rc;
    if (value_stride < width) return fail(KOEMI_ERR_INVALID, "value_stride must be at least the width");
    if (rows == 0) return KOEMI_OK;
    if (values == nullptr || gate_weight == nullptr || value_weight == nullptr || output_weight == nullptr || out == nullptr) {
        return fail(KOEMI_ERR_INVALID, "values, weights and out must be non-NULL");
    }
    if (kept != nullptr && (kept_bytes < koemi_dense_gated_feed_forward_kept(rows, hidden_width, dtype) || !aligned(kept, 256))) {
        return fail(KOEMI_ERR_WORKSPACE, "kept must hold %zu bytes from a multiple of 256", koemi_dense_gated_feed_forward_kept(rows, hidden_width, dtype));
    }
    const size_t need = koemi_dense_gated_feed_forward_workspace(rows, width, hidden_width, out_width, dtype, 0);
    if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256)) {
        return fail(KOEMI_ERR_WORKSPACE, "the feed-forward block needs %zu workspace bytes from a multiple of 256", need);
    }
    const Problem q{values, gate_weight, value_weight, output_weight, gate_bias, value_bias, output_bias, rows, width, hidden_width, out_width, value_stride, dtype};
    if (dtype == KOEMI_F32) return forward<float>(q, out, kept, workspace, as_stream(stream));
    if (dtype == KOEMI_F16) return forward<__half>(q, out, kept, workspace, as_stream(stream));
    return forward<__nv_bfloat16>(q, out, kept, workspace, as_stream(stream));
}

extern "C" int koemi_dense_gated_feed_forward_backward(const void *values, int64_t value_stride, const void *gate_weight,
                                                       const void *value_weight, const void *output_weight, const void *kept,
                                                       size_t kept_bytes, const void *grad_out, void *grad_values,
                                                       void *grad_gate_weight, void *grad_value_weight, void *grad_output_weight,
                                                       void *grad_gate_bias, void *grad_value_bias, void *grad_output_bias,
                                                       int64_t rows, int64_t width, int64_t hidden_width, int64_t out_width,
                                                       int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    const int rc = check(rows, width, hidden_width, out_width, dtype);
    if (rc != KOEMI_OK) return rc;
    if (value_stride < width) return fail(KOEMI_ERR_INVALID, "value_stride must be at least the width");
    if (rows == 0) {  // sums of no rows
        const size_t size = dtype_size(dtype);
        const struct { void *p; int64_t count; } sums[] = {{grad_gate_weight, hidden_width * width}, {grad_value_weight, hidden_width * width},
                                                           {grad_output_weight, out_width * hidden_width}, {grad_gate_bias, hidden_width},
                                                           {grad_value_bias, hidden_width}, {grad_output_bias, out_width}};
        for (const auto &sum : sums) {
            if (sum.p != nullptr) KOEMI_CUDA_TRY(cudaMemsetAsync(sum.p, 0, size * static_cast<size_t>(sum.count), as_stream(stream)));
        }
        return KOEMI_OK;
    }
    if (values == nullptr || gate_weight == nullptr || value_weight == nullptr || output_weight == nullptr || grad_out == nullptr || kept == nullptr) {
        return fail(KOEMI_ERR_INVALID, "values, weights, kept and grad_out must be non-NULL");
    }
    if (kept_bytes < koemi_dense_gated_feed_forward_kept(rows, hidden_width, dtype) || !aligned(kept, 256)) {
        return fail(KOEMI_ERR_WORKSPACE, "kept must hold %zu bytes from a multiple of 256", koemi_dense_gated_feed_forward_kept(rows, hidden_width, dtype));
    }
    const size_t need = koemi_dense_gated_feed_forward_workspace(rows, width, hidden_width, out_width, dtype, 1);
    if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256)) {
        return fail(KOEMI_ERR_WORKSPACE, "the feed-forward block's backward needs %zu workspace bytes from a multiple of 256", need);
    }
    const Problem q{values, gate_weight, value_weight, output_weight, nullptr, nullptr, nullptr, rows, width, hidden_width, out_width, value_stride, dtype};
    const Gradients g{grad_out, grad_values, grad_gate_weight, grad_value_weight, grad_output_weight, grad_gate_bias, grad_value_bias, grad_output_bias};
    if (dtype == KOEMI_F32) return backward<float>(q, g, kept, workspace, as_stream(stream));
    if (dtype == KOEMI_F16) return backward<__half>(q, g, kept, workspace, as_stream(stream));
    return backward<__nv_bfloat16>(q, g, kept, workspace, as_stream(stream));
}
