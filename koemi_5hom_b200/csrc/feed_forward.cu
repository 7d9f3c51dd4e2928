// The gated feed-forward block, forward and backward, on tcgen05 tensor cores:
//
//   p = x Wg^T + bg, q = x Wv^T + bv, h = silu(p) q, y = h Wo^T + bo;
//   dh = dy Wo, dq = dh a, dp = dh b with a = silu(p), b = q s (1 + p (1 - s)), s = sigmoid(p),
//   dx = dp Wg + dq Wv, dWg = dp^T x, dWv = dq^T x, dWo = dy^T h, and the
//   biases' gradients are the column sums of dp, dq and dy.
//
// One matrix product kernel with three epilogues:
//   kGate   p and q of the same hidden units side by side in one accumulator,
//           h from both (and a, b for the backward): both projections, the
//           activation and the product in one pass over x;
//   kInner  dh, and from it dp and dq (dh is never stored);
//   kOut    the plain product, with a bias or without.
// Its operands are row-major matrices of 16-bit values read by TMA, each with K
// along its rows (K-major) or down its columns (MN-major): the transposed
// products of the backward need no transposed copy.
//
// fp32 values are split into three bf16 parts (8 bits each, together the 24 of
// fp32), x = x0 + x1 + x2 with |x1| <= 2^-8 |x0|, |x2| <= 2^-17 |x0|, and a
// product is the six part products that matter, x0 y0, x0 y1, x1 y0, x1 y1, x0 y2
// and x2 y0: x0 y0 in one accumulator, the others, 2^-8 of it and less, in a
// second one, where they are not cut off at the first one's last place. What is
// left out is about 2^-24 of |x y|, one rounding of fp32. Six bf16 products run
// several times faster than fp32 FMAs. 16-bit operands whose rows TMA cannot
// describe (a width that is no multiple of 8, a start off 16 bytes) are copied to
// padded rows first.
//
// In 16 bits h, dp and dq are rounded to the type between two products, because
// the tensor cores take no wider operand; an fp16 entry of dp or dq under 2^-14
// loses digits by that and one under 2^-25 all of them. A result's error is that
// of two roundings, 1.4 times that of one. The few rows' kernel, which could keep
// h wider, rounds it alike, so that a row's result has the same roundings in
// every batch and the backward, which reads that h, belongs to the y returned. The
// biases' gradients sum the dp and dq whose products the weights' gradients are. a
// and b stay fp32: in 16 bits they would cost the gradients two roundings more
// (bf16 3.1e-3 for 2.4e-3 of a gradient's norm). All sums are fp32.
//
// Many rows are bound by the tensor cores: 32768 rows of 2048 -> 4096 -> 2048 in
// bf16 take 805 us for the gate's products, 369 for y, 469 for dh with dp and dq,
// and 1861 for the four products behind them: 4.95 TFLOP at 1.41 PFLOP/s, where a
// plain library product reaches 1.65 in a burst and 1.37 under the power limit.
#include <algorithm>
#include <atomic>

#include "umma.cuh"
#include "vec.cuh"

namespace koemi {
namespace {

constexpr int kBM = 128;  // accumulator rows of a CTA
constexpr int kBK = 64;   // K of a stage: 128 bytes of 16-bit values, the swizzle's span
constexpr int kEpilogueWarps = 8;
constexpr int kLoaders = 2;  // warps that load, every other stage each
constexpr int kThreads = (kLoaders + 1 + kEpilogueWarps) * 32;
constexpr uint32_t kABytes = kBM * kBK * 2;
constexpr uint32_t kRingBytes = 192 * 1024;
constexpr int kMaxStages = 8;
constexpr int kMaxJobs = 4;
// An epilogue warp's staging area: 32 rows of up to 64 bytes, 16 apart so that
// rows written 16 bytes a lane fall into different banks.
constexpr int kStagedRow = 64 + 16;
constexpr uint32_t kStagedBytes = 32 * kStagedRow;
// The tensor cores cut off what an fp32 accumulator cannot hold, which 256
// instructions in a row turn into 2e-6 of the result. Where that is too much,
// for fp32 values, the accumulators are added up in registers, rounded to
// nearest, every kPass K blocks (32 instructions on x0 y0).
constexpr int kPass = 8;
constexpr uint32_t kBiasBytes = 128 * sizeof(float);  // an epilogue warp's columns' biases
constexpr uint32_t kTmemColumns = 512;
constexpr size_t kSmemBytes = 1024 + kRingBytes + kEpilogueWarps * (kStagedBytes + kBiasBytes) + 256;
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

// Division by a number that the host knows, of values below 2^31.
struct Divisor {
    uint32_t magic, shift;
    __device__ __forceinline__ int of(int n) const {
        return magic == 0 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), magic) >> shift);
    }
};

// One product, D = A B, or A B + A' B' (two segments of K). What every role
// reads first comes first: parameters are fetched from memory a line at a time.
struct Job {
    int tiles, m_tiles, band, total_k, k_per_split, splits;
    int a_rows;              // rows of A that a CTA loads of a tile
    int first_blocks;        // K blocks of the first segment
    int per_split, per_band; // tiles of a part of K, and of a band of rows in it
    Divisor by_split, by_band, by_rows, by_last_rows;  // rows of a band, and of the last one
    int a_mn, b_mn;          // MN-major operands
    uint32_t idesc;
    int64_t m, n;            // rows and columns of the result (kGate: hidden units)
    const void *bias0, *bias1;
    void *out;               // kOut
    int64_t ld_out;
    Parts first, second;     // kGate: first = h; kInner: first = dp, second = dq
    float *a_kept, *b_kept;  // kGate: a and b written (NULL: not wanted); kInner: read. In blocks, see kept_at
    int64_t kept_blocks;     // of 16 columns
    float *partials;         // splits > 1: raw accumulators [split][gate | value][m][ld_partial]
    int64_t ld_partial;
    CUtensorMap a[2], b[2];  // a segment's operands; kGate: b[0] and b[1] are the gate's and the value's weights
};

// Independent products in one launch, in two classes of equal K: the tiles of
// the longer class go round the places first, `ahead` places get one more, the
// others catch up on `catch_up` tiles of the second class, and the rest go round.
struct GemmArgs {
    int job_count, first_jobs;
    int first_tiles, second_tiles, ahead, catch_up, places;
    int early;               // the kernel before writes no B: the first stages' are loaded while it ends
    int *status;
    Job jobs[kMaxJobs];
};

// ------------------------------------------------------------------- PTX

__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// All threads of the pair. Orders no memory but barriers set up before
// fence_barrier_init: a release would wait for every store under way, 1700
// clocks at a tile's end. What one CTA sends to the other's barriers is waited
// for there before the last of these.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The address that `local` has in the first CTA of the pair.
__device__ __forceinline__ uint32_t in_leader(uint32_t local) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(local));
    return remote;
}

// Says that accumulator columns have been read. Relaxed: they are in registers,
// and a release would wait for the results' stores (2000 clocks a tile).
__device__ __forceinline__ void arrive_leader(uint64_t *bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_leader(smem_addr(bar))) : "memory");
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

// One lane of a converged warp. The loaders' and the multiplier's whole loops
// run in such a lane: a warp that parts and meets again for every K block waits
// each time until its copies or matrix instructions have left (150 to 250 clocks).
__device__ __forceinline__ bool elect() {
    uint32_t chosen;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(chosen));
    return chosen != 0;
}

// Whether the phase is complete, without waiting. A wait behind copies or matrix
// instructions comes back late, ready or not, so the next stage is asked for
// between those of this one.
template <bool kCluster>
__device__ __forceinline__ bool test(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    if constexpr (kCluster) {
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(smem_addr(bar)), "r"(parity) : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(smem_addr(bar)), "r"(parity) : "memory");
    }
    return done != 0;
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
__device__ __forceinline__ Tile tile_at(const Job &a, int t) {
    Tile tile;
    tile.split = a.by_split.of(t);
    t -= tile.split * a.per_split;
    const int band = a.by_band.of(t), inside = t - band * a.per_band;
    const bool last = (band + 1) * a.band > a.m_tiles;
    const int rows = last ? a.m_tiles - band * a.band : a.band;
    tile.n = last ? a.by_last_rows.of(inside) : a.by_rows.of(inside);
    tile.m = band * a.band + (inside - tile.n * rows);
    tile.k_begin = tile.split * a.k_per_split;
    tile.k_end = min(a.total_k, tile.k_begin + a.k_per_split);
    return tile;
}

// The tiles of one place (a CTA or a pair), the same for all its roles.
struct Walk {
    int place, phase = 0, round = 0;
    __device__ explicit Walk(int p) : place(p) {}
    __device__ __forceinline__ bool next(const GemmArgs &a, int &job, Tile &tile) {
        int t = -1;
        if (phase == 0) {
            t = place + round * a.places;
            job = 0;
            if (t >= a.first_tiles) t = -1, phase = 1, round = 0;
        }
        if (phase == 1) {
            const int behind = a.places - a.ahead;
            t = place - a.ahead + round * behind;
            job = a.first_jobs;
            if (round >= a.catch_up || place < a.ahead || t >= a.second_tiles) t = -1, phase = 2, round = 0;
        }
        if (phase == 2) {
            const int turn = place >= a.ahead ? place - a.ahead : place - a.ahead + a.places;
            t = a.catch_up * (a.places - a.ahead) + turn + round * a.places;
            job = a.first_jobs;
            if (t >= a.second_tiles) return false;
        }
        ++round;
        while (t >= a.jobs[job].tiles) t -= a.jobs[job++].tiles;
        tile = tile_at(a.jobs[job], t);
        return true;
    }
};

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
    if (kWide % W == 0 && left >= kWide && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
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

// Where columns of a result go, as the epilogues see it. Direct: a thread
// stores its row's columns itself.
struct DirectStore {
    int64_t row, column, left;
    bool live;
    __device__ __forceinline__ bool inside() const { return live; }
    __device__ __forceinline__ int64_t own_row() const { return row; }
    template <int kWide, typename E>
    __device__ __forceinline__ void operator()(E *base, int64_t ld, const float (&in)[kWide]) const {
        if (live && left > 0) store_values<kWide>(base + row * ld + column, left, in);
    }
};

// 32 bytes at a multiple of 32: a whole sector with one instruction.
__device__ __forceinline__ void store_sector(void *p, const uint4 &a, const uint4 &b) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w),
                 "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
}

__device__ __forceinline__ void load_sector(const void *p, uint4 &a, uint4 &b) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                 : "l"(p));
}

// 16 columns of a warp's 32 rows, lane r holding row r: whole sectors where the
// rows allow it, else through shared memory, so that a warp stores contiguous
// entries of a row (2-byte stores down 32 rows took 6 us of a tile).
struct TileStore {
    uint8_t *area;
    int64_t row0, column, left;  // the warp's first row; columns from here to the result's last
    int rows;                    // its rows inside the result
    int lane;
    __device__ __forceinline__ bool inside() const { return lane < rows; }
    __device__ __forceinline__ int64_t own_row() const { return row0 + lane; }
    template <typename E>
    __device__ __forceinline__ void operator()(E *base, int64_t ld, const float (&in)[16]) const {
        constexpr int W = Pack<E>::kWidth, kPieces = 16 / W;
        uint4 pieces[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            float part[W];
#pragma unroll
            for (int e = 0; e < W; ++e) part[e] = in[i * W + e];
            pieces[i] = pack(part, E());
        }
        E *dst = base + row0 * ld + column;
        if (left >= 16 && ((reinterpret_cast<uintptr_t>(dst) | static_cast<uintptr_t>(ld * sizeof(E))) & 31) == 0) {
            if (lane < rows) {
#pragma unroll
                for (int i = 0; i < kPieces; i += 2) store_sector(dst + lane * ld + i * W, pieces[i], pieces[i + 1]);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) *reinterpret_cast<uint4 *>(area + lane * kStagedRow + 16 * i) = pieces[i];
        __syncwarp();
        const int c = lane & 15;
        if (c < left) {
#pragma unroll 1
            for (int r = lane >> 4; r < rows; r += 2) dst[r * ld + c] = reinterpret_cast<const E *>(area + r * kStagedRow)[c];
        }
        __syncwarp();
    }
};

template <int kWide, typename T, typename Store>
__device__ __forceinline__ void store_parts(const Store &store, const Parts &to, const float (&in)[kWide]) {
    using E = typename Operand16<T>::type;
    E *dst = static_cast<E *>(to.base);
    if constexpr (Operand16<T>::kParts == 1) {
        store(dst, to.ld, in);
    } else {
        float rest[kWide], part[kWide];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
#pragma unroll
            for (int j = 0; j < kWide; ++j) {
                rest[j] = k == 0 ? in[j] : rest[j] - part[j];
                part[j] = __bfloat162float(__float2bfloat16_rn(rest[j]));
            }
            store(dst + k * to.part_stride, to.ld, part);
        }
    }
}

// 16-bit results leave room for the approximate exponential and reciprocal
// (relative error about 1e-6; exp(-p) of 2^128 and more gives 0).
template <typename T>
__device__ __forceinline__ float sigmoid_of(float p) {
    if constexpr (sizeof(T) == 4) {
        return 1.0f / (1.0f + expf(-p));
    } else {
        float e, s;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(p * -1.4426950408889634f));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + e));
        return s;
    }
}

template <int kWide, typename T>
__device__ __forceinline__ void add_bias(const void *bias, int64_t column, int64_t left, float (&v)[kWide]) {
    if (bias == nullptr) return;
    float b[kWide];
    load_values<kWide>(static_cast<const T *>(bias) + column, left, b);
#pragma unroll
    for (int j = 0; j < kWide; ++j) v[j] += b[j];
}

template <int kWide>
__device__ __forceinline__ void add_staged(const float *bias, float (&v)[kWide]) {
#pragma unroll
    for (int j = 0; j < kWide / 4; ++j) {
        const float4 b = reinterpret_cast<const float4 *>(bias)[j];
        v[4 * j] += b.x, v[4 * j + 1] += b.y, v[4 * j + 2] += b.z, v[4 * j + 3] += b.w;
    }
}

// Where a and b of a row's 8 columns lie: blocks of 32 rows and 16 columns, two
// halves of 8 columns each, the rows side by side. The writer's and the reader's
// lane r both hold row r, so that a warp moves a kilobyte at a stretch (row by
// row, 32 sectors each: the reading kernel took 540 us for 32768 x 4096).
__device__ __forceinline__ float *kept_at(float *base, int64_t blocks, int64_t row, int64_t column) {
    return base + ((row >> 5) * blocks + (column >> 4)) * 512 + (column & 8) * 32 + (row & 31) * 8;
}

// kWide kept values of a row.
template <int kWide>
struct KeptRow {
    uint4 raw[kWide / 4];
    __device__ __forceinline__ void load(float *base, int64_t blocks, int64_t row, int64_t column, bool live) {
#pragma unroll
        for (int i = 0; i < kWide / 4; i += 2) {
            if (live) {
                load_sector(kept_at(base, blocks, row, column + 4 * i), raw[i], raw[i + 1]);
            } else {
                raw[i] = raw[i + 1] = make_uint4(0, 0, 0, 0);
            }
        }
    }
    static __device__ __forceinline__ void store(float *base, int64_t blocks, int64_t row, int64_t column, const float (&in)[kWide]) {
#pragma unroll
        for (int i = 0; i < kWide; i += 8) {
            uint4 v[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                v[k] = make_uint4(__float_as_uint(in[i + 4 * k]), __float_as_uint(in[i + 4 * k + 1]), __float_as_uint(in[i + 4 * k + 2]),
                                  __float_as_uint(in[i + 4 * k + 3]));
            }
            store_sector(kept_at(base, blocks, row, column + i), v[0], v[1]);
        }
    }
    __device__ __forceinline__ void times(const float (&in)[kWide], float (&out)[kWide]) const {
#pragma unroll
        for (int i = 0; i < kWide / 4; ++i) {
            out[4 * i] = in[4 * i] * __uint_as_float(raw[i].x);
            out[4 * i + 1] = in[4 * i + 1] * __uint_as_float(raw[i].y);
            out[4 * i + 2] = in[4 * i + 2] * __uint_as_float(raw[i].z);
            out[4 * i + 3] = in[4 * i + 3] * __uint_as_float(raw[i].w);
        }
    }
};

// kGate on kWide hidden units of one row.
template <int kWide, typename T, typename Store>
__device__ __forceinline__ void finish_gate(const Job &a, const Store &store, float (&p)[kWide], float (&q)[kWide]) {
    if (a.a_kept == nullptr) {
#pragma unroll
        for (int j = 0; j < kWide; ++j) q[j] *= p[j] * sigmoid_of<T>(p[j]);
    } else {
        float slope[kWide];
#pragma unroll
        for (int j = 0; j < kWide; j += 2) {
            const float2 s = make_float2(sigmoid_of<T>(p[j]), sigmoid_of<T>(p[j + 1])), x = make_float2(p[j], p[j + 1]), y = make_float2(q[j], q[j + 1]);
            const float2 one = make_float2(1.0f, 1.0f);
            const float2 rest = fma2(s, make_float2(-1.0f, -1.0f), one);  // 1 - s
            const float2 b = mul2(y, mul2(s, fma2(x, rest, one))), a = mul2(x, s), h = mul2(y, a);
            slope[j] = b.x, slope[j + 1] = b.y;
            p[j] = a.x, p[j + 1] = a.y;
            q[j] = h.x, q[j + 1] = h.y;
        }
        if (store.inside()) {
            KeptRow<kWide>::store(a.a_kept, a.kept_blocks, store.own_row(), store.column, p);
            KeptRow<kWide>::store(a.b_kept, a.kept_blocks, store.own_row(), store.column, slope);
        }
    }
    store_parts<kWide, T>(store, a.first, q);
}

// kInner on kWide hidden units of one row of dh.
template <int kWide, typename T, typename Store>
__device__ __forceinline__ void finish_inner(const Job &j, const Store &store, const KeptRow<kWide> &a, const KeptRow<kWide> &b, const float (&dh)[kWide]) {
    float out[kWide];
    b.times(dh, out);
    store_parts<kWide, T>(store, j.first, out);
    a.times(dh, out);
    store_parts<kWide, T>(store, j.second, out);
}

template <int kWide, typename T, typename Store>
__device__ __forceinline__ void finish_out(const Job &a, const Store &store, float (&y)[kWide]) {
    store(static_cast<T *>(a.out), a.ld_out, y);
}

// ------------------------------------------------------------------- kernel
//
// Two warps load, every other stage each, one multiplies, eight finish tiles: two
// per quarter of the accumulator's lanes, each on half of its columns. Two
// accumulators, so a tile is finished while the next is multiplied. kCtas = 2: a pair of CTAs
// computes 256 rows with one instruction; each loads its 128 rows of A and half
// of B's columns, so an SM reads a third fewer bytes per product than with a
// 128 x 256 tile of its own (32768 rows of 2048 -> 4096 -> 2048: 923 to 856 us of
// the gate's product when pairs came in, 805 now). fp32: a K block is three stages, one a part, each
// loaded once for all the products of its parts. Every wait is bounded; one that
// gives up raises the CTA's abort flag and the status word, and all roles leave.
template <typename T, int kEpilogue, int kTileN, int kCtas>
__global__ __launch_bounds__(kThreads, 1) void gemm_kernel(const __grid_constant__ GemmArgs args) {
    constexpr uint32_t kBBytes = static_cast<uint32_t>(kTileN / kCtas) * kBK * 2;
    constexpr uint32_t kStage = kABytes + kBBytes;
    constexpr int kStages = kRingBytes / kStage < kMaxStages ? kRingBytes / kStage : kMaxStages;
    constexpr int kUnits = kEpilogue == kGate ? kTileN / 2 : kTileN;  // result columns of a tile
    constexpr int kParts = Operand16<T>::kParts;
    constexpr bool kPasses = kParts > 1;
    constexpr int kAccumulator = kPasses ? 2 * kTileN : kTileN;  // TMEM columns
    static_assert(2 * kAccumulator <= static_cast<int>(kTmemColumns), "two accumulators");
    static_assert(kStages >= kParts + 2, "a K block's parts stay while the next is loaded");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    uint8_t *staged = ring + kRingBytes;
    uint64_t *full = reinterpret_cast<uint64_t *>(staged + kEpilogueWarps * (kStagedBytes + kBiasBytes));
    uint64_t *empty = full + kMaxStages;
    uint64_t *acc_full = empty + kMaxStages;
    uint64_t *acc_empty = acc_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = kCtas == 1 ? 0 : static_cast<int>(cta_rank());
    pdl_trigger();
    Walk walk(blockIdx.x / kCtas);
    int job = 0;
    Tile tile{};
    bool more = walk.next(args, job, tile);  // the parameters come in while barriers and TMEM are set up
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
    if (threadIdx.x == 32) {
        prefetch_tensor_map(&args.jobs[job].a[0]);
        prefetch_tensor_map(&args.jobs[job].b[kEpilogue == kGate && kCtas == 2 ? rank : 0]);
    }
    if (warp == kLoaders) {
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

    if (warp < kLoaders) {
        if (elect()) {
            int stage = 0, turn = 0;
            uint32_t phase = 0;
            bool ok = true, first = true, next_empty = false;
            auto advance = [&] {
                turn ^= 1;
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            };
            // B's part of K block kb, and the stage's bytes announced; A's part
            auto load_b = [&](const Job &j, int kb, int part) {
                const int segment = kEpilogue != kGate && kb >= j.first_blocks;
                const CUtensorMap *mb = kEpilogue == kGate && kCtas == 2 ? &j.b[rank] : &j.b[segment];
                const int32_t k = (segment ? kb - j.first_blocks : kb) * kBK;
                const int32_t column = kEpilogue == kGate ? tile.n * kUnits : tile.n * kTileN + rank * (kTileN / kCtas);
                uint8_t *to = ring + stage * kStage + kABytes;
                const uint32_t bar = kCtas == 1 ? smem_addr(&full[stage]) : in_leader(smem_addr(&full[stage]));
                if (rank == 0) mbar_arrive_expect_tx(&full[stage], (kBBytes + j.a_rows * (kBK * 2)) * kCtas);
                if constexpr (kEpilogue == kGate) {  // K-major: the units' gate rows, then their value rows
                    load_box<kCtas>(to, mb, bar, k, column, part);
                    if (kCtas == 1) load_box<1>(to + kBBytes / 2, &j.b[1], bar, k, column, part);
                } else if (j.b_mn) {
#pragma unroll
                    for (int c = 0; c < kTileN / kCtas / 64; ++c) load_box<kCtas>(to + c * 8192, mb, bar, column + 64 * c, k, part);
                } else {
                    load_box<kCtas>(to, mb, bar, k, column, part);
                }
            };
            auto load_a = [&](const Job &j, int kb, int part) {
                const int segment = kEpilogue != kGate && kb >= j.first_blocks;
                const CUtensorMap *ma = &j.a[segment];
                const int32_t k = (segment ? kb - j.first_blocks : kb) * kBK, row = (tile.m * kCtas + rank) * kBM;
                uint8_t *to = ring + stage * kStage;
                const uint32_t bar = kCtas == 1 ? smem_addr(&full[stage]) : in_leader(smem_addr(&full[stage]));
                if (j.a_mn) {
                    load_box<kCtas>(to, ma, bar, row, k, part);
                    load_box<kCtas>(to + kABytes / 2, ma, bar, row + 64, k, part);
                } else {
                    load_box<kCtas>(to, ma, bar, k, row, part);
                }
            };
            for (; more && ok; more = walk.next(args, job, tile)) {
                const Job &j = args.jobs[job];
                int ready = 0;  // stages of this tile whose B is under way
                if (first && args.early) {
                    ready = min(kStages, (tile.k_end - tile.k_begin) * kParts);
                    for (int i = 0; i < ready; ++i, advance()) {
                        if (turn == warp) load_b(j, tile.k_begin + i / kParts, i % kParts);
                    }
                    stage = turn = 0;
                    phase = 0;
                }
                if (first) pdl_wait();
                first = false;
                for (int kb = tile.k_begin; kb < tile.k_end && ok; ++kb) {
#pragma unroll 1
                    for (int part = 0; part < kParts; ++part, --ready, advance()) {
                        if (turn != warp) continue;
                        if (ready <= 0) {
                            ok = next_empty || wait<kCtas == 2>(&empty[stage], phase ^ 1, abort, args.status);
                            if (!ok) break;
                            const int s = stage + kLoaders < kStages ? stage + kLoaders : stage + kLoaders - kStages;
                            next_empty = test<kCtas == 2>(&empty[s], s > stage ? phase ^ 1 : phase);
                            load_b(j, kb, part);
                        }
                        load_a(j, kb, part);
                    }
                }
            }
            if (first) pdl_wait();
            // the last stages' releases, which the pair's leader sends, have come before the CTA ends
            for (int i = 0; i < kStages && ok; ++i, advance()) {
                if (turn == warp) ok = wait<kCtas == 2>(&empty[stage], phase ^ 1, abort, args.status);
            }
            if (*abort && warp == 0 && rank == 0) {  // copies still under way land before the CTA ends
                for (int s = 0; s < kStages; ++s) {
                    for (uint32_t spin = 0; spin < (1u << 16) && !mbar_try_wait<kCtas == 2>(&full[s], s < stage ? phase : phase ^ 1); ++spin) {
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == kLoaders) {
        if (rank == 0 && elect()) {
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true, next_full = false;
            auto next_accumulator = [&] {
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1;
                }
            };
            for (; more && ok; more = walk.next(args, job, tile)) {
                const int a_mn = args.jobs[job].a_mn, b_mn = args.jobs[job].b_mn;
                const uint32_t idesc = args.jobs[job].idesc;
                // 16 of K: 16 rows of 128 bytes, or 32 bytes of every row (addresses count 16 bytes)
                const uint64_t step_a = a_mn ? 2048 >> 4 : 32 >> 4, step_b = b_mn ? 2048 >> 4 : 32 >> 4;
                const uint64_t kind_a = a_mn ? sw128_mnmajor_desc(0) : sw128_kmajor_desc(0);
                const uint64_t kind_b = b_mn ? sw128_mnmajor_desc(0) : sw128_kmajor_desc(0);
                const uint32_t base = smem_addr(ring);
                uint32_t d = 0;
                // A's part from one stage, B's from another; on the way, whether the stage behind has come
                auto multiply_parts = [&](uint32_t to, int stage_a, int stage_b, bool fresh, bool ask) {
                    const uint64_t da = kind_a | (base + stage_a * kStage) >> 4, db = kind_b | (base + stage_b * kStage + kABytes) >> 4;
#pragma unroll
                    for (int k = 0; k < kBK / 16; ++k) {
                        mma<kCtas>(to, da + k * step_a, db + k * step_b, idesc, !fresh || k > 0);
                        if (k == 1 && ask) next_full = test<kCtas == 2>(&full[stage], phase);
                    }
                };
                for (int kb = tile.k_begin; kb < tile.k_end && ok; ++kb) {
                    const bool fresh = kb == tile.k_begin || (kPasses && (kb - tile.k_begin) % kPass == 0);
                    if (fresh) {
                        if (kb > tile.k_begin) {
                            commit<kCtas>(&acc_full[acc]);
                            next_accumulator();
                        }
                        ok = wait<kCtas == 2>(&acc_empty[acc], acc_phase ^ 1, abort, args.status);
                        if (!ok) break;
                        tc_fence_after();
                        d = tmem + static_cast<uint32_t>(acc * kAccumulator);
                    }
                    int at[kParts];
#pragma unroll
                    for (int part = 0; part < kParts; ++part) {
                        ok = next_full || wait<kCtas == 2>(&full[stage], phase, abort, args.status);
                        if (!ok) break;
                        tc_fence_after();
                        at[part] = stage;
                        if (++stage == kStages) {
                            stage = 0;
                            phase ^= 1;
                        }
                        if (part == 0) {
                            multiply_parts(d, at[0], at[0], fresh, true);
                            if (kParts == 1) commit<kCtas>(&empty[at[0]]);
                        } else if (part == 1) {
                            multiply_parts(d + kTileN, at[0], at[part], fresh, false);
                            multiply_parts(d + kTileN, at[part], at[0], false, false);
                            multiply_parts(d + kTileN, at[part], at[part], false, true);
                            commit<kCtas>(&empty[at[part]]);
                        } else {
                            multiply_parts(d + kTileN, at[0], at[part], false, false);
                            multiply_parts(d + kTileN, at[part], at[0], false, true);
                            commit<kCtas>(&empty[at[0]]);
                            commit<kCtas>(&empty[at[part]]);
                        }
                    }
                }
                if (ok) {
                    commit<kCtas>(&acc_full[acc]);
                    next_accumulator();
                }
            }
            for (int b = 0; b < 2 && ok; ++b) {  // the other CTA's releases of the accumulators have come, too
                ok = wait<kCtas == 2>(&acc_empty[acc], acc_phase ^ 1, abort, args.status);
                next_accumulator();
            }
        }
        __syncwarp();
    } else {
        // Groups of 16 columns, alternately for the two warps of a quarter, in a
        // loop that is not unrolled: a tile's epilogue runs once or twice a
        // launch of a small problem, at the speed that its code is fetched.
        const int quarter = warp & 3, part = (warp - kLoaders - 1) >> 2;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        constexpr int kGroups = kUnits / 16, kSides = kEpilogue == kGate ? 2 : 1;
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
        TileStore store{staged + (warp - kLoaders - 1) * kStagedBytes, 0, 0, 0, 0, lane};
        float *const biases = reinterpret_cast<float *>(staged + kEpilogueWarps * kStagedBytes + (warp - kLoaders - 1) * kBiasBytes);
        bool first = true;
        // a warp that has given up still meets the others at every tile
        for (; more; more = walk.next(args, job, tile)) {
            const Job &j = args.jobs[job];
            store.row0 = static_cast<int64_t>(tile.m * kCtas + rank) * kBM + quarter * 32;
            store.rows = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(32), j.m - store.row0)));
            const int64_t first_column = static_cast<int64_t>(tile.n) * kUnits;
            KeptRow<16> kept_a, kept_b;  // kInner: of the group to come
            auto request = [&](int g) {
                if constexpr (kEpilogue == kInner) {
                    if (j.splits > 1 || g >= kGroups) return;
                    kept_a.load(j.a_kept, j.kept_blocks, store.row0 + lane, first_column + g * 16, lane < store.rows && first_column + g * 16 < j.n);
                    kept_b.load(j.b_kept, j.kept_blocks, store.row0 + lane, first_column + g * 16, lane < store.rows && first_column + g * 16 < j.n);
                }
            };
            // 16 columns of the warp's rows (kGate: of p and of q)
            auto finish = [&](int g, float (&v)[kSides][16]) {
                store.column = first_column + g * 16;
                store.left = j.n - store.column;
                if (store.left <= 0) return;
                if (j.splits > 1) {  // parts of the sums are parked
                    float *base = j.partials + kSides * tile.split * j.m * j.ld_partial;
#pragma unroll
                    for (int k = 0; k < kSides; ++k) store(base + k * j.m * j.ld_partial, j.ld_partial, v[k]);
                } else if constexpr (kEpilogue == kGate) {
                    if (j.bias0 != nullptr) add_staged<16>(biases + g / 2 * 16, v[0]);
                    if (j.bias1 != nullptr) add_staged<16>(biases + kUnits / 2 + g / 2 * 16, v[1]);
                    finish_gate<16, T>(j, store, v[0], v[1]);
                } else if constexpr (kEpilogue == kInner) {
                    const KeptRow<16> a = kept_a, b = kept_b;
                    request(g + 2);
                    finish_inner<16, T>(j, store, a, b, v[0]);
                } else {
                    if (j.bias0 != nullptr) add_staged<16>(biases + g / 2 * 16, v[0]);
                    finish_out<16, T>(j, store, v[0]);
                }
            };
            if (first) pdl_wait();  // before anything of the kernel before is read, and anything written
            first = false;
            request(part);
            if constexpr (kEpilogue != kInner) {  // the biases of the warp's columns, while the tile is multiplied
                if (j.splits == 1 && (j.bias0 != nullptr || j.bias1 != nullptr)) {
                    __syncwarp();
#pragma unroll 1
                    for (int i = lane; i < kSides * kUnits / 2; i += 32) {
                        const int side = i / (kUnits / 2), c = i % (kUnits / 2);
                        const int64_t column = first_column + (part + 2 * (c / 16)) * 16 + c % 16;
                        const T *bias = static_cast<const T *>(side == 0 ? j.bias0 : j.bias1);
                        biases[i] = bias != nullptr && column < j.n ? to_acc(bias[column]) : 0.0f;
                    }
                    __syncwarp();
                }
            }
            if constexpr (kPasses) {
                constexpr int kMine = kGroups / 2;
                float sum[kMine][kSides][16];
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
#pragma unroll
                    for (int k = 0; k < kSides; ++k) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) sum[i][k][e] = 0.0f;
                    }
                }
                for (int kb = tile.k_begin; kb < tile.k_end && ok; kb += kPass) {
                    ok = wait<kCtas == 2>(&acc_full[acc], acc_phase, abort, args.status);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t from = tmem + lanes + static_cast<uint32_t>(acc * kAccumulator + part * 16);
#pragma unroll
                    for (int i = 0; i < kMine; ++i) {
#pragma unroll
                        for (int k = 0; k < kSides; ++k) {
#pragma unroll
                            for (int which = 0; which < 2; ++which) {  // x0 y0, and the rest
                                uint32_t raw[16];
                                KOEMI_TMEM_LD16(from + which * kTileN + k * kUnits + i * 32, raw);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) sum[i][k][e] += __uint_as_float(raw[e]);
                            }
                        }
                    }
                    release();
                }
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    if (ok) finish(part + 2 * i, sum[i]);
                }
            } else {
                ok = ok && wait<kCtas == 2>(&acc_full[acc], acc_phase, abort, args.status);
                tc_fence_after();
                const uint32_t from = tmem + lanes + static_cast<uint32_t>(acc * kAccumulator);
#pragma unroll 1
                for (int g = part; g < kGroups && ok; g += 2) {
                    uint32_t raw[kSides][16];
                    float v[kSides][16];
#pragma unroll
                    for (int k = 0; k < kSides; ++k) KOEMI_TMEM_LD16(from + k * kUnits + g * 16, raw[k]);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < kSides; ++k) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) v[k][e] = __uint_as_float(raw[k][e]);
                    }
                    if (g + 2 >= kGroups) release();
                    finish(g, v);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (kCtas == 2) cluster_sync();  // the pair ends together
    if (warp == kLoaders) {
        tc_fence_after();
        if constexpr (kCtas == 1) {
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
        } else {
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
        }
    }
}

// The splits' accumulators added in order, then the epilogue: 8 columns a
// thread. grid.y: the job. (Joined by the last CTA of a tile to come, through a
// counter, the same took 3 to 6 times as long: one CTA reads what here the whole GPU does.)
template <typename T, int kEpilogue>
__global__ __launch_bounds__(256) void join_kernel(const __grid_constant__ GemmArgs args) {
    const Job &j = args.jobs[blockIdx.y];
    pdl_wait();
    const int64_t groups = (j.n + 7) / 8;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (j.splits == 1 || i >= groups * j.m) return;
    const int64_t row = i / groups, column = (i - row * groups) * 8;
    constexpr int kSides = kEpilogue == kGate ? 2 : 1;
    const int64_t side = j.m * j.ld_partial;
    const float *src = j.partials + row * j.ld_partial + column;
    KeptRow<8> kept_a, kept_b;
    if constexpr (kEpilogue == kInner) {
        kept_a.load(j.a_kept, j.kept_blocks, row, column, true);
        kept_b.load(j.b_kept, j.kept_blocks, row, column, true);
    }
    float sum[kSides][8] = {};
#pragma unroll 4
    for (int s = 0; s < j.splits; ++s) {
#pragma unroll
        for (int k = 0; k < kSides; ++k) {
            // ld_partial is a multiple of 16; not through the read-only path: the kernel before wrote them
            const float4 *from = reinterpret_cast<const float4 *>(src + (kSides * s + k) * side);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float4 v = from[i];
                sum[k][4 * i] += v.x, sum[k][4 * i + 1] += v.y, sum[k][4 * i + 2] += v.z, sum[k][4 * i + 3] += v.w;
            }
        }
    }
    const DirectStore store{row, column, j.n - column, true};
    if constexpr (kEpilogue == kGate) {
        add_bias<8, T>(j.bias0, column, store.left, sum[0]);
        add_bias<8, T>(j.bias1, column, store.left, sum[1]);
        finish_gate<8, T>(j, store, sum[0], sum[1]);
    } else if constexpr (kEpilogue == kInner) {
        finish_inner<8, T>(j, store, kept_a, kept_b, sum[0]);
    } else {
        add_bias<8, T>(j.bias0, column, store.left, sum[0]);
        finish_out<8, T>(j, store, sum[0]);
    }
}

// ------------------------------------------------------------------ few rows
//
// A few rows (tokens at decode) are bound by the weights' bytes: a warp takes the
// dot products of few_units units with every row on the FMA units, straight from
// the weights as they lie (fp32 too: no parts), 16 bytes a lane at a time. The
// tensor cores' tiles are 128 rows high and their sums parted along K. Measured,
// here and there, 2048 -> 4096 -> 2048: 1 row 16 and 25 us in bf16, 22 and 99 in
// fp32; 4 rows 23 and 25 (1024 -> 2048 -> 1024: 14 and 17); 8 rows in fp32 43 and
// 99; with rows that no 16-byte load fits (3229 -> 2690 -> 3229) 2 rows of bf16 39
// and 50, 8 of fp32 86 and 110. Hence the limit, next to which the two meet:
int64_t few_limit(int64_t width, int64_t hidden, int dtype) {
    return dtype == KOEMI_F32 ? 8 : width % 8 == 0 && hidden % 8 == 0 ? 4 : 2;
}
// Units of a warp. Loads by element want more of them to an x: 1 row of 3229 ->
// 2690 -> 3229 bf16 30 us with 2, 23 with 4 (2048 -> 4096 -> 2048, 16 bytes a load: 17 and 19).
constexpr int few_units(bool vector) { return vector ? 2 : 4; }
// Steps of 32 lanes whose weights a warp asks for together.
constexpr int few_asked(bool vector, int dots) { return (vector ? 16 : 32) / dots; }

struct FewArgs {
    const void *x, *w0, *w1;   // kGate: the gate's and the value's weights; kOut: w0
    const void *bias0, *bias1;
    int64_t ld_x, width, units;
    int rows;
    int share;                 // warps that part the width of one's units (a power of two up to 8)
    void *out;                 // kOut: [rows, units]; kGate: h as the second product reads it
    int64_t ld_out;
    Parts parts;               // kGate: h for the backward (base NULL: not wanted)
    float *a_kept, *b_kept;
    int64_t kept_blocks;
};

// 16 bytes of a row of weights, or one value, as they lie.
template <typename T, bool kVec>
struct Piece {
    uint4 raw;
    T one;
    __device__ __forceinline__ void load(const T *p, bool live) {
        if constexpr (kVec) {
            raw = live ? load_stream(p) : make_uint4(0, 0, 0, 0);
        } else {
            one = live ? __ldg(p) : from_acc<T>(0.0f);
        }
    }
    template <int W>
    __device__ __forceinline__ void values(float (&out)[W]) const {
        if constexpr (kVec) {
            unpack(raw, out, T());
        } else {
            out[0] = to_acc(one);
        }
    }
};

template <typename T, int kEpilogue, int R, bool kVec>
__global__ __launch_bounds__(256) void few_rows_kernel(const __grid_constant__ FewArgs args) {
    constexpr int W = kVec ? Pack<T>::kWidth : 1, kSides = kEpilogue == kGate ? 2 : 1;
    constexpr int kFewUnits = few_units(kVec), N = kFewUnits * kSides, kAsked = few_asked(kVec, N);
    __shared__ float sums[8][N * R];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, part = warp & (args.share - 1);
    // units behind the last are the last once more, and not stored
    const int64_t unit0 = (static_cast<int64_t>(blockIdx.x) * 8 + warp) / args.share * kFewUnits;
    pdl_trigger();
    const T *w[N];
#pragma unroll
    for (int u = 0; u < kFewUnits; ++u) {
        const int64_t unit = min(unit0 + u, args.units - 1);
#pragma unroll
        for (int k = 0; k < kSides; ++k) w[u * kSides + k] = static_cast<const T *>(k == 0 ? args.w0 : args.w1) + unit * args.width;
    }
    const T *x = static_cast<const T *>(args.x);
    float sum[N][R];
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int r = 0; r < R; ++r) sum[n][r] = 0.0f;
    }
    bool waited = false;
    for (int64_t base = part * (kAsked * 32 * W); base < args.width; base += args.share * (kAsked * 32 * W)) {
        Piece<T, kVec> pieces[kAsked][N];
#pragma unroll
        for (int i = 0; i < kAsked; ++i) {
            const int64_t c = base + (i * 32 + lane) * W;
#pragma unroll
            for (int n = 0; n < N; ++n) pieces[i][n].load(w[n] + c, c < args.width);
        }
        if (!waited) {  // the first weights are under way while the kernel before ends
            pdl_wait();
            waited = true;
        }
#pragma unroll
        for (int i = 0; i < kAsked; ++i) {
            const int64_t c = base + (i * 32 + lane) * W;
            if (c >= args.width) continue;
            float wv[N][W];
#pragma unroll
            for (int n = 0; n < N; ++n) pieces[i][n].values(wv[n]);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                // a row behind the last is the last once more; not through the read-only path: the kernel before may have written it
                const T *from = x + min(r, args.rows - 1) * args.ld_x + c;
                float xv[W];
                if constexpr (kVec) {
                    unpack(*reinterpret_cast<const uint4 *>(from), xv, T());
                } else {
                    xv[0] = to_acc(*from);
                }
#pragma unroll
                for (int n = 0; n < N; ++n) {
#pragma unroll
                    for (int e = 0; e < W; ++e) sum[n][r] = fmaf(wv[n][e], xv[e], sum[n][r]);
                }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            sum[n][r] = warp_sum(sum[n][r]);
            if (lane == 0) sums[warp][n * R + r] = sum[n][r];
        }
    }
    if (!waited) pdl_wait();  // a part behind the width
    __syncthreads();
    if (part != 0 || lane >= args.rows) return;
    // lane r of the first part's warp adds and finishes row r
#pragma unroll
    for (int u = 0; u < kFewUnits; ++u) {
        const int64_t unit = unit0 + u;
        if (unit >= args.units) continue;
        float v[kSides];
#pragma unroll
        for (int k = 0; k < kSides; ++k) {
            v[k] = 0.0f;
            for (int i = 0; i < args.share; ++i) v[k] += sums[warp + i][(u * kSides + k) * R + lane];
            const T *bias = static_cast<const T *>(k == 0 ? args.bias0 : args.bias1);
            if (bias != nullptr) v[k] += to_acc(bias[unit]);
        }
        T *out = static_cast<T *>(args.out) + lane * args.ld_out + unit;
        if constexpr (kEpilogue == kGate) {  // h in the type, as the tensor cores' path rounds it
            const float s = sigmoid_of<T>(v[0]), a = v[0] * s;
            if (args.parts.base != nullptr) {
                *(kept_at(args.a_kept, args.kept_blocks, lane, unit & ~7) + (unit & 7)) = a;
                *(kept_at(args.b_kept, args.kept_blocks, lane, unit & ~7) + (unit & 7)) = v[1] * (s * fmaf(v[0], 1.0f - s, 1.0f));
                const float h[1] = {a * v[1]};
                store_parts<1, T>(DirectStore{lane, unit, 1, true}, args.parts, h);
            }
            *out = from_acc<T>(a * v[1]);
        } else {
            *out = from_acc<T>(v[0]);
        }
    }
}

template <typename T, int kEpilogue>
int few_rows(FewArgs args, bool dependent, cudaStream_t stream) {
    constexpr int W = Pack<T>::kWidth;
    const bool vector = args.width % W == 0 && args.ld_x % W == 0 && aligned(args.x, 16) && aligned(args.w0, 16) && aligned(args.w1, 16);
    auto kernel = vector ? few_rows_kernel<T, kEpilogue, 1, true> : few_rows_kernel<T, kEpilogue, 1, false>;
    if (args.rows > 1) kernel = vector ? few_rows_kernel<T, kEpilogue, 2, true> : few_rows_kernel<T, kEpilogue, 2, false>;
    if (args.rows > 2) kernel = vector ? few_rows_kernel<T, kEpilogue, 4, true> : few_rows_kernel<T, kEpilogue, 4, false>;
    if constexpr (sizeof(T) == 4) {
        if (args.rows > 4) kernel = vector ? few_rows_kernel<T, kEpilogue, 8, true> : few_rows_kernel<T, kEpilogue, 8, false>;
    }
    // warps share units until 8 an SM (16 with loads by element) have work, and while each has a step of its
    // own: 1 row of 2048 -> 4096 -> 2048 bf16 19 us without, 16 with, 18 where steps are not full
    const int units = few_units(vector);
    const int64_t groups = ceil_div(args.units, units), want = (vector ? 8 : 16) * sm_count();
    const int64_t step = few_asked(vector, units * (kEpilogue == kGate ? 2 : 1)) * 32 * (vector ? W : 1);
    args.share = 1;
    while (args.share < 8 && groups * args.share < want && 2 * args.share * step <= args.width) args.share *= 2;
    const int64_t blocks = ceil_div(groups * args.share, 8);
    KOEMI_CUDA_TRY(launch_programmatic(dependent, kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, dim3(1, 1, 1), args));
    return KOEMI_OK;
}

// ------------------------------------------------------------ packed operands

struct PackJob {
    const void *src;
    int64_t rows, columns, ld;
    Parts to;
};
constexpr int kMaxPacks = 5;
struct PackArgs {
    PackJob jobs[kMaxPacks];
};

// Row-major matrices copied (fp32: split) to rows of a multiple of 16 columns, zeros
// behind the last. grid.y: the matrix. Bound by bytes: 3 us for 4096 x 128 and its weights in fp32.
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(const __grid_constant__ PackArgs args) {
    const PackJob &job = args.jobs[blockIdx.y];
    const int64_t groups = job.to.ld / 8, count = groups * job.rows;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = i / groups, column = (i - row * groups) * 8;
        float v[8];
        load_values<8>(static_cast<const T *>(job.src) + row * job.ld + column, job.columns - column, v);
        store_parts<8, T>(DirectStore{row, column, 8, true}, job.to, v);
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
// Bound by latency at small sizes (4096 rows of 256, 256 and 128 fp32 columns: 8 us, and 4 for the totals).
template <typename T>
__global__ __launch_bounds__(256) void column_sums_kernel(const __grid_constant__ SumArgs args) {
    using E = typename Operand16<T>::type;
    __shared__ float parts[8][33];
    pdl_trigger();
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
    pdl_wait();
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

int64_t round16(int64_t v) { return (v + 15) / 16 * 16; }  // whole sectors of 16-bit values
size_t round256(size_t v) { return (v + 255) & ~size_t(255); }

int encode(CUtensorMap *map, const Matrix &matrix, bool half, bool mn_major, int box_rows) {
    const CUtensorMapDataType type = half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const uint64_t dims[3] = {static_cast<uint64_t>(matrix.columns), static_cast<uint64_t>(matrix.rows), static_cast<uint64_t>(matrix.parts)};
    const uint64_t part = static_cast<uint64_t>(matrix.parts > 1 ? matrix.part_stride : matrix.ld) * 2;
    const uint64_t strides[2] = {static_cast<uint64_t>(matrix.ld) * 2, part};
    const uint32_t box[3] = {64, mn_major ? 64u : static_cast<uint32_t>(box_rows), 1};
    return encode_tensor_map(map, type, 3, matrix.base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// One product as the host sees it. kGate: one A, B the two weights, n hidden units.
struct Product {
    Matrix a[2], b[2];
    int segments;
    bool a_mn, b_mn;
    int64_t m, n;
};

int blocks_of(const Product &p, int segment) {
    return static_cast<int>(ceil_div(p.a_mn ? p.a[segment].rows : p.a[segment].columns, kBK));
}
int total_k_of(const Product &p, bool gate) { return blocks_of(p, 0) + (!gate && p.segments > 1 ? blocks_of(p, 1) : 0); }

// How a launch is cut: its tiles' columns, CTAs a tile, and each product's parts of K.
struct Cut {
    int tile_n, ctas, splits[kMaxJobs];
};

int64_t tiles_of(const Product &p, bool gate, int tile_n, int ctas) {
    return ceil_div(p.m, kBM * ctas) * ceil_div(p.n, gate ? tile_n / 2 : tile_n);
}

// The cheapest cut by clocks. An SM takes about 52 bytes a clock from L2
// (measured with all SMs loading: 128 x 256 tiles 51, 128 x 128 tiles 53), which
// is what a K block of every shape but a pair's 256 x 256 waits for; its
// products take the tensor cores 2 clocks a column (six products a block of
// fp32). A product is parted along K where a whole tile of it would outlast an
// even share of the work. A launch adds about 6500 clocks for its first loads
// and its last epilogue; parts of K add a kernel and their accumulators' way
// through L2. Products of one group are in at most two classes of equal K, the
// longer first.
Cut cut_of(const Product *const *products, int count, bool gate, int sms) {
    const int parts = products[0]->a[0].parts;
    Cut best{128, 1, {1, 1, 1, 1}};
    double least = 1e300;
    const struct { int tile_n, ctas; } shapes[] = {{256, 2}, {128, 2}, {256, 1}, {128, 1}, {64, 1}};
    int64_t rows = 0;
    for (int i = 0; i < count; ++i) rows = std::max(rows, products[i]->m);
    for (const auto &shape : shapes) {
        if (parts > 1 && shape.tile_n > 128) continue;  // two accumulators of two parts, and their sums in registers
        if (shape.ctas == 2 && rows <= kBM) continue;
        const double loaded = static_cast<double>(std::min<int64_t>(rows, kBM)) + shape.tile_n / shape.ctas;
        const double clocks = std::max(shape.tile_n * (parts > 1 ? 12.0 : 2.0), parts * loaded * kBK * 2 / 52.0);
        const double places = std::max(1, sms / shape.ctas);
        double work = 0;
        for (int i = 0; i < count; ++i) work += static_cast<double>(tiles_of(*products[i], gate, shape.tile_n, shape.ctas)) * total_k_of(*products[i], gate) * clocks;
        for (int eager = 0; eager < 2; ++eager) {  // parts of K as long as an even share, or shorter ones
            Cut cut{shape.tile_n, shape.ctas, {1, 1, 1, 1}};
            const double share = std::max(work / places / (1 + eager), 3000.0);
            double load = 0, longest = 0, joined = 0;
            for (int i = 0; i < count; ++i) {
                const int total = total_k_of(*products[i], gate);
                int splits = static_cast<int>(std::min(64.0, total * clocks / share + (eager ? 0.999 : 0.3)));
                splits = std::max(1, std::min(splits, total));
                const int per = static_cast<int>(ceil_div(total, splits));
                splits = static_cast<int>(ceil_div(total, per));  // every part has blocks
                cut.splits[i] = splits;
                const double tiles = static_cast<double>(tiles_of(*products[i], gate, shape.tile_n, shape.ctas)) * splits;
                longest = std::max(longest, per * clocks);
                load += tiles * per * clocks;
                if (splits > 1) joined += (gate ? 2.0 : 1.0) * static_cast<double>(products[i]->m) * static_cast<double>(products[i]->n) * (splits + 1) * 4;
            }
            // an even share, rounded up to whole tiles of the shortest product
            const Product &last = *products[count - 1];
            const double shortest = ceil_div(total_k_of(last, gate), cut.splits[count - 1]) * clocks;
            double cost = std::max(longest, std::ceil(load / places / shortest - 1e-9) * shortest) + 6500;
            if (joined > 0) cost += 9000 + joined / 2500;
            if (cost < least) least = cost, best = cut;
        }
    }
    return best;
}

size_t partial_bytes(const Cut &cut, int i, const Product &p, bool gate) {
    return cut.splits[i] == 1 ? 0 : round256(static_cast<size_t>(cut.splits[i]) * (gate ? 2 : 1) * p.m * round16(p.n) * sizeof(float));
}

// What the products of one launch, cut alike, need for their partial sums.
size_t partial_bytes(const Cut &cut, const Product *const *products, int count, bool gate) {
    size_t bytes = 0;
    for (int i = 0; i < count; ++i) bytes += partial_bytes(cut, i, *products[i], gate);
    return bytes;
}
template <typename T, int kEpilogue, int kTileN, int kCtas>
int launch_shape(GemmArgs &args, bool dependent, cudaStream_t stream) {
    auto kernel = gemm_kernel<T, kEpilogue, kTileN, kCtas>;
    // once a device: the most that any launch takes
    static std::atomic<bool> allowed[64];
    int device = 0;
    KOEMI_CUDA_TRY(cudaGetDevice(&device));
    if (device >= 64 || !allowed[device].load(std::memory_order_acquire)) {
        KOEMI_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemBytes)));
        if (device < 64) allowed[device].store(true, std::memory_order_release);
    }
    args.places = std::min(args.first_tiles + args.second_tiles, sm_count() / kCtas);
    const int first = args.jobs[0].k_per_split, second = args.jobs[args.job_count - 1].k_per_split;
    args.ahead = args.first_tiles % args.places;
    args.catch_up = args.ahead > 0 && args.second_tiles > 0 ? first / second : 0;
    if (args.ahead == 0) args.catch_up = 0;
    args.early = dependent;
    KOEMI_CUDA_TRY(launch_programmatic(dependent, kernel, dim3(static_cast<unsigned>(args.places * kCtas)), dim3(kThreads), kSmemBytes, stream,
                                       dim3(kCtas, 1, 1), args));
    return KOEMI_OK;
}

// n / d == umulhi(n, magic) >> shift for 0 <= n < 2^31: magic = ceil(2^(32 + shift) / d) exceeds 2^(32 + shift) / d
// by less than 1, so the quotient by less than n / 2^(32 + shift) < 1 / d with 2^shift >= d / 2.
Divisor divisor(int d) {
    if (d == 1) return Divisor{0, 0};
    uint32_t shift = 0;
    while ((int64_t(2) << shift) < d) ++shift;
    return Divisor{static_cast<uint32_t>(((uint64_t(1) << (32 + shift)) + d - 1) / d), shift};
}

// Independent products in one launch, those of the longer K first; jobs: their
// epilogues' fields. dependent: the stream's last kernel, which writes none of
// the products' B, may still be running when this one starts; all before it has
// ended, because no launch that comes first in a call is a dependent one. The cut is that of all of them, wanted or not, so that the
// workspace does not depend on which are.
template <typename T, int kEpilogue>
int multiply(const Product *const *products, const Job *jobs, int count, const Cut &cut, char *partials, bool dependent,
              cudaStream_t stream) {
    constexpr bool gate = kEpilogue == kGate;
    const bool half = std::is_same<typename Operand16<T>::type, __half>::value;
    GemmArgs args{};
    args.status = device_status_word();
    int64_t tiles[2] = {0, 0}, most = 0;
    for (int i = 0; i < count; ++i) {
        const Product &p = *products[i];
        if (kEpilogue == kOut && jobs[i].out == nullptr) {  // not wanted: the others are cut as beside it
            partials += partial_bytes(cut, i, p, gate);
            continue;
        }
        const int at = args.job_count++;
        Job &j = args.jobs[at] = jobs[i];
        j.total_k = total_k_of(p, gate);
        j.first_blocks = blocks_of(p, 0);
        j.splits = cut.splits[i];
        j.k_per_split = static_cast<int>(ceil_div(j.total_k, j.splits));
        j.a_mn = p.a_mn;
        j.b_mn = p.b_mn;
        // few rows: the others of the accumulator hold whatever the stage held, and are not stored
        j.a_rows = !p.a_mn && p.m < kBM ? static_cast<int>(ceil_div(p.m, 8) * 8) : kBM;
        j.m = p.m;
        j.n = p.n;
        j.m_tiles = static_cast<int>(ceil_div(p.m, kBM * cut.ctas));
        const int64_t n_tiles = ceil_div(p.n, gate ? cut.tile_n / 2 : cut.tile_n);
        const int64_t own = j.m_tiles * n_tiles * j.splits;
        if (own > INT32_MAX / 2) return fail(KOEMI_ERR_INVALID, "feed-forward sizes are too large");
        j.tiles = static_cast<int>(own);
        j.band = std::min(j.m_tiles, 16 / cut.ctas);
        j.per_split = static_cast<int>(j.m_tiles * n_tiles);
        j.per_band = static_cast<int>(j.band * n_tiles);
        j.by_split = divisor(j.per_split);
        j.by_band = divisor(j.per_band);
        j.by_rows = divisor(j.band);
        j.by_last_rows = divisor(j.m_tiles % j.band == 0 ? j.band : j.m_tiles % j.band);
        j.partials = reinterpret_cast<float *>(partials);
        j.ld_partial = round16(p.n);
        partials += partial_bytes(cut, i, p, gate);
        j.idesc = 1u << 4 | (half ? 0u : 1u << 7 | 1u << 10) | (p.a_mn ? 1u << 15 : 0u) | (p.b_mn ? 1u << 16 : 0u) |
                  static_cast<uint32_t>(cut.tile_n >> 3) << 17 | static_cast<uint32_t>(kBM * cut.ctas >> 4) << 24;
        for (int s = 0; s < (gate ? 2 : p.segments); ++s) {
            int rc = s > 0 && gate ? KOEMI_OK : encode(&j.a[s], p.a[s], half, p.a_mn, j.a_rows);
            if (rc == KOEMI_OK) rc = encode(&j.b[s], p.b[s], half, p.b_mn, gate ? cut.tile_n / 2 : cut.tile_n / cut.ctas);
            if (rc != KOEMI_OK) return rc;
        }
        const bool first = args.jobs[0].k_per_split == j.k_per_split && args.first_jobs == at;
        tiles[first ? 0 : 1] += own;
        if (first) ++args.first_jobs;
        if (tiles[0] + tiles[1] > INT32_MAX / 2) return fail(KOEMI_ERR_INVALID, "feed-forward sizes are too large");
        if (j.splits > 1) most = std::max(most, ceil_div(p.n, 8) * p.m);
    }
    if (args.job_count == 0) return KOEMI_OK;
    args.first_tiles = static_cast<int>(tiles[0]);
    args.second_tiles = static_cast<int>(tiles[1]);
    int rc = KOEMI_OK;
    if (cut.tile_n == 64) {
        rc = launch_shape<T, kEpilogue, 64, 1>(args, dependent, stream);
    } else if (cut.tile_n == 128) {
        rc = cut.ctas == 2 ? launch_shape<T, kEpilogue, 128, 2>(args, dependent, stream) : launch_shape<T, kEpilogue, 128, 1>(args, dependent, stream);
    } else if constexpr (sizeof(T) == 2) {
        rc = cut.ctas == 2 ? launch_shape<T, kEpilogue, 256, 2>(args, dependent, stream) : launch_shape<T, kEpilogue, 256, 1>(args, dependent, stream);
    }
    if (rc != KOEMI_OK) return rc;
    if (most > 0) {
        KOEMI_CUDA_TRY(launch_programmatic(true, join_kernel<T, kEpilogue>, dim3(static_cast<unsigned>(ceil_div(most, 256)), static_cast<unsigned>(args.job_count)),
                                           dim3(256), 0, stream, dim3(1, 1, 1), args));
    }
    return KOEMI_OK;
}

// Hands out 256-byte aligned parts of a workspace; without one it only counts,
// for operands that TMA reads as they lie (direct) or for any.
struct Pool {
    char *base;
    size_t used = 0;
    bool direct = false;
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

// What the backward needs of the forward: h (in parts), a and b.
struct Kept {
    Parts h;
    float *a, *b;
    int64_t ld;
};

Kept kept_of(Pool &pool, int64_t rows, int64_t hidden, int dtype, bool with_slopes) {
    Kept kept{};
    kept.ld = round16(hidden);
    const size_t count = static_cast<size_t>(rows) * kept.ld;
    kept.h = Parts{pool.take(count * 2 * parts_of(dtype)), kept.ld, rows * kept.ld};
    if (with_slopes) {
        const size_t blocks = static_cast<size_t>(ceil_div(rows, 32)) * kept.ld / 16;
        kept.a = static_cast<float *>(pool.take(blocks * 512 * sizeof(float)));
        kept.b = static_cast<float *>(pool.take(blocks * 512 * sizeof(float)));
    }
    return kept;
}

// `src` as an operand: itself where TMA reads it, else a packed copy, noted in `jobs`.
Matrix operand(Pool &pool, const void *src, int64_t rows, int64_t columns, int64_t ld, int dtype, PackArgs &jobs, int &count) {
    const bool direct = pool.base == nullptr ? pool.direct : aligned(src, 16);
    if (dtype != KOEMI_F32 && direct && ld % 8 == 0) return Matrix{src, rows, columns, ld, 0, 1};
    const int64_t padded = round16(columns);
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
    Cut gate_cut, out_cut;
    char *partials;
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
    const Product *gate = &plan.gate, *out = &plan.out;
    const int sms = sm_count();
    plan.gate_cut = cut_of(&gate, 1, true, sms);
    plan.out_cut = cut_of(&out, 1, false, sms);
    plan.partials = static_cast<char *>(pool.take(std::max(partial_bytes(plan.gate_cut, &gate, 1, true), partial_bytes(plan.out_cut, &out, 1, false))));
}

// h of few rows, as the second product reads it.
size_t few_bytes(int64_t rows, int64_t hidden, int dtype) { return static_cast<size_t>(rows) * round16(hidden) * dtype_size(dtype); }

int too_small(size_t need) {
    return fail(KOEMI_ERR_WORKSPACE, "the feed-forward block needs %zu workspace bytes from a multiple of 256 here", need);
}

template <typename T>
int forward_few(const Problem &q, void *y, void *kept_base, void *workspace, size_t room, cudaStream_t stream) {
    Pool pool{static_cast<char *>(workspace)}, kept_pool{static_cast<char *>(kept_base)};
    void *h = pool.take(few_bytes(q.rows, q.hidden, q.dtype));
    if (pool.used > room) return too_small(pool.used);
    const Kept kept = kept_of(kept_pool, q.rows, q.hidden, q.dtype, true);
    const int rows = static_cast<int>(q.rows);
    FewArgs gate{q.x, q.wg, q.wv, q.bg, q.bv, q.ld_x, q.width, q.hidden, rows, 1, h, round16(q.hidden), kept.h, kept.a, kept.b, kept.ld / 16};
    if (kept_base == nullptr) gate.parts.base = nullptr;
    const int rc = few_rows<T, kGate>(gate, false, stream);
    if (rc != KOEMI_OK) return rc;
    const FewArgs out{h, q.wo, nullptr, q.bo, nullptr, round16(q.hidden), q.hidden, q.out_width, rows, 1, y, q.out_width, Parts{}, nullptr, nullptr, 0};
    return few_rows<T, kOut>(out, true, stream);
}

template <typename T>
int forward(const Problem &q, void *y, void *kept, void *workspace, size_t room, cudaStream_t stream) {
    if (q.rows <= few_limit(q.width, q.hidden, q.dtype)) return forward_few<T>(q, y, kept, workspace, room, stream);
    ForwardPlan plan{};
    Pool pool{static_cast<char *>(workspace)};
    plan_forward(plan, q, pool, static_cast<char *>(kept), kept != nullptr);
    if (pool.used > room) return too_small(pool.used);
    int rc = pack_all<T>(plan.jobs, plan.job_count, stream);
    if (rc != KOEMI_OK) return rc;
    const Product *first = &plan.gate, *second = &plan.out;
    Job gate{};
    gate.bias0 = q.bg;
    gate.bias1 = q.bv;
    gate.first = plan.kept.h;
    gate.a_kept = plan.kept.a;
    gate.b_kept = plan.kept.b;
    gate.kept_blocks = plan.kept.ld / 16;
    rc = multiply<T, kGate>(&first, &gate, 1, plan.gate_cut, plan.partials, false, stream);
    if (rc != KOEMI_OK) return rc;
    Job out{};
    out.bias0 = q.bo;
    out.out = y;
    out.ld_out = q.out_width;
    return multiply<T, kOut>(&second, &out, 1, plan.out_cut, plan.partials, true, stream);
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
    const Product *last[kMaxJobs];  // the products behind inner, the longer first, and where they go
    void *results[kMaxJobs];
    SumArgs sums;
    Cut inner_cut, last_cut;
    char *partials;
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
    const int64_t ld = round16(q.hidden);
    const size_t bytes = static_cast<size_t>(q.rows) * ld * 2 * parts_of(q.dtype);
    plan.dp = Parts{pool.take(bytes), ld, q.rows * ld};
    plan.dq = Parts{pool.take(bytes), ld, q.rows * ld};
    const Matrix dp = matrix_of(plan.dp, q.rows, q.hidden, q.dtype), dq = matrix_of(plan.dq, q.rows, q.hidden, q.dtype);
    plan.inner = Product{{plan.dy, {}}, {plan.wo, {}}, 1, false, true, q.rows, q.hidden};
    plan.values = Product{{dp, dq}, {plan.wg, plan.wv}, 2, false, true, q.rows, q.width};
    plan.gate_weight = Product{{dp, {}}, {plan.x, {}}, 1, true, true, q.hidden, q.width};
    plan.value_weight = Product{{dq, {}}, {plan.x, {}}, 1, true, true, q.hidden, q.width};
    plan.output_weight = Product{{plan.dy, {}}, {matrix_of(plan.kept.h, q.rows, q.hidden, q.dtype), {}}, 1, true, true, q.out_width, q.hidden};
    const Product *candidates[] = {&plan.gate_weight, &plan.value_weight, &plan.output_weight, &plan.values};
    void *results[] = {g.dwg, g.dwv, g.dwo, g.dx};
    const bool values_first = total_k_of(plan.values, false) > total_k_of(plan.gate_weight, false);
    for (int i = 0; i < kMaxJobs; ++i) {
        const int at = values_first ? (i + 3) % 4 : i;
        plan.last[i] = candidates[at];
        plan.results[i] = results[at];
    }
    const Product *inner = &plan.inner;
    const int sms = sm_count();
    plan.inner_cut = cut_of(&inner, 1, false, sms);
    plan.last_cut = cut_of(plan.last, kMaxJobs, false, sms);
    plan.partials = static_cast<char *>(pool.take(std::max(partial_bytes(plan.inner_cut, &inner, 1, false), partial_bytes(plan.last_cut, plan.last, kMaxJobs, false))));
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
int backward(const Problem &q, const Gradients &g, const void *kept, void *workspace, size_t room, cudaStream_t stream) {
    BackwardPlan plan{};
    Pool pool{static_cast<char *>(workspace)};
    plan_backward(plan, q, g, pool, static_cast<char *>(const_cast<void *>(kept)));
    if (pool.used > room) return too_small(pool.used);
    int rc = pack_all<T>(plan.jobs, plan.job_count, stream);
    if (rc != KOEMI_OK) return rc;
    bool dependent = false;
    if (g.dx != nullptr || g.dwg != nullptr || g.dwv != nullptr || g.dbg != nullptr || g.dbv != nullptr) {
        const Product *product = &plan.inner;
        Job inner{};
        inner.first = plan.dp;
        inner.second = plan.dq;
        inner.a_kept = plan.kept.a;
        inner.b_kept = plan.kept.b;
        inner.kept_blocks = plan.kept.ld / 16;
        rc = multiply<T, kInner>(&product, &inner, 1, plan.inner_cut, plan.partials, false, stream);
        dependent = true;
    }
    if (rc == KOEMI_OK) {
        Job jobs[kMaxJobs]{};
        for (int i = 0; i < kMaxJobs; ++i) {
            jobs[i].out = plan.results[i];
            jobs[i].ld_out = plan.last[i]->n;
        }
        rc = multiply<T, kOut>(plan.last, jobs, kMaxJobs, plan.last_cut, plan.partials, dependent, stream);
    }
    if (rc != KOEMI_OK) return rc;
    if (g.dbg != nullptr || g.dbv != nullptr || g.dbo != nullptr) {
        const unsigned columns = static_cast<unsigned>(plan.sums.ld);
        column_sums_kernel<T><<<dim3((columns + 31) / 32, plan.sums.chunks, 3), 256, 0, stream>>>(plan.sums);
        KOEMI_LAUNCH_CHECK();
        KOEMI_CUDA_TRY(launch_programmatic(true, column_totals_kernel<T>, dim3((columns + 127) / 128, 3), dim3(128), 0, stream, dim3(1, 1, 1), plan.sums));
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

int misaligned() { return fail(KOEMI_ERR_INVALID, "feed-forward pointers must be aligned to their type"); }

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
                                                           int dtype, int pass) {
    if (rows < 1 || check(rows, width, hidden_width, out_width, dtype) != KOEMI_OK) return 0;
    const Problem q{nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, rows, width, hidden_width, out_width, width, dtype};
    Pool pool{nullptr, 0, (pass & KOEMI_FEED_FORWARD_ALIGNED) != 0};
    if (pass & KOEMI_FEED_FORWARD_BACKWARD) {
        BackwardPlan plan{};
        plan_backward(plan, q, Gradients{}, pool, nullptr);
    } else if (rows <= few_limit(width, hidden_width, dtype)) {
        pool.take(few_bytes(rows, hidden_width, dtype));
    } else {
        ForwardPlan plan{};
        plan_forward(plan, q, pool, nullptr, (pass & KOEMI_FEED_FORWARD_KEEPS) != 0);
    }
    return std::max<size_t>(pool.used, 256);
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
    if (!aligned({values, gate_weight, value_weight, output_weight, gate_bias, value_bias, output_bias, out}, dtype_size(dtype))) return misaligned();
    if (kept != nullptr && (kept_bytes < koemi_dense_gated_feed_forward_kept(rows, hidden_width, dtype) || !aligned(kept, 256))) {
        return fail(KOEMI_ERR_WORKSPACE, "kept must hold %zu bytes from a multiple of 256", koemi_dense_gated_feed_forward_kept(rows, hidden_width, dtype));
    }
    if (workspace == nullptr || !aligned(workspace, 256)) return fail(KOEMI_ERR_WORKSPACE, "the workspace must start at a multiple of 256");
    const Problem q{values, gate_weight, value_weight, output_weight, gate_bias, value_bias, output_bias, rows, width, hidden_width, out_width, value_stride, dtype};
    if (dtype == KOEMI_F32) return forward<float>(q, out, kept, workspace, workspace_bytes, as_stream(stream));
    if (dtype == KOEMI_F16) return forward<__half>(q, out, kept, workspace, workspace_bytes, as_stream(stream));
    return forward<__nv_bfloat16>(q, out, kept, workspace, workspace_bytes, as_stream(stream));
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
    if (!aligned({values, gate_weight, value_weight, output_weight, grad_out, grad_values, grad_gate_weight, grad_value_weight, grad_output_weight,
                  grad_gate_bias, grad_value_bias, grad_output_bias}, dtype_size(dtype))) {
        return misaligned();
    }
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
    if (workspace == nullptr || !aligned(workspace, 256)) return fail(KOEMI_ERR_WORKSPACE, "the workspace must start at a multiple of 256");
    const Problem q{values, gate_weight, value_weight, output_weight, nullptr, nullptr, nullptr, rows, width, hidden_width, out_width, value_stride, dtype};
    const Gradients g{grad_out, grad_values, grad_gate_weight, grad_value_weight, grad_output_weight, grad_gate_bias, grad_value_bias, grad_output_bias};
    if (dtype == KOEMI_F32) return backward<float>(q, g, kept, workspace, workspace_bytes, as_stream(stream));
    if (dtype == KOEMI_F16) return backward<__half>(q, g, kept, workspace, workspace_bytes, as_stream(stream));
    return backward<__nv_bfloat16>(q, g, kept, workspace, workspace_bytes, as_stream(stream));
}
