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
//
// The logits are read once and their gradient is written once, in one pass
// over the rows, bound by HBM. Up to 1024 entries a warp holds a row in
// registers. Up to 64 KB a CTA of 64 to 256 threads does: a bulk copy brings
// the row into shared memory, a thread takes up to 256 bytes of it into
// registers, which frees the buffer for the next row's copy, adds its
// exponentials up relative to its warp's maximum, and the warps' (maximum,
// sum) pairs meet at a barrier; then it forms the gradient from its registers.
// fp32 entries are kept as exponentials, 16-bit ones as they came, with a
// second exponential: half the registers, so that 512 threads hold two rows of
// 64 KB and one row's arithmetic hides the other's latency. Up to 512 KB a
// cluster of 2 to 8 CTAs holds a row so, 64 KB a CTA, and the CTAs exchange
// their (maximum, sum) through distributed shared memory. Longer rows are
// walked twice from memory, the second time mostly from L2.
//
// Read and written at the device's copy bandwidth, these take (time, fraction
// of it): 8192 x 32768 bf16 182 us, 0.90; 8192 x 16384 fp32 189 us, 0.87; 1024
// x 131072 fp32 185 us, 0.89; 2048 x 131072 bf16 221 us, 0.74, with the cluster's
// exchange in every row; rows that are not whole packets pay a barrier more
// and the edges' own stores, 4096 x 50257 bf16 201 us, 0.63; evaluation reads
// only, and the exponentials' share shows: 8192 x 32768 bf16 105 us,
// 0.78. What these replaced: 128 bytes of a row to each of twice as many
// threads (half the work per row and warp that is not per entry) 8192 x 32768
// bf16 196 us; the next row's copy after the row's reduction, 187 us and 123 in
// evaluation; the row in chunks with a barrier each, 209 us and more; one CTA
// for 128 KB 4096 x 50257 bf16 196 us and 4096 x 32768 fp32 196 us, as the
// cluster, but 266 us for rows of 256 KB, walked.
// Every row belongs to one CTA or cluster and their sums are added in a fixed
// order by a second kernel, so equal inputs give equal bits.
#include "vec.cuh"

namespace koemi {
namespace {

constexpr int kPolicyBlocks = 2368;     // most CTAs of a launch: 16 per SM
constexpr int kWarpRow = 1024;          // entries a warp holds
constexpr int kSmBytes = 128 * 1024;    // of rows, in the registers of an SM
constexpr int kSliceBytes = 64 * 1024;  // of a row, in one CTA: longer rows are split over a cluster
constexpr int kMaxCluster = 8;
constexpr int64_t kCountedRows = 16384; // up to here every CTA counts the valid rows itself
constexpr float kLog2e = 1.4426950408889634f;

// Row r of the logits starts at (r / inner) * outer_stride + (r % inner) *
// inner_stride elements.
struct PolicyRows {
    int64_t rows, vocab, inner, outer_stride, inner_stride;  // rows up to 2^31, inner up to rows
    __device__ __forceinline__ int64_t start(int64_t row) const {
        const uint32_t r = static_cast<uint32_t>(row), n = static_cast<uint32_t>(inner), outer = r / n;
        return outer * outer_stride + (r - outer * n) * inner_stride;
    }
};

struct PolicyTerms {
    const int64_t *targets;
    const float *old, *advantages, *reference;  // reference may be NULL: no KL term
    const uint8_t *valid;                       // may be NULL: every row
    float clip_low, clip_high, beta;
};

__device__ __forceinline__ bool aligned_to(const void *p, unsigned bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// 1 / (valid rows), by one CTA. 16 flags at a time where they are aligned.
__device__ float inverse_count(const uint8_t *valid, int64_t rows) {
    __shared__ int32_t sums[32];
    if (valid == nullptr) return 1.0f / static_cast<float>(rows > 0 ? rows : 1);
    int32_t count = 0;
    const int64_t packets = aligned_to(valid, 16) ? rows / 16 : 0;
    for (int64_t i = threadIdx.x; i < packets; i += blockDim.x) {
        const uint4 raw = load_cached(valid + 16 * i);
        // a bool is one byte of value 0 or 1
        count += __popc(__vcmpne4(raw.x, 0) & 0x01010101u) + __popc(__vcmpne4(raw.y, 0) & 0x01010101u) +
                 __popc(__vcmpne4(raw.z, 0) & 0x01010101u) + __popc(__vcmpne4(raw.w, 0) & 0x01010101u);
    }
    for (int64_t i = 16 * packets + threadIdx.x; i < rows; i += blockDim.x) count += valid[i] != 0;
    count = __reduce_add_sync(0xffffffffu, count);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = count;
    __syncthreads();
    int64_t all = 0;
    for (unsigned w = 0; w < blockDim.x / 32; ++w) all += sums[w];
    __syncthreads();
    return 1.0f / static_cast<float>(all > 0 ? all : 1);
}

__global__ void policy_count_kernel(const uint8_t *__restrict__ valid, int64_t rows, float *__restrict__ inverse) {
    const float v = inverse_count(valid, rows);
    if (threadIdx.x == 0) *inverse = v;
}

__device__ __forceinline__ float ex2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Two fp32 operations in one issue slot.
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
template <int kWidth>
__device__ __forceinline__ float packet_max(const float (&v)[kWidth]) {
    float m = v[0];
#pragma unroll
    for (int i = 1; i < kWidth; ++i) m = fmaxf(m, v[i]);
    return m;
}

// e^(v - m), m a maximum: the difference is exact to half a unit in its last
// place whatever the logits' magnitude (the type's lowest value in every entry
// gives a uniform row); ex2.approx adds 2 units. A maximum of nothing but -inf
// counts as 0, so that its entries give 0.
__device__ __forceinline__ float origin(float max) { return max == -INFINITY ? 0.0f : max; }
__device__ __forceinline__ float exp_from(float v, float from) { return ex2_approx((v - from) * kLog2e); }

__device__ __forceinline__ float redux_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
// A maximum and the sum of e^(entry - it) over a thread's, a warp's, a row's entries.
struct Partial {
    float max, sum;
};
__device__ __forceinline__ Partial warp_merge(Partial p) {
    const float m = redux_max(p.max);
    return Partial{m, warp_sum(p.sum * exp_from(p.max, origin(m)))};
}
__device__ __forceinline__ float lse_of(Partial p) { return p.max + logf(p.sum); }

// What a forward kernel writes beside the gradient. For the backward a row
// leaves its maximum and its sum, which give the same softmax as the forward's;
// with sums NULL only its log-sum-exp, which rounds at the logits' magnitude:
// near 1e6 its probabilities are 2% off, and a row of the type's lowest value,
// which absorbs the logarithm, gets 1 in every entry for 1 / vocab.
struct PolicyOut {
    const float *inverse;  // NULL: the CTA counts the valid rows
    float *log_probs, *lse, *sums, *slopes;  // lse: the maxima where sums is given
    double2 *partials;
    __device__ __forceinline__ void keep(int64_t index, Partial p, float slope) const {
        lse[index] = sums != nullptr ? p.max : lse_of(p);
        if (sums != nullptr) sums[index] = p.sum;
        slopes[index] = slope;
    }
    __device__ __forceinline__ void skip(int64_t index) const {
        log_probs[index] = 0.0f;
        keep(index, Partial{0.0f, 1.0f}, 0.0f);
    }
};

// A row's scalars, and what follows from its log-sum-exp: every thread takes
// the slope (two ex2.approx), one thread per row the loss and the KL term
// (expf and expm1f: exp(d) - d - 1 cancels).
struct __align__(16) RowTerms {
    int target;  // -1 outside the vocabulary, -2 in a row that is not valid
    float old, advantage, reference;
    __device__ __forceinline__ bool valid() const { return target != -2; }
};
__device__ __forceinline__ RowTerms load_terms(const PolicyTerms &terms, int64_t index, int vocab) {
    if (terms.valid != nullptr && terms.valid[index] == 0) return RowTerms{-2, 0.0f, 0.0f, 0.0f};
    const int64_t id = terms.targets[index];
    return RowTerms{id >= 0 && id < vocab ? static_cast<int>(id) : -1, terms.old[index], terms.advantages[index],
                    terms.reference != nullptr ? terms.reference[index] : 0.0f};
}
struct RowScalars : RowTerms {
    float chosen;  // the target's logit
    __device__ __forceinline__ RowScalars(const RowTerms &row, float logit) : RowTerms(row), chosen(target >= 0 ? logit : NAN) {}
    // from the maximum, not from the log-sum-exp, which rounds at its own magnitude
    __device__ __forceinline__ float log_prob(Partial p) const { return (chosen - p.max) - logf(p.sum); }
    // d loss / d log-prob, of a row alone
    __device__ __forceinline__ float slope(const PolicyTerms &terms, float lp) const {
        const float r = exp_from(lp, old), free = r * advantage;
        const float clipped = fminf(fmaxf(r, 1.0f - terms.clip_low), 1.0f + terms.clip_high) * advantage;
        float s = free <= clipped ? -free : 0.0f;
        if (terms.reference != nullptr) s += terms.beta * (1.0f - exp_from(reference, lp));
        return isnan(free) || isnan(clipped) ? NAN : s;
    }
    __device__ void add_loss(const PolicyTerms &terms, float lp, double &loss, double &kl) const {
        const float r = expf(lp - old), free = r * advantage;
        const float clipped = fminf(fmaxf(r, 1.0f - terms.clip_low), 1.0f + terms.clip_high) * advantage;
        loss -= isnan(free) || isnan(clipped) ? NAN : fminf(free, clipped);
        if (terms.reference != nullptr) {
            const float d = reference - lp, k = expm1f(d) - d;
            kl += k;
            loss += terms.beta * k;
        }
    }
    // the row's results, by one thread
    __device__ void finish(const PolicyTerms &terms, const PolicyOut &out, int64_t index, float lp, Partial p,
                           float scaled_slope, double &loss, double &kl) const {
        add_loss(terms, lp, loss, kl);
        out.log_probs[index] = lp;
        out.keep(index, p, scaled_slope);
    }
};

// Up to 1024 entries: a warp per row, entry v in lane v % 32.
template <typename T, int kPer>
__global__ __launch_bounds__(256) void policy_warp_kernel(PolicyRows shape, PolicyTerms terms,
                                                          const T *__restrict__ logits, PolicyOut result,
                                                          T *__restrict__ grad_logits) {
    __shared__ double2 sums[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, vocab = static_cast<int>(shape.vocab);
    const float scale = result.inverse != nullptr ? *result.inverse : inverse_count(terms.valid, shape.rows);
    double loss_sum = 0.0, kl_sum = 0.0;  // advantages cancel: fp32 sums would lose what is left
    for (int64_t row = int64_t(blockIdx.x) * 8 + warp; row < shape.rows; row += int64_t(gridDim.x) * 8) {
        T *out = grad_logits == nullptr ? nullptr : grad_logits + row * vocab;
        const RowTerms row_terms = load_terms(terms, row, vocab);
        if (!row_terms.valid()) {
            if (out != nullptr) {
                for (int v = lane; v < vocab; v += 32) out[v] = from_acc<T>(0.0f);
            }
            if (lane == 0) result.skip(row);
            continue;
        }
        const T *in = logits + shape.start(row);
        const RowScalars scalars(row_terms, row_terms.target >= 0 ? to_acc(in[row_terms.target]) : NAN);
        // loaded as they are and converted later: every load is on its way first
        T raw[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            raw[j] = from_acc<T>(-INFINITY);
            if (lane + 32 * j < vocab) raw[j] = in[lane + 32 * j];
        }
        float e[kPer];
        Partial p{-INFINITY, 0.0f};
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            e[j] = to_acc(raw[j]);
            p.max = fmaxf(p.max, e[j]);
        }
        p.max = redux_max(p.max);
        const float from = origin(p.max);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            e[j] = exp_from(e[j], from);
            p.sum += e[j];
        }
        p.sum = warp_sum(p.sum);
        const float lp = scalars.log_prob(p), slope = scalars.slope(terms, lp) * scale;
        if (lane == 0) scalars.finish(terms, result, row, lp, p, slope, loss_sum, kl_sum);
        if (out != nullptr) {
            const float factor = -slope / p.sum;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const int v = lane + 32 * j;
                if (v < vocab) out[v] = from_acc<T>(fmaf(e[j], factor, v == scalars.target ? slope : 0.0f));
            }
        }
    }
    if (lane == 0) sums[warp] = make_double2(loss_sum, kl_sum);
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) {
            loss_sum += sums[w].x;
            kl_sum += sums[w].y;
        }
        result.partials[blockIdx.x] = make_double2(loss_sum, kl_sum);
    }
}

// A row in packets of 16 bytes at 16-byte boundaries: packet c holds entries
// c width - skip and following; the first and the last may be partly outside.
template <typename T>
struct Packets {
    static constexpr int kWidth = Pack<T>::kWidth;
    const T *base;  // the boundary at or before the row's start
    int skip, vocab, count;
    int first, end;  // packets first .. end - 1 are whole
    __device__ __forceinline__ Packets(const T *row, int vocab_) : vocab(vocab_) {
        skip = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
        base = row - skip;
        count = (skip + vocab + kWidth - 1) / kWidth;
        first = skip > 0 ? 1 : 0;
        end = (skip + vocab) / kWidth;
    }
    __device__ __forceinline__ bool whole(int c) const { return c >= first && c < end; }
    // packet c lies inside the tensor that ends before `tensor_end`
    __device__ __forceinline__ bool inside(int c, const T *tensor, const T *tensor_end) const {
        const T *packet = base + int64_t(c) * kWidth;
        return packet >= tensor && packet + kWidth <= tensor_end;
    }
    __device__ __forceinline__ bool in_row(int c, int i) const {
        return static_cast<unsigned>(c * kWidth + i - skip) < static_cast<unsigned>(vocab);
    }
    // entries of a packet that is partly (or all) outside, one by one
    __device__ __forceinline__ void load_partly(int c, float (&v)[kWidth]) const {
#pragma unroll
        for (int i = 0; i < kWidth; ++i) v[i] = in_row(c, i) ? to_acc(base[int64_t(c) * kWidth + i]) : -INFINITY;
    }
    // Whether the packets of the row at `out` lie as this row's.
    __device__ __forceinline__ bool fits(const T *out) const {
        return reinterpret_cast<uintptr_t>(out) % 16 / sizeof(T) == static_cast<unsigned>(skip);
    }
    // v into packet c of the row at `out`: whole, or one by one
    __device__ __forceinline__ void store(T *out, bool whole_packet, int c, const float (&v)[kWidth]) const {
        T *to = out - skip + int64_t(c) * kWidth;
        if (whole_packet) {
            __stcs(reinterpret_cast<uint4 *>(to), pack(v, T()));
            return;
        }
#pragma unroll
        for (int i = 0; i < kWidth; ++i) {
            if (in_row(c, i)) to[i] = from_acc<T>(v[i]);
        }
    }
};

// Zeros into a row of the gradient, by kRowThreads neighbouring threads: from
// packet `first` on, `count` of them or, the last slice, to the row's end.
template <typename T, int kRowThreads>
__device__ void clear_row(T *out, int vocab, int first = 0, int count = 0) {
    const Packets<T> packets(out, vocab);
    const float zeros[Packets<T>::kWidth] = {};
    const int end = count > 0 ? first + count : packets.count;
    for (int c = first + static_cast<int>(threadIdx.x % kRowThreads); c < end; c += kRowThreads) packets.store(out, packets.whole(c), c, zeros);
}

// The warps' partials of a row, merged by every warp alike: the row's partial
// from one barrier. `place` alternates between two rows.
template <int kThreads>
__device__ __forceinline__ Partial block_merge(Partial p, Partial (*place)[32], int parity) {
    constexpr int kWarps = kThreads / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) place[parity][warp] = p;
    __syncthreads();
    p = lane < kWarps ? place[parity][lane] : Partial{-INFINITY, 0.0f};
    return warp_merge(p);
}

__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_addr(dst)),
                 "l"(src), "r"(bytes), "r"(smem_addr(bar))
                 : "memory");
}

// Two entries at a time of a packet's words.
__device__ __forceinline__ float2 word_of(uint32_t w, __nv_bfloat16) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&w)); }
__device__ __forceinline__ float2 word_of(uint32_t w, __half) { return __half22float2(*reinterpret_cast<__half2 *>(&w)); }
// The larger entries of two packets; a NaN is passed over (the sum shows it).
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b, __nv_bfloat16) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162 *>(&a), *reinterpret_cast<__nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
}
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b, __half) {
    const __half2 m = __hmax2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
}
template <typename T>
__device__ __forceinline__ float row_part_max(const uint4 &m, T type) {
    const uint32_t w = word_max(word_max(m.x, m.y, type), word_max(m.z, m.w, type), type);
    const float2 v = word_of(w, type);
    return fmaxf(v.x, v.y);
}
__device__ __forceinline__ float row_part_max(const uint4 &m, float) {
    return fmaxf(fmaxf(__uint_as_float(m.x), __uint_as_float(m.y)), fmaxf(__uint_as_float(m.z), __uint_as_float(m.w)));
}
template <typename T>
__device__ __forceinline__ uint4 packet_larger(const uint4 &a, const uint4 &b, T type) {
    return make_uint4(word_max(a.x, b.x, type), word_max(a.y, b.y, type), word_max(a.z, b.z, type), word_max(a.w, b.w, type));
}
__device__ __forceinline__ uint4 packet_larger(const uint4 &a, const uint4 &b, float) {
    auto larger = [](uint32_t x, uint32_t y) { return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y))); };
    return make_uint4(larger(a.x, b.x), larger(a.y, b.y), larger(a.z, b.z), larger(a.w, b.w));
}
__device__ __forceinline__ float2 exp_from(float2 v, float from) {
    v = mul2(add2(v, make_float2(-from, -from)), make_float2(kLog2e, kLog2e));
    return make_float2(ex2_approx(v.x), ex2_approx(v.y));
}

__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Four floats into the same place of CTA `rank` of the cluster, counted on its
// barrier in the same place as `bar`.
__device__ __forceinline__ void store_to_rank(float4 *local, uint64_t *bar, int rank, float4 v) {
    asm volatile(
        "{\n\t.reg .b32 a, b;\n\tmapa.shared::cluster.u32 a, %0, %2;\n\tmapa.shared::cluster.u32 b, %1, %2;\n\t"
        "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [a], {%3, %4, %5, %6}, [b];\n\t}" ::"r"(smem_addr(local)),
        "r"(smem_addr(bar)), "r"(rank), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
        : "memory");
}

// A CTA per row at a time, kThreadBytes of it in a thread's registers. kExact:
// every row is whole packets (16-byte aligned rows, a vocabulary of whole
// packets). [logits, logits_end) is the tensor, with whatever its strides skip.
// kSplit: a cluster per row; each CTA takes `slice` packets of it, the last
// one the rest, and they give each other their (maximum, sum, target's logit).
template <typename T, int kThreads, int kThreadBytes, bool kExact, bool kSplit>
__global__ __launch_bounds__(kThreads, kSmBytes / kThreadBytes / kThreads) void policy_row_kernel(
    PolicyRows shape, PolicyTerms terms, const T *__restrict__ logits, const T *logits_end, PolicyOut result,
    T *__restrict__ grad_logits, int buffers, uint32_t buffer_bytes, int cluster, int slice, int *status) {
    constexpr int kWidth = Pack<T>::kWidth, kPackets = kThreadBytes / 16;
    // whether the next row is loaded as soon as this one is in registers, at a
    // barrier more, or after the row's only barrier: small rows have several
    // buffers and many CTAs
    constexpr bool kEarly = kThreads > 64;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    constexpr int kTable = 64;
    __shared__ uint64_t full[4];
    __shared__ Partial merged[2][32];
    // the scalars of kTable of the CTA's rows, loaded at once: their latency is
    // paid once per table and not in every row
    __shared__ RowTerms table[kTable];
    __shared__ float4 met[2][kSplit ? kMaxCluster : 1];  // the CTAs' parts of two rows
    __shared__ uint64_t meeting[2];
    const int rank = kSplit ? static_cast<int>(blockIdx.x % cluster) : 0, first = rank * slice;  // the slice's first packet
    const int64_t first_row = kSplit ? blockIdx.x / cluster : blockIdx.x, row_step = kSplit ? gridDim.x / cluster : gridDim.x;
    const bool last_slice = !kSplit || rank == cluster - 1;
    int64_t table_end = 0;  // rows of the CTA's that have been in the table
    const int vocab = static_cast<int>(shape.vocab);
    auto live = [&](int64_t row, int64_t index) {
        if (index < table_end) return table[index % kTable].valid();
        return terms.valid == nullptr || terms.valid[row] != 0;
    };
    // thread 0's: the next row to load (nothing: bytes 0), found while there is time
    __shared__ struct {
        const T *from;
        int64_t row, index;
        uint32_t to, bytes;
        int buffer, loads;
    } next;
    auto find_next = [&] {
        for (; next.row < shape.rows && !live(next.row, next.index); next.row += row_step) ++next.index;
        next.bytes = 0;
        if (next.row >= shape.rows) return;
        const Packets<T> packets(logits + shape.start(next.row), vocab);
        const int from = kExact || first > 0 || packets.inside(0, logits, logits_end) ? first : first + 1;
        const int to = !last_slice ? first + slice
                       : kExact || packets.inside(packets.count - 1, logits, logits_end) ? packets.count : packets.count - 1;
        next.from = packets.base + int64_t(from) * kWidth;
        next.to = next.buffer * buffer_bytes + (from - first) * 16;
        next.bytes = static_cast<uint32_t>(to - from) * 16;
        next.row += row_step;
        ++next.index;
    };
    auto load_next = [&] {
        const uint32_t bytes = next.bytes;
        if (bytes == 0) return;
        uint64_t *bar = &full[next.buffer];
        mbar_arrive_expect_tx(bar, bytes);
        bulk_load(smem_raw + next.to, next.from, bytes, bar);
        next.buffer = next.buffer + 1 == buffers ? 0 : next.buffer + 1;
        ++next.loads;
    };
    if (threadIdx.x == 0) {
        for (int b = 0; b < buffers; ++b) mbar_init(&full[b], 1);
        next.row = first_row;
        next.index = next.buffer = next.loads = 0;
        mbar_init(&meeting[0], 1);
        mbar_init(&meeting[1], 1);
        fence_barrier_init();
    }
    if (kSplit) cluster_sync();  // every CTA's barriers are ready before one stores into another
    const float scale = result.inverse != nullptr ? *result.inverse : inverse_count(terms.valid, shape.rows);
    double loss_sum = 0.0, kl_sum = 0.0;  // advantages cancel: fp32 sums would lose what is left
    bool dead = false;  // a copy never arrived: go on without waiting or loading
    int taken = 0, buffer = 0;
    uint32_t parity = 0;
    int64_t index = 0;
    for (int64_t row = first_row; row < shape.rows; row += row_step, ++index) {
        if (index == table_end) {
            __syncthreads();
            if (threadIdx.x < kTable) {
                const int64_t r = row + int64_t(threadIdx.x) * row_step;
                if (r < shape.rows) table[threadIdx.x] = load_terms(terms, r, vocab);
            }
            table_end += kTable;
            __syncthreads();
            if (threadIdx.x == 0 && index == 0) {
                for (int b = 0; b < buffers; ++b) {
                    find_next();
                    load_next();
                }
                find_next();
            }
        }
        const RowTerms row_terms = table[index % kTable];
        T *out = grad_logits == nullptr ? nullptr : grad_logits + row * vocab;
        if (!row_terms.valid()) {
            if (out != nullptr) clear_row<T, kThreads>(out, vocab, first, last_slice ? 0 : slice);
            if (threadIdx.x == kThreads - 1 && rank == 0) result.skip(row);
            continue;
        }
        const T *in = logits + (kExact ? 0 : shape.start(row));
        const Packets<T> packets(in, vocab);
        const int count = last_slice ? packets.count - first : slice;  // of the slice
        unsigned char *place = smem_raw + buffer * buffer_bytes;
        const uint4 *staged = reinterpret_cast<const uint4 *>(place) + threadIdx.x;
        if (!dead) dead = !mbar_wait_bounded(&full[buffer], parity, status);
        if (++buffer == buffers) {
            buffer = 0;
            parity ^= 1;
        }
        // the entries of the first and the last packet, a thread each: in
        // shared memory those outside the row become -inf
        const int edge_packet = threadIdx.x < kWidth ? 0 : packets.count - 1, edge_place = threadIdx.x % kWidth;
        const bool on_edge = !kExact && threadIdx.x < 2 * kWidth && !packets.whole(edge_packet) &&
                             (threadIdx.x < kWidth ? rank == 0 : last_slice);
        T edge = from_acc<T>(-INFINITY);
        if (!kExact) {
            if (on_edge) {
                const int entry = edge_packet * kWidth + edge_place;
                T *cell = reinterpret_cast<T *>(place) + (entry - first * kWidth);
                if (packets.in_row(edge_packet, edge_place)) {
                    edge = packets.inside(edge_packet, logits, logits_end) ? *cell : packets.base[entry];
                }
                *cell = edge;
                fence_proxy_async();  // before a copy takes the place
            }
            __syncthreads();
        }

        // the target's entry and packet, and the packet's place in the slice
        const int at = row_terms.target + packets.skip, packet = row_terms.target >= 0 ? at / kWidth : -1;
        const bool here = packet >= first && packet < first + count;
        float chosen = here ? to_acc(reinterpret_cast<const T *>(place)[at - first * kWidth]) : NAN;
        uint4 kept[kPackets];
        if (kExact && count == kPackets * kThreads) {
#pragma unroll
            for (int j = 0; j < kPackets; ++j) kept[j] = staged[j * kThreads];
        } else {
            float nothing[kWidth];
#pragma unroll
            for (int i = 0; i < kWidth; ++i) nothing[i] = -INFINITY;
#pragma unroll
            for (int j = 0; j < kPackets; ++j) {
                kept[j] = pack(nothing, T());
                if (static_cast<int>(threadIdx.x) + j * kThreads < count) kept[j] = staged[j * kThreads];
            }
        }
        if (kEarly) {
            __syncthreads();
            if (threadIdx.x == 0 && !dead) load_next();
        }
        uint4 largest = kept[0];
#pragma unroll
        for (int j = 1; j < kPackets; ++j) largest = packet_larger(largest, kept[j], T());
        Partial p{redux_max(row_part_max(largest, T())), 0.0f};
        const float from = origin(p.max);
        float2 sums = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < kPackets; ++j) {
            if (j * kThreads >= count) continue;
            if constexpr (sizeof(T) == 4) {
                const float2 x = exp_from(make_float2(__uint_as_float(kept[j].x), __uint_as_float(kept[j].y)), from);
                const float2 y = exp_from(make_float2(__uint_as_float(kept[j].z), __uint_as_float(kept[j].w)), from);
                sums = add2(sums, add2(x, y));
                kept[j] = make_uint4(__float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(y.x), __float_as_uint(y.y));
            } else {
                sums = add2(sums, exp_from(word_of(kept[j].x, T()), from));
                sums = add2(sums, exp_from(word_of(kept[j].y, T()), from));
                sums = add2(sums, exp_from(word_of(kept[j].z, T()), from));
                sums = add2(sums, exp_from(word_of(kept[j].w, T()), from));
            }
        }
        p.sum = warp_sum(sums.x + sums.y);
        Partial all = block_merge<kThreads>(p, merged, taken & 1);
        if (kSplit) {
            float4 *parts = met[taken & 1];
            uint64_t *bar = &meeting[taken & 1];
            // a CTA that gave up sends no more: the others give up too
            if (threadIdx.x == 0 && !dead) mbar_arrive_expect_tx(bar, cluster * sizeof(float4));
            if (threadIdx.x < cluster && !dead) store_to_rank(parts + rank, bar, threadIdx.x, make_float4(all.max, all.sum, chosen, 0.0f));
            if (!dead) dead = !mbar_wait_bounded<true>(bar, static_cast<uint32_t>(taken >> 1) & 1, status);
            const int lane = threadIdx.x & 31;
            all = warp_merge(lane < cluster ? Partial{parts[lane].x, parts[lane].y} : Partial{-INFINITY, 0.0f});
            if (packet >= 0) chosen = parts[packet / slice < cluster ? packet / slice : cluster - 1].z;
        }
        if (threadIdx.x == 0) {
            if (!kEarly && !dead) load_next();
            find_next();
        }
        ++taken;

        const RowScalars scalars(row_terms, chosen);
        const float lp = scalars.log_prob(all), slope = scalars.slope(terms, lp) * scale;
        if (threadIdx.x == kThreads - 1 && rank == 0) scalars.finish(terms, result, row, lp, all, slope, loss_sum, kl_sum);
        if (out != nullptr) {
            // of an fp32 warp with nothing but -inf: 0
            const float factor = -__fdividef(slope, all.sum) * (sizeof(T) == 4 ? exp_from(p.max, all.max) : 1.0f);
            const bool fits = kExact || packets.fits(out);
#pragma unroll
            for (int j = 0; j < kPackets; ++j) {
                const int c = first + threadIdx.x + j * kThreads;
                if (c >= first + count) continue;
                // from here a value of its own: else the first loop's fp32
                // entries would be kept across the barrier, and spilled
                asm("" : "+r"(kept[j].x), "+r"(kept[j].y), "+r"(kept[j].z), "+r"(kept[j].w));
                float v[kWidth];
                unpack(kept[j], v, T());
#pragma unroll
                for (int i = 0; i < kWidth; i += 2) {
                    float2 e = make_float2(v[i], v[i + 1]);
                    if constexpr (sizeof(T) == 2) e = exp_from(e, all.max);
                    e = mul2(e, make_float2(factor, factor));
                    v[i] = e.x;
                    v[i + 1] = e.y;
                }
                if (kExact || (fits && packets.whole(c))) {
                    packets.store(out, true, c, v);
                } else if (!fits) {
                    packets.store(out, false, c, v);
                }
            }
            // the entries of packets that are not whole, and the target's again
            // by the thread that stored it
            const float weight = -__fdividef(slope, all.sum);
            const bool edges = !kExact && fits, target_on_edge = edges && !packets.whole(packet);
            if (edges && on_edge && packets.in_row(edge_packet, edge_place)) {
                const int v = edge_packet * kWidth + edge_place - packets.skip;
                out[v] = from_acc<T>(fmaf(exp_from(to_acc(edge), all.max), weight, v == scalars.target ? slope : 0.0f));
            }
            if (here && (packet - first) % kThreads == threadIdx.x && !target_on_edge) {
                out[scalars.target] = from_acc<T>(fmaf(exp_from(scalars.chosen, all.max), weight, slope));
            }
        }
    }
    if (threadIdx.x == 0 && dead) {  // no copy may land after the CTA's end
        for (int b = 0; b < buffers; ++b) {
            const int loads = (next.loads + buffers - 1 - b) / buffers;
            if (loads > 0) mbar_wait_bounded(&full[b], (loads - 1) & 1, status);
        }
    }
    if (kSplit) cluster_sync();  // no CTA ends while another may store into it
    if (threadIdx.x == kThreads - 1 && rank == 0) result.partials[first_row] = make_double2(loss_sum, kl_sum);
}

// Longer rows, in blocks of 1024 threads x 32 entries, walked twice.
constexpr int kWalkThreads = 1024;
template <typename T>
__global__ __launch_bounds__(kWalkThreads) void policy_walk_kernel(PolicyRows shape, PolicyTerms terms,
                                                                   const T *__restrict__ logits, PolicyOut result,
                                                                   T *__restrict__ grad_logits) {
    constexpr int kWidth = Pack<T>::kWidth, kPackets = 32 / kWidth / 2;  // in flight per thread
    __shared__ Partial merged[2][32];
    const int vocab = static_cast<int>(shape.vocab);
    const float scale = result.inverse != nullptr ? *result.inverse : inverse_count(terms.valid, shape.rows);
    double loss_sum = 0.0, kl_sum = 0.0;  // advantages cancel: fp32 sums would lose what is left
    int taken = 0;
    for (int64_t row = blockIdx.x; row < shape.rows; row += gridDim.x) {
        T *out = grad_logits == nullptr ? nullptr : grad_logits + row * vocab;
        const RowTerms row_terms = load_terms(terms, row, vocab);
        if (!row_terms.valid()) {
            if (out != nullptr) clear_row<T, kWalkThreads>(out, vocab);
            if (threadIdx.x == 0) result.skip(row);
            continue;
        }
        const T *in = logits + shape.start(row);
        const RowScalars scalars(row_terms, row_terms.target >= 0 ? to_acc(in[row_terms.target]) : NAN);
        const Packets<T> packets(in, vocab);
        auto walk = [&](auto &&each) {
            for (int first = threadIdx.x; first < packets.count; first += kPackets * kWalkThreads) {
                uint4 raw[kPackets];
#pragma unroll
                for (int j = 0; j < kPackets; ++j) {
                    const int c = first + j * kWalkThreads;
                    raw[j] = packets.whole(c) ? load_cached(packets.base + int64_t(c) * kWidth) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < kPackets; ++j) {
                    const int c = first + j * kWalkThreads;
                    if (c >= packets.count) continue;
                    float v[kWidth];
                    if (packets.whole(c)) {
                        unpack(raw[j], v, T());
                    } else {
                        packets.load_partly(c, v);
                    }
                    each(c, v);
                }
            }
        };
        Partial p{-INFINITY, 0.0f};
        walk([&](int, const float (&v)[kWidth]) {
            const float m = packet_max(v);
            if (m > p.max) {
                p.sum *= exp_from(p.max, m);
                p.max = m;
            }
            const float from = origin(p.max);
#pragma unroll
            for (int i = 0; i < kWidth; ++i) p.sum += exp_from(v[i], from);
        });
        const Partial all = block_merge<kWalkThreads>(warp_merge(p), merged, taken++ & 1);
        const float lp = scalars.log_prob(all), slope = scalars.slope(terms, lp) * scale;
        if (threadIdx.x == 0) scalars.finish(terms, result, row, lp, all, slope, loss_sum, kl_sum);
        if (out != nullptr) {
            const float factor = -slope / all.sum;
            const bool fits = packets.fits(out);
            const int at = scalars.target + packets.skip, packet = scalars.target >= 0 ? at / kWidth : -1;
            walk([&](int c, float (&v)[kWidth]) {
#pragma unroll
                for (int i = 0; i < kWidth; ++i) v[i] = exp_from(v[i], all.max) * factor;
                if (packet == c) {
#pragma unroll
                    for (int i = 0; i < kWidth; ++i) v[i] += at % kWidth == i ? slope : 0.0f;
                }
                packets.store(out, fits && packets.whole(c), c, v);
            });
        }
    }
    if (threadIdx.x == 0) result.partials[blockIdx.x] = make_double2(loss_sum, kl_sum);
}

constexpr int kFinishThreads = 256;
__global__ __launch_bounds__(kFinishThreads) void policy_finish_kernel(const double2 *__restrict__ partials, int count,
                                                                       const float *__restrict__ inverse,
                                                                       const uint8_t *__restrict__ valid, int64_t rows,
                                                                       float *__restrict__ loss, float *__restrict__ kl) {
    __shared__ double sums[2][kFinishThreads / 32];
    double l = 0.0, k = 0.0;
    for (int i = threadIdx.x; i < count; i += kFinishThreads) {
        l += partials[i].x;
        k += partials[i].y;
    }
    const float scale = inverse != nullptr ? *inverse : inverse_count(valid, rows);
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, offset);
        k += __shfl_xor_sync(0xffffffffu, k, offset);
    }
    if ((threadIdx.x & 31) == 0) {
        sums[0][threadIdx.x >> 5] = l;
        sums[1][threadIdx.x >> 5] = k;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kFinishThreads / 32; ++w) {
            l += sums[0][w];
            k += sums[1][w];
        }
        *loss = static_cast<float>(l * scale);
        *kl = static_cast<float>(k * scale);
    }
}

// The gradient from what the forward kept of its rows: kRowThreads threads take
// a row's packets (or, grid.y > 1, every grid.y-th run of them). held: grad_logits holds it for a
// factor of one, which stays. A 16-bit gradient under another factor is formed
// again from the logits: as many bytes as scaling it, and one rounding, where a
// product of the rounded gradient would have two (8192 x 32768 bf16, 75% of the
// rows valid: 166 us, the product 175; 65536 x 1000 53 and 48).
constexpr int kBackwardThreads = 256;
template <typename T, int kRowThreads>
__global__ __launch_bounds__(kBackwardThreads) void policy_backward_kernel(
    PolicyRows shape, const T *__restrict__ logits, const int64_t *__restrict__ targets,
    const uint8_t *__restrict__ valid, const float *__restrict__ lse, const float *__restrict__ sums,
    const float *__restrict__ slopes, const float *__restrict__ grad_loss, T *__restrict__ grad_logits, bool held) {
    constexpr int kWidth = Pack<T>::kWidth, kPackets = 4;
    const float scale = *grad_loss;
    if (held && scale == 1.0f) return;
    constexpr int kRows = kBackwardThreads / kRowThreads;  // of a CTA at a time
    const int thread = threadIdx.x % kRowThreads, run = blockIdx.y * kRowThreads * kPackets;
    const int vocab = static_cast<int>(shape.vocab), step = static_cast<int>(gridDim.y) * kRowThreads * kPackets;
    for (int64_t row = int64_t(blockIdx.x) * kRows + threadIdx.x / kRowThreads; row < shape.rows; row += int64_t(gridDim.x) * kRows) {
        const T *in = logits + shape.start(row);
        T *out = grad_logits + row * vocab;
        if (valid != nullptr && valid[row] == 0) {
            if (blockIdx.y == 0) clear_row<T, kRowThreads>(out, vocab);
            continue;
        }
        const Packets<T> packets(in, vocab);
        const bool fits = packets.fits(out);
        const float slope = slopes[row] * scale, from = lse[row], factor = sums != nullptr ? -slope / sums[row] : -slope;
        const int64_t target = targets[row];
        const int at = static_cast<int>(target) + packets.skip, packet = target >= 0 && target < vocab ? at / kWidth : -1;
        for (int first = run + thread; first < packets.count; first += step) {
            uint4 raw[kPackets];
#pragma unroll
            for (int j = 0; j < kPackets; ++j) {
                const int c = first + j * kRowThreads;
                raw[j] = packets.whole(c) ? load_cached(packets.base + int64_t(c) * kWidth) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < kPackets; ++j) {
                const int c = first + j * kRowThreads;
                if (c >= packets.count) continue;
                float v[kWidth];
                if (packets.whole(c)) {
                    unpack(raw[j], v, T());
                } else {
                    packets.load_partly(c, v);
                }
#pragma unroll
                for (int i = 0; i < kWidth; ++i) v[i] = exp_from(v[i], from) * factor;
                if (packet == c) {
#pragma unroll
                    for (int i = 0; i < kWidth; ++i) v[i] += at % kWidth == i ? slope : 0.0f;
                }
                packets.store(out, fits && packets.whole(c), c, v);
            }
        }
    }
}

// grad *= *factor, unless the factor is one. grad is 16-byte aligned.
template <typename T>
__global__ __launch_bounds__(256) void policy_scale_kernel(T *__restrict__ grad, int64_t count,
                                                           const float *__restrict__ factor) {
    constexpr int kWidth = Pack<T>::kWidth;
    const float f = *factor;
    if (f == 1.0f) return;
    const int64_t packets = count / kWidth, thread = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    for (int64_t i = thread; i < packets; i += int64_t(gridDim.x) * blockDim.x) {
        float v[kWidth];
        unpack(reinterpret_cast<const uint4 *>(grad)[i], v, T());
#pragma unroll
        for (int j = 0; j < kWidth; ++j) v[j] *= f;
        reinterpret_cast<uint4 *>(grad)[i] = pack(v, T());
    }
    if (thread < count - packets * kWidth) {
        T *tail = grad + packets * kWidth + thread;
        *tail = from_acc<T>(to_acc(*tail) * f);
    }
}

// Takes a flag out of a dtype.
bool take_flag(int &dtype, int flag) {
    const bool given = (dtype & flag) != 0;
    dtype &= ~flag;
    return given;
}

PolicyRows rows_of(int64_t rows, int64_t vocab, int64_t inner_rows, int64_t outer_stride, int64_t inner_stride) {
    // one run of rows, however long, is a run of all of them
    return PolicyRows{rows, vocab, inner_rows > rows && rows > 0 ? rows : inner_rows, outer_stride, inner_stride};
}

int check_policy(const PolicyRows &shape) {
    if (shape.rows < 0 || shape.rows > (int64_t(1) << 31)) return fail(KOEMI_ERR_INVALID, "rows must be in [0, 2^31]");
    if (shape.vocab < 1 || shape.vocab > (int64_t(1) << 30)) return fail(KOEMI_ERR_INVALID, "vocab must be in [1, 2^30]");
    if (shape.inner < 1) return fail(KOEMI_ERR_INVALID, "inner_rows must be positive");
    return KOEMI_OK;
}

// The clusters of `size` CTAs that run at the same time, two CTAs on an SM.
template <typename Kernel>
int resident_clusters(Kernel kernel, int threads, int shared, int size) {
    cudaLaunchConfig_t config{};
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = size;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.gridDim = dim3(size);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.attrs = &attribute;
    config.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) != cudaSuccess || clusters < 1) {
        cudaGetLastError();
        clusters = 2 * sm_count() / size;
    }
    return clusters;
}

// `blocks`: the partial sums that the kernel leaves.
template <typename T, int kThreads, int kThreadBytes, bool kSplit>
int launch_rows(int64_t bytes, bool exact, const PolicyRows &shape, const PolicyTerms &terms, const T *logits,
                const PolicyOut &result, T *grad, unsigned &blocks, cudaStream_t stream) {
    constexpr int kPerSm = kSmBytes / kThreadBytes / kThreads;
    const int cluster = kSplit ? static_cast<int>(ceil_div(bytes, kSliceBytes)) : 1;
    const int slice = static_cast<int>(ceil_div(ceil_div(bytes, 16), cluster));
    // as many buffers as fit beside the other CTAs of the SM
    const uint32_t buffer_bytes = static_cast<uint32_t>(ceil_div(slice * 16, 128) * 128), room = 222 * 1024 / kPerSm - 2048;
    const int buffers = static_cast<int>(room / buffer_bytes > 3 ? 3 : room / buffer_bytes);
    const int64_t outer = (shape.rows - 1) / shape.inner, inner = (shape.rows < shape.inner ? shape.rows : shape.inner) - 1;
    const T *end = logits + outer * shape.outer_stride + inner * shape.inner_stride + shape.vocab;
    auto kernel = exact ? policy_row_kernel<T, kThreads, kThreadBytes, true, kSplit>
                        : policy_row_kernel<T, kThreads, kThreadBytes, false, kSplit>;
    const int shared = buffers * static_cast<int>(buffer_bytes);
    // the most that any call wants, not this one's: another thread's launch may stand between the two calls
    KOEMI_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(room)));
    int64_t places = kSplit ? resident_clusters(kernel, kThreads, shared, cluster) : int64_t(sm_count()) * kPerSm;
    if (places > kPolicyBlocks) places = kPolicyBlocks;  // a partial sum each
    blocks = static_cast<unsigned>(shape.rows < places ? shape.rows : places);
    KOEMI_CUDA_TRY(launch_programmatic(false, kernel, dim3(blocks * cluster), dim3(kThreads), static_cast<size_t>(shared), stream,
                                       dim3(cluster), shape, terms, logits, end, result, grad, buffers, buffer_bytes, cluster,
                                       slice, device_status_word()));
    return KOEMI_OK;
}

// Up to here (packets) eight threads, and a warp, take a row of the backward; a
// CTA takes longer ones: 65536 x 64 bf16 19 us with eight threads and 33 with a
// warp, 16384 x 1100 27 us with a warp and 53 with a CTA.
constexpr int kTinyRow = 32, kShortRow = 1024;

// The row kernel with the fewest threads that hold the row.
template <typename T>
int launch_held(int64_t bytes, bool exact, const PolicyRows &shape, const PolicyTerms &terms, const T *logits,
                const PolicyOut &result, T *grad, unsigned &blocks, cudaStream_t stream) {
    auto go = [&](auto launch) { return launch(bytes, exact, shape, terms, logits, result, grad, blocks, stream); };
    if (bytes <= 64 * 128) return go(launch_rows<T, 64, 128, false>);
    if (bytes <= 64 * 256) return go(launch_rows<T, 64, 256, false>);
    if (bytes <= 128 * 256) return go(launch_rows<T, 128, 256, false>);
    if (bytes <= 256 * 256) return go(launch_rows<T, 256, 256, false>);
    return go(launch_rows<T, 256, 256, true>);
}

template <typename T, int kPer>
int launch_warps(const PolicyRows &shape, const PolicyTerms &terms, const T *logits, const PolicyOut &result, T *grad,
                 unsigned &blocks, cudaStream_t stream) {
    const int64_t wanted = ceil_div(shape.rows, 8);
    blocks = static_cast<unsigned>(wanted < kPolicyBlocks ? wanted : kPolicyBlocks);
    policy_warp_kernel<T, kPer><<<blocks, 256, 0, stream>>>(shape, terms, logits, result, grad);
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

template <typename T>
int policy_forward(const PolicyRows &shape, const PolicyTerms &terms, const void *logits, float *loss, float *kl,
                   float *log_probs, float *lse, float *sums, float *slopes, void *grad_logits, void *workspace,
                   cudaStream_t stream) {
    float *inverse = static_cast<float *>(workspace);
    PolicyOut result{nullptr, log_probs, lse, sums, slopes, reinterpret_cast<double2 *>(static_cast<unsigned char *>(workspace) + 256)};
    const T *in = static_cast<const T *>(logits);
    T *grad = static_cast<T *>(grad_logits);
    unsigned blocks = 0;
    if (terms.valid != nullptr && shape.rows > kCountedRows) {
        policy_count_kernel<<<1, 1024, 0, stream>>>(terms.valid, shape.rows, inverse);
        KOEMI_LAUNCH_CHECK();
        result.inverse = inverse;
    }
    if (shape.rows > 0) {
        // rows that can start inside a packet may touch one packet more
        const bool inside = !aligned(logits, 16) || shape.outer_stride * sizeof(T) % 16 != 0 || shape.inner_stride * sizeof(T) % 16 != 0;
        const int64_t entries = shape.vocab + (inside ? Pack<T>::kWidth - 1 : 0);
        int rc;
        // 65536 x 257 fp32: 45 us with 12 entries a lane, 48 us with 16
        if (shape.vocab <= 256) {
            rc = launch_warps<T, 8>(shape, terms, in, result, grad, blocks, stream);
        } else if (shape.vocab <= 384) {
            rc = launch_warps<T, 12>(shape, terms, in, result, grad, blocks, stream);
        } else if (shape.vocab <= 512) {
            rc = launch_warps<T, 16>(shape, terms, in, result, grad, blocks, stream);
        } else if (shape.vocab <= kWarpRow) {
            rc = launch_warps<T, 32>(shape, terms, in, result, grad, blocks, stream);
        } else if (entries * int64_t(sizeof(T)) <= kMaxCluster * kSliceBytes) {
            const bool exact = !inside && shape.vocab % Pack<T>::kWidth == 0;
            rc = launch_held<T>(entries * sizeof(T), exact, shape, terms, in, result, grad, blocks, stream);
        } else {
            const int64_t places = 2 * int64_t(sm_count());
            blocks = static_cast<unsigned>(shape.rows < places ? shape.rows : places);
            policy_walk_kernel<T><<<blocks, kWalkThreads, 0, stream>>>(shape, terms, in, result, grad);
            KOEMI_LAUNCH_CHECK();
            rc = KOEMI_OK;
        }
        if (rc != KOEMI_OK) return rc;
    }
    policy_finish_kernel<<<1, kFinishThreads, 0, stream>>>(result.partials, static_cast<int>(blocks), result.inverse,
                                                           terms.valid, shape.rows, loss, kl);
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

template <typename T>
int policy_backward(const PolicyRows &shape, const void *logits, const int64_t *targets, const uint8_t *valid,
                    const float *lse, const float *sums, const float *slopes, const float *grad_loss, void *grad_logits,
                    bool held, cudaStream_t stream) {
    // threads of a row, rows of a CTA at a time, and for few long rows several CTAs a row
    const int64_t packets = ceil_div(shape.vocab, Pack<T>::kWidth), most = 8 * int64_t(sm_count());
    auto go = [&](auto kernel, int row_threads) {
        const int64_t turns = ceil_div(shape.rows, kBackwardThreads / row_threads), x = turns < most ? turns : most;
        const int64_t runs = ceil_div(packets, row_threads * 4), wanted = ceil_div(most, x);
        const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>(wanted < runs ? wanted : runs));
        kernel<<<grid, kBackwardThreads, 0, stream>>>(shape, static_cast<const T *>(logits), targets, valid, lse, sums, slopes,
                                                      grad_loss, static_cast<T *>(grad_logits), held);
    };
    if (packets <= kTinyRow) {
        go(policy_backward_kernel<T, 8>, 8);
    } else if (packets <= kShortRow) {
        go(policy_backward_kernel<T, 32>, 32);
    } else {
        go(policy_backward_kernel<T, kBackwardThreads>, kBackwardThreads);
    }
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

template <typename T>
int policy_scale(void *grad, int64_t count, const float *factor, cudaStream_t stream) {
    const int64_t blocks = ceil_div(count, 256 * Pack<T>::kWidth);
    policy_scale_kernel<T><<<static_cast<unsigned>(blocks < 1184 ? blocks : 1184), 256, 0, stream>>>(
        static_cast<T *>(grad), count, factor);
    KOEMI_LAUNCH_CHECK();
    return KOEMI_OK;
}

}  // namespace
}  // namespace koemi

using namespace koemi;

extern "C" size_t koemi_think_policy_loss_workspace(void) { return 256 + kPolicyBlocks * sizeof(double2); }

extern "C" int koemi_think_policy_loss_forward(const void *logits, int64_t rows, int64_t vocab, int64_t inner_rows,
                                               int64_t outer_stride, int64_t inner_stride, const int64_t *targets,
                                               const float *old_log_probs, const float *advantages,
                                               const float *reference_log_probs, const uint8_t *valid, float clip_low,
                                               float clip_high, float kl_weight, float *loss, float *kl,
                                               float *log_probs, float *lse, float *slopes, void *grad_logits,
                                               int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    const PolicyRows shape = rows_of(rows, vocab, inner_rows, outer_stride, inner_stride);
    const int rc = check_policy(shape);
    if (rc != KOEMI_OK) return rc;
    if (!(clip_low >= 0.0f && clip_high >= 0.0f)) return fail(KOEMI_ERR_INVALID, "clip widths must be non-negative");
    if (loss == nullptr || kl == nullptr || workspace == nullptr ||
        (rows > 0 && (logits == nullptr || targets == nullptr || old_log_probs == nullptr || advantages == nullptr ||
                      log_probs == nullptr || lse == nullptr || slopes == nullptr))) {
        return fail(KOEMI_ERR_INVALID, "policy loss tensors and workspace must be non-NULL");
    }
    if (!aligned(grad_logits, 16)) return fail(KOEMI_ERR_INVALID, "grad_logits must be 16-byte aligned");
    if (workspace_bytes < koemi_think_policy_loss_workspace()) {
        return fail(KOEMI_ERR_WORKSPACE, "the policy loss's workspace is smaller than koemi_think_policy_loss_workspace()");
    }
    const PolicyTerms terms{targets, old_log_probs, advantages, reference_log_probs, valid, clip_low, clip_high, kl_weight};
    float *sums = take_flag(dtype, KOEMI_POLICY_SUMS) && lse != nullptr ? lse + rows : nullptr;
    cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case KOEMI_F32: return policy_forward<float>(shape, terms, logits, loss, kl, log_probs, lse, sums, slopes, grad_logits, workspace, s);
        case KOEMI_F16: return policy_forward<__half>(shape, terms, logits, loss, kl, log_probs, lse, sums, slopes, grad_logits, workspace, s);
        case KOEMI_BF16: return policy_forward<__nv_bfloat16>(shape, terms, logits, loss, kl, log_probs, lse, sums, slopes, grad_logits, workspace, s);
        default: return fail(KOEMI_ERR_INVALID, "unsupported policy loss dtype %d", dtype);
    }
}

extern "C" int koemi_think_policy_loss_backward(const void *logits, int64_t rows, int64_t vocab, int64_t inner_rows,
                                                int64_t outer_stride, int64_t inner_stride, const int64_t *targets,
                                                const uint8_t *valid, const float *lse, const float *slopes,
                                                const float *grad_loss, void *grad_logits, int dtype, void *stream) {
    clear_error();
    const PolicyRows shape = rows_of(rows, vocab, inner_rows, outer_stride, inner_stride);
    const int rc = check_policy(shape);
    if (rc != KOEMI_OK) return rc;
    if (rows == 0) return KOEMI_OK;
    if (logits == nullptr || targets == nullptr || lse == nullptr || slopes == nullptr || grad_loss == nullptr ||
        grad_logits == nullptr) {
        return fail(KOEMI_ERR_INVALID, "policy loss backward tensors must be non-NULL");
    }
    if (!aligned(grad_logits, 16)) return fail(KOEMI_ERR_INVALID, "grad_logits must be 16-byte aligned");
    const float *sums = take_flag(dtype, KOEMI_POLICY_SUMS) ? lse + rows : nullptr;
    const bool held = take_flag(dtype, KOEMI_POLICY_HELD);
    cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case KOEMI_F32: return policy_backward<float>(shape, logits, targets, valid, lse, sums, slopes, grad_loss, grad_logits, held, s);
        case KOEMI_F16: return policy_backward<__half>(shape, logits, targets, valid, lse, sums, slopes, grad_loss, grad_logits, held, s);
        case KOEMI_BF16: return policy_backward<__nv_bfloat16>(shape, logits, targets, valid, lse, sums, slopes, grad_loss, grad_logits, held, s);
        default: return fail(KOEMI_ERR_INVALID, "unsupported policy loss dtype %d", dtype);
    }
}

extern "C" int koemi_think_policy_loss_scale(void *grad_logits, int64_t count, const float *factor, int dtype,
                                             void *stream) {
    clear_error();
    if (count < 0) return fail(KOEMI_ERR_INVALID, "count must be non-negative");
    if (count == 0) return KOEMI_OK;
    if (grad_logits == nullptr || factor == nullptr) return fail(KOEMI_ERR_INVALID, "grad_logits and factor must be non-NULL");
    if (!aligned(grad_logits, 16)) return fail(KOEMI_ERR_INVALID, "grad_logits must be 16-byte aligned");
    cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case KOEMI_F32: return policy_scale<float>(grad_logits, count, factor, s);
        case KOEMI_F16: return policy_scale<__half>(grad_logits, count, factor, s);
        case KOEMI_BF16: return policy_scale<__nv_bfloat16>(grad_logits, count, factor, s);
        default: return fail(KOEMI_ERR_INVALID, "unsupported policy loss dtype %d", dtype);
    }
}
