// PTX of the tcgen05 matrix instructions that the tensor-core kernels share:
// operand descriptors, the instruction and its completion, accumulator reads,
// and a wait that watches its CTA's abort flag.
#pragma once

#include "common.cuh"

namespace koemi {

__device__ __forceinline__ uint64_t sw128_kmajor_desc(uint32_t smem_address) {
    uint64_t desc = 0;
    desc |= static_cast<uint64_t>((smem_address & 0x3FFFF) >> 4);  // start address
    desc |= static_cast<uint64_t>(1) << 16;                          // LBO (unused for swizzled K-major)
    desc |= static_cast<uint64_t>(1024 >> 4) << 32;                  // SBO: 8 rows x 128 B
    desc |= static_cast<uint64_t>(1) << 46;                          // descriptor version (sm100)
    desc |= static_cast<uint64_t>(2) << 61;                          // 128-byte swizzle
    return desc;
}

// A tile whose rows are K (128 bytes of M or N each, 64 K rows a tile, tiles of
// 64 M or N entries one after the other): repeats along M or N every 8192
// bytes, along K every 8 rows.
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t smem_address) {
    uint64_t desc = 0;
    desc |= static_cast<uint64_t>((smem_address & 0x3FFFF) >> 4);
    desc |= static_cast<uint64_t>(8192 >> 4) << 16;  // LBO: the next 64 entries of M or N
    desc |= static_cast<uint64_t>(1024 >> 4) << 32;  // SBO: the next 8 rows of K
    desc |= static_cast<uint64_t>(1) << 46;
    desc |= static_cast<uint64_t>(2) << 61;
    return desc;
}

__device__ __forceinline__ void umma_f16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ void umma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

#define KOEMI_TMEM_LD32(taddr, v)                                                                              \
    asm volatile(                                                                                              \
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, " \
        "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"    \
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),     \
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]),             \
          "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]),           \
          "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]),           \
          "=r"(v[29]), "=r"(v[30]), "=r"(v[31])                                                                \
        : "r"(taddr))

#define KOEMI_TMEM_LD16(taddr, v)                                                                              \
    asm volatile(                                                                                              \
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, " \
        "%14, %15}, [%16];"                                                                                    \
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),     \
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]),             \
          "=r"(v[15])                                                                                          \
        : "r"(taddr))

__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Bounded wait that also watches the CTA abort flag.
__device__ __forceinline__ bool wait_or_abort(uint64_t *bar, uint32_t parity, volatile int *abort, int *status) {
    for (uint32_t spin = 0; spin < kWaitSpinLimit; ++spin) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((spin & 255) == 255 && *abort) return false;
    }
    *abort = 1;
    if (status != nullptr) atomicExch(status, KOEMI_ERR_TIMEOUT);
    return false;
}

}  // namespace koemi
