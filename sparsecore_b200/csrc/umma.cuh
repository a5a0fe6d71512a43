// Fifth-generation tensor cores (tcgen05) with a pair of CTAs on one tile:
// the instructions as functions, and the descriptors of their operands.
//
// cta_group::2: the two CTAs of a cluster multiply one 256 x N tile.  Each
// holds its 128 rows of A, its half of B's rows and, in its tensor memory,
// its 128 rows of the result; one thread of the first CTA issues for both.
#pragma once

#include "tma.cuh"

namespace slb {

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Address, in the cluster's window, of the first CTA's copy of a shared
// variable.
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_addr(p)));
    return a;
}

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}

// mbar_wait for arrivals from the other CTA of the cluster.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, unsigned phase, unsigned* status) {
    const uint32_t a = smem_addr(bar);
    for (long long it = 0; it < kSpinLimit; ++it) {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
            " selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(a), "r"(phase)
            : "memory");
        if (done) return true;
    }
    atomicOr(status, 1u);
    return false;
}

// TMA box at (x, y, z) into this CTA's shared memory, completing on a
// barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst)), "r"(cols) : "memory");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 rows of tensor memory, a row a thread.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A . B for one step of 16 along the sum.
__device__ __forceinline__ void umma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}

// One arrival on the barrier at this offset in both CTAs once all MMAs
// issued so far are done (and their operands read).
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     smem_addr(bar)),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
}

// Shared-memory operand in boxes of 128-byte rows with the 128-byte swizzle.
// K-major: rows are the operand's rows, 64 of its columns each; groups of 8
// rows are 1024 bytes apart.  MN-major: rows are steps along the sum, 64 of
// the operand's rows each; groups of 8 steps are 1024 bytes apart and the
// next 64 rows one box of 64 steps, 8192 bytes, further.
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, bool mn_major) {
    const uint64_t lead = mn_major ? 8192 >> 4 : 1;
    return static_cast<uint64_t>((addr & 0x3FFFF) >> 4) | lead << 16 | static_cast<uint64_t>(1024 >> 4) << 32 |
           static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}

// 16-bit operands of one type, 32-bit sums, a tile of 256 x n.
__device__ __forceinline__ uint32_t umma_idesc(bool bf16, bool a_mn, bool b_mn, int n) {
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
           static_cast<uint32_t>(n >> 3) << 17 | (256u >> 4) << 24;
}

}  // namespace slb
