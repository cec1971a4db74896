// Thin wrappers over the PTX of the 5th-generation tensor cores, tensor-map copies and mbarriers, all waits bounded.
#pragma once

#include <cuda.h>

#include "gact_common.cuh"

namespace gact {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}

// Waits for a phase of a barrier, at most `limit` polls.  A wait that runs out sets *dead (shared memory); every later wait of
// the block then returns at once, so the block runs to its end without waiting for anything again.  The default spans whole
// products: a poll takes a quarter of a microsecond (layer norm's rings: 8), the longest reductions a few tenths of a second.
constexpr uint32_t kWaitLimit = 1u << 23;
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, uint32_t limit, volatile int* dead) {
    for (uint32_t i = 0; i < limit; i++) {
        if (mbar_try(bar, parity)) return true;
        if (*dead) return false;
    }
    *dead = 1;
    return false;
}
// the same for copies that are still in flight when a block has given up
__device__ __forceinline__ void mbar_drain(uint32_t bar, uint32_t parity, uint32_t limit) {
    for (uint32_t i = 0; i < limit && !mbar_try(bar, parity); i++) {}
}

// a block that gave up: the device's error word and, for the host's next call, the word in its memory
__device__ __forceinline__ void report_wait(int* error_word, int* host_word) {
    atomicExch(error_word, 1);
    if (host_word) {
        *(volatile int*)host_word = 1;
        __threadfence_system();
    }
}

// address of the same shared-memory variable in block `rank` of the cluster
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// all threads of both blocks; everything written before is visible after
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrive on a barrier of any block of the cluster.  (Default scope: what the other block is told about - operand tiles, TMEM
// that has been read - it touches through the tensor core only, ordered by fence.proxy.async and tcgen05.fence before the
// arrival.  A release at cluster scope would wait for the thread's outstanding global accesses: a microsecond per stage.)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// CG: 1, or 2 for a pair of blocks that works on one tile.  2-D tile copy of this GPU's own memory into this block's shared
// memory; x counts elements along the contiguous axis.  With CG = 2 the barrier may be the other block's.
template <int CG> __device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

template <int CG> __device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols) {
    if constexpr (CG == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
}
template <int CG> __device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
    if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// D (TMEM, fp32) += A B for one K of 16; `add` = 0 starts a new sum.  CG = 2: issued by one block for both, each holding half
// of A's rows, half of B's columns, and the accumulators of its rows.
template <int CG> __device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    if constexpr (CG == 1)
        asm volatile("{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
    else
        asm volatile("{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p; }"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
// the barrier (CG = 2: at this address in both blocks) is arrived on once every earlier tcgen05.mma of this thread has finished
template <int CG> __device__ __forceinline__ void mma_commit(uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"((uint16_t)3) : "memory");
}

// 32 lanes x 32 columns of fp32 accumulators: lane l of the warp gets TMEM lane (its quarter) + l, columns c .. c + 31
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
          "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Shared-memory operand descriptor for tiles written by a tensor map with 128-byte swizzle (atoms of 8 rows x 128 bytes,
// 1024-byte aligned).
//   K-major  (rows = M or N, 64 K-elements per row): the next 8 rows are 1024 bytes on; 16 more K-elements are 32 bytes on.
//   MN-major (rows = K, 64 M- or N-elements per row): the next 8 K-rows are 1024 bytes on, the next 64 M/N-elements
//            `chunk` bytes on; 16 more K-rows are 2048 bytes on.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t chunk) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)((chunk >> 4) & 0x3fffu) << 16) | ((uint64_t)(1024u >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// Instruction descriptor of kind::f16: fp32 accumulator, both operands fp16 (0) or bf16 (1), majorness, shape.
static __host__ __device__ constexpr uint32_t mma_idesc(int m, int n, bool bf16, bool a_mn, bool b_mn) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

}  // namespace gact
