// aw4_tc.cuh -- barriers, bulk tensor copies and 5th-generation tensor core
// instructions (sm_100a), as thin wrappers of their PTX.
#pragma once

#include <cuda.h>
#include <stdint.h>

namespace aw4 {

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}

// ---- barriers ---------------------------------------------------------------

__device__ __forceinline__ void bar_init(uint32_t bar, int arrivals) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The barrier at the same place in the pair's first block.
__device__ __forceinline__ uint32_t in_first_block(uint32_t bar) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(bar));
    return r;
}
// Arrivals there.  An arrival that names no scope orders memory within its own block only.  `release`: what this
// thread has written, or has seen written by a wait, is there for the thread whose wait of kind kWaitPair sees the arrival.
// `relaxed`: no memory is handed over; tensor memory is ordered by the tcgen05 fences around arrival and wait.
__device__ __forceinline__ void bar_arrive_pair_release(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void bar_arrive_pair_relaxed(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ uint32_t block_in_pair() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void pair_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Whose arrivals a wait is for: the own block's threads and copies and the tensor core's commits, or
// the other block's threads too, by either kind of arrival.
enum WaitKind { kWaitOwn, kWaitPair, kWaitPairRelaxed };
template <WaitKind KIND = kWaitOwn>
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    if constexpr (KIND == kWaitPair)
        asm volatile(
            "{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
            : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    else if constexpr (KIND == kWaitPairRelaxed)
        asm volatile(
            "{ .reg .pred p; mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
            : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    else
        asm volatile(
            "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
            : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Waits for the phase of this parity to end.  Every wait has a limit in tries
// and in time (`limit`, in ns), by default far above the longest tile: past it, or once another waiter of
// the block has given up (`gave_up`), it returns false and the block winds
// down.  With a limit of 0 it returns false at once.
constexpr int kWaitTries = 1 << 24;
constexpr uint64_t kWaitNs = 2000000000ull;
template <WaitKind KIND = kWaitOwn>
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up, uint64_t limit) {
    uint64_t from = 0;
    for (int i = 0; limit && i < kWaitTries; ++i) {
        if (bar_try<KIND>(bar, parity)) return true;
        if ((i & 63) == 63) {
            if (*gave_up) return false;
            const uint64_t t = now_ns();
            if (!from) from = t;
            if (t - from > limit) break;
        }
    }
    *gave_up = 1;
    return false;
}
// The same for a block that winds down and lets its own work in flight end.
__device__ __forceinline__ void bar_drain(uint32_t bar, uint32_t parity) {
    const uint64_t from = now_ns();
    for (int i = 0; i < kWaitTries && !bar_try(bar, parity); ++i)
        if (now_ns() - from > kWaitNs) break;
}

__device__ __forceinline__ void fence_async_smem() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// ---- bulk tensor copies -----------------------------------------------------

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// ---- tensor memory and tensor core, in pairs of blocks ------------------------
//
// A pair's product is 256 x n: each block holds 128 of the rows in its tensor
// memory, those rows of the first operand and half the columns of the second in its shared
// memory.  One thread of the pair's first block issues for both.

// Both by the same warp of each block of the pair.
__device__ __forceinline__ void tmem_alloc(uint32_t smem_slot, int cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_slot), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t taddr, int cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// The barrier of both blocks gets one arrival when every product issued so far by this thread is done.
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tc_mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{ .reg .pred p; setp.ne.u32 p, %4, 0;\n"
        "  tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p; }"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
// 32 columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_load32(uint32_t taddr, uint32_t v[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory operand descriptor of a tile whose rows (the product's inner
// dimension) are 128-byte lines of 64 two-byte values, swizzled by 128 bytes:
// groups of eight rows follow each other by 1024 bytes, groups of 64
// columns by `column_stride`.
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t column_stride) {
    return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(column_stride >> 4) << 16) |
           ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// Instruction descriptor: float32 sums, both operands with their columns
// contiguous (the inner dimension strided), 256 x n.
__device__ __forceinline__ uint32_t tc_idesc(bool bf16, int n) {
    const uint32_t type = bf16 ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(n >> 3) << 17) |
           ((256u >> 4) << 24);
}

}  // namespace aw4
