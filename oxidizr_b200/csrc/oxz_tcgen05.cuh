// The tensor-core path of sm_100a as the loss head's products use it: mbarriers with bounded waits, TMA tile loads, and
// tcgen05.mma on a pair of SMs (cta_group::2) with its accumulators in tensor memory. Thin wrappers over single instructions.
#pragma once

#include <stdint.h>

namespace oxz {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// The address of the same place in the shared memory of block `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_smem(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// bar: a peer_smem address. What it tells is that accumulators have been read (ordered by the tcgen05 fences), no memory: the narrow
// default scope will do, and does not wait for the stores in flight as a cluster-wide release would.
__device__ __forceinline__ void mbar_arrive_peer(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}

// What a block that gives up leaves for its other warps (shared) and for the host (mapped memory).
struct WaitState {
    volatile uint32_t* dead;
    int32_t* expired;
};
// A wait gives up after WAIT_NS of waiting that are at least LEAST_TRIES tries: what a try takes depends on the rest of its warp (2 us where
// all of it waits, 25 ns where other lanes are elsewhere, both measured), so tries alone would bound it to anything from a twentieth of a
// second to minutes; time alone would count what the block spends off the SM. The clock is not read in a wait of fewer than 256 tries.
constexpr uint64_t WAIT_NS = 4000000000ull;
constexpr uint32_t LEAST_TRIES = 1u << 16, MOST_TRIES = 1u << 30;
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const WaitState& w) {
    uint64_t from = 0;
    for (uint32_t i = 0; i < MOST_TRIES; i++) {
        if (mbar_try(bar, parity)) return true;
        if ((i & 255) == 255) {
            if (*w.dead) return false;
            uint64_t now;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (from == 0) from = now;
            if (i >= LEAST_TRIES && now - from > WAIT_NS) break;
        }
    }
    *w.dead = 1;
    *reinterpret_cast<volatile int32_t*>(w.expired) = 1;
    __threadfence_system();
    return false;
}

// A box of a 3-d tensor map into this block's shared memory; the bytes are counted on `bar`, which may be the pair's first block's.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const void* map, int32_t x, int32_t y, int32_t z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
// A box from this block's shared memory into a tensor map's memory, or added to it in f32; what lies outside is left out. `from` has been
// written by this thread's warp (store_fence, then a warp barrier). One thread of the warp; store_read<N> waits until the shared
// memory of all but the last N stores may be written again, store_done until all are in memory.
__device__ __forceinline__ void tma_store(const void* map, int32_t x, int32_t y, int32_t z, uint32_t from) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n\tcp.async.bulk.commit_group;"
                 ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(from) : "memory");
}
__device__ __forceinline__ void tma_add(const void* map, int32_t x, int32_t y, int32_t z, uint32_t from) {
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n\tcp.async.bulk.commit_group;"
                 ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(from) : "memory");
}
__device__ __forceinline__ void store_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
template <int N> __device__ __forceinline__ void store_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void st_shared16(uint32_t to, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ void tma_prefetch_map(const void* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

__device__ __forceinline__ void tmem_alloc_pair(uint32_t to_smem, uint32_t columns) {  // one warp of each block of the pair
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to_smem), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t addr, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns) : "memory");
}
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// D[256 x N] (+)= A[256 x 16] B[N x 16]^T over the two blocks of a pair: 128 rows of A and D and half of B's rows in each.
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p; }"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
// Arrives at `bar` (same place in both blocks) once the pair's products issued so far have read and written what they use.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((uint16_t)3) : "memory");
}

// Columns of this warp's 32 lanes of tensor memory: x[c] is column c of the thread's row. Complete after tmem_wait(), which every array
// loaded before it passes through (arrived()), so that nothing that reads them is moved above the wait.
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&x)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]), "=f"(x[8]), "=f"(x[9]), "=f"(x[10]), "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15]), "=f"(x[16]), "=f"(x[17]), "=f"(x[18]), "=f"(x[19]), "=f"(x[20]), "=f"(x[21]), "=f"(x[22]), "=f"(x[23]), "=f"(x[24]), "=f"(x[25]), "=f"(x[26]), "=f"(x[27]), "=f"(x[28]), "=f"(x[29]), "=f"(x[30]), "=f"(x[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&x)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]), "=f"(x[8]), "=f"(x[9]), "=f"(x[10]), "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void arrived(float (&x)[32]) {
    asm volatile("" : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]), "+f"(x[6]), "+f"(x[7]), "+f"(x[8]), "+f"(x[9]), "+f"(x[10]), "+f"(x[11]), "+f"(x[12]), "+f"(x[13]), "+f"(x[14]), "+f"(x[15]), "+f"(x[16]), "+f"(x[17]), "+f"(x[18]), "+f"(x[19]), "+f"(x[20]), "+f"(x[21]), "+f"(x[22]), "+f"(x[23]), "+f"(x[24]), "+f"(x[25]), "+f"(x[26]), "+f"(x[27]), "+f"(x[28]), "+f"(x[29]), "+f"(x[30]), "+f"(x[31]));
}
__device__ __forceinline__ void arrived(float (&x)[16]) {
    asm volatile("" : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]), "+f"(x[6]), "+f"(x[7]), "+f"(x[8]), "+f"(x[9]), "+f"(x[10]), "+f"(x[11]), "+f"(x[12]), "+f"(x[13]), "+f"(x[14]), "+f"(x[15]));
}

// Shared-memory operand descriptors for tiles that TMA wrote with the 128-byte swizzle, in boxes of 64 elements (128 bytes) by
// 64 lines, 8192 bytes each.
//   K along the 128 bytes: lines are rows of the operand; 8 lines (1024 bytes) form a group, groups follow each other.
//   K along the lines: the 128 bytes hold 64 rows of the operand, the next 64 are one box (8192 bytes) on; 8 lines form a group.
constexpr uint32_t BOX_BYTES = 8192;
__device__ __forceinline__ uint64_t operand(uint32_t addr, bool k_along_lines) {
    const uint64_t leading = k_along_lines ? BOX_BYTES >> 4 : 1, stride = 1024 >> 4;
    return (uint64_t)((addr >> 4) & 0x3fff) | leading << 16 | stride << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// f32 accumulators, both operands bf16 or both f16
__host__ __device__ __forceinline__ uint32_t instruction(bool bf16, bool a_along_lines, bool b_along_lines, uint32_t m, uint32_t n) {
    const uint32_t fmt = bf16 ? 1 : 0;
    return 1u << 4 | fmt << 7 | fmt << 10 | (uint32_t)a_along_lines << 15 | (uint32_t)b_along_lines << 16 | (n >> 3) << 17 | (m >> 4) << 24;
}

}  // namespace oxz
