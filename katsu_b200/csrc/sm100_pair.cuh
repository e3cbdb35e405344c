// Cluster-level instructions for kernels that run tcgen05 MMAs on pairs of thread blocks (cta_group::2):
// cluster rank and barrier, shared-window addresses of the peer, remote barrier arrival, paired tensor-memory
// allocation, the MMA / commit forms that span both blocks, and TMA loads whose bytes are counted on a barrier
// of the pair's leader.  No load here is shared between blocks by the copy engine.
#pragma once

#include "sm100.cuh"

namespace sm100 {

__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// Shared-window address of the same variable in block `rank` of the cluster.
__device__ __forceinline__ uint32_t map_to_rank(const void *local, uint32_t rank) {
    uint32_t out;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(smem_u32(local)), "r"(rank));
    return out;
}

// Writes to the variable at this place in block `rank`'s shared memory and counts the 16 bytes on the barrier at `bar`'s place
// there: the data and its signal in one, with nothing of the thread's earlier work waited for.
__device__ __forceinline__ void st_async_v4(const void *local, uint64_t *bar, uint32_t rank, float4 v) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(map_to_rank(local, rank)),
                 "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(map_to_rank(bar, rank))
                 : "memory");
}

__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// Whole-warp bounded wait (mbar_wait_warp) for what other blocks of the cluster have written.
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}

__device__ __forceinline__ bool mbar_wait_warp_cluster(uint64_t *bar, uint32_t parity, int *status, int code) {
    // (every lane acquires: each reads the data itself)
    if (__all_sync(0xffffffffu, mbar_try_wait_cluster(bar, parity) ? 1 : 0)) return true;
    const bool ok = mbar_wait_warp(bar, parity, status, code);
    mbar_try_wait_cluster(bar, parity);
    return ok;
}

// Arrival on a barrier of the other block.  Relaxed: what these arrivals publish lives in tensor memory and is
// ordered by tcgen05.wait / tcgen05.fence around them, not by the memory model; a release at cluster scope made
// every arrival wait for the thread's earlier global and shared writes to drain (measured: ~2 000 clk per k-block).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync_all() {
    cluster_arrive();
    cluster_wait();
}

__device__ __forceinline__ void tmem_alloc_pair(uint32_t *smem_slot, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_slot)), "r"(columns)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(columns) : "memory");
}

// Arrives on the barrier at shared-window address `addr` (this block's or the peer's) once every MMA issued so far
// by this thread has completed.
__device__ __forceinline__ void mma_commit_pair(uint32_t addr) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(addr) : "memory");
}

// The same on the barrier at this place in both blocks of the pair.
__device__ __forceinline__ void mma_commit_both(uint64_t *bar) {
    mma_commit_pair(smem_u32(bar));
    mma_commit_pair(map_to_rank(bar, 1));
}

__device__ __forceinline__ void tma_load_3d_pair(void *smem_dst, const CUtensorMap *map, uint32_t bar_addr, int c0, int c1,
                                                 int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_addr), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

// D[tmem of both blocks] (+)= A[both blocks' shared memory, 128 rows each] * B[halves in both blocks' shared memory], 16-bit
// operands, f32 accumulator: 256 x N x 16 per instruction; issued by one thread of the leader block.  The TMA loads below bring
// a block's own tile into its own shared memory; the bytes are counted on the barrier at `bar_addr`, which may be the leader's.
__device__ __forceinline__ void mma_f16_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                             bool accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}

// The same with signed 8-bit operands and a 32-bit integer accumulator: 256 x N x 32 per instruction.
__device__ __forceinline__ void mma_i8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n"
        "}\n"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}

__device__ __forceinline__ void tma_load_4d_pair(void *smem_dst, const CUtensorMap *map, uint32_t bar_addr, int c0, int c1,
                                                 int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_addr), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

__device__ __forceinline__ void tma_load_5d_pair(void *smem_dst, const CUtensorMap *map, uint32_t bar_addr, int c0, int c1,
                                                 int c2, int c3, int c4) {
    asm volatile(
        "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], "
        "[%2];"
        ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_addr), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
        : "memory");
}

}  // namespace sm100
