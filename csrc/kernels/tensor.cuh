// Tensor-core and tensor-copy primitives (sm_100a): tcgen05 with TMEM
// accumulators, tiled bulk copies, and the proxy fence between plain
// shared-memory stores and the tensor core's reads.
#pragma once

#include <cstdint>
#include <cuda.h>

#include "ptx.cuh"

namespace engram {

// Tiled copy of one box at (x, y, z), completing its bytes on `bar`.
__device__ __forceinline__ void tensor_load_3d(void *dst_smem, const CUtensorMap *map, int x, int y, int z,
                                               uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_addr(dst_smem)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
                 : "memory");
}

// Tiled copy of one box to (x, y, z); what lies outside the tensor is not
// written.  A bulk group of the calling thread.
__device__ __forceinline__ void tensor_store_3d(const CUtensorMap *map, int x, int y, int z, const void *src_smem) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x),
                 "r"(y), "r"(z), "r"(smem_addr(src_smem))
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// At most N of this thread's groups still read shared memory.
template <int N> __device__ __forceinline__ void bulk_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void prefetch_tensor_map(const CUtensorMap *map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Plain shared-memory stores before it are visible to the async proxy after.
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The MMAs here run on a pair of SMs (a cluster of two blocks, the even one of
// them the leader): each block holds half of the rows of A and of the result,
// and half of the columns of B.

// TMEM: `columns` columns of 128 lanes x 32 bits in both blocks of the pair (a
// warp of each calls it); the address lands in `*slot`.
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}

__device__ __forceinline__ void tmem_free(uint32_t address, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
}

// 32 consecutive columns of this warp's 32 lanes (lane = row).  The values are
// there after tmem_wait_loads.
__device__ __forceinline__ void tmem_load32(uint32_t address, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
                 "%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]),
                   "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]),
                   "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]),
                   "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(address));
}

__device__ __forceinline__ void tmem_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tensor_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// `bar` of both blocks gets one arrival when every MMA this thread issued so far is done.
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     smem_addr(bar)),
                 "h"(uint16_t(3))
                 : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// All threads of the pair (stores before it are visible after it).
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The leader's barrier at the place of this block's `bar`.
__device__ __forceinline__ uint32_t leader_barrier(const uint64_t *bar) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_addr(bar)));
    return at;
}
// Arrives there.  What it announces are operands for the pair's MMAs, which this
// SM's own tensor core reads: fence_async_shared before it orders them, and no
// thread of the other block reads them.  (A release at cluster scope took a
// third of a stage's time.)
__device__ __forceinline__ void mbar_arrive_leader(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Shared-memory operand stored with its non-reduction dimension contiguous and
// the 128-byte swizzle: atoms of 64 16-bit elements x 8 reduction steps (1 KB);
// `chunk_stride` bytes to the next 64 elements, `step_stride` to the next 8
// reduction steps.
__device__ __forceinline__ uint64_t mma_operand(const void *smem, uint32_t chunk_stride, uint32_t step_stride) {
    return uint64_t((smem_addr(smem) & 0x3FFFFu) >> 4) | (uint64_t(chunk_stride >> 4) << 16) |
           (uint64_t(step_stride >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

// bf16 x bf16 -> fp32, both operands transposed as above, 256 x n outputs.
__device__ __forceinline__ uint32_t mma_shape_bf16(uint32_t n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | ((n >> 3) << 17) | ((256u >> 4) << 24);
}

// One 256 x n x 16 step of the pair into TMEM at `d`; `add` 0 overwrites.  The leader issues it.
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, uint32_t add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                 "l"(a), "l"(b), "r"(shape), "r"(add)
                 : "memory");
}

} // namespace engram
