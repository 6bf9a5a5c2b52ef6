// Fifth-generation tensor cores and what feeds them: descriptors, tensor memory, bulk copies.
#pragma once

#include <cstdint>
#include <cuda.h>            // CUtensorMap
#include <cuda_runtime.h>

#include "tcq_mbarrier.cuh"

namespace tcq {

// ---- shared memory descriptors (64 bits: address / 16, leading and stride byte offsets / 16, version 1 at bit 46, swizzle at bit 61)
// Rows of 128 bytes in the 128-byte swizzle, eight rows to an atom of 1024 bytes (what a TMA load of that swizzle leaves).
__device__ __forceinline__ uint64_t desc_rows128(uint32_t smem) {
    return uint64_t((smem & 0x3FFFFu) >> 4) | uint64_t(1) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
// 32 rows of 16 bytes, one behind the other.
__device__ __forceinline__ uint64_t desc_rows16(uint32_t smem) {
    return uint64_t((smem & 0x3FFFFu) >> 4) | uint64_t(128 >> 4) << 32 | uint64_t(1) << 46;
}

// ---- tensor memory.  CTAS = 2: the form for a pair of CTAs on neighbouring SMs (ranks 2i and 2i + 1 of a cluster); a kernel uses one form only.
template <int CTAS = 1>
__device__ __forceinline__ void tmem_alloc(uint32_t smem_to, uint32_t columns) {       // a whole warp
    if constexpr (CTAS == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_to), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_to), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
}
template <int CTAS = 1>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {           // the same warp
    if constexpr (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// One arrival at the barrier when all that this thread has issued before is done.
__device__ __forceinline__ void tc_commit(uint32_t mbar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(mbar) : "memory");
}
// The pair's form: one arrival at the barrier of this place in both CTAs.
__device__ __forceinline__ void tc_commit_pair(uint32_t mbar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(mbar), "h"(uint16_t(3)) : "memory");
}
// 512 bytes (32 rows of 16) to four columns of lanes 0-31, and again to the other three quarters of the lanes.
// (pair: each CTA's own bytes to its own columns, asked for by the first CTA alone)
template <int CTAS = 1>
__device__ __forceinline__ void tc_copy_scales(uint32_t tmem, uint64_t desc) {
    if constexpr (CTAS == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// N consecutive columns of this warp's 32 lanes.
template <int N> __device__ __forceinline__ void tmem_load(uint32_t tmem, uint32_t (&v)[N]);
template <> __device__ __forceinline__ void tmem_load<8>(uint32_t tmem, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(tmem));
}
template <> __device__ __forceinline__ void tmem_load<16>(uint32_t tmem, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(tmem));
}
template <> __device__ __forceinline__ void tmem_load<32>(uint32_t tmem, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
                   "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
                   "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]) : "r"(tmem));
}

// One lane of a whole warp, always the same.  A warp that loads or issues stays together and lets this lane do it: what the instructions
// take is then known to be the same for the warp, and a stage of the products takes half the time to issue.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
    return p != 0;
}

// ---- bulk copies to shared memory, counted by an mbarrier
__device__ __forceinline__ void tma_load(uint32_t smem, const CUtensorMap* map, int x, int y, uint32_t mbar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem), "l"(map), "r"(x), "r"(y), "r"(mbar) : "memory");
}
// To this CTA's memory, counted by a barrier of the pair's first CTA (a shared::cluster address).
__device__ __forceinline__ void tma_load_pair(uint32_t smem, const CUtensorMap* map, int x, int y, uint32_t mbar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem), "l"(map), "r"(x), "r"(y), "r"(mbar) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t smem, const void* from, uint32_t bytes, uint32_t mbar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem), "l"(from), "r"(bytes), "r"(mbar) : "memory");
}

// ---- clusters
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this place in another CTA of the cluster.
__device__ __forceinline__ uint32_t map_rank(uint32_t smem, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem), "r"(rank));
    return a;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t smem, uint32_t rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(map_rank(smem, rank)) : "memory");
    return v;
}

// A map of [rows][width] bytes, `pitch` bytes a row (a multiple of 16), cut into boxes of [box_rows][128 bytes] in the 128-byte swizzle.
cudaError_t make_byte_map(CUtensorMap* map, const void* base, long long width, long long rows, long long pitch, int box_rows);

// A map of [rows][width] 16-bit numbers, `ld` from row to row (a multiple of 8), cut into boxes of [box_rows][64] in the same swizzle.
cudaError_t make_16bit_map(CUtensorMap* map, const void* base, long long width, long long rows, long long ld, int box_rows);

// A map of scales as rows of 512 bytes, cut into boxes of `box_rows` of them, one behind the other.
cudaError_t make_scale_map(CUtensorMap* map, const void* base, long long rows, int box_rows);

}  // namespace tcq
