// tcgen05 over a pair of CTAs (cta_group::2): one M = 256 MMA whose accumulator's rows 0 .. 127 lie in the even CTA's tensor
// memory and 128 .. 255 in the odd one's; every CTA holds its 128 rows of A and half of B's rows in shared memory.  Operands come by
// tensor-map copies with the 128-byte swizzle.
#pragma once
#include <cuda.h>

#include "umma.cuh"

namespace mlxs {

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// all threads of the cluster's CTAs; what was written before is seen by the others after
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of `saddr` (this CTA's shared memory) in the cluster's CTA `rank`
__device__ __forceinline__ uint32_t map_to_rank(uint32_t saddr, uint32_t rank) {
    uint32_t d;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(saddr), "r"(rank));
    return d;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {   // by cluster address
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// a wait whose other side is in another CTA of the cluster
__device__ __forceinline__ bool mbar_try_wait_cluster(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t limit = (1u << 20)) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    for (uint32_t i = 1; i < limit; ++i) {
        if (mbar_try_wait_cluster(bar, parity)) return true;
        if ((i & 63u) == 63u && *abort_flag) return false;
    }
    return false;
}
// A wait of this CTA has run out: before the CTAs meet for the last time every one of the cluster is told, so that none goes on with what is missing
__device__ __forceinline__ void cluster_abort(volatile int* abort_flag, uint32_t n_ctas) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(const_cast<int*>(abort_flag));
    for (uint32_t r = 0; r < n_ctas; ++r) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_to_rank(at, r)), "r"(1u) : "memory");
}
// after a give-up: copies and products in flight end before the memory goes
__device__ __forceinline__ void abort_drain() { for (int i = 0; i < 2000; ++i) __nanosleep(1000); }
// Tensor-map copies into this CTA's shared memory whose bytes count on a barrier of either CTA of the pair.  The innermost
// coordinate is a multiple of 16 bytes; no multicast.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int32_t c0, int32_t c1, int32_t c2, int32_t c3, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int32_t c0, int32_t c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// both CTAs of the pair allocate and free together
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* slot_smem, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot_smem)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t taddr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
// Operand descriptor, 128-byte swizzle, tiles based at multiples of 1024 bytes.  K-major: rows of 128 bytes (64 inputs), sbo = bytes
// of 8 rows (1024), lbo unused.  M-major: rows of 128 bytes are 64 of M at one k; sbo = bytes of 8 k (1024), lbo = bytes to the
// next 64 of M.
__device__ __forceinline__ uint64_t umma_desc_sw128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) | ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) |
           (1ull << 46) | (2ull << 61);
}
// K-major descriptors by their low words (address >> 4, lbo 16 bytes: 1 << 16), which alone change along a tile, and the high word they share; one CTA
constexpr uint32_t UMMA_SW128_HI = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ void umma_f16_lo(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}"
        ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// M = 256 over the pair; a_m_major: A's descriptor is M-major
__device__ __forceinline__ uint32_t umma_idesc_pair(uint32_t fmt, uint32_t n, bool a_m_major) {
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (a_m_major ? 1u << 15 : 0u) | ((n >> 3) << 17) | ((256u >> 4) << 24);
}
__device__ __forceinline__ void umma_f16_pair(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
        : "memory");
}
// all MMAs issued so far complete -> one arrival on the barrier at this offset in every CTA of `mask`
__device__ __forceinline__ void umma_commit_pair(uint32_t bar, uint16_t mask) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(mask) : "memory");
}
}  // namespace mlxs
