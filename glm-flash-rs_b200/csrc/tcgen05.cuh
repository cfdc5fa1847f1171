// Blackwell tensor-core helpers of the dense products: tensor memory, tcgen05.mma on operands in shared memory (128-byte swizzle, K-major),
// tensor copies, waits with a bound.
#pragma once
#include "tensor_map.cuh"

namespace gf {

__device__ __forceinline__ void t5_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void t5_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// CG: CTAs of a group (1, or 2 that work on one product)
template <int CG>
__device__ __forceinline__ void t5_alloc(uint32_t *slot_smem, uint32_t cols) {
    if (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot_smem)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot_smem)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <int CG>
__device__ __forceinline__ void t5_dealloc(uint32_t taddr, uint32_t cols) {
    if (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
// D[tmem] (+)= A[smem] * B[smem]^T, 16-bit operands of one type, fp32 accumulators
template <int CG>
__device__ __forceinline__ void t5_mma(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    if (CG == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// arrives on the barrier (CG 2: of both CTAs) once every product that this thread has issued is done
template <int CG>
__device__ __forceinline__ void t5_commit(uint64_t *bar) {
    if (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// 32 columns of this thread's lane, complete on return
__device__ __forceinline__ void t5_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// K-major tile of 64 16-bit elements a row (128 bytes, swizzled), groups of 8 rows 1024 bytes apart, base 1024-aligned.  A step of 16 elements
// moves the start address by 32 bytes.
__device__ __forceinline__ uint64_t t5_desc(uint32_t smem_addr) {
    return (uint64_t)((smem_addr >> 4) & 0x3fffu) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// kind::f16, fp32 accumulators, both operands K-major and of one type
__device__ __forceinline__ uint32_t t5_idesc(int m, int n, bool bf16) {
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
__device__ __forceinline__ bool t5_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ uint32_t t5_cta_rank() {
    uint32_t r;
    asm("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
// address in the cluster of an object at the same offset in CTA `cta`
__device__ __forceinline__ uint32_t t5_of_cta(const void *p, uint32_t cta) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(cta));
    return r;
}
__device__ __forceinline__ void t5_arrive_cluster(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// Tensor copies of 64-element blocks k, k + 1, .. of the rows from y on: a box of several blocks (three dimensions), or of one (two).
// Of a pair: its bytes count on a barrier of either CTA, named by its address in the cluster.
__device__ __forceinline__ void t5_load_pair(void *dst, const CUtensorMap *map, bool blocks, int k, int y, uint32_t bar) {
    if (blocks)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(smem_u32(dst)), "l"((uint64_t)map), "r"(0), "r"(y), "r"(k), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(smem_u32(dst)), "l"((uint64_t)map), "r"(64 * k), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void t5_load(void *dst, const CUtensorMap *map, bool blocks, int k, int y, uint64_t *bar) {
    if (blocks)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(smem_u32(dst)), "l"((uint64_t)map), "r"(0), "r"(y), "r"(k), "r"(smem_u32(bar)) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(smem_u32(dst)), "l"((uint64_t)map), "r"(64 * k), "r"(y), "r"(smem_u32(bar)) : "memory");
}

// Wait for a phase.  Gives up when the CTA's abort flag is up, when another CTA has set the status word, or after a number of polls (seconds);
// then both are set.  SLEEP: nanoseconds that a poll may sleep.
template <uint32_t SLEEP>
__device__ __forceinline__ bool t5_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int *status, int code) {
    if (mbar_try_wait(bar, parity)) return true;
    for (uint32_t i = 0; i < 4000000u; ++i) {
        if (SLEEP ? mbar_try_wait_hint(bar, parity, SLEEP) : mbar_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
        if ((i & 15u) == 15u && *reinterpret_cast<volatile int *>(status) != 0) { *abort_flag = 1; return false; }
    }
    *abort_flag = 1;
    atomicExch(status, code);
    return false;
}

// After a give-up: products in flight have read their operands (each takes a fraction of a microsecond).
__device__ __forceinline__ void t5_settle() {
    for (int i = 0; i < 100; ++i) __nanosleep(1000);
}

// position in a ring of barriers and the parity of its phase
struct T5Ring {
    uint32_t slot = 0, parity = 0;
    __device__ __forceinline__ void next(uint32_t depth) {
        if (++slot == depth) { slot = 0; parity ^= 1; }
    }
};

}  // namespace gf
