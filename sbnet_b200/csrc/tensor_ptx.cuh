// Thin wrappers over the tcgen05 (fifth-generation tensor core) and TMEM instructions, shared-memory
// operand descriptors, two-dimensional TMA loads and the cluster controls used by the matrix kernels, which
// run as pairs of CTAs (cta_group::2): one instruction multiplies 256 rows, 128 of them in each CTA's shared
// memory and TMEM, and each CTA holds half of the other operand.  sm_100a only.
#pragma once
#include "async_ptx.cuh"

namespace sbnet {

// One lane of a converged warp, chosen by the hardware.
__device__ __forceinline__ bool elect_one()
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// A bounded wait made by a whole warp, with one outcome for all of its lanes (a lane that gave up alone would
// leave the others behind at the next warp-wide instruction).
static __device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* abortFlag,
                                                      unsigned int* timeouts)
{
    return __all_sync(0xffffffffu, mbar_wait_quick(bar, parity, abortFlag, timeouts));
}

// ---- tensor memory -------------------------------------------------------------------------------
// Whole-warp calls, made by one warp of each CTA of the pair; `cols` is a power of two >= 32.  The warp that
// allocates also frees.
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols)
{
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish()
{
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols)
{
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
// 32 lanes x 32 columns of 32-bit words: lane i of the warp gets row i (of the warp's quarter of the lanes).
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// ---- matrix multiply ------------------------------------------------------------------------------
// Shared-memory operand of 16-bit elements in the 128-byte swizzle.  A tile arrives by TMA as boxes of
// 64 elements (128 bytes) x rows; eight rows (1,024 bytes) are the swizzle's repeating unit.
//  K-major : a box row is one row of the matrix, 64 steps of the reduction; the next eight rows are 1,024
//            bytes on (stride offset).  One instruction takes 16 reduction steps: 32 bytes along the row.
//  MN-major: a box row is one step of the reduction, 64 rows of the matrix; the next eight steps are 1,024
//            bytes on (stride offset), the next 64 rows are the next box, 64 steps * 128 bytes on (leading
//            offset).  16 reduction steps are 2,048 bytes.
template <bool MN> __device__ __forceinline__ uint64_t operand_desc(uint32_t smem)
{
    const uint64_t lead = MN ? 8192 >> 4 : 1, stride = 1024 >> 4;
    return (uint64_t)((smem & 0x3ffff) >> 4) | (lead << 16) | (stride << 32) | (1ull << 46) | (2ull << 61);
}
template <bool MN> constexpr uint32_t kDescStep = MN ? 2048 >> 4 : 32 >> 4;

// kind::f16, fp32 accumulators; format 0 = f16, 1 = bf16 (both operands); M = 256 over the pair.
template <bool A_MN, bool B_MN> __device__ __forceinline__ constexpr uint32_t instr_desc(int format, int n)
{
    return (1u << 4) | ((uint32_t)format << 7) | ((uint32_t)format << 10) | ((A_MN ? 1u : 0u) << 15) |
           ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (16u << 24);
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
// Arrives on the barrier at this offset in both CTAs once every tcgen05.mma this thread has issued is done.
__device__ __forceinline__ void mma_commit_pair(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"((uint16_t)3)
                 : "memory");
}

// ---- the pair -----------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Address, in the cluster's shared window, of this offset in the first CTA of the pair.
__device__ __forceinline__ uint32_t in_first_cta(uint32_t addr)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(0));
    return r;
}
// Relaxed: hands over TMEM, which tcgen05.wait::ld and the tcgen05 fences order.  A release at cluster scope would
// wait for this thread's global stores as well.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr)
{
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// Behind fence_async_smem: hands this CTA's shared memory to the tensor cores.  Released at CTA scope: what is handed
// over is read by this SM; at cluster scope the arrival would wait for the thread's global stores.
__device__ __forceinline__ void mbar_arrive_cluster_release(uint32_t addr)
{
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// ---- loads ------------------------------------------------------------------------------------------
// Into this CTA's shared memory; the bytes are counted on a barrier of either CTA of the pair (a cluster
// address).  c0 (the contiguous coordinate) times the element size is a multiple of 16 bytes at every call.
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
// Shared memory -> matrix; rows and columns outside it are dropped (no coordinate is negative).  The issuing thread closes
// the group and waits for it.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(src), "r"(c0), "r"(c1)
                 : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map)
{
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

} // namespace sbnet
