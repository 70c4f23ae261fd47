// qagg_tcgen05.cuh -- device helpers of the kernels that multiply on the fifth-generation tensor cores (qagg_mx_gemm.cu): tensor
// memory, shared-memory operand descriptors, instruction descriptors, bounded waits.
#pragma once

#include "qagg_async.cuh"

#include <cuda.h>

namespace qagg {

// ---- waits ------------------------------------------------------------------------------------------------------------------
// try_wait suspends the thread for a while in hardware before it answers.  A wait is for one stage of a ring or one chain of products, a
// few microseconds however long the product as a whole; one that has lasted TC_WAIT_NS gives up: *broken ends every later wait of the
// CTA at once, the status word tells the host.
constexpr unsigned long long TC_WAIT_NS = 4000000000ull;
__device__ __forceinline__ unsigned long long clock_ns()
{
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ bool mbar_suspend_wait(unsigned long long* bar, unsigned parity)
{
    unsigned ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(smem_addr(bar)), "r"(parity)
                 : "memory");
    return ok != 0;
}
// Arrive at the same barrier of CTA `rank` of the cluster.  CTA scope is enough here, and a release to the whole cluster cost the warp
// 1900 cycles each time: what the arrival announces is this SM's own tensor and shared memory, and it is this SM's half of the
// pair's product that reads them.
__device__ __forceinline__ void mbar_arrive_remote(unsigned long long* bar, unsigned rank)
{
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, %1;\n\tmbarrier.arrive.shared::cluster.b64 _, [r];\n\t}" ::"r"(smem_addr(bar)),
                 "r"(rank)
                 : "memory");
}
__device__ __forceinline__ void tc_wait(unsigned long long* bar, unsigned parity, unsigned* broken, unsigned* status, unsigned long long limitNs = TC_WAIT_NS)
{
    if (mbar_suspend_wait(bar, parity))
        return;
    const unsigned long long began = clock_ns();
    while (!mbar_suspend_wait(bar, parity))
    {
        if (*reinterpret_cast<volatile unsigned*>(broken))
            return;
        if (clock_ns() - began > limitNs)
        {
            *reinterpret_cast<volatile unsigned*>(broken) = 1u;
            atomicOr(status, 1u);
            return;
        }
    }
}

// True in one lane of a converged warp.  The tensor cores' instructions take uniform registers; behind this (rather than lane == 0)
// the compiler knows their operands to be uniform.  With lane == 0 each instruction cost its thread about 150 cycles.
__device__ __forceinline__ bool elect_one()
{
    unsigned ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}

// ---- copies -----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_2d(unsigned dst, const void* tmap, int x0, int x1, unsigned long long* bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(tmap),
                 "r"(smem_addr(bar)), "r"(x0), "r"(x1)
                 : "memory");
}
// untiled copy: both addresses and the size are multiples of 16 bytes
__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned long long* bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_addr(bar))
                 : "memory");
}
// generic-proxy stores to shared memory become visible to the tensor cores and the copy engine
__device__ __forceinline__ void fence_async_shared()
{
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// ---- tensor memory ------------------------------------------------------------------------------------------------------------
// 128 lanes x 512 columns of 32 bits; warp w of a CTA reaches lanes 32 * (w % 4) .. + 31.  An address is lane << 16 | column.
// PAIR: for products that two CTAs of a cluster (ranks 0 and 1) make together; both of them call these.
template <bool PAIR = false>
__device__ __forceinline__ void tmem_alloc(unsigned* slot, unsigned columns)
{
    if constexpr (PAIR)
    {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        return;
    }
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <bool PAIR = false>
__device__ __forceinline__ void tmem_free(unsigned base, unsigned columns)
{
    if constexpr (PAIR)
    {
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
        return;
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
}
__device__ __forceinline__ void tc_fence_before()
{
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after()
{
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// 16 columns of this warp's 32 lanes: register j of lane l is column j
__device__ __forceinline__ void tmem_load16(unsigned addr, unsigned (&r)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_load_wait()
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// 32 columns of 16 lanes: registers 4 g, 4 g + 1 are columns 8 g + 2 (l % 4), + 1 of lane l / 4, registers 4 g + 2, + 3 those of lane l / 4 + 8
__device__ __forceinline__ void tmem_store_16x256b(unsigned addr, const unsigned (&r)[16])
{
    asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15])
                 : "memory");
}
// Two 16 x 16 matrices of bytes from shared memory, transposed.  Lanes 0-15 give the rows' addresses of the first, 16-31 of the second.
// Registers 0 and 1 (first matrix), 2 and 3: bytes of column l / 4 (second register: + 8), rows 4 (l % 4) .. + 3.
__device__ __forceinline__ void ldmatrix_trans_b8(unsigned addr, unsigned (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// Registers per thread of this warp's group of four warps, whose warps all get here, from LAUNCHED to N.  (A decrease to more than a warp
// has is an illegal instruction.)
template <int N, int LAUNCHED>
__device__ __forceinline__ void set_registers()
{
    if constexpr (N > LAUNCHED)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    else if constexpr (N < LAUNCHED)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void tmem_store_wait()
{
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// 512 bytes of shared memory (32 rows of 16 bytes) -> 4 columns, repeated in the four groups of 32 lanes: a tile of block scales
// (PAIR: in each of the two CTAs, from its own shared memory at the same address)
template <bool PAIR = false>
__device__ __forceinline__ void tmem_copy_scales(unsigned addr, unsigned long long desc)
{
    if constexpr (PAIR)
    {
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(addr), "l"(desc) : "memory");
        return;
    }
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(addr), "l"(desc) : "memory");
}

// ---- products -----------------------------------------------------------------------------------------------------------------
// Operand in shared memory.  128-byte swizzle: rows of 128 bytes, the 16-byte pieces of row r at piece ^ (r & 7), eight rows per
// 1024-byte group.  K-major (a row = 128 bytes along the contraction): stride = bytes from eight rows to the next eight; leading
// unused.  MN-major (a row = 64 values across it): stride = bytes from eight contraction rows to the next eight, leading = bytes
// from 64 values to the next 64.  No swizzle (scale tiles): stride = bytes from eight 16-byte rows to the next eight.
constexpr unsigned SWIZZLE_NONE = 0, SWIZZLE_128B = 2;
__device__ __forceinline__ unsigned long long smem_desc(unsigned addr, unsigned leading, unsigned stride, unsigned swizzle)
{
    return (unsigned long long) ((addr >> 4) & 0x3fffu) | ((unsigned long long) ((leading >> 4) & 0x3fffu) << 16) |
           ((unsigned long long) ((stride >> 4) & 0x3fffu) << 32) | (1ull << 46) | ((unsigned long long) swizzle << 61);
}
// bf16 x bf16 -> fp32, m x n; transB: operand B is MN-major
__host__ __device__ constexpr unsigned idesc_bf16(int n, bool transB, int m = 128)
{
    return (1u << 4) | (1u << 7) | (1u << 10) | ((transB ? 1u : 0u) << 16) | ((unsigned) (n >> 3) << 17) | ((unsigned) (m >> 4) << 24);
}
// e2m1 x e2m1 with one power-of-two scale per 32 values -> fp32, m x n; sf: which pair of a scale word's four bytes
__host__ __device__ constexpr unsigned idesc_mxf4(int n, unsigned sf, int m = 128)
{
    return (sf << 4) | (1u << 7) | (1u << 10) | ((unsigned) (n >> 3) << 17) | (1u << 23) | ((unsigned) (m >> 4) << 24) | (sf << 29);
}
// D (+)= A B, A in tensor memory (16 contraction values in 8 columns), B in shared memory
__device__ __forceinline__ void mma_bf16_ts(unsigned d, unsigned a, unsigned long long b, unsigned idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((unsigned) add)
                 : "memory");
}
// The same by two CTAs: 256 rows, 128 of A and D in each one's tensor memory, half of B's columns in each one's shared memory, at the same
// addresses.  Issued by rank 0.
__device__ __forceinline__ void mma_bf16_ts_pair(unsigned d, unsigned a, unsigned long long b, unsigned idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((unsigned) add)
                 : "memory");
}
// D (+)= A B over 64 contraction values, both in shared memory, block scales in tensor memory
// (PAIR: two CTAs, 256 rows, half of A's and of B's rows in each one's shared memory; the scales of its own 128 rows of A and of all of
// B's in each one's tensor memory)
template <bool PAIR = false>
__device__ __forceinline__ void mma_mxf4_ss(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned scaleA, unsigned scaleB, bool add)
{
    if constexpr (PAIR)
    {
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                     "r"(scaleA), "r"(scaleB), "r"((unsigned) add)
                     : "memory");
        return;
    }
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"(scaleA), "r"(scaleB), "r"((unsigned) add)
                 : "memory");
}
// arrive on `bar` when all products and scale copies this thread has issued are done
__device__ __forceinline__ void tc_commit(unsigned long long* bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// the same for products of two CTAs: arrives at the barrier of both
__device__ __forceinline__ void tc_commit_pair(unsigned long long* bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)), "h"((unsigned short) 3)
                 : "memory");
}

// ---- clusters -----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned cluster_rank()
{
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// all threads of all CTAs of the cluster; orders shared-memory accesses across it
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned cluster_address(unsigned addr, unsigned rank)
{
    unsigned remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    return remote;
}
__device__ __forceinline__ float4 cluster_load4(unsigned remote)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
    return v;
}

} // namespace qagg
