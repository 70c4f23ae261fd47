// qagg_mx_gemm.cu -- products of microscaled matrices on the tensor cores (form: qagg_mx.cuh, instructions: qagg_tcgen05.cuh).
//
//   k_mx_times  y(o, t)  = sum_k w(k, o) x(k, t) + bias(o), both packed in fp4: the tensor cores take codes and block scales as
//               they are.
//   k_mx_grad   dw(o, i) = sum_t dy(o, t) x(i, t)   and   dx(i, t) = sum_o w(i, o) dy(o, t), x or w packed (fp4 or int8) and dy
//               dense.  The packed operand's blocks run across the contraction, so its scales cannot go with a block-scaled
//               product; it is expanded to bf16 (exact) on the way, straight into tensor memory, as operand A.
//
// Both: 128 x n output tiles, dealt to one resident CTA per SM.  A copy warp feeds a ring of shared-memory stages and runs ahead into
// the next tile, one thread issues the products, eight (or four) result warps hold the tile's sums in registers.
//
// The sums.  The tensor cores add to their fp32 accumulator with truncation: n instructions lose less than n units of 2^-23 of the
// largest sum on the way, 6.8e-6 of a sum of positive values after 512 of them.  So a chain ends after CHAIN instructions where the output is fp32; the
// result warps add its value to their registers (round to nearest) and hand the accumulator back, which takes about 2000 cycles
// from the last product to the next.  Two accumulators in turn hide that, and the next tile begins while this one is being
// written.  (A 256-wide tile of the 4-bit product has room for one.)
// 16-bit outputs, which round more coarsely, have longer chains.
//
// Where there are fewer tiles than SMs the contraction is split over the CTAs of a cluster, whose partial sums are added through
// distributed shared memory in rank order: no workspace, no atomics, the same bits on every run.
#include "qagg_mx.cuh"
#include "qagg_mx_groups.h"
#include "qagg_tcgen05.cuh"

#include <algorithm>
#include <atomic>
#include <cstring>
#include <mutex>
#include <string>
#include <type_traits>

namespace qagg {

// set by a bounded wait that ran out; qagg_mx_check takes it, in one step, and reads what it took
__device__ unsigned g_mxStatus, g_mxTaken;
__global__ void k_mx_take_status()
{
    g_mxTaken = atomicExch(&g_mxStatus, 0u);
}
// A wait of the product kernels on a barrier that nothing completes, and one more behind it, which returns at once.
__global__ void __launch_bounds__(32) k_mx_wait_selftest(unsigned long long limitNs)
{
    __shared__ unsigned long long bar;
    __shared__ unsigned broken;
    if (threadIdx.x == 0)
    {
        mbar_init(&bar, 1);
        broken = 0;
        tc_wait(&bar, 0, &broken, &g_mxStatus, limitNs);
        tc_wait(&bar, 0, &broken, &g_mxStatus);
    }
}

constexpr int MAX_STAGES = 8;
constexpr int GEMM_SMEM_MAX = 224 * 1024; // dynamic; barriers and scales take a little more
// Nearly all of an SM's shared memory, always: a second CTA on the SM, of these kernels or of any other that uses tensor memory, would
// wait for the columns this one holds, and CTAs of two clusters that each wait for the other's would never meet at their cluster
// barriers.
constexpr int GEMM_SMEM_MIN = 200 * 1024;
// Tensor-core instructions in a row on one accumulator.  After 32 the sums are within 3e-7; with a single accumulator, where every
// chain costs its hand-over, 64 are taken: within 6e-7, as a sum in plain fp32 is.  A 16-bit result's own rounding is half a step: 4096
// units of 2^-23 for fp16, 32768 for bf16; chains for them lose a 32nd of that at most.
// The planes of an fp32 or fp16 dy count as instructions of their own.  A step takes the smallest plane first: the other way round all
// twelve instructions of an fp32 step truncated a sum that the first four had made large (132 x 512 x 256: 3.9e-7, so 7e-8).
constexpr int CHAIN = 32, CHAIN_SINGLE = 64, CHAIN_FP16 = 128, CHAIN_BF16 = 1024;
template <class T, bool SINGLE>
constexpr int CHAIN_OF = std::is_same_v<T, __half> ? CHAIN_FP16 : std::is_same_v<T, __nv_bfloat16> ? CHAIN_BF16 : SINGLE ? CHAIN_SINGLE : CHAIN;

struct GemmBars
{
    unsigned long long full[MAX_STAGES];  // copies of the stage have landed
    unsigned long long conv[MAX_STAGES];  // gradients: packed operand expanded into tensor memory
    unsigned long long dense[MAX_STAGES]; // gradients, dense loaders: their part of the stage is written
    unsigned long long empty[MAX_STAGES]; // products that read the stage are done
    unsigned long long ready[2];          // the accumulator holds a finished chain
    unsigned long long taken[2];          // the result warps have it
    unsigned tmem;
    unsigned broken;
};

// place in the ring of stages and the parity of its current round
struct Ring
{
    int s = 0;
    unsigned par = 0;
    __device__ __forceinline__ void next(int stages)
    {
        if (++s == stages)
        {
            s = 0;
            par ^= 1;
        }
    }
};

// this CTA's steps of the contraction
__device__ __forceinline__ void split_range(int steps, int rank, int splits, int& first, int& count)
{
    first = (int) ((long long) steps * rank / splits);
    count = (int) ((long long) steps * (rank + 1) / splits) - first;
}

// The copies this thread started have landed, after a wait ran out too (or a bounded wait for them ran out as well), before the CTA goes.
__device__ __forceinline__ void drain_copies(GemmBars* bars, long long issued, int stages)
{
    const unsigned long long began = clock_ns();
    for (long long i = issued > stages ? issued - stages : 0; i < issued; ++i)
        while (!mbar_suspend_wait(&bars->full[i % stages], (unsigned) (i / stages) & 1) && clock_ns() - began < TC_WAIT_NS)
            ;
}

// First warp, all lanes: barriers.  The copies may start right after this, before the CTA has met.
__device__ __forceinline__ void init_barriers(GemmBars* bars, int stages, int convCount, int denseCount, int resultWarps)
{
    const int lane = threadIdx.x & 31, s = lane >> 2;
    if (s < stages)
        mbar_init(lane & 2 ? (lane & 1 ? &bars->empty[s] : &bars->dense[s]) : (lane & 1 ? &bars->conv[s] : &bars->full[s]),
                  (lane & 3) == 1 ? convCount : (lane & 3) == 2 ? denseCount : 1);
    if (lane < 2)
    {
        mbar_init(&bars->ready[lane], 1);
        mbar_init(&bars->taken[lane], resultWarps);
    }
    if (lane == 0)
        bars->broken = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_shared();
    __syncwarp();
}
static_assert(MAX_STAGES <= 8, "four lanes of a warp per stage");

// ---- results ------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ unsigned pack2(float a, float b, __half*)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ unsigned pack2(float a, float b, __nv_bfloat16*)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
}

// `cols` columns (a multiple of 16) of a finished chain, set or added to the registers.
template <bool PAIR, int ACC>
__device__ __forceinline__ void take_chain(GemmBars* bars, int buf, unsigned par, unsigned tmem, int cols, bool firstChain, float (&acc)[ACC])
{
    tc_wait(&bars->ready[buf], par, &bars->broken, &g_mxStatus);
    __syncwarp();
    tc_fence_after();
#pragma unroll
    for (int p = 0; p < ACC / 16; ++p)
        if (p * 16 < cols)
        {
            unsigned r[16];
            tmem_load16(tmem + p * 16, r);
            tmem_load_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j)
                acc[p * 16 + j] = firstChain ? __uint_as_float(r[j]) : acc[p * 16 + j] + __uint_as_float(r[j]);
        }
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0)
    {
        if constexpr (PAIR)
            mbar_arrive_remote(&bars->taken[buf], 0);
        else
            mbar_arrive(&bars->taken[buf]);
    }
}
// A CTA's only tile with a single chain goes from tensor memory to its place sixteen columns at a time: the loop is a tenth of the code that
// registers holding the whole tile need, and a launch of a few microseconds spends much of them on fetching instructions.
// f(j, values): columns j .. j + 15.
template <class F>
__device__ __forceinline__ void drain_chain(GemmBars* bars, unsigned tmem, int cols, bool nothing, F f)
{
    if (!nothing)
        tc_wait(&bars->ready[0], 0, &bars->broken, &g_mxStatus);
    __syncwarp();
    tc_fence_after();
#pragma unroll 1
    for (int j = 0; j < cols; j += 16)
    {
        float v[16];
        if (nothing)
        {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                v[e] = 0.0f;
        }
        else
        {
            unsigned r[16];
            tmem_load16(tmem + j, r);
            tmem_load_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e)
                v[e] = __uint_as_float(r[e]);
        }
        f(j, v);
    }
}
// Which accumulator a chain uses, and the parity of its barriers' phase.
struct Chains
{
    int buf = 0;
    unsigned par = 0;
    __device__ __forceinline__ void next(int bufs)
    {
        if (++buf >= bufs)
        {
            buf = 0;
            par ^= 1;
        }
    }
};

// Sums of one lane (row m of the tile) and `cols` columns from n on, straight to the output:
//   columns  out[n * ld + m]: 32 lanes are 32 neighbours (`partner`: the lane whose row is m ^ 1; 16-bit types are stored in pairs)
//   rows     out[m * ld + n], fp32: 16 bytes a thread where the alignment allows
template <class T, int ACC>
__device__ __forceinline__ void write_columns(T* out, long long ld, long long m, long long M, long long n, long long N, int cols, const float (&acc)[ACC], float bias,
                                              int partner, bool pairs)
{
    const long long left = N - n;
    const int c = (int) (left < cols ? left : cols);
    if constexpr (sizeof(T) == 2)
    {
        if (pairs) // uniform: all rows of the tile exist, ld is even, the base 4-byte aligned
        {
            const bool odd = m & 1;
            T* p = out + (n + odd) * ld + (m & ~1LL);
            const long long two = 2 * ld;
#pragma unroll
            for (int j = 0; j < ACC; j += 2)
            {
                // this lane stores column j (even row) or j + 1 (odd row) of its pair of rows
                const float a = acc[j] + bias, b = acc[j + 1] + bias;
                const float got = __shfl_sync(0xffffffffu, odd ? a : b, partner);
                const unsigned v = odd ? pack2(got, b, (T*) nullptr) : pack2(a, got, (T*) nullptr);
                if (j + (odd ? 1 : 0) < c)
                    *reinterpret_cast<unsigned*>(p) = v;
                p += two;
            }
            return;
        }
    }
    if (m >= M)
        return;
    T* p = out + n * ld + m;
#pragma unroll
    for (int j = 0; j < ACC; ++j)
    {
        if (j < c)
            put(p, acc[j] + bias);
        p += ld;
    }
}
template <int ACC>
__device__ __forceinline__ void write_row(float* out, long long ld, long long m, long long M, long long n, long long N, int cols, const float (&acc)[ACC], bool add, bool vec)
{
    if (m >= M)
        return;
    const long long left = N - n;
    const int c = (int) (left < cols ? left : cols);
    float* p = out + m * ld + n;
#pragma unroll
    for (int j = 0; j < ACC; j += 4)
    {
        if (vec && j + 4 <= c)
        {
            float4* q = reinterpret_cast<float4*>(p + j);
            float4 v = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
            if (add)
            {
                const float4 o = *q;
                v = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
            }
            *q = v;
        }
        else
        {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (j + e < c)
                    p[j + e] = add ? p[j + e] + acc[j + e] : acc[j + e];
        }
    }
}

// Split contraction: each CTA leaves its partial sums in its shared memory ([n][128 rows], or for rows [m][bn + 4]), and CTA `rank` adds
// up and writes its share of the tile's columns (rows).  Called by all threads; result warps have put their sums down.
// wide: four neighbours of the output are one aligned word of 4 * sizeof(T) bytes.
__device__ __forceinline__ void put4(float* p, const float4& s) { *reinterpret_cast<float4*>(p) = s; }
template <class T>
__device__ __forceinline__ void put4(T* p, const float4& s)
{
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2(s.x, s.y, p), pack2(s.z, s.w, p));
}
template <int SPLITS, bool ROWS, class T>
__device__ __forceinline__ void reduce_parts(float* buf, int rank, int bn, T* out, long long ld, long long m0, long long M, long long n0, long long N, const float* bias,
                                             bool add, bool wide)
{
    const long long restM = M - m0, restN = N - n0;
    const int rows = (int) (restM < 128 ? restM : 128), cols = (int) (restN < bn ? restN : bn);
    const int pitch = ROWS ? bn + 4 : 128;
    const int lines = ROWS ? rows : cols, width = ROWS ? cols : rows;
    const int perLine = (width + 3) / 4;
    const int u1 = lines * perLine * (rank + 1) / SPLITS;
#pragma unroll 1
    for (int u = lines * perLine * rank / SPLITS + (int) threadIdx.x; u < u1; u += blockDim.x)
    {
        const int l = u / perLine, w = (u - l * perLine) * 4;
        const unsigned at = smem_addr(buf + l * pitch + w);
        float4 v[SPLITS];
#pragma unroll
        for (int k = 0; k < SPLITS; ++k)
            v[k] = cluster_load4(cluster_address(at, k));
        const long long col = (ROWS ? n0 : m0) + w;
        T* p = out + ((ROWS ? m0 : n0) + l) * ld + col;
        float4 s = v[0];
#pragma unroll
        for (int k = 1; k < SPLITS; ++k)
            s = make_float4(s.x + v[k].x, s.y + v[k].y, s.z + v[k].z, s.w + v[k].w);
        float e[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (w + j < width)
            {
                if constexpr (ROWS)
                    e[j] += add ? (float) p[j] : 0.0f;
                else
                    e[j] += bias ? bias[col + j] : 0.0f;
            }
        if (wide && w + 4 <= width)
            put4(p, make_float4(e[0], e[1], e[2], e[3]));
        else
        {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (w + j < width)
                    put(p + j, e[j]);
        }
    }
}
template <bool ROWS, class T>
__device__ __forceinline__ void reduce_cluster(float* buf, int splits, int rank, int bn, T* out, long long ld, long long m0, long long M, long long n0, long long N,
                                               const float* bias, bool add, bool wide)
{
    __syncwarp();
    cluster_sync();
    if (splits == 2)
        reduce_parts<2, ROWS>(buf, rank, bn, out, ld, m0, M, n0, N, bias, add, wide);
    else if (splits == 4)
        reduce_parts<4, ROWS>(buf, rank, bn, out, ld, m0, M, n0, N, bias, add, wide);
    else
        reduce_parts<8, ROWS>(buf, rank, bn, out, ld, m0, M, n0, N, bias, add, wide);
    __syncwarp();
    cluster_sync(); // nobody leaves while its partial sums are being read
}
template <bool ROWS, int ACC>
__device__ __forceinline__ void put_partial(float* buf, int bn, int m, int col0, int cols, const float (&acc)[ACC])
{
    if constexpr (ROWS)
    {
#pragma unroll
        for (int j = 0; j < ACC; j += 4)
            if (j < cols)
                *reinterpret_cast<float4*>(buf + m * (bn + 4) + col0 + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
    }
    else
    {
#pragma unroll
        for (int j = 0; j < ACC; ++j)
            if (j < cols)
                buf[(col0 + j) * 128 + m] = acc[j];
    }
}

// ---- 4-bit product --------------------------------------------------------------------------------------------------------------

struct TimesArgs
{
    const unsigned char* scaleW;
    const unsigned char* scaleX;
    const float* bias;
    void* y;
    long long ld, O, T, K;
    int bn, stages, splits, tilesM, tiles;
    int pairs, wide4; // y: two rows of a column can be written at once, four of them
};

constexpr int TT = 384;  // copy, product, allocating and spare warp; eight result warps
constexpr int TIMES_NARROW = 32;
constexpr int TK = 256;  // contraction values per stage: 128 bytes of codes
constexpr int TIMES_PAIR = 256; // width of a tile that two CTAs make
// codes of 128 rows of W and `rows` of X, scales of W's and of bn of X's
__host__ __device__ inline int times_stage_bytes(int bn, int rows)
{
    return 128 * 128 + rows * 128 + 1024 + (bn > 128 ? 2048 : 1024);
}

// ACC: most columns of the tile that one result warp holds.  The narrow tiles of few tokens have a kernel of their own, whose results are
// a quarter of the code: a launch that lasts 3 us feels the instruction fetches (128: 1400 cycles to put the sums down).
// PAIR: two CTAs make a 256 x 256 tile together, each with half of W's and of X's rows: 35 KB a step for each instead of 51.
template <class T, int ACC, bool PAIR>
__global__ void __launch_bounds__(TT, 1) k_mx_times(const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapX, const TimesArgs a)
{
    extern __shared__ unsigned char dyn[];
    __shared__ GemmBars bars;
    unsigned char* stage0 = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t) 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int bn = a.bn, S = a.stages, share = PAIR ? bn / 2 : bn, stageBytes = times_stage_bytes(bn, share);
    const unsigned codesBytes = 16384 + share * 128;
    const int steps = (int) ((a.K + TK - 1) / TK);
    const int rank = PAIR || a.splits > 1 ? (int) cluster_rank() : 0;
    int first = 0, count = steps;
    if (!PAIR)
        split_range(steps, rank, a.splits, first, count);
    const int firstTile = PAIR ? blockIdx.x >> 1 : blockIdx.x, tileStep = PAIR ? gridDim.x >> 1 : gridDim.x;
    const long long chunks = mx_scale_tiles(a.K); // scale tiles along the contraction, 128 values each
    const int resultWarps = bn > 128 ? 8 : 4;
    const int bufs = bn > 128 ? 1 : 2; // accumulators, 128 columns apart
    constexpr unsigned SIDE = 256;     // block scales: 24 columns a stage
    const int chainSteps = (bufs == 1 ? CHAIN_OF<T, true> : CHAIN_OF<T, false>) / 4;

    // The copying thread's time per step counts: what depends on the tile alone is worked out once per tile.
    struct Source
    {
        int m0, n0, rowsX;
        const unsigned char *scaleW, *scaleX;
    };
    auto source_of = [&](int tile) {
        const int m = (tile % a.tilesM) * (PAIR ? 2 : 1) + (PAIR ? rank : 0), n0 = tile / a.tilesM * bn;
        // (a CTA of a pair may have no rows of W: codes outside read as zero, scales are taken from the last rows)
        const long long rowTile = m * 128LL < a.O ? m : (a.O - 1) / 128;
        return Source{m * 128, n0 + (PAIR ? rank * share : 0), bn > 128 && n0 + 128 < a.T ? 2 : 1, a.scaleW + rowTile * chunks * 512,
                      a.scaleX + (long long) (n0 / 128) * chunks * 512};
    };
    auto copy_step = [&](const Source& src, int i, int s) {
        const unsigned at = smem_addr(stage0) + s * stageBytes, sw = at + codesBytes;
        const int k = first + i;
        const unsigned bytes = chunks - 2 * k < 2 ? 512 : 1024;
        unsigned long long* full = &bars.full[s];
        mbar_arrive_expect_tx(full, codesBytes + bytes * (1 + src.rowsX));
        tma_load_2d(at, &mapW, k * 128, src.m0, full);
        tma_load_2d(at + 16384, &mapX, k * 128, src.n0, full);
        bulk_load(sw, src.scaleW + k * 1024LL, bytes, full);
        bulk_load(sw + 1024, src.scaleX + k * 1024LL, bytes, full);
        if (src.rowsX == 2)
            bulk_load(sw + 2048, src.scaleX + (chunks + 2LL * k) * 512, bytes, full);
    };
    int early = 0; // steps of the first tile whose copies start before the CTA has met
    if (warp == 0)
    {
        init_barriers(&bars, S, 1, 1, PAIR ? 2 * resultWarps : resultWarps);
        if (elect_one())
        {
            const Source src = source_of(firstTile);
            for (; early < count && early < S; ++early)
                copy_step(src, early, early);
        }
        early = count < S ? count : S;
        __syncwarp();
    }
    if (warp == 2)
        tmem_alloc<PAIR>(&bars.tmem, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    if (PAIR)
        cluster_sync(); // the other CTA's barriers exist
    tc_fence_after();
    const unsigned tm = bars.tmem;

    if (warp == 0)
    {
        if (elect_one())
        {
            Ring ring;
            for (int i = 0; i < early; ++i)
                ring.next(S);
            long long issued = early;
            for (int tile = firstTile; tile < a.tiles; tile += tileStep)
            {
                const Source src = source_of(tile);
                for (int i = tile == firstTile ? early : 0; i < count; ++i, ++issued)
                {
                    if (issued >= S)
                        tc_wait(&bars.empty[ring.s], ring.par ^ 1, &bars.broken, &g_mxStatus);
                    if (*reinterpret_cast<volatile unsigned*>(&bars.broken))
                    {
                        tile = a.tiles;
                        break;
                    }
                    copy_step(src, i, ring.s);
                    ring.next(S);
                }
            }
            drain_copies(&bars, issued, S);
        }
    }
    else if (warp == 1 && (!PAIR || rank == 0))
    {
        if (elect_one())
        {
            Ring ring;
            Chains chain;
            bool fresh = true; // accumulators that no chain has used
            const unsigned id0 = idesc_mxf4(bn, 0, PAIR ? 256 : 128), id2 = idesc_mxf4(bn, 2, PAIR ? 256 : 128);
            const unsigned long long dW = smem_desc(smem_addr(stage0), 16, 1024, SWIZZLE_128B);
            const unsigned long long dX = dW + (16384 >> 4);
            const unsigned long long dS = smem_desc(smem_addr(stage0) + codesBytes, 16, 128, SWIZZLE_NONE);
            for (int tile = firstTile; tile < a.tiles; tile += tileStep)
            {
                const long long n0 = (long long) (tile / a.tilesM) * bn;
                const bool twoX = bn > 128 && n0 + 128 < a.T;
                int inChain = 0;
                for (int i = 0; i < count; ++i)
                {
                    if (inChain == 0 && !fresh)
                        tc_wait(&bars.taken[chain.buf], chain.par ^ 1, &bars.broken, &g_mxStatus);
                    tc_wait(&bars.full[ring.s], ring.par, &bars.broken, &g_mxStatus);
                    if (PAIR)
                        tc_wait(&bars.conv[ring.s], ring.par, &bars.broken, &g_mxStatus); // the other CTA's copies
                    tc_fence_after();
                    const unsigned d = tm + chain.buf * 128;
                    const unsigned long long off = (unsigned long long) (unsigned) (ring.s * stageBytes) >> 4;
                    const unsigned long long w = dW + off, x = dX + off, sc = dS + off;
                    const unsigned sa = tm + SIDE + ring.s * 24, sb = sa + 8; // eight columns of W's scales, sixteen of X's
                    const long long left = a.K - (long long) (first + i) * TK;
                    const bool more = inChain > 0;
                    tmem_copy_scales<PAIR>(sa, sc);
                    tmem_copy_scales<PAIR>(sb, sc + (1024 >> 4));
                    if (twoX)
                        tmem_copy_scales<PAIR>(sb + 4, sc + (2048 >> 4));
                    mma_mxf4_ss<PAIR>(d, w, x, id0, sa, sb, more);
                    if (left > 64)
                        mma_mxf4_ss<PAIR>(d, w + 2, x + 2, id2, sa, sb, true);
                    if (left > 128)
                    {
                        tmem_copy_scales<PAIR>(sa + 4, sc + (512 >> 4));
                        tmem_copy_scales<PAIR>(sb + 8, sc + (1536 >> 4));
                        if (twoX)
                            tmem_copy_scales<PAIR>(sb + 12, sc + (2560 >> 4));
                        mma_mxf4_ss<PAIR>(d, w + 4, x + 4, id0, sa + 4, sb + 8, true);
                        if (left > 192)
                            mma_mxf4_ss<PAIR>(d, w + 6, x + 6, id2, sa + 4, sb + 8, true);
                    }
                    if constexpr (PAIR)
                        tc_commit_pair(&bars.empty[ring.s]);
                    else
                        tc_commit(&bars.empty[ring.s]);
                    ring.next(S);
                    if (++inChain == chainSteps || i + 1 == count)
                    {
                        if constexpr (PAIR)
                            tc_commit_pair(&bars.ready[chain.buf]);
                        else
                            tc_commit(&bars.ready[chain.buf]);
                        chain.next(bufs);
                        fresh = fresh && chain.buf != 0;
                        inChain = 0;
                    }
                }
            }
        }
    }
    else if (PAIR && warp == 3 && rank == 1)
    {
        if (elect_one())
        {
            Ring ring; // tells the issuing CTA of the copies that have landed here
            for (int tile = firstTile; tile < a.tiles; tile += tileStep)
                for (int i = 0; i < count; ++i)
                {
                    tc_wait(&bars.full[ring.s], ring.par, &bars.broken, &g_mxStatus);
                    mbar_arrive_remote(&bars.conv[ring.s], 0);
                    ring.next(S);
                }
        }
    }
    else if (warp >= 4)
    {
        const int rw = warp - 4, quad = rw & 3, half = rw >> 2;
        if (rw < resultWarps)
        {
            const int cols = bn > 128 ? 128 : bn;
            const unsigned mine = tm + ((unsigned) (quad * 32) << 16) + half * 128;
            const int m = quad * 32 + lane;
            Chains chain;
            for (int tile = firstTile; tile < a.tiles; tile += tileStep)
            {
                const long long m0 = (long long) (tile % a.tilesM) * (PAIR ? 256 : 128) + (PAIR ? rank * 128 : 0), n0 = (long long) (tile / a.tilesM) * bn;
                const float bias = a.bias && a.splits == 1 && m0 + m < a.O ? a.bias[m0 + m] : 0.0f;
                float* buf = reinterpret_cast<float*>(stage0);
                if (!PAIR && a.tiles <= tileStep && count <= chainSteps)
                {
                    drain_chain(&bars, mine, cols, count == 0, [&](int j, const float(&v)[16]) {
                        if (a.splits > 1)
                            put_partial<false>(buf, bn, m, half * 128 + j, 16, v);
                        else
                            write_columns((T*) a.y, a.ld, m0 + m, a.O, n0 + half * 128 + j, a.T, 16, v, bias, lane ^ 1, a.pairs && m0 + 128 <= a.O);
                    });
                    break;
                }
                float acc[ACC];
#pragma unroll
                for (int j = 0; j < ACC; ++j)
                    acc[j] = 0.0f;
                for (int i = 0; i < count; i += chainSteps, chain.next(bufs))
                    take_chain<PAIR>(&bars, chain.buf, chain.par, mine + chain.buf * 128, cols, i == 0, acc);
                if (!PAIR && a.splits > 1)
                    put_partial<false>(buf, bn, m, half * 128, cols, acc);
                else
                    write_columns((T*) a.y, a.ld, m0 + m, a.O, n0 + half * 128, a.T, cols, acc, bias, lane ^ 1, a.pairs && m0 + 128 <= a.O);
            }
        }
    }
    __syncwarp();
    if (!PAIR && a.splits > 1) // one tile per cluster
        reduce_cluster<false, T>(reinterpret_cast<float*>(stage0), a.splits, rank, bn, (T*) a.y, a.ld, (long long) (blockIdx.x % a.tilesM) * 128, a.O,
                                 (long long) (blockIdx.x / a.tilesM) * bn, a.T, a.bias, false, a.wide4);
    tc_fence_before();
    if (PAIR)
        cluster_sync(); // neither goes while the other may still arrive at its barriers or use its memory
    __syncthreads();
    if (warp == 2)
        tmem_free<PAIR>(tm, TMEM_COLS);
}

// ---- 4-bit product, a few tokens ------------------------------------------------------------------------------------------------
// Up to four tokens read the weights once and do little with them: no tensor cores, no tensor maps, one short launch.  A warp takes one
// output row (two where there are enough), a lane every 32nd block of it: 16 bytes, the next ones on their way.  Twice an element is an
// integer of at most 12, looked up four at a time by PRMT, so a block's products are integer dot products, exact: with mag the
// magnitudes of w and x signed, sum w x = sum mag x - 2 * (sum over negative w of mag x).  x is decoded once per CTA, into shared
// memory.  Only the sum over blocks is in fp32.
// When it is chosen: times_few.

// four codes (16 bits) -> magnitudes times two; mask: 0xff where the code is negative, 0x80 where not
__device__ __forceinline__ unsigned fp4_magnitudes(unsigned c, unsigned& mask)
{
    // a selector's top bit spreads the chosen byte's sign (__byte_perm ignores that bit)
    asm("prmt.b32 %0, %1, %1, %2;" : "=r"(mask) : "r"(0x80808080u), "r"(c));
    return __byte_perm(0x03020100u, 0x0c080604u, c & 0x7777u);
}
// v * 2^e, e from -256 to 252
__device__ __forceinline__ float scale_by(float v, int e)
{
    if ((unsigned) (e + 126) < 253u)
        return v * __uint_as_float((unsigned) (e + 127) << 23);
    const int h = e >> 1; // two factors that are floats
    auto pow2 = [](int k) { return __uint_as_float(k > -127 ? (unsigned) (k + 127) << 23 : 0x00400000u >> (-127 - k)); };
    return v * pow2(h) * pow2(e - h);
}

template <class T, int NT, int R>
__global__ void __launch_bounds__(256) k_mx_times_few(const unsigned char* __restrict__ codesW, const unsigned char* __restrict__ scalesW,
                                                      const unsigned char* __restrict__ codesX, const unsigned char* __restrict__ scalesX,
                                                      const float* __restrict__ bias, T* __restrict__ y, long long ld, int O, int tokens, int blocks)
{
    extern __shared__ __align__(16) unsigned char few[];
    uint4* x = reinterpret_cast<uint4*>(few);                 // [token][block][2]: 32 signed bytes
    unsigned char* xs = few + (size_t) NT * blocks * 32;      // [token][block]
    const int lane = threadIdx.x & 31;
    const int unit = blockIdx.x * 8 + (threadIdx.x >> 5);
    // two rows 32 apart: their scale bytes lie together
    const int row0 = R == 2 ? unit / 64 * 128 + unit / 32 % 2 * 64 + unit % 32 : unit;
    const long long chunks = (blocks + 3) / 4, pitch = blocks * 16LL;
    const unsigned char *pw[R], *ps[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
    {
        const int o = min(row0 + 32 * r, O - 1);
        pw[r] = codesW + o * pitch;
        ps[r] = scalesW + (o >> 7) * chunks * 512 + (o & 31) * 16 + (o >> 5 & 3) * 4;
    }
    uint4 wc[R];
    unsigned wb[R];
    auto fetch = [&](int b) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (b < blocks)
            {
                wc[r] = __ldcs(reinterpret_cast<const uint4*>(pw[r]) + b);
                wb[r] = ps[r][(b >> 2) * 512LL + (b & 3)];
            }
    };
    fetch(lane);
    for (int i = threadIdx.x; i < NT * blocks; i += 256)
    {
        const int t = i / blocks, b = i - t * blocks;
        if (t >= tokens)
            break;
        const uint4 c = reinterpret_cast<const uint4*>(codesX + t * pitch)[b];
        xs[i] = scalesX[(b >> 2) * 512LL + t * 16 + (b & 3)];
        unsigned v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
        {
            const unsigned w = (&c.x)[q >> 1];
            unsigned mask;
            const unsigned mag = fp4_magnitudes(q & 1 ? w >> 16 : w & 0xffffu, mask);
            v[q] = __vsub4(mag, 2u * (mag & mask));
        }
        x[2 * i] = make_uint4(v[0], v[1], v[2], v[3]);
        x[2 * i + 1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
    __syncthreads();
    float sum[R][NT] = {};
    for (int b = lane; b < blocks; b += 32)
    {
        uint4 w[R];
        unsigned ws[R];
#pragma unroll
        for (int r = 0; r < R; ++r)
            w[r] = wc[r], ws[r] = wb[r];
        fetch(b + 32);
        int all[R][NT] = {}, negative[R][NT] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            uint4 xv[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t)
                xv[t] = x[2 * (t * blocks + b) + h];
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                {
                    const unsigned c = (&w[r].x)[2 * h + (q >> 1)];
                    unsigned mask;
                    const unsigned mag = fp4_magnitudes(q & 1 ? c >> 16 : c & 0xffffu, mask);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                    {
                        all[r][t] = __dp4a((int) mag, (int) (&xv[t].x)[q], all[r][t]);
                        negative[r][t] = __dp4a((int) (mag & mask), (int) (&xv[t].x)[q], negative[r][t]);
                    }
                }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
        {
            const unsigned xb = xs[t * blocks + b];
#pragma unroll
            for (int r = 0; r < R; ++r)
            {
                const float v = scale_by((float) (all[r][t] - 2 * negative[r][t]), (int) (ws[r] + xb) - 256); // both operands are doubled
                sum[r][t] += ws[r] == 255u || xb == 255u ? __uint_as_float(0x7fffffffu) : v;
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t)
        {
#pragma unroll
            for (int d = 16; d > 0; d /= 2)
                sum[r][t] += __shfl_xor_sync(0xffffffffu, sum[r][t], d);
            const int o = row0 + 32 * r;
            if (lane == 0 && t < tokens && o < O)
                put(y + t * ld + o, sum[r][t] + (bias ? bias[o] : 0.0f));
        }
}

template <class T>
static cudaError_t launch_times_few(cudaStream_t st, const void* wc, const void* ws, const void* xc, const void* xs, const float* bias, T* y, long long ld, long long O,
                                    int tokens, long long K, int sms)
{
    const int blocks = (int) mx_blocks(K);
    const bool two = O >= sms * 48LL; // a warp for every two rows still fills the SMs
    const unsigned grid = (unsigned) (((two ? (O + 127) / 128 * 64 : O) + 7) / 8);
    const auto launch = [&](auto kernel, int nt) {
        kernel<<<grid, 256, nt * blocks * 33, st>>>((const unsigned char*) wc, (const unsigned char*) ws, (const unsigned char*) xc, (const unsigned char*) xs, bias, y, ld, (int) O,
                                                    tokens, blocks);
        return cudaGetLastError();
    };
    if (tokens == 1)
        return two ? launch(k_mx_times_few<T, 1, 2>, 1) : launch(k_mx_times_few<T, 1, 1>, 1);
    if (tokens == 2)
        return two ? launch(k_mx_times_few<T, 2, 2>, 2) : launch(k_mx_times_few<T, 2, 1>, 2);
    return two ? launch(k_mx_times_few<T, 4, 2>, 4) : launch(k_mx_times_few<T, 4, 1>, 4);
}

// ---- gradients --------------------------------------------------------------------------------------------------------------------

struct GradArgs
{
    const unsigned char* scales;
    const void* dy;     // dense operand, for the loaders
    long long ldDy;
    void* out;
    long long ld;
    long long I;        // rows of the packed matrix: lanes of the tile
    long long C;        // columns of the packed matrix: the contraction
    long long N;        // the other dimension
    int bn, stages, splits, tilesM, tiles;
    int vec;            // dy can be read 16 bytes a time
    int wide, wide4;    // out: rows can be written 16 bytes a time, columns in pairs of rows; four neighbours at once
    int add;
    int pair;
};

constexpr int GK = 64; // contraction values per stage

// packed part of a stage: 64 contraction values x 128 rows of codes, and the scale tile they lie in (128 values x 128 rows)
__host__ __device__ inline int grad_codes_bytes(int format)
{
    return GK * (format == QAGG_MXFP4 ? 64 : 128);
}
constexpr int GRAD_SCALE_BYTES = 512, GRAD_SCALE_ROOM = 1024; // stages stay multiples of 1024 bytes

// Codes to bf16.  v: four codes of one row (int8), or four bytes with one code of an even and one of an odd row each (fp4), from
// contraction values k..k+3; pair 0 is (k, k + 1), pair 1 (k + 2, k + 3).
// int8: 0x43 over a code byte is the bf16 number 128 + (its low seven bits) with bit 7 moved aside; q = low - (bit 7), so
// q = (128 + low) - (128 or 256), and 256 is 0x4380.  fp4: the element's exponent and mantissa bits, set where bf16 has them, give
// its value times 2^-126, subnormal included; one multiplication puts two copies of a nibble where sign and the rest belong.  The
// multiplier has the 2^126 in it (X <= 1: largest magnitudes below 16) or the step takes two.  All products are exact.
__device__ __forceinline__ unsigned bf16x2_mul(unsigned a, unsigned b)
{
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const unsigned*>(&r);
}
__device__ __forceinline__ unsigned bf16x2_sub(unsigned a, unsigned b)
{
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const unsigned*>(&r);
}
__device__ __forceinline__ unsigned expand_int8(unsigned v, int pair, unsigned scale)
{
    const unsigned x = __byte_perm(v, 0x43434343u, pair ? 0x4342 : 0x4140);
    return bf16x2_mul(bf16x2_sub(x & 0xff7fff7fu, x & 0xff80ff80u), scale);
}
__device__ __forceinline__ unsigned expand_fp4(unsigned v, int pair, bool odd, bool large, unsigned scale)
{
    const unsigned x = __byte_perm(v, 0, pair ? 0x4342 : 0x4140);
    const unsigned t = (odd ? (x & 0x00f000f0u) * 0x104u : (x & 0x000f000fu) * 0x1040u) & 0x81c081c0u;
    return large ? bf16x2_mul(bf16x2_mul(t, 0x7e807e80u), scale) : bf16x2_mul(t, scale); // 0x7e80: 2^126
}
// multiplier of a block as bf16 bits: 2^X / 64 (int8; subnormal below byte 7), 2^X or 2^(X + 126) (fp4)
constexpr unsigned FP4_LARGE = 128; // scale bytes above this have no 2^(X + 126)
template <int FMT>
__device__ __forceinline__ unsigned scale_bf16(unsigned byte, bool large)
{
    if (FMT == QAGG_MXFP4 && !large)
        return (byte + 126u) << 7;
    if (byte == 255u)
        return 0x7fffu;
    if (FMT == QAGG_MXINT8)
        return byte > 6u ? (byte - 6u) << 7 : 1u << byte;
    return byte ? byte << 7 : 0x40u;
}

// Eight dense values as sums of bf16 planes, exactly: the top eight significant bits by truncation, the next eight, the rest (fp16 has
// eleven: two planes; fp32 twenty-four: three).  Infinities and NaN stay in the first plane, which the second form sees to.
template <class T, int NP, bool SPECIAL>
__device__ __forceinline__ void split8(const Raw8<T>& raw, unsigned (&w)[NP][4])
{
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        float v[2] = {(float) e[2 * i], (float) e[2 * i + 1]};
#pragma unroll
        for (int k = 0; k < NP; ++k)
        {
            unsigned top[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                const unsigned bits = __float_as_uint(v[h]);
                const bool special = SPECIAL && (bits & 0x7f800000u) == 0x7f800000u;
                top[h] = special && v[h] != v[h] ? 0x7fff0000u : bits;
                if (k + 1 < NP)
                    v[h] = special ? 0.0f : v[h] - __uint_as_float(bits & 0xffff0000u);
            }
            w[k][i] = __byte_perm(top[0], top[1], 0x7632);
        }
    }
}
template <class T>
__device__ __forceinline__ bool any_special(const Raw8<T>& raw)
{
    if constexpr (sizeof(T) == 2)
    {
        const __half2* e = reinterpret_cast<const __half2*>(&raw);
        __half2 zero = __float2half2_rn(0.0f); // stays 0 unless a value is infinite or NaN
#pragma unroll
        for (int i = 0; i < 4; ++i)
            zero = __hfma2(e[i], __float2half2_rn(0.0f), zero);
        return (*reinterpret_cast<const unsigned*>(&zero) & 0x7fff7fffu) != 0u;
    }
    else
    {
        const float* e = reinterpret_cast<const float*>(&raw);
        float zero = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            zero = __fmaf_rn(e[i], 0.0f, zero);
        return zero != 0.0f;
    }
}

// WEIGHT: dw, lanes = i, columns = o, contraction over the tokens; the dense operand is MN-major (o runs fastest).
// otherwise: dx, lanes = i, columns = t, contraction over o; the dense operand is K-major.
// DENSE 0: dy is bf16 and the copy engine can take it.  DENSE 1..3: that many bf16 planes, made by loader warps from TD.
template <bool WEIGHT, int FMT, int DENSE, bool PAIR, class TD, class TO>
__global__ void __launch_bounds__(GradGroups<(DENSE > 0), PAIR>::threads, 1) k_mx_grad(const __grid_constant__ CUtensorMap mapCodes, const __grid_constant__ CUtensorMap mapDy, const GradArgs a)
{
    using G = GradGroups<(DENSE > 0), PAIR>;
    constexpr int NP = DENSE ? DENSE : 1;
    constexpr int CHAIN_STEPS = CHAIN_OF<TO, G::accumulators == 1> / 4 / NP;
    constexpr int WIDEST = G::widest, SLOTS = G::slots, BUFS = G::accumulators;
    extern __shared__ unsigned char dyn[];
    __shared__ GemmBars bars;
    __shared__ __align__(16) unsigned short scaleRows[4 * G::expand][GK]; // per expanding warp: its block's multipliers for one step
    unsigned char* stage0 = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t) 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int bn = a.bn, S = a.stages;
    const int share = PAIR ? bn / 2 : bn; // columns of dy that this CTA brings
    const int denseBytes = share * 128 * NP;
    const int stageBytes = denseBytes + grad_codes_bytes(FMT) + GRAD_SCALE_ROOM;
    const int steps = (int) ((a.C + GK - 1) / GK);
    const int rank = PAIR || a.splits > 1 ? (int) cluster_rank() : 0;
    int first = 0, count = steps;
    if (!PAIR)
        split_range(steps, rank, a.splits, first, count);
    const int firstTile = PAIR ? blockIdx.x >> 1 : blockIdx.x, tileStep = PAIR ? gridDim.x >> 1 : gridDim.x;
    auto tile_m0 = [&](int tile) { return (long long) (tile % a.tilesM) * (PAIR ? 256 : 128) + (PAIR ? rank * 128 : 0); };
    auto tile_n0 = [&](int tile) { return (long long) (tile / a.tilesM) * bn; };

    // what a copied step needs, worked out once per tile
    struct Source
    {
        int codes, n0;
        const unsigned char* scales;
    };
    const long long scaleRow = mx_scale_tiles(a.I) * GRAD_SCALE_BYTES; // from 128 contraction values to the next
    auto source_of = [&](int tile) {
        const int m0 = (int) tile_m0(tile);
        // (a CTA of a pair may have no rows of the packed matrix: codes outside read as zero, scales are taken from the last rows)
        const long long rowTile = m0 < a.I ? m0 / 128 : (a.I - 1) / 128;
        return Source{FMT == QAGG_MXFP4 ? m0 / 2 : m0, (int) tile_n0(tile) + (PAIR ? rank * share : 0), a.scales + rowTile * GRAD_SCALE_BYTES};
    };
    auto copy_step = [&](const Source& src, int i, int s) {
        const unsigned at = smem_addr(stage0) + s * stageBytes;
        const int k0 = (first + i) * GK;
        unsigned long long* full = &bars.full[s];
        mbar_arrive_expect_tx(full, grad_codes_bytes(FMT) + GRAD_SCALE_BYTES + (DENSE ? 0 : denseBytes));
        tma_load_2d(at + denseBytes, &mapCodes, src.codes, k0, full);
        bulk_load(at + denseBytes + grad_codes_bytes(FMT), src.scales + (k0 >> 7) * scaleRow, GRAD_SCALE_BYTES, full);
        if constexpr (DENSE == 0)
        {
            if constexpr (WEIGHT)
                for (int n = 0; n < share; n += 64)
                    tma_load_2d(at + n * 128, &mapDy, src.n0 + n, k0, full);
            else
                tma_load_2d(at, &mapDy, k0, src.n0, full);
        }
    };
    int early = 0; // steps of the first tile whose copies start before the CTA has met
    if (warp == 0)
    {
        init_barriers(&bars, S, G::convArrivals, G::denseArrivals, G::takenArrivals);
        if (elect_one())
        {
            const Source src = source_of(firstTile);
            for (; early < count && early < S; ++early)
                copy_step(src, early, early);
        }
        early = count < S ? count : S;
        __syncwarp();
    }
    // Loaders of the dense operand: rows of 64 contiguous values (128 bytes a plane), in units of eight values.  A thread has two units a
    // step (one of a pair's, which has half of the columns), the second 64 columns (rows of 64 tokens) further: 8192 bytes in the
    // stage, a constant in memory.
    constexpr int THREADS = DENSE ? 128 * G::load : 512, UNITS = PAIR ? 1 : 2;
    static_assert(THREADS * 2 == GRAD_WIDEST_DENSE * 8, "two units a thread");
    struct Units
    {
        Raw8<TD> raw[UNITS];
    };
    const int unit = threadIdx.x - G::firstLoad * 32; // 8 row + piece of the row
    const long long unitStride = WEIGHT ? 64 : 64 * a.ldDy, stepStride = WEIGHT ? GK * a.ldDy : GK;
    const TD* from = nullptr;       // the first unit's next values
    int have0 = 0, have1 = 0;       // WEIGHT: how many of the units' eight columns exist; otherwise eight where their token does
    int left = 0;                   // contraction values from this thread's next one on
    int nextTile = firstTile, nextStep = 0;
    auto fetch = [&](Units& v) { // the next step that this CTA has
        if (nextTile >= a.tiles || count == 0)
            return;
        if (nextStep == 0)
        {
            const int c = (unit & 7) * 8, r = unit >> 3;
            const long long n0 = tile_n0(nextTile) + (PAIR ? rank * share : 0), k0 = (long long) first * GK;
            const long long line = (WEIGHT ? k0 : n0) + r, col = (WEIGHT ? n0 : k0) + c; // token, output
            from = (const TD*) a.dy + line * a.ldDy + col;
            left = (int) (a.C - k0) - (WEIGHT ? r : c);
            if constexpr (WEIGHT)
            {
                const long long cols = a.N - col;
                have0 = (int) (cols < 0 ? 0 : cols < 8 ? cols : 8);
                have1 = share <= 64 || cols <= 64 ? 0 : (int) (cols < 72 ? cols - 64 : 8);
            }
            else
            {
                have0 = line < a.N ? 8 : 0;
                have1 = share > 64 && line + 64 < a.N ? 8 : 0;
            }
        }
        const int most = WEIGHT ? (left > 0 ? 8 : 0) : left < 0 ? 0 : left < 8 ? left : 8;
        v.raw[0] = load8(from, min(have0, most), a.vec);
        if constexpr (UNITS == 2)
            v.raw[UNITS - 1] = load8(from + unitStride, min(have1, most), a.vec);
        from += stepStride;
        left -= GK;
        if (++nextStep == count)
        {
            nextStep = 0;
            nextTile += tileStep;
        }
    };
    Units even = {}, odd = {};
    if (DENSE > 0 && warp >= G::firstLoad)
    {
        fetch(even);
        fetch(odd);
    }
    if (warp == 2)
        tmem_alloc<PAIR>(&bars.tmem, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    if (PAIR)
        cluster_sync(); // the other CTA's barriers exist
    tc_fence_after();
    const unsigned tm = bars.tmem;
    const unsigned tmA = tm + G::side;

    if (warp < 4)
    {
        set_registers<G::regsMisc, G::regsLaunch>();
        if (warp == 0 && elect_one())
        {
            Ring ring;
            for (int i = 0; i < early; ++i)
                ring.next(S);
            long long issued = early;
            for (int tile = firstTile; tile < a.tiles; tile += tileStep)
            {
                const Source src = source_of(tile);
                for (int i = tile == firstTile ? early : 0; i < count; ++i, ++issued)
                {
                    if (issued >= S)
                        tc_wait(&bars.empty[ring.s], ring.par ^ 1, &bars.broken, &g_mxStatus);
                    if (*reinterpret_cast<volatile unsigned*>(&bars.broken))
                    {
                        tile = a.tiles;
                        break;
                    }
                    copy_step(src, i, ring.s);
                    ring.next(S);
                }
            }
            drain_copies(&bars, issued, S);
        }
        else if (warp == 1 && (!PAIR || rank == 0) && elect_one())
        {
            Ring ring;
            Chains chain;
            bool fresh = true; // accumulators that no chain has used
            int slot = 0;
            const unsigned idesc = idesc_bf16(bn, WEIGHT, PAIR ? 256 : 128);
            const unsigned long long d0 = WEIGHT ? smem_desc(smem_addr(stage0), 8192, 1024, SWIZZLE_128B) : smem_desc(smem_addr(stage0), 16, 1024, SWIZZLE_128B);
            constexpr unsigned KSTEP = (WEIGHT ? 2048 : 32) >> 4;
            for (int tile = firstTile; tile < a.tiles; tile += tileStep)
            {
                int inChain = 0;
                for (int i = 0; i < count; ++i)
                {
                    if (inChain == 0 && !fresh)
                        tc_wait(&bars.taken[chain.buf], chain.par ^ 1, &bars.broken, &g_mxStatus);
                    // the expanding warps saw the copies land before they arrived
                    if constexpr (DENSE > 0)
                        tc_wait(&bars.dense[ring.s], ring.par, &bars.broken, &g_mxStatus);
                    tc_wait(&bars.conv[ring.s], ring.par, &bars.broken, &g_mxStatus);
                    tc_fence_after();
                    const unsigned long long d = d0 + ((unsigned) (ring.s * stageBytes) >> 4);
                    const unsigned ta = tmA + slot * 32, acc = tm + chain.buf * WIDEST;
                    slot = (slot + 1) % SLOTS;
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p) // small planes first, onto small sums: see CHAIN
#pragma unroll
                        for (int j = 0; j < GK / 16; ++j)
                            if constexpr (PAIR)
                                mma_bf16_ts_pair(acc, ta + j * 8, d + p * (share * 128 >> 4) + j * KSTEP, idesc, inChain > 0 || p < NP - 1 || j > 0);
                            else
                                mma_bf16_ts(acc, ta + j * 8, d + p * (share * 128 >> 4) + j * KSTEP, idesc, inChain > 0 || p < NP - 1 || j > 0);
                    if constexpr (PAIR)
                        tc_commit_pair(&bars.empty[ring.s]);
                    else
                        tc_commit(&bars.empty[ring.s]);
                    ring.next(S);
                    if (++inChain == CHAIN_STEPS || i + 1 == count)
                    {
                        if constexpr (PAIR)
                            tc_commit_pair(&bars.ready[chain.buf]);
                        else
                            tc_commit(&bars.ready[chain.buf]);
                        chain.next(BUFS);
                        fresh = fresh && chain.buf != 0;
                        inChain = 0;
                    }
                }
            }
        }
    }
    else if (warp < G::firstResult)
    {
        set_registers<G::regsExpand, G::regsLaunch>();
        // Expand: lanes 32 * quad .. of the tile are one block of the packed matrix, so a warp has one scale per contraction value.
        // The codes lie [contraction value][row]; ldmatrix transposes 16 x 16 bytes of them into the order in which a 16 x 256-bit
        // store to tensor memory takes pairs of contraction values.  With fp4 that puts row 16 h + 2 b + o of the block on lane
        // 16 h + 8 o + b; the result warps know.  Several groups of warps take the steps in turn.
        const int quad = warp & 3, group = (warp - G::firstExpand) >> 2;
        const unsigned char* scaleAt = stage0 + denseBytes + grad_codes_bytes(FMT) + lane * 16 + quad; // of contraction value `lane` of a tile
        unsigned short* mult = scaleRows[warp - G::firstExpand];
        // rows of the code tile are 128 (fp4: 64) bytes, their 16-byte pieces swizzled by the copy
        constexpr int ROW = FMT == QAGG_MXFP4 ? 64 : 128;
        unsigned rowAt[2]; // this lane's row address for ldmatrix, for each 16 rows of the block (fp4: one piece holds all 32)
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            const int piece = FMT == QAGG_MXFP4 ? quad : quad * 2 + h;
            rowAt[h] = smem_addr(stage0) + denseBytes + lane * ROW + ((FMT == QAGG_MXFP4 ? piece ^ ((lane >> 1) & 3) : piece ^ (lane & 7)) << 4);
        }
        // Slot n % SLOTS of tensor memory is free when the products of step n - SLOTS are done.  With no more stages than slots the
        // copies of this step had to wait for them already.  With more, their stage has been handed back, and cannot be handed back
        // once more (which would make the parity ambiguous) before this warp has done its part of step n - SLOTS + stages > n.
        int n = 0, stage = 0, oldStage = SLOTS < S ? S - SLOTS : 0, slot = 0; // n: step, over all tiles; oldStage: that of step n - SLOTS
        unsigned par = 0, oldPar = 1;                                      // parities of their rounds
        auto advance = [&](int k) { // k <= G::expand <= S, SLOTS
            n += k;
            slot = (slot + k) % SLOTS;
            if ((stage += k) >= S)
            {
                stage -= S;
                par ^= 1;
            }
            if ((oldStage += k) >= S)
            {
                oldStage -= S;
                oldPar ^= 1;
            }
        };
        for (int tile = firstTile; tile < a.tiles; tile += tileStep)
        {
            int i = 0;
            for (; i < count && n % G::expand != group; ++i) // steps of the other groups
                advance(1);
            for (; i < count; i += G::expand)
            {
                tc_wait(&bars.full[stage], par, &bars.broken, &g_mxStatus);
                __syncwarp(); // also: the multipliers of the previous step have been read
                const unsigned off = stage * stageBytes;
                // piece g of a block half is 16 contraction values: two registers
                constexpr int HALVES = FMT == QAGG_MXINT8 ? 2 : 1;
                unsigned c[HALVES][8];
#pragma unroll
                for (int h = 0; h < HALVES; ++h)
                {
                    ldmatrix_trans_b8(rowAt[h] + off, reinterpret_cast<unsigned(&)[4]>(c[h][0]));
                    ldmatrix_trans_b8(rowAt[h] + off + 32 * ROW, reinterpret_cast<unsigned(&)[4]>(c[h][4]));
                }
                const unsigned char* sb = scaleAt + off + ((first + i) & 1) * 8;
                const unsigned b0 = sb[0], b1 = sb[4];
                const bool large = FMT == QAGG_MXFP4 && __any_sync(0xffffffffu, b0 > FP4_LARGE || b1 > FP4_LARGE);
                mult[lane] = (unsigned short) scale_bf16<FMT>(b0, large);
                mult[lane + 32] = (unsigned short) scale_bf16<FMT>(b1, large);
                __syncwarp();
                uint2 sc[4]; // multipliers of contraction values 16 g + 4 (lane % 4) .. + 3
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    sc[g] = *reinterpret_cast<const uint2*>(mult + 16 * g + 4 * (lane & 3));
                if (S > SLOTS && n >= SLOTS)
                {
                    tc_wait(&bars.empty[oldStage], oldPar, &bars.broken, &g_mxStatus);
                    __syncwarp();
                }
                tc_fence_after();
                const unsigned to = tmA + ((unsigned) (quad * 32) << 16) + slot * 32;
                const auto expand = [&](auto large_) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                    {
                        unsigned r[16];
#pragma unroll
                        for (int g = 0; g < 4; ++g)
#pragma unroll
                            for (int e = 0; e < 2; ++e) // rows l / 4, l / 4 + 8 of the half
                            {
                                const unsigned v = FMT == QAGG_MXINT8 ? c[h % HALVES][2 * g + e] : c[0][2 * g + h];
                                constexpr bool LARGE = decltype(large_)::value;
                                r[4 * g + 2 * e] = FMT == QAGG_MXINT8 ? expand_int8(v, 0, sc[g].x) : expand_fp4(v, 0, e, LARGE, sc[g].x);
                                r[4 * g + 2 * e + 1] = FMT == QAGG_MXINT8 ? expand_int8(v, 1, sc[g].y) : expand_fp4(v, 1, e, LARGE, sc[g].y);
                            }
                        tmem_store_16x256b(to + ((unsigned) (h * 16) << 16), r);
                    }
                };
                if (FMT == QAGG_MXFP4 && large)
                    expand(std::true_type());
                else
                    expand(std::false_type());
                tmem_store_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                {
                    if constexpr (PAIR)
                        mbar_arrive_remote(&bars.conv[stage], 0);
                    else
                        mbar_arrive(&bars.conv[stage]);
                }
                advance(min(G::expand, count - i));
            }
        }
    }
    else if (warp < G::firstLoad)
    {
        set_registers<G::regsResult, G::regsLaunch>();
        const int rw = warp - G::firstResult, quad = rw & 3, half = rw >> 2;
        {
            const int cols = bn / G::result;
            const unsigned mine = tm + ((unsigned) (quad * 32) << 16) + half * cols;
            const int m = quad * 32 + (FMT == QAGG_MXFP4 ? (lane & 16) + 2 * (lane & 7) + ((lane >> 3) & 1) : lane);
            Chains chain;
            for (int tile = firstTile; tile < a.tiles; tile += tileStep)
            {
                const long long m0 = tile_m0(tile), n0 = tile_n0(tile);
                float* buf = reinterpret_cast<float*>(stage0);
                const int partner = lane ^ (FMT == QAGG_MXFP4 ? 8 : 1);
                if (!PAIR && a.tiles <= tileStep && count <= CHAIN_STEPS)
                {
                    drain_chain(&bars, mine, cols, count == 0, [&](int j, const float(&v)[16]) {
                        if (a.splits > 1)
                            put_partial<WEIGHT>(buf, bn, m, half * cols + j, 16, v);
                        else if constexpr (WEIGHT)
                            write_row((float*) a.out, a.ld, m0 + m, a.I, n0 + half * cols + j, a.N, 16, v, a.add != 0, a.wide != 0);
                        else
                            write_columns((TO*) a.out, a.ld, m0 + m, a.I, n0 + half * cols + j, a.N, 16, v, 0.0f, partner, a.wide && m0 + 128 <= a.I);
                    });
                    break;
                }
                constexpr int ACC = WIDEST / G::result;
                float acc[ACC];
#pragma unroll
                for (int j = 0; j < ACC; ++j)
                    acc[j] = 0.0f;
                for (int i = 0; i < count; i += CHAIN_STEPS, chain.next(BUFS))
                    take_chain<PAIR>(&bars, chain.buf, chain.par, mine + chain.buf * WIDEST, cols, i == 0, acc);
                if (!PAIR && a.splits > 1)
                    put_partial<WEIGHT>(buf, bn, m, half * cols, cols, acc);
                else if constexpr (WEIGHT)
                    write_row((float*) a.out, a.ld, m0 + m, a.I, n0 + half * cols, a.N, cols, acc, a.add != 0, a.wide != 0);
                else
                    write_columns((TO*) a.out, a.ld, m0 + m, a.I, n0 + half * cols, a.N, cols, acc, 0.0f, partner, a.wide && m0 + 128 <= a.I);
            }
        }
    }
    else if constexpr (DENSE > 0)
    {
        // Two steps' values are on their way (behind the fence, which would wait for them) while an earlier one is split and stored.
        set_registers<G::regsLoad, G::regsLaunch>();
        unsigned char* mine = stage0 + (unit >> 3) * 128 + (((unit & 7) ^ (unit >> 3 & 7)) << 4);
        Ring ring;
        long long done = 0;
        auto put_step = [&](const Units& v) {
            if (done >= S)
                tc_wait(&bars.empty[ring.s], ring.par ^ 1, &bars.broken, &g_mxStatus);
            ++done;
            unsigned char* at = mine + ring.s * stageBytes;
#pragma unroll
            for (int q = 0; q < UNITS; ++q)
            {
                unsigned w[NP][4];
                if (NP == 1)
                    *reinterpret_cast<uint4*>(w[0]) = v.raw[q].a;
                else if (any_special(v.raw[q]))
                    split8<TD, NP, true>(v.raw[q], w);
                else
                    split8<TD, NP, false>(v.raw[q], w);
                if (q == 0 || share > 64)
#pragma unroll
                    for (int p = 0; p < NP; ++p)
                        *reinterpret_cast<uint4*>(at + q * 8192 + p * share * 128) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0)
            {
                if constexpr (PAIR)
                    mbar_arrive_remote(&bars.dense[ring.s], 0);
                else
                    mbar_arrive(&bars.dense[ring.s]);
            }
            ring.next(S);
        };
        const long long mySteps = firstTile < a.tiles ? (long long) ((a.tiles - 1 - firstTile) / tileStep + 1) * count : 0;
        for (long long n = 0; n < mySteps; n += 2)
        {
            put_step(even);
            fetch(even);
            if (n + 1 < mySteps)
            {
                put_step(odd);
                fetch(odd);
            }
        }
    }
    __syncwarp();
    if (!PAIR && a.splits > 1) // one tile per cluster
        reduce_cluster<WEIGHT, TO>(reinterpret_cast<float*>(stage0), a.splits, rank, bn, (TO*) a.out, a.ld, tile_m0(blockIdx.x), a.I, tile_n0(blockIdx.x), a.N, nullptr,
                                   a.add != 0, a.wide4);
    tc_fence_before();
    if (PAIR)
        cluster_sync(); // neither goes while the other may still arrive at its barriers or use its memory
    __syncthreads();
    if (warp == 2)
        tmem_free<PAIR>(tm, TMEM_COLS);
}

// ---- launches -----------------------------------------------------------------------------------------------------------------

// Tile width and split of the contraction, by a count of cycles: a CTA runs waves * steps / splits steps, each as long as its products
// (2 * bn * planes: 8192 bf16 or 32768 fp4 multiply-adds a cycle), its copies (46 bytes a cycle from L2) or its preparation
// (`least`: expanding a step takes the warps 450 cycles, splitting a dense one 1300) take, whichever is most; then the last tile's
// result goes out.
struct Shape
{
    int bn, splits;
};
static Shape choose_shape(long long tilesM, long long N, int steps, int sms, const int* widths, int nWidths, int planes, int fixedBytes, int columnBytes, double least)
{
    Shape best = {widths[0], 1};
    double bestCost = 1e300;
    for (int i = 0; i < nWidths; ++i)
    {
        const int bn = widths[i];
        if (i > 0 && bn < 128 && N > bn)
            break; // several narrow tiles would read the other operand once each
        const long long tiles = tilesM * ((N + bn - 1) / bn);
        const double step = 50.0 + std::max(std::max(2.0 * bn * planes, (fixedBytes + (double) bn * columnBytes) / 46.0), least);
        for (int s = 1; s <= 8; s *= 2)
        {
            if (s > 1 && s > steps)
                break;
            const long long waves = (tiles * s + sms - 1) / sms;
            // split: every wave starts anew and ends with an exchange, and clusters of eight are slow to be placed (a 2048 x 2048
            // product with one token: 10.3 us in eights, 5.9 in fours); otherwise tiles follow one another without a gap
            const double cost = step * waves * ((steps + s - 1) / s) + (s > 1 ? waves * (5000.0 + 4.0 * bn) : 3000.0 + 4.0 * bn) + (s == 8 ? 9000.0 : 0.0);
            if (cost < bestCost)
            {
                bestCost = cost;
                best = {bn, s};
            }
        }
    }
    return best;
}

static int stages_for(int stageBytes, int most)
{
    return std::max(2, std::min(most, (GEMM_SMEM_MAX - 1024) / stageBytes));
}
static int smem_for(int stageBytes, int stages, int resultBytes)
{
    return std::max(GEMM_SMEM_MIN, 1024 + std::max(stageBytes * stages, resultBytes));
}

// The kernels' limit of dynamic shared memory is raised once per device.
template <auto KERNEL, class... Args>
static cudaError_t launch_cluster(dim3 grid, int threads, int smem, dim3 cluster, cudaStream_t st, Args... args)
{
    static std::atomic<unsigned long long> raised{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess)
        return e;
    if (!(raised.load(std::memory_order_relaxed) >> dev & 1)) // devices 0..63: launch_cfg_for_current_device has seen to it
    {
        e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, GEMM_SMEM_MAX);
        if (e != cudaSuccess)
            return e;
        raised.fetch_or(1ull << dev);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster.x;
    attr[0].val.clusterDim.y = cluster.y;
    attr[0].val.clusterDim.z = cluster.z;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, KERNEL, args...);
    return e != cudaSuccess ? e : cudaGetLastError();
}

// boxes of boxBytes x boxCols codes, the 16-byte pieces of a row swizzled within it
static bool codes_map(CUtensorMap* m, const void* codes, long long M, long long N, int format, int boxBytes, int boxCols)
{
    return encode_map_tiled(m, 1, codes, mx_pitch(M, format), N, mx_pitch(M, format), boxBytes, boxCols, boxBytes);
}

template <bool WEIGHT, int FMT, int DENSE, class TD, class TO>
static cudaError_t launch_grad(cudaStream_t st, const CUtensorMap& mc, const CUtensorMap& md, GradArgs a, int sms)
{
    constexpr int NP = DENSE ? DENSE : 1;
    if constexpr (WEIGHT || DENSE == 0 || std::is_same_v<TD, TO> || std::is_same_v<TO, float>)
        if (a.pair)
        {
            const int stageBytes = a.bn / 2 * 128 * NP + grad_codes_bytes(FMT) + GRAD_SCALE_ROOM;
            a.stages = stages_for(stageBytes, MAX_STAGES);
            const int smem = smem_for(stageBytes, a.stages, 0);
            return launch_cluster<k_mx_grad<WEIGHT, FMT, DENSE, true, TD, TO>>(dim3((unsigned) (2 * std::min(a.tiles, sms / 2))), GradGroups<(DENSE > 0), true>::threads, smem,
                                                                              dim3(2, 1, 1), st, mc, md, a);
        }
    const int stageBytes = a.bn * 128 * NP + grad_codes_bytes(FMT) + GRAD_SCALE_ROOM;
    a.stages = stages_for(stageBytes, MAX_STAGES);
    const int smem = smem_for(stageBytes, a.stages, a.splits > 1 ? 128 * (a.bn + 4) * 4 : 0);
    const dim3 grid((unsigned) (a.splits > 1 ? a.tiles : std::min(a.tiles, sms)), 1, (unsigned) a.splits);
    return launch_cluster<k_mx_grad<WEIGHT, FMT, DENSE, false, TD, TO>>(grid, GradGroups<(DENSE > 0), false>::threads, smem, dim3(1, 1, a.splits), st, mc, md, a);
}

template <bool WEIGHT, int FMT, class TO>
static cudaError_t launch_grad_dense(cudaStream_t st, const CUtensorMap& mc, const CUtensorMap& md, const GradArgs& a, int dyType, bool tma, int sms)
{
    if (dyType == QAGG_BF16)
        return tma ? launch_grad<WEIGHT, FMT, 0, __nv_bfloat16, TO>(st, mc, md, a, sms) : launch_grad<WEIGHT, FMT, 1, __nv_bfloat16, TO>(st, mc, md, a, sms);
    if (dyType == QAGG_F16)
        return launch_grad<WEIGHT, FMT, 2, __half, TO>(st, mc, md, a, sms);
    return launch_grad<WEIGHT, FMT, 3, float, TO>(st, mc, md, a, sms);
}

// Two CTAs on a 256 x 256 (with loaders 256 x 128) tile, or one on 128 x bn: cycles as in choose_shape, with what a pair waits for its
// one accumulator.  Loaders and splitting warps take a CTA by itself 2000 cycles a step of 128 columns, each of a pair 1200.
static bool pair_pays(long long I, long long N, const GradArgs& a, int sms, int format, bool tma)
{
    const int codes = grad_codes_bytes(format), width = tma ? GRAD_PAIR : GRAD_WIDEST_DENSE;
    const double one = (tma ? std::max(2.0 * a.bn, (codes + a.bn * 128.0) / 46.0) : 2000.0) * ((a.tiles + sms - 1) / sms);
    const long long pairs = (I + 255) / 256 * ((N + width - 1) / width);
    const double two = (tma ? std::max(512.0, (codes + 16384.0) / 46.0) * 1.25 : 1200.0) * ((pairs + sms / 2 - 1) / (sms / 2));
    return two < one;
}

// What both gradients check and set up.  tokens x outputs is dy; `contraction` of the two is summed over.
static int grad_common(const char* who, bool weight, void* stream, const void* dy, int dyType, int64_t ldDy, const void* codes, const void* scales, int format, void* out,
                       int outType, int64_t ldOut, int64_t O, int64_t I, int64_t T, int add)
{
    const int64_t C = weight ? T : O, N = weight ? O : T;
    int rc = mx_check_dims(who, I, C);
    if (!rc)
        rc = mx_check_dims(who, O, T);
    if (rc)
        return rc;
    if (!mx_type_ok(dyType) || !mx_type_ok(outType) || (format != QAGG_MXFP4 && format != QAGG_MXINT8))
        return fail(QAGG_EINVAL, std::string(who) + ": unknown element type or format");
    if (ldDy < O || ldOut < (weight ? O : I))
        return fail(QAGG_EINVAL, std::string(who) + ": ld is less than the number of rows");
    if (N > 65535LL * 64)
        return fail(QAGG_EINVAL, std::string(who) + ": matrix dimension too large");
    if (I == 0 || N == 0 || (C == 0 && add))
        return QAGG_OK;
    if (!out || (C > 0 && (!dy || !codes || !scales)))
        return fail(QAGG_EINVAL, std::string(who) + ": null pointer");
    if (((uintptr_t) out & (mx_type_bytes(outType) - 1)) || ((uintptr_t) dy & (mx_type_bytes(dyType) - 1)) || (((uintptr_t) codes | (uintptr_t) scales) & 15))
        return fail(QAGG_EINVAL, std::string(who) + ": codes and scales must be 16-byte aligned, the others aligned to their type");
    LaunchCfg cfg;
    rc = launch_cfg_for_current_device(&cfg);
    if (rc)
        return rc;
    GradArgs a = {};
    a.scales = (const unsigned char*) scales;
    a.dy = dy;
    a.ldDy = ldDy;
    a.out = out;
    a.ld = ldOut;
    a.I = I;
    a.C = C;
    a.N = N;
    a.add = add != 0;
    a.vec = (((uintptr_t) dy | (uintptr_t) (ldDy * mx_type_bytes(dyType))) & 15) == 0;
    const bool tma = dyType == QAGG_BF16 && a.vec;
    static const int wide[] = {GRAD_WIDEST, GRAD_WIDEST_DENSE, 64};
    const Shape sh = choose_shape((I + 127) / 128, N, (int) ((C + GK - 1) / GK), cfg.numSMs, tma ? wide : wide + 1, tma ? 3 : 2, dyType == QAGG_BF16 ? 1 : dyType == QAGG_F16 ? 2 : 3,
                                  grad_codes_bytes(format), GK * mx_type_bytes(dyType), tma ? 450.0 : 1300.0);
    a.bn = sh.bn;
    a.splits = sh.splits;
    a.tilesM = (int) ((I + 127) / 128);
    a.tiles = a.tilesM * (int) ((N + a.bn - 1) / a.bn);
    // with loaders a pair's kernel exists for outputs of dy's type and fp32 (and is not worth one more for the others)
    if (a.splits == 1 && (tma || weight || outType == dyType || outType == QAGG_F32) && pair_pays(I, N, a, cfg.numSMs, format, tma))
    {
        a.pair = 1;
        a.bn = tma ? GRAD_PAIR : GRAD_WIDEST_DENSE;
        a.tilesM = (int) ((I + 255) / 256);
        a.tiles = a.tilesM * (int) ((N + a.bn - 1) / a.bn);
    }
    a.wide = weight ? ((((uintptr_t) out | (uintptr_t) (ldOut * 4)) & 15) == 0) : ((uintptr_t) out & 3) == 0 && (ldOut & 1) == 0;
    a.wide4 = (((uintptr_t) out | (uintptr_t) (ldOut * mx_type_bytes(outType))) & (4 * mx_type_bytes(outType) - 1)) == 0;
    alignas(64) CUtensorMap mc, md;
    std::memset(&mc, 0, sizeof(mc));
    std::memset(&md, 0, sizeof(md));
    if (C > 0 && !codes_map(&mc, codes, I, C, format, format == QAGG_MXFP4 ? 64 : 128, GK))
        return fail(QAGG_ECUDA, std::string(who) + ": tensor map of the codes could not be made");
    if (C > 0 && tma && !encode_map_tiled(&md, 2, dy, O, T, ldDy * 2, 64, weight ? GK : a.pair ? a.bn / 2 : a.bn, 128))
        return fail(QAGG_ECUDA, std::string(who) + ": tensor map of dy could not be made");
    const cudaStream_t st = (cudaStream_t) stream;
    cudaError_t e;
    if (weight)
        e = format == QAGG_MXFP4 ? launch_grad_dense<true, QAGG_MXFP4, float>(st, mc, md, a, dyType, tma, cfg.numSMs)
                                 : launch_grad_dense<true, QAGG_MXINT8, float>(st, mc, md, a, dyType, tma, cfg.numSMs);
    else if (outType == QAGG_F32)
        e = format == QAGG_MXFP4 ? launch_grad_dense<false, QAGG_MXFP4, float>(st, mc, md, a, dyType, tma, cfg.numSMs)
                                 : launch_grad_dense<false, QAGG_MXINT8, float>(st, mc, md, a, dyType, tma, cfg.numSMs);
    else if (outType == QAGG_F16)
        e = format == QAGG_MXFP4 ? launch_grad_dense<false, QAGG_MXFP4, __half>(st, mc, md, a, dyType, tma, cfg.numSMs)
                                 : launch_grad_dense<false, QAGG_MXINT8, __half>(st, mc, md, a, dyType, tma, cfg.numSMs);
    else
        e = format == QAGG_MXFP4 ? launch_grad_dense<false, QAGG_MXFP4, __nv_bfloat16>(st, mc, md, a, dyType, tma, cfg.numSMs)
                                 : launch_grad_dense<false, QAGG_MXINT8, __nv_bfloat16>(st, mc, md, a, dyType, tma, cfg.numSMs);
    return check_cuda(e, "gradient product kernel launch");
}

} // namespace qagg

using namespace qagg;

extern "C" {

int qagg_mx_times(void* stream, const void* w_codes, const void* w_scales, const void* x_codes, const void* x_scales, const float* bias, void* y, int y_type, int64_t ld_y,
                  int64_t O, int64_t T, int64_t K)
{
    int rc = mx_check_dims("qagg_mx_times", K, O);
    if (!rc)
        rc = mx_check_dims("qagg_mx_times", K, T);
    if (!rc)
        rc = mx_check_dims("qagg_mx_times", O, T);
    if (rc)
        return rc;
    if (!mx_type_ok(y_type))
        return fail(QAGG_EINVAL, "qagg_mx_times: unknown element type");
    if (ld_y < O)
        return fail(QAGG_EINVAL, "qagg_mx_times: ld is less than the number of rows");
    if (O == 0 || T == 0)
        return QAGG_OK;
    if (!y || (K > 0 && (!w_codes || !w_scales || !x_codes || !x_scales)))
        return fail(QAGG_EINVAL, "qagg_mx_times: null pointer");
    if (((uintptr_t) y & (mx_type_bytes(y_type) - 1)) || ((uintptr_t) bias & 3) ||
        (((uintptr_t) w_codes | (uintptr_t) w_scales | (uintptr_t) x_codes | (uintptr_t) x_scales) & 15))
        return fail(QAGG_EINVAL, "qagg_mx_times: codes and scales must be 16-byte aligned, the others aligned to their type");
    LaunchCfg cfg;
    rc = launch_cfg_for_current_device(&cfg);
    if (rc)
        return rc;
    if (times_few(O, T, K))
    {
        const auto few = [&](auto* p) { return launch_times_few((cudaStream_t) stream, w_codes, w_scales, x_codes, x_scales, bias, p, ld_y, O, (int) T, K, cfg.numSMs); };
        return check_cuda(y_type == QAGG_F32 ? few((float*) y) : y_type == QAGG_F16 ? few((__half*) y) : few((__nv_bfloat16*) y), "4-bit product kernel launch");
    }
    TimesArgs a = {};
    a.scaleW = (const unsigned char*) w_scales;
    a.scaleX = (const unsigned char*) x_scales;
    a.bias = bias;
    a.y = y;
    a.ld = ld_y;
    a.O = O;
    a.T = T;
    a.K = K;
    static const int widths[] = {256, 128, 64, 32, 16};
    const Shape sh = choose_shape((O + 127) / 128, T, (int) ((K + TK - 1) / TK), cfg.numSMs, widths, 5, 1, 128 * (128 + 8), 128 + 8, 0.0);
    a.bn = sh.bn;
    a.splits = sh.splits;
    a.tilesM = (int) ((O + 127) / 128);
    a.tiles = a.tilesM * (int) ((T + a.bn - 1) / a.bn);
    a.pairs = ((uintptr_t) y & 3) == 0 && (ld_y & 1) == 0;
    a.wide4 = (((uintptr_t) y | (uintptr_t) (ld_y * mx_type_bytes(y_type))) & (4 * mx_type_bytes(y_type) - 1)) == 0;
    // two CTAs on a 256 x 256 tile, or one on 128 x bn: cycles as in choose_shape
    const long long pairs = (O + 255) / 256 * ((T + 255) / 256);
    const bool pair = a.splits == 1 && 1.05 * 780.0 * ((pairs + cfg.numSMs / 2 - 1) / (cfg.numSMs / 2)) <
                                           std::max(2.0 * a.bn, (128 + a.bn) * 136.0 / 46.0) * ((a.tiles + cfg.numSMs - 1) / cfg.numSMs);
    if (pair)
    {
        a.bn = TIMES_PAIR;
        a.tilesM = (int) ((O + 255) / 256);
        a.tiles = (int) pairs;
    }
    const int stageBytes = times_stage_bytes(a.bn, pair ? a.bn / 2 : a.bn);
    a.stages = stages_for(stageBytes, MAX_STAGES);
    const int smem = smem_for(stageBytes, a.stages, a.splits > 1 ? 128 * a.bn * 4 : 0);
    alignas(64) CUtensorMap mw, mx;
    std::memset(&mw, 0, sizeof(mw));
    std::memset(&mx, 0, sizeof(mx));
    if (K > 0 && (!codes_map(&mw, w_codes, K, O, QAGG_MXFP4, 128, 128) || !codes_map(&mx, x_codes, K, T, QAGG_MXFP4, 128, pair ? a.bn / 2 : a.bn)))
        return fail(QAGG_ECUDA, "qagg_mx_times: tensor maps of the codes could not be made");
    const dim3 grid((unsigned) (pair ? 2 * std::min(a.tiles, cfg.numSMs / 2) : a.splits > 1 ? a.tiles : std::min(a.tiles, cfg.numSMs)), 1, (unsigned) a.splits);
    const dim3 cluster(pair ? 2 : 1, 1, a.splits);
    const cudaStream_t st = (cudaStream_t) stream;
    const auto launch = [&](auto* t) {
        using T_ = std::remove_pointer_t<decltype(t)>;
        if (pair)
            return launch_cluster<k_mx_times<T_, 128, true>>(grid, TT, smem, cluster, st, mw, mx, a);
        if (a.bn <= TIMES_NARROW)
            return launch_cluster<k_mx_times<T_, TIMES_NARROW, false>>(grid, TT, smem, cluster, st, mw, mx, a);
        return launch_cluster<k_mx_times<T_, 128, false>>(grid, TT, smem, cluster, st, mw, mx, a);
    };
    const cudaError_t e = y_type == QAGG_F32 ? launch((float*) nullptr) : y_type == QAGG_F16 ? launch((__half*) nullptr) : launch((__nv_bfloat16*) nullptr);
    return check_cuda(e, "4-bit product kernel launch");
}

int qagg_mx_weight_grad(void* stream, const void* dy, int dy_type, int64_t ld_dy, const void* x_codes, const void* x_scales, int format, float* dw, int64_t O, int64_t I,
                        int64_t T, int add)
{
    return grad_common("qagg_mx_weight_grad", true, stream, dy, dy_type, ld_dy, x_codes, x_scales, format, dw, QAGG_F32, O, O, I, T, add);
}

int qagg_mx_input_grad(void* stream, const void* dy, int dy_type, int64_t ld_dy, const void* w_codes, const void* w_scales, int format, void* dx, int dx_type, int64_t ld_dx,
                       int64_t O, int64_t I, int64_t T)
{
    return grad_common("qagg_mx_input_grad", false, stream, dy, dy_type, ld_dy, w_codes, w_scales, format, dx, dx_type, ld_dx, O, I, T, 0);
}

int qagg_mx_check(void* stream)
{
    const cudaStream_t st = (cudaStream_t) stream;
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    int rc = check_cuda(cudaStreamIsCapturing(st, &capture), "qagg_mx_check");
    if (rc)
        return rc;
    if (capture != cudaStreamCaptureStatusNone)
        return fail(QAGG_ESTATE, "qagg_mx_check: the stream is being captured");
    // another stream's capture, on this thread or another, is not to be disturbed by the calls below, which do not concern it
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    rc = check_cuda(cudaThreadExchangeStreamCaptureMode(&mode), "qagg_mx_check");
    if (rc)
        return rc;
    unsigned status = 0;
    rc = check_cuda(cudaStreamSynchronize(st), "qagg_mx_check");
    if (!rc)
    {
        static std::mutex one; // g_mxTaken is one word per device
        const std::lock_guard<std::mutex> guard(one);
        k_mx_take_status<<<1, 1, 0, st>>>();
        cudaError_t e = cudaGetLastError();
        if (e == cudaSuccess)
            e = cudaMemcpyFromSymbolAsync(&status, g_mxTaken, sizeof(status), 0, cudaMemcpyDeviceToHost, st);
        if (e == cudaSuccess)
            e = cudaStreamSynchronize(st);
        rc = check_cuda(e, "qagg_mx_check");
    }
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (rc || !status)
        return rc;
    return fail(QAGG_ETIMEOUT, "qagg_mx_check: a bounded wait inside a product kernel ran out on this device; results since the last check may be invalid");
}

int qagg_mx_wait_selftest(void* stream, int64_t limit_ns)
{
    if (limit_ns < 1 || limit_ns > 1000000000)
        return fail(QAGG_EINVAL, "qagg_mx_wait_selftest: the limit must be 1 .. 10^9 ns");
    k_mx_wait_selftest<<<1, 32, 0, (cudaStream_t) stream>>>((unsigned long long) limit_ns);
    return check_cuda(cudaGetLastError(), "product wait self-test launch");
}

} // extern "C"
