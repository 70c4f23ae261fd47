// qagg_mx_gemm.cu -- products of microscaled matrices on the tensor cores (form: qagg_mx.cuh, instructions: qagg_tcgen05.cuh).
//
//   k_mx_times  y(o, t)  = sum_k w(k, o) x(k, t) + bias(o), both packed in fp4: the tensor cores take codes and block scales as
//               they are.
//   k_mx_grad   dw(o, i) = sum_t dy(o, t) x(i, t)   and   dx(i, t) = sum_o w(i, o) dy(o, t), x or w packed (fp4 or int8) and dy
//               dense.  The packed operand's blocks run across the contraction, so its scales cannot go with a block-scaled
//               product; it is expanded to bf16 (exact) on the way, straight into tensor memory, as operand A.
//
// Both: one CTA per 128 x n output tile; a copy warp feeds a ring of shared-memory stages, one thread issues the products, eight
// warps take the result from tensor memory.  Where there are fewer tiles than SMs the contraction is split over the CTAs of a cluster,
// whose partial sums are added through distributed shared memory in rank order: no workspace, no atomics, the same bits on every run.
#include "qagg_mx.cuh"
#include "qagg_tcgen05.cuh"

#include <algorithm>
#include <cstring>
#include <string>

namespace qagg {

// set by a bounded wait that ran out; read and cleared by qagg_mx_check
__device__ unsigned g_mxStatus;

constexpr int GT = 384;            // threads: copy warp, product warp, allocating warp, spare, eight result warps
constexpr int GT_DENSE = 640;      // and eight warps that bring a dense operand which the copy engine cannot take
constexpr unsigned TMEM_COLS = 512;
constexpr int MAX_STAGES = 8;
constexpr int GEMM_SMEM_MAX = 224 * 1024; // dynamic; barriers and scale pairs take a little more
// More than half of an SM's shared memory, always: a second CTA on the SM would wait for tensor memory (all columns are taken),
// and CTAs of two clusters that each wait for the other's tensor memory would never meet at their cluster barriers.
constexpr int GEMM_SMEM_MIN = 118 * 1024;

struct GemmBars
{
    unsigned long long full[MAX_STAGES];  // copies of the stage have landed
    unsigned long long conv[MAX_STAGES];  // grad: packed operand expanded into tensor memory
    unsigned long long dense[MAX_STAGES]; // grad, dense loaders: their part of the stage is written
    unsigned long long empty[MAX_STAGES]; // products that read the stage are done
    unsigned long long done;              // all products are done
    unsigned tmem;
    unsigned broken;
};

__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// First and last-but-one step of this CTA's part of the contraction.
__device__ __forceinline__ void split_range(int steps, int rank, int splits, int& first, int& count)
{
    first = (int) ((long long) steps * rank / splits);
    count = (int) ((long long) steps * (rank + 1) / splits) - first;
}

// ---- results ------------------------------------------------------------------------------------------------------------------
// The tile D (128 lanes m x bn columns n) goes out as
//   columns  out[(n0 + n) * ld + m0 + m], any type: 32 lanes are 32 neighbours, so straight from the registers
//   rows     out[(m0 + m) * ld + n0 + n], fp32: through shared memory, whose rows are then written 16 values a thread apart
// Eight warps (`warp` 0..7 of them): lanes 32 * (warp % 4), 32-column pieces alternating between warp / 4 = 0, 1.
template <bool ROWS, class T>
__device__ __forceinline__ void write_tile(unsigned tmemD, bool zero, int bn, int warp, float* buf, int splits, int rank, T* out, long long ld, long long m0,
                                           long long M, long long n0, long long N, const float* bias, bool add)
{
    const int lane = threadIdx.x & 31, quad = warp & 3;
    const int m = quad * 32 + lane;
    const int pitch = ROWS ? bn + 4 : 128; // ROWS: [m][n], else [n][m]
    const bool viaShared = ROWS || splits > 1;
    if (warp >= 0)
    {
        const float b = bias && m0 + m < M && splits == 1 ? bias[m0 + m] : 0.0f;
        for (int c = (warp >> 2) * 32; c < bn; c += 64)
        {
            unsigned r[32];
            if (zero)
            {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    r[j] = 0;
            }
            else
                tmem_load32(tmemD + ((unsigned) (quad * 32) << 16) + c, r);
            if (viaShared)
            {
                if (ROWS)
                {
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        *reinterpret_cast<uint4*>(buf + m * pitch + c + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
                }
                else
                {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (c + j < bn)
                            buf[(c + j) * pitch + m] = __uint_as_float(r[j]);
                }
            }
            else if (m0 + m < M)
            {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (c + j < bn && n0 + c + j < N)
                        put(out + (n0 + c + j) * ld + m0 + m, __uint_as_float(r[j]) + b);
            }
        }
    }
    if (!viaShared)
        return;
    __syncwarp();
    if (splits > 1)
        cluster_sync();
    else
        __syncthreads();
    // this CTA's share of the tile: rows (ROWS) or columns, four values a time
    const int lines = ROWS ? 128 : bn, width = ROWS ? bn : 128;
    const int l0 = lines * rank / splits, l1 = lines * (rank + 1) / splits;
    const unsigned base = smem_addr(buf);
    if (warp >= 0)
    {
        const int perLine = width / 4;
        for (int u = l0 * perLine + warp * 32 + lane; u < l1 * perLine; u += 256)
        {
            const int l = u / perLine, w = (u - l * perLine) * 4;
            const unsigned at = base + (unsigned) (l * pitch + w) * 4;
            float4 s = *reinterpret_cast<const float4*>(buf + l * pitch + w);
            if (splits > 1)
            {
                s = cluster_load4(at, 0);
                for (int k = 1; k < splits; ++k)
                {
                    const float4 v = cluster_load4(at, k);
                    s.x += v.x;
                    s.y += v.y;
                    s.z += v.z;
                    s.w += v.w;
                }
            }
            const float e[4] = {s.x, s.y, s.z, s.w};
            const long long line = (ROWS ? m0 : n0) + l, col = (ROWS ? n0 : m0) + w;
            const long long nl = ROWS ? M : N, nc = ROWS ? N : M;
            if (line >= nl)
                continue;
            T* p = out + line * ld + col;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < nc)
                {
                    if constexpr (ROWS)
                        p[j] = add ? p[j] + e[j] : e[j];
                    else
                        put(p + j, e[j] + (bias ? bias[col + j] : 0.0f));
                }
        }
    }
    __syncwarp();
    if (splits > 1)
        cluster_sync(); // nobody leaves while its partial sums are being read
}

// After a wait ran out: the copies this thread started have landed (or a bounded wait for them ran out too) before the CTA goes.
__device__ __forceinline__ void drain_copies(GemmBars* bars, int issued, int stages)
{
    const unsigned long long began = clock_ns();
    for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
        while (!mbar_suspend_wait(&bars->full[i % stages], (i / stages) & 1) && clock_ns() - began < TC_WAIT_NS)
            ;
}

__device__ __forceinline__ void gemm_setup(GemmBars* bars, int stages, int convCount, int denseCount)
{
    if (threadIdx.x == 0)
    {
        for (int s = 0; s < stages; ++s)
        {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->conv[s], convCount);
            mbar_init(&bars->dense[s], denseCount);
            mbar_init(&bars->empty[s], 1);
        }
        mbar_init(&bars->done, 1);
        bars->broken = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_shared();
    }
    if (threadIdx.x >> 5 == 2)
        tmem_alloc(&bars->tmem, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
}

// ---- 4-bit product --------------------------------------------------------------------------------------------------------------

struct TimesArgs
{
    const unsigned char* scaleW;
    const unsigned char* scaleX;
    const float* bias;
    void* y;
    long long ld, O, T, K;
    int bn, stages, splits;
};

constexpr int TK = 256; // contraction values per stage: 128 bytes of codes

__host__ __device__ inline int times_stage_bytes(int bn)
{
    return 128 * 128 + bn * 128 + 1024 + (bn > 128 ? 2048 : 1024);
}

template <class T>
__global__ void __launch_bounds__(GT, 1) k_mx_times(const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapX, const TimesArgs a)
{
    extern __shared__ unsigned char dyn[];
    __shared__ GemmBars bars;
    unsigned char* stage0 = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t) 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int bn = a.bn, S = a.stages, stageBytes = times_stage_bytes(bn);
    const long long m0 = (long long) blockIdx.x * 128, n0 = (long long) blockIdx.y * bn;
    const int steps = (int) ((a.K + TK - 1) / TK);
    const int rank = a.splits > 1 ? (int) cluster_rank() : 0;
    int first, count;
    split_range(steps, rank, a.splits, first, count);
    const long long chunks = mx_scale_tiles(a.K); // scale tiles along the contraction, 128 values each
    const int rowsX = bn > 128 && n0 + 128 < a.T ? 2 : 1;

    gemm_setup(&bars, S, 1, 1);
    const unsigned tm = bars.tmem;
    const unsigned scales = tm + 256; // 24 columns a stage: 8 of W, 16 of X
    if (warp == 0 && lane == 0)
    {
        for (int i = 0; i < count; ++i)
        {
            const int s = i % S;
            if (i >= S)
                tc_wait(&bars.empty[s], ((i / S) & 1) ^ 1, &bars.broken, &g_mxStatus);
            if (*reinterpret_cast<volatile unsigned*>(&bars.broken))
            {
                drain_copies(&bars, i, S);
                break;
            }
            const unsigned at = smem_addr(stage0 + (size_t) s * stageBytes);
            const int k = first + i;
            const unsigned nch = (unsigned) (chunks - 2LL * k < 2 ? 1 : 2);
            mbar_arrive_expect_tx(&bars.full[s], 128 * 128 + bn * 128 + nch * 512 * (1 + rowsX));
            tma_load_2d(at, &mapW, k * 128, (int) m0, &bars.full[s]);
            tma_load_2d(at + 16384, &mapX, k * 128, (int) n0, &bars.full[s]);
            const unsigned sw = at + 16384 + bn * 128;
            bulk_load(sw, a.scaleW + ((m0 / 128) * chunks + 2LL * k) * 512, nch * 512, &bars.full[s]);
            for (int r = 0; r < rowsX; ++r)
                bulk_load(sw + 1024 + r * 1024, a.scaleX + ((n0 / 128 + r) * chunks + 2LL * k) * 512, nch * 512, &bars.full[s]);
        }
    }
    else if (warp == 1 && lane == 0)
    {
        for (int i = 0; i < count; ++i)
        {
            const int s = i % S;
            tc_wait(&bars.full[s], (i / S) & 1, &bars.broken, &g_mxStatus);
            tc_fence_after();
            const unsigned at = smem_addr(stage0 + (size_t) s * stageBytes);
            const unsigned sw = at + 16384 + bn * 128;
            const long long left = a.K - (long long) (first + i) * TK;
            const int nch = left > 128 ? 2 : 1;
            const int nk = left >= TK ? 4 : (int) ((left + 63) / 64);
            const unsigned sa = scales + s * 24, sb = sa + 8;
            for (int c = 0; c < nch; ++c)
            {
                tmem_copy_scales(sa + c * 4, smem_desc(sw + c * 512, 16, 128, SWIZZLE_NONE));
                for (int r = 0; r < rowsX; ++r)
                    tmem_copy_scales(sb + c * 8 + r * 4, smem_desc(sw + 1024 + r * 1024 + c * 512, 16, 128, SWIZZLE_NONE));
            }
            for (int j = 0; j < nk; ++j)
                mma_mxf4_ss(tm, smem_desc(at + j * 32, 16, 1024, SWIZZLE_128B), smem_desc(at + 16384 + j * 32, 16, 1024, SWIZZLE_128B), idesc_mxf4(bn, (j & 1) * 2),
                            sa + (j >> 1) * 4, sb + (j >> 1) * 8, i + j > 0);
            tc_commit(&bars.empty[s]);
        }
        tc_commit(&bars.done);
    }
    __syncwarp();
    // every thread sees the end of the products before shared memory is used again and tensor memory is given back
    tc_wait(&bars.done, 0, &bars.broken, &g_mxStatus);
    __syncwarp();
    tc_fence_after();
    write_tile<false, T>(tm, count == 0, bn, warp - 4, reinterpret_cast<float*>(stage0), a.splits, rank, (T*) a.y, a.ld, m0, a.O, n0, a.T, a.bias, false);
    tc_fence_before();
    __syncthreads();
    if (warp == 2)
        tmem_free(tm, TMEM_COLS);
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
    int bn, stages, splits, vec, add;
};

constexpr int GK = 64; // contraction values per stage

__host__ __device__ inline int grad_codes_bytes(int format)
{
    return GK * (format == QAGG_MXFP4 ? 64 : 128);
}

// Two values of this lane, k and k + 1, as bf16: codes b0, b1 (fp4: the byte that holds the value, `nib` the shift to it) times the
// scale pair.  int8: 0x43 over a code byte is the bf16 number 128 + (its low seven bits) with bit 7 moved aside; q = low - (bit 7),
// so q = (128 + low) - (128 or 256), and 256 is 0x4380.  fp4: exponent and mantissa bits set where bf16 has them give the value
// times 2^-126, subnormal included.
template <int FMT>
__device__ __forceinline__ unsigned expand2(unsigned b0, unsigned b1, unsigned nib, unsigned scale)
{
    unsigned v = b0 + (b1 << 16), r;
    if constexpr (FMT == QAGG_MXINT8)
    {
        const unsigned mag = (v & 0x007f007fu) | 0x43004300u, sub = (v & 0x00800080u) | 0x43004300u;
        const __nv_bfloat162 q = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&mag), *reinterpret_cast<const __nv_bfloat162*>(&sub));
        const __nv_bfloat162 e = __hmul2(q, *reinterpret_cast<const __nv_bfloat162*>(&scale));
        r = *reinterpret_cast<const unsigned*>(&e);
    }
    else
    {
        v >>= nib;
        const unsigned t = ((v << 6) & 0x01c001c0u) | ((v << 12) & 0x80008000u), up = 0x7e807e80u; // 2^126
        const __nv_bfloat162 q = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&t), *reinterpret_cast<const __nv_bfloat162*>(&up));
        const __nv_bfloat162 e = __hmul2(q, *reinterpret_cast<const __nv_bfloat162*>(&scale));
        r = *reinterpret_cast<const unsigned*>(&e);
    }
    return r;
}
// multiplier of a block as bf16 bits: 2^X (fp4), 2^X / 64 (int8; subnormal below byte 7)
template <int FMT>
__device__ __forceinline__ unsigned scale_bf16(unsigned byte)
{
    if (byte == 255u)
        return 0x7fffu;
    if (FMT == QAGG_MXINT8)
        return byte > 6u ? (byte - 6u) << 7 : 1u << byte;
    return byte ? byte << 7 : 0x40u;
}

// A dense value as a sum of bf16 planes, exactly: the top eight significant bits by truncation, the next eight, the rest (fp16 has
// eleven: two planes; fp32 twenty-four: three).  Infinities and NaN stay in the first plane.
template <class T, int NP>
__device__ __forceinline__ void split_planes(T x, unsigned short (&p)[NP])
{
    if constexpr (NP == 1)
        p[0] = __bfloat16_as_ushort((__nv_bfloat16) x);
    else
    {
        float v = (float) x;
        const bool finite = (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u;
        if (!finite)
        {
            p[0] = v != v ? 0x7fff : (unsigned short) (__float_as_uint(v) >> 16);
#pragma unroll
            for (int k = 1; k < NP; ++k)
                p[k] = 0;
            return;
        }
#pragma unroll
        for (int k = 0; k < NP; ++k)
        {
            const unsigned top = __float_as_uint(v) & 0xffff0000u;
            p[k] = (unsigned short) (top >> 16);
            v -= __uint_as_float(top);
        }
    }
}

// WEIGHT: dw, lanes = i, columns = o, contraction over the tokens; the dense operand is MN-major (o runs fastest).
// otherwise: dx, lanes = i, columns = t, contraction over o; the dense operand is K-major.
// DENSE 0: dy is bf16 and the copy engine can take it.  DENSE 1..3: that many bf16 planes, made by eight loader warps from T.
template <bool WEIGHT, int FMT, int DENSE, class TD, class TO>
__global__ void __launch_bounds__(DENSE ? GT_DENSE : GT, 1) k_mx_grad(const __grid_constant__ CUtensorMap mapCodes, const __grid_constant__ CUtensorMap mapDy, const GradArgs a)
{
    constexpr int NP = DENSE ? DENSE : 1;
    extern __shared__ unsigned char dyn[];
    __shared__ GemmBars bars;
    __shared__ unsigned scalePairs[8][2][16];
    unsigned char* stage0 = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t) 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int bn = a.bn, S = a.stages;
    const int denseBytes = bn * 128 * NP;
    const int stageBytes = denseBytes + grad_codes_bytes(FMT);
    const long long m0 = (long long) blockIdx.x * 128, n0 = (long long) blockIdx.y * bn;
    const int steps = (int) ((a.C + GK - 1) / GK);
    const int rank = a.splits > 1 ? (int) cluster_rank() : 0;
    int first, count;
    split_range(steps, rank, a.splits, first, count);

    gemm_setup(&bars, S, 8, 8);
    const unsigned tm = bars.tmem;
    const unsigned tmA = tm + 256; // 32 columns a stage
    if (warp == 0 && lane == 0)
    {
        for (int i = 0; i < count; ++i)
        {
            const int s = i % S;
            if (i >= S)
                tc_wait(&bars.empty[s], ((i / S) & 1) ^ 1, &bars.broken, &g_mxStatus);
            if (*reinterpret_cast<volatile unsigned*>(&bars.broken))
            {
                drain_copies(&bars, i, S);
                break;
            }
            const unsigned at = smem_addr(stage0 + (size_t) s * stageBytes);
            const int k0 = (first + i) * GK;
            mbar_arrive_expect_tx(&bars.full[s], grad_codes_bytes(FMT) + (DENSE ? 0 : denseBytes));
            tma_load_2d(at + denseBytes, &mapCodes, (int) (FMT == QAGG_MXFP4 ? m0 / 2 : m0), k0, &bars.full[s]);
            if constexpr (DENSE == 0)
            {
                if constexpr (WEIGHT)
                    for (int n = 0; n < bn; n += 64)
                        tma_load_2d(at + n * 128, &mapDy, (int) n0 + n, k0, &bars.full[s]);
                else
                    tma_load_2d(at, &mapDy, k0, (int) n0, &bars.full[s]);
            }
        }
    }
    else if (warp == 1 && lane == 0)
    {
        const unsigned idesc = idesc_bf16(bn, WEIGHT);
        for (int i = 0; i < count; ++i)
        {
            const int s = i % S;
            const unsigned par = (i / S) & 1;
            tc_wait(&bars.full[s], par, &bars.broken, &g_mxStatus);
            if constexpr (DENSE > 0)
                tc_wait(&bars.dense[s], par, &bars.broken, &g_mxStatus);
            tc_wait(&bars.conv[s], par, &bars.broken, &g_mxStatus);
            tc_fence_after();
            const unsigned at = smem_addr(stage0 + (size_t) s * stageBytes);
            // smallest plane first: its products are added while the sum of this step is small
#pragma unroll
            for (int p = NP - 1; p >= 0; --p)
#pragma unroll
                for (int j = 0; j < GK / 16; ++j)
                {
                    const unsigned b = at + p * bn * 128;
                    const unsigned long long desc = WEIGHT ? smem_desc(b + j * 2048, 8192, 1024, SWIZZLE_128B) : smem_desc(b + j * 32, 16, 1024, SWIZZLE_128B);
                    mma_bf16_ts(tm, tmA + s * 32 + j * 8, desc, idesc, i > 0 || j > 0 || p < NP - 1);
                }
            tc_commit(&bars.empty[s]);
        }
        tc_commit(&bars.done);
    }
    else if (warp >= 4 && warp < 12)
    {
        // expand: lanes 32 * quad .. are one block of the packed matrix; this warp takes 32 of the stage's 64 contraction values
        const int quad = warp & 3, half = (warp - 4) >> 2;
        const long long tilesM = mx_scale_tiles(a.I);
        const unsigned nib = FMT == QAGG_MXFP4 ? (lane & 1) * 4 : 0;
        const unsigned char* mine = a.scales + (m0 / 128) * 512 + lane * 16 + quad;
        auto fetch = [&](int i) -> unsigned {
            const long long k = (long long) (first + i) * GK + half * 32; // the scale tiles cover whole groups of 128 columns
            return mine[k / 128 * tilesM * 512 + (k % 128) / 32 * 4];
        };
        unsigned byte = count > 0 ? fetch(0) : 0;
        for (int i = 0; i < count; ++i)
        {
            const int s = i % S;
            unsigned* pairs = scalePairs[warp - 4][i & 1];
            const unsigned mineScale = scale_bf16<FMT>(byte);
            const unsigned next = __shfl_down_sync(0xffffffffu, mineScale, 1);
            if ((lane & 1) == 0)
                pairs[lane / 2] = mineScale | (next << 16);
            if (i + 1 < count)
                byte = fetch(i + 1);
            __syncwarp();
            tc_wait(&bars.full[s], (i / S) & 1, &bars.broken, &g_mxStatus);
            __syncwarp();
            const unsigned char* codes = stage0 + (size_t) s * stageBytes + denseBytes +
                                         (FMT == QAGG_MXFP4 ? half * 32 * 64 + quad * 16 + lane / 2 : half * 32 * 128 + quad * 32 + lane);
            constexpr int ROW = FMT == QAGG_MXFP4 ? 64 : 128;
            unsigned r[16];
#pragma unroll
            for (int j = 0; j < 16; ++j)
                r[j] = expand2<FMT>(codes[(2 * j) * ROW], codes[(2 * j + 1) * ROW], nib, pairs[j]);
            tc_fence_after(); // the stage's previous products, whose end the copy warp saw, have read this part of tensor memory
            tmem_store16(tmA + ((unsigned) (quad * 32) << 16) + s * 32 + half * 16, r);
            tmem_store_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
                mbar_arrive(&bars.conv[s]);
        }
    }
    else if (DENSE > 0 && warp >= 12)
    {
        // bring the dense operand: rows of 64 contiguous values (128 bytes a plane), eight values a thread and turn
        const TD* dy = (const TD*) a.dy;
        const int t = threadIdx.x - GT;
        for (int i = 0; i < count; ++i)
        {
            const int s = i % S;
            if (i >= S)
                tc_wait(&bars.empty[s], ((i / S) & 1) ^ 1, &bars.broken, &g_mxStatus);
            unsigned char* at = stage0 + (size_t) s * stageBytes;
            const long long k0 = (long long) (first + i) * GK;
            for (int u = t; u < bn * 8; u += 256)
            {
                // row r of piece `atom` in the stage; its place in dy
                const int c = u & 7, r = WEIGHT ? (u >> 3) & 63 : u >> 3, atom = WEIGHT ? u >> 9 : 0;
                const long long line = WEIGHT ? k0 + r : n0 + r;               // token
                const long long col = (WEIGHT ? n0 + atom * 64 : k0) + c * 8;   // output
                const long long lines = WEIGHT ? a.C : a.N, cols = WEIGHT ? a.N : a.C;
                TD v[8];
                const TD* src = dy + line * a.ldDy + col;
                if (line < lines && col + 8 <= cols && a.vec)
                {
                    uint4* q = reinterpret_cast<uint4*>(v);
                    q[0] = *reinterpret_cast<const uint4*>(src);
                    if constexpr (sizeof(TD) == 4)
                        q[1] = *(reinterpret_cast<const uint4*>(src) + 1);
                }
                else
                {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        v[e] = line < lines && col + e < cols ? src[e] : (TD) 0.0f;
                }
                unsigned short pl[8][NP];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    split_planes<TD, NP>(v[e], pl[e]);
                unsigned char* dst = at + atom * 8192 + r * 128 + ((c ^ (r & 7)) << 4);
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    *reinterpret_cast<uint4*>(dst + p * bn * 128) =
                        make_uint4(pl[0][p] | (unsigned) pl[1][p] << 16, pl[2][p] | (unsigned) pl[3][p] << 16, pl[4][p] | (unsigned) pl[5][p] << 16,
                                   pl[6][p] | (unsigned) pl[7][p] << 16);
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0)
                mbar_arrive(&bars.dense[s]);
        }
    }
    __syncwarp();
    tc_wait(&bars.done, 0, &bars.broken, &g_mxStatus);
    __syncwarp();
    tc_fence_after();
    const int resultWarp = warp < 12 ? warp - 4 : -1;
    write_tile<WEIGHT, TO>(tm, count == 0, bn, resultWarp, reinterpret_cast<float*>(stage0), a.splits, rank, (TO*) a.out, a.ld, m0, a.I, n0, a.N, nullptr, a.add != 0);
    tc_fence_before();
    __syncthreads();
    if (warp == 2)
        tmem_free(tm, TMEM_COLS);
}

// ---- launches -----------------------------------------------------------------------------------------------------------------

// Tile width and split of the contraction.  Costs in units of a 256-wide step: a CTA runs steps / splits of them, then its result.
struct Shape
{
    int bn, splits;
};
static Shape choose_shape(long long tilesM, long long N, int steps, int sms, int widest, int narrowest)
{
    Shape best = {widest, 1};
    double bestCost = 1e300;
    for (int bn = widest; bn >= narrowest; bn /= 2)
    {
        if (bn < widest && bn < 128 && N > bn)
            break; // several narrow tiles would read the other operand once each
        const long long tiles = tilesM * ((N + bn - 1) / bn);
        for (int s = 1; s <= 8; s *= 2)
        {
            if (s > 1 && s > steps)
                break;
            const long long waves = (tiles * s + sms - 1) / sms;
            const double step = std::max(bn, 96) / 256.0;
            const double cost = waves * (step * ((steps + s - 1) / s) + 4.0 + 6.0 * bn / 256.0 + (s > 1 ? 2.0 : 0.0));
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

template <class K, class... Args>
static cudaError_t launch_cluster(K kernel, dim3 grid, int threads, int smem, int splits, cudaStream_t st, Args... args)
{
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess)
        return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = splits;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return e != cudaSuccess ? e : cudaGetLastError();
}

static bool codes_map(CUtensorMap* m, const void* codes, long long M, long long N, int format, int boxBytes, int boxCols, bool swizzle)
{
    return encode_map_tiled(m, 1, codes, mx_pitch(M, format), N, mx_pitch(M, format), boxBytes, boxCols, swizzle);
}

template <bool WEIGHT, int FMT, int DENSE, class TD, class TO>
static cudaError_t launch_grad(cudaStream_t st, const CUtensorMap& mc, const CUtensorMap& md, GradArgs a, int sms)
{
    constexpr int NP = DENSE ? DENSE : 1;
    const int stageBytes = a.bn * 128 * NP + grad_codes_bytes(FMT);
    a.stages = stages_for(stageBytes, MAX_STAGES);
    const int smem = smem_for(stageBytes, a.stages, WEIGHT ? 128 * (a.bn + 4) * 4 : a.splits > 1 ? 128 * a.bn * 4 : 0);
    const dim3 grid((unsigned) ((a.I + 127) / 128), (unsigned) ((a.N + a.bn - 1) / a.bn), (unsigned) a.splits);
    return launch_cluster(k_mx_grad<WEIGHT, FMT, DENSE, TD, TO>, grid, DENSE ? GT_DENSE : GT, smem, a.splits, st, mc, md, a);
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
    const int planes = dyType == QAGG_BF16 ? 1 : dyType == QAGG_F16 ? 2 : 3;
    const Shape sh = choose_shape((I + 127) / 128, N, (int) ((C + GK - 1) / GK), cfg.numSMs, planes > 1 ? 128 : 256, 64);
    a.bn = sh.bn;
    a.splits = sh.splits;
    alignas(64) CUtensorMap mc, md;
    std::memset(&mc, 0, sizeof(mc));
    std::memset(&md, 0, sizeof(md));
    if (C > 0 && !codes_map(&mc, codes, I, C, format, format == QAGG_MXFP4 ? 64 : 128, GK, false))
        return fail(QAGG_ECUDA, std::string(who) + ": tensor map of the codes could not be made");
    if (C > 0 && tma && !encode_map_tiled(&md, 2, dy, O, T, ldDy * 2, 64, weight ? GK : a.bn, true))
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
    TimesArgs a = {};
    a.scaleW = (const unsigned char*) w_scales;
    a.scaleX = (const unsigned char*) x_scales;
    a.bias = bias;
    a.y = y;
    a.ld = ld_y;
    a.O = O;
    a.T = T;
    a.K = K;
    const Shape sh = choose_shape((O + 127) / 128, T, (int) ((K + TK - 1) / TK), cfg.numSMs, 256, 16);
    a.bn = sh.bn;
    a.splits = sh.splits;
    const int stageBytes = times_stage_bytes(a.bn);
    a.stages = stages_for(stageBytes, MAX_STAGES);
    const int smem = smem_for(stageBytes, a.stages, a.splits > 1 ? 128 * a.bn * 4 : 0);
    alignas(64) CUtensorMap mw, mx;
    std::memset(&mw, 0, sizeof(mw));
    std::memset(&mx, 0, sizeof(mx));
    if (K > 0 && (!codes_map(&mw, w_codes, K, O, QAGG_MXFP4, 128, 128, true) || !codes_map(&mx, x_codes, K, T, QAGG_MXFP4, 128, a.bn, true)))
        return fail(QAGG_ECUDA, "qagg_mx_times: tensor maps of the codes could not be made");
    const dim3 grid((unsigned) ((O + 127) / 128), (unsigned) ((T + a.bn - 1) / a.bn), (unsigned) a.splits);
    const cudaStream_t st = (cudaStream_t) stream;
    cudaError_t e;
    if (y_type == QAGG_F32)
        e = launch_cluster(k_mx_times<float>, grid, GT, smem, a.splits, st, mw, mx, a);
    else if (y_type == QAGG_F16)
        e = launch_cluster(k_mx_times<__half>, grid, GT, smem, a.splits, st, mw, mx, a);
    else
        e = launch_cluster(k_mx_times<__nv_bfloat16>, grid, GT, smem, a.splits, st, mw, mx, a);
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
    int rc = check_cuda(cudaStreamSynchronize((cudaStream_t) stream), "qagg_mx_check");
    if (rc)
        return rc;
    unsigned status = 0;
    rc = check_cuda(cudaMemcpyFromSymbol(&status, g_mxStatus, sizeof(status)), "qagg_mx_check");
    if (rc || !status)
        return rc;
    const unsigned zero = 0;
    rc = check_cuda(cudaMemcpyToSymbol(g_mxStatus, &zero, sizeof(zero)), "qagg_mx_check");
    return rc ? rc : fail(QAGG_ETIMEOUT, "qagg_mx_check: a bounded wait inside a product kernel ran out; its results are invalid");
}

} // extern "C"
