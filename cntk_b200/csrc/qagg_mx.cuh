// qagg_mx.cuh -- the microscaled (MX) matrix form shared by qagg_mx.cu (quantize, unquantize, activations) and qagg_mx_gemm.cu (4-bit
// product, gradients from packed operands).
//
// A packed M x N matrix has blocks of 32 rows in each column.  A block shares the scale 2^X, kept as the byte X + 127 (255: the
// block held a NaN or an infinity, every value of it is NaN), and value = element * 2^X with
//   QAGG_MXFP4   element = sign, 0 .5 1 1.5 2 3 4 6; two to a byte, the even row in the low half; X = floor(log2 max) - 2
//   QAGG_MXINT8  element = q / 64, q = -127..127; one to a byte;                                X = floor(log2 max)
// Columns are padded to whole blocks.  Scale bytes lie in tiles of 128 columns x 4 blocks (512 bytes), inside a tile at
// (column % 32) * 16 + (column % 128 / 32) * 4 + block % 4: the order in which the tensor cores take block scales, so the product
// copies tiles as they are.  The four bytes of one column in a tile are one aligned word.
//
// Every value of either format is exactly a bfloat16 (at most 7 significant bits, exponent range included: the smallest int8
// step, 2^-133, is the smallest subnormal), which is why the gradients can use the tensor cores' bf16 products without rounding
// the packed operand again.
#pragma once

#include "../../include/qagg.h"
#include "qagg_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>

namespace qagg {

constexpr int MX_BLOCK = 32;

__host__ __device__ inline long long mx_blocks(long long M)
{
    return (M + MX_BLOCK - 1) / MX_BLOCK;
}
// bytes from one packed column to the next: whole blocks, so always a multiple of 16
__host__ __device__ inline long long mx_pitch(long long M, int format)
{
    return mx_blocks(M) * (format == QAGG_MXFP4 ? 16 : 32);
}
__host__ __device__ inline long long mx_scale_tiles(long long M)
{
    return (mx_blocks(M) + 3) / 4;
}

// 2^X of a scale byte below 255 (byte 0 is 2^-127, a subnormal), and its reciprocal
__device__ __forceinline__ float mx_scale(unsigned byte)
{
    return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}
__device__ __forceinline__ float mx_scale_inv(unsigned byte)
{
    return __uint_as_float(byte < 254u ? (254u - byte) << 23 : 0x00400000u);
}

// eight values of one column as they were loaded
template <class T>
struct Raw8;
template <>
struct Raw8<float>
{
    uint4 a, b;
};
template <>
struct Raw8<__half>
{
    uint4 a;
};
template <>
struct Raw8<__nv_bfloat16>
{
    uint4 a;
};

// n = values that exist (0..8); the others read as zero.  vec: the address is 16-byte aligned.
template <class T>
__device__ __forceinline__ Raw8<T> load8(const T* p, int n, bool vec)
{
    Raw8<T> r = {};
    if (vec && n == 8)
    {
        const uint4* q = reinterpret_cast<const uint4*>(p);
        r.a = __ldcs(q);
        if constexpr (sizeof(T) == 4)
            r.b = __ldcs(q + 1);
    }
    else
    {
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n)
                e[i] = p[i];
    }
    return r;
}
// argument checks shared by the entry points (host)
int mx_check_dims(const char* who, long long M, long long N);
bool mx_type_ok(int type);
inline int mx_type_bytes(int type)
{
    return type == QAGG_F32 ? 4 : 2;
}

} // namespace qagg
