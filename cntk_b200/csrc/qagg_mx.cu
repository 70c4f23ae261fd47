// qagg_mx.cu -- microscaled matrices: quantize (along rows or, transposing, along columns), unquantize, and pointwise layers
// that keep their input in 8 bits for the backward pass.  The form is described in qagg_mx.cuh.
//
// All kernels here move each value once and are bound by HBM.  One CTA takes one scale tile: 128 packed columns x 4 blocks.
// Sixteen threads share a column's 128 rows, eight values each (one 16-byte load of a 16-bit type), so a block's largest magnitude
// takes two shuffles and the tile's 512 scale bytes are collected in shared memory and leave as full lines.
#include "qagg_mx.cuh"

#include <algorithm>
#include <string>

namespace qagg {

constexpr int MXT = 256;              // threads per CTA
constexpr int MX_TILE = 128;          // rows and columns of a tile
constexpr int MX_PASS = MXT / 16;     // columns per pass
constexpr int MX_PASSES = MX_TILE / MX_PASS;

// ---- eight values of one column -------------------------------------------------------------------------------------------

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&v)[8])
{
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = to_float(e[i]);
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], int n, bool vec)
{
    Raw8<T> r;
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        e[i] = from_float<T>(v[i]);
    if (vec && n == 8)
    {
        uint4* q = reinterpret_cast<uint4*>(p);
        __stcs(q, r.a);
        if constexpr (sizeof(T) == 4)
            __stcs(q + 1, r.b);
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n)
                p[i] = e[i];
    }
}

// ---- elements ---------------------------------------------------------------------------------------------------------------

// Scale byte of a block from the largest magnitude's bit pattern (as an integer: NaN > infinity > every number).  The exponent
// field is floor(log2) + 127, and 0 for subnormals, where X is held at -127 anyway.
template <int FMT>
__device__ __forceinline__ unsigned scale_byte(unsigned top)
{
    if (top >= 0x7f800000u)
        return 255u;
    const unsigned e = top >> 23;
    return FMT == QAGG_MXFP4 ? (e > 2u ? e - 2u : 0u) : e;
}

// x / 2^X is exact (a value whose quotient is subnormal is far below the first rounding border).  int8: q by adding 1.5 * 2^23,
// which rounds to an integer, ties to even, in the low bits.  fp4: the hardware's conversion, nearest even, held at 6.
template <int FMT, int N>
__device__ __forceinline__ void encode(const float (&v)[N], unsigned byte, unsigned (&out)[N / (FMT == QAGG_MXFP4 ? 8 : 4)])
{
    const float inv = mx_scale_inv(byte);
    const bool bad = byte == 255u;
    if constexpr (FMT == QAGG_MXFP4)
    {
#pragma unroll
        for (int w = 0; w < N / 8; ++w)
        {
            unsigned r = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                r |= (unsigned) __nv_cvt_float2_to_fp4x2(make_float2(v[8 * w + 2 * i] * inv, v[8 * w + 2 * i + 1] * inv), __NV_E2M1, cudaRoundNearest) << (8 * i);
            out[w] = bad ? 0u : r;
        }
    }
    else
    {
#pragma unroll
        for (int w = 0; w < N / 4; ++w)
        {
            unsigned q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const float a = fminf(fmaxf(v[4 * w + i] * inv, -127.0f / 64.0f), 127.0f / 64.0f);
                q[i] = __float_as_uint(__fmaf_rn(a, 64.0f, 12582912.0f));
            }
            const unsigned r = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
            out[w] = bad ? 0u : r;
        }
    }
}
// eight elements -> values
template <int FMT>
__device__ __forceinline__ void decode8(const unsigned* w, unsigned byte, float (&v)[8])
{
    const float s = byte == 255u ? __uint_as_float(0x7fffffffu) : mx_scale(byte);
    if constexpr (FMT == QAGG_MXFP4)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t) (w[0] >> (8 * i)), __NV_E2M1);
            const float2 f = __half22float2(__half2(h));
            v[2 * i] = f.x * s;
            v[2 * i + 1] = f.y * s;
        }
    }
    else
    {
        // element first, then the scale: q / 64 * 2^X, each product exact, down to the smallest scale
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = ((float) (signed char) (w[i / 4] >> (8 * (i % 4))) * 0.015625f) * s;
    }
}

// ---- pointwise functions -----------------------------------------------------------------------------------------------------

template <int ACT>
__device__ __forceinline__ float act_value(float x)
{
    if constexpr (ACT == QAGG_ACT_RELU)
        return x > 0.0f ? x : (x != x ? x : 0.0f);
    else if constexpr (ACT == QAGG_ACT_SIGMOID)
        return __fdiv_rn(1.0f, 1.0f + expf(-x));
    else if constexpr (ACT == QAGG_ACT_TANH)
        return tanhf(x);
    else if constexpr (ACT == QAGG_ACT_GELU)
        return x * (0.5f * (1.0f + erff(x * 0.70710678118654752f)));
    else
        return __fdiv_rn(x, 1.0f + expf(-x));
}
// derivative; with e = exp(-|x|) no form here overflows or cancels
template <int ACT>
__device__ __forceinline__ float act_slope(float x)
{
    if constexpr (ACT == QAGG_ACT_RELU)
        return x > 0.0f ? 1.0f : (x != x ? x : 0.0f);
    else if constexpr (ACT == QAGG_ACT_SIGMOID)
    {
        const float e = expf(-fabsf(x)), d = 1.0f + e;
        return __fdiv_rn(e, d * d);
    }
    else if constexpr (ACT == QAGG_ACT_TANH)
    {
        const float e = expf(-2.0f * fabsf(x)), d = 1.0f + e;
        return __fdiv_rn(4.0f * e, d * d);
    }
    else if constexpr (ACT == QAGG_ACT_GELU)
        return __fmaf_rn(x * 0.39894228040143268f, expf(-0.5f * x * x), 0.5f * (1.0f + erff(x * 0.70710678118654752f)));
    else
    {
        const float e = expf(-fabsf(x)), d = 1.0f + e;
        const float s = __fdiv_rn(x >= 0.0f ? 1.0f : e, d); // the sigmoid of x
        return __fmaf_rn(x, __fdiv_rn(e, d * d), s);
    }
}

// ---- quantize along the rows; with ACT >= 0 also y = f(x) --------------------------------------------------------------------

template <class T, int FMT, int ACT>
__global__ void __launch_bounds__(MXT) k_mx_quantize(const T* x, long long ldx, unsigned char* codes, unsigned char* scales, T* y, long long ldy,
                                                     long long M, long long N, int vecX, int vecY)
{
    __shared__ __align__(16) unsigned char tile[512];
    const long long row0 = (long long) blockIdx.x * MX_TILE;
    const long long col0 = (long long) blockIdx.y * MX_TILE;
    const int tid = threadIdx.x, seg = tid & 15;
    if (tid < 32)
        reinterpret_cast<uint4*>(tile)[tid] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const long long row = row0 + seg * 8;
    const int n = row >= M ? 0 : (int) (M - row < 8 ? M - row : 8);
    const bool block = (row0 + (seg & ~3) * 8) < M; // this thread's block exists
    const long long pitch = mx_pitch(M, FMT);
    constexpr int HALF = sizeof(T) == 4 ? MX_PASSES / 2 : MX_PASSES; // loads in flight per thread: 64 bytes and up
#pragma unroll
    for (int h = 0; h < MX_PASSES; h += HALF)
    {
        Raw8<T> raw[HALF];
#pragma unroll
        for (int p = 0; p < HALF; ++p)
        {
            const long long col = col0 + (h + p) * MX_PASS + (tid >> 4);
            raw[p] = load8(x + col * ldx + row, col < N ? n : 0, vecX);
        }
#pragma unroll
        for (int p = 0; p < HALF; ++p)
        {
            const int c = (h + p) * MX_PASS + (tid >> 4);
            const long long col = col0 + c;
            float v[8];
            unpack8(raw[p], v);
            unsigned top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const unsigned byte = scale_byte<FMT>(top);
            if (col < N && block)
            {
                unsigned w[FMT == QAGG_MXFP4 ? 1 : 2];
                encode<FMT, 8>(v, byte, w);
                unsigned char* at = codes + col * pitch + (FMT == QAGG_MXFP4 ? row / 2 : row);
                if constexpr (FMT == QAGG_MXFP4)
                    *reinterpret_cast<unsigned*>(at) = w[0];
                else
                    *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
                if ((seg & 3) == 0)
                    tile[(c & 31) * 16 + (c >> 5) * 4 + (seg >> 2)] = (unsigned char) byte;
                if constexpr (ACT >= 0)
                {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        v[i] = act_value<ACT>(v[i]);
                    store8(y + col * ldy + row, v, n, vecY);
                }
            }
        }
    }
    __syncthreads();
    if (tid < 32)
        reinterpret_cast<uint4*>(scales + ((long long) blockIdx.y * gridDim.x + blockIdx.x) * 512)[tid] = reinterpret_cast<const uint4*>(tile)[tid];
}

// ---- quantize the transpose: blocks along the columns of x -------------------------------------------------------------------
// A 128 x 128 tile of x goes through shared memory as it lies (rows contiguous); a thread then takes one packed column (a row of
// x) and 32 of its values, which neighbouring lanes read from neighbouring addresses.
template <class T, int FMT>
__global__ void __launch_bounds__(MXT) k_mx_quantize_t(const T* __restrict__ x, long long ldx, unsigned char* __restrict__ codes,
                                                       unsigned char* __restrict__ scales, long long M, long long N, int vecX)
{
    extern __shared__ __align__(16) unsigned char smem[];
    T* s = reinterpret_cast<T*>(smem);
    __shared__ __align__(16) unsigned char tile[512];
    const long long col0 = (long long) blockIdx.x * MX_TILE; // columns of x: the packed matrix's rows
    const long long row0 = (long long) blockIdx.y * MX_TILE; // rows of x: the packed matrix's columns
    const int tid = threadIdx.x;
    if (tid < 32)
        reinterpret_cast<uint4*>(tile)[tid] = make_uint4(0, 0, 0, 0);
    {
        const int seg = tid & 15;
        const long long row = row0 + seg * 8;
        const int n = row >= M ? 0 : (int) (M - row < 8 ? M - row : 8);
#pragma unroll
        for (int p = 0; p < MX_PASSES; ++p)
        {
            const int c = p * MX_PASS + (tid >> 4);
            const Raw8<T> r = load8(x + (col0 + c) * ldx + row, col0 + c < N ? n : 0, vecX);
            *reinterpret_cast<Raw8<T>*>(s + c * MX_TILE + seg * 8) = r;
        }
    }
    __syncthreads();
    const long long pitch = mx_pitch(N, FMT);
#pragma unroll 1
    for (int u = tid; u < MX_TILE * 4; u += MXT)
    {
        const int r = u & (MX_TILE - 1), b = u / MX_TILE;
        if (row0 + r >= M || col0 + b * MX_BLOCK >= N)
            continue;
        float v[32];
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i)
        {
            v[i] = to_float(s[(b * MX_BLOCK + i) * MX_TILE + r]);
            top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
        }
        const unsigned byte = scale_byte<FMT>(top);
        unsigned w[FMT == QAGG_MXFP4 ? 4 : 8];
        encode<FMT, 32>(v, byte, w);
        uint4* at = reinterpret_cast<uint4*>(codes + (row0 + r) * pitch + (col0 + b * MX_BLOCK) / (FMT == QAGG_MXFP4 ? 2 : 1));
        at[0] = make_uint4(w[0], w[1], w[2], w[3]);
        if constexpr (FMT == QAGG_MXINT8)
            at[1] = make_uint4(w[4], w[5], w[6], w[7]);
        tile[(r & 31) * 16 + (r >> 5) * 4 + b] = (unsigned char) byte;
    }
    __syncthreads();
    if (tid < 32)
        reinterpret_cast<uint4*>(scales + ((long long) blockIdx.y * gridDim.x + blockIdx.x) * 512)[tid] = reinterpret_cast<const uint4*>(tile)[tid];
}

// ---- unquantize; with ACT >= 0 the backward pass of a pointwise layer: out = in * f'(value) ----------------------------------

template <class T, int FMT, int ACT>
__global__ void __launch_bounds__(MXT) k_mx_unquantize(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales, const T* in,
                                                       long long ldin, T* out, long long ldout, long long M, long long N, int vecIn, int vecOut)
{
    __shared__ __align__(16) unsigned char tile[512];
    const long long row0 = (long long) blockIdx.x * MX_TILE;
    const long long col0 = (long long) blockIdx.y * MX_TILE;
    const int tid = threadIdx.x, seg = tid & 15;
    const long long row = row0 + seg * 8;
    const int n = row >= M ? 0 : (int) (M - row < 8 ? M - row : 8);
    const long long pitch = mx_pitch(M, FMT);
    constexpr int W = FMT == QAGG_MXFP4 ? 1 : 2;
    constexpr int HALF = sizeof(T) == 4 && ACT >= 0 ? MX_PASSES / 2 : MX_PASSES;
    if (tid < 32)
        reinterpret_cast<uint4*>(tile)[tid] = __ldcs(reinterpret_cast<const uint4*>(scales + ((long long) blockIdx.y * gridDim.x + blockIdx.x) * 512) + tid);
    __syncthreads();
#pragma unroll
    for (int h = 0; h < MX_PASSES; h += HALF)
    {
        unsigned w[HALF][W];
        Raw8<T> raw[ACT >= 0 ? HALF : 1];
#pragma unroll
        for (int p = 0; p < HALF; ++p)
        {
            const long long col = col0 + (h + p) * MX_PASS + (tid >> 4);
            const bool have = col < N && n > 0;
            const unsigned char* at = codes + col * pitch + (FMT == QAGG_MXFP4 ? row / 2 : row);
            if constexpr (FMT == QAGG_MXFP4)
                w[p][0] = have ? __ldcs(reinterpret_cast<const unsigned*>(at)) : 0u;
            else
            {
                const uint2 q = have ? __ldcs(reinterpret_cast<const uint2*>(at)) : make_uint2(0, 0);
                w[p][0] = q.x;
                w[p][1] = q.y;
            }
            if constexpr (ACT >= 0)
                raw[p] = load8(in + col * ldin + row, have ? n : 0, vecIn);
        }
#pragma unroll
        for (int p = 0; p < HALF; ++p)
        {
            const int c = (h + p) * MX_PASS + (tid >> 4);
            const long long col = col0 + c;
            if (col >= N || n == 0)
                continue;
            float v[8];
            decode8<FMT>(w[p], tile[(c & 31) * 16 + (c >> 5) * 4 + (seg >> 2)], v);
            if constexpr (ACT >= 0)
            {
                float g[8];
                unpack8(raw[p], g);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    v[i] = g[i] * act_slope<ACT>(v[i]);
            }
            store8(out + col * ldout + row, v, n, vecOut);
        }
    }
}

// ---- launches -----------------------------------------------------------------------------------------------------------------

bool mx_type_ok(int type)
{
    return type == QAGG_F32 || type == QAGG_F16 || type == QAGG_BF16;
}
static bool format_ok(int format)
{
    return format == QAGG_MXFP4 || format == QAGG_MXINT8;
}

int mx_check_dims(const char* who, long long M, long long N)
{
    if (M < 0 || N < 0)
        return fail(QAGG_EINVAL, std::string(who) + ": negative matrix dimension");
    // tiles of 128 columns are the grid's second dimension (65535 at most); tensor maps take 31-bit coordinates
    if (M >= (1LL << 30) || N > 65535LL * MX_TILE)
        return fail(QAGG_EINVAL, std::string(who) + ": matrix dimension too large (rows < 2^30, columns <= 65535 * 128)");
    return QAGG_OK;
}

static int vec_ok(const void* p, long long ld, int type)
{
    return (((uintptr_t) p | (uintptr_t) (ld * mx_type_bytes(type))) & 15) == 0;
}

static dim3 tile_grid(long long M, long long N)
{
    return dim3((unsigned) mx_scale_tiles(M), (unsigned) ((N + MX_TILE - 1) / MX_TILE));
}

template <class T, int FMT>
static cudaError_t launch_quantize(cudaStream_t st, const T* x, long long ld, void* codes, void* scales, long long M, long long N, int transpose, int vec)
{
    if (!transpose)
        k_mx_quantize<T, FMT, -1><<<tile_grid(M, N), MXT, 0, st>>>(x, ld, (unsigned char*) codes, (unsigned char*) scales, nullptr, 0, M, N, vec, 0);
    else
    {
        constexpr int bytes = MX_TILE * MX_TILE * (int) sizeof(T);
        if (bytes > 48 * 1024 - 512)
        {
            const cudaError_t e = cudaFuncSetAttribute(k_mx_quantize_t<T, FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
            if (e != cudaSuccess)
                return e;
        }
        k_mx_quantize_t<T, FMT><<<tile_grid(N, M), MXT, bytes, st>>>(x, ld, (unsigned char*) codes, (unsigned char*) scales, M, N, vec);
    }
    return cudaGetLastError();
}

// calls f(T) for the element type, g(ACT) for the function
template <class F>
static cudaError_t by_type(int type, F f)
{
    if (type == QAGG_F32)
        return f((float*) nullptr);
    if (type == QAGG_F16)
        return f((__half*) nullptr);
    return f((__nv_bfloat16*) nullptr);
}
template <int A>
struct ActTag
{
    static constexpr int value = A;
};
template <class F>
static cudaError_t by_act(int act, F f)
{
    switch (act)
    {
    case QAGG_ACT_RELU: return f(ActTag<QAGG_ACT_RELU>());
    case QAGG_ACT_SIGMOID: return f(ActTag<QAGG_ACT_SIGMOID>());
    case QAGG_ACT_TANH: return f(ActTag<QAGG_ACT_TANH>());
    case QAGG_ACT_GELU: return f(ActTag<QAGG_ACT_GELU>());
    default: return f(ActTag<QAGG_ACT_SILU>());
    }
}

} // namespace qagg

using namespace qagg;

extern "C" {

int64_t qagg_mx_code_bytes(int64_t M, int64_t N, int format)
{
    if (M < 0 || N < 0 || !format_ok(format))
        return fail(QAGG_EINVAL, "qagg_mx_code_bytes: bad arguments");
    return N * mx_pitch(M, format);
}

int64_t qagg_mx_scale_bytes(int64_t M, int64_t N)
{
    if (M < 0 || N < 0)
        return fail(QAGG_EINVAL, "qagg_mx_scale_bytes: bad arguments");
    return (N + 127) / 128 * mx_scale_tiles(M) * 512;
}

int qagg_mx_quantize(void* stream, const void* x, int type, int64_t ld, void* codes, void* scales, int64_t M, int64_t N, int format, int transpose)
{
    int rc = transpose ? mx_check_dims("qagg_mx_quantize", N, M) : mx_check_dims("qagg_mx_quantize", M, N);
    if (rc)
        return rc;
    if (!mx_type_ok(type) || !format_ok(format))
        return fail(QAGG_EINVAL, "qagg_mx_quantize: unknown element type or format");
    if (ld < M)
        return fail(QAGG_EINVAL, "qagg_mx_quantize: ld is less than the number of rows");
    if (M == 0 || N == 0)
        return QAGG_OK;
    if (!x || !codes || !scales)
        return fail(QAGG_EINVAL, "qagg_mx_quantize: null pointer");
    if ((((uintptr_t) codes | (uintptr_t) scales) & 15) || ((uintptr_t) x & (mx_type_bytes(type) - 1)))
        return fail(QAGG_EINVAL, "qagg_mx_quantize: codes and scales must be 16-byte aligned, x aligned to its type");
    const int vec = vec_ok(x, ld, type);
    return check_cuda(by_type(type, [&](auto* t) {
                          using T = std::remove_pointer_t<decltype(t)>;
                          return format == QAGG_MXFP4 ? launch_quantize<T, QAGG_MXFP4>((cudaStream_t) stream, (const T*) x, ld, codes, scales, M, N, transpose, vec)
                                                      : launch_quantize<T, QAGG_MXINT8>((cudaStream_t) stream, (const T*) x, ld, codes, scales, M, N, transpose, vec);
                      }),
                      "microscaled quantize kernel launch");
}

int qagg_mx_unquantize(void* stream, const void* codes, const void* scales, void* out, int type, int64_t ld, int64_t M, int64_t N, int format)
{
    int rc = mx_check_dims("qagg_mx_unquantize", M, N);
    if (rc)
        return rc;
    if (!mx_type_ok(type) || !format_ok(format))
        return fail(QAGG_EINVAL, "qagg_mx_unquantize: unknown element type or format");
    if (ld < M)
        return fail(QAGG_EINVAL, "qagg_mx_unquantize: ld is less than the number of rows");
    if (M == 0 || N == 0)
        return QAGG_OK;
    if (!codes || !scales || !out)
        return fail(QAGG_EINVAL, "qagg_mx_unquantize: null pointer");
    if ((((uintptr_t) codes | (uintptr_t) scales) & 15) || ((uintptr_t) out & (mx_type_bytes(type) - 1)))
        return fail(QAGG_EINVAL, "qagg_mx_unquantize: codes and scales must be 16-byte aligned, out aligned to its type");
    const int vec = vec_ok(out, ld, type);
    return check_cuda(by_type(type, [&](auto* t) {
                          using T = std::remove_pointer_t<decltype(t)>;
                          const dim3 grid = tile_grid(M, N);
                          if (format == QAGG_MXFP4)
                              k_mx_unquantize<T, QAGG_MXFP4, -1><<<grid, MXT, 0, (cudaStream_t) stream>>>((const unsigned char*) codes, (const unsigned char*) scales, nullptr, 0,
                                                                                                          (T*) out, ld, M, N, 0, vec);
                          else
                              k_mx_unquantize<T, QAGG_MXINT8, -1><<<grid, MXT, 0, (cudaStream_t) stream>>>((const unsigned char*) codes, (const unsigned char*) scales, nullptr, 0,
                                                                                                           (T*) out, ld, M, N, 0, vec);
                          return cudaGetLastError();
                      }),
                      "microscaled unquantize kernel launch");
}

static int check_act(const char* who, const void* a, int64_t lda, const void* b, int64_t ldb, int type, int act, const void* codes, const void* scales, int64_t M, int64_t N)
{
    int rc = mx_check_dims(who, M, N);
    if (rc)
        return rc;
    if (!mx_type_ok(type) || act < QAGG_ACT_RELU || act > QAGG_ACT_SILU)
        return fail(QAGG_EINVAL, std::string(who) + ": unknown element type or function");
    if (lda < M || ldb < M)
        return fail(QAGG_EINVAL, std::string(who) + ": ld is less than the number of rows");
    if (M == 0 || N == 0)
        return QAGG_OK;
    if (!a || !b || !codes || !scales)
        return fail(QAGG_EINVAL, std::string(who) + ": null pointer");
    if ((((uintptr_t) codes | (uintptr_t) scales) & 15) || (((uintptr_t) a | (uintptr_t) b) & (mx_type_bytes(type) - 1)))
        return fail(QAGG_EINVAL, std::string(who) + ": codes and scales must be 16-byte aligned, the others aligned to their type");
    return QAGG_OK;
}

int qagg_mx_act_forward(void* stream, const void* x, int type, int64_t ld_x, int act, void* y, int64_t ld_y, void* codes, void* scales, int64_t M, int64_t N)
{
    const int rc = check_act("qagg_mx_act_forward", x, ld_x, y, ld_y, type, act, codes, scales, M, N);
    if (rc || M == 0 || N == 0)
        return rc;
    return check_cuda(by_type(type, [&](auto* t) {
                          using T = std::remove_pointer_t<decltype(t)>;
                          return by_act(act, [&](auto tag) {
                              k_mx_quantize<T, QAGG_MXINT8, decltype(tag)::value><<<tile_grid(M, N), MXT, 0, (cudaStream_t) stream>>>(
                                  (const T*) x, ld_x, (unsigned char*) codes, (unsigned char*) scales, (T*) y, ld_y, M, N, vec_ok(x, ld_x, type), vec_ok(y, ld_y, type));
                              return cudaGetLastError();
                          });
                      }),
                      "activation kernel launch");
}

int qagg_mx_act_backward(void* stream, const void* dy, int type, int64_t ld_dy, const void* codes, const void* scales, int act, void* dx, int64_t ld_dx, int64_t M, int64_t N)
{
    const int rc = check_act("qagg_mx_act_backward", dy, ld_dy, dx, ld_dx, type, act, codes, scales, M, N);
    if (rc || M == 0 || N == 0)
        return rc;
    return check_cuda(by_type(type, [&](auto* t) {
                          using T = std::remove_pointer_t<decltype(t)>;
                          return by_act(act, [&](auto tag) {
                              k_mx_unquantize<T, QAGG_MXINT8, decltype(tag)::value><<<tile_grid(M, N), MXT, 0, (cudaStream_t) stream>>>(
                                  (const unsigned char*) codes, (const unsigned char*) scales, (const T*) dy, ld_dy, (T*) dx, ld_dx, M, N, vec_ok(dy, ld_dy, type),
                                  vec_ok(dx, ld_dx, type));
                              return cudaGetLastError();
                          });
                      }),
                      "activation backward kernel launch");
}

} // extern "C"
