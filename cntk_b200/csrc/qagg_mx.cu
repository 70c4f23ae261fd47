// qagg_mx.cu -- microscaled matrices: quantize (along rows or, transposing, along columns), unquantize, and pointwise layers
// that keep their input in 8 bits for the backward pass.  The form is described in qagg_mx.cuh.
//
// All kernels here move each value once and are bound by HBM.  One CTA takes one scale tile: 128 packed columns x 4 blocks.
// A thread takes 32 bytes of dense values at a time, with one 256-bit access where they are aligned (sixteen values of a 16-bit type,
// eight fp32): what a block costs, the largest magnitude, the scale, the addresses, is shared by more values than with 16 bytes, and a
// warp still reads and writes whole sectors.  Two or four threads share a block; the tile's 512 scale bytes are collected in shared
// memory and leave as full lines.
#include "qagg_mx.cuh"

#include <algorithm>
#include <string>
#include <type_traits>

namespace qagg {

constexpr int MXT = 256;     // threads per CTA
constexpr int MX_TILE = 128; // rows and columns of a tile
template <class T, bool ACT = false>
struct Shape // of the threads over a tile; ACT: with a function's arithmetic, which needs the registers
{
    static constexpr int V = 32 / sizeof(T);  // values per thread and turn
    static constexpr int LANES = MX_TILE / V; // threads per column
    static constexpr int COLS = MXT / LANES;  // columns per pass
    static constexpr int PASSES = MX_TILE / COLS;
    static constexpr int FLIGHT = ACT ? 1 : 4; // passes whose loads are in flight together
    static constexpr int PARTS = MX_BLOCK / V; // threads per block
};
struct Raw32
{
    uint4 a, b;
};
// how a matrix may be accessed: 32 bytes a time, 16, or value by value
constexpr int VEC32 = 2, VEC16 = 1;

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

// 32 bytes of values: n of them exist, the others read as zero.  Dense values pass once: first to leave L2, so that codes and scales, which
// the next kernel wants, stay (2048 x 16384 to int8 and back: 50.5 us with plain streaming accesses, 44.8 so).
template <class T>
__device__ __forceinline__ Raw32 load32(const T* p, int n, int vec)
{
    constexpr int V = Shape<T>::V;
    Raw32 r;
    if (vec == VEC32 && n == V)
    {
        asm volatile("ld.global.L1::no_allocate.L2::evict_first.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r.a.x), "=r"(r.a.y), "=r"(r.a.z), "=r"(r.a.w), "=r"(r.b.x), "=r"(r.b.y), "=r"(r.b.z), "=r"(r.b.w)
                     : "l"(p));
        return r;
    }
    r.a = r.b = make_uint4(0, 0, 0, 0);
    if (vec && n == V)
    {
        const uint4* q = reinterpret_cast<const uint4*>(p);
        r.a = __ldcs(q);
        r.b = __ldcs(q + 1);
        return r;
    }
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < n)
            e[i] = p[i];
    return r;
}
template <class T>
__device__ __forceinline__ void unpack32(const Raw32& r, float (&v)[Shape<T>::V])
{
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < Shape<T>::V; ++i)
        v[i] = to_float(e[i]);
}
template <class T>
__device__ __forceinline__ void store32(T* p, const float (&v)[Shape<T>::V], int n, int vec)
{
    constexpr int V = Shape<T>::V;
    Raw32 r;
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < V; ++i)
        e[i] = from_float<T>(v[i]);
    if (vec == VEC32 && n == V)
        asm volatile("st.global.L1::no_allocate.L2::evict_first.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r.a.x), "r"(r.a.y), "r"(r.a.z), "r"(r.a.w), "r"(r.b.x), "r"(r.b.y),
                     "r"(r.b.z), "r"(r.b.w)
                     : "memory");
    else if (vec && n == V)
    {
        uint4* q = reinterpret_cast<uint4*>(p);
        __stcs(q, r.a);
        __stcs(q + 1, r.b);
    }
    else
    {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n)
                p[i] = e[i];
    }
}

// Matrices whose columns are not 16-byte aligned: a warp's columns of one pass (32 bytes a lane) are read and written value by value,
// neighbouring lanes neighbouring values, and change hands in the warp's kilobyte of shared memory.
template <class T>
struct Exchange
{
    static constexpr int V = Shape<T>::V;
    T v[V]; // value 32 j + lane of the warp's columns, 128 rows each
    __device__ __forceinline__ void fetch(const T* first, long long ld, int rows, int cols)
    {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int j = 0; j < V; ++j)
        {
            const int at = j * 32 + lane, c = at / MX_TILE, r = at % MX_TILE;
            v[j] = c < cols && r < rows ? first[c * ld + r] : from_float<T>(0.0f);
        }
    }
    __device__ __forceinline__ Raw32 take(T* room) const // what load32 gives
    {
        const int lane = threadIdx.x & 31;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < V; ++j)
            room[j * 32 + lane] = v[j];
        __syncwarp();
        return reinterpret_cast<const Raw32*>(room)[lane];
    }
    static __device__ __forceinline__ void put(T* room, const float (&value)[V], T* first, long long ld, int rows, int cols)
    {
        const int lane = threadIdx.x & 31;
        Raw32 r;
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int i = 0; i < V; ++i)
            e[i] = from_float<T>(value[i]);
        __syncwarp();
        reinterpret_cast<Raw32*>(room)[lane] = r;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < V; ++j)
        {
            const int at = j * 32 + lane, c = at / MX_TILE, r_ = at % MX_TILE;
            if (c < cols && r_ < rows)
                first[c * ld + r_] = room[at];
        }
    }
};

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

// A block's scale as its elements need it.  int8: q is the low byte of x * 2^(6 - X) + 1.5 * 2^23, whose one rounding is to the integer,
// nearest even; where 2^(6 - X) is no float, or the largest element would round up to 128, the quotient is taken first and held.
// fp4: the hardware's conversion of x / 2^X (exact), nearest even, held at 6.
template <int FMT>
struct BlockEncoder
{
    float inv; // 1 / 2^X, int8: 2^(6 - X)
    bool rare, bad;
    unsigned byte;
    __device__ __forceinline__ explicit BlockEncoder(unsigned top)
    {
        byte = scale_byte<FMT>(top);
        bad = byte == 255u;
        if constexpr (FMT == QAGG_MXFP4)
        {
            inv = mx_scale_inv(byte);
            rare = false;
        }
        else
        {
            rare = byte < 6u || (top & 0x7f0000u) == 0x7f0000u; // (top: also of NaN and infinity, whose byte is 255)
            inv = rare || bad ? mx_scale_inv(byte) : __uint_as_float((260u - byte) << 23);
        }
    }
    // four int8 or (in 16 bits) four fp4 codes
    __device__ __forceinline__ unsigned encode4(float a, float b, float c, float d) const
    {
        if (bad)
            return 0u;
        if constexpr (FMT == QAGG_MXFP4)
            return (unsigned) __nv_cvt_float2_to_fp4x2(make_float2(a * inv, b * inv), __NV_E2M1, cudaRoundNearest) |
                   (unsigned) __nv_cvt_float2_to_fp4x2(make_float2(c * inv, d * inv), __NV_E2M1, cudaRoundNearest) << 8;
        float v[4] = {a, b, c, d};
        float scale = inv;
        if (rare)
        {
            asm volatile(""); // a branch
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = fminf(fmaxf(v[i] * inv, -127.0f / 64.0f), 127.0f / 64.0f);
            scale = 64.0f;
        }
        unsigned q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            q[i] = __float_as_uint(__fmaf_rn(v[i], scale, 12582912.0f));
        return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
    }
};
// Codes -> values.  int8: a code with its sign bit turned, set under the exponent of 2^23, is the float 2^23 + 128 + q; times 2^(X - 6) less
// (2^23 + 128) 2^(X - 6) in one fused step it is the value, exactly.  Where that difference overflows (X > 103, or NaN: s is then NaN in
// either form) 2^23 + 128 is taken off first.
template <int FMT>
struct BlockDecoder
{
    float s, off;
    bool rare;
    __device__ __forceinline__ explicit BlockDecoder(unsigned byte)
    {
        if constexpr (FMT == QAGG_MXFP4)
            s = mx_scale(byte);
        else
        {
            s = byte > 6u ? __uint_as_float((byte - 6u) << 23) : __uint_as_float(0x10000u << byte); // subnormal below byte 7
            off = s * -8388736.0f;
        }
        if (byte == 255u)
            s = __uint_as_float(0x7fffffffu);
        rare = byte > 230u;
    }
    __device__ __forceinline__ void decode4(unsigned w, float (&v)[4]) const
    {
        if constexpr (FMT == QAGG_MXFP4)
        {
            const float2 lo = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t) (w & 0xffu), __NV_E2M1)));
            const float2 hi = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t) (w >> 8 & 0xffu), __NV_E2M1)));
            v[0] = lo.x * s, v[1] = lo.y * s, v[2] = hi.x * s, v[3] = hi.y * s;
        }
        else
        {
            const unsigned u = w ^ 0x80808080u;
            const float f[4] = {__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)),
                                __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443))};
            if (rare)
            {
                asm volatile(""); // a branch: not four more instructions for everybody
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[i] = (f[i] - 8388736.0f) * s;
            }
            else
            {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[i] = __fmaf_rn(f[i], s, off);
            }
        }
    }
};

// ---- pointwise functions -----------------------------------------------------------------------------------------------------
// In fp32 whatever the type, from the hardware's exponential and reciprocal, whose errors of one or two units of 2^-23 apply to
// e = exp(-|x|) <= 1 and 1 / (1 + e), so that no form here overflows or cancels.  With 16-bit types the exponential's argument is rounded as
// it comes, which is small beside half a step of the type.  fp32 results are good to a few units of the result itself, subnormal ones
// included: there the argument's roundings are made up for.  With expf, normcdff and IEEE quotients the kernels were bound by
// their instructions: gelu of 4096 x 8192 bf16 took 53 us forward and 66 backward for 26 us of HBM traffic each (now 37 and 38), of fp32 88
// and 100 for 46 (now 61 and 64).
template <class T>
__device__ __forceinline__ float exp2_approx(float x)
{
    float r;
    if constexpr (sizeof(T) == 4)
        asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    else
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_approx(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// the smaller of |x| and a limit beyond which exponentials are 0; NaN stays
__device__ __forceinline__ float magnitude_to(float x, float limit)
{
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(x)), "f"(limit));
    return r;
}
// log2(e) in two floats
constexpr float LOG2E = 1.44269502f, LOG2E_REST = 1.92596299e-8f, LN2 = 0.693147182f;
// exp(-k |x|), k = 1 or 2
template <class T>
__device__ __forceinline__ float exp_minus(float k, float x)
{
    if constexpr (sizeof(T) == 4)
    {
        // 2^(high + low) = 2^high + 2^high low ln 2, low being what the first product's rounding left
        const float a = magnitude_to(x, 128.0f) * k, high = a * -LOG2E;
        const float low = __fmaf_rn(a, -LOG2E_REST, __fmaf_rn(a, -LOG2E, -high)), e = exp2_approx<T>(high);
        return __fmaf_rn(e * LN2, low, e);
    }
    else
        return exp2_approx<T>(fabsf(x) * (-LOG2E * k));
}

// Phi(-|x|), the normal distribution's lower tail, and e = exp(-x^2 / 2), as (a1 t + a2 t^2 + ...) e, t = 1 / (1 + c |x|): the form of Abramowitz
// and Stegun, Handbook of Mathematical Functions, 7.1.26, whose own five terms are good to 1.5e-7 of 1 but to 2e-3 of the tail at 5.
// 16-bit types: six terms, within 2.4e-7 near 0 and 2.4e-5 of the tail everywhere (half a step of fp16 is 4.9e-4).  fp32: nine terms,
// fitted for the least largest relative error over |x| = 0 .. 14.5, 3.4e-8.
template <class T>
__device__ __forceinline__ float normal_tail(float x, float& e)
{
    if constexpr (sizeof(T) == 4)
    {
        const float a = magnitude_to(x, 16.0f), s = a * a, high = s * (-0.5f * LOG2E);
        float low = __fmaf_rn(s, -0.5f * LOG2E_REST, __fmaf_rn(s, -0.5f * LOG2E, -high));
        low = __fmaf_rn(__fmaf_rn(a, a, -s), -0.5f * LOG2E, low); // and what the square's left
        e = exp2_approx<T>(high);
        e = __fmaf_rn(e * LN2, low, e);
        const float t = rcp_approx(__fmaf_rn(0.34f, a, 1.0f));
        float p = __fmaf_rn(-0.0258764457f, t, 0.138357103f);
        p = __fmaf_rn(p, t, -0.270871073f);
        p = __fmaf_rn(p, t, 0.199717611f);
        p = __fmaf_rn(p, t, -0.0431062728f);
        p = __fmaf_rn(p, t, 0.114713587f);
        p = __fmaf_rn(p, t, 0.115351707f);
        p = __fmaf_rn(p, t, 0.136092231f);
        p = __fmaf_rn(p, t, 0.135621578f);
        return p * t * e;
    }
    else
    {
        const float t = rcp_approx(__fmaf_rn(0.296f, fabsf(x), 1.0f));
        e = exp2_approx<T>(x * x * (-0.5f * LOG2E));
        float p = __fmaf_rn(-0.0822813883f, t, 0.243228272f);
        p = __fmaf_rn(p, t, -0.045148883f);
        p = __fmaf_rn(p, t, 0.156217799f);
        p = __fmaf_rn(p, t, 0.109275274f);
        p = __fmaf_rn(p, t, 0.118709125f);
        return p * t * e;
    }
}
// Phi(x)
template <class T>
__device__ __forceinline__ float normal(float x, float& e)
{
    const float tail = normal_tail<T>(x, e);
    return x < 0.0f ? tail : 1.0f - tail;
}

template <int ACT, class T>
__device__ __forceinline__ float act_value(float x)
{
    if constexpr (ACT == QAGG_ACT_RELU)
        return x > 0.0f ? x : (x != x ? x : 0.0f);
    else if constexpr (ACT == QAGG_ACT_TANH)
    {
        if constexpr (sizeof(T) == 4)
            return tanhf(x);
        else
        {
            const float e = exp_minus<T>(2.0f, x);
            const float t = (1.0f - e) * rcp_approx(1.0f + e);
            return fabsf(x) < 0.02f ? __fmaf_rn(x * x * x, -0.33333333f, x) : copysignf(t, x);
        }
    }
    else if constexpr (ACT == QAGG_ACT_GELU)
    {
        float e;
        return x * normal<T>(x, e); // not x - x Phi(-x), which is NaN at infinity
    }
    else
    {
        const float e = exp_minus<T>(1.0f, x);
        const float r = rcp_approx(1.0f + e), s = x < 0.0f ? e * r : r; // the sigmoid of x
        return ACT == QAGG_ACT_SIGMOID ? s : x * s;
    }
}
// derivative
template <int ACT, class T>
__device__ __forceinline__ float act_slope(float x)
{
    if constexpr (ACT == QAGG_ACT_RELU)
        return x > 0.0f ? 1.0f : (x != x ? x : 0.0f);
    else if constexpr (ACT == QAGG_ACT_GELU)
    {
        float e;
        const float c = normal<T>(x, e);
        return __fmaf_rn(x * 0.39894228040143268f, e, c);
    }
    else
    {
        const float e = exp_minus<T>(ACT == QAGG_ACT_TANH ? 2.0f : 1.0f, x), r = rcp_approx(1.0f + e);
        const float d = e * r * r; // s (1 - s), s the sigmoid of |x| (tanh: of 2 |x|)
        if constexpr (ACT == QAGG_ACT_SIGMOID)
            return d;
        else if constexpr (ACT == QAGG_ACT_TANH)
            return 4.0f * d;
        else
            return __fmaf_rn(x, d, x < 0.0f ? e * r : r);
    }
}

// Bit pattern, as a float's, of the largest magnitude of a thread's 32 bytes; 16-bit types two at a time.
template <class T>
__device__ __forceinline__ unsigned largest32(const Raw32& raw)
{
    const uint4 r = raw.a, q = raw.b;
    if constexpr (sizeof(T) == 4)
        return max(max(max(r.x & 0x7fffffffu, r.y & 0x7fffffffu), max(r.z & 0x7fffffffu, r.w & 0x7fffffffu)),
                   max(max(q.x & 0x7fffffffu, q.y & 0x7fffffffu), max(q.z & 0x7fffffffu, q.w & 0x7fffffffu)));
    else
        return __vmaxu2(__vmaxu2(__vmaxu2(r.x & 0x7fff7fffu, r.y & 0x7fff7fffu), __vmaxu2(r.z & 0x7fff7fffu, r.w & 0x7fff7fffu)),
                        __vmaxu2(__vmaxu2(q.x & 0x7fff7fffu, q.y & 0x7fff7fffu), __vmaxu2(q.z & 0x7fff7fffu, q.w & 0x7fff7fffu)));
}
template <class T, int THREADS>
__device__ __forceinline__ unsigned largest_of_block(unsigned top)
{
#pragma unroll
    for (int d = 1; d < THREADS; d *= 2)
    {
        const unsigned o = __shfl_xor_sync(0xffffffffu, top, d);
        top = sizeof(T) == 4 ? max(top, o) : __vmaxu2(top, o);
    }
    if constexpr (sizeof(T) == 4)
        return top;
    const unsigned t = max(top & 0xffffu, top >> 16);
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
        return t << 16;
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short) t)));
}

// ---- quantize along the rows; with ACT >= 0 also y = f(x) --------------------------------------------------------------------

template <class T, int FMT, int ACT>
__global__ void __launch_bounds__(MXT, (ACT >= 0 ? 5 : 4)) k_mx_quantize(const T* x, long long ldx, unsigned char* codes, unsigned char* scales, T* y, long long ldy,
                                                     long long M, long long N, int vecX, int vecY)
{
    using S = Shape<T, (ACT >= 0)>;
    __shared__ __align__(16) unsigned char tile[512];
    const long long row0 = (long long) blockIdx.x * MX_TILE;
    const long long col0 = (long long) blockIdx.y * MX_TILE;
    const int tid = threadIdx.x, seg = tid % S::LANES, c0 = tid / S::LANES;
    if (tid < 32)
        reinterpret_cast<uint4*>(tile)[tid] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const long long row = row0 + seg * S::V;
    const int n = row >= M ? 0 : (int) (M - row < S::V ? M - row : S::V);
    const int b = seg * S::V / MX_BLOCK;              // block within the tile
    const bool block = row0 + b * MX_BLOCK < M;       // it exists
    const long long pitch = mx_pitch(M, FMT);
    const T* px = x + (col0 + c0) * ldx + row;
    T* py = y + (col0 + c0) * ldy + row;
    unsigned char* pc = codes + (col0 + c0) * pitch + (FMT == QAGG_MXFP4 ? row / 2 : row);
    const int cols = (int) (N - col0 - c0 < MX_TILE ? N - col0 - c0 : MX_TILE); // columns from this thread's first on
    // value by value: the warp's rows and columns, from its first column on
    __shared__ __align__(32) unsigned char rooms[MXT / 32][1024];
    T* room = reinterpret_cast<T*>(rooms[tid >> 5]);
    const int lane0 = (tid & 31) / S::LANES;
    const int rows = (int) (M - row0 < MX_TILE ? M - row0 : MX_TILE);
    const auto one = [&](const Raw32& raw, int c, unsigned char* at, T* yAt) { // c: column of the tile, from this thread's first
        const BlockEncoder<FMT> enc(largest_of_block<T, S::PARTS>(largest32<T>(raw)));
        float v[S::V];
        unpack32<T>(raw, v);
        if (c < cols && block)
        {
            unsigned w[S::V / 4];
#pragma unroll
            for (int q = 0; q < S::V / 4; ++q)
                w[q] = enc.encode4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
            if constexpr (FMT == QAGG_MXFP4 && S::V == 8)
                *reinterpret_cast<unsigned*>(at) = w[0] | w[1] << 16;
            else if constexpr (FMT == QAGG_MXFP4)
                *reinterpret_cast<uint2*>(at) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
            else if constexpr (S::V == 8)
                *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
            else
                *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
            if (seg % S::PARTS == 0)
                tile[((c0 + c) & 31) * 16 + ((c0 + c) >> 5) * 4 + b] = (unsigned char) enc.byte;
        }
        if constexpr (ACT >= 0)
        {
#pragma unroll
            for (int i = 0; i < S::V; ++i)
                v[i] = act_value<ACT, T>(v[i]);
            if (vecY)
            {
                if (c < cols && block)
                    store32(yAt, v, n, vecY);
            }
            else
                Exchange<T>::put(room, v, yAt - seg * S::V - lane0 * ldy, ldy, rows, cols + lane0 - c);
        }
    };
    if (vecX)
    {
#pragma unroll 1
        for (int h = 0; h < MX_TILE; h += S::FLIGHT * S::COLS)
        {
            Raw32 raw[S::FLIGHT];
#pragma unroll
            for (int p = 0; p < S::FLIGHT; ++p)
                raw[p] = load32(px + p * S::COLS * ldx, h + p * S::COLS < cols ? n : 0, vecX);
#pragma unroll
            for (int p = 0; p < S::FLIGHT; ++p)
                one(raw[p], h + p * S::COLS, pc + p * S::COLS * pitch, py + p * S::COLS * ldy);
            px += S::FLIGHT * S::COLS * ldx;
            py += S::FLIGHT * S::COLS * ldy;
            pc += S::FLIGHT * S::COLS * pitch;
        }
    }
    else
    {
        px -= seg * S::V + lane0 * ldx; // the warp's first
        Exchange<T> next;
        next.fetch(px, ldx, rows, cols + lane0);
#pragma unroll 1
        for (int h = 0; h < MX_TILE; h += S::COLS)
        {
            const Raw32 raw = next.take(room);
            px += S::COLS * ldx;
            if (h + S::COLS < MX_TILE)
                next.fetch(px, ldx, rows, cols + lane0 - h - S::COLS);
            one(raw, h, pc, py);
            py += S::COLS * ldy;
            pc += S::COLS * pitch;
        }
    }
    __syncthreads();
    if (tid < 32)
        reinterpret_cast<uint4*>(scales + ((long long) blockIdx.y * gridDim.x + blockIdx.x) * 512)[tid] = reinterpret_cast<const uint4*>(tile)[tid];
}

// ---- quantize the transpose: blocks along the columns of x -------------------------------------------------------------------
// 128 rows x 64 columns of x, half a scale tile, go through shared memory as they lie (rows contiguous); a thread then takes one packed
// column (a row of x) and a block of its values, which neighbouring lanes read from neighbouring addresses, once for the largest and
// once to encode.  Half tiles and few registers put five CTAs on an SM, so that some load while others encode: 9304 x 2048 fp32 takes
// 19 us where whole tiles took 24.
constexpr int MXT_COLS = 64;
template <class T, int FMT>
__global__ void __launch_bounds__(MXT, 5) k_mx_quantize_t(const T* __restrict__ x, long long ldx, unsigned char* __restrict__ codes,
                                                          unsigned char* __restrict__ scales, long long M, long long N, int vecX)
{
    using S = Shape<T>;
    __shared__ __align__(32) T s[MXT_COLS * MX_TILE + 16];
    auto at = [](int c) { return c * MX_TILE + c / MX_BLOCK * 16; }; // the second block 16 values further: see below
    __shared__ unsigned char bytes[MX_TILE][2];
    // neighbouring CTAs take neighbouring rows of x, which lie together in memory
    const long long tilesR = (M + MX_TILE - 1) / MX_TILE, tileR = blockIdx.x % tilesR, half = blockIdx.x / tilesR;
    const long long col0 = half * MXT_COLS; // columns of x: the packed matrix's rows
    const long long row0 = tileR * MX_TILE; // rows of x: the packed matrix's columns
    const int tid = threadIdx.x;
    if (vecX)
    {
        const int seg = tid % S::LANES;
        const long long row = row0 + seg * S::V;
        const int n = row >= M ? 0 : (int) (M - row < S::V ? M - row : S::V);
#pragma unroll
        for (int c = 0; c < MXT_COLS; c += S::COLS)
        {
            const int k = c + tid / S::LANES;
            const Raw32 r = load32(x + (col0 + k) * ldx + row, col0 + k < N ? n : 0, vecX);
            uint4* to = reinterpret_cast<uint4*>(s + at(k) + seg * S::V);
            to[0] = r.a;
            to[1] = r.b;
        }
    }
    else
    {
        // neighbouring threads neighbouring rows, two columns a turn
        const int r = tid % MX_TILE;
        const T* px = x + (col0 + tid / MX_TILE) * ldx + row0 + r;
#pragma unroll 16
        for (int c = tid / MX_TILE; c < MXT_COLS; c += MXT / MX_TILE, px += MXT / MX_TILE * ldx)
            s[at(c) + r] = row0 + r < M && col0 + c < N ? *px : from_float<T>(0.0f);
    }
    __syncthreads();
    const long long pitch = mx_pitch(N, FMT);
    const int r = tid >> 1, b = tid & 1; // two lanes: 32 (int8: 64) neighbouring bytes; sixteen rows, two blocks: different banks
    unsigned char byte = 0;
    if (row0 + r < M && col0 + b * MX_BLOCK < N)
    {
        const T* v = s + at(b * MX_BLOCK) + r;
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < MX_BLOCK; ++i)
            top = max(top, __float_as_uint(to_float(v[i * MX_TILE])) & 0x7fffffffu);
        const BlockEncoder<FMT> enc(top);
        byte = (unsigned char) enc.byte;
        uint4* to = reinterpret_cast<uint4*>(codes + (row0 + r) * pitch + (col0 + b * MX_BLOCK) / (FMT == QAGG_MXFP4 ? 2 : 1));
        unsigned w[4];
#pragma unroll
        for (int q = 0; q < 8; ++q)
        {
            const T* e = v + 4 * q * MX_TILE;
            const unsigned c = enc.encode4(to_float(e[0]), to_float(e[MX_TILE]), to_float(e[2 * MX_TILE]), to_float(e[3 * MX_TILE]));
            if constexpr (FMT == QAGG_MXFP4)
                w[q / 2] = q & 1 ? w[q / 2] | c << 16 : c;
            else
                w[q & 3] = c;
            if (FMT == QAGG_MXINT8 ? (q & 3) == 3 : q == 7)
                to[FMT == QAGG_MXINT8 ? q / 4 : 0] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    bytes[r][b] = byte;
    __syncthreads();
    if (tid < MX_TILE) // the other half of the tile is another CTA's
        *reinterpret_cast<unsigned short*>(scales + (tileR * mx_scale_tiles(N) + half / 2) * 512 + (tid & 31) * 16 + (tid >> 5) * 4 + (half & 1) * 2) =
            (unsigned short) (bytes[tid][0] | bytes[tid][1] << 8);
}

// ---- unquantize; with ACT >= 0 the backward pass of a pointwise layer: out = in * f'(value) ----------------------------------

template <class T, int FMT, int ACT>
__global__ void __launch_bounds__(MXT, (ACT >= 0 ? 5 : 4)) k_mx_unquantize(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales, const T* in,
                                                       long long ldin, T* out, long long ldout, long long M, long long N, int vecIn, int vecOut)
{
    using S = Shape<T, (ACT >= 0)>;
    __shared__ __align__(16) unsigned char tile[512];
    const long long row0 = (long long) blockIdx.x * MX_TILE;
    const long long col0 = (long long) blockIdx.y * MX_TILE;
    const int tid = threadIdx.x, seg = tid % S::LANES, c0 = tid / S::LANES;
    const long long row = row0 + seg * S::V;
    const int n = row >= M ? 0 : (int) (M - row < S::V ? M - row : S::V);
    const int b = seg * S::V / MX_BLOCK;
    const long long pitch = mx_pitch(M, FMT);
    const unsigned char* pc = codes + (col0 + c0) * pitch + (FMT == QAGG_MXFP4 ? row / 2 : row);
    const T* pi = in + (col0 + c0) * ldin + row;
    T* po = out + (col0 + c0) * ldout + row;
    const int cols = (int) (N - col0 - c0 < MX_TILE ? N - col0 - c0 : MX_TILE); // columns from this thread's first on
    __shared__ __align__(32) unsigned char rooms[MXT / 32][1024];
    T* room = reinterpret_cast<T*>(rooms[tid >> 5]);
    const int lane0 = (tid & 31) / S::LANES;
    const int rows = (int) (M - row0 < MX_TILE ? M - row0 : MX_TILE);
    if (tid < 32)
        reinterpret_cast<uint4*>(tile)[tid] = __ldcs(reinterpret_cast<const uint4*>(scales + ((long long) blockIdx.y * gridDim.x + blockIdx.x) * 512) + tid);
    __syncthreads();
#pragma unroll 1
    for (int h = 0; h < MX_TILE; h += S::FLIGHT * S::COLS)
    {
        unsigned w[S::FLIGHT][S::V / 4];
        Raw32 raw[ACT >= 0 ? S::FLIGHT : 1];
#pragma unroll
        for (int p = 0; p < S::FLIGHT; ++p)
        {
            const bool have = h + p * S::COLS < cols && n > 0;
            const unsigned char* at = pc + p * S::COLS * pitch;
#pragma unroll
            for (int q = 0; q < S::V / 4; ++q)
                w[p][q] = 0;
            if (have)
            {
                if constexpr (FMT == QAGG_MXFP4)
                {
                    uint2 q = make_uint2(0, 0);
                    if constexpr (S::V == 8)
                        q.x = __ldcs(reinterpret_cast<const unsigned*>(at));
                    else
                        q = __ldcs(reinterpret_cast<const uint2*>(at));
                    w[p][0] = q.x & 0xffffu;
                    w[p][1] = q.x >> 16;
                    if constexpr (S::V == 16)
                    {
                        w[p][2] = q.y & 0xffffu;
                        w[p][3] = q.y >> 16;
                    }
                }
                else if constexpr (S::V == 8)
                {
                    const uint2 q = __ldcs(reinterpret_cast<const uint2*>(at));
                    w[p][0] = q.x;
                    w[p][1] = q.y;
                }
                else
                {
                    const uint4 q = __ldcs(reinterpret_cast<const uint4*>(at));
                    w[p][0] = q.x;
                    w[p][1] = q.y;
                    w[p][2] = q.z;
                    w[p][3] = q.w;
                }
            }
            if constexpr (ACT >= 0)
            {
                const T* at = pi + p * S::COLS * ldin;
                if (vecIn)
                    raw[p] = load32(at, have ? n : 0, vecIn);
                else
                {
                    Exchange<T> e;
                    e.fetch(at - seg * S::V - lane0 * ldin, ldin, rows, cols + lane0 - h - p * S::COLS);
                    raw[p] = e.take(room);
                }
            }
        }
#pragma unroll
        for (int p = 0; p < S::FLIGHT; ++p)
        {
            const int c = h + p * S::COLS;
            const BlockDecoder<FMT> dec(tile[((c0 + c) & 31) * 16 + ((c0 + c) >> 5 & 3) * 4 + b]);
            float v[S::V];
#pragma unroll
            for (int q = 0; q < S::V / 4; ++q)
                dec.decode4(w[p][q], reinterpret_cast<float(&)[4]>(v[4 * q]));
            if constexpr (ACT >= 0)
            {
                float g[S::V];
                unpack32<T>(raw[p], g);
#pragma unroll
                for (int i = 0; i < S::V; ++i)
                    v[i] = g[i] * act_slope<ACT, T>(v[i]);
            }
            T* at = po + p * S::COLS * ldout;
            if (vecOut)
            {
                if (c < cols && n > 0)
                    store32(at, v, n, vecOut);
            }
            else
                Exchange<T>::put(room, v, at - seg * S::V - lane0 * ldout, ldout, rows, cols + lane0 - c);
        }
        pc += S::FLIGHT * S::COLS * pitch;
        pi += S::FLIGHT * S::COLS * ldin;
        po += S::FLIGHT * S::COLS * ldout;
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
    const uintptr_t low = (uintptr_t) p | (uintptr_t) (ld * mx_type_bytes(type));
    return (low & 31) == 0 ? VEC32 : (low & 15) == 0 ? VEC16 : 0;
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
        const dim3 tiles = tile_grid(N, M); // of scales; two CTAs each
        k_mx_quantize_t<T, FMT><<<tiles.x * tiles.y * 2, MXT, 0, st>>>(x, ld, (unsigned char*) codes, (unsigned char*) scales, M, N, vec);
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
    const int rc = mx_check_dims("qagg_mx_code_bytes", M, N);
    if (rc)
        return rc;
    if (!format_ok(format))
        return fail(QAGG_EINVAL, "qagg_mx_code_bytes: unknown format");
    return N * mx_pitch(M, format);
}

int64_t qagg_mx_scale_bytes(int64_t M, int64_t N)
{
    const int rc = mx_check_dims("qagg_mx_scale_bytes", M, N);
    if (rc)
        return rc;
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
    if (a == b && lda != ldb && N > 1)
        return fail(QAGG_EINVAL, std::string(who) + ": in place the two ld must be the same");
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
