// vt_mx.cuh -- microscaled block formats and the activations of a learned layer.
//
// A row is cut into blocks of 32 columns; the last block may be short and is
// padded with zeros.  Each block has one exponent byte E and its values are
// small codes times a power of two:
//   8 bits: e = max(floor(log2 max|x|), -120), E = e + 127,
//           code = clamp(rne(x 2^(6 - e)), -127, 127), value = code 2^(e - 6)
//   4 bits: e = max(floor(log2 max|x|) - 2, -126), E = e + 127,
//           code = e2m1(x 2^-e) rounded to nearest even, saturated at 6,
//           value = e2m1 2^e, e2m1 in {0, .5, 1, 1.5, 2, 3, 4, 6} and negatives
// A block that holds a NaN or an infinity has E = 255 and stands for NaN.
// Scaling by a power of two is exact in binary32, so the code's rounding is the
// only rounding, and an 8-bit value fits bfloat16 without another one.  The
// lower bounds of e keep 2^(6 - e), 2^-e and the scales normal numbers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "vt_abi.cuh"

namespace vt {

enum : int { ACT_IDENTITY = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };
constexpr uint32_t MX_BLOCK = 32;

// ---- types ----

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v)
{
    return __bfloat162float(v);
}
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}

// ---- pairs of binary32 values in one 64-bit register ----
//
// sm_100 adds and multiplies two at once, which halves the instructions of the activations; they
// share the issue slots with conversions and shared-memory traffic and are what the fused kernels
// spend most of them on.

typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float x, float y)
{
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpair(f32x2 v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b)
{
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b)
{
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c)
{
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 both(float x) { return pair(x, x); }

// 8 values of a row, as 16-byte words (one, or two for binary32)
template <typename T> struct Vec8 {
    static constexpr int WORDS = sizeof(T) * 8 / 16;
    uint4 w[WORDS];
    __device__ __forceinline__ void load(const T *p)
    {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    }
    __device__ __forceinline__ void store(T *p) const
    {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) reinterpret_cast<uint4 *>(p)[i] = w[i];
    }
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void unpack(float *v) const
    {
        const T *t = reinterpret_cast<const T *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(t[i]);
    }
    __device__ __forceinline__ void pack(const float *v)
    {
        T *t = reinterpret_cast<T *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(v[i]);
    }
};

// 32 bytes at a 32-byte boundary
__device__ __forceinline__ void store32(void *p, const uint32_t *w)
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
__device__ __forceinline__ void load32(const void *p, uint32_t *w)
{
    asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi)
{
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi)
{
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <typename T> __device__ __forceinline__ uint32_t pack2(f32x2 v)
{
    const float2 x = unpair(v);
    return pack2<T>(x.x, x.y);
}
// Binary32 bits of the larger magnitude of two 16-bit numbers whose sign bits are clear
template <typename T> __device__ __forceinline__ uint32_t top_of_pair(uint32_t w);
template <> __device__ __forceinline__ uint32_t top_of_pair<__half>(uint32_t w)
{
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(w & 0xffffu, w >> 16))));
}
template <> __device__ __forceinline__ uint32_t top_of_pair<__nv_bfloat16>(uint32_t w) { return max(w << 16, w & 0xffff0000u); }
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w)
{
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// 32 columns of a row from packed pairs, for rows that start on 32 bytes and hold whole 32-byte pieces,
// which are whole sectors of L2.
template <typename T> __device__ __forceinline__ void store_row32(T *row, uint32_t col, uint32_t cols, const uint32_t *w)
{
    if (col < cols) store32(row + col, w);
    if (col + 16u < cols) store32(row + col + 16u, w + 8);
}
// The same for any rows: a warp's 32 rows by 32 columns (a lane a row of packed pairs) turned in shared memory, so
// that a row's 32 columns are one access.  (A lane storing its own row's columns touches 32 rows an access: 277867 x 195
// in bfloat16 took 557 us that way.)  `rows` of the 32 exist; out is the first one, a matrix of `cols` columns.
constexpr uint32_t TURN_WORDS = 32u * 17u;
template <typename T>
__device__ __forceinline__ void store_turned(T *out, uint32_t rows, uint32_t col, uint32_t cols, const uint32_t *w, uint32_t *turn)
{
    const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) turn[lane * 17u + i] = w[i];
    __syncwarp();
    const unsigned short *from = reinterpret_cast<const unsigned short *>(turn) + lane;
    unsigned short *to = reinterpret_cast<unsigned short *>(out) + col + lane;
    if (col + lane < cols) {
        if (rows == 32u) {
#pragma unroll 8
            for (uint32_t r = 0; r < 32; ++r) to[(uint64_t)r * cols] = from[r * 34u];
        } else {
            for (uint32_t r = 0; r < rows; ++r) to[(uint64_t)r * cols] = from[r * 34u];
        }
    }
    __syncwarp();
}

// ---- formats ----

// Exponent field of a block from the bits of its largest magnitude (sign bit clear).
__device__ __forceinline__ uint32_t mx8_exponent(uint32_t top_bits)
{
    const uint32_t f = top_bits >> 23;
    return f < 7u ? 7u : f;
}
__device__ __forceinline__ uint32_t mx4_exponent(uint32_t top_bits)
{
    const uint32_t f = top_bits >> 23;
    return f == 255u ? 255u : f < 3u ? 1u : f - 2u;
}
// 2^(6 - e) and 2^(e - 6) of an 8-bit block.  E = 255 gives 2^-122 (its codes are set to zero) and NaN.  Below 7,
// which is never written here, the scale is a subnormal number.
__device__ __forceinline__ float mx8_inverse(uint32_t E) { return __uint_as_float((260u - E) << 23); }
__device__ __forceinline__ float mx8_scale(uint32_t E)
{
    return __uint_as_float(E == 255u ? 0x7fc00000u : E < 7u ? 1u << (E + 16u) : (E - 6u) << 23);
}
// 2^-e and 2^e of a 4-bit block.
__device__ __forceinline__ float mx4_inverse(uint32_t E) { return __uint_as_float((254u - E) << 23); }
__device__ __forceinline__ float mx4_scale(uint32_t E)  // E = 0, which is never written here, is 2^-127
{
    return __uint_as_float(E == 255u ? 0x7fc00000u : E == 0u ? 0x00400000u : E << 23);
}
// Four 8-bit codes in a word.  Adding 1.5 2^23 rounds to the nearest whole number, ties to even, and leaves
// it in the low byte: two instructions a pair, where conversions would share the pipe of the activations'
// exponentials and reciprocals, which bounds these kernels next to HBM.
__device__ __forceinline__ uint32_t mx8_codes(f32x2 a, f32x2 b, f32x2 inverse)
{
    const float2 x = unpair(mul2(a, inverse)), y = unpair(mul2(b, inverse));
    const f32x2 magic = both(12582912.0f);
    const float2 u = unpair(add2(pair(fminf(fmaxf(x.x, -127.0f), 127.0f), fminf(fmaxf(x.y, -127.0f), 127.0f)), magic));
    const float2 v = unpair(add2(pair(fminf(fmaxf(y.x, -127.0f), 127.0f), fminf(fmaxf(y.y, -127.0f), 127.0f)), magic));
    return __byte_perm(__byte_perm(__float_as_uint(u.x), __float_as_uint(u.y), 0x0040),
                       __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x0040), 0x5410);
}
// Eight e2m1 codes in a word, the first in the lowest nibble; rounds to nearest even and saturates.
__device__ __forceinline__ uint32_t mx4_word(const f32x2 *v)
{
    const float2 a = unpair(v[0]), b = unpair(v[1]), c = unpair(v[2]), d = unpair(v[3]);
    uint32_t r;
    asm("{\n.reg .b8 p, q, r, s;\n"
        "cvt.rn.satfinite.e2m1x2.f32 p, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 q, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 r, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 s, %8, %7;\n"
        "mov.b32 %0, {p, q, r, s};\n}"
        : "=r"(r) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y), "f"(d.x), "f"(d.y));
    return r;
}
// e2m1 magnitudes doubled are 0 1 2 3 4 6 8 12
__device__ __forceinline__ float mx4_value(uint32_t nibble)
{
    const float m = 0.5f * (float)((0xc8643210u >> ((nibble & 7u) * 4u)) & 15u);
    return nibble & 8u ? -m : m;
}

// ---- activations (binary32 throughout; the caller rounds once) ----

__device__ __forceinline__ float exp2_approx(float x)  // within 2^-22 of 2^x, relative
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float reciprocal_approx(float x)  // within 1 ulp
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b)  // a NaN stays one
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b)
{
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// 1 / (1 + 2^x): the logistic of -x ln 2
__device__ __forceinline__ f32x2 logistic2(f32x2 x)
{
    const float2 a = unpair(x);
    const float2 b = unpair(add2(pair(exp2_approx(a.x), exp2_approx(a.y)), both(1.0f)));
    return pair(reciprocal_approx(b.x), reciprocal_approx(b.y));
}

// gelu_tanh(x) = x logistic(c (x + a x^3)), c = 2 sqrt(2 / pi), a = 0.044715.  Outside [-15, 15]
// the logistic is 0 or 1 in binary32; the bound keeps x^3 finite.
constexpr float GELU_C = 1.5957691216057308f, GELU_A = 0.044715f, LOG2_E = 1.4426950408889634f;

// Value and slope of the activation of two numbers; what is not wanted is not computed.
template <int ACT, bool VALUE, bool SLOPE>
__device__ __forceinline__ void act_pair(f32x2 x, f32x2 &value, f32x2 &slope)
{
    if constexpr (ACT == ACT_RELU) {
        const float2 v = unpair(x);
        value = pair(max_nan(v.x, 0.0f), max_nan(v.y, 0.0f));
        if constexpr (SLOPE)  // of a zero itself, and of a NaN
            slope = pair(v.x > 0.0f ? 1.0f : v.x < 0.0f ? 0.0f : v.x, v.y > 0.0f ? 1.0f : v.y < 0.0f ? 0.0f : v.y);
    } else if constexpr (ACT == ACT_SILU) {
        const f32x2 p = logistic2(mul2(x, both(-LOG2_E)));
        value = mul2(x, p);
        if constexpr (SLOPE) slope = fma2(value, fma2(p, both(-1.0f), both(1.0f)), p);
    } else if constexpr (ACT == ACT_GELU) {
        const float2 v = unpair(x);
        const f32x2 c = pair(min_nan(max_nan(v.x, -15.0f), 15.0f), min_nan(max_nan(v.y, -15.0f), 15.0f));
        const f32x2 cc = mul2(c, c);
        const f32x2 p = logistic2(mul2(c, fma2(cc, both(-LOG2_E * GELU_C * GELU_A), both(-LOG2_E * GELU_C))));
        if constexpr (VALUE) value = mul2(x, p);
        if constexpr (SLOPE)
            slope = fma2(mul2(mul2(c, p), fma2(p, both(-1.0f), both(1.0f))), fma2(cc, both(3.0f * GELU_C * GELU_A), both(GELU_C)), p);
    } else {
        value = x;
        slope = both(1.0f);
    }
}
template <int ACT> __device__ __forceinline__ f32x2 act_value2(f32x2 x)
{
    f32x2 v, s;
    act_pair<ACT, true, false>(x, v, s);
    return v;
}
template <int ACT> __device__ __forceinline__ f32x2 act_slope2(f32x2 x)
{
    f32x2 v, s;
    act_pair<ACT, false, true>(x, v, s);
    return s;
}

// Two of a word's four 8-bit codes (bytes i and i + 1, sign bits turned) as numbers: a turned
// byte under the exponent of 2^23 is 2^23 + 128 + code.
__device__ __forceinline__ f32x2 code_pair(uint32_t turned, int i)
{
    return add2(pair(__uint_as_float(__byte_perm(turned, 0x4b000000u, 0x7440u | i)),
                     __uint_as_float(__byte_perm(turned, 0x4b000000u, 0x7440u | (i + 1)))),
                both(-8388736.0f));
}

// ---- dispatch: one instantiation per activation / type ----

template <int V> struct IntC { static constexpr int value = V; };
template <typename T> struct TypeC { using type = T; };

template <typename F> inline vt_status with_act(int act, F f)
{
    switch (act) {
    case ACT_IDENTITY: return f(IntC<ACT_IDENTITY>());
    case ACT_RELU: return f(IntC<ACT_RELU>());
    case ACT_SILU: return f(IntC<ACT_SILU>());
    case ACT_GELU: return f(IntC<ACT_GELU>());
    }
    return set_error(VT_ERR_INVALID, "unknown activation %d", act);
}

template <typename F> inline vt_status with_type(int dtype, F f)
{
    switch (dtype) {
    case VT_F32: return f(TypeC<float>());
    case VT_F16: return f(TypeC<__half>());
    case VT_BF16: return f(TypeC<__nv_bfloat16>());
    }
    return set_error(VT_ERR_INVALID, "unknown element type %d", dtype);
}

template <typename F> inline vt_status with_type16(int dtype, F f)
{
    switch (dtype) {
    case VT_F16: return f(TypeC<__half>());
    case VT_BF16: return f(TypeC<__nv_bfloat16>());
    }
    return set_error(VT_ERR_INVALID, "products take binary16 or bfloat16 (type %d given)", dtype);
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned32(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; }
// Whether all addresses (nulls among them) are a T's: the kernels touch nothing narrower
template <typename T, typename... P> inline bool on_elements(const P *...p)
{
    return ((reinterpret_cast<uintptr_t>(p) | ...) & (sizeof(T) - 1u)) == 0;
}
inline uint32_t mx_blocks(uint32_t cols) { return cols / MX_BLOCK + (cols % MX_BLOCK != 0); }
inline int sm_count()  // of the current device, asked for once
{
    static std::atomic<int> known[64];
    int dev = 0, sms = 0;
    cudaGetDevice(&dev);
    std::atomic<int> &k = known[dev & 63];
    if ((sms = k.load(std::memory_order_relaxed)) == 0) {
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) sms = 148;
        else k.store(sms, std::memory_order_relaxed);
    }
    return sms;
}

}  // namespace vt
