// Shared by the feed-forward operators (nf_rms_norm.hip, nf_gated_ff*.hip): element types, 16-byte vectors of a row, the 8-bit block format.
#pragma once

#include "nf_common.h"

typedef __bf16 ff_bf16;
typedef _Float16 ff_half;
typedef ff_bf16 ff_bf16x8 __attribute__((ext_vector_type(8)));
typedef ff_half ff_half8 __attribute__((ext_vector_type(8)));
typedef float ff_f32x16 __attribute__((ext_vector_type(16)));
typedef float ff_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned ff_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned ff_u32x2 __attribute__((ext_vector_type(2)));
typedef ff_bf16 ff_bf16x2 __attribute__((ext_vector_type(2)));

// a row's 16-byte vectors need not start at a 16-byte address (odd row lengths): the hardware loads and stores them at any element's address
template <typename T>
struct FfVec;
template <>
struct FfVec<float> {
    static constexpr int N = 4;
    typedef float V __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct FfVec<ff_bf16> {
    static constexpr int N = 8;
    typedef ff_bf16 V __attribute__((ext_vector_type(8), aligned(2)));
};
template <>
struct FfVec<ff_half> {
    static constexpr int N = 8;
    typedef ff_half V __attribute__((ext_vector_type(8), aligned(2)));
};

// elements c .. c + N - 1 of a row of `dim` as float; those behind the row's end are 0
template <typename T>
__device__ __forceinline__ void ff_load_row(const T* row, int c, int dim, float* v) {
    constexpr int N = FfVec<T>::N;
    if (c + N <= dim) {
        const typename FfVec<T>::V t = *reinterpret_cast<const typename FfVec<T>::V*>(row + c);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = (float)t[j];
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = c + j < dim ? (float)row[c + j] : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void ff_store_row(T* row, int c, int dim, const float* v) {
    constexpr int N = FfVec<T>::N;
    if (c + N <= dim) {
        typename FfVec<T>::V t;
#pragma unroll
        for (int j = 0; j < N; ++j) t[j] = (T)v[j];
        *reinterpret_cast<typename FfVec<T>::V*>(row + c) = t;
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (c + j < dim) row[c + j] = (T)v[j];
    }
}

// ---- the 8-bit form: 32 consecutive values of a row share the scale 2^e, e the least whole number with max|block| <= 448 * 2^e (448 is
//      e4m3's largest value), stored as the byte e + 127; a block of zeros has e = -127, one with an infinity or a NaN the byte 255 and all
//      its values are NaN.  This is the format that the matrix instruction scales by itself (v_mfma_scale_f32_*_f8f6f4).
__device__ __forceinline__ unsigned ff_scale_byte(float top) {
    const unsigned u = __float_as_uint(top) & 0x7fffffffu;
    if (u >= 0x7f800000u) return 255u;
    // 448 * 2^e = 1.75 * 2^(e + 8): the exponent field says floor(log2), the mantissa whether 1.75 is enough.  Subnormal maxima are below
    // 448 * 2^-127 and take the least exponent.
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e <= -127 ? 0u : (unsigned)(e + 127);
}
// 2^-e of a scale byte below 255: 2^127 .. 2^-127, the last of them (byte 254) subnormal
__device__ __forceinline__ float ff_scale_inverse(unsigned byte) { return __uint_as_float(byte < 254u ? (254u - byte) << 23 : 0x400000u); }

// float -> e4m3, nearest, ties to even, |v| <= 448 or NaN
__device__ __forceinline__ unsigned ff_e4m3_soft(float v) {
    const unsigned u = __float_as_uint(v), sign = (u >> 24) & 0x80u;
    const float a = __uint_as_float(u & 0x7fffffffu);
    if (!(a <= 464.f)) return sign | 0x7fu;
    int e = (int)((u >> 23) & 0xffu) - 127;
    if (e < -6) e = -6;
    const float m = rintf(ldexpf(a, 3 - e));          // in steps of 2^(e - 3): 8 .. 16 for a normal value, 0 .. 8 below
    const int n = (int)m;
    return sign | (unsigned)(((e + 7) << 3) + n - 8);
}
// four floats -> four e4m3 bytes, the first in the low byte
__device__ __forceinline__ unsigned ff_e4m3x4(float a, float b, float c, float d) {
#if defined(__HIP_DEVICE_COMPILE__)
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    return (unsigned)r;
#else
    return ff_e4m3_soft(a) | ff_e4m3_soft(b) << 8 | ff_e4m3_soft(c) << 16 | ff_e4m3_soft(d) << 24;
#endif
}

// eight e4m3 bytes (the first in lo's low byte) times 2^(byte - 127), in bfloat16: exact, but for what lies below its least value, 2^-133
__device__ __forceinline__ ff_bf16x8 ff_from_e4m3x8(unsigned lo, unsigned hi, unsigned byte) {
#if defined(__HIP_DEVICE_COMPILE__)
    const float s = __uint_as_float(byte << 23);          // the instruction takes the exponent field: 2^(byte - 127)
    ff_bf16x2 v[4];
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
    return __builtin_bit_cast(ff_bf16x8, v);
#else
    ff_bf16x8 v;
    for (int j = 0; j < 8; ++j) {
        const unsigned b = ((j < 4 ? lo : hi) >> (8 * (j & 3))) & 255u, e = (b >> 3) & 15u, m = b & 7u;
        float f = (b & 127u) == 127u || byte == 255u ? NAN : ldexpf(e ? (float)(8 + m) : (float)m, (e ? (int)e : 1) - 10 + (int)byte - 127);
        v[j] = (ff_bf16)(b & 128u ? -f : f);
    }
    return v;
#endif
}

enum { FF_F32 = 0, FF_BF16 = 1, FF_F16 = 2 };
enum { FF_SILU = 0, FF_GELU = 1, FF_RELU = 2 };

// act(g) and act'(g).  The hardware's exponential and reciprocal: good to about (1 + |g|) 2^-23, below what the float32 sums behind g are off by.  gelu's erfc by the
// Chebyshev fit of Numerical Recipes (section 6.2, erfcc: 1.2e-7 of its value everywhere, so that the tail keeps its digits); the library's erff costs four times
// the instructions, and beside the products of a narrow block those are what counts.
__device__ __forceinline__ void ff_act(int act, float g, float& a, float& slope) {
    if (act == FF_SILU) {
        const float s = nf_rcp(1.f + __expf(-g));
        a = g * s;
        slope = s * (1.f + g * (1.f - s));
    } else if (act == FF_GELU) {
        const float z = fabsf(g) * 0.70710678118654752f, t = nf_rcp(fmaf(0.5f, z, 1.f));
        float p = fmaf(t, 0.17087277f, -0.82215223f);
        p = fmaf(t, p, 1.48851587f);
        p = fmaf(t, p, -1.13520398f);
        p = fmaf(t, p, 0.27886807f);
        p = fmaf(t, p, -0.18628806f);
        p = fmaf(t, p, 0.09678418f);
        p = fmaf(t, p, 0.37409196f);
        p = fmaf(t, p, 1.00002368f);
        p = fmaf(t, p, -1.26551223f);
        const float tail = 0.5f * t * __expf(fmaf(-z, z, p));          // half of erfc(z)
        const float cdf = g < 0.f ? tail : 1.f - tail;
        a = g * cdf;
        slope = fmaf(g, 0.39894228040143268f * __expf(-z * z), cdf);
    } else {
        a = g > 0.f ? g : (g != g ? g : 0.f);
        slope = g > 0.f ? 1.f : 0.f;
    }
}

// ---- stores of 4 consecutive values of a row (`left`: how many the row still has)
template <typename T>
__device__ __forceinline__ void ff_put(T* p, int left, const ff_f32x4& v) {
    if (left >= 4) {
        typedef T V4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
        *reinterpret_cast<V4*>(p) = V4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    } else {
        for (int c = 0; c < left; ++c) p[c] = (T)v[c];
    }
}
// the three bf16 parts of a float, each rounded, which makes the third exact.  Where the first would round to an infinity, near the largest float, it is cut off instead: the rest is
// then positive and of 16 bits, and the other two hold it.  An infinity or a NaN keeps its value in the first part and zeros in the others.
__device__ __forceinline__ void ff_split3(float v, ff_bf16* part) {
    const unsigned u = __float_as_uint(v);
    float hi = (float)(ff_bf16)v;
    if (!(fabsf(hi) <= 3.4028235e38f)) hi = __uint_as_float(u & 0xffff0000u);
    if (v != v) hi = v;
    float rest = v - hi;
    if (!(fabsf(v) <= 3.4028235e38f)) rest = 0.f;
    const float mid = (float)(ff_bf16)rest;
    part[0] = (ff_bf16)hi;
    part[1] = (ff_bf16)mid;
    part[2] = (ff_bf16)(rest - mid);
}

// A float16 backward pass multiplies dg and du as float16 values, and with gradients as small as they are without a loss scale these fall among the subnormal ones: at dy = 1e-5 a
// tenth of their bits.  They are linear in dy, so they are made of dy times a power of two and the results divided by it, exactly.  The largest |dy| goes to 2^-4 .. 2^-3: dg and du
// may be 2^19 times as large as it, and are normal numbers down to 2^-11 of it.  Never below 1: larger gradients are as they were.
__device__ __forceinline__ float ff_grad_scale(float top) {
    const unsigned e = (__float_as_uint(top) >> 23) & 255u;
    return top > 0.f && e < 123u ? __uint_as_float((250u - e) << 23) : 1.f;          // 2^(-4 - (e - 127)); zeros, infinities: 1
}
