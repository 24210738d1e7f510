// Device helpers for microscaled 4-bit matrices: conversions, block scales, loads of 16- and 32-bit elements.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bsq_device.cuh"
#include "bsq_fp4.hpp"

namespace bsq {
namespace {

// Elements of a floating type as 32-bit words: what the largest magnitude and the test for Inf / NaN need.  larger(a, b): the larger magnitude of each element of
// a and b, NaN where there is one; the sign bits of its result say nothing (one instruction, where clearing the sign and comparing take two).
// Adding kCarry to a magnitude sets the top bit for Inf and NaN and for nothing else.
template <int TYPE> struct Words;
template <> struct Words<kF32> {
    static constexpr int kPer = 1;
    static constexpr unsigned kAbs = 0x7fffffffu, kCarry = 0x00800000u, kTop = 0x80000000u;
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
        float r;
        asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
        return __float_as_uint(r);
    }
    static __device__ __forceinline__ unsigned drop(unsigned w) { return (w & kAbs) >= 0x7f800000u ? 0u : w & kAbs; }
    static __device__ __forceinline__ float top(unsigned m) { return __uint_as_float(m & kAbs); }
};
template <> struct Words<kBf16> {
    static constexpr int kPer = 2;
    static constexpr unsigned kAbs = 0x7fff7fffu, kCarry = 0x00800080u, kTop = 0x80008000u;
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
        unsigned r;
        asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ unsigned drop(unsigned w) {
        return ((w & 0x7fffu) >= 0x7f80u ? 0u : (w & 0x7fffu)) | ((w >> 16 & 0x7fffu) >= 0x7f80u ? 0u : (w & 0x7fff0000u));
    }
    static __device__ __forceinline__ float top(unsigned m) { return __uint_as_float(max(m & 0x7fffu, m >> 16 & 0x7fffu) << 16); }
};
template <> struct Words<kF16> {
    static constexpr int kPer = 2;
    static constexpr unsigned kAbs = 0x7fff7fffu, kCarry = 0x04000400u, kTop = 0x80008000u;
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
        unsigned r;
        asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ unsigned drop(unsigned w) {
        return ((w & 0x7fffu) >= 0x7c00u ? 0u : (w & 0x7fffu)) | ((w >> 16 & 0x7fffu) >= 0x7c00u ? 0u : (w & 0x7fff0000u));
    }
    static __device__ __forceinline__ float top(unsigned m) { return __half2float(__ushort_as_half((unsigned short)max(m & 0x7fffu, m >> 16 & 0x7fffu))); }
};
template <int TYPE> __device__ __forceinline__ bool not_finite(unsigned w) { return (((w & Words<TYPE>::kAbs) + Words<TYPE>::kCarry) & Words<TYPE>::kTop) != 0; }

// The elements of a word
template <int TYPE> __device__ __forceinline__ float word_elem(unsigned w, int i) {
    if (TYPE == kF32) return __uint_as_float(w);
    if (TYPE == kBf16) return __uint_as_float(i ? (w & 0xffff0000u) : (w << 16));
    return __half2float(__ushort_as_half((unsigned short)(i ? (w >> 16) : (w & 0xffffu))));
}

// Eight values to the nearest e2m1, ties to even, saturated; element i in bits 4 i.
__device__ __forceinline__ unsigned e2m1_pack8(const float (&v)[8]) {
    unsigned r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// Eight codes as four pairs of FP16 (exact)
__device__ __forceinline__ void e2m1_unpack8(unsigned codes, unsigned (&h)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
}
// The nearest E4M3 byte of x >= 0, ties to even, saturated at 448
__device__ __forceinline__ unsigned ue4m3_byte(float x) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(x));
    return r & 0xffu;
}
// A block scale's value; NaN for the bytes that mean NaN
template <int FMT> __device__ __forceinline__ float fp4_scale_value(unsigned byte) {
    if (FMT == kMxFp4) return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fffffffu : byte << 23);
    return (byte & 0x7fu) == 0x7fu ? __uint_as_float(0x7fffffffu) : e4m3_decode(byte & 0x7fu);
}

// The exponent of an NVFP4 matrix scale: the smallest t with amax <= 2688 * 2^t (2688 = 448 * 6, the largest block scale times the
// largest element), kept where 2^t and its products with block scales and reciprocals stay normal.  Powers of two keep every
// decision of the quantiser exact: halfway points times block scales have 7 significant bits, and scaling by 2^t adds none.
__device__ __forceinline__ int nvfp4_matrix_exp(float amax) {
    const unsigned b = __float_as_uint(amax);
    if (!(amax > 0.0f) || b >= 0x7f800000u) return 0;
    const int t = (int)(b >> 23) - 127 - 11 + ((b & 0x7fffffu) > 0x280000u ? 1 : 0);     // 2688 = 1.3125 * 2^11
    return min(max(t, -110), 117);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }   // -126 <= e <= 127

__device__ __forceinline__ void ld_words8(const void *p, unsigned (&w)[8]) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
}
__device__ __forceinline__ void st_words8(void *p, const unsigned (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// Two FP32 values in one word of a 16-bit type
template <int TYPE> __device__ __forceinline__ unsigned pack_pair(float lo, float hi) {
    if (TYPE == kBf16) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const unsigned *>(&r);
    }
    const __half2 r = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned *>(&r);
}
template <int TYPE> __device__ __forceinline__ void store_elem(void *out, uint64_t i, float v) {
    if (TYPE == kF32) static_cast<float *>(out)[i] = v;
    else if (TYPE == kBf16) static_cast<__nv_bfloat16 *>(out)[i] = __float2bfloat16_rn(v);
    else static_cast<__half *>(out)[i] = __float2half_rn(v);
}

}  // namespace
}  // namespace bsq
