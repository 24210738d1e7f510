// Decoding of 4-bit values to BF16, exact, eight at a time.
#pragma once

#include "bsq_fp4.cuh"

namespace bsq {
namespace {

constexpr float kNvHold = 4096.0f;                               // NVFP4: decoded values are held 2^12 smaller

__device__ __forceinline__ unsigned mul_bf16x2(unsigned a, unsigned b) {
    unsigned r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Eight codes to BF16, times a scale.  Sign and the three magnitude bits are moved to where BF16 has its sign, the last two bits of its exponent and
// the first of its mantissa: read as BF16 that is the element times 2^-126 (also for 0 and 0.5, which are subnormal in both), and multiplying brings it
// back.  Word i holds elements i and i + 4: columns of a group of 8 come out in the order 0 4 1 5 2 6 3 7, which the epilogue undoes for nothing.
// ONE (MXFP4): the factor holds the 2^126 as well, which scales up to 2 leave room for.
template <int FMT, bool ONE = false> __device__ __forceinline__ uint4 decode8(unsigned x, unsigned scale2) {
    // (shifts to the left, which go to the multiply pipe: the integer pipe with its half rate is what decoding is short of)
    const unsigned y = x >> 6;
    unsigned w[4];
    w[0] = ((x << 12) & 0x80008000u) | ((x << 6) & 0x01C001C0u);
    w[1] = ((x << 8) & 0x80008000u) | ((x << 2) & 0x01C001C0u);
    w[2] = ((x << 4) & 0x80008000u) | ((y << 4) & 0x01C001C0u);
    w[3] = (x & 0x80008000u) | (y & 0x01C001C0u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (FMT == kMxFp4 && !ONE) w[i] = mul_bf16x2(w[i], 0x7E807E80u);  // 2^126: the element itself, exact; the scale's range needs a product of its own
        w[i] = mul_bf16x2(w[i], scale2);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// The factors of decode8 from two scale bytes (each in the low byte of its word): the first in the low half.  NVFP4: s * 2^(126 - 12), exact in BF16.
template <int FMT> __device__ __forceinline__ unsigned decode_scales(unsigned b0, unsigned b1) {
    if (FMT == kMxFp4) {
        const unsigned h0 = b0 == 0 ? 0x0040u : b0 == 255 ? 0x7FFFu : b0 << 7, h1 = b1 == 0 ? 0x0040u : b1 == 255 ? 0x7FFFu : b1 << 7;
        return h0 | (h1 << 16);
    }
    unsigned f;
    asm("{\n\t.reg .b16 e;\n\tcvt.u16.u32 e, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, e;\n\t}" : "=r"(f) : "r"((b0 | (b1 << 8)) & 0x7f7fu));
    const float2 s = __half22float2(*reinterpret_cast<const __half2 *>(&f));
    return pack_pair<kBf16>(s.x * 2.076918743413931e34f, s.y * 2.076918743413931e34f);
}

// ... of MXFP4 bytes up to 128 (scales up to 2), times 2^126
__device__ __forceinline__ unsigned decode_scales_one(unsigned b0, unsigned b1) {
    return (b0 ? (b0 + 126u) << 7 : 0x3F00u) | (b1 ? (b1 + 126u) << 23 : 0x3F000000u);
}

}  // namespace
}  // namespace bsq
