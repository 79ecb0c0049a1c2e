// Microscaled (MX) number formats, shared by the kernels that write or read
// them (sm_100a).
//
// A block is 32 consecutive elements of a row with one power-of-two scale
// (OCP Microscaling Formats v1.0): value = 2^(scale - 127) * element, the
// elements e4m3 (MXFP8) or e2m1 (MXFP4, element 2i in the low nibble of byte
// i). Conversion, per block: with amax the largest magnitude,
//   scale = max(0, floor(log2(amax)) + 127 - emax),   emax = 8 (e4m3), 2 (e2m1)
//   element = x * 2^(127 - scale), rounded to nearest even, saturating.
// floor(log2(amax)) + 127 is amax's exponent field, so the scale is a
// subtraction on its bits, and multiplying by the inverse scale is exact: the
// element's rounding is the only one. amax below 2^-126 (zero included) gives
// scale 0. A block holding an infinity or NaN gets scale 255 (NaN) and zero
// elements, so the whole block reads as NaN and the fault stays visible.
#pragma once

#include <cstdint>

namespace ds3 {

constexpr int kMxBlock = 32;
constexpr int kMxFp8 = 0, kMxFp4 = 1;             // ds3_cuda_mx_t
constexpr int kMxEmaxFp8 = 8, kMxEmaxFp4 = 2;

// Scale byte of a block from the bits of its largest magnitude (sign cleared).
template <int EMAX>
__device__ __forceinline__ uint32_t mx_scale(uint32_t amax_bits)
{
    const uint32_t e = amax_bits >> 23;
    if (e == 255u) return 255u;
    return e > (uint32_t)EMAX ? e - EMAX : 0u;
}

// 2^(127 - scale), or 0 for the NaN scale (the block's elements become 0).
// scale <= 254 - EMAX otherwise, so the exponent field stays normal.
__device__ __forceinline__ float mx_inv_scale(uint32_t scale)
{
    return scale == 255u ? 0.0f : __uint_as_float((254u - scale) << 23);
}

// 2^(scale - 127); scale 0 is the subnormal 2^-127, 255 is NaN.
__device__ __forceinline__ float mx_scale_value(uint32_t scale)
{
    if (scale == 255u) return __uint_as_float(0x7fc00000u);
    return scale ? __uint_as_float(scale << 23) : __uint_as_float(0x00400000u);
}

// x * inv for a block whose scale is `scale`: 0 where the block is NaN (an
// infinity or NaN times 0 would not be).
__device__ __forceinline__ float mx_scaled(float x, uint32_t scale, float inv)
{
    return scale == 255u ? 0.0f : x * inv;
}

// Two floats to e4m3 (lo in the low byte), four to a word.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d)
{
    return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}

// Eight floats to e2m1, element 0 in the low nibble of byte 0.
__device__ __forceinline__ uint32_t e2m1x8(const float *v)
{
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

}  // namespace ds3
