// Microscaled 4-bit numbers: e2m1 codes, 32 of them along c with a power of two in common (E8M0).
#pragma once
#include "ksmm_common.h"

namespace ksmm {

// The exponent of a block's scale is floor(log2 of its largest magnitude) - 2, so that this one becomes 4 to 7.99 (and is
// rounded to 6 from 5 on: that saturates by a quarter at most), and -120 at least: what is below 2^-122 becomes zero, and
// no scale is a subnormal number.  A block that holds an infinity or a NaN has the scale 255, which stands for NaN.
constexpr int MX_LOWEST = 7, MX_NAN = 255;  // biased by 127

static inline int64_t mx_blocks(int c) { return ((int64_t)c + 31) / 32; }

// magnitude as bits: ordered like the values, infinities and NaNs above
__device__ __forceinline__ uint32_t mx_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// the scale's byte from the bits of the largest magnitude as fp32
__device__ __forceinline__ int mx_scale(uint32_t top)
{
    const int e = (int)(top >> 23);
    return e == 255 ? MX_NAN : e - 2 > MX_LOWEST ? e - 2 : MX_LOWEST;
}
__device__ __forceinline__ float mx_power(int scale) { return __builtin_bit_cast(float, (uint32_t)scale << 23); }

// eight values as codes, the first in the lowest bits: v / 2^e to the nearest e2m1 number, ties to the even code, at most 6
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8], float power)
{
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], power, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], power, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], power, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], power, 3);
    return r;
}
// what eight codes stand for, before their scale
__device__ __forceinline__ void mx_decode8(uint32_t r, float (&v)[8])
{
    const float2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r, 1.f, 1);
    const float2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r, 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r, 1.f, 3);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
}
// the power of two that a scale's byte stands for (0: 2^-127), NaN for 255
__device__ __forceinline__ float mx_scale_value(int scale)
{
    return scale == MX_NAN ? __builtin_nanf("") : scale == 0 ? __builtin_bit_cast(float, 0x00400000u) : mx_power(scale);
}

}  // namespace ksmm
