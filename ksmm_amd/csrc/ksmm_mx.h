// Microscaled 4-bit numbers: e2m1 codes, 32 of them along c with a power of two in common (E8M0).
#pragma once
#include "ksmm_common.h"

namespace ksmm {

// The exponent of a block's scale is floor(log2 of its largest magnitude) - 2, so that this one becomes 4 to 7.99 (and is
// rounded to 6 from 5 on: that saturates by a quarter at most), and -120 at least: what is below 2^-122 becomes zero, and
// no scale is a subnormal number.  A block that holds an infinity or a NaN has the scale 255, which stands for NaN.
constexpr int MX_LOWEST = 7, MX_NAN = 255;  // biased by 127

static inline int64_t mx_blocks(int c) { return ((int64_t)c + 31) / 32; }

// magnitudes as bits: ordered like the values, infinities and NaNs above
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

// ---- reading an operand ---------------------------------------------------------------------------------
// A thread takes blocks of one place kb that lie side by side in memory: those of D consecutive d_i (batch-size-first), or of D
// consecutive rows (batch-size-last).  Their 32 values of c are `step` elements apart; where that is D, they are one run of 32 * D.
typedef uint32_t uint4_any __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at an element's alignment

template <typename T, int D> struct MxGroup {
    T v[32 * D];  // value k of block j at k * D + j
};

// count: of the 32 values those that are there, here: of the D blocks; the rest is zeros
template <typename T, int D> __device__ __forceinline__ void mx_load(MxGroup<T, D> &g, const T *x, int64_t step, int count, int here)
{
    constexpr int E = 16 / (int)sizeof(T);  // values a vector
    if (step == D && here == D) {
        const int have = count * D;
#pragma unroll
        for (int j = 0; j < 32 * D / E; ++j) {
            if ((j + 1) * E <= have) {
                const uint4_t q = *(const uint4_any *)(x + j * E);
                __builtin_memcpy(&g.v[j * E], &q, 16);
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i) g.v[j * E + i] = j * E + i < have ? x[j * E + i] : (T)0;
            }
        }
    } else if (here == D) {
        struct __attribute__((packed, aligned(sizeof(T)))) Run {
            T e[D];
        };
#pragma unroll
        for (int k = 0; k < 32; ++k) {
            Run r = {};
            if (k < count) r = *(const Run *)(x + k * step);
#pragma unroll
            for (int j = 0; j < D; ++j) g.v[k * D + j] = r.e[j];
        }
    } else {
#pragma unroll
        for (int k = 0; k < 32; ++k)
#pragma unroll
            for (int j = 0; j < D; ++j) g.v[k * D + j] = k < count && j < here ? x[k * step + j] : (T)0;
    }
}

// block j of the group: its codes and its scale's byte
template <typename T, int D> __device__ __forceinline__ int mx_quantize(const MxGroup<T, D> &g, int j, uint4_t &code)
{
    uint32_t top = 0;
    if constexpr (sizeof(T) == 2) {
        uint16_t most = 0;
#pragma unroll
        for (int k = 0; k < 32; ++k) {
            const uint16_t bits = __builtin_bit_cast(uint16_t, g.v[k * D + j]) & 0x7fffu;
            most = bits > most ? bits : most;
        }
        top = mx_bits((float)__builtin_bit_cast(half_t, most));
    } else {
#pragma unroll
        for (int k = 0; k < 32; ++k) {
            const uint32_t bits = mx_bits(g.v[k * D + j]);
            top = bits > top ? bits : top;
        }
    }
    const int scale = mx_scale(top);
    const float power = mx_power(scale);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        uint32_t r = 0;
        if constexpr (sizeof(T) == 2) {
            const T *v = &g.v[q * 8 * D + j];
            r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, half2_t{v[0], v[D]}, power, 0);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, half2_t{v[2 * D], v[3 * D]}, power, 1);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, half2_t{v[4 * D], v[5 * D]}, power, 2);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, half2_t{v[6 * D], v[7 * D]}, power, 3);
        } else {
            const float *v = (const float *)&g.v[q * 8 * D + j];
            const float e[8] = {v[0], v[D], v[2 * D], v[3 * D], v[4 * D], v[5 * D], v[6 * D], v[7 * D]};
            r = mx_encode8(e, power);
        }
        code[q] = scale == MX_NAN ? 0 : r;
    }
    return scale;
}

// What the product kernels are given.
struct MxProduct {
    const void *x;
    const uint8_t *x_scales;  // null: x has values
    const uint8_t *w, *w_scales;
    const void *bias;
    void *y;
    int64_t batch;
    int a, b, c, d, cb;
    int slots;             // of 16 bytes in LDS for a row's codes, odd
    int runs, units;       // runs of D consecutive d_i, and a times as many units of work
    int units_per;         // of them a workgroup takes
    int b_tiles, tiles_per;  // tiles of 32 outputs, and those a workgroup takes
    int splits, unit_groups;
    int64_t tiles, token_tiles;  // (without LDS)
};
int mx_run_half(MxProduct p, bool last, bool gated, int act, hipStream_t s);
int mx_run_float(MxProduct p, bool last, bool gated, int act, hipStream_t s);
// whether an operand's codes fit LDS, so that it is quantised there
bool mx_in_lds(int c, int d, int bs_last);

}  // namespace ksmm
