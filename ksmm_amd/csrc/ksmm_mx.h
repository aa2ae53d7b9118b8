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

// t / d for 0 <= t, t d < 2^32 (m is less than d 2^-32 too large): a multiplication where the compiler takes 30 instructions
struct MxDiv {
    uint32_t d, m;
    MxDiv() = default;
    __host__ __device__ __forceinline__ explicit MxDiv(int d) : d((uint32_t)d), m(0xffffffffu / (uint32_t)d + 1) {}
    __device__ __forceinline__ int operator()(int t) const { return d == 1 ? t : (int)__umulhi((uint32_t)t, m); }
};

// ---- reading an operand ---------------------------------------------------------------------------------
// A thread takes the blocks of one place kb of D consecutive d_i (batch-size-last D is 1): their 32 values of c are `step` elements
// apart, and one run of 32 * D where that is D.
typedef uint32_t uint4_any __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at an element's alignment

template <typename T, int D> struct MxGroup {
    T v[32 * D];  // value k of block j at k * D + j
};

// count (1 ..) of the 32 values are there.  Those behind are read as the last ones that are: that changes no largest magnitude, and
// mx_quantize leaves them out of the codes; a branch around each load would cost more than the loads.
template <typename T, int D> __device__ __forceinline__ void mx_load(MxGroup<T, D> &g, const T *x, int64_t step, int count)
{
    constexpr int E = 16 / (int)sizeof(T);  // values a vector
    struct __attribute__((packed, aligned(sizeof(T)))) Run {
        T e[D];
    };
    int last = (count < 32 ? count : 32) - 1;
    asm volatile("" : "+v"(last));  // (offsets of 32 loads are not to be kept in registers from one step of rows to the next)
    // (a vector that is read in another's place has the same blocks in the same places: not so where D does not divide it)
    if (step == D && (E % D == 0 ? (last + 1) * D % E == 0 : last == 31)) {
        const int end = (last + 1) * D / E - 1;
#pragma unroll
        for (int j = 0; j < 32 * D / E; ++j) {
            const uint4_t q = *(const uint4_any *)(x + (j < end ? j : end) * E);
            __builtin_memcpy(&g.v[j * E], &q, 16);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 32; ++k) {
            const Run r = *(const Run *)(x + (k < last ? k : last) * step);
#pragma unroll
            for (int j = 0; j < D; ++j) g.v[k * D + j] = r.e[j];
        }
    }
}

// block j of the group: its codes and its scale's byte
template <typename T, int D> __device__ __forceinline__ int mx_quantize(const MxGroup<T, D> &g, int j, int count, uint4_t &code)
{
    uint32_t top = 0;
    if constexpr (sizeof(T) == 2) {
        typedef uint16_t ushort2_v __attribute__((ext_vector_type(2)));
        ushort2_v most = {0, 0};
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
            const ushort2_v bits = {__builtin_bit_cast(uint16_t, g.v[k * D + j]), __builtin_bit_cast(uint16_t, g.v[(k + 1) * D + j])};
            most = __builtin_elementwise_max(most, bits & (uint16_t)0x7fff);
        }
        top = mx_bits((float)__builtin_bit_cast(half_t, (uint16_t)(most[0] > most[1] ? most[0] : most[1])));
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
        const int there = count - 8 * q;
        const uint32_t mask = scale == MX_NAN || there <= 0 ? 0u : there >= 8 ? ~0u : (1u << 4 * there) - 1;
        code[q] = r & mask;
    }
    return scale;
}

// ---- a quarter of a block a lane: 8 values of D consecutive d_i that are one run in memory.  Lanes that follow one another read
// bytes that do, where a block a lane has 64 lines of the cache in every load (25088 x 768 of (1,192,768,2): 31 us for 15)
template <typename T, int D> struct MxQuarter {
    T v[8 * D];
};
// count of the 8 values are there (may be none, or more); the rest is zeros.  (Values that are not are read as the last that is, in this
// quarter or one before: a branch around each load is a wait of its own)
template <typename T, int D> __device__ __forceinline__ void mx_load(MxQuarter<T, D> &g, const T *x, int count)
{
    constexpr int E = 16 / (int)sizeof(T);
    if (count >= 8) {
#pragma unroll
        for (int j = 0; j < 8 * D / E; ++j) {
            const uint4_t q = *(const uint4_any *)(x + j * E);
            __builtin_memcpy(&g.v[j * E], &q, 16);
        }
    } else {
        struct __attribute__((packed, aligned(sizeof(T)))) Run {
            T e[D];
        } r[8];
        asm volatile("" : "+v"(count));  // (as above)
#pragma unroll
        for (int k = 0; k < 8; ++k) r[k] = *(const Run *)(x + (k < count ? k : count - 1) * D);
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int j = 0; j < D; ++j) g.v[k * D + j] = k < count ? r[k].e[j] : (T)0;
    }
}
// its part of the codes of the four lanes' block j, and the scale's byte (in each of them; all four take part)
template <typename T, int D> __device__ __forceinline__ int mx_quantize(const MxQuarter<T, D> &g, int j, uint32_t &code)
{
    uint32_t top = 0;
    if constexpr (sizeof(T) == 2) {
        uint16_t most = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint16_t bits = __builtin_bit_cast(uint16_t, g.v[k * D + j]) & 0x7fffu;
            most = bits > most ? bits : most;
        }
        top = most;
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t bits = mx_bits(g.v[k * D + j]);
            top = bits > top ? bits : top;
        }
    }
    top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xb1, 0xf, 0xf, true));  // lanes 1 0 3 2
    top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4e, 0xf, 0xf, true));  // 2 3 0 1
    if constexpr (sizeof(T) == 2) top = mx_bits((float)__builtin_bit_cast(half_t, (uint16_t)top));
    const int scale = mx_scale(top);
    const float power = mx_power(scale);
    uint32_t r = 0;
    if constexpr (sizeof(T) == 2) {
        const T *v = &g.v[j];
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, half2_t{v[0], v[D]}, power, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, half2_t{v[2 * D], v[3 * D]}, power, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, half2_t{v[4 * D], v[5 * D]}, power, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, half2_t{v[6 * D], v[7 * D]}, power, 3);
    } else {
        const float *v = (const float *)&g.v[j];
        const float e[8] = {v[0], v[D], v[2 * D], v[3 * D], v[4 * D], v[5 * D], v[6 * D], v[7 * D]};
        r = mx_encode8(e, power);
    }
    code = scale == MX_NAN ? 0u : r;
    return scale;
}

// What the product kernels are given.
struct MxProduct {
    const void *x;
    const uint8_t *x_scales;  // null: x has values
    uint8_t *codes_out, *scales_out;  // where these go as codes, or null
    const uint8_t *w, *w_scales;
    const void *bias;
    void *y;
    const void *dy;  // (gradients only)
    bool finite;     // of codes, without an activation: results beyond the type's range are its largest (gradients only)
    uint32_t first;  // workgroup of the launch, of all
    int64_t batch;
    int a, b, c, d, cb;
    int slots;                    // of 16 bytes in LDS for a row's codes, odd
    int run_d, runs, units;       // d_i of a unit of work, units of an a_i and of all
    int b_tiles, tiles_per;       // tiles of 32 outputs, and those a workgroup takes
    int chunk_tiles, splits;      // tiles at a time, and workgroups that share the tiles
    int64_t tiles, token_tiles;  // (without LDS); steps of rows
    int raw_rows, raw_pitch;     // rows at a time whose values go through LDS on their way to codes (0: straight), and values from one to the next
    int tile_rows, wave_tiles;   // rows a step, and of a workgroup's waves those that lie along the outputs
    int row_splits;              // workgroups that share the steps
    MxDiv by_cb, by_run_d;
};
int mx_slope_half(const MxProduct &p, bool last, bool gated, int act, hipStream_t s);
int mx_slope_float(const MxProduct &p, bool last, bool gated, int act, hipStream_t s);
// by the type of x and y, the layout and whether two projections make one output
int mx_half_first_plain(const MxProduct &p, int act, hipStream_t s);
int mx_half_first_gated(const MxProduct &p, int act, hipStream_t s);
int mx_half_last_plain(const MxProduct &p, int act, hipStream_t s);
int mx_half_last_gated(const MxProduct &p, int act, hipStream_t s);
int mx_float_first_plain(const MxProduct &p, int act, hipStream_t s);
int mx_float_first_gated(const MxProduct &p, int act, hipStream_t s);
int mx_float_last_plain(const MxProduct &p, int act, hipStream_t s);
int mx_float_last_gated(const MxProduct &p, int act, hipStream_t s);

// d_i that a thread converts together: all of up to four, else four, two or one (three of six would be runs of 6 bytes: 25088 rows of (6,64,6) in
// fp16 81 us to codes and 106 back for 51 and 59)
inline int mx_run_of(int d) { return d <= 4 ? d : d % 4 == 0 ? 4 : d % 2 == 0 ? 2 : 1; }

// Weights from the caches: d_i of a workgroup (16 of more are pieces of 32 bytes at least), tiles of outputs at a time (a wave each,
// or with d_i of their own some), and LDS
constexpr int MX_WAVES = 8;
constexpr int MX_LINE = 144, MX_STAGE = 32 * MX_LINE;  // of a wave for its results: 128 bytes of 32 lines, 16 between them for the banks' sake
constexpr int64_t MX_LDS_MOST = 80 * 1024;             // two workgroups a compute unit
constexpr int64_t MX_LDS_ALL = 160 * 1024;
inline int mx_unit_of(int d, bool last) { return last ? 1 : d <= 16 ? d : 16; }
inline int mx_chunk_of(int unit, bool last) { return last || unit == 1 ? MX_WAVES : unit < MX_WAVES ? MX_WAVES / unit : 1; }
inline int64_t mx_codes_lds(int tt, int c, int d, bool last)
{
    const int64_t cb = mx_blocks(c), unit = mx_unit_of(d, last), rows = 32 * tt;
    return unit * rows * (cb | 1) * 16 + (unit * rows * cb + 15) / 16 * 16;
}
// Five d_i and more go through LDS on their way to codes: bytes of a row (16 more than its vectors: rows meet other banks), and rows at a
// time, all of them or as few times as two workgroups a compute unit allow
inline int64_t mx_raw_row(int c, int d, int size) { return ((int64_t)mx_unit_of(d, false) * c * size + 15) / 16 * 16 + 16; }
inline int mx_raw_rows(int tt, int c, int d, int size)
{
    const int64_t fit = (MX_LDS_MOST - mx_codes_lds(tt, c, d, false)) / mx_raw_row(c, d, size), rows = 32 * tt;
    const int64_t times = fit < 1 ? rows : (rows + fit - 1) / fit;
    return (int)((rows + times - 1) / times);
}
inline int64_t mx_wide_lds(int tt, int c, int d, int size, bool last)
{
    if (last) return mx_codes_lds(tt, c, d, last) + MX_WAVES * MX_STAGE;
    const int64_t unit = mx_unit_of(d, last), results = 32 * tt * (mx_chunk_of((int)unit, last) * 32 * unit * size + 4);
    const int64_t raw = d > 4 ? mx_raw_rows(tt, c, d, size) * mx_raw_row(c, d, size) : 0;
    return mx_codes_lds(tt, c, d, last) + (results > raw ? results : raw);
}
// whether an operand's codes fit LDS, so that it is quantised there
inline bool mx_in_lds(int c, int d, int size, bool last) { return mx_wide_lds(1, c, d, size, last) <= MX_LDS_ALL; }

}  // namespace ksmm
