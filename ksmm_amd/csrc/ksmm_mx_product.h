// Products of microscaled 4-bit numbers, quantised on the way: the kernels, for one type of x and y.
//
// A workgroup takes rows of the batch and a unit of work: one a_i and D consecutive d_i (batch-size-last one d_i).  It quantises its
// rows of x into LDS, where they take 17 bytes for 32 values, and its waves multiply them with tiles of 32 outputs, whose codes are in
// registers (ks_mx_held_kernel) or come from the caches (ks_mx_wide_kernel).  x quantised in a launch of its own would be written
// and read once more, and again by every tile of outputs: (1,768,192,2) gated fp16, 25088 rows 135 us for 82 of the same kernel.
// Every row of a tile's operand is read where the lane that holds the result wants it: row 8j + 4h + i of a tile is its row
// 16h + 4j + i, so that a lane ends up with 16 consecutive outputs of a row of the batch (batch-size-last: 16 consecutive rows of
// one output), which with those of all D leave as whole vectors.
//
// What bounds them: at full batches HBM and waits at the barrier of the two roles, never the matrix cores (0.1 of their time).
// (1,768,192,2) gated fp16, 25088 rows: 96 MB in 29 us, 3.4 TB/s; (4,192,192,1) fp16: 39 MB in 15, (12,64,64,1) 77 MB in 14, a copy's rate.
#pragma once
#include <algorithm>
#include <type_traits>

#include "ksmm_act.h"
#include "ksmm_mx.h"

namespace ksmm {

namespace {

typedef int int8_v __attribute__((ext_vector_type(8)));

__device__ __forceinline__ int8_v mx_widen(uint4_t v) { return int8_v{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; }
__device__ __forceinline__ float16_t mx_mfma(uint4_t a, int sa, uint4_t b, int sb, float16_t c)
{
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_widen(a), mx_widen(b), c, 4, 4, 0, sa, 0, sb);
}

// N elements to p, as 16-byte stores at the elements' alignment
template <typename T, int N> __device__ __forceinline__ void mx_store(T *p, const T (&v)[N])
{
    constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
    for (int j = 0; j < N / E; ++j) {
        uint4_t q;
        __builtin_memcpy(&q, &v[j * E], 16);
        *(uint4_any *)(p + j * E) = q;
    }
}

// one step: which byte of the scales is a constant of the instruction
template <bool LAST> __device__ __forceinline__ float16_t mx_step(uint4_t w, int sw, uint4_t x, int sx, int byte, float16_t c)
{
    const int8_v a = mx_widen(LAST ? x : w), b = mx_widen(LAST ? w : x);
    const int sa = LAST ? sx : sw, sb = LAST ? sw : sx;
    switch (byte) {
    case 0: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, 4, 0, sa, 0, sb);
    case 1: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, 4, 1, sa, 1, sb);
    case 2: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, 4, 2, sa, 2, sb);
    default: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, 4, 3, sa, 3, sb);
    }
}
// GELU in fp32: the form of activate()'s for fp16, with two coefficients more and p = 0.43, fitted in the same way: 8.5e-8 of Phi's tail up to
// u = 9.6.  With its roundings 3.9e-8 off (2-norms, normal z; what 1 + erf gives in fp32: 3.7e-8), and of a value far below zero by what its
// exponent 0.72 z^2 is off by in fp32, 1.2e-7 z^2 (the epilogues' form, three coefficients less: 8.4e-8, and a hundredth of the value at -8).
__device__ __forceinline__ float mx_gelu(float z)
{
    const float q = fabsf(z) * 0.84932180028801907f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3579984828f, q, 1.0f));
    float poly = fmaf(0.0368345306f, t, -0.1551079629f);
    poly = fmaf(poly, t, 0.1917208133f);
    poly = fmaf(poly, t, -0.0427444251f);
    poly = fmaf(poly, t, 0.1233610324f);
    poly = fmaf(poly, t, 0.1024936934f);
    poly = fmaf(poly, t, 0.1221848693f);
    poly = fmaf(poly, t, 0.1212574870f);
    const float ex = __builtin_amdgcn_exp2f(-(q * q)), part = poly * t;
    return z * (z >= 0.f ? fmaf(-part, ex, 1.f) : part * ex);
}
// Of one factor in fp32 GELU is 17 instructions; the library's erfc, good to the last bits of the smallest values too, takes three times as
// many, and is for those that are multiplied with another projection.
template <typename T, bool GATED, int ACT> __device__ __forceinline__ float mx_act(float z)
{
    float slope;
    if constexpr (ACT == KSMM_ACT_GELU && sizeof(T) == 4 && !GATED) return mx_gelu(z);
    return activate<T, ACT, false, true>(z, slope);
}

// in fp16's range (NaN stays)
__device__ __forceinline__ float mx_within_half(float z) { return z > 65504.f ? 65504.f : z < -65504.f ? -65504.f : z; }

// act of a lane's sums of one d_i
template <typename T, int D, bool GATED, int ACT> __device__ __forceinline__ void mx_activate(const float16_t (&acc)[GATED ? 2 : 1], int j, T (&v)[16 * D])
{
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float z = mx_act<T, GATED, ACT>(acc[0][i]);
        if constexpr (GATED) z *= acc[1][i];
        if constexpr (sizeof(T) == 2) asm("" : "+v"(z));  // (rounded to fp32 in every kernel: else the last product and this conversion can be one)
        v[i * D + j] = (T)z;
    }
}

// Stores of a wave's tile, 32 lines (rows of the batch, or batch-size-last outputs) of 32 * D values in a row, of which every lane has a
// half: straight from the lanes every instruction writes 64 pieces of 16 bytes apart; by way of LDS lanes that follow one another write
// bytes that do.  `stage`: MX_STAGE bytes of the wave's own; y: the first line, `pitch` values to the next.
template <typename T, int N> __device__ __forceinline__ void mx_store_lines(uint8_t *stage, T *y, int64_t pitch, const T (&v)[N], int lane)
{
    constexpr int PIECE = N * (int)sizeof(T) % 64 == 0 ? 64 : 32, PIECES = N * (int)sizeof(T) / PIECE;  // bytes of a lane at a time
    static_assert(PIECES * PIECE == N * (int)sizeof(T), "pieces of a lane's values");
    constexpr int CHUNKS = PIECE / 16, LANES = 2 * CHUNKS;  // of 16 bytes; lanes that share a line
    const int l32 = lane & 31, half = lane >> 5;
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) __builtin_memcpy(__builtin_assume_aligned(stage + l32 * MX_LINE + half * PIECE + i * 16, 16), (const char *)v + q * PIECE + i * 16, 16);
        __builtin_amdgcn_wave_barrier();
        const int line = lane / LANES, chunk = lane % LANES;
        // (both halves of a lane's values are N apart)
        char *to = (char *)(y + line * pitch) + (chunk / CHUNKS) * (N * (int)sizeof(T)) + q * PIECE + chunk % CHUNKS * 16;
        const int64_t step = pitch * (64 / LANES) * (int64_t)sizeof(T);
#pragma unroll
        for (int i = 0; i < 32 * LANES / 64; ++i) {
            const uint4_t r = *(const uint4_t *)(stage + (line + i * (64 / LANES)) * MX_LINE + chunk * 16);
            *(uint4_any *)to = r;
            to += step;
        }
    }
}

// stores of a lane's results: tile t of 32 rows of those from n0 on, tile bt of the p.b outputs that begin at `from` of an a_i's `rows`
template <typename T, bool LAST, int D>
__device__ __forceinline__ void mx_results(const MxProduct &p, const T (&v)[16 * D], int ai, int d0, int bt, int lane, int64_t n0, int t, int here, uint8_t *stage,
                                           int rows, int from = 0)
{
    const int l32 = lane & 31, half = lane >> 5;
    if ((t + 1) * 32 <= here && (bt + 1) * 32 <= p.b) {
        const int64_t pitch = LAST ? (int64_t)p.d * p.batch : (int64_t)p.a * rows * p.d;
        T *const y = (T *)p.y + (LAST ? (((int64_t)ai * rows + from + bt * 32) * p.d + d0) * p.batch + n0 + t * 32
                                      : (((n0 + t * 32) * p.a + ai) * rows + from + bt * 32) * p.d + d0);
        mx_store_lines<T, 16 * D>(stage, y, pitch, v, lane);
        return;
    }
    if constexpr (LAST) {
        const int o = bt * 32 + l32, n = t * 32 + 16 * half;
        T *const y = (T *)p.y + (((int64_t)ai * rows + from + o) * p.d + d0) * p.batch + n0 + n;
        if (o >= p.b) return;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (n + i < here) y[i] = v[i];
    } else {
        const int o = bt * 32 + 16 * half, n = t * 32 + l32;
        T *const y = (T *)p.y + (((n0 + n) * p.a + ai) * rows + from + o) * p.d + d0;
        struct __attribute__((packed, aligned(sizeof(T)))) Run {
            T e[D];
        };
        if (n >= here) return;
        if (o + 16 <= p.b) {
            mx_store<T, 16 * D>(y, v);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                Run r;
#pragma unroll
                for (int j = 0; j < D; ++j) r.e[j] = v[i * D + j];
                if (o + i < p.b) *(Run *)(y + (int64_t)i * p.d) = r;
            }
        }
    }
}

// ---- weights in registers ---------------------------------------------------------------------------------
// A wave holds the codes of its 32 outputs (of all D, gate and up) for the whole launch, KS steps of 64 along c, and walks down the
// batch: a workgroup's eight waves are tiles of outputs times runs of rows.  Four more waves quantise the rows of the next step into
// the other of two buffers in LDS and have the values of the step after that on their way: waits for what is loaded would be waits for the
// stores before it too (one counter), which only waves that store nothing do not make ((1,768,192,2) gated fp16, 25088 rows 40 us for 29).
constexpr int MX_CONSUMERS = 8, MX_PRODUCERS = 4;
constexpr int mx_scale_bytes(int ks) { return ks <= 4 ? 4 : ks <= 8 ? 8 : 16; }  // of a row and one half of each step
// blocks of 32 rows, or quarters of them, that a producer's thread takes, and of these those on their way at once: 64 registers of values
constexpr int mx_rounds(int ks, int quarters) { return quarters == 1 ? (ks + 3) / 4 : ks; }
// Lanes a block.  Four of them read what is one run in memory with a quarter of the lines a load, but find the scale four times: in fp32
// (1,768,192,2) gated takes 58 us for 64, in fp16 36 for 29.  (Of 16 steps the rounds would be too many to keep; blocks of three d_i that
// end inside 32 are read three values at a time: (1,192,48,3) in fp16 27 us for 13.)
template <typename T> constexpr int mx_quarters(bool last, int ks, int d) { return last || ks > 8 || (sizeof(T) == 2 && d != 3) ? 1 : 4; }
// Rows that a lane reads together, batch-size-last: of 2-byte values two, 256 bytes a load instead of 128, where that leaves the producers
// work ((1,192,768,2) 25088 rows 40.7 -> 35.2 us, (1,48,48,16) 32 -> 29; of three steps, 96 pairs a step for 256 threads, (1,768,192,2) 42.5 -> 44.5)
template <typename T> constexpr int mx_pairs(bool last, int ks) { return last && sizeof(T) == 2 && (ks == 1 || ks > 4) ? 2 : 1; }
constexpr int mx_ahead(int rounds, int registers)
{
    int n = 64 / registers < 8 ? 64 / registers : 8;
    if (n > rounds) n = rounds;
    while (rounds % n) --n;
    return n;
}

// the weights of a wave's 32 outputs, those of tile bt
template <bool LAST, int D, int G, int KS> struct MxHeld {
    static constexpr int SB = mx_scale_bytes(KS), SW = (KS + 3) / 4;
    uint4_t w[D][G][KS];
    int sw[D][G][SW], scale[D][G][KS];
    __device__ __forceinline__ void load(const MxProduct &p, int ai, int d0, int bt, int l32, int run, int half)
    {
        const int wo = bt * 32 + (LAST ? l32 : run), o = wo < p.b ? wo : p.b - 1;  // (outputs behind the last one are read as the last one)
#pragma unroll
        for (int j = 0; j < D; ++j)
#pragma unroll
            for (int q = 0; q < G; ++q) {
                const int64_t at = (((int64_t)ai * p.d + d0 + j) * (G * p.b) + q * p.b + o) * p.cb;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int kb = 2 * s + half;
                    const bool there = kb < p.cb;
                    w[j][q][s] = there ? *(const uint4_t *)(p.w + (at + kb) * 16) : uint4_t{0, 0, 0, 0};
                    scale[j][q][s] = there ? p.w_scales[at + kb] : 127;
                }
            }
    }
    // (said to the compiler: the weights are there, and no step waits for them again, which would be for all stores before it too)
    __device__ __forceinline__ void arrived()
    {
#pragma unroll
        for (int j = 0; j < D; ++j)
#pragma unroll
            for (int q = 0; q < G; ++q) {
#pragma unroll
                for (int s = 0; s < KS; ++s) sw[j][q][s / 4] = s % 4 ? sw[j][q][s / 4] | scale[j][q][s] << 8 * (s % 4) : scale[j][q][s];
#pragma unroll
                for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(w[j][q][s]));
#pragma unroll
                for (int s = 0; s < SW; ++s) asm volatile("" : "+v"(sw[j][q][s]));
            }
    }
    // sums of row `row` of x in LDS with d_i j's weights; bias: of the wave's tile, or null
    __device__ __forceinline__ void sums(const uint8_t *codes, const uint8_t *scales, int slots, int row, int j, int l32, int half, const float *bias, float16_t (&acc)[G]) const
    {
        int sx[SW];
#pragma unroll
        for (int i = 0; i < SW; ++i) sx[i] = ((const int *)(scales + row * 2 * SB + half * SB))[i];
        auto steps = [&](auto biased) {
#pragma unroll
            for (int q = 0; q < G; ++q) {
                acc[q] = float16_t{};
                if constexpr (decltype(biased)::value)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[q][i] = bias[(q * D + j) * 32 + (LAST ? l32 : 16 * half + i)];
            }
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const uint4_t x = *(const uint4_t *)(codes + (row * slots + 2 * s + half) * 16);
#pragma unroll
                for (int q = 0; q < G; ++q) acc[q] = mx_step<LAST>(w[j][q][s], sw[j][q][s / 4], x, sx[s / 4], s % 4, acc[q]);
            }
        };
        if (bias)
            steps(std::true_type());
        else
            steps(std::false_type());
    }
};
// scales of blocks behind the last one, of `words` words each `apart` bytes from the other buffer's: they are read, with weights of zeros, but
// not as NaN; and the biases of `tiles` tiles from tile0 on, (tile, gate and up, D, 32 outputs)
template <typename T, int D, int G> __device__ __forceinline__ void mx_prepare(const MxProduct &p, uint8_t *scales, int apart, int words, float *bias, int ai, int d0, int tile0)
{
    for (int k = 0; k < 2; ++k)
        for (int i = threadIdx.x; i < words; i += blockDim.x) ((uint32_t *)(scales + k * apart))[i] = 0x7f7f7f7fu;
    if (p.bias)
        for (int i = threadIdx.x; i < p.wave_tiles * G * 32 * D; i += blockDim.x) {
            const int j = i / 32 % D, q = i / 32 / D % G, out = (tile0 + i / 32 / D / G) * 32 + i % 32;
            bias[i] = out < p.b ? (float)((const T *)p.bias)[((int64_t)ai * (G * p.b) + q * p.b + out) * p.d + d0 + j] : 0.f;
        }
}

template <typename T, bool LAST, int D, bool GATED, int ACT, int KS>
__global__ __launch_bounds__(64 * (MX_CONSUMERS + MX_PRODUCERS)) void ks_mx_held_kernel(MxProduct p)
{
    constexpr int G = GATED ? 2 : 1, SB = mx_scale_bytes(KS), P = mx_pairs<T>(LAST, KS), R = (mx_rounds(KS, mx_quarters<T>(LAST, KS, D)) + P - 1) / P;
    constexpr int BLOCKS = LAST ? P : D;  // of a task: rows, or d_i of one
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int TN = p.tile_rows, buffer = D * TN * (p.slots * 16 + 2 * SB);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, half = lane >> 5;
    const int run = 16 * ((l32 >> 2) & 1) + 4 * (l32 >> 3) + (l32 & 3);  // the row that this lane reads of the operand whose rows are dealt out
    int blk = (int)(p.first + blockIdx.x);
    const int first = blk % p.row_splits;
    blk /= p.row_splits;
    const int unit = blk % p.units, ai = unit / p.runs, d0 = (unit - ai * p.runs) * D;
    const int tile0 = blk / p.units * p.wave_tiles;
    float *const bias = (float *)(smem + 2 * buffer);
    uint8_t *const stage = smem + 2 * buffer + p.wave_tiles * G * D * 128 + wave * MX_STAGE;
    const int tasks = TN / P * p.cb, batch = (int)p.batch, row_tiles = (int)p.token_tiles;  // (steps past the end are counted in 32 bits)
    const int turns = p.codes_out ? p.splits : 0, mine = blk / p.units;  // (workgroups of the same rows hand out the codes in turn)

    // what a thread loads for the step of rows n0 on: the blocks of task t, or batch-size-first a quarter of them
    constexpr int Q = mx_quarters<T>(LAST, KS, D);
    typedef std::conditional_t<Q == 1, MxGroup<T, BLOCKS>, MxQuarter<T, D>> Load;
    const MxDiv by(LAST ? TN / P : p.cb);
    const int quarter = threadIdx.x & 3;  // (batch-size-first: a thread has the same of all its blocks)
    // row * 256 + kb of task t
    auto place = [&](int t) {
        const int u = t / Q, v = by(u), rest = u - v * (LAST ? TN / P : p.cb);
        return LAST ? rest * P * 256 + v : v * 256 + rest;
    };
    // rows that are not there: whatever LDS has, they are other columns of the product
    auto there = [&](int t, int at, int n0) { return t < tasks * Q && (at >> 8) < batch - n0; };
    auto fetch = [&](Load &f, int t, int at, int n0) {
        if (!there(t, at, n0)) return;
        const int n = at >> 8, kb = at & 255;
        if constexpr (LAST)
            mx_load<T, P>(f, (const T *)p.x + (((int64_t)ai * p.c + kb * 32) * p.d + d0) * p.batch + (n0 + n < batch - P ? n0 + n : batch - P), (int64_t)p.d * p.batch, p.c - kb * 32);
        else if constexpr (Q == 1)
            mx_load<T, D>(f, (const T *)p.x + ((((int64_t)n0 + n) * p.a + ai) * p.c + kb * 32) * D, D, p.c - kb * 32);
        else
            mx_load<T, D>(f, (const T *)p.x + ((((int64_t)n0 + n) * p.a + ai) * p.c + kb * 32 + quarter * 8) * D, p.c - kb * 32 - quarter * 8);
    };
    auto keep = [&](const Load &f, int t, int at, int n0, int which, bool emit) {
        if (!there(t, at, n0)) return;
        const int n = at >> 8, kb = at & 255;
        uint8_t *const codes = smem + which * buffer, *const scales = codes + D * TN * p.slots * 16;
#pragma unroll
        for (int j = 0; j < BLOCKS; ++j) {
            // (of two rows the last one of the batch goes with the one before it, which has been found once already, here or a step ago)
            const int at_row = LAST ? (n < batch - n0 - P ? n : batch - n0 - P) + j : n, row = LAST ? at_row : j * TN + n;
            if (P > 1 && row < 0) continue;
            const int64_t block = (((int64_t)ai * p.d + d0 + (LAST ? 0 : j)) * p.batch + n0 + at_row) * p.cb + kb;
            int scale;
            if constexpr (Q == 1) {
                uint4_t code;
                scale = mx_quantize<T, BLOCKS>(f, j, p.c - kb * 32, code);
                *(uint4_t *)(codes + (row * p.slots + kb) * 16) = code;
                if (emit) *(uint4_t *)(p.codes_out + block * 16) = code;
            } else {
                uint32_t code;
                scale = mx_quantize<T, D>(f, j, code);
                *(uint32_t *)(codes + (row * p.slots + kb) * 16 + quarter * 4) = code;
                if (emit) *(uint32_t *)(p.codes_out + block * 16 + quarter * 4) = code;
            }
            if (Q == 1 || quarter == 0) {
                scales[row * 2 * SB + (kb & 1) * SB + (kb >> 1)] = (uint8_t)scale;
                if (emit) p.scales_out[block] = (uint8_t)scale;
            }
        }
    };
    auto prepare = [&] { mx_prepare<T, D, G>(p, smem + D * TN * p.slots * 16, buffer, D * TN * SB / 2, bias, ai, d0, tile0); };

    if (wave >= MX_CONSUMERS) {
        const int t0 = threadIdx.x - 64 * MX_CONSUMERS;
        constexpr int AHEAD = mx_ahead(R, BLOCKS * (int)sizeof(T) * 8 / Q);
        Load f[AHEAD];
        int at[R];
#pragma unroll
        for (int r = 0; r < R; ++r) at[r] = place(t0 + r * 64 * MX_PRODUCERS);
#pragma unroll
        for (int r = 0; r < AHEAD; ++r) fetch(f[r], t0 + r * 64 * MX_PRODUCERS, at[r], first * TN);
        prepare();
        __syncthreads();
        int which = 0, turn = turns ? 0 : -1;
        for (int tile = first; tile < row_tiles; tile += p.row_splits, which ^= 1) {
            const bool emit = turn == mine;
            if (turns) turn = turn + 1 < turns ? turn + 1 : 0;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                keep(f[r % AHEAD], t0 + r * 64 * MX_PRODUCERS, at[r], tile * TN, which, emit);
                const int next = (r + AHEAD) % R;
                if (r + AHEAD < R || tile + p.row_splits < row_tiles)
                    fetch(f[r % AHEAD], t0 + next * 64 * MX_PRODUCERS, at[next], (r + AHEAD < R ? tile : tile + p.row_splits) * TN);
            }
            __syncthreads();
        }
        return;
    }

    const int wb = wave & (p.wave_tiles - 1), wt = wave / p.wave_tiles, per_wave = TN / 32 / (MX_CONSUMERS / p.wave_tiles);
    const int bt = tile0 + wb;
    const bool busy = bt < p.b_tiles;
    MxHeld<LAST, D, G, KS> held;
    if (busy) held.load(p, ai, d0, bt, l32, run, half);
    prepare();
    __syncthreads();
    held.arrived();
    int which = 0;
    for (int tile = first; tile < row_tiles; tile += p.row_splits, which ^= 1) {
        const int n0 = tile * TN, here = batch - n0 < TN ? batch - n0 : TN;
        __syncthreads();
        if (!busy) continue;
        const uint8_t *const codes = smem + which * buffer, *const scales = codes + D * TN * p.slots * 16;
        for (int t = wt * per_wave; t < (wt + 1) * per_wave && t * 32 < here; ++t) {
            T v[16 * D];
#pragma unroll
            for (int j = 0; j < D; ++j) {
                float16_t acc[G];
                held.sums(codes, scales, p.slots, j * TN + t * 32 + (LAST ? run : l32), j, l32, half, p.bias ? bias + wb * G * D * 32 : nullptr, acc);
                mx_activate<T, D, GATED, ACT>(acc, j, v);
            }
            mx_results<T, LAST, D>(p, v, ai, d0, bt, lane, n0, t, here, stage, p.b);
        }
    }
}

// ---- weights from the caches: few rows, more weights than registers hold, or d_i that no thread takes together --------------------
// A workgroup quantises 32 * TT rows of a unit (one a_i; all d_i, or runs of 16 of more) into LDS; its waves take tiles of 32 outputs
// of one d_i each, and leave their results in LDS, from where they go out a line of a row, all d_i, at a time (batch-size-last, where
// a unit is one d_i, and where a tile is all of a workgroup's, straight from the wave).  Four steps along c of codes are on their way, the
// first ones before x is.  Of few rows a launch is bound by what follows one another, not by a rate: eight waves quantise, chunks of
// outputs are as small as one workgroup a compute unit allows (see mx_launch_wide), and what divides is multiplied with.
// D: all d_i of up to four, which a thread quantises together; 0: five and more; -1: x comes as codes.  (Kernels of their own: what they do not
// run of the others' instructions costs a launch of few rows a tenth.)
template <typename T, bool LAST, int D, int TT, bool GATED, int ACT> __global__ __launch_bounds__(64 * MX_WAVES) void ks_mx_wide_kernel(MxProduct p)
{
    constexpr int TN = 32 * TT, G = GATED ? 2 : 1;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, half = lane >> 5;
    const int run = 16 * ((l32 >> 2) & 1) + 4 * (l32 >> 3) + (l32 & 3);  // the row that this lane reads of the operand whose rows are dealt out
    uint8_t *const codes = smem, *const scales = codes + (size_t)p.run_d * TN * p.slots * 16;
    T *const stage = (T *)(scales + (p.run_d * TN * p.cb + 15) / 16 * 16);  // of the workgroup: rows of `pitch`; batch-size-last of the waves
    const uint32_t group = p.first + blockIdx.x, rest = group / (uint32_t)p.splits, split = group - rest * (uint32_t)p.splits, tile = rest / (uint32_t)p.units;
    const int unit = (int)(rest - tile * (uint32_t)p.units), ai = p.runs == 1 ? unit : unit / p.runs, d0 = (unit - ai * p.runs) * p.run_d;
    const int64_t n0 = (int64_t)tile * TN;
    const int here = (int)(p.batch - n0 < TN ? p.batch - n0 : TN);                 // rows of the batch
    const int dc = LAST ? 1 : p.d - d0 < p.run_d ? p.d - d0 : p.run_d;             // d_i of the unit
    const int rows_w = G * p.b, pitch = p.chunk_tiles * 32 * p.run_d + 4 / (int)sizeof(T);  // (an odd number of words: rows meet other banks)
    // ---- x into LDS
    auto keep = [&](int j, int n, int kb, uint4_t code, int scale, bool emit) {
        const int row = j * TN + n;
        *(uint4_t *)(codes + ((size_t)row * p.slots + kb) * 16) = code;
        scales[row * p.cb + kb] = (uint8_t)scale;
        if (emit) {
            const int64_t block = (((int64_t)ai * p.d + d0 + j) * p.batch + n0 + n) * p.cb + kb;
            *(uint4_t *)(p.codes_out + block * 16) = code;
            p.scales_out[block] = (uint8_t)scale;
        }
    };
    const bool emit = p.codes_out && split == 0;
    const MxDiv by_cb = p.by_cb, by_dc = dc == p.run_d ? p.by_run_d : MxDiv(dc);
    const int chunk_first = (int)split * p.tiles_per, chunk_end = chunk_first + p.tiles_per < p.b_tiles ? chunk_first + p.tiles_per : p.b_tiles;
    // ---- a wave's work: a tile of outputs of one d_i, and the codes of its next AHEAD steps along c
    constexpr int AHEAD = 4;
    struct {
        int j, bt;
        int64_t at[G];
        uint4_t w[AHEAD][G];
        int s[AHEAD][G];
    } job;
    auto load = [&](int kb, int r) {
        const bool there = kb < p.cb;
#pragma unroll
        for (int q = 0; q < G; ++q) {
            job.w[r][q] = there ? *(const uint4_t *)(p.w + (job.at[q] + kb) * 16) : uint4_t{0, 0, 0, 0};
            job.s[r][q] = there ? p.w_scales[job.at[q] + kb] : 127;
        }
    };
    auto begin = [&](int chunk, int i) {
        const int tile = by_dc(i);
        job.j = i - tile * dc;
        job.bt = chunk + tile;
        // (outputs behind the last one are read as the last one and not stored)
        const int wo = job.bt * 32 + (LAST ? l32 : run), o = wo < p.b ? wo : p.b - 1;
#pragma unroll
        for (int q = 0; q < G; ++q) job.at[q] = (((int64_t)ai * p.d + d0 + job.j) * rows_w + q * p.b + o) * p.cb;
#pragma unroll
        for (int r = 0; r < AHEAD; ++r)
            if (2 * r < p.cb) load(2 * r + half, r);
    };
    auto jobs_of = [&](int chunk) { return (chunk_end - chunk < p.chunk_tiles ? chunk_end - chunk : p.chunk_tiles) * dc; };
    // (the first ones are on their way before x is)
    if (wave < jobs_of(chunk_first)) begin(chunk_first, wave);
    if constexpr (D < 0) {  // they are copied
        for (int t = threadIdx.x; t < TN * p.cb * dc; t += 64 * MX_WAVES) {
            const int u = by_cb(t), kb = t - u * p.cb, j = u / TN, n = u - j * TN;
            if (n >= here) continue;
            const int64_t block = (((int64_t)ai * p.d + d0 + j) * p.batch + n0 + n) * p.cb + kb;
            keep(j, n, kb, *(const uint4_t *)((const uint8_t *)p.x + block * 16), p.x_scales[block], false);
        }
    } else if constexpr (LAST) {
        constexpr int P = TT == 1 ? 1 : mx_pairs<T>(true, 16);  // ((1,1024,1024,1) fp16, 25088 rows 86 -> 60 us)
        for (int t = threadIdx.x; t < TN / P * p.cb; t += 64 * MX_WAVES) {
            const int kb = t / (TN / P), n = (t - kb * (TN / P)) * P;
            if (n >= here) continue;  // (whatever LDS has there, it is another column of the product)
            // (of two rows the last one of the batch goes with the one before it)
            const int first = n < here - P ? n : here - P;
            MxGroup<T, P> g;
            mx_load<T, P>(g, (const T *)p.x + (((int64_t)ai * p.c + kb * 32) * p.d + d0) * p.batch + n0 + first, (int64_t)p.d * p.batch, p.c - kb * 32);
#pragma unroll
            for (int j = 0; j < P; ++j) {
                uint4_t code;
                const int scale = mx_quantize<T, P>(g, j, p.c - kb * 32, code);
                if (P == 1 || first + j >= 0) keep(0, first + j, kb, code, scale, emit);
            }
        }
    } else if constexpr (D > 0) {
        constexpr int SIZE = 2 * D * (int)sizeof(T), TIMES = 64 / SIZE < 4 ? 64 / SIZE : 4;  // (64 registers of values on their way)
        const int total = here * p.cb * 4, quarter = threadIdx.x & 3;
        for (int t0 = threadIdx.x; t0 < total; t0 += 64 * MX_WAVES * TIMES) {
            MxQuarter<T, D> g[TIMES];
            int n[TIMES], kb[TIMES];
#pragma unroll
            for (int r = 0; r < TIMES; ++r) {
                const int t = t0 + r * 64 * MX_WAVES, u = t / 4;
                n[r] = by_cb(u);
                kb[r] = u - n[r] * p.cb;
                if (t < total) mx_load<T, D>(g[r], (const T *)p.x + (((n0 + n[r]) * p.a + ai) * p.c + kb[r] * 32 + quarter * 8) * D, p.c - kb[r] * 32 - quarter * 8);
            }
#pragma unroll
            for (int r = 0; r < TIMES; ++r) {
                if (t0 + r * 64 * MX_WAVES >= total) break;
#pragma unroll
                for (int j = 0; j < D; ++j) {
                    uint32_t code;
                    const int row = j * TN + n[r], scale = mx_quantize<T, D>(g[r], j, code);
                    const int64_t block = (((int64_t)ai * p.d + d0 + j) * p.batch + n0 + n[r]) * p.cb + kb[r];
                    ((uint32_t *)(codes + ((size_t)row * p.slots + kb[r]) * 16))[quarter] = code;
                    if (emit) ((uint32_t *)(p.codes_out + block * 16))[quarter] = code;
                    if (quarter == 0) {
                        scales[row * p.cb + kb[r]] = (uint8_t)scale;
                        if (emit) p.scales_out[block] = (uint8_t)scale;
                    }
                }
            }
        }
    } else {
        // as they lie into LDS, where a thread gathers a block
        constexpr int E = 16 / (int)sizeof(T), AHEAD = 4;
        const bool whole = dc == p.d;
        const int length = whole ? p.c * dc : dc, vectors = (length + E - 1) / E, lines = whole ? 1 : p.c;  // runs of a row
        const MxDiv by_vectors(vectors), by_lines(lines);
        for (int first = 0; first < here; first += p.raw_rows) {
            const int rows = here - first < p.raw_rows ? here - first : p.raw_rows, total = rows * lines * vectors;
            if (first > 0) __syncthreads();
            for (int i0 = threadIdx.x; i0 < total; i0 += 64 * MX_WAVES * AHEAD) {
                uint4_t q[AHEAD];
                int to[AHEAD], left[AHEAD];
#pragma unroll
                for (int r = 0; r < AHEAD; ++r) {
                    const int i = i0 + r * 64 * MX_WAVES < total ? i0 + r * 64 * MX_WAVES : i0;  // (behind the end the first one again)
                    const int u = by_vectors(i), e = (i - u * vectors) * E, n = by_lines(u), line = u - n * lines;
                    const T *from = (const T *)p.x + (((n0 + first + n) * p.a + ai) * p.c + line) * p.d + d0 + e;
                    left[r] = length - e;
                    to[r] = n * p.raw_pitch + line * dc + e;
                    if (left[r] >= E) {
                        q[r] = *(const uint4_any *)from;
                    } else {
                        T v[E];
#pragma unroll
                        for (int k = 0; k < E; ++k) v[k] = from[k < left[r] ? k : 0];
                        __builtin_memcpy(&q[r], v, 16);
                    }
                }
#pragma unroll
                for (int r = 0; r < AHEAD; ++r) {
                    if (whole || dc % E == 0) {
                        __builtin_memcpy(__builtin_assume_aligned(stage + to[r], 16), &q[r], 16);
                    } else {
                        T v[E];
                        __builtin_memcpy(v, &q[r], 16);
#pragma unroll
                        for (int k = 0; k < E; ++k)
                            if (k < left[r]) stage[to[r] + k] = v[k];
                    }
                }
            }
            __syncthreads();
            const MxDiv by_rows(rows);
            for (int t = threadIdx.x; t < rows * p.cb * dc; t += 64 * MX_WAVES) {
                const int u = by_dc(t), j = t - u * dc, kb = by_rows(u), n = u - kb * rows, count = p.c - kb * 32, last = (count < 32 ? count : 32) - 1;
                const T *from = stage + n * p.raw_pitch + kb * 32 * dc + j;
                MxGroup<T, 1> g;
#pragma unroll
                for (int k = 0; k < 32; ++k) g.v[k] = from[(k < last ? k : last) * dc];
                uint4_t code;
                const int scale = mx_quantize<T, 1>(g, 0, count, code);
                keep(j, first + n, kb, code, scale, emit);
            }
        }
    }
    __syncthreads();
    // ---- products, a chunk of tiles of outputs at a time
    const bool alone = !LAST && (D == 1 || D == -1) && p.d == 1 && p.chunk_tiles == 1;  // (one wave's lines are all there is)
    const T *const bias = (const T *)p.bias;
    for (int chunk = chunk_first; chunk < chunk_end; chunk += p.chunk_tiles) {
        const int jobs = jobs_of(chunk);
        for (int i = wave; i < jobs; i += MX_WAVES) {
            if (chunk > chunk_first || i > wave) begin(chunk, i);
            const int j = job.j, bt = job.bt;
            float16_t acc[TT][G];
#pragma unroll
            for (int q = 0; q < G; ++q) {
                float16_t add = {};
                if (bias) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int out = LAST ? bt * 32 + l32 : bt * 32 + 16 * half + i;
                        add[i] = (float)bias[((int64_t)ai * rows_w + q * p.b + (out < p.b ? out : p.b - 1)) * p.d + d0 + j];
                    }
                }
#pragma unroll
                for (int t = 0; t < TT; ++t) acc[t][q] = add;
            }
            constexpr int XS = TT == 1 ? AHEAD : 1;  // steps whose codes of x are read at once
            for (int k0 = 0; k0 < p.cb; k0 += 2 * AHEAD) {
#pragma unroll
                for (int r0 = 0; r0 < AHEAD; r0 += XS) {
                    uint4_t x[XS][TT];
                    int sx[XS][TT];
#pragma unroll
                    for (int r = 0; r < XS; ++r) {
                        const int kb = k0 + 2 * (r0 + r) + half, at = kb < p.cb ? kb : p.cb - 1;  // (behind the last block: with weights of zeros, but not as NaN)
#pragma unroll
                        for (int t = 0; t < TT; ++t) {
                            const int row = j * TN + t * 32 + (LAST ? run : l32);
                            x[r][t] = *(const uint4_t *)(codes + ((size_t)row * p.slots + at) * 16);
                            sx[r][t] = kb < p.cb ? scales[row * p.cb + at] : 127;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < XS; ++r) {
                        const int k = k0 + 2 * (r0 + r);
                        if (k >= p.cb) break;
                        const auto &w = job.w[r0 + r];
                        const auto &sw = job.s[r0 + r];
#pragma unroll
                        for (int t = 0; t < TT; ++t)
#pragma unroll
                            for (int q = 0; q < G; ++q) acc[t][q] = LAST ? mx_mfma(x[r][t], sx[r][t], w[q], sw[q], acc[t][q]) : mx_mfma(w[q], sw[q], x[r][t], sx[r][t], acc[t][q]);
                        if (k + 2 * AHEAD < p.cb) load(k + 2 * AHEAD + half, r0 + r);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                T v[16];
                if constexpr (D == -1 && !GATED && ACT == KSMM_ACT_NONE && sizeof(T) == 2) {
                    if (p.finite) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[t][0][i] = mx_within_half(acc[t][0][i]);
                    }
                }
                mx_activate<T, 1, GATED, ACT>(acc[t], 0, v);
                if (LAST || alone) {
                    if (t * 32 < here) mx_results<T, LAST, 1>(p, v, ai, d0, bt, lane, n0, t, here, (uint8_t *)stage + wave * MX_STAGE, p.b);
                } else {
                    T *const to = stage + (t * 32 + l32) * pitch + ((bt - chunk) * 32 + 16 * half) * dc + j;
#pragma unroll
                    for (int i = 0; i < 16; ++i) to[i * dc] = v[i];
                }
            }
        }
        if (!LAST && !alone) {
            __syncthreads();
            // pieces of a line that lie together: all of it, or with more d_i than the unit's, those of an output
            constexpr int E = 16 / (int)sizeof(T);
            const int outs = (chunk + p.chunk_tiles) * 32 < p.b ? p.chunk_tiles * 32 : p.b - chunk * 32, tiles_out = (chunk_end - chunk) * 32;
            const int lines = outs < tiles_out ? outs : tiles_out;  // outputs of the chunk
            const int piece = dc == p.d ? lines * dc : dc, pieces = dc == p.d ? 1 : lines, vectors = (piece + E - 1) / E;
            const MxDiv by_vectors(vectors), by_pieces(pieces);
            for (int i = threadIdx.x; i < here * pieces * vectors; i += 64 * MX_WAVES) {
                const int u = by_vectors(i), e = (i - u * vectors) * E, n = by_pieces(u), q = u - n * pieces;
                const T *from = stage + n * pitch + q * dc + e;
                T *to = (T *)p.y + (((n0 + n) * p.a + ai) * p.b + chunk * 32 + q) * p.d + d0 + e;
                if (e + E <= piece) {
                    T v[E];
                    if (sizeof(T) == 4 || dc % 2 == 0 || pieces == 1) {  // (words)
                        __builtin_memcpy(v, __builtin_assume_aligned(from, 4), 16);
                    } else {
#pragma unroll
                        for (int k = 0; k < E; ++k) v[k] = from[k];
                    }
                    mx_store<T, E>(to, v);
                } else {
                    for (int k = 0; k < piece - e; ++k) to[k] = from[k];
                }
            }
            __syncthreads();
        }
    }
}

// `grid` workgroups of a kernel
inline int mx_launch(void (*fn)(MxProduct), MxProduct p, int64_t grid, int threads, int64_t lds, hipStream_t s)
{
    return in_launches(grid, threads, [&](uint32_t first, unsigned groups) {
        p.first = first;
        return launch_kernel(fn, groups, (unsigned)threads, (size_t)lds, s, p);
    });
}

inline int64_t mx_held_lds(int d, bool gated, int ks, int cb, int rows, int tiles, int consumers)
{
    return 2LL * d * rows * ((cb | 1) * 16 + 2 * mx_scale_bytes(ks)) + (int64_t)tiles * (gated ? 2 : 1) * 32 * d * 4 + consumers * MX_STAGE;
}

template <typename T, bool LAST, int D, int TT, bool GATED> int mx_launch_wide(MxProduct p, int act, hipStream_t s)
{
    p.slots = p.cb | 1;
    p.run_d = mx_unit_of(p.d, LAST);
    p.runs = (p.d + p.run_d - 1) / p.run_d;
    p.units = p.a * p.runs;
    p.b_tiles = (p.b + 31) / 32;
    p.chunk_tiles = mx_chunk_of(p.run_d, LAST);
    p.token_tiles = (p.batch + 32 * TT - 1) / (32 * TT);
    // outputs are split over workgroups, each of which quantises its rows anew, as far as there is one for a compute unit at most ((1,192,768,2)
    // fp16 of 3136 rows in 98 of them 16.0 us, in 196 12.9; of 6272 in 196 17.3, in 392 19.3), and into smaller chunks where that leaves room
    const int64_t groups = p.token_tiles * p.units;
    while (p.chunk_tiles > 1 && groups * ((p.b_tiles + p.chunk_tiles / 2 - 1) / (p.chunk_tiles / 2)) <= 256) p.chunk_tiles /= 2;
    const int most = (p.b_tiles + p.chunk_tiles - 1) / p.chunk_tiles;
    const int64_t want = std::max<int64_t>(1, 256 / groups);
    p.splits = (int)(want < most ? want : most);
    p.tiles_per = (most + p.splits - 1) / p.splits * p.chunk_tiles;
    p.splits = (p.b_tiles + p.tiles_per - 1) / p.tiles_per;
    const int64_t grid = groups * p.splits;
    if (grid > 0x7fffffffLL) return KSMM_ERR_TOO_LARGE;
    const int lds = (int)mx_wide_lds(TT, p.c, p.d, (int)sizeof(T), LAST);
    p.by_cb = MxDiv(p.cb);
    p.by_run_d = MxDiv(p.run_d);
    p.raw_pitch = (int)(mx_raw_row(p.c, p.d, (int)sizeof(T)) / (int)sizeof(T));
    p.raw_rows = mx_raw_rows(TT, p.c, p.d, (int)sizeof(T));
    int rc = KSMM_OK;
    with_act(act, [&](auto which) {
        constexpr int ACT = decltype(which)::value;
        if constexpr (GATED || ACT != KSMM_ACT_SILU) {
            auto fn = &ks_mx_wide_kernel<T, LAST, D, TT, GATED, ACT>;
            if (lds > 64 * 1024) rc = ensure_dynamic_lds((const void *)fn, (int)MX_LDS_ALL);  // (set once a kernel: for all of its sizes)
            if (rc == KSMM_OK) rc = mx_launch(fn, p, grid, 64 * MX_WAVES, lds, s);
        }
    });
    return rc;
}

// registers of a thread
inline int mx_registers(const void *kernel)
{
    hipFuncAttributes a;
    if (hipFuncGetAttributes(&a, kernel) == hipSuccess) return a.numRegs;
    (void)hipGetLastError();  // (its answer is not needed)
    return 512;
}

// the rest of the sizes, with `tiles` of outputs a workgroup
inline void mx_held_tiles(MxProduct &p, int consumers, int tiles)
{
    p.wave_tiles = tiles;
    p.tile_rows = 32 * consumers / tiles;
    p.token_tiles = (p.batch + p.tile_rows - 1) / p.tile_rows;
    p.splits = (p.b_tiles + tiles - 1) / tiles;
}
// sizes of a launch whose weights are held by `consumers` waves: `most` blocks a step of a workgroup
inline void mx_held_sizes(MxProduct &p, bool last, int consumers, int most)
{
    p.slots = p.cb | 1;
    p.runs = last ? p.d : 1;
    p.units = p.a * p.runs;
    p.b_tiles = (p.b + 31) / 32;
    // the more waves share their rows the less often these are quantised, but none should idle
    int idle = 1 << 30;
    for (int tiles = consumers; tiles >= 1; tiles /= 2) {
        const int over = (p.b_tiles + tiles - 1) / tiles * tiles - p.b_tiles;
        if (over < idle && 32 * consumers / tiles * p.cb <= most) {
            p.wave_tiles = tiles;
            idle = over;
        }
    }
    mx_held_tiles(p, consumers, p.wave_tiles);
}
inline int64_t mx_held_groups(const MxProduct &p) { return (int64_t)p.units * p.splits; }
// workgroups that share the steps of one tile of outputs: one a compute unit, or two where the registers of both fit; one more would be a
// second round.  Those of the same rows lie on the same XCD where that is a multiple of eight apart
inline int64_t mx_held_splits(const MxProduct &p, int a_unit)
{
    const int64_t most = std::max<int64_t>(1, 256 * a_unit / mx_held_groups(p));
    return most >= 8 ? most / 8 * 8 : most;
}

template <typename T, bool LAST, int D, bool GATED, int KS> int mx_launch_held(MxProduct p, int act, hipStream_t s)
{
    constexpr int Q = mx_quarters<T>(LAST, KS, D), P = mx_pairs<T>(LAST, KS);
    mx_held_sizes(p, LAST, MX_CONSUMERS, 64 * MX_PRODUCERS * P * ((mx_rounds(KS, Q) + P - 1) / P) / Q);
    int64_t most = mx_held_splits(p, 1);
    if (p.token_tiles > most && mx_held_lds(D, GATED, KS, p.cb, p.tile_rows, p.wave_tiles, MX_CONSUMERS) <= 80 * 1024) {
        with_act(act, [&](auto which) {
            constexpr int ACT = decltype(which)::value;
            if constexpr (GATED || ACT != KSMM_ACT_SILU) {
                static const int registers = mx_registers((const void *)&ks_mx_held_kernel<T, LAST, D, GATED, ACT, KS>);
                if (registers <= 80) most = mx_held_splits(p, 2);  // (six waves of each SIMD's 512)
            }
        });
    }
    p.row_splits = (int)std::min(p.token_tiles, most);
    const int64_t grid = mx_held_groups(p) * p.row_splits;
    if (grid > 0x7fffffffLL) return KSMM_ERR_TOO_LARGE;
    const int lds = (int)mx_held_lds(D, GATED, KS, p.cb, p.tile_rows, p.wave_tiles, MX_CONSUMERS);
    int rc = KSMM_OK;
    with_act(act, [&](auto which) {
        constexpr int ACT = decltype(which)::value;
        if constexpr (GATED || ACT != KSMM_ACT_SILU) {
            auto fn = &ks_mx_held_kernel<T, LAST, D, GATED, ACT, KS>;
            if (lds > 64 * 1024) rc = ensure_dynamic_lds((const void *)fn, (int)MX_LDS_ALL);  // (set once a kernel: for all of its sizes)
            if (rc == KSMM_OK) rc = mx_launch(fn, p, grid, 64 * (MX_CONSUMERS + MX_PRODUCERS), lds, s);
        }
    });
    return rc;
}

// steps of 64 along c that a kernel is made for
template <typename T, bool LAST, int D, bool GATED, int KS, int... MORE> int mx_held(const MxProduct &p, int act, hipStream_t s)
{
    // registers (168 of them): the weights' codes, sums and results of a wave; with more it spills (4 d_i: all of them live longer)
    constexpr int SIZE = (int)sizeof(T), HELD = 4 * D * (GATED ? 2 : 1) * KS + 16 * (GATED ? 2 : 1) + 4 * D * SIZE;
    constexpr bool fits = D < 4 ? HELD <= (D == 3 ? 104 : 112) : SIZE == 2 && D * (GATED ? 2 : 1) * KS <= 8;
    if constexpr (fits) {
        if (p.cb <= 2 * KS) return mx_launch_held<T, LAST, D, GATED, KS>(p, act, s);
        if constexpr (sizeof...(MORE) > 0) return mx_held<T, LAST, D, GATED, MORE...>(p, act, s);
    }
    return KSMM_ERR_BAD_ALGO;
}

template <typename T, bool LAST, int D, bool GATED> int mx_pick(const MxProduct &p, int act, hipStream_t s)
{
    const int unit = mx_unit_of(p.d, LAST), chunk = mx_chunk_of(unit, LAST);
    auto groups = [&](int rows) { return (p.batch + rows - 1) / rows * p.a * ((p.d + unit - 1) / unit) * ((p.b + 32 * chunk - 1) / (32 * chunk)); };
    if constexpr (D > 0) {
        // fewer than these are done sooner by workgroups of one step, which all begin at once: (1,768,192,2) gated fp16 of 32 rows in 4.9 us
        // for 7.2, of 1000 in 6.6 for 7.8; with 252 of them 4000 rows of (2,96,72,3) in fp32 take 9.4 for 8.2
        if (groups(32) > 192 && p.batch >= mx_pairs<T>(LAST, 1)) {
            const int rc = mx_held<T, LAST, D, GATED, 1, 2, 3, 4, 6, 8, 16>(p, act, s);
            if (rc != KSMM_ERR_BAD_ALGO) return rc;
        }
    }
    // twice the rows for the same weights, where that leaves a workgroup for a compute unit without splits, or there are many more weights than x
    // ((1,1536,384,2) gated fp16 of 3136 rows 35 -> 28 us, (1,128,128,8) 12 -> 17)
    const bool many = (p.batch + 63) / 64 * p.a * ((p.d + unit - 1) / unit) >= 256, heavy = (GATED ? 2 : 1) * p.b >= 256 * (int)sizeof(T) && groups(64) >= 256;
    if (p.batch > 32 && (many || heavy) && mx_wide_lds(2, p.c, p.d, (int)sizeof(T), LAST) <= MX_LDS_MOST) return mx_launch_wide<T, LAST, D, 2, GATED>(p, act, s);
    return mx_launch_wide<T, LAST, D, 1, GATED>(p, act, s);
}

template <typename T, bool GATED> int mx_last(const MxProduct &p, int act, hipStream_t s)
{
    return p.x_scales ? mx_pick<T, true, -1, GATED>(p, act, s) : mx_pick<T, true, 1, GATED>(p, act, s);
}
template <typename T, bool GATED> int mx_first(const MxProduct &p, int act, hipStream_t s)
{
    switch (p.x_scales ? -1 : p.d) {
    case -1: return mx_pick<T, false, -1, GATED>(p, act, s);
    case 1: return mx_pick<T, false, 1, GATED>(p, act, s);
    case 2: return mx_pick<T, false, 2, GATED>(p, act, s);
    case 3: return mx_pick<T, false, 3, GATED>(p, act, s);
    case 4: return mx_pick<T, false, 4, GATED>(p, act, s);
    default: return mx_pick<T, false, 0, GATED>(p, act, s);
    }
}

}  // namespace

}  // namespace ksmm
