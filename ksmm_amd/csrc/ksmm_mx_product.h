// Products of microscaled 4-bit numbers, quantised on the way: the kernel, for one type of x and y.
//
// A workgroup takes 32 * TT rows of the batch and a unit of work: one a_i and D consecutive d_i (batch-size-last one d_i).  It
// quantises its rows of x into LDS, where they take 17 bytes for 32 values, and its waves multiply them with tiles of 32
// outputs, whose codes come from the caches.  Every row of a tile's operand is read where the lane that holds the result wants it:
// row 8j + 4h + i of a tile is its row 16h + 4j + i, so that a lane ends up with 16 consecutive outputs of a row of the batch
// (batch-size-last: 16 consecutive rows of one output), which with those of all D leave as whole vectors.
#pragma once
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

constexpr int MX_WAVES = 4;

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

template <typename T, bool LAST, int D, int TT, bool GATED, int ACT> __global__ __launch_bounds__(64 * MX_WAVES) void ks_mx_fused_kernel(MxProduct p)
{
    constexpr int TN = 32 * TT, G = GATED ? 2 : 1;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    uint8_t *const codes = smem, *const scales = smem + (size_t)D * TN * p.slots * 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, half = lane >> 5;
    const int run = 16 * ((l32 >> 2) & 1) + 4 * (l32 >> 3) + (l32 & 3);  // the row that this lane reads of the operand whose rows are dealt out
    int64_t blk = blockIdx.x;
    const int split = (int)(blk % p.splits);
    blk /= p.splits;
    const int first_unit = (int)(blk % p.unit_groups) * p.units_per;
    const int64_t n0 = blk / p.unit_groups * TN;
    const int here = (int)(p.batch - n0 < TN ? p.batch - n0 : TN);  // rows of the batch
    const int rows_w = G * p.b, last_unit = first_unit + p.units_per < p.units ? first_unit + p.units_per : p.units;
    const int tile_end = (split + 1) * p.tiles_per < p.b_tiles ? (split + 1) * p.tiles_per : p.b_tiles;

    for (int unit = first_unit; unit < last_unit; ++unit) {
        const int ai = unit / p.runs, d0 = (unit - ai * p.runs) * D;
        if (unit > first_unit) __syncthreads();  // (the codes before are no longer read)
        // ---- x into LDS
        if (p.x_scales) {
            for (int t = threadIdx.x; t < D * TN * p.cb; t += 64 * MX_WAVES) {
                const int kb = t % p.cb, row = t / p.cb, j = row / TN, n = row - j * TN;
                uint4_t code = {0, 0, 0, 0};
                int scale = 127;
                if (n < here) {
                    const int64_t block = (((int64_t)ai * p.d + d0 + j) * p.batch + n0 + n) * p.cb + kb;
                    code = *(const uint4_t *)((const uint8_t *)p.x + block * 16);
                    scale = p.x_scales[block];
                }
                *(uint4_t *)(codes + ((size_t)row * p.slots + kb) * 16) = code;
                scales[row * p.cb + kb] = (uint8_t)scale;
            }
        } else if constexpr (LAST) {
            constexpr int V = sizeof(T) == 2 ? 4 : 2;
            for (int t = threadIdx.x; t < TN / V * p.cb; t += 64 * MX_WAVES) {
                const int kb = t / (TN / V), n = (t - kb * (TN / V)) * V;
                MxGroup<T, V> g;
                const int there = here - n < 0 ? 0 : here - n < V ? here - n : V, count = p.c - kb * 32;
                const int64_t step = (int64_t)p.d * p.batch;
                mx_load<T, V>(g, (const T *)p.x + (((int64_t)ai * p.c + kb * 32) * p.d + d0) * p.batch + n0 + n, step, there ? count : 0, there);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    uint4_t code;
                    const int scale = mx_quantize<T, V>(g, j, code);
                    *(uint4_t *)(codes + ((size_t)(n + j) * p.slots + kb) * 16) = code;
                    scales[(n + j) * p.cb + kb] = (uint8_t)scale;
                }
            }
        } else {
            for (int t = threadIdx.x; t < TN * p.cb; t += 64 * MX_WAVES) {
                const int n = t / p.cb, kb = t - n * p.cb;
                MxGroup<T, D> g;
                mx_load<T, D>(g, (const T *)p.x + (((n0 + n) * p.a + ai) * p.c + kb * 32) * p.d + d0, p.d, n < here ? p.c - kb * 32 : 0, D);
#pragma unroll
                for (int j = 0; j < D; ++j) {
                    uint4_t code;
                    const int scale = mx_quantize<T, D>(g, j, code);
                    *(uint4_t *)(codes + ((size_t)(j * TN + n) * p.slots + kb) * 16) = code;
                    scales[(j * TN + n) * p.cb + kb] = (uint8_t)scale;
                }
            }
        }
        __syncthreads();
        // ---- products
        for (int bt = split * p.tiles_per + wave; bt < tile_end; bt += MX_WAVES) {
            float16_t acc[TT][D][G];
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
                for (int j = 0; j < D; ++j)
#pragma unroll
                    for (int q = 0; q < G; ++q) acc[t][j][q] = float16_t{};
            // (outputs behind the last one are read as the last one and not stored)
            const int wo = bt * 32 + (LAST ? l32 : run), o = wo < p.b ? wo : p.b - 1;
            const int xr = LAST ? run : l32;
            int64_t at[D][G];
#pragma unroll
            for (int j = 0; j < D; ++j)
#pragma unroll
                for (int q = 0; q < G; ++q) at[j][q] = (((int64_t)ai * p.d + d0 + j) * rows_w + q * p.b + o) * p.cb;
            for (int k0 = 0; k0 < p.cb; k0 += 2) {
                const int kb = k0 + half;
                const bool there = kb < p.cb;
                uint4_t w[D][G];
                int sw[D][G];
#pragma unroll
                for (int j = 0; j < D; ++j)
#pragma unroll
                    for (int q = 0; q < G; ++q) {
                        w[j][q] = there ? *(const uint4_t *)(p.w + (at[j][q] + kb) * 16) : uint4_t{0, 0, 0, 0};
                        sw[j][q] = there ? p.w_scales[at[j][q] + kb] : 127;
                    }
#pragma unroll
                for (int t = 0; t < TT; ++t)
#pragma unroll
                    for (int j = 0; j < D; ++j) {
                        const int row = j * TN + t * 32 + xr;
                        const uint4_t x = there ? *(const uint4_t *)(codes + ((size_t)row * p.slots + kb) * 16) : uint4_t{0, 0, 0, 0};
                        const int sx = there ? scales[row * p.cb + kb] : 127;
#pragma unroll
                        for (int q = 0; q < G; ++q)
                            acc[t][j][q] = LAST ? mx_mfma(x, sx, w[j][q], sw[j][q], acc[t][j][q]) : mx_mfma(w[j][q], sw[j][q], x, sx, acc[t][j][q]);
                    }
            }
            // ---- results
            const T *const bias = (const T *)p.bias;
            if constexpr (LAST) {
                float add[G];
#pragma unroll
                for (int q = 0; q < G; ++q) add[q] = bias ? (float)bias[((int64_t)ai * rows_w + q * p.b + o) * p.d + d0] : 0.f;
                T *const y = (T *)p.y + (((int64_t)ai * p.b + wo) * p.d + d0) * p.batch + n0;
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                    const int n = t * 32 + 16 * half;
                    T v[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float slope, z = activate<T, ACT, false>(acc[t][0][0][i] + add[0], slope);
                        if constexpr (GATED) z *= acc[t][0][G - 1][i] + add[G - 1];
                        v[i] = (T)z;
                    }
                    if (wo >= p.b) continue;
                    if (n + 16 <= here) {
                        mx_store<T, 16>(y + n, v);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (n + i < here) y[n + i] = v[i];
                    }
                }
            } else {
                const int o0 = bt * 32 + 16 * half;
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                    const int n = t * 32 + l32;
                    T v[16 * D];
#pragma unroll
                    for (int j = 0; j < D; ++j)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int oi = o0 + i < p.b ? o0 + i : p.b - 1;
                            float slope, z = acc[t][j][0][i];
                            if (bias) z += (float)bias[((int64_t)ai * rows_w + oi) * p.d + d0 + j];
                            z = activate<T, ACT, false>(z, slope);
                            if constexpr (GATED) {
                                float u = acc[t][j][G - 1][i];
                                if (bias) u += (float)bias[((int64_t)ai * rows_w + p.b + oi) * p.d + d0 + j];
                                z *= u;
                            }
                            v[i * D + j] = (T)z;
                        }
                    if (n >= here) continue;
                    T *const y = (T *)p.y + (((n0 + n) * p.a + ai) * p.b + o0) * p.d + d0;
                    if (p.d == D && o0 + 16 <= p.b) {
                        mx_store<T, 16 * D>(y, v);
                    } else {
                        struct __attribute__((packed, aligned(sizeof(T)))) Run {
                            T e[D];
                        };
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            if (o0 + i >= p.b) continue;
                            Run r;
#pragma unroll
                            for (int j = 0; j < D; ++j) r.e[j] = v[i * D + j];
                            *(Run *)(y + (int64_t)i * p.d) = r;
                        }
                    }
                }
            }
        }
    }
}

// d_i that a unit takes: all of up to four, else a divisor
inline int mx_run_of(int d) { return d <= 4 ? d : d % 4 == 0 ? 4 : d % 3 == 0 ? 3 : d % 2 == 0 ? 2 : 1; }
// tiles of 32 rows: what 128 accumulators hold
constexpr int mx_rows_of(int d, bool gated) { return d * (gated ? 2 : 1) <= 2 ? 4 : d * (gated ? 2 : 1) <= 4 ? 2 : 1; }
inline int64_t mx_lds(int tt, int d, int cb) { return (int64_t)d * 32 * tt * (16 * (cb | 1) + cb); }
constexpr int64_t MX_LDS_MOST = 80 * 1024;  // two workgroups a compute unit

template <typename T, bool LAST, int D, int TT, bool GATED> int mx_launch(MxProduct p, int act, hipStream_t s)
{
    p.slots = p.cb | 1;
    p.runs = p.d / D;
    p.units = p.a * p.runs;
    p.b_tiles = (p.b + 31) / 32;
    p.token_tiles = (p.batch + 32 * TT - 1) / (32 * TT);
    // units whose values share a line of 128 bytes go to one workgroup, unless there are few
    p.units_per = 1;
    if (!LAST) {
        const int64_t bytes = (int64_t)(p.d == D ? p.c * D : D) * (int64_t)sizeof(T);
        const int64_t share = bytes >= 128 ? 1 : 128 / bytes;
        if (p.token_tiles * p.units / share >= 1024) p.units_per = (int)(share < p.units ? share : p.units);
    }
    p.unit_groups = (p.units + p.units_per - 1) / p.units_per;
    // outputs are split over workgroups, each of which quantises its rows anew, until there are 1024
    const int64_t groups = p.token_tiles * p.unit_groups;
    const int most = (p.b_tiles + MX_WAVES - 1) / MX_WAVES;
    const int64_t want = groups >= 1024 ? 1 : (1024 + groups - 1) / groups;
    p.splits = (int)(want < most ? want : most);
    p.tiles_per = (p.b_tiles + p.splits - 1) / p.splits;
    p.splits = (p.b_tiles + p.tiles_per - 1) / p.tiles_per;
    const int64_t grid = groups * p.splits;
    if (grid > 0x7fffffffLL) return KSMM_ERR_TOO_LARGE;
    const int lds = (int)mx_lds(TT, D, p.cb);
    int rc = KSMM_OK;
    with_act(act, [&](auto which) {
        constexpr int ACT = decltype(which)::value;
        if constexpr (GATED || ACT != KSMM_ACT_SILU) {
            auto fn = &ks_mx_fused_kernel<T, LAST, D, TT, GATED, ACT>;
            if (lds > 64 * 1024) rc = ensure_dynamic_lds((const void *)fn, lds);
            if (rc != KSMM_OK) return;
            hipLaunchKernelGGL(fn, dim3((unsigned)grid), dim3(64 * MX_WAVES), lds, s, p);
            if (hipGetLastError() != hipSuccess) rc = KSMM_ERR_LAUNCH;
        }
    });
    return rc;
}

template <typename T, bool LAST, int D, bool GATED> int mx_pick(const MxProduct &p, int act, hipStream_t s)
{
    constexpr int TT = mx_rows_of(D, GATED);
    if constexpr (TT > 1) {
        if (p.batch > 32 && mx_lds(TT, D, p.cb) <= MX_LDS_MOST) return mx_launch<T, LAST, D, TT, GATED>(p, act, s);
    }
    return mx_launch<T, LAST, D, 1, GATED>(p, act, s);
}

template <typename T> int mx_run(const MxProduct &p, bool last, bool gated, int act, hipStream_t s)
{
    if (last) return gated ? mx_pick<T, true, 1, true>(p, act, s) : mx_pick<T, true, 1, false>(p, act, s);
    switch (mx_run_of(p.d)) {
    case 1: return gated ? mx_pick<T, false, 1, true>(p, act, s) : mx_pick<T, false, 1, false>(p, act, s);
    case 2: return gated ? mx_pick<T, false, 2, true>(p, act, s) : mx_pick<T, false, 2, false>(p, act, s);
    case 3: return gated ? mx_pick<T, false, 3, true>(p, act, s) : mx_pick<T, false, 3, false>(p, act, s);
    default: return gated ? mx_pick<T, false, 4, true>(p, act, s) : mx_pick<T, false, 4, false>(p, act, s);
    }
}

}  // namespace

}  // namespace ksmm
