// Gradients of what an activation was applied to, of products of microscaled 4-bit numbers: z is computed again.
//
//     dz = dy act'(z),  gated: dg = dy u act'(g), du = dy act(g)
//
// What is kept of the forward pass are the operands' codes, 17 bytes for 32 values; of a call that writes z and another one that reads it
// again two of the five passes over tensors of b features are left out.  The work is that of the forward kernel whose weights are in
// registers: eight waves (four) multiply and store, four bring the next step's codes of x and its dy into LDS, as they lie.
// What bounds it: HBM.  (1,768,192,2) gated in fp16, 25088 rows: 236 MB in 46 us, 5.1 TB/s, what a copy reaches; the kernel that multiplies
// the values in fp16 once more takes 80.
// dz has the tensors' type, as gradients between two layers have: in fp16 it is rounded before dx, dW and dbias sum it, 2.9e-4 off
// (rms) for 2.1e-4 of one rounding alone.  In 32 bits its traffic would be 390 MB for 236, and dx and dW, 115 us of a pass, were on fp32
// matrix cores, at an eighth of the rate.
#pragma once
#include "ksmm_mx_product.h"

namespace ksmm {

namespace {

// waves that multiply: with more than 4 bytes of D a value the dy of eight would not fit LDS, nor their registers the gradients
template <typename T, int D> constexpr int mx_slope_waves() { return D * (int)sizeof(T) <= 4 ? MX_CONSUMERS : MX_CONSUMERS / 2; }

// bytes from one line of dy in LDS (a row of the batch; batch-size-last an output) to the next: 16 more than there are, for the banks' sake
template <typename T, bool LAST, int D> __host__ __device__ constexpr int mx_dy_pitch(int rows, int tiles) { return (LAST ? rows : tiles * 32 * D) * (int)sizeof(T) + 16; }

template <typename T, bool LAST, int D, bool GATED, int ACT, int KS>
__global__ __launch_bounds__(64 * (mx_slope_waves<T, D>() + MX_PRODUCERS)) void ks_mx_slope_kernel(MxProduct p)
{
    constexpr int G = GATED ? 2 : 1, SB = mx_scale_bytes(KS), R = mx_rounds(KS, 1), E = 16 / (int)sizeof(T), THREADS = 64 * MX_PRODUCERS, C = mx_slope_waves<T, D>();
    constexpr int V = 32 * C * 32 * D / E / THREADS;  // vectors of dy that a producer's thread takes
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int TN = p.tile_rows, pitch = mx_dy_pitch<T, LAST, D>(TN, p.wave_tiles), scales_at = D * TN * p.slots * 16, dy_at = scales_at + D * TN * 2 * SB;
    const int buffer = dy_at + (LAST ? p.wave_tiles * 32 : TN) * pitch;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, half = lane >> 5;
    const int run = 16 * ((l32 >> 2) & 1) + 4 * (l32 >> 3) + (l32 & 3);  // the row that this lane reads of the operand whose rows are dealt out
    int blk = (int)(p.first + blockIdx.x);
    const int first = blk % p.row_splits;
    blk /= p.row_splits;
    const int unit = blk % p.units, ai = unit / p.runs, d0 = (unit - ai * p.runs) * D;
    const int tile0 = blk / p.units * p.wave_tiles;
    float *const bias = (float *)(smem + 2 * buffer);
    uint8_t *const stage = smem + 2 * buffer + p.wave_tiles * G * D * 128 + wave * MX_STAGE;
    const int tasks = TN * p.cb, batch = (int)p.batch, row_tiles = (int)p.token_tiles;
    auto prepare = [&] { mx_prepare<T, D, G>(p, smem + scales_at, buffer, D * TN * SB / 2, bias, ai, d0, tile0); };

    if (wave >= C) {
        const int t0 = threadIdx.x - 64 * C;
        const MxDiv by_cb(p.cb), by_line(LAST ? TN / E : p.wave_tiles * 32 * D / E);
        const int outs = p.b - tile0 * 32;  // from the workgroup's first tile on
        uint4_t code[D][R], dy[V];
        int scale[D][R];
        // task r's row of the step and its block, or a row that never is there
        auto place = [&](int r, int &n, int &kb) {
            const int t = t0 + r * THREADS;
            n = by_cb(t);
            kb = t - n * p.cb;
            if (t >= tasks) n = 1 << 30;
        };
        auto fetch = [&](int n0) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                int n, kb;
                place(r, n, kb);
                if (n >= batch - n0) continue;
#pragma unroll
                for (int j = 0; j < D; ++j) {
                    const int64_t block = (((int64_t)ai * p.d + d0 + j) * p.batch + n0 + n) * p.cb + kb;
                    code[j][r] = *(const uint4_t *)((const uint8_t *)p.x + block * 16);
                    scale[j][r] = p.x_scales[block];
                }
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int i = t0 + v * THREADS, line = by_line(i), e = (i - line * (int)by_line.d) * E;
                int left = LAST ? (line < outs ? batch - n0 - e : 0) : line < batch - n0 ? outs * D - e : 0;  // values from this vector on
                if (left <= 0) continue;
                const T *from = (const T *)p.dy + (LAST ? (((int64_t)ai * p.b + tile0 * 32 + line) * p.d + d0) * p.batch + n0 + e
                                                        : ((((int64_t)n0 + line) * p.a + ai) * p.b + tile0 * 32) * D + e);
                if (left >= E) {
                    dy[v] = *(const uint4_any *)from;
                } else {
                    asm volatile("" : "+v"(left));  // (offsets are not to be kept in registers from one step to the next)
                    T part[E];
#pragma unroll
                    for (int k = 0; k < E; ++k) part[k] = from[k < left ? k : 0];
                    __builtin_memcpy(&dy[v], part, 16);
                }
            }
        };
        auto keep = [&](int n0, int which) {
            uint8_t *const codes = smem + which * buffer, *const scales = codes + scales_at, *const lines = codes + dy_at;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                int n, kb;
                place(r, n, kb);
                if (n >= batch - n0) continue;  // (whatever LDS has, it is another column of the product)
#pragma unroll
                for (int j = 0; j < D; ++j) {
                    const int row = j * TN + n;
                    *(uint4_t *)(codes + (row * p.slots + kb) * 16) = code[j][r];
                    scales[row * 2 * SB + (kb & 1) * SB + (kb >> 1)] = (uint8_t)scale[j][r];
                }
            }
            // (values that are not there: they are not stored)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int i = t0 + v * THREADS, line = by_line(i), e = (i - line * (int)by_line.d) * E;
                *(uint4_t *)(lines + line * pitch + e * (int)sizeof(T)) = dy[v];
            }
        };
        fetch(first * TN);
        prepare();
        __syncthreads();
        int which = 0;
        for (int tile = first; tile < row_tiles; tile += p.row_splits, which ^= 1) {
            keep(tile * TN, which);
            if (tile + p.row_splits < row_tiles) fetch((tile + p.row_splits) * TN);
            __syncthreads();
        }
        return;
    }

    const int wb = wave & (p.wave_tiles - 1), wt = wave / p.wave_tiles, per_wave = TN / 32 / (C / p.wave_tiles);
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
        const uint8_t *const codes = smem + which * buffer, *const scales = codes + scales_at, *const lines = codes + dy_at;
        for (int t = wt * per_wave; t < (wt + 1) * per_wave && t * 32 < here; ++t) {
            // a lane's 16 outputs of a row, of all D (batch-size-last: 16 rows of one output)
            const uint8_t *const from = LAST ? lines + (wb * 32 + l32) * pitch + (t * 32 + 16 * half) * (int)sizeof(T)
                                             : lines + (t * 32 + l32) * pitch + (wb * 32 + 16 * half) * D * (int)sizeof(T);
            T v[16 * D], u[GATED ? 16 * D : 1];
#pragma unroll
            for (int i = 0; i < 16 * D / E; ++i) {
                const uint4_t q = *(const uint4_t *)(from + i * 16);
                __builtin_memcpy(&v[i * E], &q, 16);
            }
#pragma unroll
            for (int j = 0; j < D; ++j) {
                float16_t acc[G];
                held.sums(codes, scales, p.slots, j * TN + t * 32 + (LAST ? run : l32), j, l32, half, p.bias ? bias + wb * G * D * 32 : nullptr, acc);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float slope;
                    const float dy = (float)v[i * D + j], f = activate<T, ACT, true, true>(acc[0][i], slope);
                    float down = dy * slope, other = dy * f;
                    if constexpr (GATED) down *= acc[1][i];
                    asm volatile("" : "+v"(down), "+v"(other));  // (here, and not behind the products of all D, whose sums would not fit the registers)
                    v[i * D + j] = (T)down;
                    if constexpr (GATED) u[i * D + j] = (T)other;
                }
            }
            mx_results<T, LAST, D>(p, v, ai, d0, bt, lane, n0, t, here, stage, G * p.b);
            if constexpr (GATED) mx_results<T, LAST, D>(p, u, ai, d0, bt, lane, n0, t, here, stage, G * p.b, p.b);
        }
    }
}

template <typename T, bool LAST, int D, bool GATED, int KS> int mx_launch_slope(MxProduct p, int act, hipStream_t s)
{
    constexpr int C = mx_slope_waves<T, D>();
    mx_held_sizes(p, LAST, C, 64 * MX_PRODUCERS * mx_rounds(KS, 1));
    auto bytes = [&] {
        return mx_held_lds(D, GATED, KS, p.cb, p.tile_rows, p.wave_tiles, C) + 2LL * (LAST ? p.wave_tiles * 32 : p.tile_rows) * mx_dy_pitch<T, LAST, D>(p.tile_rows, p.wave_tiles);
    };
    while (bytes() > MX_LDS_ALL && p.wave_tiles < C) mx_held_tiles(p, C, 2 * p.wave_tiles);  // (fewer rows of codes)
    const int64_t lds = bytes();
    if (lds > MX_LDS_ALL) return KSMM_ERR_BAD_ALGO;
    p.row_splits = (int)std::min(p.token_tiles, mx_held_splits(p, 1));
    const int64_t grid = mx_held_groups(p) * p.row_splits;
    if (grid > 0x7fffffffLL) return KSMM_ERR_TOO_LARGE;
    if (!p.y) return KSMM_OK;  // (asked only)
    int rc = KSMM_OK;
    with_act(act, [&](auto which) {
        constexpr int ACT = decltype(which)::value;
        if constexpr (GATED || ACT == KSMM_ACT_GELU) {
            auto fn = &ks_mx_slope_kernel<T, LAST, D, GATED, ACT, KS>;
            if (lds > 64 * 1024) rc = ensure_dynamic_lds((const void *)fn, (int)MX_LDS_ALL);  // (set once a kernel: for all of its sizes)
            if (rc == KSMM_OK) rc = mx_launch(fn, p, grid, 64 * (C + MX_PRODUCERS), lds, s);
        }
    });
    return rc;
}

template <typename T, bool LAST, int D, bool GATED, int KS, int... MORE> int mx_slope_steps(const MxProduct &p, int act, hipStream_t s)
{
    // registers, 168 of them or 256: the weights' codes, sums, and gradients of gate and up
    constexpr int G = GATED ? 2 : 1, HELD = 4 * D * G * KS + 16 * G + 4 * D * G * (int)sizeof(T);
    if constexpr (HELD <= (mx_slope_waves<T, D>() == MX_CONSUMERS ? 112 : 176)) {
        if (p.cb <= 2 * KS) return mx_launch_slope<T, LAST, D, GATED, KS>(p, act, s);
        if constexpr (sizeof...(MORE) > 0) return mx_slope_steps<T, LAST, D, GATED, MORE...>(p, act, s);
    }
    return KSMM_ERR_BAD_ALGO;
}
template <typename T, bool LAST, int D> int mx_slope(const MxProduct &p, bool gated, int act, hipStream_t s)
{
    return gated ? mx_slope_steps<T, LAST, D, true, 1, 2, 3, 4, 6, 8>(p, act, s) : mx_slope_steps<T, LAST, D, false, 1, 2, 3, 4, 6, 8>(p, act, s);
}

}  // namespace

}  // namespace ksmm
