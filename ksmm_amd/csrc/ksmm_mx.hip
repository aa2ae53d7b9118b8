// Kronecker-sparse products of microscaled 4-bit numbers (e2m1, blocks of 32 along c with a power of two in common).
//
//     xq[a_i, c_i, d_i, n] = 2^e rne(x / 2^e),  e = floor(log2 max |x| of the block) - 2
//     y[a_i, b_i, d_i, n]  = act(sum_c Wq[a_i, b_i, c_i, d_i] xq[a_i, c_i, d_i, n] + bias[a_i, b_i, d_i])
//
// Operands are kept as the a*d matrices that the products take, (a*d, rows, c) with c in blocks of 32, the last one filled
// with zeros: 16 bytes of codes a block, the even place in the lower half of a byte, and a byte of scale.  That is what a lane
// of the scaled matrix instructions holds: 32 numbers of one row and their scale.
//
// Here: conversions, the products of rows whose codes no workgroup's LDS holds, and the C entry points.  Conversions are short workgroups, of
// which each loads once and waits for it: 24.4 MB of 25088 x 384 in fp16 take 6.6 to 7.0 us to codes and 8.0 back (medians, of one run's dispatches
// 6.3 and 7.8 at least), 22.6 MB of 768 x 6501 in fp32 batch-size-last 8.7 and 7.8, where a copy takes 4.7 and 4.4; of that 2 us are a
// launch's start and end.
#include "ksmm_mx_product.h"

namespace ksmm {

namespace {

struct MxOperand {
    const void *x;  // dequantising: written
    uint8_t *codes, *scales;
    int64_t rows;
    int a, c, d, cb;
    bool last;
    uint32_t first;  // workgroup of the launch, of all (batch-size-last)
    int64_t blocks;  // a * d * rows * cb
    bool small;      // tasks that the two divide by multiplying
    MxDiv by_cb, by_a;
};
// task t as (n, ai, kb), t = (n a + ai) cb + kb
__device__ __forceinline__ int64_t mx_place(const MxOperand &p, int64_t t, int &ai, int &kb)
{
    if (p.small) {
        const int i = (int)t, u = p.by_cb(i), n = p.by_a(u);
        kb = i - u * p.cb;
        ai = u - n * p.a;
        return n;
    }
    const int64_t u = t / p.cb, n = u / p.a;
    kb = (int)(t - u * p.cb);
    ai = (int)(u - n * p.a);
    return n;
}
constexpr int THREADS = 256;

// ---- batch-size-first, all d_i of up to four in a row: four lanes a block, so that lanes that follow one another read and write 16 * D
// bytes that do (a block a lane took 24 us for 25088 x 384 in fp16)
template <typename T, int D, bool BACK> __device__ __forceinline__ void mx_rows(const MxOperand &p, int64_t group, int64_t groups)
{
    constexpr int E = 16 / (int)sizeof(T), N = 8 * D;
    const int64_t tasks = p.blocks / D * 4;
    const int quarter = threadIdx.x & 3;
    for (int64_t i = group * THREADS + threadIdx.x; i < tasks; i += groups * THREADS) {
        int ai, kb;
        const int64_t n = mx_place(p, i >> 2, ai, kb);
        const int count = p.c - kb * 32 - quarter * 8;
        T *const x = (T *)p.x + ((n * p.a + ai) * p.c + kb * 32 + quarter * 8) * D;
        T v[N];
        if constexpr (!BACK) {
            if (count >= 8) {
#pragma unroll
                for (int j = 0; j < N / E; ++j) {
                    const uint4_t q = *(const uint4_any *)(x + j * E);
                    __builtin_memcpy(&v[j * E], &q, 16);
                }
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] = j < count * D ? x[j] : (T)0;
            }
        }
#pragma unroll
        for (int j = 0; j < D; ++j) {
            const int64_t block = (((int64_t)ai * D + j) * p.rows + n) * p.cb + kb;
            if constexpr (BACK) {
                float e[8];
                mx_decode8(((const uint32_t *)p.codes)[block * 4 + quarter], e);
                const float power = mx_scale_value(p.scales[block]);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k * D + j] = (T)(e[k] * power);
            } else {
                float e[8];
                uint32_t top = 0;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    e[k] = (float)v[k * D + j];
                    top = max(top, mx_bits(e[k]));
                }
                top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xb1, 0xf, 0xf, true));  // lanes 1 0 3 2
                top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4e, 0xf, 0xf, true));  // 2 3 0 1
                const int scale = mx_scale(top);
                ((uint32_t *)p.codes)[block * 4 + quarter] = scale == MX_NAN ? 0u : mx_encode8(e, mx_power(scale));
                if (quarter == 0) p.scales[block] = (uint8_t)scale;
            }
        }
        if constexpr (BACK) {
            if (count >= 8) {
#pragma unroll
                for (int j = 0; j < N / E; ++j) {
                    uint4_t q;
                    __builtin_memcpy(&q, &v[j * E], 16);
                    *(uint4_any *)(x + j * E) = q;
                }
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (j < count * D) x[j] = v[j];
            }
        }
    }
}

// ---- batch-size-first, D of more d_i: blocks that lie side by side, a thread each
template <typename T, int D, bool BACK> __device__ __forceinline__ void mx_runs(const MxOperand &p, int64_t group, int64_t groups)
{
    struct __attribute__((packed, aligned(sizeof(T)))) Run {
        T e[D];
    };
    const int64_t tasks = p.blocks / D;
    const int runs = p.d / D;
    for (int64_t i = group * THREADS + threadIdx.x; i < tasks; i += groups * THREADS) {
        const int64_t t = i / runs;
        int ai, kb;
        const int64_t n = mx_place(p, t, ai, kb);
        const int d0 = (int)(i - t * runs) * D, count = p.c - kb * 32;
        T *const x = (T *)p.x + ((n * p.a + ai) * p.c + kb * 32) * p.d + d0;
        MxGroup<T, D> g;
        if constexpr (!BACK) mx_load<T, D>(g, x, p.d, count);
#pragma unroll
        for (int j = 0; j < D; ++j) {
            const int64_t block = (((int64_t)ai * p.d + d0 + j) * p.rows + n) * p.cb + kb;
            if constexpr (BACK) {
                const uint4_t code = *(const uint4_t *)(p.codes + block * 16);
                const float power = mx_scale_value(p.scales[block]);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float e[8];
                    mx_decode8(code[q], e);
#pragma unroll
                    for (int k = 0; k < 8; ++k) g.v[(8 * q + k) * D + j] = (T)(e[k] * power);
                }
            } else {
                uint4_t code;
                const int scale = mx_quantize<T, D>(g, j, count, code);
                *(uint4_t *)(p.codes + block * 16) = code;
                p.scales[block] = (uint8_t)scale;
            }
        }
        if constexpr (BACK) {
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                Run r;
#pragma unroll
                for (int j = 0; j < D; ++j) r.e[j] = g.v[k * D + j];
                if (k < count) *(Run *)(x + (int64_t)k * p.d) = r;
            }
        }
    }
}

// ---- batch-size-last: a workgroup takes 64 rows of four blocks of a d_i.  Lanes lie along the rows in x, and along the blocks of a row
// among the codes, which change places in LDS.
template <typename T, bool BACK> __device__ __forceinline__ void mx_columns(const MxOperand &p, uint32_t group)
{
    __shared__ uint4_t codes[64 * 4 + 4];
    __shared__ uint8_t scales[64 * 4];
    // (in 32 bits: a workgroup begins with these, and lives for 32 loads)
    const uint32_t quads = (uint32_t)(p.cb + 3) / 4, u = group / quads, row_tiles = (uint32_t)((p.rows + 63) / 64), block_at = u / row_tiles;
    const int kb0 = (int)(group - u * quads) * 4, ai = (int)(block_at / (uint32_t)p.d), di = (int)block_at - ai * p.d;
    const int64_t n0 = (int64_t)(u - block_at * row_tiles) * 64;
    const int row = threadIdx.x & 63, kb = kb0 + (threadIdx.x >> 6), count = p.c - kb * 32;
    const int64_t step = (int64_t)p.d * p.rows, n = n0 + row;
    T *const x = (T *)p.x + (((int64_t)ai * p.c + kb * 32) * p.d + di) * p.rows + n;
    const int other = threadIdx.x >> 2, other_kb = kb0 + (threadIdx.x & 3);
    const int64_t block = (((int64_t)ai * p.d + di) * p.rows + n0 + other) * p.cb + other_kb;
    const bool there = n0 + other < p.rows && other_kb < p.cb;
    // (a row's four blocks are a slot of 16 bytes each, one more for every 16 rows, so that both sides meet few of the same banks)
    const int mine = row * 4 + (threadIdx.x >> 6) + row / 16, place = other * 4 + (threadIdx.x & 3) + other / 16;
    if constexpr (BACK) {
        if (there) {
            codes[place] = *(const uint4_t *)(p.codes + block * 16);
            scales[threadIdx.x] = p.scales[block];
        }
        __syncthreads();
        if (n >= p.rows || count <= 0) return;
        const uint4_t code = codes[mine];
        const float power = mx_scale_value(scales[row * 4 + (threadIdx.x >> 6)]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float e[8];
            mx_decode8(code[q], e);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (8 * q + k < count) x[(8 * q + k) * step] = (T)(e[k] * power);
        }
    } else {
        if (n < p.rows && count > 0) {
            MxGroup<T, 1> g;
            mx_load<T, 1>(g, x, step, count);
            uint4_t code;
            const int scale = mx_quantize<T, 1>(g, 0, count, code);
            codes[mine] = code;
            scales[row * 4 + (threadIdx.x >> 6)] = (uint8_t)scale;
        }
        __syncthreads();
        if (there) {
            *(uint4_t *)(p.codes + block * 16) = codes[place];
            p.scales[block] = scales[threadIdx.x];
        }
    }
}

template <typename T, int D, bool BACK> __global__ __launch_bounds__(THREADS) void ks_mx_rows_kernel(MxOperand p)
{
    mx_rows<T, D, BACK>(p, blockIdx.x, gridDim.x);
}
template <typename T, int D, bool BACK> __global__ __launch_bounds__(THREADS) void ks_mx_runs_kernel(MxOperand p)
{
    mx_runs<T, D, BACK>(p, blockIdx.x, gridDim.x);
}
template <typename T, bool BACK> __global__ __launch_bounds__(THREADS) void ks_mx_columns_kernel(MxOperand p)
{
    mx_columns<T, BACK>(p, p.first + blockIdx.x);
}
// ---- both operands of a product back to values, for its gradients: workgroups of the one behind those of the other (a launch each for
// (2,96,72,3) fp32, 1970 rows takes 6.6 us, this one 3.9).  D: d_i of x together, 0 batch-size-last
template <typename T, int D> __global__ __launch_bounds__(THREADS) void ks_mx_values_kernel(MxOperand x, MxOperand w, uint32_t w_groups)
{
    if (blockIdx.x < w_groups) {
        mx_columns<T, true>(w, blockIdx.x);
        return;
    }
    const uint32_t group = blockIdx.x - w_groups, groups = gridDim.x - w_groups;
    if constexpr (D == 0) {
        mx_columns<T, true>(x, group);
    } else {
        if (D == 3 || x.d == D)
            mx_rows<T, D, true>(x, group, groups);
        else if constexpr (D != 3)
            mx_runs<T, D, true>(x, group, groups);
    }
}

// 32 numbers and their scale of row `row` (< rows, else zeros), block kb (< cb, else zeros)
__device__ __forceinline__ int8_v mx_operand(const uint8_t *codes, const uint8_t *scales, int64_t row, bool there, int kb, int cb, int *scale)
{
    int8_v r = {0, 0, 0, 0, 0, 0, 0, 0};
    *scale = 127;
    if (there && kb < cb) {
        const uint4_t v = *(const uint4_t *)(codes + (row * cb + kb) * 16);
        r[0] = (int)v[0], r[1] = (int)v[1], r[2] = (int)v[2], r[3] = (int)v[3];
        *scale = scales[row * cb + kb];
    }
    return r;
}

// Codes beyond LDS (c of 8500 and more): operands from the caches, x quantised in a launch before.  (1,512,9000,1) fp16: one row 38 us, 4096 rows
// 139, 272 TF (c of 8000, which LDS holds: 20 and 81).
// A wave computes 32 outputs of 32 rows: row 8j + 4(lane / 32) + i of the tile is an output, column lane % 32 a row of the batch.
template <typename T, bool LAST, bool GATED, int ACT> __global__ __launch_bounds__(256) void ks_mx_product_kernel(MxProduct p)
{
    const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
    const int64_t tile = blockIdx.x * 4LL + (threadIdx.x >> 6);
    if (tile >= p.tiles) return;
    const int bt = (int)(tile % p.b_tiles);
    const int64_t nt = tile / p.b_tiles % p.token_tiles;
    const int block = (int)(tile / p.b_tiles / p.token_tiles), ai = block / p.d, di = block % p.d;
    const int rows_w = GATED ? 2 * p.b : p.b;
    const int64_t n = nt * 32 + l32;
    const int bi = bt * 32 + l32;
    float16_t acc = {}, up = {};
    for (int kb = half; kb - half < p.cb; kb += 2) {
        int sx, sw, su;
        const int8_v x = mx_operand((const uint8_t *)p.x, p.x_scales, (int64_t)block * p.batch + n, n < p.batch, kb, p.cb, &sx);
        const int64_t row = (int64_t)block * rows_w + bi;
        const int8_v w = mx_operand(p.w, p.w_scales, row, bi < p.b, kb, p.cb, &sw);
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, acc, 4, 4, 0, sw, 0, sx);
        if constexpr (GATED) {
            const int8_v u = mx_operand(p.w, p.w_scales, row + p.b, bi < p.b, kb, p.cb, &su);
            up = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(u, x, up, 4, 4, 0, su, 0, sx);
        }
    }
    if (n >= p.batch) return;
    const T *bias = (const T *)p.bias;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int o = bt * 32 + 8 * (i / 4) + 4 * half + (i & 3);
        if (o >= p.b) continue;
        float z = acc[i];
        if (bias) z += (float)bias[((int64_t)ai * rows_w + o) * p.d + di];
        if constexpr (!GATED && ACT == KSMM_ACT_NONE && sizeof(T) == 2)
            if (p.finite) z = mx_within_half(z);
        z = mx_act<T, GATED, ACT>(z);
        if constexpr (GATED) z *= up[i] + (bias ? (float)bias[((int64_t)ai * rows_w + p.b + o) * p.d + di] : 0.f);
        if constexpr (sizeof(T) == 2) asm("" : "+v"(z));
        const int64_t f = ((int64_t)ai * p.b + o) * p.d + di;
        ((T *)p.y)[LAST ? f * p.batch + n : n * p.a * p.b * p.d + f] = (T)z;
    }
}

// workgroups of a conversion
int64_t groups_of(const MxOperand &p)
{
    if (p.last) return (p.rows + 63) / 64 * ((p.cb + 3) / 4) * p.a * p.d;
    const int run = mx_run_of(p.d);
    return std::min<int64_t>((p.blocks / run * (p.d == run ? 4 : 1) + THREADS - 1) / THREADS, 65536);
}
template <typename T, int D, bool BACK> int convert_rows(const MxOperand &p, hipStream_t s)
{
    const unsigned groups = (unsigned)groups_of(p);
    if constexpr (D != 3)  // (never three of more)
        if (p.d != D) return launch_kernel(&ks_mx_runs_kernel<T, D, BACK>, groups, THREADS, 0, s, p);
    return launch_kernel(&ks_mx_rows_kernel<T, D, BACK>, groups, THREADS, 0, s, p);
}
template <typename T, bool BACK> int convert(const MxOperand &p, hipStream_t s)
{
    if (groups_of(p) > 0x7fffffffLL) return KSMM_ERR_TOO_LARGE;
    if (p.last)
        return in_launches(groups_of(p), THREADS, [&](uint32_t first, unsigned groups) {
            MxOperand part = p;
            part.first = first;
            return launch_kernel(&ks_mx_columns_kernel<T, BACK>, groups, THREADS, 0, s, part);
        });
    switch (mx_run_of(p.d)) {
    case 1: return convert_rows<T, 1, BACK>(p, s);
    case 2: return convert_rows<T, 2, BACK>(p, s);
    case 3: return convert_rows<T, 3, BACK>(p, s);
    default: return convert_rows<T, 4, BACK>(p, s);
    }
}

template <typename T> int values_of(const MxOperand &x, const MxOperand &w, hipStream_t s)
{
    const int64_t x_groups = groups_of(x), w_groups = groups_of(w);
    if (x_groups + w_groups > THREADS_MOST / THREADS) {
        const int rc = convert<T, true>(w, s);
        return rc == KSMM_OK ? convert<T, true>(x, s) : rc;
    }
    auto launch = [&](auto fn) { return launch_kernel(fn, (unsigned)(x_groups + w_groups), THREADS, 0, s, x, w, (uint32_t)w_groups); };
    switch (x.last ? 0 : mx_run_of(x.d)) {
    case 0: return launch(&ks_mx_values_kernel<T, 0>);
    case 1: return launch(&ks_mx_values_kernel<T, 1>);
    case 2: return launch(&ks_mx_values_kernel<T, 2>);
    case 3: return launch(&ks_mx_values_kernel<T, 3>);
    default: return launch(&ks_mx_values_kernel<T, 4>);
    }
}

template <typename T, bool LAST, bool GATED> int product(const MxProduct &p, int act, hipStream_t s)
{
    const int64_t grid = (p.tiles + 3) / 4;
    if (grid > 0x7fffffffLL) return KSMM_ERR_TOO_LARGE;
    int rc = KSMM_OK;
    with_act(act, [&](auto which) { rc = launch_kernel(&ks_mx_product_kernel<T, LAST, GATED, decltype(which)::value>, (unsigned)grid, 256, 0, s, p); });
    return rc;
}
template <typename T> int product(MxProduct p, bool last, bool gated, int act, hipStream_t s)
{
    p.b_tiles = (p.b + 31) / 32;
    p.token_tiles = (p.batch + 31) / 32;
    p.tiles = (int64_t)p.a * p.d * p.b_tiles * p.token_tiles;
    if (last) return gated ? product<T, true, true>(p, act, s) : product<T, true, false>(p, act, s);
    return gated ? product<T, false, true>(p, act, s) : product<T, false, false>(p, act, s);
}

// sizes of an operand; tensors of 2^31 elements and more are refused, and so are operands whose codes would take 2^35 bytes
int check_operand(int64_t rows, int a, int c, int d, int dtype)
{
    if (dtype != KSMM_F32 && dtype != KSMM_F16) return KSMM_ERR_BAD_DTYPE;
    return ksmm_validate(rows, a, 1, c, d, dtype, dtype, dtype, 0);
}
MxOperand operand(const void *x, void *codes, void *scales, int64_t rows, int a, int c, int d, int bs_last)
{
    const int cb = (int)mx_blocks(c);
    // (MxDiv: t d < 2^32 of the largest t)
    const int64_t tasks = (int64_t)a * rows * cb;
    return MxOperand{x,  (uint8_t *)codes, (uint8_t *)scales, rows, a, c, d, cb, bs_last != 0, 0, (int64_t)a * d * rows * cb, tasks < (1LL << 32) / std::max(a, cb) && tasks < 1LL << 31,
                     MxDiv(cb), MxDiv(a)};
}
int64_t values(int64_t rows, int a, int c, int d) { return rows * a * c * d; }
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

}  // namespace

}  // namespace ksmm

using namespace ksmm;

extern "C" {

int64_t ksmm_mx_blocks(int64_t rows, int a, int c, int d)
{
    const int rc = check_operand(rows, a, c, d, KSMM_F16);
    return rc != KSMM_OK ? rc : (int64_t)a * d * rows * mx_blocks(c);
}

static int convert_operand(const void *x, const void *codes, const void *scales, int64_t rows, int a, int c, int d, int dtype, int bs_last,
                   bool back, void *stream)
{
    const int rc = check_operand(rows, a, c, d, dtype);
    if (rc != KSMM_OK) return rc;
    if (!x || !codes || !scales) return KSMM_ERR_NULL_POINTER;
    const MxOperand p = operand(x, (void *)codes, (void *)scales, rows, a, c, d, bs_last);
    if (((uintptr_t)codes & 15) != 0) return KSMM_ERR_WORKSPACE;
    const Span t[] = {{x, values(rows, a, c, d) * (int64_t)dtype_size(dtype)}}, q[] = {{codes, p.blocks * 16}, {scales, p.blocks}};
    if (any_overlap(t, q) || overlaps(codes, p.blocks * 16, scales, p.blocks)) return KSMM_ERR_ALIAS;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == KSMM_F32) return back ? convert<float, true>(p, s) : convert<float, false>(p, s);
    return back ? convert<half_t, true>(p, s) : convert<half_t, false>(p, s);
}

int ksmm_mx_quantize(const void *x, void *codes, void *scales, int64_t rows, int a, int c, int d, int dtype, int bs_last, void *stream)
{
    return convert_operand(x, codes, scales, rows, a, c, d, dtype, bs_last, false, stream);
}

int ksmm_mx_dequantize(const void *codes, const void *scales, void *x, int64_t rows, int a, int c, int d, int dtype, int bs_last, void *stream)
{
    return convert_operand(x, codes, scales, rows, a, c, d, dtype, bs_last, true, stream);
}

int ksmm_mx_values(const void *x_codes, const void *x_scales, void *x, const void *w_codes, const void *w_scales, void *w, int64_t batch, int64_t rows,
                   int a, int c, int d, int dtype, int bs_last, void *stream)
{
    int rc = check_operand(batch, a, c, d, dtype);
    if (rc != KSMM_OK) return rc;
    if ((int64_t)a * d > 0x7fffffffLL) return KSMM_ERR_TOO_LARGE;
    rc = check_operand(rows, a * d, c, 1, dtype);
    if (rc != KSMM_OK) return rc;
    if (!x_codes || !x_scales || !x || !w_codes || !w_scales || !w) return KSMM_ERR_NULL_POINTER;
    if ((((uintptr_t)x_codes | (uintptr_t)w_codes) & 15) != 0) return KSMM_ERR_WORKSPACE;
    const MxOperand px = operand(x, (void *)x_codes, (void *)x_scales, batch, a, c, d, bs_last), pw = operand(w, (void *)w_codes, (void *)w_scales, rows, a * d, c, 1, 1);
    const int64_t size = (int64_t)dtype_size(dtype), x_bytes = values(batch, a, c, d) * size, w_bytes = values(rows, a * d, c, 1) * size;
    const Span in[] = {{x_codes, px.blocks * 16}, {x_scales, px.blocks}, {w_codes, pw.blocks * 16}, {w_scales, pw.blocks}}, out[] = {{x, x_bytes}, {w, w_bytes}};
    if (any_overlap(in, out)) return KSMM_ERR_ALIAS;
    return dtype == KSMM_F32 ? values_of<float>(px, pw, (hipStream_t)stream) : values_of<half_t>(px, pw, (hipStream_t)stream);
}

static int check_product(int64_t batch, int a, int b, int c, int d, int dtype, int act, int gated)
{
    if (dtype != KSMM_F32 && dtype != KSMM_F16) return KSMM_ERR_BAD_DTYPE;
    if (b > 0x3fffffff || batch > 0x7fffff00) return KSMM_ERR_TOO_LARGE;
    const int rc = ksmm_validate(batch, a, gated ? 2 * b : b, c, d, dtype, dtype, dtype, 0);
    if (rc != KSMM_OK) return rc;
    if (act != KSMM_ACT_NONE && act != KSMM_ACT_GELU && (act != KSMM_ACT_SILU || !gated)) return KSMM_ERR_BAD_EPILOGUE;
    return KSMM_OK;
}

int64_t ksmm_mx_forward_workspace(int64_t batch, int a, int b, int c, int d, int dtype, int bs_last, int gated)
{
    const int rc = check_product(batch, a, b, c, d, dtype, KSMM_ACT_NONE, gated);
    if (rc != KSMM_OK) return rc;
    if (mx_in_lds(c, d, (int)dtype_size(dtype), bs_last != 0)) return 0;
    const int64_t blocks = (int64_t)a * d * batch * mx_blocks(c);
    return align256(blocks * 16) + align256(blocks);
}

// the product of an operand, or of values whose codes LDS holds
static int launch_product(const MxProduct &p, int dtype, bool last, bool gated, int act, hipStream_t s)
{
    static int (*const fused[2][2][2])(const MxProduct &, int, hipStream_t) = {
        {{mx_half_first_plain, mx_half_first_gated}, {mx_half_last_plain, mx_half_last_gated}},
        {{mx_float_first_plain, mx_float_first_gated}, {mx_float_last_plain, mx_float_last_gated}}};
    if (mx_in_lds(p.c, p.d, (int)dtype_size(dtype), last)) return fused[dtype == KSMM_F32][last][gated](p, act, s);
    return dtype == KSMM_F32 ? product<float>(p, last, gated, act, s) : product<half_t>(p, last, gated, act, s);
}

int ksmm_mx_forward(const void *x, const void *x_scales, const void *w, const void *w_scales, const void *bias, void *y, void *codes_out,
                    void *scales_out, void *workspace, int64_t workspace_bytes, int64_t batch, int a, int b, int c, int d, int dtype,
                    int bs_last, int act, int gated, void *stream)
{
    int rc = check_product(batch, a, b, c, d, dtype, act, gated);
    if (rc != KSMM_OK) return rc;
    if (!x || !w || !w_scales || !y || (!codes_out != !scales_out)) return KSMM_ERR_NULL_POINTER;
    if (x_scales) codes_out = scales_out = nullptr;  // (they are there)
    const int rows_w = gated ? 2 * b : b, cb = (int)mx_blocks(c);
    const int64_t need = x_scales ? 0 : ksmm_mx_forward_workspace(batch, a, b, c, d, dtype, bs_last, gated);
    if (((uintptr_t)w & 15) != 0 || (x_scales && ((uintptr_t)x & 15) != 0) || ((uintptr_t)codes_out & 15) != 0) return KSMM_ERR_WORKSPACE;
    if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0)) return KSMM_ERR_WORKSPACE;
    const int64_t blocks = (int64_t)a * d * batch * cb, w_blocks = (int64_t)a * d * rows_w * cb, size = (int64_t)dtype_size(dtype);
    const Span in[] = {{x, x_scales ? blocks * 16 : values(batch, a, c, d) * size}, {x_scales, blocks}, {w, w_blocks * 16}, {w_scales, w_blocks},
                       {bias, (int64_t)a * rows_w * d * size}};
    const Span out[] = {{y, values(batch, a, b, d) * size}, {codes_out, blocks * 16}, {scales_out, blocks}, {need ? workspace : nullptr, need}};
    if (any_overlap(in, out)) return KSMM_ERR_ALIAS;
    MxProduct p{x, (const uint8_t *)x_scales, (uint8_t *)codes_out, (uint8_t *)scales_out, (const uint8_t *)w, (const uint8_t *)w_scales, bias, y, nullptr, false, 0, batch, a, b, c, d, cb};
    hipStream_t s = (hipStream_t)stream;
    if (need > 0) {  // (no workgroup's LDS holds the codes: x is quantised in a launch of its own)
        uint8_t *const codes = codes_out ? (uint8_t *)codes_out : (uint8_t *)workspace;
        uint8_t *const scales = codes_out ? (uint8_t *)scales_out : codes + align256(blocks * 16);
        rc = ksmm_mx_quantize(x, codes, scales, batch, a, c, d, dtype, bs_last, stream);
        if (rc != KSMM_OK) return rc;
        p.x = codes;
        p.x_scales = scales;
    }
    return launch_product(p, dtype, bs_last != 0, gated != 0, act, s);
}

int ksmm_mx_sums(const void *x, const void *x_scales, const void *w, const void *w_scales, const void *bias, void *z, int64_t batch, int a, int b, int c, int d,
                 int dtype, int bs_last, void *stream)
{
    const int rc = check_product(batch, a, b, c, d, dtype, KSMM_ACT_NONE, 0);
    if (rc != KSMM_OK) return rc;
    if (!x || !x_scales || !w || !w_scales || !z) return KSMM_ERR_NULL_POINTER;
    if (((uintptr_t)w & 15) != 0 || ((uintptr_t)x & 15) != 0) return KSMM_ERR_WORKSPACE;
    const int cb = (int)mx_blocks(c);
    const int64_t blocks = (int64_t)a * d * batch * cb, w_blocks = (int64_t)a * d * b * cb, size = (int64_t)dtype_size(dtype);
    const Span in[] = {{x, blocks * 16}, {x_scales, blocks}, {w, w_blocks * 16}, {w_scales, w_blocks}, {bias, (int64_t)a * b * d * size}};
    const Span out[] = {{z, values(batch, a, b, d) * size}};
    if (any_overlap(in, out)) return KSMM_ERR_ALIAS;
    const MxProduct p{x, (const uint8_t *)x_scales, nullptr, nullptr, (const uint8_t *)w, (const uint8_t *)w_scales, bias, z, nullptr, true, 0, batch, a, b, c, d, cb};
    return launch_product(p, dtype, bs_last != 0, false, KSMM_ACT_NONE, (hipStream_t)stream);
}

int ksmm_mx_slope(const void *x, const void *x_scales, const void *w, const void *w_scales, const void *bias, const void *dy, void *dz, int64_t batch,
                  int a, int b, int c, int d, int dtype, int bs_last, int act, int gated, void *stream)
{
    const int rc = check_product(batch, a, b, c, d, dtype, act, gated);
    if (rc != KSMM_OK) return rc;
    if (!gated && act == KSMM_ACT_NONE) return KSMM_ERR_BAD_EPILOGUE;
    const int rows_w = gated ? 2 * b : b, cb = (int)mx_blocks(c);
    MxProduct p{x, (const uint8_t *)x_scales, nullptr, nullptr, (const uint8_t *)w, (const uint8_t *)w_scales, bias, dz, dy, false, 0, batch, a, b, c, d, cb};
    if (dz) {
        if (!x || !x_scales || !w || !w_scales || !dy) return KSMM_ERR_NULL_POINTER;
        const int64_t blocks = (int64_t)a * d * batch * cb, w_blocks = (int64_t)a * d * rows_w * cb, size = (int64_t)dtype_size(dtype);
        if (((uintptr_t)w & 15) != 0 || ((uintptr_t)x & 15) != 0) return KSMM_ERR_WORKSPACE;
        const Span in[] = {{x, blocks * 16}, {x_scales, blocks}, {w, w_blocks * 16}, {w_scales, w_blocks}, {bias, (int64_t)a * rows_w * d * size},
                           {dy, values(batch, a, b, d) * size}};
        const Span out[] = {{dz, values(batch, a, rows_w, d) * size}};
        if (any_overlap(in, out)) return KSMM_ERR_ALIAS;
    }
    return (dtype == KSMM_F32 ? mx_slope_float : mx_slope_half)(p, bs_last != 0, gated != 0, act, (hipStream_t)stream);
}

}  // extern "C"
