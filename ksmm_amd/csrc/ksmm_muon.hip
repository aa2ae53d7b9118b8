// Updates of Kronecker-sparse factors made orthogonal block by block (Newton-Schulz), with momentum before and the new
// weights after.
//
//     m' = beta m + g,  u = g + beta m' (Nesterov) or m'          (without momentum u = g)
//     X0 = u / (|u|_F + eps) for each block (c x b) of each of `parts` column ranges
//     A = X X^T,  X <- p0 X + (p1 A + p2 A A) X                   `steps` times; X taken with its smaller side as rows
//     w' = (1 - lr decay) w - lr sqrt(max(1, b/c)) X              (without weights: X itself)
//
// A factor in kernel format IS its blocks one after the other, each in a row of memory: nothing is laid out again.
//
// Blocks that fit the LDS of a compute unit with their Gram matrix go through all steps in one launch, a workgroup
// each (ks_muon_block_kernel).  Larger ones go step by step through tiles in global memory (ks_muon_gemm_kernel).  The
// polynomial has slope p0 at zero: rounding errors of X grow up to p0^steps (485 for five of 3.4445) times, which is why
// every product is fp32 (32-bit matrix instructions) whatever the type of the update.
#include "ksmm_common.h"

namespace ksmm {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

struct MuonArgs {
    const void *grad;        // T
    const float *m_in;       // momentum, or null
    float *m_out;
    const void *w_in;        // T, or null: the result is X
    const float *master_in;  // fp32 weights that stand behind w, or null
    float *master_out;
    void *out;               // T: w', or X
    int c, b, parts;         // blocks of c x b, `parts` side by side
    int steps, nesterov;
    float beta, keep, rate;  // w' = keep w - rate X
    float p0, p1, p2, eps;
};

// where element (row, col) of matrix `id` lies: (blocks * c, parts * b)
__device__ __forceinline__ int64_t matrix_base(const MuonArgs &a, int64_t id)
{
    const int64_t block = id / a.parts;
    return block * a.c * a.parts * a.b + (id - block * a.parts) * a.b;
}
template <typename T> __device__ __forceinline__ float update_of(const MuonArgs &a, int64_t at)
{
    float u = (float)((const T *)a.grad)[at];
    if (a.m_in) {
        const float m = fmaf(a.beta, a.m_in[at], u);
        a.m_out[at] = m;
        u = a.nesterov ? fmaf(a.beta, m, u) : m;
    }
    return u;
}
template <typename T> __device__ __forceinline__ void finish(const MuonArgs &a, int64_t at, float x)
{
    if (a.w_in) {
        const float w = fmaf(a.keep, a.master_in ? a.master_in[at] : (float)((const T *)a.w_in)[at], -a.rate * x);
        if (a.master_in) a.master_out[at] = w;
        ((T *)a.out)[at] = (T)w;
    } else {
        ((T *)a.out)[at] = (T)x;
    }
}

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// ---- blocks that fit LDS -------------------------------------------------------------------------------
constexpr int HELD = 8;  // 16 x 16 tiles of X a wave holds between reading the old X and writing the new one
__host__ __device__ constexpr int up16(int v) { return (v + 15) / 16 * 16; }
__host__ __device__ constexpr int64_t block_lds(int m, int n)
{
    return 4 * ((int64_t)up16(m) * (up16(n) + 4) + (int64_t)up16(m) * (up16(m) + 4));
}

template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void ks_muon_block_kernel(MuonArgs a)
{
    extern __shared__ __attribute__((aligned(16))) float smem[];
    __shared__ float red[WAVES];
    const bool flip = a.c > a.b;
    const int m = flip ? a.b : a.c, n = flip ? a.c : a.b, M = up16(m), N = up16(n), ldx = N + 4, ldg = M + 4;
    float *const X = smem, *const G = smem + M * ldx;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, q = lane >> 4;
    const int64_t base = matrix_base(a, blockIdx.x), pitch = (int64_t)a.parts * a.b;
    const int count = a.c * a.b;

    for (int i = tid; i < M * ldx; i += 64 * WAVES) X[i] = 0.f;
    __syncthreads();
    float ss = 0.f;
    for (int i = tid; i < count; i += 64 * WAVES) {
        const int r = i / a.b, k = i - r * a.b;
        const float u = update_of<T>(a, base + r * pitch + k);
        X[flip ? k * ldx + r : r * ldx + k] = u;
        ss = fmaf(u, u, ss);
    }
    ss = wave_sum(ss);
    if (lane == 0) red[wave] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) ss += red[i];
    const float scale = 1.f / (sqrtf(ss) + a.eps);
    for (int i = tid; i < M * ldx; i += 64 * WAVES) X[i] *= scale;
    __syncthreads();

    const int mt = M / 16, nt = N / 16, pairs = mt * (mt + 1) / 2, tiles = mt * nt;
    // tile t of the upper triangle: (row, col >= row)
    auto upper = [&](int t, int &i, int &j) {
        i = 0;
        int left = mt;
        while (t >= left) {
            t -= left;
            --left;
            ++i;
        }
        j = i + t;
    };
    // S(16 rows from i0) times S'(16 rows from j0) transposed, K columns of both
    auto rows_product = [&](const float *s, int lds, int i0, const float *t, int ldt, int j0, int K) {
        f4 acc = {0.f, 0.f, 0.f, 0.f};
        const float *ps = s + (i0 + l16) * lds + 4 * q, *pt = t + (j0 + l16) * ldt + 4 * q;
        for (int k = 0; k < K; k += 16) {
            const f4 x = *(const f4 *)(ps + k), y = *(const f4 *)(pt + k);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], acc, 0, 0, 0);
        }
        return acc;
    };
    for (int step = 0; step < a.steps; ++step) {
        for (int t = wave; t < pairs; t += WAVES) {
            int i, j;
            upper(t, i, j);
            const f4 v = rows_product(X, ldx, 16 * i, X, ldx, 16 * j, N);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 16 * i + 4 * q + e, s = 16 * j + l16;
                G[r * ldg + s] = v[e];
                if (i != j) G[s * ldg + r] = v[e];
            }
        }
        __syncthreads();
        f4 hold[HELD];
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const int t = wave + h * WAVES;
            if (t >= pairs) break;
            int i, j;
            upper(t, i, j);
            const f4 v = rows_product(G, ldg, 16 * i, G, ldg, 16 * j, M);
#pragma unroll
            for (int e = 0; e < 4; ++e) hold[h][e] = fmaf(a.p2, v[e], a.p1 * G[(16 * i + 4 * q + e) * ldg + 16 * j + l16]);
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const int t = wave + h * WAVES;
            if (t >= pairs) break;
            int i, j;
            upper(t, i, j);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 16 * i + 4 * q + e, s = 16 * j + l16;
                G[r * ldg + s] = hold[h][e];
                if (i != j) G[s * ldg + r] = hold[h][e];
            }
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const int t = wave + h * WAVES;
            if (t >= tiles) break;
            const int i0 = t / nt * 16, j0 = t % nt * 16;
            f4 acc = {0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < M; k += 16) {
                const f4 x = *(const f4 *)(G + (i0 + l16) * ldg + 4 * q + k);
                const float *y = X + (k + 4 * q) * ldx + j0 + l16;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e * ldx], acc, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) hold[h][e] = fmaf(a.p0, X[(i0 + 4 * q + e) * ldx + j0 + l16], acc[e]);
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const int t = wave + h * WAVES;
            if (t >= tiles) break;
            const int i0 = t / nt * 16, j0 = t % nt * 16;
#pragma unroll
            for (int e = 0; e < 4; ++e) X[(i0 + 4 * q + e) * ldx + j0 + l16] = hold[h][e];
        }
        __syncthreads();
    }
    for (int i = tid; i < count; i += 64 * WAVES) {
        const int r = i / a.b, k = i - r * a.b;
        finish<T>(a, base + r * pitch + k, X[flip ? k * ldx + r : r * ldx + k]);
    }
}

// ---- larger blocks: a launch a product --------------------------------------------------------------------
// In the workspace each matrix lies as M x N, both multiples of 64 (zeros past its own sides).
constexpr int TILE = 64, CHUNKS = 16;
__host__ __device__ constexpr int up64(int v) { return (v + 63) / 64 * 64; }

// u into the workspace, and the sums of its squares, CHUNKS a matrix
template <typename T>
__global__ __launch_bounds__(256) void ks_muon_load_kernel(MuonArgs a, float *__restrict__ x, float *__restrict__ squares, int M, int N)
{
    __shared__ float red[4];
    const int64_t id = blockIdx.x / CHUNKS, chunk = blockIdx.x % CHUNKS;
    const bool flip = a.c > a.b;
    const int64_t base = matrix_base(a, id), pitch = (int64_t)a.parts * a.b;
    // in the order of memory: rows and columns as they are stored, padded alike
    const int R = flip ? N : M, K = flip ? M : N;
    const int64_t total = (int64_t)R * K, per = (total + CHUNKS - 1) / CHUNKS, end = min(total, (chunk + 1) * per);
    x += id * M * N;
    float ss = 0.f;
    for (int64_t i = chunk * per + threadIdx.x; i < end; i += 256) {
        const int r = (int)(i / K), k = (int)(i - (int64_t)r * K);
        const float u = r < a.c && k < a.b ? update_of<T>(a, base + r * pitch + k) : 0.f;
        x[flip ? (int64_t)k * N + r : (int64_t)r * N + k] = u;
        ss = fmaf(u, u, ss);
    }
    ss = wave_sum(ss);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
    __syncthreads();
    if (threadIdx.x == 0) squares[id * CHUNKS + chunk] = (red[0] + red[1]) + (red[2] + red[3]);
}

enum { GRAM, POLY, APPLY };
// C (rows x cols) of 64 x 64 tiles, K in slabs of 16.
//   GRAM   G = s^2 X X^T      POLY   Q = p1 G + p2 G G      APPLY  X' = s (p0 X + Q X), the last one: the results
// s = 1 / (|u| + eps) in the first step, whose X is u itself; later 1.  GRAM and POLY are symmetric: upper tiles only.
template <typename T, int WHAT>
__global__ __launch_bounds__(256) void ks_muon_gemm_kernel(MuonArgs a, const float *__restrict__ left, const float *__restrict__ right,
                                                           float *__restrict__ out, const float *__restrict__ squares, int M, int N, int last)
{
    constexpr int TK = 32, LDI = TK + 4, LDO = TILE + 8;
    __shared__ __attribute__((aligned(16))) float sl[2][TILE * LDI];
    __shared__ __attribute__((aligned(16))) float sr[2][WHAT == APPLY ? TK * LDO : TILE * LDI];
    const int mt = M / TILE, per = WHAT == APPLY ? mt * (N / TILE) : mt * (mt + 1) / 2;
    const int64_t id = blockIdx.x / per;
    int t = (int)(blockIdx.x - id * per), ti, tj;
    if (WHAT == APPLY) {
        ti = t % mt;
        tj = t / mt;
    } else {
        ti = 0;
        for (int rest = mt; t >= rest; --rest, ++ti) t -= rest;
        tj = ti + t;
    }
    const int K = WHAT == GRAM ? N : M, ldl = WHAT == GRAM ? N : M, ldr = WHAT == POLY ? M : N, i0 = ti * TILE, j0 = tj * TILE;
    const float *const L = left + id * M * ldl, *const R = right + id * M * ldr;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, q = lane >> 4;
    const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;

    f4 lr[2], rr[2];
    auto gload = [&](int k0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int v = tid + i * 256, row = v / (TK / 4), k = v % (TK / 4) * 4;
            lr[i] = *(const f4 *)(L + (int64_t)(i0 + row) * ldl + k0 + k);
            if (WHAT == APPLY) {
                const int kk = v / (TILE / 4), col = v % (TILE / 4) * 4;
                rr[i] = *(const f4 *)(R + (int64_t)(k0 + kk) * ldr + j0 + col);
            } else {
                rr[i] = *(const f4 *)(R + (int64_t)(j0 + row) * ldr + k0 + k);
            }
        }
    };
    auto lstore = [&](int buf) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int v = tid + i * 256, row = v / (TK / 4), k = v % (TK / 4) * 4;
            *(f4 *)(sl[buf] + row * LDI + k) = lr[i];
            if (WHAT == APPLY)
                *(f4 *)(sr[buf] + v / (TILE / 4) * LDO + v % (TILE / 4) * 4) = rr[i];
            else
                *(f4 *)(sr[buf] + row * LDI + k) = rr[i];
        }
    };
    f4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
    gload(0);
    lstore(0);
    __syncthreads();
    for (int k0 = 0, buf = 0; k0 < K; k0 += TK, buf ^= 1) {
        if (k0 + TK < K) gload(k0 + TK);
#pragma unroll
        for (int k = 0; k < TK; k += 16) {
            f4 x[2], y[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                x[i] = *(const f4 *)(sl[buf] + (wi + 16 * i + l16) * LDI + k + 4 * q);
                if (WHAT == APPLY) {
                    const float *p = sr[buf] + (k + 4 * q) * LDO + wj + 16 * i + l16;
                    y[i] = f4{p[0], p[LDO], p[2 * LDO], p[3 * LDO]};
                } else {
                    y[i] = *(const f4 *)(sr[buf] + (wj + 16 * i + l16) * LDI + k + 4 * q);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i][e], y[j][e], acc[i][j], 0, 0, 0);
        }
        if (k0 + TK < K) lstore(buf ^ 1);
        __syncthreads();
    }
    float s = 1.f;
    if (WHAT != POLY && squares) {
        float ss = 0.f;
        for (int i = 0; i < CHUNKS; ++i) ss += squares[id * CHUNKS + i];
        s = 1.f / (sqrtf(ss) + a.eps);
    }
    const int64_t base = matrix_base(a, id), pitch = (int64_t)a.parts * a.b;
    const bool flip = a.c > a.b;
    const int m = flip ? a.b : a.c, n = flip ? a.c : a.b;
    out += id * M * (WHAT == APPLY ? N : M);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = i0 + wi + 16 * i + 4 * q + e, c = j0 + wj + 16 * j + l16;
                if (WHAT == GRAM) {
                    const float v = acc[i][j][e] * s * s;
                    out[(int64_t)r * M + c] = v;
                    if (ti != tj) out[(int64_t)c * M + r] = v;
                } else if (WHAT == POLY) {
                    const float v = fmaf(a.p2, acc[i][j][e], a.p1 * L[(int64_t)r * M + c]);
                    out[(int64_t)r * M + c] = v;
                    if (ti != tj) out[(int64_t)c * M + r] = v;
                } else {
                    const float v = fmaf(a.p0, R[(int64_t)r * N + c], acc[i][j][e]) * s;
                    if (!last)
                        out[(int64_t)r * N + c] = v;
                    else if (r < m && c < n)
                        finish<T>(a, base + (flip ? (int64_t)c * pitch + r : (int64_t)r * pitch + c), v);
                }
            }
}

// ---- choices ----------------------------------------------------------------------------------------------
int launched() { return hipGetLastError() == hipSuccess ? KSMM_OK : KSMM_ERR_LAUNCH; }
constexpr int64_t LDS_MOST = 160 * 1024 - 256;

bool fits_lds(int m, int n)
{
    const int64_t mt = up16(m) / 16, nt = up16(n) / 16;
    return block_lds(m, n) <= LDS_MOST && mt * nt <= 16 * HELD && mt * (mt + 1) / 2 <= 16 * HELD;
}

template <typename T, int WAVES> int run_block(const MuonArgs &a, int64_t matrices, int lds, hipStream_t s)
{
    const auto fn = &ks_muon_block_kernel<T, WAVES>;
    if (lds > 64 * 1024) {
        const int rc = ensure_dynamic_lds((const void *)fn, (int)LDS_MOST);
        if (rc != KSMM_OK) return rc;
    }
    hipLaunchKernelGGL(fn, dim3((unsigned)matrices), dim3(64 * WAVES), lds, s, a);
    return launched();
}

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
struct Space {
    int M, N;
    int64_t x[2], gram, poly, squares, total;
};
Space space(int64_t matrices, int c, int b)
{
    Space w;
    const int m = std::min(c, b), n = std::max(c, b);
    w.M = up64(m);
    w.N = up64(n);
    int64_t at = 0;
    auto take = [&](int64_t floats) {
        const int64_t was = at;
        at += align256(4 * floats);
        return was;
    };
    w.x[0] = take(matrices * w.M * w.N);
    w.x[1] = take(matrices * w.M * w.N);
    w.gram = take(matrices * w.M * w.M);
    w.poly = take(matrices * w.M * w.M);
    w.squares = take(matrices * CHUNKS);
    w.total = at;
    return w;
}

template <typename T> int run(const MuonArgs &a, int64_t matrices, char *ws, hipStream_t s)
{
    const int m = std::min(a.c, a.b), n = std::max(a.c, a.b);
    if (fits_lds(m, n)) {
        const int lds = (int)block_lds(m, n), tiles = up16(m) / 16 * (up16(n) / 16);
        return tiles <= 1 ? run_block<T, 1>(a, matrices, lds, s) : tiles <= 4 ? run_block<T, 4>(a, matrices, lds, s) : run_block<T, 16>(a, matrices, lds, s);
    }
    const Space w = space(matrices, a.c, a.b);
    const int64_t mt = w.M / TILE, half = matrices * mt * (mt + 1) / 2, full = matrices * mt * (w.N / TILE);
    if (full > 0x7fffffffLL || matrices * CHUNKS > 0x7fffffffLL) return KSMM_ERR_TOO_LARGE;
    float *x = (float *)(ws + w.x[0]), *y = (float *)(ws + w.x[1]), *gram = (float *)(ws + w.gram), *poly = (float *)(ws + w.poly);
    float *const squares = (float *)(ws + w.squares);
    hipLaunchKernelGGL((ks_muon_load_kernel<T>), dim3((unsigned)(matrices * CHUNKS)), dim3(256), 0, s, a, x, squares, w.M, w.N);
    for (int i = 0; i < a.steps; ++i) {
        const float *const sq = i == 0 ? squares : nullptr;
        hipLaunchKernelGGL((ks_muon_gemm_kernel<T, GRAM>), dim3((unsigned)half), dim3(256), 0, s, a, x, x, gram, sq, w.M, w.N, 0);
        hipLaunchKernelGGL((ks_muon_gemm_kernel<T, POLY>), dim3((unsigned)half), dim3(256), 0, s, a, gram, gram, poly, sq, w.M, w.N, 0);
        hipLaunchKernelGGL((ks_muon_gemm_kernel<T, APPLY>), dim3((unsigned)full), dim3(256), 0, s, a, poly, x, y, sq, w.M, w.N, i + 1 == a.steps);
        std::swap(x, y);
    }
    return launched();
}

int check(const ksmm_muon_desc *d, int64_t blocks, int c, int b, int parts, int dtype)
{
    if (!d) return KSMM_ERR_NULL_POINTER;
    if (blocks < 1 || c < 1 || b < 1 || parts < 1) return KSMM_ERR_BAD_PATTERN;
    if (dtype != KSMM_F32 && dtype != KSMM_F16) return KSMM_ERR_BAD_DTYPE;
    if (d->steps < 1) return KSMM_ERR_BAD_ALGO;
    if ((double)blocks * c * b * parts > 2147483647.0 || blocks * parts > 0x7fffffffLL) return KSMM_ERR_TOO_LARGE;
    return KSMM_OK;
}

}  // namespace

}  // namespace ksmm

using namespace ksmm;

extern "C" {

int64_t ksmm_muon_workspace(int64_t blocks, int c, int b, int parts)
{
    if (blocks < 1 || c < 1 || b < 1 || parts < 1) return KSMM_ERR_BAD_PATTERN;
    if ((double)blocks * c * b * parts > 2147483647.0) return KSMM_ERR_TOO_LARGE;
    return fits_lds(std::min(c, b), std::max(c, b)) ? 0 : space(blocks * parts, c, b).total;
}

int ksmm_muon_update(const ksmm_muon_desc *desc, const void *grad, const float *momentum, float *momentum_out, const void *weight,
                     const float *master, float *master_out, void *out, void *workspace, int64_t workspace_bytes, int64_t blocks, int c,
                     int b, int parts, int dtype, void *stream)
{
    const int rc = check(desc, blocks, c, b, parts, dtype);
    if (rc != KSMM_OK) return rc;
    if (!grad || !out || (momentum && !momentum_out) || (master && (!master_out || !weight))) return KSMM_ERR_NULL_POINTER;
    const int64_t need = ksmm_muon_workspace(blocks, c, b, parts);
    if (need < 0) return (int)need;
    if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0)) return KSMM_ERR_WORKSPACE;
    MuonArgs a;
    a.grad = grad;
    a.m_in = momentum;
    a.m_out = momentum_out;
    a.w_in = weight;
    a.master_in = master;
    a.master_out = master_out;
    a.out = out;
    a.c = c;
    a.b = b;
    a.parts = parts;
    a.steps = desc->steps;
    a.nesterov = desc->nesterov;
    a.beta = desc->beta;
    a.keep = desc->keep;
    a.rate = desc->rate;
    a.p0 = desc->coefficients[0];
    a.p1 = desc->coefficients[1];
    a.p2 = desc->coefficients[2];
    a.eps = desc->eps;
    return dtype == KSMM_F32 ? run<float>(a, blocks * parts, (char *)workspace, (hipStream_t)stream)
                             : run<half_t>(a, blocks * parts, (char *)workspace, (hipStream_t)stream);
}

}  // extern "C"
