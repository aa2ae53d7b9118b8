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
// X, its Gram matrix and the polynomial of that are held in 22 bits, whatever the type of the update, and multiplied with fp32 sums.
#include "ksmm_mfma.h"
#include <algorithm>
#include <cmath>
#include <initializer_list>

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
    int steps, nesterov, follow;
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
// the weight that is updated: the master, or what lies in its place if that is not its rounding any more (`follow`)
template <typename T> __device__ __forceinline__ float weight_of(const MuonArgs &a, int64_t at)
{
    if (!a.master_in) return (float)((const T *)a.w_in)[at];
    const float m = a.master_in[at];
    if (!a.follow) return m;
    const T w = ((const T *)a.w_in)[at];
    return (T)m == w ? m : (float)w;
}
template <typename T> __device__ __forceinline__ void finish(const MuonArgs &a, int64_t at, float x)
{
    if (a.w_in) {
        const float w = fmaf(a.keep, weight_of<T>(a, at), -a.rate * x);
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

// fp32 values as two fp16 ones, x = hi + lo / 2048: 22 bits.  A product of two such is three matrix instructions
// (hi hi, and hi lo + lo hi in sums of their own; what lo lo would add is below the last bit), 96 clocks for 32 x 32 x 16
// where the 32-bit instructions take 512.  The 22 bits are those of values from 6e-5 on; below, where hi is subnormal, they end at
// 1.5e-11 (an entry of an orthogonal 1536 x 384 is 1e-3).  Coefficients with which a value could pass 60000 are refused (in_range).
// (1,1536,384,2) of two parts is 5.6e-8 off in the 2-norm; the same steps in plain fp32 are 1.1e-7.
constexpr float SPLIT = 2048.f;
__device__ __forceinline__ void split(float v, half_t &hi, half_t &lo)
{
    hi = (half_t)v;
    lo = (half_t)((v - (float)hi) * SPLIT);
}

// ---- blocks that fit LDS -------------------------------------------------------------------------------
// X and its Gram matrix (which the polynomial replaces) in LDS, hi and lo apart, sides padded to 32 with zeros; tiles of
// 16 x 16 are dealt to the waves.  G and Q are symmetric: upper tiles only, and both operands of G G are rows.  Few of these
// matrices fill no chip: what counts is the latency of fifteen products in a row, and for blocks that fill LDS its reads, 4 KB for
// three instructions (128 x 128: 11 MB in five steps, 36 us at 128 bytes a clock).
// (6,64,64,1) 17.7 us, (1,128,128,3) 70, with momentum and weights 74 (on 32-bit instructions 28 and 133).  Blocks of more than 64
// tiles (8 a wave) spill 90 registers a thread.
__host__ __device__ constexpr int up16(int v) { return (v + 15) / 16 * 16; }
__host__ __device__ constexpr int up32(int v) { return (v + 31) / 32 * 32; }
__host__ __device__ constexpr int64_t block_lds(int m, int n)
{
    return 4 * ((int64_t)up32(m) * (up32(n) + 8) + (int64_t)up32(m) * (up32(m) + 8));
}

// HELD: tiles of X a wave holds between reading the old X and writing the new one
template <typename T, int WAVES, int HELD>
__global__ __launch_bounds__(64 * WAVES) void ks_muon_block_kernel(MuonArgs a)
{
    constexpr int THREADS = 64 * WAVES, PER = HELD * 4, ONCE = PER < 16 ? PER : 16;  // elements a thread, and loaded at a time
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    __shared__ float red[WAVES];
    const bool flip = a.c > a.b;
    const int m = flip ? a.b : a.c, n = flip ? a.c : a.b, M = up32(m), N = up32(n), ldx = N + 8, ldg = M + 8;
    half_t *const XH = (half_t *)smem, *const XL = XH + M * ldx, *const GH = XL + M * ldx, *const GL = GH + M * ldg;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, q = lane >> 4;
    const int64_t base = matrix_base(a, blockIdx.x);

    // the thread's elements tid, tid + THREADS, ..: row and column as stored, without a division each
    struct Walk {
        int r, k, dr, dk, c, b, pitch, ld;
        bool flip;
        __device__ __forceinline__ void next()
        {
            r += dr;
            k += dk;
            if (k >= b) {
                k -= b;
                ++r;
            }
        }
        __device__ __forceinline__ bool in() const { return r < c; }
        __device__ __forceinline__ int place() const { return in() ? r * pitch + k : 0; }  // in the tensors
        __device__ __forceinline__ int inside() const { return flip ? k * ld + r : r * ld + k; }  // in X
    };
    const Walk start{tid / a.b, tid % a.b, THREADS / a.b, THREADS % a.b, a.c, a.b, a.parts * a.b, ldx, flip};
    auto walk = [&]() {
        Walk w = start;
        asm volatile("" : "+v"(w.r), "+v"(w.k));  // (each walk is made anew: the places of one are not held for the next)
        return w;
    };
    for (int i = tid; i < 2 * M * (ldx + ldg) / 8; i += THREADS) ((uint4_t *)smem)[i] = uint4_t{0u, 0u, 0u, 0u};
    float u[PER], ss = 0.f;
    {
        Walk at = walk(), to = walk();
        const T *const grad = (const T *)a.grad + base;
#pragma unroll
        for (int first = 0; first < PER; first += ONCE) {
            float mom[ONCE];
#pragma unroll
            for (int e = 0; e < ONCE; ++e, at.next()) {
                const float g = (float)grad[at.place()];
                u[first + e] = at.in() ? g : 0.f;
                if (a.m_in) mom[e] = a.m_in[base + at.place()];
            }
            if (a.m_in) {
#pragma unroll
                for (int e = 0; e < ONCE; ++e, to.next()) {
                    const float v = fmaf(a.beta, mom[e], u[first + e]);
                    if (to.in()) {
                        a.m_out[base + to.place()] = v;
                        u[first + e] = a.nesterov ? fmaf(a.beta, v, u[first + e]) : v;
                    }
                }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) ss = fmaf(u[e], u[e], ss);
    ss = wave_sum(ss);
    if (lane == 0) red[wave] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) ss += red[i];
    const float scale = 1.f / (sqrtf(ss) + a.eps);
    {
        Walk at = walk();
#pragma unroll
        for (int e = 0; e < PER; ++e, at.next())
            if (at.in()) split(u[e] * scale, XH[at.inside()], XL[at.inside()]);
    }
    __syncthreads();

    const int mt = up16(m) / 16, nt = up16(n) / 16, pairs = mt * (mt + 1) / 2, tiles = mt * nt;
    // the wave's tiles: of the upper triangle (row, col >= row), and of X
    int pi[HELD], pj[HELD], xi[HELD], xj[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        int t = wave + h * WAVES, left = mt;
        xi[h] = t / nt * 16;
        xj[h] = t % nt * 16;
        pi[h] = 0;
        while (left > 0 && t >= left) {
            t -= left;
            --left;
            ++pi[h];
        }
        pj[h] = pi[h] + t;
    }
    // where the lane's part of a tile at (0, 0) lies: operand rows of X and G; columns of X; four of a row of G, rows of G and X
    int at_x = l16 * ldx + 8 * q, at_g = l16 * ldg + 8 * q, at_c = (8 * q + (l16 >> 2)) * ldx + 4 * (l16 & 3);
    int at_p = l16 * ldg + 4 * q, at_r = 4 * q * ldg + l16, at_o = 4 * q * ldx + l16;
    // (the addresses of all tiles would be held through the steps, and spilled: each product makes its own)
    auto fresh = [&]() { asm volatile("" : "+v"(at_x), "+v"(at_g), "+v"(at_c), "+v"(at_p), "+v"(at_r), "+v"(at_o)); };
    // rows i0.. of (sh, sl) times rows j0.. of it, transposed, over K columns
    auto rows_product = [&](const half_t *sh, const half_t *sl, int ld, int at, int i0, int j0, int K) {
        const int x = at + i0 * ld, y = at + j0 * ld;
        f4 main = {0.f, 0.f, 0.f, 0.f}, cross = {0.f, 0.f, 0.f, 0.f};
        half8_t xh = *(const half8_t *)(sh + x), xl = *(const half8_t *)(sl + x), yh = *(const half8_t *)(sh + y), yl = *(const half8_t *)(sl + y);
        for (int k = 32; k <= K; k += 32) {  // the next operands are read while these multiply
            const int to = min(k, K - 32);
            const half8_t ph = *(const half8_t *)(sh + x + to), pl = *(const half8_t *)(sl + x + to);
            const half8_t rh = *(const half8_t *)(sh + y + to), rl = *(const half8_t *)(sl + y + to);
            main = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, yh, main, 0, 0, 0);
            cross = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, yl, cross, 0, 0, 0);
            cross = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl, yh, cross, 0, 0, 0);
            xh = ph;
            xl = pl;
            yh = rh;
            yl = rl;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) main[e] = fmaf(cross[e], 1.f / SPLIT, main[e]);
        return main;
    };
    // element e of a lane's tile: row 4 q + e, column l16
    auto store_pair = [&](const f4 &v, int i, int j) {
        half4_t h, l;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            half_t vh, vl;
            split(v[e], vh, vl);
            h[e] = vh;
            l[e] = vl;
            if (i != j) {
                GH[at_r + (16 * i + e) * ldg + 16 * j] = vh;
                GL[at_r + (16 * i + e) * ldg + 16 * j] = vl;
            }
        }
        *(half4_t *)(GH + at_p + 16 * j * ldg + 16 * i) = h;
        *(half4_t *)(GL + at_p + 16 * j * ldg + 16 * i) = l;
    };
    auto wide = [&](const half_t *h, const half_t *l, int at) { return fmaf((float)l[at], 1.f / SPLIT, (float)h[at]); };
    // 8 k of column l16: X[k0 + 8 q ..][j0 + l16]
    auto columns = [&](const half_t *s, int k0, int j0) {
        typedef short4_t __attribute__((address_space(3))) * lds_ptr;
        typedef short short8_t __attribute__((ext_vector_type(8)));
        const half_t *p = s + at_c + k0 * ldx + j0;
        const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 4 * ldx));
        return __builtin_bit_cast(half8_t, short8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
    };
    // the wave's tiles of X stay in registers too, unrounded
    f4 mine[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h)
        if (wave + h * WAVES < tiles)
#pragma unroll
            for (int e = 0; e < 4; ++e) mine[h][e] = wide(XH, XL, at_o + (xi[h] + e) * ldx + xj[h]);
    for (int step = 0; step < a.steps; ++step) {
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            if (wave + h * WAVES >= pairs) break;
            fresh();
            store_pair(rows_product(XH, XL, ldx, at_x, 16 * pi[h], 16 * pj[h], N), pi[h], pj[h]);
        }
        __syncthreads();
        f4 hold[HELD];
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            if (wave + h * WAVES >= pairs) break;
            fresh();
            const int i = pi[h], j = pj[h];
            const f4 v = rows_product(GH, GL, ldg, at_g, 16 * i, 16 * j, M);
            const half4_t gh = *(const half4_t *)(GH + at_p + 16 * j * ldg + 16 * i), gl = *(const half4_t *)(GL + at_p + 16 * j * ldg + 16 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) hold[h][e] = fmaf(a.p2, v[e], a.p1 * fmaf((float)gl[e], 1.f / SPLIT, (float)gh[e]));
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            if (wave + h * WAVES >= pairs) break;
            fresh();
            store_pair(hold[h], pi[h], pj[h]);
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            if (wave + h * WAVES >= tiles) break;
            fresh();
            const int j0 = xj[h], x = at_g + xi[h] * ldg;
            f4 main = {0.f, 0.f, 0.f, 0.f}, cross = {0.f, 0.f, 0.f, 0.f};
            half8_t xh = *(const half8_t *)(GH + x), xl = *(const half8_t *)(GL + x), yh = columns(XH, 0, j0), yl = columns(XL, 0, j0);
            for (int k = 32; k <= M; k += 32) {
                const int to = min(k, M - 32);
                const half8_t ph = *(const half8_t *)(GH + x + to), pl = *(const half8_t *)(GL + x + to);
                const half8_t rh = columns(XH, to, j0), rl = columns(XL, to, j0);
                main = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, yh, main, 0, 0, 0);
                cross = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, yl, cross, 0, 0, 0);
                cross = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl, yh, cross, 0, 0, 0);
                xh = ph;
                xl = pl;
                yh = rh;
                yl = rl;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) mine[h][e] = fmaf(a.p0, mine[h][e], fmaf(cross[e], 1.f / SPLIT, main[e]));
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            if (wave + h * WAVES >= tiles) break;
            fresh();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int to = at_o + (xi[h] + e) * ldx + xj[h];
                split(mine[h][e], XH[to], XL[to]);
            }
        }
        __syncthreads();
    }
    Walk at = walk(), to = walk();
#pragma unroll
    for (int first = 0; first < PER; first += ONCE) {
        float w[ONCE];
        if (a.w_in) {
#pragma unroll
            for (int e = 0; e < ONCE; ++e, at.next()) w[e] = weight_of<T>(a, base + at.place());
        }
#pragma unroll
        for (int e = 0; e < ONCE; ++e, to.next()) {
            if (!to.in()) continue;
            float v = wide(XH, XL, to.inside());
            if (a.w_in) {
                v = fmaf(a.keep, w[e], -a.rate * v);
                if (a.master_in) a.master_out[base + to.place()] = v;
            }
            ((T *)a.out)[base + to.place()] = (T)v;
        }
    }
}

// ---- larger blocks: a launch a product --------------------------------------------------------------------
// In the workspace each matrix lies as X (M x N) and as its transpose, M and N multiples of 64 (zeros past its own
// sides): with G and Q symmetric, every product is one of rows with rows, and its operands come straight from memory.  They
// lie there as the instructions take them: 32 rows x 16 k are 1 KB in a row, 16 bytes a lane (operands gathered from plain
// rows took 58 us a product of (1,1536,384,2) pairs, bound by addresses).
constexpr int TILE = 64, STEP = 16;
__host__ __device__ constexpr int up64(int v) { return (v + 63) / 64 * 64; }

// where element (r, k) of a matrix of K columns lies: lane r % 32 + 32 * (k % 16 / 8) of piece (r / 32, k / 16)
__device__ __forceinline__ int64_t operand_at(int r, int k, int K)
{
    return ((int64_t)(r >> 5) * (K >> 4) + (k >> 4)) * 512 + (((k >> 3) & 1) * 32 + (r & 31)) * 8 + (k & 7);
}
struct Split {
    half_t *hi, *lo;
    // four values, k to k + 3 (4 divides k)
    __device__ __forceinline__ void put(int64_t at, const f4 &v) const
    {
        half4_t h, l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h[i] = (half_t)v[i];
            l[i] = (half_t)((v[i] - (float)h[i]) * SPLIT);
        }
        *(half4_t *)(hi + at) = h;
        *(half4_t *)(lo + at) = l;
    }
    __device__ __forceinline__ f4 get(int64_t at) const
    {
        const half4_t h = *(const half4_t *)(hi + at), l = *(const half4_t *)(lo + at);
        f4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = fmaf((float)l[i], 1.f / SPLIT, (float)h[i]);
        return v;
    }
};

// u (fp32, as it is stored in memory, blocks next to each other) and the sums of its squares, `chunks` a matrix
template <typename T>
__global__ __launch_bounds__(256) void ks_muon_load_kernel(MuonArgs a, float *__restrict__ u, float *__restrict__ squares, int chunks)
{
    __shared__ float red[4];
    const int64_t id = blockIdx.x / chunks, chunk = blockIdx.x - id * chunks;
    const int64_t base = matrix_base(a, id), pitch = (int64_t)a.parts * a.b;
    const int total = a.c * a.b, per = (total + chunks - 1) / chunks, end = min((int64_t)total, (chunk + 1) * per);
    u += id * total;
    float ss = 0.f;
    for (int i = chunk * per + threadIdx.x; i < end; i += 256) {
        const int r = i / a.b, k = i - r * a.b;
        const float v = update_of<T>(a, base + r * pitch + k);
        u[i] = v;
        ss = fmaf(v, v, ss);
    }
    ss = wave_sum(ss);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
    __syncthreads();
    if (threadIdx.x == 0) squares[id * chunks + chunk] = (red[0] + red[1]) + (red[2] + red[3]);
}

// X0 and its transpose from u, 64 x 64 at a time (as they lie in memory: c x b)
__global__ __launch_bounds__(256) void ks_muon_split_kernel(MuonArgs a, const float *__restrict__ u, const float *__restrict__ squares, int chunks,
                                                            Split straight, Split turned, int R, int K)
{
    __shared__ float tile[64][65];
    __shared__ float norm;
    const int tk = K / 64, per = R / 64 * tk;
    const int64_t id = blockIdx.x / per;
    const int t = (int)(blockIdx.x - id * per), r0 = t / tk * 64, k0 = t % tk * 64;
    if (threadIdx.x < 64) {
        float ss = 0.f;
        for (int i = threadIdx.x; i < chunks; i += 64) ss += squares[id * chunks + i];
        ss = wave_sum(ss);
        if (threadIdx.x == 0) norm = 1.f / (sqrtf(ss) + a.eps);
    }
    __syncthreads();
    const float scale = norm;
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    u += id * a.c * a.b;
    const int64_t base = id * R * K;
#pragma unroll 4
    for (int i = w; i < 64; i += 4) {
        const int r = r0 + i, k = k0 + l;
        tile[i][l] = r < a.c && k < a.b ? u[(int64_t)r * a.b + k] * scale : 0.f;
    }
    __syncthreads();
    // lane: a row, four k at a time
#pragma unroll
    for (int k = 4 * w; k < 64; k += 16) {
        straight.put(base + operand_at(r0 + l, k0 + k, K), f4{tile[l][k], tile[l][k + 1], tile[l][k + 2], tile[l][k + 3]});
        turned.put(base + operand_at(k0 + l, r0 + k, R), f4{tile[k][l], tile[k + 1][l], tile[k + 2][l], tile[k + 3][l]});
    }
}

enum { GRAM, POLY, APPLY };
// C = L R^T (rows of L, rows of R), a 64 x 64 tile a workgroup; four groups of four waves share K and add up in LDS.
//   GRAM   G = X X^T      POLY   Q = p1 G + p2 G G      APPLY  X'^T = p0 X^T + X^T Q, or the results
// Stored are the transposes of the tiles (what a lane holds lies in a row there; G and Q are symmetric), by APPLY both.
// (GRAM and POLY compute both triangles: with few matrices there are more CUs than tiles.)
// A wave multiplies whole tiles of 64 x 64 (four of 32 x 32: an operand from the L1, whose 64 bytes a clock are what bounds
// this, serves two of them); the GROUPS waves of a workgroup share K and add up in LDS.
template <typename T, int WHAT, int GROUPS>
__global__ __launch_bounds__(64 * GROUPS, 2) void ks_muon_gemm_kernel(MuonArgs a, Split left, Split right, Split x, Split out, Split turned, int M, int N,
                                                                   int last, int tiles)
{
    extern __shared__ __attribute__((aligned(16))) float sums[];  // GROUPS x 64 x 64, then 4 x 32 x 33
    // a range of tiles an XCD: a matrix's operands are read through few of the L2s
    const int per_xcd = (tiles + 7) / 8, lid = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per_xcd || lid >= tiles) return;
    const int mt = M / TILE, per = WHAT == APPLY ? mt * (N / TILE) : mt * mt;
    const int64_t id = lid / per;
    const int t = (int)(lid - id * per), tj = t % mt, ti = t / mt;  // (tiles that share rows of L are neighbours)
    const int K = WHAT == GRAM ? N : M, rows_l = WHAT == APPLY ? N : M;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, lq = lane >> 5;
    const int64_t at_l = id * rows_l * K + operand_at(ti * TILE, 0, K) + lane * 8, at_r = id * M * K + operand_at(tj * TILE, 0, K) + lane * 8;
    const int64_t half = (int64_t)(K >> 4) * 512;  // to the other 32 rows
    const half_t *const lh = left.hi + at_l, *const ll = left.lo + at_l, *const rh = right.hi + at_r, *const rl = right.lo + at_r;
    // element e of a lane's 32 x 32: row 8 * (e / 4) + 4 * lq + e % 4, column l32.  A wave finishes MINE fours of rows of one
    constexpr int MINE = 16 / GROUPS;
    static_assert(MINE * GROUPS == 16 && MINE <= 4, "waves");
    const int quarter = wave * MINE / 4, group = wave % (4 / MINE);
    const int i0 = ti * TILE + (quarter >> 1) * 32, j0 = tj * TILE + (quarter & 1) * 32;
    f4 old[MINE];
    float16_t main[2][2], cross[2][2];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 16; ++e) main[q >> 1][q & 1][e] = cross[q >> 1][q & 1][e] = 0.f;
    struct Operands {
        half8_t xh[2], xl[2], yh[2], yl[2];
    };
    const int steps = K / STEP;
    auto load = [&](Operands &o, int s) {
        const int64_t at = (int64_t)min(s, steps - 1) * 512;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            o.xh[q] = *(const half8_t *)(lh + at + q * half);
            o.xl[q] = *(const half8_t *)(ll + at + q * half);
            o.yh[q] = *(const half8_t *)(rh + at + q * half);
            o.yl[q] = *(const half8_t *)(rl + at + q * half);
        }
    };
    auto multiply = [&](const Operands &o) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            main[p >> 1][p & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(o.xh[p >> 1], o.yh[p & 1], main[p >> 1][p & 1], 0, 0, 0);
            cross[p >> 1][p & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(o.xh[p >> 1], o.yl[p & 1], cross[p >> 1][p & 1], 0, 0, 0);
            cross[p >> 1][p & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(o.xl[p >> 1], o.yh[p & 1], cross[p >> 1][p & 1], 0, 0, 0);
        }
    };
    // loads run two steps ahead: the compiler must neither move them behind the products nor sink them to their use
    Operands ring[3];
    load(ring[0], wave);
    load(ring[1], wave + GROUPS);
    int s = wave;
    for (; s + 2 * GROUPS < steps; s += 3 * GROUPS) {
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            load(ring[(q + 2) % 3], s + (q + 2) * GROUPS);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            multiply(ring[q]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (WHAT != GRAM) {
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int r = 8 * (group * MINE + k) + 4 * lq;
            old[k] = x.get(WHAT == POLY ? id * M * M + operand_at(j0 + l32, i0 + r, M) : id * M * N + operand_at(j0 + l32, i0 + r, N));
        }
    }
    if (s < steps) multiply(ring[0]);
    if (s + GROUPS < steps) multiply(ring[1]);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 16; ++e) sums[((wave * 4 + q) * 16 + e) * 64 + lane] = fmaf(cross[q >> 1][q & 1][e], 1.f / SPLIT, main[q >> 1][q & 1][e]);
    __syncthreads();
    f4 v[MINE];
#pragma unroll
    for (int k = 0; k < MINE; ++k) {
        v[k] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < GROUPS; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[k][e] += sums[((q * 4 + quarter) * 16 + 4 * (group * MINE + k) + e) * 64 + lane];
    }
    if (WHAT == APPLY) __syncthreads();
    float *const turn = sums + quarter * 32 * 33;  // [j][i]
#pragma unroll
    for (int k = 0; k < MINE; ++k) {
        const int r = 8 * (group * MINE + k) + 4 * lq;
        if (WHAT == GRAM) {
            out.put(id * M * M + operand_at(j0 + l32, i0 + r, M), v[k]);
        } else if (WHAT == POLY) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[k][e] = fmaf(a.p2, v[k][e], a.p1 * old[k][e]);
            out.put(id * M * M + operand_at(j0 + l32, i0 + r, M), v[k]);
        } else {
            // rows of X^T are i, of X are j: X[j0 + l32][i0 + r ..]
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[k][e] = fmaf(a.p0, old[k][e], v[k][e]);
                turn[l32 * 33 + r + e] = v[k][e];
            }
            if (!last) out.put(id * M * N + operand_at(j0 + l32, i0 + r, N), v[k]);
        }
    }
    if (WHAT != APPLY) return;
    __syncthreads();
    const int64_t base = matrix_base(a, id), pitch = (int64_t)a.parts * a.b;
    const bool flip = a.c > a.b;
    const int m = flip ? a.b : a.c, n = flip ? a.c : a.b;
#pragma unroll
    for (int k = 0; k < MINE; ++k) {
        const int r = 8 * (group * MINE + k) + 4 * lq;
        if (!last) {
            turned.put(id * M * N + operand_at(i0 + l32, j0 + r, M), f4{turn[r * 33 + l32], turn[(r + 1) * 33 + l32], turn[(r + 2) * 33 + l32], turn[(r + 3) * 33 + l32]});
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // along the rows of memory
                const int i = i0 + (flip ? r + e : l32), j = j0 + (flip ? l32 : r + e);
                if (j < m && i < n) finish<T>(a, base + (flip ? (int64_t)i * pitch + j : (int64_t)j * pitch + i), turn[(j - j0) * 33 + i - i0]);
            }
        }
    }
}

// ---- choices ----------------------------------------------------------------------------------------------
int launched() { return hipGetLastError() == hipSuccess ? KSMM_OK : KSMM_ERR_LAUNCH; }
constexpr int64_t LDS_MOST = 160 * 1024 - 256;

// In one launch where X fits LDS and the waves' registers: (6,64,64,1) 17.7 us, by launches of products 73;
// (1,192,48,2) of two parts 29 for 80; (1,128,128,3) 70 for 84, 64 such matrices 70 for 104.
bool fits_lds(int m, int n)
{
    const int64_t mt = up16(m) / 16, nt = up16(n) / 16;
    return block_lds(m, n) <= LDS_MOST && mt * nt <= 16 * 8;
}

template <typename T, int WAVES, int HELD> int run_block(const MuonArgs &a, int64_t matrices, int lds, hipStream_t s)
{
    const auto fn = &ks_muon_block_kernel<T, WAVES, HELD>;
    if (lds > 64 * 1024) {
        const int rc = ensure_dynamic_lds((const void *)fn, (int)LDS_MOST);
        if (rc != KSMM_OK) return rc;
    }
    hipLaunchKernelGGL(fn, dim3((unsigned)matrices), dim3(64 * WAVES), lds, s, a);
    return launched();
}

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
struct Space {
    int M, N, chunks;
    int64_t x[4], gram, poly, squares, u, total;  // x: two of X, two of its transpose; bytes
};
Space space(int64_t matrices, int c, int b)
{
    Space w;
    const int m = std::min(c, b), n = std::max(c, b);
    w.M = up64(m);
    w.N = up64(n);
    w.chunks = (int)std::max<int64_t>(1, std::min<int64_t>(256, 1024 / matrices));
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t was = at;
        at += align256(bytes);
        return was;
    };
    for (int64_t &x : w.x) x = take(4 * matrices * w.M * w.N);
    w.gram = take(4 * matrices * w.M * w.M);
    w.poly = take(4 * matrices * w.M * w.M);
    w.squares = take(4 * matrices * w.chunks);
    w.u = w.x[1];  // (the second X is written after u was read)
    w.total = at;
    return w;
}

template <typename T> int run(const MuonArgs &a, int64_t matrices, char *ws, hipStream_t s)
{
    const int m = std::min(a.c, a.b), n = std::max(a.c, a.b);
    if (fits_lds(m, n)) {
        const int lds = (int)block_lds(m, n), tiles = up16(m) / 16 * (up16(n) / 16);
        if (tiles <= 1) return run_block<T, 1, 1>(a, matrices, lds, s);
        if (tiles <= 4) return run_block<T, 4, 1>(a, matrices, lds, s);
        if (tiles <= 16) return run_block<T, 16, 1>(a, matrices, lds, s);
        return tiles <= 64 ? run_block<T, 16, 4>(a, matrices, lds, s) : run_block<T, 16, 8>(a, matrices, lds, s);
    }
    const Space w = space(matrices, a.c, a.b);
    const int64_t mt = w.M / TILE, square = matrices * mt * mt, full = matrices * mt * (w.N / TILE);
    if (full > 0x7fffffffLL || matrices * w.chunks > 0x7fffffffLL) return KSMM_ERR_TOO_LARGE;
    const bool flip = a.c > a.b;
    auto split = [&](int64_t at, int64_t values) { return Split{(half_t *)(ws + at), (half_t *)(ws + at) + values}; };
    const int64_t values = matrices * w.M * w.N;
    Split x = split(w.x[0], values), y = split(w.x[1], values), xt = split(w.x[2], values), yt = split(w.x[3], values);
    const Split gram = split(w.gram, matrices * w.M * w.M), poly = split(w.poly, matrices * w.M * w.M);
    float *const u = (float *)(ws + w.u), *const squares = (float *)(ws + w.squares);
    hipLaunchKernelGGL((ks_muon_load_kernel<T>), dim3((unsigned)(matrices * w.chunks)), dim3(256), 0, s, a, u, squares, w.chunks);
    hipLaunchKernelGGL(ks_muon_split_kernel, dim3((unsigned)full), dim3(256), 0, s, a, u, squares, w.chunks, flip ? xt : x, flip ? x : xt,
                       flip ? w.N : w.M, flip ? w.M : w.N);
    int rc = KSMM_OK;
    auto gemm = [&](auto fn, int groups, int64_t tiles, Split l, Split r, Split old, Split out, Split turned, bool last) {
        const int lds = groups * TILE * TILE * 4;
        if (lds > 64 * 1024 && rc == KSMM_OK) rc = ensure_dynamic_lds((const void *)fn, lds);
        if (rc != KSMM_OK) return;
        hipLaunchKernelGGL(fn, dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(64 * groups), lds, s, a, l, r, old, out, turned, w.M, w.N, last, (int)tiles);
    };
    // waves that share K: 8 for the square products, whose tiles are few, 4 for the others ((1,1536,384,2) of two parts 200 us; before
    // loads were kept ahead 223, 4 everywhere 227, 8 everywhere 241; (1,256,256,16) 104; 115, 112, 116)
    for (int i = 0; i < a.steps; ++i) {
        gemm(&ks_muon_gemm_kernel<T, GRAM, 8>, 8, square, x, x, x, gram, gram, false);
        gemm(&ks_muon_gemm_kernel<T, POLY, 8>, 8, square, gram, gram, gram, poly, poly, false);
        gemm(&ks_muon_gemm_kernel<T, APPLY, 4>, 4, full, xt, poly, x, y, yt, i + 1 == a.steps);
        std::swap(x, y);
        std::swap(xt, yt);
    }
    return rc == KSMM_OK ? launched() : rc;
}

// sizes are rounded up, and chunks and walks step over the end, in 32 bits
bool too_large(int64_t blocks, int c, int b, int parts) { return (double)blocks * c * b * parts > 2147483647.0 - 4096.0; }

// A step is a polynomial of the singular values, which are at most one in X0.  Whether any with such values can leave what pairs of
// fp16 numbers hold: no entry of X, its Gram matrix or the polynomial of that is larger than the largest singular value of each.
bool in_range(const float *p, int steps)
{
    const double p0 = p[0], p1 = p[1], p2 = p[2], most = 60000.0;
    auto largest = [](double top, auto f, std::initializer_list<double> inner) {  // of |f| on [0, top]: at the top, or where its slope is zero
        double v = std::fabs(f(top));
        for (double at : inner)
            if (at > 0 && at < top) v = std::max(v, std::fabs(f(at)));
        return v;
    };
    const double root = 9 * p1 * p1 - 20 * p0 * p2, q = root > 0 ? std::sqrt(root) : 0.0;
    // p0 + 3 p1 t + 5 p2 t^2 = 0, t the square of a singular value
    const double t0 = p2 != 0 ? (-3 * p1 + q) / (10 * p2) : p1 != 0 ? -p0 / (3 * p1) : 0.0, t1 = p2 != 0 ? (-3 * p1 - q) / (10 * p2) : 0.0;
    double s = 1.0;
    for (int i = 0; i < steps; ++i) {
        const double gram = s * s, poly = largest(gram, [&](double g) { return p1 * g + p2 * g * g; }, {p2 != 0 ? -p1 / (2 * p2) : 0.0});
        const double next = largest(s, [&](double x) { return x * (p0 + x * x * (p1 + x * x * p2)); }, {t0 > 0 ? std::sqrt(t0) : 0.0, t1 > 0 ? std::sqrt(t1) : 0.0});
        if (!(gram <= most && poly <= most && next <= most)) return false;
        if (next == s) break;  // (and so it goes on)
        s = next;
    }
    return true;
}

int check(const ksmm_muon_desc *d, int64_t blocks, int c, int b, int parts, int dtype)
{
    if (!d) return KSMM_ERR_NULL_POINTER;
    if (blocks < 1 || c < 1 || b < 1 || parts < 1) return KSMM_ERR_BAD_PATTERN;
    if (dtype != KSMM_F32 && dtype != KSMM_F16) return KSMM_ERR_BAD_DTYPE;
    if (d->steps < 1) return KSMM_ERR_BAD_ALGO;
    if (too_large(blocks, c, b, parts)) return KSMM_ERR_TOO_LARGE;
    return in_range(d->coefficients, d->steps) ? KSMM_OK : KSMM_ERR_BAD_ALGO;
}

}  // namespace

}  // namespace ksmm

using namespace ksmm;

extern "C" {

int64_t ksmm_muon_workspace(int64_t blocks, int c, int b, int parts)
{
    if (blocks < 1 || c < 1 || b < 1 || parts < 1) return KSMM_ERR_BAD_PATTERN;
    if (too_large(blocks, c, b, parts)) return KSMM_ERR_TOO_LARGE;
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
    {
        // (momentum, masters and weights may be updated in their place, and nowhere else)
        const int64_t values = blocks * parts * c * b, wide = 4 * values, size = values * (int64_t)dtype_size(dtype);
        const bool own_m = momentum_out == momentum, own_master = master_out == master, own_w = out == weight;
        const Span in[] = {{grad, size}, {own_m ? nullptr : momentum, wide}, {own_w ? nullptr : weight, size}, {own_master ? nullptr : master, wide}};
        const Span written[] = {{momentum ? momentum_out : nullptr, wide}, {master ? master_out : nullptr, wide}, {out, size}, {need ? workspace : nullptr, need}};
        if (any_overlap(in, written)) return KSMM_ERR_ALIAS;
    }
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
    a.follow = desc->follow;
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
