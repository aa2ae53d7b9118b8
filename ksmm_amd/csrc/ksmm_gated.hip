// Gated projection: two factors of one pattern that share their input, the activation of one and the product in one
// kernel.
//
//     z[a_i, p, b_i, d_i, n] = sum_c W[a_i, p, b_i, c_i, d_i] x[a_i, c_i, d_i, n] + bias[a_i, p, b_i, d_i]    (p = 0, 1)
//     h[a_i, b_i, d_i, n]    = act(z[a_i, 0, b_i, d_i, n]) * z[a_i, 1, b_i, d_i, n]
//
// The weights of both lie side by side, (a*d*c, 2*b), gate columns first: as kernel-format weights they are ONE factor
// with pattern (a, 2b, c, d), which is what the gradients of input and weights run as, on the kernels that any factor
// has.  z itself never reaches memory on the way forward; backward it is computed again, and
//     dz[0] = dh * z1 * act'(z0),  dz[1] = dh * act(z0)
// leave the kernel in its place (MODE 1).  Sums are fp32; h is rounded once, from fp32.  So is dz, and the gradients, sums over it, once
// more: dz in the tensors' type is what the 16-bit matrix instructions take.  In fp16 that costs gradients 2.9e-4 in the 2-norm for
// 2.1e-4 of the last rounding alone, and the range of the type, as the same layers apart would; a training pass over
// (1,768,192,2), 25088 rows, is 285 us, and in fp32, where dz has 32 bits, 1340.
//
// An MFMA tile has 32 rows of weights.  Batch-size-first these are 16 gate and 16 up columns of the same outputs, dealt
// so that a lane (which holds rows 8j + 4*(lane/32) + i) has gate and up of 8 outputs in a row: the product needs no
// other lane's values and leaves as whole vectors.  Batch-size-last the operands swap sides: a lane holds one output's
// gate (or up) at 16 batch elements in a row, and gate and up are two tiles of the same lanes.
#include "ksmm_act.h"
#include "ksmm_mfma.h"

namespace ksmm {

namespace {

struct GatedArgs {
    const void *x, *w, *bias, *dh;
    void *out;  // h, or dz (MODE 1)
    int64_t batch;
    int a, b, c, d;
    int act;
};

// ---- MFMA operands: KS k values of one row or column a lane --------------------------------------------
// fp16: 8 k in a row from 8 * (lane / 32) on, one 32x32x16.  fp32: 4 k in a row from 4 * (lane / 32) on, four 32x32x2
// (the order of k within a sum is free, as long as both operands have the same)
template <typename T> struct op;
template <> struct op<half_t> {
    static constexpr int KS = 16, PER = 8;
    typedef half8_t type;
    __device__ static __forceinline__ float16_t mfma(type a, type b, float16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct op<float> {
    static constexpr int KS = 8, PER = 4;
    typedef float4_t type;
    __device__ static __forceinline__ float16_t mfma(type a, type b, float16_t c)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// column of a weight row (gate columns 0..tb-1, up columns tb..) that row r of the 16 + 16 tile holds
__device__ __forceinline__ int mixed_col(int r, int tb)
{
    const int rg = r >> 2, hh = rg & 1, j = rg >> 1;
    return (j >> 1) * tb + 8 * hh + 4 * (j & 1) + (r & 3);
}
// batch element that row r of a batch-size-last tile holds: a lane ends up with 16 in a row
__device__ __forceinline__ int run_col(int r)
{
    const int rg = r >> 2;
    return 16 * (rg & 1) + 4 * (rg >> 1) + (r & 3);
}

// k-outer operand S[k][col], columns by groups of 4: group rg (0..7) of the operand at column at(rg)
template <typename F> __device__ __forceinline__ half8_t k_outer(const half_t *s, int ld, int k0, int lane, F at)
{
    const int kq = lane >> 5, i16 = lane & 15, rg = 4 * ((lane >> 4) & 1) + (i16 & 3);
    const half_t *p = s + (k0 + 8 * kq + (i16 >> 2)) * ld + at(rg);
    typedef short4_t __attribute__((address_space(3))) * lds_ptr;
    typedef short short8_t __attribute__((ext_vector_type(8)));
    const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p));
    const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 4 * ld));
    return __builtin_bit_cast(half8_t, short8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
}
template <typename F> __device__ __forceinline__ float4_t k_outer(const float *s, int ld, int k0, int lane, F at)
{
    const float *p = s + (k0 + 4 * (lane >> 5)) * ld + at((lane & 31) >> 2) + (lane & 3);
    return float4_t{p[0], p[ld], p[2 * ld], p[3 * ld]};
}
// k-inner operand S[idx][k]
template <typename T> __device__ __forceinline__ typename op<T>::type k_inner(const T *s, int ld, int idx0, int k0, int lane)
{
    return *(const typename op<T>::type *)(s + (idx0 + (lane & 31)) * ld + k0 + op<T>::PER * (lane >> 5));
}

template <typename T> constexpr int EPV = 16 / (int)sizeof(T);
template <typename T, int N> struct Run {
    T e[N];
};
// count (<= N) elements from p on, the rest zeros; all of them in one or more 16-byte loads at element alignment
template <typename T, int N> __device__ __forceinline__ Run<T, N> load_run(const T *p, int count)
{
    Run<T, N> r;
    if (count >= N) {
        __builtin_memcpy(&r, p, sizeof(r));
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) r.e[e] = e < count ? p[e] : (T)0.f;
    }
    return r;
}
// elements from `first` on (all of them in one or more 16-byte stores)
template <typename T, int N> __device__ __forceinline__ void store_run(T *p, int first, const Run<T, N> &r)
{
    if (first <= 0) {
        __builtin_memcpy(p, &r, sizeof(r));
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e >= first) p[e] = r.e[e];
    }
}

// ---- tiles ---------------------------------------------------------------------------------------------
// Workgroup: TB outputs (2 * TB weight columns) of D neighbouring d_i of one a_i x TN rows of the batch; WB x WN waves.
// x and W arrive in slabs of TK, through registers into two LDS buffers in turn.  Batch-size-first a thread takes D * E
// values of a row, the E k of D neighbouring d_i, and writes them as D chunks of one d_i each (ALL: D is all of d, and
// these values lie in a row).
// Vectors that would cross the end of a row of weights, or of a batch-size-last row, are moved back to end with it, and
// so are their results: some outputs are computed twice.  They are stored once, by the vector that they were in before: the compiler
// rounds products of different places in a lane in different ways (to fp16 through fp32, or at once), and what would remain of two
// stores is whichever comes last.  (b >= 8, batch-size-last batch >= 16.)
template <typename T, bool LAST, int D, int TB, int TN, int TK, int WB, int WN> struct Tile {
    static constexpr int THREADS = 64 * WB * WN, E = EPV<T>;
    static constexpr int BT = TB / WB / (LAST ? 32 : 16), NT = TN / WN / 32;  // MFMA tiles a wave: outputs (16, or 32 as gate and up), rows
    static constexpr int LDW = pads<T>::outer(2 * TB), LDX = LAST ? pads<T>::outer(TN) : pads<T>::inner(TK);
    static constexpr int W_PLANE = TK * LDW, X_PLANE = LAST ? TK * LDX : TN * LDX;
    static constexpr int BUF = D * (W_PLANE + X_PLANE), LDS_BYTES = 2 * BUF * (int)sizeof(T);
    static constexpr int W_UNITS = D * TK * 2 * TB / E, X_UNITS = TK * TN / E;
    static constexpr int W_PER = W_UNITS / THREADS, X_PER = X_UNITS / THREADS;
    static_assert(W_UNITS % THREADS == 0 && X_UNITS % THREADS == 0 && TK % op<T>::KS == 0 && (!LAST || D == 1), "shape");
    static_assert(LDS_BYTES <= 160 * 1024, "LDS");
};

template <typename T, bool LAST, int D, bool ALL, int TB, int TN, int TK, int WB, int WN, int MODE>
__global__ __launch_bounds__(64 * WB *WN, 2) void ks_gated_kernel(GatedArgs g, int b_tiles, int n_tiles, int blocks)
{
    typedef Tile<T, LAST, D, TB, TN, TK, WB, WN> C;
    typedef op<T> O;
    constexpr int E = C::E;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    T *const lds = (T *)smem;
    auto ws = [&](int buf, int p) { return lds + buf * C::BUF + p * C::W_PLANE; };
    auto xs = [&](int buf, int p) { return lds + buf * C::BUF + D * C::W_PLANE + p * C::X_PLANE; };

    // each XCD gets a contiguous range of tiles: those that share rows of x share an L2
    const int per_xcd = (blocks + 7) / 8, lid = (blockIdx.x % 8) * per_xcd + blockIdx.x / 8;
    if (lid >= blocks) return;
    const int a = g.a, b = g.b, c = g.c, d = ALL ? D : g.d, dg = ALL ? 1 : d / D;
    const int bt = lid % b_tiles, rest = lid / b_tiles;
    // (batch-size-first the d_i of an a_i share cache lines of x and h: they are neighbours)
    const int grp = LAST ? rest / n_tiles : rest % (a * dg), nt = LAST ? rest % n_tiles : rest / (a * dg);
    const int a_i = grp / dg, d0 = ALL ? 0 : (grp - a_i * dg) * D;
    const int b0 = bt * TB, B = (int)g.batch, n0 = nt * TN;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wb = wave / WN, wn = wave % WN;
    const int lq = lane >> 5, l32 = lane & 31;
    const int64_t in_size = (int64_t)a * c * d;
    const T *const w = (const T *)g.w + (int64_t)(a_i * d + d0) * c * 2 * b;
    const T *const x = LAST ? (const T *)g.x + ((int64_t)a_i * c * d + d0) * B : (const T *)g.x + (int64_t)a_i * c * d + d0;

    // what a thread loads: places in the first slab
    const T *wp[C::W_PER], *xp[C::X_PER];
#pragma unroll
    for (int i = 0; i < C::W_PER; ++i) {
        const int v = tid + i * C::THREADS, col = v % (2 * TB / E) * E, row = v / (2 * TB / E);
        wp[i] = w + ((int64_t)(row / TK) * c + row % TK) * 2 * b + col / TB * b + min(b0 + col % TB, b - E);
    }
#pragma unroll
    for (int i = 0; i < C::X_PER; ++i) {
        const int v = tid + i * C::THREADS;
        if constexpr (LAST)
            xp[i] = x + (int64_t)(v / (TN / E)) * d * B + min(n0 + v % (TN / E) * E, B - E);
        else  // (rows past the batch: the last one again, not stored)
            xp[i] = x + min(n0 + v / (TK / E), B - 1) * in_size + (int64_t)(v % (TK / E) * E) * d;
    }
    const int64_t w_step = (int64_t)TK * 2 * b, x_step = LAST ? (int64_t)TK * d * B : (int64_t)TK * d;
    Run<T, E> wr[C::W_PER];
    Run<T, D * E> xr[C::X_PER];
    auto gload = [&](int s, bool whole) {
#pragma unroll
        for (int i = 0; i < C::W_PER; ++i) {
            const T *const from = wp[i] + s * w_step;
            if (whole)
                wr[i] = load_run<T, E>(from, E);
            else  // past the block's rows: zeros
                wr[i] = load_run<T, E>(from, s * TK + (tid + i * C::THREADS) / (2 * TB / E) % TK < c ? E : 0);
        }
#pragma unroll
        for (int i = 0; i < C::X_PER; ++i) {
            const int v = tid + i * C::THREADS;
            const T *const from = xp[i] + s * x_step;
            if constexpr (LAST) {
                xr[i] = load_run<T, E>(from, whole || s * TK + v / (TN / E) < c ? E : 0);
            } else {
                const int count = whole ? E : min(max(c - s * TK - v % (TK / E) * E, 0), E);
                if constexpr (ALL) {
                    xr[i] = load_run<T, D * E>(from, count * D);
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const Run<T, D> q = load_run<T, D>(from + (int64_t)e * d, e < count ? D : 0);
#pragma unroll
                        for (int p = 0; p < D; ++p) xr[i].e[e * D + p] = q.e[p];
                    }
                }
            }
        }
    };
    auto lstore = [&](int buf) {
#pragma unroll
        for (int i = 0; i < C::W_PER; ++i) {
            const int v = tid + i * C::THREADS, cv = v % (2 * TB / E), row = v / (2 * TB / E);
            *(Run<T, E> *)__builtin_assume_aligned(ws(buf, row / TK) + (row % TK) * C::LDW + cv * E, 16) = wr[i];
        }
#pragma unroll
        for (int i = 0; i < C::X_PER; ++i) {
            const int v = tid + i * C::THREADS;
            if constexpr (LAST) {
                *(Run<T, E> *)__builtin_assume_aligned(xs(buf, 0) + v / (TN / E) * C::LDX + v % (TN / E) * E, 16) = xr[i];
            } else {
#pragma unroll
                for (int p = 0; p < D; ++p) {
                    Run<T, E> q;
#pragma unroll
                    for (int e = 0; e < E; ++e) q.e[e] = xr[i].e[e * D + p];
                    *(Run<T, E> *)__builtin_assume_aligned(xs(buf, p) + v / (TK / E) * C::LDX + v % (TK / E) * E, 16) = q;
                }
            }
        }
    };

    constexpr int PARTS = LAST ? 2 : 1;  // accumulators an output tile: gate and up apart, or both in one
    float16_t acc[D][PARTS][C::BT][C::NT];
    const T *const bias = (const T *)g.bias;
    // the lane's outputs of tile i: a run of 8 (E at a time, each moved back on its own), or one; and by how much they were moved
    auto run_at = [&](int i, int e) { return min(b0 + (wb * C::BT + i) * 16 + 8 * lq + e, b - E); };
    auto run_moved = [&](int i, int e) { return b0 + (wb * C::BT + i) * 16 + 8 * lq + e - run_at(i, e); };
    auto one_at = [&](int i) {
        const int at = b0 + (wb * C::BT + i) * 32 + l32 / E * E;
        return min(at, b - E) + l32 % E;
    };
    auto one_moved = [&](int i) { return b0 + (wb * C::BT + i) * 32 + l32 - one_at(i); };
    // the sums start at the bias: its loads go out before those of the first slab
    constexpr int BIAS = LAST ? 1 : 8 * D;
    T bv[2][C::BT][BIAS];
    if (bias) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < C::BT; ++i) {
                const T *const from = bias + ((int64_t)(a_i * 2 + q) * b) * d + d0;
                if constexpr (LAST) {
                    bv[q][i][0] = from[(int64_t)one_at(i) * d];
                } else if constexpr (ALL) {
#pragma unroll
                    for (int h = 0; h < 8; h += E) __builtin_memcpy(&bv[q][i][h * D], from + (int64_t)run_at(i, h) * D, E * D * sizeof(T));
                } else {
#pragma unroll
                    for (int h = 0; h < 8; ++h) __builtin_memcpy(&bv[q][i][h * D], from + (int64_t)(run_at(i, h / E * E) + h % E) * d, D * sizeof(T));
                }
            }
    } else {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < C::BT; ++i)
#pragma unroll
                for (int e = 0; e < BIAS; ++e) bv[q][i][e] = (T)0.f;
    }
    const int steps = (c + TK - 1) / TK;
    gload(0, TK <= c);
#pragma unroll
    for (int p = 0; p < D; ++p)
#pragma unroll
        for (int i = 0; i < C::BT; ++i)
#pragma unroll
            for (int j = 0; j < C::NT; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    if constexpr (LAST) {
                        acc[p][0][i][j][e] = (float)bv[0][i][0];
                        acc[p][PARTS - 1][i][j][e] = (float)bv[1][i][0];
                    } else {
                        acc[p][0][i][j][e] = (float)bv[e / 8][i][e % 8 * D + p];
                    }
                }
    lstore(0);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        const int buf = s & 1;
        if (s + 1 < steps) {
            if ((s + 2) * TK <= c)
                gload(s + 1, true);
            else
                gload(s + 1, false);
        }
#pragma unroll
        for (int k0 = 0; k0 < TK; k0 += O::KS)
#pragma unroll
            for (int p = 0; p < D; ++p) {
                const T *wl = ws(buf, p), *xl = xs(buf, p);
                typename O::type fw[PARTS][C::BT], fx[C::NT];
#pragma unroll
                for (int q = 0; q < PARTS; ++q)
#pragma unroll
                    for (int i = 0; i < C::BT; ++i) {
                        if constexpr (LAST) {
                            const int col = q * TB + (wb * C::BT + i) * 32;
                            fw[q][i] = k_outer(wl, C::LDW, k0, lane, [&](int rg) { return col + 4 * rg; });
                        } else {
                            const int col = (wb * C::BT + i) * 16;
                            fw[q][i] = k_outer(wl, C::LDW, k0, lane, [&](int rg) { return col + mixed_col(4 * rg, TB); });
                        }
                    }
#pragma unroll
                for (int j = 0; j < C::NT; ++j) {
                    const int n = (wn * C::NT + j) * 32;
                    if constexpr (LAST)
                        fx[j] = k_outer(xl, C::LDX, k0, lane, [&](int rg) { return n + run_col(4 * rg); });
                    else
                        fx[j] = k_inner<T>(xl, C::LDX, n, k0, lane);
                }
#pragma unroll
                for (int q = 0; q < PARTS; ++q)
#pragma unroll
                    for (int i = 0; i < C::BT; ++i)
#pragma unroll
                        for (int j = 0; j < C::NT; ++j)
                            acc[p][q][i][j] = LAST ? O::mfma(fx[j], fw[q][i], acc[p][q][i][j]) : O::mfma(fw[q][i], fx[j], acc[p][q][i][j]);
            }
        if (s + 1 < steps) lstore(buf ^ 1);
        __syncthreads();
    }

    const T *const dh = (const T *)g.dh;
    T *const out = (T *)g.out;
    const int64_t out_size = (int64_t)a * b * d;
    // (nearly all tiles have no vector that was moved: one branch around everything, where one at each vector took 2 to 23 % of a call)
    auto finish_tile = [&](auto act_of, auto moved_of) {
        constexpr int ACT = decltype(act_of)::value;
        constexpr bool MOVED = decltype(moved_of)::value;
        // N values of gate and up (and of dh) at a time: a vector of the result, stored from element `first` on
        auto finish = [&](auto zg, auto zu, const T *dh_at, T *to_g, T *to_u, int first, auto count) {
            constexpr int N = decltype(count)::value;
            Run<T, N> in, r0, r1;
            if constexpr (MODE == 1) in = load_run<T, N>(dh_at, N);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float gate = zg(e), up = zu(e);
                float slope = 0.f;
                const float v = activate<T, ACT, MODE == 1>(gate, slope);
                if constexpr (MODE == 0) {
                    r0.e[e] = (T)(v * up);
                } else {
                    const float t = (float)in.e[e];
                    r0.e[e] = (T)(t * up * slope);
                    r1.e[e] = (T)(t * v);
                }
            }
            store_run<T, N>(to_g, first, r0);
            if constexpr (MODE == 1) store_run<T, N>(to_u, first, r1);
        };
        if constexpr (LAST) {
            // a lane: one output, 16 rows of the batch in a row, E at a time
#pragma unroll
            for (int i = 0; i < C::BT; ++i) {
                if (b0 + (wb * C::BT + i) * 32 >= b || (MOVED && l32 % E < one_moved(i))) continue;
                const int64_t bi = one_at(i);
                const int64_t fg = (a_i * 2 * (int64_t)b + bi) * d + d0, fh = (a_i * (int64_t)b + bi) * d + d0;
#pragma unroll
                for (int j = 0; j < C::NT; ++j)
#pragma unroll
                    for (int v = 0; v < 16; v += E) {
                        const int at = n0 + (wn * C::NT + j) * 32 + 16 * lq + v;
                        if (at >= B) continue;
                        const int n = min(at, B - E);
                        finish([&](int e) { return acc[0][0][i][j][v + e]; }, [&](int e) { return acc[0][PARTS - 1][i][j][v + e]; },
                               dh + fh * B + n, out + (MODE == 0 ? fh : fg) * B + n, out + (fg + (int64_t)b * d) * B + n, MOVED ? at - n : 0,
                               std::integral_constant<int, E>());
                    }
            }
        } else {
            // a lane: one row of the batch, 8 outputs of D neighbouring d_i
#pragma unroll
            for (int j = 0; j < C::NT; ++j) {
                const int n = n0 + (wn * C::NT + j) * 32 + l32;
                if (n >= B) continue;
                const T *const dh_n = dh + n * out_size + d0;
                T *const out_n = out + n * (MODE + 1) * out_size + d0;
#pragma unroll
                for (int i = 0; i < C::BT; ++i) {
                    if (b0 + (wb * C::BT + i) * 16 + 8 * lq >= b) continue;
                    if constexpr (ALL) {
#pragma unroll
                        for (int h = 0; h < 8; h += E) {
                            const int64_t fh = ((int64_t)a_i * b + run_at(i, h)) * D, fg = fh + (int64_t)a_i * b * D * MODE;
#pragma unroll
                            for (int q = 0; q < D; ++q)  // vector q of the E * D values
                                finish([&](int e) { return acc[(q * E + e) % D][0][i][j][h + (q * E + e) / D]; },
                                       [&](int e) { return acc[(q * E + e) % D][0][i][j][8 + h + (q * E + e) / D]; }, dh_n + fh + q * E,
                                       out_n + fg + q * E, out_n + fg + (int64_t)b * D + q * E, MOVED ? run_moved(i, h) * D - q * E : 0,
                                       std::integral_constant<int, E>());
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < 8; ++h) {
                            if (MOVED && h % E < run_moved(i, h / E * E)) continue;
                            const int64_t at = run_at(i, h / E * E) + h % E, fh = ((int64_t)a_i * b + at) * d, fg = fh + (int64_t)a_i * b * d * MODE;
                            finish([&](int e) { return acc[e][0][i][j][h]; }, [&](int e) { return acc[e][0][i][j][8 + h]; }, dh_n + fh,
                                   out_n + fg, out_n + fg + (int64_t)b * d, 0, std::integral_constant<int, D>());
                        }
                    }
                }
            }
        }
    };
    with_act(g.act, [&](auto act_of) {
        if ((b0 + TB <= b || b % (LAST ? 32 : 8) == 0) && (!LAST || n0 + TN <= B || B % E == 0))
            finish_tile(act_of, std::false_type());
        else
            finish_tile(act_of, std::true_type());
    });
}

// ---- fp16 in aligned vectors: a ring of slabs ----------------------------------------------------------
// The tile above spends its time waiting: a slab of 32 k is a quarter of a microsecond of products, its loads take two.
// Here they go straight to LDS (no registers), three slabs of 16 k ahead, and a workgroup stays for many tiles.  Two workgroups a CU:
// one multiplies while the other finishes a tile (GLU in the vector ALU takes as long as the products of c = 192).
//
// What counts as landed is counted by hand: a slab's loads are followed by those of two more (2 * L of them), and, in a tile's last two
// iterations, by the loads that its end needs (bias of the next tile, dh; EARLY of them, each an instruction of its own in the
// compiled code).  Those are ordinary loads, and the compiler, which does not see the ones to LDS, waits for them at the
// head of the next tile with everything issued before: its first three slabs, and this one's stores.  So a tile begins with its slabs
// landed, and stores do not run on behind it.
//
// d_i = 2: a row's (k, d_i) pairs are split into the operands of both d_i when they are read (one v_perm a register).
// The sums start at the bias: one product of (bias, 0, ..) and (1, 0, ..).  Results go through 4 KB of LDS a wave, and
// leave as rows of 128 bytes.
//
// A kernel an activation: with a branch on it inside, MODE 1 with 128 outputs of one d_i or 64 of two spills 21 to 34 registers a lane
// around its stores, and the number of one activation's registers costs the others time ((1,768,192,2), 25088 rows, a
// training pass 285 us; in one kernel 314, and 301 while GELU had a coefficient less).
//
// (1,768,192,2), 25088 rows forward 52 us: 29.6 GFLOP at 566 TFLOP/s; 96 MB of x and h, 1.9 TB/s.  The matrix cores are busy for 31 %
// of the SIMDs' time: what is left is the wait at each tile's head, and the vector ALU's work on the results, which the other
// workgroup's products cover in part.
constexpr int vmcnt_imm(int n) { return (n & 15) | (7 << 4) | (15 << 8) | (((n >> 4) & 3) << 14); }
typedef __attribute__((address_space(3))) unsigned char *lds_bytes_t;

// 16 bytes a lane from base (uniform) + offset to LDS, 1024 bytes a wave from `to` on
__device__ __forceinline__ void to_lds(const void *base, uint32_t offset, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(to) : "memory", "m0");
}

template <bool LAST, int D, int TB, int MODE> struct Ring {
    static constexpr int WB = 2, WN = 2, TN = 128, TK = 16, ST = 4, THREADS = 256;
    static constexpr int BT = TB / WB / (LAST ? 32 : 16), NT = 2, PARTS = LAST ? 2 : 1;
    static constexpr int W_CPR = 2 * TB / 8, X_CPR = LAST ? TN / 8 : TK * D / 8, X_ROWS = LAST ? TK : TN;  // 16-byte chunks a row
    static constexpr int W_PLANE = TK * W_CPR * 16, W_BYTES = D * W_PLANE, X_BYTES = X_ROWS * X_CPR * 16, STAGE = W_BYTES + X_BYTES;
    static constexpr int LW = W_BYTES / 16 / THREADS, LX = X_BYTES / 16 / THREADS, L = LW + LX;
    static constexpr int UNITS = LAST ? BT : NT;                       // pieces of 32 rows that a wave's results leave in
    static constexpr int O_CPR = LAST ? 8 : TB / WB * D * 2 / 16;      // chunks a row of them
    static constexpr int O_IT = 32 * O_CPR / 64, PIECE = 32 * O_CPR * 16;
    static constexpr int LDS_BYTES = ST * STAGE + 4 * PIECE;
    static constexpr int BIASES = LAST ? 2 * BT : D * BT, EARLY = BIASES + (MODE ? O_IT : 0);
    static constexpr int WAIT = (ST - 2) * L;
    static_assert(W_BYTES % (16 * THREADS) == 0 && X_BYTES % (16 * THREADS) == 0 && (!LAST || D == 1) && D <= 2, "loads");
    static_assert(TB == 64 || TB == 128, "weight swizzle");
    static_assert(WAIT + EARLY <= 63 && LDS_BYTES <= 80 * 1024, "ring");
    static_assert(BT * PARTS * NT * D * 16 <= 128, "accumulators");
};

// where chunk cc of row `row` lies (and, as these are their own inverses, what the chunk that lies there is)
template <int TB, bool LAST> __device__ __forceinline__ int w_swizzle(int row, int cc)
{
    if (LAST) return cc ^ (4 * (row & 3));                  // operands of 32 columns in a row: 4 rows x 64 bytes at a time
    const int r = cc ^ (2 * (row & 3));                     // 16 gate and 16 up columns: 4 rows x (32 + 32)
    return TB == 128 ? r ^ ((r >> 4) * 8) : r;
}
template <bool LAST, int CPR> __device__ __forceinline__ int x_swizzle(int row, int cc)
{
    if (LAST) return cc ^ (4 * (row & 3));
    return cc ^ (CPR == 2 ? (row >> 3) & 1 : (row >> 2) & 3);
}
template <int CPR> __device__ __forceinline__ int o_swizzle(int row, int cc) { return cc ^ (CPR == 8 ? (row >> 1) & 7 : (row >> 2) & 3); }

template <bool LAST, int D, int TB, int MODE, int ACT>
__global__ __launch_bounds__(256, 2) void ks_gated_ring_kernel(GatedArgs g, int b_tiles, int tiles)
{
    typedef Ring<LAST, D, TB, MODE> C;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_bytes_t)smem;
    const int a = g.a, b = g.b, c = g.c, d = LAST ? g.d : D, groups = LAST ? a * d : a, B = (int)g.batch;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wb = wave / C::WN, wn = wave % C::WN;
    const int l32 = lane & 31, lq = lane >> 5, steps = c / C::TK;
    // each XCD has a range of tiles, dealt to its workgroups in turn: those at work share rows of x in their L2
    const int per_xcd = (tiles + 7) / 8, first = (blockIdx.x & 7) * per_xcd, last = min(tiles, first + per_xcd), stride = gridDim.x / 8;
    const int mine = first + (blockIdx.x >> 3);
    if (mine >= last) return;
    const half_t *const x = (const half_t *)g.x, *const w = (const half_t *)g.w, *const bias = (const half_t *)g.bias;
    const half_t *const dh = (const half_t *)g.dh;
    half_t *const out = (half_t *)g.out;
    const int64_t in_size = (int64_t)a * c * d, out_size = (int64_t)a * b * d;

    struct At {
        int grp, b0, n0;
    };
    auto at = [&](int t) {
        const int bt = t % b_tiles, rest = t / b_tiles;
        return At{rest % groups, bt * TB, rest / groups * C::TN};
    };

    // ---- loads: slab `ls` of tile `lt` next
    uint32_t woff[C::LW], xoff[C::LX];
    const char *wsrc, *xsrc;
    const int64_t w_step = (int64_t)C::TK * 2 * b * 2, x_step = LAST ? (int64_t)C::TK * d * B * 2 : (int64_t)C::TK * D * 2;
    int lt = mine, ls = 0;
    auto begin_loads = [&]() {
        const At p = at(lt);
#pragma unroll
        for (int i = 0; i < C::LW; ++i) {
            const int v = tid + i * C::THREADS, row = v / C::W_CPR, cc = w_swizzle<TB, LAST>(row, v % C::W_CPR);
            const int part = cc / (TB / 8), col = p.b0 + cc % (TB / 8) * 8;
            woff[i] = (uint32_t)((((row / C::TK) * c + row % C::TK) * 2 * b + part * b + min(col, b - 8)) * 2);
        }
#pragma unroll
        for (int i = 0; i < C::LX; ++i) {
            const int v = tid + i * C::THREADS, row = v / C::X_CPR, cc = x_swizzle<LAST, C::X_CPR>(row, v % C::X_CPR);
            xoff[i] = LAST ? (uint32_t)((row * d * B + min(cc * 8, B - 8 - p.n0)) * 2)
                           : (uint32_t)((min(row, B - 1 - p.n0) * (int)in_size + cc * 8) * 2);
        }
        const int a_i = LAST ? p.grp / d : p.grp, d_i = LAST ? p.grp - a_i * d : 0;
        wsrc = (const char *)(w + (int64_t)(a_i * d + d_i) * c * 2 * b);
        xsrc = (const char *)(LAST ? x + ((int64_t)a_i * c * d + d_i) * B + p.n0 : x + p.n0 * in_size + (int64_t)a_i * c * D);
    };
    uint32_t to = lds0 + wave * 1024;
    int slot = 0;
    auto issue = [&]() {
#pragma unroll
        for (int i = 0; i < C::LW; ++i) to_lds(wsrc, woff[i], to + i * (C::THREADS * 16));
#pragma unroll
        for (int i = 0; i < C::LX; ++i) to_lds(xsrc, xoff[i], to + C::W_BYTES + i * (C::THREADS * 16));
        slot = slot + 1 == C::ST ? 0 : slot + 1;
        to = lds0 + wave * 1024 + slot * C::STAGE;
        wsrc += w_step;
        xsrc += x_step;
        if (++ls == steps) {
            // (behind the last tile its loads are repeated: the counts stay what they are)
            ls = 0;
            lt = lt + stride < last ? lt + stride : lt;
            begin_loads();
        }
    };

    // ---- operands
    uint32_t wa[C::PARTS][C::BT], xa[LAST ? C::NT : D];
    {
        const int i16 = lane & 15, hs = (lane >> 4) & 1, row = 8 * lq + (i16 >> 2);
#pragma unroll
        for (int q = 0; q < C::PARTS; ++q)
#pragma unroll
            for (int i = 0; i < C::BT; ++i) {
                int cc, half;
                if (LAST) {
                    cc = q * (TB / 8) + (wb * C::BT + i) * 4 + 2 * hs + ((i16 & 3) >> 1);
                    half = i16 & 1;
                } else {  // mixed_col: rows of the operand 4 * (4 * hs + (i16 & 3)) ..
                    cc = hs * (TB / 8) + (wb * C::BT + i) * 2 + (i16 & 1);
                    half = (i16 >> 1) & 1;
                }
                wa[q][i] = lds0 + row * (C::W_CPR * 16) + w_swizzle<TB, LAST>(row, cc) * 16 + half * 8;
            }
        if (LAST) {
#pragma unroll
            for (int j = 0; j < C::NT; ++j) {  // run_col
                const int cc = (wn * C::NT + j) * 4 + 2 * (i16 & 1) + hs, half = (i16 >> 1) & 1;
                xa[j % (LAST ? C::NT : D)] = lds0 + C::W_BYTES + row * (C::X_CPR * 16) + x_swizzle<LAST, C::X_CPR>(row, cc) * 16 + half * 8;
            }
        } else {
#pragma unroll
            for (int p = 0; p < D; ++p) {
                const int r = wn * C::NT * 32 + l32;
                xa[p] = lds0 + C::W_BYTES + r * (C::X_CPR * 16) + x_swizzle<LAST, C::X_CPR>(r, lq * D + p) * 16;
            }
        }
    }
    auto outer = [&](uint32_t addr, int row_bytes) {
        typedef short4_t __attribute__((address_space(3))) * lds_ptr;
        typedef short short8_t __attribute__((ext_vector_type(8)));
        const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds_bytes_t)(uintptr_t)addr);
        const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds_bytes_t)(uintptr_t)(addr + 4 * row_bytes));
        return __builtin_bit_cast(half8_t, short8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
    };
    auto inner = [&](uint32_t addr) {
        typedef uint4_t __attribute__((address_space(3))) * lds_ptr;
        return *(lds_ptr)(lds_bytes_t)(uintptr_t)addr;
    };

    // ---- bias: of row lane % 32 of each weight tile (of column lane % 32, batch-size-last)
    half_t bv[C::BIASES];
    auto load_bias = [&](int t) {
        const At p = at(t);
        const int a_i = LAST ? p.grp / d : p.grp, d_i = LAST ? p.grp - a_i * d : 0;
        const half_t *const from = bias ? bias + (int64_t)a_i * 2 * b * d + d_i : w;  // (no bias: anything, not used)
#pragma unroll
        for (int i = 0; i < C::BT; ++i)
#pragma unroll
            for (int q = 0; q < C::BIASES / C::BT; ++q) {
                int64_t k;
                if (LAST) {
                    k = ((int64_t)q * b + min(p.b0 + (wb * C::BT + i) * 32 + l32, b - 1)) * d;
                } else {
                    const int col = mixed_col(l32, 16);
                    k = ((int64_t)(col >> 4) * b + min(p.b0 + (wb * C::BT + i) * 16 + (col & 15), b - 1)) * D + q;
                }
                bv[i * (C::BIASES / C::BT) + q] = from[bias ? k : 0];
            }
    };
    auto unit_operand = [&](half_t v) { return half8_t{lq == 0 ? v : (half_t)0.f, (half_t)0.f, (half_t)0.f, (half_t)0.f, (half_t)0.f, (half_t)0.f, (half_t)0.f, (half_t)0.f}; };

    // ---- results: rows of a unit, 16 bytes a lane
    unsigned char *const piece = smem + C::ST * C::STAGE + wave * C::PIECE;
    const int o_row = lane / C::O_CPR, o_cc = lane % C::O_CPR;
    constexpr int O_STEP = 64 / C::O_CPR;
    // where chunk o_cc of row `row` of unit u lies in the result's layout with `parts` blocks of outputs an a_i; valid?
    auto place = [&](const At &p, int u, int row, int parts, int part, int64_t *k) {
        if (LAST) {
            const int a_i = p.grp / d, d_i = p.grp - a_i * d, bi = p.b0 + (wb * C::BT + u) * 32 + row, n = p.n0 + wn * 64 + o_cc * 8;
            *k = (((int64_t)(a_i * parts + part) * b + min(bi, b - 1)) * d + d_i) * B + min(n, B - 8);
            return bi < b && n < B;
        }
        const int n = p.n0 + (wn * C::NT + u) * 32 + row, bi = p.b0 + wb * (TB / C::WB) + o_cc * 8 / D;
        *k = (int64_t)min(n, B - 1) * out_size * parts + ((int64_t)(p.grp * parts + part) * b + min(bi, b - 8 / D)) * D;
        return n < B && bi < b;
    };
    // dh of one unit: the first one's loads go out early, the next one's when its predecessor is in LDS
    uint4_t dhv[C::O_IT];
    auto load_dh = [&](const At &p, int u) {
#pragma unroll
        for (int i = 0; i < C::O_IT; ++i) {
            int64_t k;
            place(p, u, i * O_STEP + o_row, 1, 0, &k);
            dhv[i] = *(const uint4_t *)(dh + k);
        }
    };
    auto wave_sync = [&]() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
    };
    // the lane's chunk q of its row in a piece
    auto mine_at = [&](int q) { return (uint4_t *)(piece + l32 * (C::O_CPR * 16) + o_swizzle<C::O_CPR>(l32, q) * 16); };

    float16_t acc[D][C::PARTS][C::BT][C::NT];
    auto finish = [&](int t) {
        const At p = at(t);
#pragma unroll
        for (int u = 0; u < C::UNITS; ++u) {
            if constexpr (MODE == 1) {
#pragma unroll
                for (int i = 0; i < C::O_IT; ++i) {
                    const int row = i * O_STEP + o_row;
                    *(uint4_t *)(piece + row * (C::O_CPR * 16) + o_swizzle<C::O_CPR>(row, o_cc) * 16) = dhv[i];
                }
                if (u + 1 < C::UNITS) load_dh(p, u + 1);
                wave_sync();
            }
            // the lane's values of the unit: chunks of 8
            constexpr int CHUNKS = LAST ? 4 : C::BT * D;
            Run<half_t, 8> r1[MODE ? CHUNKS : 1];
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k) {
                // LAST: j = k / 2, values 8 * (k % 2) ..; else tile i = k / D, values 8 q .. of (8 outputs x D)
                const int q = LAST ? k / 2 * 4 + lq * 2 + k % 2 : (k / D * 2 + lq) * D + k % D;
                Run<half_t, 8> in, r0;
                if constexpr (MODE == 1) in = __builtin_bit_cast(Run<half_t, 8>, *mine_at(q));
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int m = LAST ? k % 2 * 8 + e : (k % D * 8 + e) / D, pl = LAST ? 0 : (k % D * 8 + e) % D;
                    const float gate = LAST ? acc[0][0][u % C::BT][k / 2 % C::NT][m] : acc[pl][0][k / D % C::BT][u % C::NT][m];
                    const float up = LAST ? acc[0][C::PARTS - 1][u % C::BT][k / 2 % C::NT][m] : acc[pl][0][k / D % C::BT][u % C::NT][8 + m];
                    float slope = 0.f;
                    const float v = activate<half_t, ACT, MODE == 1>(gate, slope);
                    if constexpr (MODE == 0) {
                        r0.e[e] = (half_t)(v * up);
                    } else {
                        const float f = (float)in.e[e];
                        r0.e[e] = (half_t)(f * up * slope);
                        r1[MODE ? k : 0].e[e] = (half_t)(f * v);
                    }
                }
                *mine_at(q) = __builtin_bit_cast(uint4_t, r0);
            }
#pragma unroll
            for (int part = 0; part <= MODE; ++part) {
                if (part == 1) {
#pragma unroll
                    for (int k = 0; k < CHUNKS; ++k) {
                        const int q = LAST ? k / 2 * 4 + lq * 2 + k % 2 : (k / D * 2 + lq) * D + k % D;
                        *mine_at(q) = __builtin_bit_cast(uint4_t, r1[MODE ? k : 0]);
                    }
                }
                wave_sync();
#pragma unroll
                for (int i = 0; i < C::O_IT; ++i) {
                    const int row = i * O_STEP + o_row;
                    const uint4_t v = *(const uint4_t *)(piece + row * (C::O_CPR * 16) + o_swizzle<C::O_CPR>(row, o_cc) * 16);
                    int64_t k;
                    if (place(p, u, row, MODE + 1, part, &k)) *(uint4_t *)(out + k) = v;
                }
                wave_sync();
            }
        }
    };

    begin_loads();
    load_bias(mine);
#pragma unroll
    for (int s = 0; s < C::ST - 1; ++s) issue();
    int read = 0;  // slot that is multiplied next
    for (int t = mine; t < last; t += stride) {
        const half8_t one = unit_operand((half_t)1.f);
#pragma unroll
        for (int p = 0; p < D; ++p)
#pragma unroll
            for (int q = 0; q < C::PARTS; ++q)
#pragma unroll
                for (int i = 0; i < C::BT; ++i) {
                    const half8_t v = unit_operand(bias ? bv[i * (C::BIASES / C::BT) + (LAST ? q : p)] : (half_t)0.f);
#pragma unroll
                    for (int j = 0; j < C::NT; ++j) {
                        float16_t z;
#pragma unroll
                        for (int e = 0; e < 16; ++e) z[e] = 0.f;
                        acc[p][q][i][j] = LAST ? op<half_t>::mfma(one, v, z) : op<half_t>::mfma(v, one, z);
                    }
                }
        for (int s = 0; s < steps; ++s) {
            if (s > steps - C::ST + 1)
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(C::WAIT + C::EARLY));
            else
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(C::WAIT));
            __syncthreads();  // the slab landed for every wave, and everyone left the one before, whose place is filled next
            issue();
            if (s == steps - C::ST + 1) {
                load_bias(t + stride < last ? t + stride : t);
                if constexpr (MODE == 1) load_dh(at(t), 0);
            }
            const uint32_t base = read * C::STAGE;
            read = read + 1 == C::ST ? 0 : read + 1;
            half8_t fx[D][C::NT];
            if constexpr (LAST) {
#pragma unroll
                for (int j = 0; j < C::NT; ++j) fx[0][j] = outer(xa[j % (LAST ? C::NT : D)] + base, C::X_CPR * 16);
            } else {
#pragma unroll
                for (int j = 0; j < C::NT; ++j) {
                    uint4_t raw[D];
#pragma unroll
                    for (int p = 0; p < D; ++p) raw[p] = inner(xa[p] + base + j * 32 * C::X_CPR * 16);
                    if constexpr (D == 1) {
                        fx[0][j] = __builtin_bit_cast(half8_t, raw[0]);
                    } else {
                        uint4_t lo, hi;
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            const uint32_t even = raw[m / 2][2 * m % 4], odd = raw[m / 2][2 * m % 4 + 1];
                            lo[m] = __builtin_amdgcn_perm(odd, even, 0x05040100u);
                            hi[m] = __builtin_amdgcn_perm(odd, even, 0x07060302u);
                        }
                        fx[0][j] = __builtin_bit_cast(half8_t, lo);
                        fx[D - 1][j] = __builtin_bit_cast(half8_t, hi);
                    }
                }
            }
#pragma unroll
            for (int p = 0; p < D; ++p)
#pragma unroll
                for (int q = 0; q < C::PARTS; ++q)
#pragma unroll
                    for (int i = 0; i < C::BT; ++i) {
                        const half8_t fw = outer(wa[q][i] + base + p * C::W_PLANE, C::W_CPR * 16);
#pragma unroll
                        for (int j = 0; j < C::NT; ++j)
                            acc[p][q][i][j] = LAST ? op<half_t>::mfma(fx[p][j], fw, acc[p][q][i][j]) : op<half_t>::mfma(fw, fx[p][j], acc[p][q][i][j]);
                    }
        }
        finish(t);
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // repeated loads land before LDS goes to someone else
}

// ---- few rows ------------------------------------------------------------------------------------------
// A workgroup takes 16 outputs of one block x 32 rows of the batch; its waves share c and add their sums in LDS, one
// output and row a thread.  Operands come straight from global memory, element by element: any shape and alignment.
constexpr int FEW_WAVES = 8;
template <typename T, bool LAST, int MODE>
__global__ __launch_bounds__(64 * FEW_WAVES) void ks_gated_few_kernel(GatedArgs g, int b_tiles, int blocks)
{
    typedef op<T> O;
    __shared__ float red[FEW_WAVES][16 * 64];
    const int per_xcd = (blocks + 7) / 8, lid = (blockIdx.x % 8) * per_xcd + blockIdx.x / 8;
    if (lid >= blocks) return;
    const int a = g.a, b = g.b, c = g.c, d = g.d, groups = a * d;
    const int bt = lid % b_tiles, rest = lid / b_tiles, grp = rest % groups, nt = rest / groups;
    const int a_i = grp / d, d_i = grp - a_i * d, b0 = bt * 16;
    const int64_t B = g.batch, n0 = (int64_t)nt * 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l32 = lane & 31, lq = lane >> 5;
    const int64_t kstride = LAST ? (int64_t)d * B : d;
    const T *const w = (const T *)g.w + (int64_t)grp * c * 2 * b;
    const int64_t n_in = min(n0 + l32, B - 1);
    const T *const x = LAST ? (const T *)g.x + ((int64_t)a_i * c * d + d_i) * B + n_in
                            : (const T *)g.x + n_in * a * c * d + (int64_t)a_i * c * d + d_i;
    const int col = mixed_col(l32, 16);  // 16 of gate, 16 of up
    const T *const wl = w + (col >> 4) * b + min(b0 + (col & 15), b - 1);
    float16_t acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    for (int k0 = wave * O::KS; k0 < c; k0 += FEW_WAVES * O::KS) {
        typename O::type fw, fx;
#pragma unroll
        for (int e = 0; e < O::PER; ++e) {
            const int k = k0 + O::PER * lq + e;
            fw[e] = k < c ? wl[(int64_t)k * 2 * b] : (T)0.f;
            fx[e] = k < c ? x[(int64_t)k * kstride] : (T)0.f;
        }
        acc = O::mfma(fw, fx, acc);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) red[wave][e * 64 + lane] = acc[e];
    __syncthreads();
    // thread: lane's row of the batch, output 8 * (lane / 32) + e
    const int e = wave, bi = b0 + 8 * lq + e;
    const int64_t n = n0 + l32;
    if (bi >= b || n >= B) return;
    float zg = 0.f, zu = 0.f;
#pragma unroll
    for (int i = 0; i < FEW_WAVES; ++i) {
        zg += red[i][e * 64 + lane];
        zu += red[i][(8 + e) * 64 + lane];
    }
    const int64_t fg = ((int64_t)(a_i * 2) * b + bi) * d + d_i, fu = fg + (int64_t)b * d, fh = ((int64_t)a_i * b + bi) * d + d_i;
    if (g.bias) {
        zg += (float)((const T *)g.bias)[fg];
        zu += (float)((const T *)g.bias)[fu];
    }
    const int64_t out_size = (int64_t)a * b * d;
    auto at = [&](int64_t f, int64_t size) { return LAST ? f * B + n : n * size + f; };
    T *const out = (T *)g.out;
    with_act(g.act, [&](auto act_of) {
        float slope = 0.f;
        const float act = activate<T, decltype(act_of)::value, MODE == 1>(zg, slope);
        if (MODE == 0) {
            out[at(fh, out_size)] = (T)(act * zu);
        } else {
            const float v = (float)((const T *)g.dh)[at(fh, out_size)];
            out[at(fg, 2 * out_size)] = (T)(v * zu * slope);
            out[at(fu, 2 * out_size)] = (T)(v * act);
        }
    });
}

// ---- choices -------------------------------------------------------------------------------------------
int launched() { return hipGetLastError() == hipSuccess ? KSMM_OK : KSMM_ERR_LAUNCH; }

template <typename T, bool LAST, int MODE> int run_few(const GatedArgs &g, hipStream_t s)
{
    const int b_tiles = (g.b + 15) / 16;
    const int64_t blocks = (int64_t)b_tiles * g.a * g.d * ((g.batch + 31) / 32);
    if (blocks > THREADS_MOST / (64 * FEW_WAVES) - 8) return KSMM_ERR_TOO_LARGE;
    hipLaunchKernelGGL((ks_gated_few_kernel<T, LAST, MODE>), dim3((unsigned)((blocks + 7) / 8 * 8)), dim3(64 * FEW_WAVES), 0, s, g, b_tiles, (int)blocks);
    return launched();
}

template <typename T, bool LAST, int D, bool ALL, int TB, int TN, int TK, int WB, int WN, int MODE> int run_tile(const GatedArgs &g, hipStream_t s)
{
    typedef Tile<T, LAST, D, TB, TN, TK, WB, WN> C;
    const int b_tiles = (g.b + TB - 1) / TB;
    const int64_t n_tiles = (g.batch + TN - 1) / TN, blocks = (int64_t)b_tiles * g.a * (g.d / D) * n_tiles;
    if (blocks > THREADS_MOST / C::THREADS - 8) return KSMM_ERR_TOO_LARGE;
    const auto fn = &ks_gated_kernel<T, LAST, D, ALL, TB, TN, TK, WB, WN, MODE>;
    if (C::LDS_BYTES > 64 * 1024) {
        const int rc = ensure_dynamic_lds((const void *)fn, C::LDS_BYTES);
        if (rc != KSMM_OK) return rc;
    }
    hipLaunchKernelGGL(fn, dim3((unsigned)((blocks + 7) / 8 * 8)), dim3(C::THREADS), C::LDS_BYTES, s, g, b_tiles, (int)n_tiles, (int)blocks);
    return launched();
}

template <bool LAST, int D, int TB, int MODE> int run_ring(const GatedArgs &g, hipStream_t s)
{
    typedef Ring<LAST, D, TB, MODE> C;
    const int b_tiles = (g.b + TB - 1) / TB;
    const int64_t tiles = (int64_t)b_tiles * g.a * (LAST ? g.d : 1) * ((g.batch + C::TN - 1) / C::TN);
    if (tiles > 0x7ffffff0LL) return KSMM_ERR_TOO_LARGE;
    const int64_t grid = std::min<int64_t>(512, (tiles + 7) / 8 * 8);  // two workgroups a CU
    int rc = KSMM_OK;
    with_act(g.act, [&](auto act_of) {
        const auto fn = &ks_gated_ring_kernel<LAST, D, TB, MODE, decltype(act_of)::value>;
        rc = ensure_dynamic_lds((const void *)fn, C::LDS_BYTES);
        if (rc != KSMM_OK) return;
        hipLaunchKernelGGL(fn, dim3((unsigned)grid), dim3(C::THREADS), C::LDS_BYTES, s, g, b_tiles, (int)tiles);
        rc = launched();
    });
    return rc;
}
// vectors of 16 bytes everywhere, and offsets inside a tile that fit 32 bits
bool ring_ok(const GatedArgs &g, bool last)
{
    const uintptr_t p = (uintptr_t)g.x | (uintptr_t)g.w | (uintptr_t)g.out | (uintptr_t)g.dh;
    if ((p & 15) || g.b % 8 || g.c % 16 || g.c < 64 || (int64_t)g.d * g.c * 2 * g.b >= 1 << 29) return false;
    if (last) return g.batch % 8 == 0 && 16 * (int64_t)g.d * g.batch < 1 << 29;
    return g.d <= 2 && (int64_t)g.a * g.c * g.d * 128 < 1 << 29;
}

// Few rows or little work: tiles of 64 x 128 would leave most of the chip idle, and their time is that of one tile, whatever
// the batch.  Workgroups of 16 outputs x 32 rows, forward, us of few rows' kernel / of tiles:
//   fp32 batch-size-first   (1,768,192,1)  512 rows 13.1/19.1,  768 rows (1152 workgroups) 19.3/19.2
//   fp32 batch-size-last    (1,768,192,2)  512 rows 14.9/20.8,  768 rows (2304) 20.0/20.9;  (1,768,192,1) 1024 rows (1536) 14.7/20.7
//   fp16 batch-size-first   (6,64,64,1)    256 rows (192) 4.1/4.8,  384 rows (288) 5.1/4.8;  (1,768,192,2) 192 rows (576) 12.9/9.4
//   fp16 batch-size-last    (1,768,192,2)  256 rows (768) 6.4/6.9,  512 rows 9.7/6.9;  (6,64,64,1) 1024 rows (768) 4.8/5.4
// Up to 32 rows weights are read once anyway.  (Tiles need 8 outputs, and batch-size-last 16 rows.)
template <typename T, bool LAST> bool few(const GatedArgs &g)
{
    const int64_t limit = sizeof(T) == 4 ? (LAST ? 2048 : 1152) : (LAST ? 768 : 256);
    return g.batch <= 32 || g.b < 8 || (int64_t)((g.b + 15) / 16) * g.a * g.d * ((g.batch + 31) / 32) <= limit;
}

// Everything else: the ring where it can run, and the tile that goes through registers.  fp16 (1,768,192,2), 25088 rows, ring/tile:
// 61/73 us forward, 213/243 backward (all of it), batch-size-last 51/58 and 183/214; with few tiles they are level
// ((1,768,192,1) 3136 rows 8.3/8.2).  Weight tiles of the ring: 128 outputs halve the reads of x ((1,768,192,1), 25088 rows
// 29.6 us for 34.8; batch-size-last (1,768,192,2) 12544 rows, 1176 tiles, 28.4 for 32.3), 64 spread better
// (6272 rows, 588 tiles, 17.2 for 18.3; (1,768,192,1) 1576 rows 6.9 for 8.9) and waste less of a b of 64 (12.6 for 17.3).
// Neighbouring d_i in one workgroup share cache lines batch-size-first; fp32 6272 rows, together/one by one: d = 2 99/124 us,
// 3 25/29, 4 29/40, 8 58/71; fp16 d = 4 16/35, 16 59/120.
template <typename T, bool LAST, int MODE> int run(const GatedArgs &g, hipStream_t s)
{
    constexpr int TK = sizeof(T) == 4 ? 16 : 32;
    if (few<T, LAST>(g)) return run_few<T, LAST, MODE>(g, s);
    if constexpr (sizeof(T) == 2) {
        if (ring_ok(g, LAST)) {
            const bool wide = (g.b % 128 == 0 || g.b > 256) && (int64_t)((g.b + 127) / 128) * g.a * g.d * ((g.batch + 127) / 128) >= 768;
            if constexpr (LAST) {
                return wide ? run_ring<true, 1, 128, MODE>(g, s) : run_ring<true, 1, 64, MODE>(g, s);
            } else {
                if (g.d == 2) return run_ring<false, 2, 64, MODE>(g, s);
                return wide ? run_ring<false, 1, 128, MODE>(g, s) : run_ring<false, 1, 64, MODE>(g, s);
            }
        }
    }
    // fp32, whose matrix instructions leave time to feed smaller tiles: 64 x 64 while those of 128 rows are fewer than two a place
    // ((4,192,192,1) batch-size-last 6501 rows, 612 tiles, 46.5 us for 52.4; (1,768,192,2) 6272 rows 84 for 93, 25088 rows, 2352
    // tiles, 299 for 291); beyond, 8 waves a tile (284 for 291, batch-size-last 260 for 264; not d = 1, 142 for 139)
    constexpr int WN = sizeof(T) == 4 ? 4 : 2;
    if constexpr (sizeof(T) == 4) {
        if ((LAST || g.d <= 2) && (int64_t)((g.b + 63) / 64) * g.a * (LAST ? g.d : 1) * ((g.batch + 127) / 128) < 1024) {
            if constexpr (LAST)
                return run_tile<T, true, 1, false, 64, 64, TK, 2, 2, MODE>(g, s);
            else
                return g.d == 1 ? run_tile<T, false, 1, true, 64, 64, TK, 2, 2, MODE>(g, s) : run_tile<T, false, 2, true, 64, 64, TK, 2, 2, MODE>(g, s);
        }
    }
    if constexpr (LAST) {
        return run_tile<T, true, 1, false, 64, 128, TK, 2, WN, MODE>(g, s);
    } else {
        if (g.d == 1) return run_tile<T, false, 1, true, 64, 128, TK, 2, 2, MODE>(g, s);
        if (g.d == 2) return run_tile<T, false, 2, true, 64, 128, TK, 2, WN, MODE>(g, s);
        if (g.d == 3) return run_tile<T, false, 3, true, 32, 128, TK, 2, 2, MODE>(g, s);
        if (g.d == 4) return run_tile<T, false, 4, true, 32, 64, TK, 2, 2, MODE>(g, s);
        if (g.d % 4 == 0) return run_tile<T, false, 4, false, 32, 64, TK, 2, 2, MODE>(g, s);
        if (g.d % 3 == 0) return run_tile<T, false, 3, false, 32, 128, TK, 2, 2, MODE>(g, s);
        if (g.d % 2 == 0) return run_tile<T, false, 2, false, 64, 128, TK, 2, 2, MODE>(g, s);
        return run_tile<T, false, 1, false, 64, 128, TK, 2, 2, MODE>(g, s);
    }
}

}  // namespace

int gated_run(const void *x, const void *w, const void *bias, const void *dh, void *out, int64_t batch, int a, int b, int c, int d,
              int dtype, int bs_last, int act, int mode, hipStream_t s)
{
    const GatedArgs g{x, w, bias, dh, out, batch, a, b, c, d, act};
    if (dtype == KSMM_F32) {
        if (bs_last) return mode ? run<float, true, 1>(g, s) : run<float, true, 0>(g, s);
        return mode ? run<float, false, 1>(g, s) : run<float, false, 0>(g, s);
    }
    if (bs_last) return mode ? run<half_t, true, 1>(g, s) : run<half_t, true, 0>(g, s);
    return mode ? run<half_t, false, 1>(g, s) : run<half_t, false, 0>(g, s);
}

}  // namespace ksmm

using namespace ksmm;

namespace {

int check(int64_t batch, int a, int b, int c, int d, int dtype, int act)
{
    if (b > 0x3fffffff || batch > 0x7fffff00) return KSMM_ERR_TOO_LARGE;  // (a tile's rows past the end are counted in 32 bits)
    if (dtype != KSMM_F32 && dtype != KSMM_F16) return KSMM_ERR_BAD_DTYPE;
    const int rc = ksmm_validate(batch, a, 2 * b, c, d, dtype, dtype, dtype, 0);
    if (rc != KSMM_OK) return rc;
    return act == KSMM_ACT_NONE || act == KSMM_ACT_GELU || act == KSMM_ACT_SILU ? KSMM_OK : KSMM_ERR_BAD_EPILOGUE;
}

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

}  // namespace

extern "C" {

int ksmm_gated_forward(const void *x, const void *w, const void *bias, void *h, int64_t batch, int a, int b, int c, int d, int dtype,
                       int bs_last, int act, void *stream)
{
    const int rc = check(batch, a, b, c, d, dtype, act);
    if (rc != KSMM_OK) return rc;
    if (!x || !w || !h) return KSMM_ERR_NULL_POINTER;
    const int64_t size = (int64_t)dtype_size(dtype), xs = (int64_t)a * c * d * batch * size, ws = (int64_t)a * c * d * 2 * b * size,
                  hs = (int64_t)a * b * d * batch * size, bs = 2 * (int64_t)a * b * d * size;
    if (overlaps(h, hs, x, xs) || overlaps(h, hs, w, ws) || overlaps(h, hs, bias, bs)) return KSMM_ERR_ALIAS;
    return gated_run(x, w, bias, nullptr, h, batch, a, b, c, d, dtype, bs_last, act, 0, (hipStream_t)stream);
}

int64_t ksmm_gated_backward_workspace(int64_t batch, int a, int b, int c, int d, int dtype, int bs_last)
{
    const int rc = check(batch, a, b, c, d, dtype, KSMM_ACT_NONE);
    if (rc != KSMM_OK) return rc;
    const ksmm_factor_desc f{nullptr, a, 2 * b, c, d, dtype, 1.f};
    const int64_t layer = ksmm_layer_backward_workspace(&f, 1, batch, dtype, bs_last, KSMM_ACT_NONE);
    return layer < 0 ? layer : layer + align256(2 * (int64_t)a * b * d * batch * (int64_t)dtype_size(dtype));
}

int ksmm_gated_backward(const void *dh, const void *x, const void *w, const void *bias, void *dx, void *dw, void *dbias, void *workspace,
                        int64_t workspace_bytes, int64_t batch, int a, int b, int c, int d, int dtype, int bs_last, int act, void *stream)
{
    int rc = check(batch, a, b, c, d, dtype, act);
    if (rc != KSMM_OK) return rc;
    if (!dh || !x || !w) return KSMM_ERR_NULL_POINTER;
    const int64_t need = ksmm_gated_backward_workspace(batch, a, b, c, d, dtype, bs_last);
    if (need < 0) return (int)need;
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0) return KSMM_ERR_WORKSPACE;
    if (!dx && !dw && !dbias) return KSMM_OK;
    {
        const int64_t size = (int64_t)dtype_size(dtype), xs = (int64_t)a * c * d * batch * size, ws = (int64_t)a * c * d * 2 * b * size,
                      hs = (int64_t)a * b * d * batch * size, bs = 2 * (int64_t)a * b * d * size;
        const void *const in[] = {dh, x, w, bias}, *const out[] = {dx, dw, dbias, workspace};
        const int64_t in_bytes[] = {hs, xs, ws, bs}, out_bytes[] = {xs, ws, bs, need};
        for (int i = 0; i < 4; ++i) {
            for (int o = 0; o < 4; ++o)
                if (overlaps(in[i], in_bytes[i], out[o], out_bytes[o])) return KSMM_ERR_ALIAS;
            for (int o = 0; o < i; ++o)
                if (overlaps(out[i], out_bytes[i], out[o], out_bytes[o])) return KSMM_ERR_ALIAS;
        }
    }
    rc = gated_run(x, w, bias, dh, workspace, batch, a, b, c, d, dtype, bs_last, act, 1, (hipStream_t)stream);
    if (rc != KSMM_OK) return rc;
    const int64_t dz = align256(2 * (int64_t)a * b * d * batch * (int64_t)dtype_size(dtype));
    const ksmm_factor_desc f{w, a, 2 * b, c, d, dtype, 1.f};
    return ksmm_layer_backward(&f, 1, &x, nullptr, workspace, dx, &dw, dbias, (char *)workspace + dz, workspace_bytes - dz, batch, dtype,
                               bs_last, KSMM_ACT_NONE, stream);
}

}  // extern "C"
