// Norms around a residual connection: what follows a block, what precedes the next one, and the gated, scaled
// addition between them in one pass over the tensors.
//
//     r' = r + alpha * gate * P(x)      P(x) = x, or norm(x) * post_weight
//     n  = norm(r') * weight + bias     norm(t) = (t - mean) / sqrt(var + eps), or t / sqrt(mean(t^2) + eps)
//
// Backward, with u = norm(x) before its weight, v = norm(r') before its weight, rho the factors 1 / sqrt(..):
//     dv = dn * weight,  D = dr' + rho_r (dv - v mean(dv v) - [mean(dv)])     ([..]: with a mean only)
//     dr = D,  dgate = sum alpha D P(x),  dP = alpha gate D,  dpost = sum dP u,  dweight = sum dn v,  dbias = sum dn
//     du = dP post_weight,  dx = rho_x (du - u mean(du u) - [mean(du)])
// r' and v are computed again from x and r (the same bytes as reading r', and not rounded), the statistics (fp32,
// four a row) come from the forward pass.
//
// What bounds it: HBM; four tensors forward, six backward.  Everything is computed in fp32; a tensor's values are
// rounded once, when they are stored.  The sums over rows are fp32 partial sums that are added in a fixed order.
#include "ksmm_common.h"
#include "ksmm_norm.h"

namespace ksmm {

namespace {

constexpr int MAX_WAVES = 16;

// ---- sums over lanes ------------------------------------------------------------------------------
template <int CTRL> __device__ __forceinline__ float dpp_add(float v)
{
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// every lane of 16 gets the sum over the 16
__device__ __forceinline__ float sum16(float v)
{
    v = dpp_add<0xB1>(v);   // the other one of a pair
    v = dpp_add<0x4E>(v);   // the other pair of four
    v = dpp_add<0x141>(v);  // the other four of eight, mirrored
    return dpp_add<0x140>(v);
}
// every lane gets the sum over the wave
__device__ __forceinline__ float sum64(float v)
{
    v = sum16(v);
    auto lane = [&](int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)); };
    return (lane(0) + lane(16)) + (lane(32) + lane(48));
}

// Sums over the TPR threads of a row.  Rows wider than a wave add up through LDS, two buffers in turn: one barrier a sum.
template <int TPR> struct RowSum {
    float *red;  // 2 x 2 x MAX_WAVES floats
    int turn = 0;
    __device__ __forceinline__ void two(float &a, float &b)
    {
        if constexpr (TPR == 16) {
            a = sum16(a);
            b = sum16(b);
        } else {
            a = sum64(a);
            b = sum64(b);
            if constexpr (TPR > 64) {
                constexpr int W = TPR / 64;
                float *const at = red + turn * 2 * MAX_WAVES;
                turn ^= 1;
                if ((threadIdx.x & 63) == 0) {
                    at[threadIdx.x >> 6] = a;
                    at[MAX_WAVES + (threadIdx.x >> 6)] = b;
                }
                __syncthreads();
                a = b = 0.f;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    a += at[i];
                    b += at[MAX_WAVES + i];
                }
            }
        }
    }
    __device__ __forceinline__ float one(float a)
    {
        float b = 0.f;
        if constexpr (TPR == 16) return sum16(a);
        if constexpr (TPR == 64) return sum64(a);
        two(a, b);
        return a;
    }
};

// What a gradient dv of v = norm(t) leaves of itself: dv - v mean(dv v) - mean(dv), given the means.  (A row of one feature has
// v^2 = 1 - eps rho^2, and so have both of a row of two behind a mean: what is left is that part of dv, which the
// difference would lose.)
__device__ __forceinline__ float project(const NormArgs &a, float dv, float v, float m1, float m2, float rho)
{
    return a.features == (a.layer ? 2 : 1) ? (dv - m1) * (a.eps * rho * rho) : fmaf(-v, m2, dv) - m1;
}

// ---- E elements of a row, at element alignment; past its end: zeros, and nothing stored ------------
// (WHOLE: E divides the row, and a piece is inside or past its end as a whole)
template <typename T, int E> struct Piece {
    T e[E];
};
template <bool WHOLE, typename T, int E> __device__ __forceinline__ void load_piece(Piece<T, E> &p, const T *row, int col, int end)
{
    if (WHOLE ? col < end : col + E <= end) {
        __builtin_memcpy(&p, row + col, sizeof(p));
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) p.e[e] = !WHOLE && col + e < end ? row[col + e] : (T)0.f;
    }
}
template <bool WHOLE, typename T, int E> __device__ __forceinline__ void store_piece(T *row, int col, int end, const Piece<T, E> &p)
{
    if (WHOLE ? col < end : col + E <= end) {
        __builtin_memcpy(row + col, &p, sizeof(p));
    } else if (!WHOLE) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (col + e < end) row[col + e] = p.e[e];
    }
}
// keeps a loop's invariant pieces as they were loaded: the compiler would hold 16-bit ones converted, in twice the registers
template <typename T, int E> __device__ __forceinline__ void opaque(Piece<T, E> &p)
{
    typedef uint32_t words __attribute__((ext_vector_type(E * sizeof(T) / 4)));
    words w = __builtin_bit_cast(words, p);
    asm volatile("" : "+v"(w));
    p = __builtin_bit_cast(Piece<T, E>, w);
}

// ---- batch-size-first -------------------------------------------------------------------------------
// A row is held by TPR threads, VPL pieces of E elements each: TPR * VPL * E are enough for it.  Rows are dealt in ranges:
// the workgroup's range starts at range * range_rows.  (Threads past the end of a row hold zeros.)
template <int TPR> __device__ __forceinline__ int row_slot()
{
    const int s = threadIdx.x / TPR;
    return TPR >= 64 ? __builtin_amdgcn_readfirstlane(s) : s;  // a row's address is uniform
}

template <typename T, int E, int TPR, int VPL, bool WHOLE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void ks_norm_rows_kernel(NormArgs a, int64_t range_rows)
{
    constexpr int ROWS = TPR < 256 ? 256 / TPR : 1;
    __shared__ float red[4 * MAX_WAVES];
    RowSum<TPR> sum{red};
    const int t = threadIdx.x % TPR, H = a.features;
    const float inv = 1.f / (float)H;
    const T *x = (const T *)a.x, *res = (const T *)a.residual, *gate = (const T *)a.gate, *post = (const T *)a.post_weight;
    const int64_t first = (int64_t)blockIdx.x * range_rows, last = min(a.batch, first + range_rows);
    Piece<T, E> w[VPL], b[VPL], pw[VPL], g[VPL];
    int64_t group_end = first;  // the gate that is held is good for rows before this one
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const int col = (j * TPR + t) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) w[j].e[e] = b[j].e[e] = pw[j].e[e] = g[j].e[e] = (T)0.f;  // (not used where they are not loaded)
        if (a.n_out && a.weight) load_piece<WHOLE>(w[j], (const T *)a.weight, col, H);
        if (a.n_out && a.bias) load_piece<WHOLE>(b[j], (const T *)a.bias, col, H);
        if (x && post) load_piece<WHOLE>(pw[j], post, col, H);
    }
    // (rows of a workgroup wider than a wave add up behind barriers: all of its threads take the same ones)
    struct Operands {
        Piece<T, E> r[VPL], x[VPL];
    };
    auto fetch = [&](Operands &o, int64_t row) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const int col = (j * TPR + t) * E;
            load_piece<WHOLE>(o.r[j], res + row * H, col, H);
            if (x) load_piece<WHOLE>(o.x[j], x + row * H, col, H);
        }
    };
    Operands next;  // a row's operands are asked for while the one before is worked on
    const int64_t start = first + row_slot<TPR>();
    if (start < last) fetch(next, start);
    for (int64_t row = start; row < last; row += ROWS) {
        const Operands now = next;
        if (row + ROWS < last) fetch(next, row + ROWS);
        const auto &rp = now.r, &xp = now.x;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            opaque(w[j]);
            opaque(b[j]);
            opaque(pw[j]);
        }
        if (x && gate && row >= group_end) {
            const int64_t group = row / a.group_rows;
            group_end = (group + 1) * a.group_rows;
#pragma unroll
            for (int j = 0; j < VPL; ++j) load_piece<WHOLE>(g[j], gate + group * H, (j * TPR + t) * E, H);
        }
        float r[VPL][E];
        float mean_x = 0.f, rho_x = 1.f;
        if (x) {
            if (post) {
                if (a.layer) {
                    float s = 0.f;
#pragma unroll
                    for (int j = 0; j < VPL; ++j)
#pragma unroll
                        for (int e = 0; e < E; ++e) s += (float)xp[j].e[e];
                    mean_x = sum.one(s) * inv;
                }
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < VPL; ++j)
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float c = (j * TPR + t) * E + e < H ? (float)xp[j].e[e] - mean_x : 0.f;
                        s = fmaf(c, c, s);
                    }
                rho_x = rsqrtf(fmaf(sum.one(s), inv, a.eps));
            }
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                opaque(g[j]);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float p = (float)xp[j].e[e];
                    if (post) p = (p - mean_x) * rho_x * (float)pw[j].e[e];
                    r[j][e] = fmaf(gate ? a.alpha * (float)g[j].e[e] : a.alpha, p, (float)rp[j].e[e]);
                }
            }
            if (a.r_out) {
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    Piece<T, E> o;
#pragma unroll
                    for (int e = 0; e < E; ++e) o.e[e] = (T)r[j][e];
                    store_piece<WHOLE>((T *)a.r_out + row * H, (j * TPR + t) * E, H, o);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) r[j][e] = (float)rp[j].e[e];
        }
        float mean_r = 0.f, rho_r = 1.f;
        if (a.n_out) {
            if (a.layer) {
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < VPL; ++j)
#pragma unroll
                    for (int e = 0; e < E; ++e) s += r[j][e];  // (zeros past the end: x and r are)
                mean_r = sum.one(s) * inv;
            }
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < VPL; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float c = (j * TPR + t) * E + e < H ? r[j][e] - mean_r : 0.f;
                    s = fmaf(c, c, s);
                }
            rho_r = rsqrtf(fmaf(sum.one(s), inv, a.eps));
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                Piece<T, E> o;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float v = (r[j][e] - mean_r) * rho_r;
                    if (a.weight) v *= (float)w[j].e[e];
                    if (a.bias) v += (float)b[j].e[e];
                    o.e[e] = (T)v;
                }
                store_piece<WHOLE>((T *)a.n_out + row * H, (j * TPR + t) * E, H, o);
            }
        }
        if (a.stats && t == 0) {
            a.stats[row] = mean_x;
            a.stats[a.batch + row] = rho_x;
            a.stats[2 * a.batch + row] = mean_r;
            a.stats[3 * a.batch + row] = rho_r;
        }
    }
}

// Gradients.  Workgroup = range of rows: `parts` ranges share a gate's group, or a range is `groups_per` whole groups
// (parts == 1).  Partial sums: slice blockIdx.x of each quantity; dgate's lie [part][group][feature].  POST: x has a norm;
// MEAN: there is a bias, or a mean is taken.
// One sum serves two gradients: with S = sum D u over the rows of a gate, dgate = alpha post_weight S and, of these rows,
// dpost_weight = alpha gate S.  What a row needs twice is converted, or computed, twice: registers decide how many
// rows are on their way from memory.
template <typename T, int E, int TPR, int VPL, bool WHOLE, bool POST, bool MEAN>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void ks_norm_rows_bwd_kernel(NormArgs a, NormGrads d, NormSplit sp)
{
    constexpr int THREADS = TPR < 256 ? 256 : TPR, ROWS = TPR < 256 ? 256 / TPR : 1, WIDE = VPL * E;
    __shared__ float red[4 * MAX_WAVES];
    __shared__ float wide[ROWS > 1 ? 256 * WIDE : 1];
    __shared__ float post_sum[POST ? THREADS * WIDE : 1];  // of the groups before
    RowSum<TPR> sum{red};
    const int t = threadIdx.x % TPR, slot = row_slot<TPR>(), H = a.features;
    const float inv = 1.f / (float)H;
    const T *const x = (const T *)a.x, *const gate = (const T *)a.gate;
    const T *const dr_in = (const T *)d.dr_out, *const dn = (const T *)d.dn_out;
    Piece<T, E> w[VPL], pw[VPL], g[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const int col = (j * TPR + t) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) w[j].e[e] = pw[j].e[e] = g[j].e[e] = (T)1.f;
        if (dn && a.weight) load_piece<WHOLE>(w[j], (const T *)a.weight, col, H);
        if (POST) load_piece<WHOLE>(pw[j], (const T *)a.post_weight, col, H);
    }
    float s_w[WIDE], s_b[MEAN ? WIDE : 1], s_u[WIDE];
#pragma unroll
    for (int i = 0; i < WIDE; ++i) {
        s_w[i] = s_b[MEAN ? i : 0] = s_u[i] = 0.f;
        if (POST) post_sum[i * THREADS + threadIdx.x] = 0.f;
    }

    // the workgroup's sum of one quantity (value i of each thread), stored to a row of floats
    auto flush = [&](auto value, float *to) {
        if constexpr (ROWS > 1) {
#pragma unroll
            for (int i = 0; i < WIDE; ++i) wide[i * 256 + threadIdx.x] = value(i);
            __syncthreads();
            for (int i = threadIdx.x; i < TPR * WIDE; i += 256) {
                const int tt = i % TPR, k = i / TPR, col = (k / E * TPR + tt) * E + k % E;
                float v = 0.f;
#pragma unroll
                for (int q = 0; q < ROWS; ++q) v += wide[k * 256 + q * TPR + tt];
                if (col < H) to[col] = v;
            }
            __syncthreads();
        } else {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int col = (j * TPR + t) * E + e;
                    if (col < H) to[col] = value(j * E + e);
                }
        }
    };

    const int64_t unit = (int64_t)blockIdx.x / sp.parts;
    const int part = (int)(blockIdx.x - unit * sp.parts);
    const int64_t g_first = unit * sp.groups_per, g_last = min(sp.groups, g_first + sp.groups_per);
    for (int64_t group = g_first; group < g_last; ++group) {
        const int64_t base = group * a.group_rows, first = base + part * sp.part_rows;
        const int64_t last = min(base + a.group_rows, first + sp.part_rows);
        if (x && gate) {
#pragma unroll
            for (int j = 0; j < VPL; ++j) load_piece<WHOLE>(g[j], gate + (sp.one_gate ? 0 : group * H), (j * TPR + t) * E, H);
        }
        // a row's operands are asked for while the one before is worked on
        struct Operands {
            Piece<T, E> r[VPL], x[VPL], n[VPL], d[VPL];
            float mean_x, rho_x, mean_r, rho_r;
        };
        auto fetch = [&](Operands &o, int64_t row) {
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                const int col = (j * TPR + t) * E;
                if (x) load_piece<WHOLE>(o.x[j], x + row * H, col, H);
                if (dn) {
                    load_piece<WHOLE>(o.r[j], (const T *)a.residual + row * H, col, H);
                    load_piece<WHOLE>(o.n[j], dn + row * H, col, H);
                }
                if (dr_in) load_piece<WHOLE>(o.d[j], dr_in + row * H, col, H);
            }
            o.mean_x = a.stats[row];
            o.rho_x = a.stats[a.batch + row];
            o.mean_r = a.stats[2 * a.batch + row];
            o.rho_r = a.stats[3 * a.batch + row];
        };
        Operands next;
        if (first + slot < last) fetch(next, first + slot);
        for (int64_t row = first + slot; row < last; row += ROWS) {
            const Operands now = next;
            if (row + ROWS < last) fetch(next, row + ROWS);
            const auto &rp = now.r, &xp = now.x, &np = now.n, &dp = now.d;
            const float mean_x = now.mean_x, rho_x = now.rho_x, mean_r = now.mean_r, rho_r = now.rho_r;
            auto u_of = [&](int j, int e) { return POST ? ((float)xp[j].e[e] - mean_x) * rho_x : (float)xp[j].e[e]; };
            auto gate_of = [&](int j, int e) { return a.alpha * (float)g[j].e[e]; };  // (ones without a gate)
            float v[VPL][E], m1 = 0.f, m2 = 0.f;
            if (dn) {
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    opaque(w[j]);
                    opaque(pw[j]);
                    opaque(g[j]);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        float r = (float)rp[j].e[e];
                        if (x) r = fmaf(gate_of(j, e), POST ? u_of(j, e) * (float)pw[j].e[e] : u_of(j, e), r);
                        const float n = (float)np[j].e[e];  // (zero past the end, and so is what it multiplies)
                        v[j][e] = (r - mean_r) * rho_r;
                        const float dv = n * (float)w[j].e[e];
                        if (MEAN) m1 += dv;
                        m2 = fmaf(dv, v[j][e], m2);
                        s_w[j * E + e] = fmaf(n, v[j][e], s_w[j * E + e]);
                        if (MEAN) s_b[MEAN ? j * E + e : 0] += n;
                    }
                }
                if (MEAN)
                    sum.two(m1, m2);
                else
                    m2 = sum.one(m2);
                m1 = MEAN && a.layer ? m1 * inv : 0.f;
                m2 *= inv;
            }
            float k1 = 0.f, k2 = 0.f;
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                opaque(w[j]);
                opaque(pw[j]);
                opaque(g[j]);
                Piece<T, E> o;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float D = dr_in ? (float)dp[j].e[e] : 0.f;
                    if (dn) D = fmaf(rho_r, project(a, (float)np[j].e[e] * (float)w[j].e[e], v[j][e], m1, m2, rho_r), D);
                    o.e[e] = (T)D;
                    // (past the end D holds the rest of a mean: nothing may be added there)
                    const bool in = WHOLE ? (j * TPR + t) * E < H : (j * TPR + t) * E + e < H;
                    D = in ? D : 0.f;
                    if (x) {
                        const float u = u_of(j, e);
                        s_u[j * E + e] = fmaf(D, u, s_u[j * E + e]);
                        float q = gate_of(j, e) * D;
                        if (POST) {
                            q *= (float)pw[j].e[e];
                            if (MEAN) k1 += q;
                            k2 = fmaf(q, u, k2);
                        }
                        v[j][e] = q;
                    }
                }
                if (d.dresidual) store_piece<WHOLE>((T *)d.dresidual + row * H, (j * TPR + t) * E, H, o);
            }
            if (x && d.dx) {
                if (POST) {
                    if (MEAN)
                        sum.two(k1, k2);
                    else
                        k2 = sum.one(k2);
                    k1 = MEAN && a.layer ? k1 * inv : 0.f;
                    k2 *= inv;
                }
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    Piece<T, E> o;
#pragma unroll
                    for (int e = 0; e < E; ++e) o.e[e] = (T)(POST ? rho_x * project(a, v[j][e], u_of(j, e), k1, k2, rho_x) : v[j][e]);
                    store_piece<WHOLE>((T *)d.dx + row * H, (j * TPR + t) * E, H, o);
                }
            }
        }
        if (x) {
            if (d.dgate)
                flush([&](int i) { return a.alpha * (POST ? (float)pw[i / E].e[i % E] : 1.f) * s_u[i]; },
                      d.dgate + (sp.one_gate ? (int64_t)blockIdx.x : (int64_t)part * sp.groups + group) * H);
            if (POST) {
#pragma unroll
                for (int i = 0; i < WIDE; ++i) post_sum[i * THREADS + threadIdx.x] += a.alpha * (float)g[i / E].e[i % E] * s_u[i];
            }
#pragma unroll
            for (int i = 0; i < WIDE; ++i) s_u[i] = 0.f;
        }
    }
    if (d.dweight) flush([&](int i) { return s_w[i]; }, d.dweight + (int64_t)blockIdx.x * H);
    if (MEAN && d.dbias) flush([&](int i) { return s_b[MEAN ? i : 0]; }, d.dbias + (int64_t)blockIdx.x * H);
    if (POST && d.dpost_weight) flush([&](int i) { return post_sum[POST ? i * THREADS + threadIdx.x : 0]; }, d.dpost_weight + (int64_t)blockIdx.x * H);
}

// ---- batch-size-last --------------------------------------------------------------------------------
// A workgroup takes 4 * LANES neighbouring rows of the batch (columns of the tensors) and all features: thread = four
// columns, one vector, and every GROUPS-th feature, FPT of them at a time, as they are stored, in registers.  ONE: that is all
// of them, and they are read once; else they are read again in each pass that the statistics need.
constexpr int COL_THREADS = 512, COL_WAVES = COL_THREADS / 64;
struct Four {
    float v[4];
};
template <typename T> struct Raw {
    T v[4];
};
// each XCD gets a contiguous range of column tiles: neighbours share cache lines
__device__ __forceinline__ int col_tile(int tiles) { return (blockIdx.x & 7) * ((tiles + 7) / 8) + (blockIdx.x >> 3); }
template <typename T> __device__ __forceinline__ Four wide_of(const Raw<T> &r)
{
    return Four{{(float)r.v[0], (float)r.v[1], (float)r.v[2], (float)r.v[3]}};
}
template <typename T> __device__ __forceinline__ void opaque(Raw<T> &r)
{
    typedef uint32_t words __attribute__((ext_vector_type(sizeof(T))));
    words w = __builtin_bit_cast(words, r);
    asm volatile("" : "+v"(w));
    r = __builtin_bit_cast(Raw<T>, w);
}
// alpha * gate, post_weight, weight and bias of every feature, as far as they fit LDS: a feature's four are one read.
// (gates of groups: alpha alone)
constexpr int PARAMS = 2048;
struct Params {
    float gate, post, weight, bias;
};
template <typename T> __device__ __forceinline__ Params params_of(const NormArgs &a, bool one_gate, int h)
{
    Params p;
    p.gate = a.gate && one_gate ? a.alpha * (float)((const T *)a.gate)[h] : a.alpha;
    p.post = a.post_weight ? (float)((const T *)a.post_weight)[h] : 1.f;
    p.weight = a.weight ? (float)((const T *)a.weight)[h] : 1.f;
    p.bias = a.bias ? (float)((const T *)a.bias)[h] : 0.f;
    return p;
}
// one row's four columns; past the last column: zeros, and nothing stored
template <typename T> __device__ __forceinline__ Raw<T> load_four(const T *row, int count)
{
    Raw<T> r;
    if (count >= 4) {
        __builtin_memcpy(&r, row, sizeof(r));
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) r.v[c] = c < count ? row[c] : (T)0.f;
    }
    return r;
}
template <typename T> __device__ __forceinline__ void store_four(T *row, int count, const Four &f)
{
    if (count >= 4) {
        const Raw<T> r{{(T)f.v[0], (T)f.v[1], (T)f.v[2], (T)f.v[3]}};
        __builtin_memcpy(row, &r, sizeof(r));
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (c < count) row[c] = (T)f.v[c];
    }
}

// every thread gets the sums of its columns over all features
template <int LANES> struct ColSum {
    float *red;  // 2 x COL_WAVES x 4 * LANES floats
    __device__ __forceinline__ void add(Four &f, int q)
    {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (LANES <= 4) f.v[c] += __shfl_xor(f.v[c], 4, 64);
            if (LANES <= 8) f.v[c] = dpp_add<0x128>(f.v[c]);  // the other eight of sixteen
            f.v[c] += __shfl_xor(f.v[c], 16, 64);
            f.v[c] += __shfl_xor(f.v[c], 32, 64);
        }
        if ((threadIdx.x & 63) < LANES) *(Four *)(red + ((q * COL_WAVES + (threadIdx.x >> 6)) * LANES + threadIdx.x % LANES) * 4) = f;
    }
    __device__ __forceinline__ void get(Four &f, int q)
    {
#pragma unroll
        for (int c = 0; c < 4; ++c) f.v[c] = 0.f;
#pragma unroll
        for (int w = 0; w < COL_WAVES; ++w) {
            const Four o = *(const Four *)(red + ((q * COL_WAVES + w) * LANES + threadIdx.x % LANES) * 4);
#pragma unroll
            for (int c = 0; c < 4; ++c) f.v[c] += o.v[c];
        }
    }
    __device__ __forceinline__ void two(Four &a, Four &b)
    {
        __syncthreads();
        add(a, 0);
        add(b, 1);
        __syncthreads();
        get(a, 0);
        get(b, 1);
    }
    __device__ __forceinline__ void one(Four &a)
    {
        __syncthreads();
        add(a, 0);
        __syncthreads();
        get(a, 0);
    }
};
// the sum over the LANES lanes side by side that hold one feature
template <int LANES> __device__ __forceinline__ float sum_lanes(const Four &f)
{
    float v = (f.v[0] + f.v[1]) + (f.v[2] + f.v[3]);
    v = dpp_add<0xB1>(v);
    v = dpp_add<0x4E>(v);
    if (LANES > 4) v = dpp_add<0x141>(v);
    return LANES > 8 ? dpp_add<0x140>(v) : v;
}

template <typename T, int LANES, int FPT, bool ONE>
__global__ __launch_bounds__(COL_THREADS) void ks_norm_cols_kernel(NormArgs a, int tiles)
{
    const int tile = col_tile(tiles);
    if (tile >= tiles) return;
    constexpr int GROUPS = COL_THREADS / LANES;
    __shared__ float red[2 * COL_WAVES * 4 * LANES];
    __shared__ Params held[PARAMS];
    ColSum<LANES> sum{red};
    const int H = a.features, grp = threadIdx.x / LANES;
    const int64_t B = a.batch, col = ((int64_t)tile * LANES + threadIdx.x % LANES) * 4;
    const int count = (int)max((int64_t)0, min((int64_t)4, B - col));  // (none: the thread adds zeros)
    const float inv = 1.f / (float)H;
    const T *const x = (const T *)a.x, *const res = (const T *)a.residual;
    const bool post = a.post_weight != nullptr, one_gate = a.group_rows == B, in_lds = H <= PARAMS;
    if (in_lds) {
        for (int h = threadIdx.x; h < H; h += COL_THREADS) held[h] = params_of<T>(a, one_gate, h);
    }
    auto params = [&](int h) { return in_lds ? held[h] : params_of<T>(a, one_gate, h); };
    const bool own_gates = a.gate && !one_gate;  // each column that of its group
    const T *gate[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) gate[c] = own_gates ? (const T *)a.gate + min(col + c, B - 1) / a.group_rows * H : nullptr;
    auto factor = [&](const Params &p, int c, int h) { return own_gates ? a.alpha * (float)gate[c][h] : p.gate; };
    Raw<T> xv[FPT] = {}, rv[FPT] = {};
    auto load = [&](int first, bool with_r) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < FPT; ++i) {
            const int h = first + i * GROUPS;
            if (h < H) {
                if (with_r) rv[i] = load_four(res + h * B + col, count);
                if (x) xv[i] = load_four(x + h * B + col, count);
            }
        }
    };
    // every feature of the thread in turn, f(i, h): its values are xv[i] and (WITH_R) rv[i]
    auto each = [&](bool with_r, auto f) __attribute__((always_inline)) {
        int first = grp;
        asm volatile("" : "+v"(first));  // (addresses are made anew in each pass, not held)
        for (; first < H; first += FPT * GROUPS) {
            if (!ONE) load(first, with_r);
#pragma unroll
            for (int i = 0; i < FPT; ++i) {
                opaque(xv[i]);  // (each pass starts from the values as they are stored: kept wide they would not fit)
                opaque(rv[i]);
                if (first + i * GROUPS < H) f(i, first + i * GROUPS);
            }
            if (ONE) break;
        }
    };
    if (ONE) load(grp, true);
    __syncthreads();
    Four mean_x = {}, rho_x = {{1.f, 1.f, 1.f, 1.f}}, mean_r = {}, rho_r = {{1.f, 1.f, 1.f, 1.f}};
    if (x && post) {
        if (a.layer) {
            each(false, [&](int i, int) {
#pragma unroll
                for (int c = 0; c < 4; ++c) mean_x.v[c] += (float)xv[i].v[c];
            });
            sum.one(mean_x);
#pragma unroll
            for (int c = 0; c < 4; ++c) mean_x.v[c] *= inv;
        }
        Four s = {};
        each(false, [&](int i, int) {
#pragma unroll
            for (int c = 0; c < 4; ++c) s.v[c] = fmaf((float)xv[i].v[c] - mean_x.v[c], (float)xv[i].v[c] - mean_x.v[c], s.v[c]);
        });
        sum.one(s);
#pragma unroll
        for (int c = 0; c < 4; ++c) rho_x.v[c] = rsqrtf(fmaf(s.v[c], inv, a.eps));
    }
    auto get_r = [&](int i, int h) {  // r', from the inputs
        Four r = wide_of(rv[i]);
        if (x) {
            const Params q = params(h);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float f = (float)xv[i].v[c], p = post ? (f - mean_x.v[c]) * rho_x.v[c] * q.post : f;
                r.v[c] = fmaf(factor(q, c, h), p, r.v[c]);
            }
        }
        return r;
    };
    Four s = {};
    each(true, [&](int i, int h) {
        const Four r = get_r(i, h);
        if (x && a.r_out) store_four((T *)a.r_out + h * B + col, count, r);
#pragma unroll
        for (int c = 0; c < 4; ++c) s.v[c] += a.layer ? r.v[c] : r.v[c] * r.v[c];
    });
    if (a.n_out) {
        sum.one(s);
        if (a.layer) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                mean_r.v[c] = s.v[c] * inv;
                s.v[c] = 0.f;
            }
            each(true, [&](int i, int h) {
                const Four r = get_r(i, h);
#pragma unroll
                for (int c = 0; c < 4; ++c) s.v[c] = fmaf(r.v[c] - mean_r.v[c], r.v[c] - mean_r.v[c], s.v[c]);
            });
            sum.one(s);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) rho_r.v[c] = rsqrtf(fmaf(s.v[c], inv, a.eps));
        each(true, [&](int i, int h) {
            const Four r = get_r(i, h);
            const Params p = params(h);
            Four o;
#pragma unroll
            for (int c = 0; c < 4; ++c) o.v[c] = fmaf((r.v[c] - mean_r.v[c]) * rho_r.v[c], p.weight, p.bias);
            store_four((T *)a.n_out + h * B + col, count, o);
        });
    }
    if (a.stats && grp == 0) {
        store_four(a.stats + col, count, mean_x);
        store_four(a.stats + B + col, count, rho_x);
        store_four(a.stats + 2 * B + col, count, mean_r);
        store_four(a.stats + 3 * B + col, count, rho_r);
    }
}

// Gradients; the sums over a workgroup's columns are its slice of the partial sums.  With one gate for all rows, S = sum D u
// serves dgate and dpost_weight (see above); gates of groups have a kernel of their own.
template <typename T, int LANES, int FPT, bool ONE>
__global__ __launch_bounds__(COL_THREADS) void ks_norm_cols_bwd_kernel(NormArgs a, NormGrads d, int tiles)
{
    const int tile = col_tile(tiles);
    if (tile >= tiles) return;
    constexpr int GROUPS = COL_THREADS / LANES;
    __shared__ float red[2 * COL_WAVES * 4 * LANES];
    __shared__ Params held[PARAMS];
    ColSum<LANES> sum{red};
    const int H = a.features, grp = threadIdx.x / LANES;
    const int64_t B = a.batch, col = ((int64_t)tile * LANES + threadIdx.x % LANES) * 4;
    const int count = (int)max((int64_t)0, min((int64_t)4, B - col));  // (past the end: zeros, which no sum minds)
    const float inv = 1.f / (float)H;
    const T *const x = (const T *)a.x, *const res = (const T *)a.residual;
    const bool post = a.post_weight != nullptr, one_gate = a.group_rows == B, in_lds = H <= PARAMS;
    if (in_lds) {
        for (int h = threadIdx.x; h < H; h += COL_THREADS) held[h] = params_of<T>(a, one_gate, h);
    }
    auto params = [&](int h) { return in_lds ? held[h] : params_of<T>(a, one_gate, h); };
    const bool own_gates = a.gate && !one_gate, writes = threadIdx.x % LANES == 0;
    const T *gate[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) gate[c] = own_gates ? (const T *)a.gate + min(col + c, B - 1) / a.group_rows * H : nullptr;
    auto factor = [&](const Params &p, int c, int h) { return own_gates ? a.alpha * (float)gate[c][h] : p.gate; };
    const T *const dr_in = (const T *)d.dr_out, *const dn = (const T *)d.dn_out;
    Four mean_x = {}, rho_x = {}, mean_r = {}, rho_r = {};
    if (count > 0) {
        mean_x = wide_of(load_four(a.stats + col, count));
        rho_x = wide_of(load_four(a.stats + B + col, count));
        mean_r = wide_of(load_four(a.stats + 2 * B + col, count));
        rho_r = wide_of(load_four(a.stats + 3 * B + col, count));
    }
    Raw<T> xv[FPT] = {}, rv[FPT] = {}, nv[FPT] = {}, dv[FPT] = {};
    auto load = [&](int first, bool with_d) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < FPT; ++i) {
            const int h = first + i * GROUPS;
            if (h < H) {
                if (x) xv[i] = load_four(x + h * B + col, count);
                if (dn) {
                    rv[i] = load_four(res + h * B + col, count);
                    nv[i] = load_four(dn + h * B + col, count);
                }
                if (with_d && dr_in) dv[i] = load_four(dr_in + h * B + col, count);
            }
        }
    };
    auto each = [&](bool with_d, auto f) __attribute__((always_inline)) {
        int first = grp;
        asm volatile("" : "+v"(first));  // (addresses are made anew in each pass, not held)
        for (; first < H; first += FPT * GROUPS) {
            if (!ONE) load(first, with_d);
#pragma unroll
            for (int i = 0; i < FPT; ++i) {
                opaque(xv[i]);  // (each pass starts from the values as they are stored: kept wide they would not fit)
                opaque(rv[i]);
                opaque(nv[i]);
                opaque(dv[i]);
                if (first + i * GROUPS < H) f(i, first + i * GROUPS);
            }
            if (ONE) break;
        }
    };
    if (ONE) load(grp, true);
    __syncthreads();
    auto get_u = [&](int i) {
        Four u = {};
        if (x) {
#pragma unroll
            for (int c = 0; c < 4; ++c) u.v[c] = post ? ((float)xv[i].v[c] - mean_x.v[c]) * rho_x.v[c] : (float)xv[i].v[c];
        }
        return u;
    };
    auto get_v = [&](int i, int h, const Params &p, const Four &u) {
        Four r = wide_of(rv[i]);
#pragma unroll
        for (int c = 0; c < 4; ++c) r.v[c] = ((x ? fmaf(factor(p, c, h), u.v[c] * p.post, r.v[c]) : r.v[c]) - mean_r.v[c]) * rho_r.v[c];
        return r;
    };
    Four m1 = {}, m2 = {};
    if (dn) {
        each(false, [&](int i, int h) {
            const Params p = params(h);
            const Four v = get_v(i, h, p, get_u(i)), n = wide_of(nv[i]);
            Four nw;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                m1.v[c] = fmaf(n.v[c], p.weight, m1.v[c]);
                m2.v[c] = fmaf(n.v[c] * p.weight, v.v[c], m2.v[c]);
                nw.v[c] = n.v[c] * v.v[c];
            }
            if (d.dweight) {
                const float q = sum_lanes<LANES>(nw);
                if (writes) d.dweight[(int64_t)tile * H + h] = q;
            }
            if (d.dbias) {
                const float q = sum_lanes<LANES>(n);
                if (writes) d.dbias[(int64_t)tile * H + h] = q;
            }
        });
        if (a.layer)
            sum.two(m1, m2);
        else
            sum.one(m2);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            m1.v[c] = a.layer ? m1.v[c] * inv : 0.f;
            m2.v[c] *= inv;
        }
        if (d.means && grp == 0) {
            store_four(d.means + col, count, m1);
            store_four(d.means + B + col, count, m2);
        }
    }
    // D of one feature
    auto get_D = [&](int i, int h, const Params &p, const Four &u) {
        Four D = dr_in ? wide_of(dv[i]) : Four{};
        if (dn) {
            const Four v = get_v(i, h, p, u);
#pragma unroll
            for (int c = 0; c < 4; ++c) D.v[c] = fmaf(rho_r.v[c], project(a, (float)nv[i].v[c] * p.weight, v.v[c], m1.v[c], m2.v[c], rho_r.v[c]), D.v[c]);
        }
        return D;
    };
    Four k1 = {}, k2 = {};
    each(true, [&](int i, int h) {
        const Params p = params(h);
        const Four u = get_u(i), D = get_D(i, h, p, u);
        if (d.dresidual) store_four((T *)d.dresidual + h * B + col, count, D);
        if (!x) return;
        Four q, s;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            q.v[c] = factor(p, c, h) * D.v[c];
            s.v[c] = (one_gate ? D.v[c] : q.v[c]) * u.v[c];
            if (post) {
                q.v[c] *= p.post;
                k1.v[c] += q.v[c];
                k2.v[c] = fmaf(q.v[c], u.v[c], k2.v[c]);
            }
        }
        if (d.dgate || d.dpost_weight) {
            const float S = sum_lanes<LANES>(s);
            if (writes && d.dgate) d.dgate[(int64_t)tile * H + h] = a.alpha * p.post * S;
            if (writes && d.dpost_weight) d.dpost_weight[(int64_t)tile * H + h] = one_gate ? p.gate * S : S;
        }
        if (!post && d.dx) store_four((T *)d.dx + h * B + col, count, q);
    });
    if (x && post && d.dx) {
        if (a.layer)
            sum.two(k1, k2);
        else
            sum.one(k2);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            k1.v[c] = a.layer ? k1.v[c] * inv : 0.f;
            k2.v[c] *= inv;
        }
        each(true, [&](int i, int h) {
            const Params p = params(h);
            const Four u = get_u(i);
            Four q = get_D(i, h, p, u);
#pragma unroll
            for (int c = 0; c < 4; ++c) q.v[c] = rho_x.v[c] * project(a, q.v[c] * factor(p, c, h) * p.post, u.v[c], k1.v[c], k2.v[c], rho_x.v[c]);
            store_four((T *)d.dx + h * B + col, count, q);
        });
    }
}

// The same in steps, for many features of few columns: a launch a step, a workgroup takes 64 columns x CHUNK features, and leaves its part of the sums over features to the
// next step.  (A step reads its operands again: what it needs of r', v and D is computed anew, unrounded.)
//   forward   X_STATS  statistics of x       MID  r', its statistics     OUT  n
//   backward  SUMS     sums over dn          RES  dr, sums over it       DX   dx
// Statistics: mean and sum of squared differences of a chunk, both taken from values in registers, put together by
// the formula for two sets, n1 n2 / (n1 + n2) (mean1 - mean2)^2.
enum { X_STATS, MID, OUT, SUMS, RES, DX };
constexpr int STEP_LANES = 16, STEP_COLS = 4 * STEP_LANES, STEP_FPT = 4, CHUNK = COL_THREADS / STEP_LANES * STEP_FPT;
struct StepSpace {
    float *x, *r, *m, *k;  // [chunk][2][batch] each
    int tiles, chunks;
};

template <typename T, int STEP>
__global__ __launch_bounds__(COL_THREADS, 4) void ks_norm_step_kernel(NormArgs a, NormGrads d, StepSpace sp)
{
    constexpr int LANES = STEP_LANES, GROUPS = COL_THREADS / LANES, FPT = STEP_FPT;
    constexpr bool FORWARD = STEP <= OUT;
    __shared__ float red[2 * COL_WAVES * 4 * LANES];
    __shared__ Params held[CHUNK];
    __shared__ float known[6][STEP_COLS];  // of a column: mean and factor of x's norm, of r's; sums
    ColSum<LANES> sum{red};
    const int blocks = sp.tiles * sp.chunks, per_xcd = (blocks + 7) / 8, lid = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per_xcd || lid >= blocks) return;
    const int tile = lid % sp.tiles, chunk = lid / sp.tiles, H = a.features, h0 = chunk * CHUNK, h_end = min(H, h0 + CHUNK);
    const int grp = threadIdx.x / LANES, lane4 = threadIdx.x % LANES * 4;
    const int64_t B = a.batch, col0 = (int64_t)tile * STEP_COLS, col = col0 + lane4;
    const int count = (int)max((int64_t)0, min((int64_t)4, B - col));  // (none: the thread adds zeros)
    const float inv = 1.f / (float)H;
    const T *const x = (const T *)a.x, *const res = (const T *)a.residual, *const dn = (const T *)d.dn_out, *const dr_in = (const T *)d.dr_out;
    const bool post = a.post_weight != nullptr, one_gate = a.group_rows == B, own_gates = a.gate && !one_gate;
    // operands
    Raw<T> xv[FPT] = {}, rv[FPT] = {}, nv[FPT] = {}, dv[FPT] = {};
#pragma unroll
    for (int i = 0; i < FPT; ++i) {
        const int h = h0 + grp + i * GROUPS;
        if (h < h_end) {
            if (x) xv[i] = load_four(x + h * B + col, count);
            if (STEP != X_STATS && (FORWARD || dn)) rv[i] = load_four(res + h * B + col, count);
            if (!FORWARD && dn) nv[i] = load_four(dn + h * B + col, count);
            if ((STEP == RES || STEP == DX) && dr_in) dv[i] = load_four(dr_in + h * B + col, count);
        }
    }
    for (int h = threadIdx.x; h < h_end - h0; h += COL_THREADS) held[h] = params_of<T>(a, one_gate, h0 + h);
    // what the steps before left
    if (threadIdx.x < STEP_COLS && col0 + threadIdx.x < B) {
        const int64_t c = col0 + threadIdx.x;
        auto statistics = [&](const float *part, int to) {
            float n = 0.f, mean = 0.f, m2 = 0.f;
            for (int k = 0; k < sp.chunks; ++k) {
                const float nk = (float)(min(H, (k + 1) * CHUNK) - k * CHUNK), mk = part[(2 * k) * B + c], sk = part[(2 * k + 1) * B + c];
                const float diff = mk - mean, both = n + nk;
                mean = fmaf(diff, nk / both, mean);
                m2 += sk + diff * diff * (n * nk / both);
                n = both;
            }
            known[to][threadIdx.x] = mean;  // (0 without a mean: the chunks' are)
            known[to + 1][threadIdx.x] = rsqrtf(fmaf(m2, inv, a.eps));
        };
        auto total = [&](const float *part, int to) {
            float s1 = 0.f, s2 = 0.f;
            for (int k = 0; k < sp.chunks; ++k) {
                s1 += part[(2 * k) * B + c];
                s2 += part[(2 * k + 1) * B + c];
            }
            known[to][threadIdx.x] = a.layer ? s1 * inv : 0.f;
            known[to + 1][threadIdx.x] = s2 * inv;
        };
        known[0][threadIdx.x] = known[2][threadIdx.x] = 0.f;
        known[1][threadIdx.x] = known[3][threadIdx.x] = 1.f;
        if (FORWARD) {
            if (STEP != X_STATS && x && post) statistics(sp.x, 0);
            if (STEP == OUT) statistics(sp.r, 2);
            if (STEP == (a.n_out ? OUT : MID) && a.stats && chunk == 0) {
                for (int q = 0; q < 4; ++q) a.stats[q * B + c] = known[q][threadIdx.x];
            }
        } else {
            for (int q = 0; q < 4; ++q) known[q][threadIdx.x] = a.stats[q * B + c];
            if (STEP != SUMS && dn) {
                total(sp.m, 4);
                if (STEP == RES && d.means && chunk == 0) {
                    d.means[c] = known[4][threadIdx.x];
                    d.means[B + c] = known[5][threadIdx.x];
                }
            }
        }
    }
    __syncthreads();
    Four mean_x, rho_x, mean_r, rho_r, m1 = {}, m2 = {};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const bool in = c < count;
        mean_x.v[c] = in ? known[0][lane4 + c] : 0.f;
        rho_x.v[c] = in ? known[1][lane4 + c] : 0.f;
        mean_r.v[c] = in ? known[2][lane4 + c] : 0.f;
        rho_r.v[c] = in ? known[3][lane4 + c] : 0.f;
        if (!FORWARD && STEP != SUMS && dn) {
            m1.v[c] = in ? known[4][lane4 + c] : 0.f;
            m2.v[c] = in ? known[5][lane4 + c] : 0.f;
        }
    }
    const T *gate[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) gate[c] = own_gates ? (const T *)a.gate + min(col + c, B - 1) / a.group_rows * H : nullptr;
    auto factor = [&](const Params &p, int c, int h) { return own_gates ? a.alpha * (float)gate[c][h] : p.gate; };
    auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < FPT; ++i) {
            const int h = h0 + grp + i * GROUPS;
            opaque(xv[i]);
            opaque(rv[i]);
            if (h < h_end) f(i, h, held[h - h0]);
        }
    };
    auto get_u = [&](int i) {
        Four u = {};
        if (x) {
#pragma unroll
            for (int c = 0; c < 4; ++c) u.v[c] = post ? ((float)xv[i].v[c] - mean_x.v[c]) * rho_x.v[c] : (float)xv[i].v[c];
        }
        return u;
    };
    auto get_r = [&](int i, int h, const Params &p, const Four &u) {
        Four r = wide_of(rv[i]);
        if (x) {
#pragma unroll
            for (int c = 0; c < 4; ++c) r.v[c] = fmaf(factor(p, c, h), u.v[c] * p.post, r.v[c]);
        }
        return r;
    };
    // this chunk's statistics of value(i, h, p)
    auto leave_statistics = [&](auto value, float *part) {
        Four mean = {}, s = {};
        if (a.layer) {
            each([&](int i, int h, const Params &p) {
                const Four v = value(i, h, p);
#pragma unroll
                for (int c = 0; c < 4; ++c) mean.v[c] += v.v[c];
            });
            sum.one(mean);
#pragma unroll
            for (int c = 0; c < 4; ++c) mean.v[c] /= (float)(h_end - h0);
        }
        each([&](int i, int h, const Params &p) {
            const Four v = value(i, h, p);
#pragma unroll
            for (int c = 0; c < 4; ++c) s.v[c] = fmaf(v.v[c] - mean.v[c], v.v[c] - mean.v[c], s.v[c]);
        });
        sum.one(s);
        if (grp == 0) {
            store_four(part + (int64_t)(2 * chunk) * B + col, count, mean);
            store_four(part + (int64_t)(2 * chunk + 1) * B + col, count, s);
        }
    };
    auto leave_sums = [&](Four &s1, Four &s2, float *part) {
        sum.two(s1, s2);
        if (grp == 0) {
            store_four(part + (int64_t)(2 * chunk) * B + col, count, s1);
            store_four(part + (int64_t)(2 * chunk + 1) * B + col, count, s2);
        }
    };
    const bool writes = threadIdx.x % LANES == 0;
    if constexpr (STEP == X_STATS) {
        leave_statistics([&](int i, int, const Params &) { return wide_of(xv[i]); }, sp.x);
    } else if constexpr (STEP == MID) {
        if (x)
            each([&](int i, int h, const Params &p) { store_four((T *)a.r_out + h * B + col, count, get_r(i, h, p, get_u(i))); });
        if (a.n_out) leave_statistics([&](int i, int h, const Params &p) { return get_r(i, h, p, get_u(i)); }, sp.r);
    } else if constexpr (STEP == OUT) {
        each([&](int i, int h, const Params &p) {
            Four o = get_r(i, h, p, get_u(i));
#pragma unroll
            for (int c = 0; c < 4; ++c) o.v[c] = fmaf((o.v[c] - mean_r.v[c]) * rho_r.v[c], p.weight, p.bias);
            store_four((T *)a.n_out + h * B + col, count, o);
        });
    } else if constexpr (STEP == SUMS) {
        Four s1 = {}, s2 = {};
        each([&](int i, int h, const Params &p) {
            Four v = get_r(i, h, p, get_u(i));
            const Four n = wide_of(nv[i]);
            Four nw;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                v.v[c] = (v.v[c] - mean_r.v[c]) * rho_r.v[c];
                nw.v[c] = n.v[c] * v.v[c];
                s1.v[c] = fmaf(n.v[c], p.weight, s1.v[c]);
                s2.v[c] = fmaf(n.v[c] * p.weight, v.v[c], s2.v[c]);
            }
            if (d.dweight) {
                const float q = sum_lanes<LANES>(nw);
                if (writes) d.dweight[(int64_t)tile * H + h] = q;
            }
            if (d.dbias) {
                const float q = sum_lanes<LANES>(n);
                if (writes) d.dbias[(int64_t)tile * H + h] = q;
            }
        });
        leave_sums(s1, s2, sp.m);
    } else {
        auto get_D = [&](int i, int h, const Params &p, const Four &u) {
            Four D = wide_of(dv[i]);
            if (dn) {
                const Four r = get_r(i, h, p, u);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float v = (r.v[c] - mean_r.v[c]) * rho_r.v[c];
                    D.v[c] = fmaf(rho_r.v[c], project(a, (float)nv[i].v[c] * p.weight, v, m1.v[c], m2.v[c], rho_r.v[c]), D.v[c]);
                }
            }
            return D;
        };
        if constexpr (STEP == RES) {
            Four k1 = {}, k2 = {};
            each([&](int i, int h, const Params &p) {
                const Four u = get_u(i), D = get_D(i, h, p, u);
                if (d.dresidual) store_four((T *)d.dresidual + h * B + col, count, D);
                if (!x) return;
                Four q, s;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    q.v[c] = factor(p, c, h) * D.v[c];
                    s.v[c] = (one_gate ? D.v[c] : q.v[c]) * u.v[c];
                    if (post) {
                        q.v[c] *= p.post;
                        k1.v[c] += q.v[c];
                        k2.v[c] = fmaf(q.v[c], u.v[c], k2.v[c]);
                    }
                }
                if (d.dgate || d.dpost_weight) {
                    const float S = sum_lanes<LANES>(s);
                    if (writes && d.dgate) d.dgate[(int64_t)tile * H + h] = a.alpha * p.post * S;
                    if (writes && d.dpost_weight) d.dpost_weight[(int64_t)tile * H + h] = one_gate ? p.gate * S : S;
                }
                if (!post && d.dx) store_four((T *)d.dx + h * B + col, count, q);
            });
            if (x && post && d.dx) leave_sums(k1, k2, sp.k);
        } else {
            // (x has a norm and its gradient is wanted)
            __syncthreads();
            if (threadIdx.x < STEP_COLS && col0 + threadIdx.x < B) {
                float s1 = 0.f, s2 = 0.f;
                for (int k = 0; k < sp.chunks; ++k) {
                    s1 += sp.k[(int64_t)(2 * k) * B + col0 + threadIdx.x];
                    s2 += sp.k[(int64_t)(2 * k + 1) * B + col0 + threadIdx.x];
                }
                known[4][threadIdx.x] = a.layer ? s1 * inv : 0.f;
                known[5][threadIdx.x] = s2 * inv;
            }
            __syncthreads();
            each([&](int i, int h, const Params &p) {
                const Four u = get_u(i);
                Four q = get_D(i, h, p, u);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float k1 = c < count ? known[4][lane4 + c] : 0.f, k2 = c < count ? known[5][lane4 + c] : 0.f;
                    q.v[c] = rho_x.v[c] * project(a, q.v[c] * factor(p, c, h) * p.post, u.v[c], k1, k2, rho_x.v[c]);
                }
                store_four((T *)d.dx + h * B + col, count, q);
            });
        }
    }
}

// Gradients of gates that belong to groups of columns: a wave sums four features over a group.  D is computed again, from
// the statistics and the two means that the kernels before left (dr as fp16 stores it is rounded, and may have left the
// type); a column's six floats serve the four features.  dr in fp32, where it is wanted, is D, and is read: a training pass of
// 768 x 25088 with 128 groups, with both norms / one, 434 / 374 us for 492 / 436 (fp16 436 / 387; 423 / 366 from rounded values).
constexpr int GATE_FEATURES = 4;
template <typename T> __global__ __launch_bounds__(256) void ks_norm_cols_gate_kernel(NormArgs a, NormGrads d, T *__restrict__ dgate, int64_t groups)
{
    const int units = (a.features + GATE_FEATURES - 1) / GATE_FEATURES;
    const int64_t wave = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), B = a.batch;
    const int64_t group = wave / units;
    if (group >= groups) return;
    const int h0 = (int)(wave - group * units) * GATE_FEATURES, last = a.features - 1, lane = threadIdx.x & 63;
    const bool known = sizeof(T) == 4 && d.dresidual;
    const T *const x = (const T *)a.x, *const res = (const T *)a.residual, *const dr = known ? (const T *)d.dresidual : (const T *)d.dr_out;
    const T *const dn = known ? nullptr : (const T *)d.dn_out;
    float gate[GATE_FEATURES], post[GATE_FEATURES], weight[GATE_FEATURES], s[GATE_FEATURES];
    int64_t row[GATE_FEATURES];  // (past the last feature: the last one again, not stored)
#pragma unroll
    for (int i = 0; i < GATE_FEATURES; ++i) {
        const int h = min(h0 + i, last);
        gate[i] = a.alpha * (float)((const T *)a.gate)[group * a.features + h];
        post[i] = a.post_weight ? (float)((const T *)a.post_weight)[h] : 1.f;
        weight[i] = a.weight ? (float)((const T *)a.weight)[h] : 1.f;
        row[i] = h * B;
        s[i] = 0.f;
    }
    for (int64_t c = group * a.group_rows + lane; c < (group + 1) * a.group_rows; c += 64) {
        const float mean_x = a.stats[c], rho_x = a.stats[B + c], mean_r = a.stats[2 * B + c], rho_r = a.stats[3 * B + c];
        const float m1 = dn ? d.means[c] : 0.f, m2 = dn ? d.means[B + c] : 0.f;
#pragma unroll
        for (int i = 0; i < GATE_FEATURES; ++i) {
            float p = (float)x[row[i] + c], D = dr ? (float)dr[row[i] + c] : 0.f;
            if (a.post_weight) p = (p - mean_x) * rho_x * post[i];
            if (dn) {
                const float v = (fmaf(gate[i], p, (float)res[row[i] + c]) - mean_r) * rho_r;
                D = fmaf(rho_r, project(a, (float)dn[row[i] + c] * weight[i], v, m1, m2, rho_r), D);
            }
            s[i] = fmaf(D, p, s[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < GATE_FEATURES; ++i) {
        s[i] = sum64(s[i]);
        if (lane == 0 && h0 + i <= last) dgate[group * a.features + h0 + i] = (T)(a.alpha * s[i]);
    }
}

// Gradients of the last norm's parameters where there is none of its result.
template <typename T> __global__ __launch_bounds__(256) void ks_norm_clear_kernel(T *__restrict__ dweight, T *__restrict__ dbias, int features)
{
    const int h = blockIdx.x * 256 + threadIdx.x;
    if (h >= features) return;
    if (dweight) dweight[h] = (T)0.f;
    if (dbias) dbias[h] = (T)0.f;
}

// ---- choices ------------------------------------------------------------------------------------------
// ranges of rows that fill the chip: workgroups of 4 waves, 2 of which fit a CU in the backward pass
constexpr int64_t FWD_RANGES = 2048, BWD_RANGES = 768;
// widest batch-size-first row that the kernels hold
constexpr int64_t WIDEST = 16384;

template <int E, int TPR, int VPL> struct Rows {
    static constexpr int e = E, tpr = TPR, vpl = VPL;
};
// The kernel that holds a row in the fewest values a thread (8 to 16): fp16 768 features in 12 a lane, 3 pieces of 8 bytes,
// are 54 us backward with both norms, in 2 pieces of 16 bytes, a third of them empty, 152.  Rates, forward/backward with both
// norms, TB/s: 768 x 25088 in fp16 4.2/3.7, 4096 x 8192 5.0/3.5, 8192 x 4096 3.5/3.3.  1024 threads have 128 registers each: the
// backward pass spills 37 to 70 of them a thread in fp32 above 4096 features, and 15 to 33 in fp16 there where 8 does not divide the row; above
// 8192 both passes do (16384 x 2048 3.7/1.5, in fp32 1.7/0.7): such rows are served, not tuned.
template <typename T, typename F> int with_rows(int64_t features, F f)
{
    constexpr int E = 16 / (int)sizeof(T);
    if constexpr (sizeof(T) == 2) {
        if (features <= 128) return f(Rows<E, 16, 1>());
        if (features <= 512) return f(Rows<E, 64, 1>());
        if (features <= 768) return f(Rows<4, 64, 3>());
        if (features <= 1024) return f(Rows<E, 64, 2>());
        if (features <= 2048) return f(Rows<E, 256, 1>());
        if (features <= 4096) return f(Rows<E, 256, 2>());
        if (features <= 8192) return f(Rows<E, 1024, 1>());
        if (features <= 16384) return f(Rows<E, 1024, 2>());
    } else {
        if (features <= 64) return f(Rows<E, 16, 1>());
        if (features <= 256) return f(Rows<E, 64, 1>());
        if (features <= 512) return f(Rows<E, 64, 2>());
        if (features <= 768) return f(Rows<E, 64, 3>());
        if (features <= 1024) return f(Rows<E, 256, 1>());
        if (features <= 2048) return f(Rows<E, 256, 2>());
        if (features <= 4096) return f(Rows<E, 1024, 1>());
        if (features <= 8192) return f(Rows<E, 1024, 2>());
        if (features <= 16384) return f(Rows<E, 1024, 4>());
    }
    return KSMM_ERR_TOO_LARGE;
}

// features a thread holds: 12 in 16 bits and 6 in 32 are what the backward pass has registers for (with 24 and 12 it
// spills, and takes twice the time)
template <typename T> constexpr int MOST = sizeof(T) == 2 ? 12 : 6;
// Lanes side by side (four columns each) of a workgroup: 8, or 4 where 8 would leave CUs without work (768 x 4000 in fp16
// forward 17.8 us for 22.5, backward 31 for 48), and where with 4 a thread holds the features that it would
// not hold, or holds half: backward from 64 * MOST / 2 features on (8 -> 4 lanes, us: 768 x 25088 in fp16 219 -> 162, 384 x 25088 in fp32
// 102 -> 90, but 192 x 25088 in fp16 46 -> 64), forward in fp32 above 64 * MOST (768 x 25088 112 -> 92, but 384 44 -> 49,
// in fp16 1500 x 8000 75 -> 80).
template <typename T> int col_lanes(int64_t batch, int64_t features, bool backward)
{
    if (batch < 32 * 192) return 4;
    const int64_t from = backward ? 32 * MOST<T> : sizeof(T) == 4 ? 64 * MOST<T> : INT64_MAX;
    return features > from && features <= 128 * MOST<T> ? 4 : 8;
}
template <typename T, typename F> int with_cols(int64_t batch, int64_t features, bool backward, F f)
{
    const int lanes = col_lanes<T>(batch, features, backward);
    const int64_t groups = COL_THREADS / lanes, per = (features + groups - 1) / groups;
    auto held = [&](auto lanes_of) {
        typedef std::integral_constant<bool, true> one;
        if (per <= MOST<T> / 2) return f(lanes_of, std::integral_constant<int, MOST<T> / 2>(), one());
        if (per <= MOST<T>) return f(lanes_of, std::integral_constant<int, MOST<T>>(), one());
        return f(lanes_of, std::integral_constant<int, MOST<T> / 2>(), std::integral_constant<bool, false>());
    };
    return lanes == 8 ? held(std::integral_constant<int, 8>()) : held(std::integral_constant<int, 4>());
}

NormSplit split_rows(int64_t batch, int64_t groups)
{
    NormSplit s;
    s.one_gate = groups <= 1;
    s.groups = groups < 1 ? 1 : groups;
    const int64_t rows = batch / s.groups;
    s.parts = (int)std::max<int64_t>(1, std::min<int64_t>(BWD_RANGES / s.groups, (rows + 7) / 8));
    s.part_rows = (rows + s.parts - 1) / s.parts;
    s.parts = (int)((rows + s.part_rows - 1) / s.part_rows);
    s.groups_per = s.parts > 1 ? 1 : (s.groups + BWD_RANGES - 1) / BWD_RANGES;
    s.ranges = (s.groups + s.groups_per - 1) / s.groups_per * s.parts;
    return s;
}

int launched() { return hipGetLastError() == hipSuccess ? KSMM_OK : KSMM_ERR_LAUNCH; }

// Batch-size-last in steps where features are many and columns few: tiles of columns alone then leave most of the chip
// idle.  Forward/backward, us in one launch -> in steps: 1500 x 500 in fp32 23/52 -> 21/33, 8000 x 500 in fp16 227/457 ->
// 60/92.  Fewer features, or more columns, are served better by the single launch, which reads its operands once: 768 x 500
// in fp16 12/27 (steps 20/35), 8000 x 2500 in fp32 222/481 (324/512), 2000 x 4000 49/98 (78/124).
bool in_steps(int64_t batch, int64_t features) { return features > 1024 && batch <= 2048; }
struct Steps {
    int tiles, chunks;
    int64_t part;  // floats of one array of partial sums
};
Steps steps_of(int64_t batch, int64_t features)
{
    Steps s;
    s.tiles = (int)((batch + STEP_COLS - 1) / STEP_COLS);
    s.chunks = (int)((features + CHUNK - 1) / CHUNK);
    s.part = 2 * (int64_t)s.chunks * batch;
    return s;
}
template <typename T, int STEP> void run_step(const NormArgs &a, const NormGrads &d, const StepSpace &sp, hipStream_t stream)
{
    const int64_t blocks = (int64_t)sp.tiles * sp.chunks;
    hipLaunchKernelGGL((ks_norm_step_kernel<T, STEP>), dim3((unsigned)((blocks + 7) / 8 * 8)), dim3(COL_THREADS), 0, stream, a, d, sp);
}

template <typename T> int forward(const NormArgs &a, int bs_last, float *ws, hipStream_t stream)
{
    if (bs_last && in_steps(a.batch, a.features)) {
        const Steps st = steps_of(a.batch, a.features);
        const StepSpace sp{ws, ws + st.part, nullptr, nullptr, st.tiles, st.chunks};
        const NormGrads none{};
        if (a.x && a.post_weight) run_step<T, X_STATS>(a, none, sp, stream);
        run_step<T, MID>(a, none, sp, stream);
        if (a.n_out) run_step<T, OUT>(a, none, sp, stream);
        return launched();
    }
    if (bs_last)
        return with_cols<T>(a.batch, a.features, false, [&](auto lanes, auto fpt, auto one) {
            constexpr int LANES = decltype(lanes)::value;
            const int tiles = (int)((a.batch + 4 * LANES - 1) / (4 * LANES));
            if (tiles > THREADS_MOST / COL_THREADS - 8) return (int)KSMM_ERR_TOO_LARGE;
            hipLaunchKernelGGL((ks_norm_cols_kernel<T, LANES, decltype(fpt)::value, decltype(one)::value>), dim3((tiles + 7) / 8 * 8),
                               dim3(COL_THREADS), 0, stream, a, tiles);
            return launched();
        });
    return with_rows<T>(a.features, [&](auto how) {
        typedef decltype(how) R;
        constexpr int TPR = R::tpr, ROWS = TPR < 256 ? 256 / TPR : 1;
        const int64_t steps = (a.batch + ROWS - 1) / ROWS, per = (steps + FWD_RANGES - 1) / FWD_RANGES * ROWS;
        const auto fn = a.features % R::e ? &ks_norm_rows_kernel<T, R::e, TPR, R::vpl, false> : &ks_norm_rows_kernel<T, R::e, TPR, R::vpl, true>;
        hipLaunchKernelGGL(fn, dim3((unsigned)((a.batch + per - 1) / per)),
                           dim3(TPR < 256 ? 256 : TPR), 0, stream, a, per);
        return launched();
    });
}

template <typename T> int backward(const NormArgs &a, const NormGrads &partial, const NormSplit &sp, int bs_last, float *ws, hipStream_t stream)
{
    if (bs_last && in_steps(a.batch, a.features)) {
        const Steps st = steps_of(a.batch, a.features);
        const StepSpace space{nullptr, nullptr, ws, ws + st.part, st.tiles, st.chunks};
        if (partial.dn_out) run_step<T, SUMS>(a, partial, space, stream);
        if (partial.dresidual || a.x) run_step<T, RES>(a, partial, space, stream);
        if (a.x && a.post_weight && partial.dx) run_step<T, DX>(a, partial, space, stream);
        return launched();
    }
    if (bs_last)
        return with_cols<T>(a.batch, a.features, true, [&](auto lanes, auto fpt, auto one) {
            constexpr int LANES = decltype(lanes)::value;
            const int tiles = (int)((a.batch + 4 * LANES - 1) / (4 * LANES));
            if (tiles > THREADS_MOST / COL_THREADS - 8) return (int)KSMM_ERR_TOO_LARGE;
            hipLaunchKernelGGL((ks_norm_cols_bwd_kernel<T, LANES, decltype(fpt)::value, decltype(one)::value>), dim3((tiles + 7) / 8 * 8),
                               dim3(COL_THREADS), 0, stream, a, partial, tiles);
            return launched();
        });
    return with_rows<T>(a.features, [&](auto how) {
        typedef decltype(how) R;
        const bool post = a.post_weight != nullptr, mean = a.layer || partial.dbias;
        constexpr int E = R::e, TPR = R::tpr, VPL = R::vpl;
        auto fn = &ks_norm_rows_bwd_kernel<T, E, TPR, VPL, false, true, true>;
        if (a.features % E) {
            if (!post) fn = &ks_norm_rows_bwd_kernel<T, E, TPR, VPL, false, false, true>;
        } else if (mean) {
            fn = post ? &ks_norm_rows_bwd_kernel<T, E, TPR, VPL, true, true, true> : &ks_norm_rows_bwd_kernel<T, E, TPR, VPL, true, false, true>;
        } else {
            fn = post ? &ks_norm_rows_bwd_kernel<T, E, TPR, VPL, true, true, false> : &ks_norm_rows_bwd_kernel<T, E, TPR, VPL, true, false, false>;
        }
        hipLaunchKernelGGL(fn, dim3((unsigned)sp.ranges), dim3(R::tpr < 256 ? 256 : R::tpr), 0, stream, a, partial, sp);
        return launched();
    });
}

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

// where the partial sums of each quantity lie
struct Layout {
    int64_t slices, slice_bytes, gate_bytes, steps, means, total;
    NormSplit split;
};
Layout layout(int64_t batch, int64_t features, int64_t groups, int dtype, int bs_last)
{
    Layout l;
    l.split = split_rows(batch, groups);
    const bool steps = bs_last && in_steps(batch, features);
    const int cols = steps ? STEP_COLS : 4 * (dtype == KSMM_F32 ? col_lanes<float>(batch, features, true) : col_lanes<half_t>(batch, features, true));
    l.slices = bs_last ? (batch + cols - 1) / cols : l.split.ranges;
    l.slice_bytes = align256(4 * l.slices * features);
    l.gate_bytes = l.split.one_gate ? l.slice_bytes : bs_last ? 0 : align256(4 * l.split.parts * l.split.groups * features);
    l.steps = 3 * l.slice_bytes + l.gate_bytes;
    l.means = l.steps + (steps ? align256(8 * steps_of(batch, features).part) : 0);
    l.total = l.means + (bs_last && !l.split.one_gate ? 8 * batch : 0);
    return l;
}

int check(const ksmm_norm_desc *d, int64_t batch, int64_t features, int dtype, int bs_last)
{
    if (!d) return KSMM_ERR_NULL_POINTER;
    if (batch < 1 || features < 1 || d->groups < 1 || batch % d->groups) return KSMM_ERR_BAD_BATCH;
    if (dtype != KSMM_F32 && dtype != KSMM_F16) return KSMM_ERR_BAD_DTYPE;
    if (d->kind != KSMM_NORM_RMS && d->kind != KSMM_NORM_LAYER) return KSMM_ERR_BAD_EPILOGUE;
    if (!d->residual) return KSMM_ERR_NULL_POINTER;
    if (features > (bs_last ? 0x7fffffffLL / 64 : WIDEST)) return KSMM_ERR_TOO_LARGE;
    if (batch > (1LL << 31) || batch * features > (1LL << 40)) return KSMM_ERR_TOO_LARGE;
    return KSMM_OK;
}

NormArgs args_of(const ksmm_norm_desc *d, int64_t batch, int64_t features)
{
    NormArgs a;
    a.x = d->x;
    a.residual = d->residual;
    a.gate = d->x ? d->gate : nullptr;
    a.post_weight = d->x ? d->post_weight : nullptr;
    a.weight = d->weight;
    a.bias = d->bias;
    a.alpha = d->alpha;
    a.eps = d->eps;
    a.layer = d->kind == KSMM_NORM_LAYER;
    a.batch = batch;
    a.features = (int)features;
    a.group_rows = batch / d->groups;
    return a;
}

// what a call reads, but for statistics and gradients
struct Operands {
    Span of[6];
};
Operands operands_of(const NormArgs &a, int64_t groups, int dtype)
{
    const int64_t vector = a.features * (int64_t)dtype_size(dtype), rows = a.batch * vector;
    return Operands{{{a.x, rows}, {a.residual, rows}, {a.gate, groups * vector}, {a.post_weight, vector}, {a.weight, vector}, {a.bias, vector}}};
}

}  // namespace

}  // namespace ksmm

using namespace ksmm;

extern "C" {

int64_t ksmm_residual_norm_forward_workspace(int64_t batch, int64_t features, int dtype, int bs_last)
{
    if (batch < 1 || features < 1) return KSMM_ERR_BAD_BATCH;
    if (dtype != KSMM_F32 && dtype != KSMM_F16) return KSMM_ERR_BAD_DTYPE;
    return bs_last && in_steps(batch, features) ? 8 * steps_of(batch, features).part : 0;
}

int ksmm_residual_norm_forward(const ksmm_norm_desc *desc, void *r_out, void *n_out, float *stats, void *workspace, int64_t workspace_bytes,
                               int64_t batch, int64_t features, int dtype, int bs_last, void *stream)
{
    const int rc = check(desc, batch, features, dtype, bs_last);
    if (rc != KSMM_OK) return rc;
    if ((desc->x && !r_out) || (!desc->x && !n_out)) return KSMM_ERR_NULL_POINTER;
    const int64_t need = ksmm_residual_norm_forward_workspace(batch, features, dtype, bs_last);
    if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0)) return KSMM_ERR_WORKSPACE;
    NormArgs a = args_of(desc, batch, features);
    const int64_t size = batch * features * (int64_t)dtype_size(dtype);
    const Span written[] = {{desc->x ? r_out : nullptr, size}, {n_out, size}, {stats, 16 * batch}, {need ? workspace : nullptr, need}};
    if (any_overlap(operands_of(a, desc->groups, dtype).of, written)) return KSMM_ERR_ALIAS;
    a.r_out = desc->x ? r_out : nullptr;
    a.n_out = n_out;
    a.stats = stats;
    return dtype == KSMM_F32 ? forward<float>(a, bs_last, (float *)workspace, (hipStream_t)stream) : forward<half_t>(a, bs_last, (float *)workspace, (hipStream_t)stream);
}

int64_t ksmm_residual_norm_backward_workspace(int64_t batch, int64_t features, int64_t groups, int dtype, int bs_last)
{
    if (batch < 1 || features < 1 || groups < 1 || batch % groups) return KSMM_ERR_BAD_BATCH;
    if (dtype != KSMM_F32 && dtype != KSMM_F16) return KSMM_ERR_BAD_DTYPE;
    return layout(batch, features, groups, dtype, bs_last).total;
}

int ksmm_residual_norm_backward(const ksmm_norm_desc *desc, const float *stats, const void *dr_out, const void *dn_out, void *dx,
                                void *dresidual, void *dgate, void *dpost_weight, void *dweight, void *dbias, void *workspace,
                                int64_t workspace_bytes, int64_t batch, int64_t features, int dtype, int bs_last, void *stream)
{
    const int rc = check(desc, batch, features, dtype, bs_last);
    if (rc != KSMM_OK) return rc;
    if (!stats || (!dr_out && !dn_out)) return KSMM_ERR_NULL_POINTER;
    if ((!desc->x && (dx || dgate || dpost_weight)) || (dgate && !desc->gate) || (dpost_weight && !desc->post_weight) ||
        (dweight && !desc->weight) || (dbias && !desc->bias))
        return KSMM_ERR_NULL_POINTER;
    const Layout l = layout(batch, features, desc->groups, dtype, bs_last);
    if (!workspace || workspace_bytes < l.total || ((uintptr_t)workspace & 15) != 0) return KSMM_ERR_WORKSPACE;
    const bool gate_alone = dgate && bs_last && !l.split.one_gate;
    if (gate_alone && l.split.groups * features > 0x7fffffffLL) return KSMM_ERR_TOO_LARGE;
    const int64_t size = batch * features * (int64_t)dtype_size(dtype);
    NormArgs a = args_of(desc, batch, features);
    {
        const int64_t vector = features * (int64_t)dtype_size(dtype);
        const Span written[] = {{dx, size}, {dresidual, size}, {dgate, desc->groups * vector}, {dpost_weight, vector}, {dweight, vector}, {dbias, vector},
                                {workspace, l.total}};
        const Span gradients[] = {{stats, 16 * batch}, {dr_out, size}, {dn_out, size}};
        if (any_overlap(operands_of(a, desc->groups, dtype).of, written) || any_overlap(gradients, written)) return KSMM_ERR_ALIAS;
    }
    const hipStream_t s = (hipStream_t)stream;
    a.stats = (float *)stats;
    char *const ws = (char *)workspace;
    NormGrads p;
    p.dr_out = dr_out;
    p.dn_out = dn_out;
    p.dx = dx;
    p.dresidual = dresidual;
    p.dweight = dweight && dn_out ? (float *)ws : nullptr;
    p.dbias = dbias && dn_out ? (float *)(ws + l.slice_bytes) : nullptr;
    p.dpost_weight = dpost_weight ? (float *)(ws + 2 * l.slice_bytes) : nullptr;
    p.dgate = dgate && !gate_alone ? (float *)(ws + 3 * l.slice_bytes) : nullptr;
    p.means = gate_alone ? (float *)(ws + l.means) : nullptr;
    int st = dtype == KSMM_F32 ? backward<float>(a, p, l.split, bs_last, (float *)(ws + l.steps), s) : backward<half_t>(a, p, l.split, bs_last, (float *)(ws + l.steps), s);
    if (st != KSMM_OK) return st;
    if (gate_alone) {
        const int64_t waves = l.split.groups * ((features + GATE_FEATURES - 1) / GATE_FEATURES);
        const dim3 blocks((unsigned)((waves + 3) / 4));
        if (dtype == KSMM_F32)
            hipLaunchKernelGGL((ks_norm_cols_gate_kernel<float>), blocks, dim3(256), 0, s, a, p, (float *)dgate, l.split.groups);
        else
            hipLaunchKernelGGL((ks_norm_cols_gate_kernel<half_t>), blocks, dim3(256), 0, s, a, p, (half_t *)dgate, l.split.groups);
        st = launched();
        if (st != KSMM_OK) return st;
    }
    if (!dn_out && (dweight || dbias)) {
        const dim3 blocks((unsigned)((features + 255) / 256));
        if (dtype == KSMM_F32)
            hipLaunchKernelGGL((ks_norm_clear_kernel<float>), blocks, dim3(256), 0, s, (float *)dweight, (float *)dbias, (int)features);
        else
            hipLaunchKernelGGL((ks_norm_clear_kernel<half_t>), blocks, dim3(256), 0, s, (half_t *)dweight, (half_t *)dbias, (int)features);
        st = launched();
        if (st != KSMM_OK) return st;
    }
    FinishJob jobs[4];
    int n = 0;
    auto finish = [&](const float *from, void *to, int64_t values, int64_t slices) {
        if (from) jobs[n++] = FinishJob{from, to, values, (int)slices, 1.f};
    };
    finish(p.dweight, dweight, features, l.slices);
    finish(p.dbias, dbias, features, l.slices);
    finish(p.dpost_weight, dpost_weight, features, l.slices);
    if (p.dgate) {
        if (l.split.one_gate)
            finish(p.dgate, dgate, features, l.slices);
        else
            finish(p.dgate, dgate, l.split.groups * features, l.split.parts);
    }
    return finish_run(jobs, n, dtype, s);
}

}  // extern "C"
