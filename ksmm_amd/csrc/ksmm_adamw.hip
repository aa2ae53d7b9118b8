// One step of AdamW over many tensors, its moments in 32 or in 8 bits.
//
//     g = s grad,  m' = beta1 m + (1 - beta1) g,  v' = beta2 v + (1 - beta2) g^2
//     w' = (1 - lr decay) w - lr / (1 - beta1^t) * m' / (sqrt(v') / sqrt(1 - beta2^t) + eps)
//
// Moments in 8 bits: 32 consecutive values of a tensor share a power of two.  m is e4m3 behind 2^(floor(log2 max |m|) - 7), v an
// unsigned e5m3 (the upper bits of an fp16 number without its sign) behind 2^(floor(log2 max v) - 14).  Both are rounded up or
// down with the probability that keeps the mean: v changes by a thousandth a step, a 60th of half a step of its type, and to
// the nearest it would stay where it is.  What decides is a hash of seed, tensor, step and place, so that a step is the same on
// every run.  A v above zero never becomes zero.  New moments are computed in 64 bits, where the decision of a value next to
// a border does not depend on the order of roundings; the weights take them in 32.
//
// What bounds it: HBM, 16 bytes a weight in fp16 with 8-bit moments and fp32 weights behind them, 28 in fp32.
#include "ksmm_common.h"
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <vector>

namespace ksmm {

namespace {

constexpr int PER = 8, THREADS = 256;
constexpr int CHUNK = THREADS * PER * 2;  // values a workgroup takes
constexpr int MOST = 64;                  // tensors a launch: their table is a kernel argument, 4 KB at most

struct Tensor {
    void *w;
    const void *g;
    float *master;
    void *m, *v;
    uint8_t *scales;  // m's, then v's
    uint32_t n, first;  // values, and the first workgroup; first's highest bit: every pointer allows vectors
};
struct Args {
    Tensor t[MOST];
    int count;
    uint32_t seed;  // the first tensor's
    int follow;
    float keep, lr, rate, root, eps;  // rate, root: of the step, or (with `step`) to be found from it
    double beta1, beta2, scale;
    int64_t step;
    const int64_t *device_step;
};
static_assert(sizeof(Args) <= 4096, "kernel arguments");

__host__ __device__ __forceinline__ uint32_t mix(uint32_t x)
{
    x = (x ^ x >> 16) * 0x6A09E667u;  // 2^32 times the fractions of sqrt(2) and sqrt(3)
    x = (x ^ x >> 15) * 0xBB67AE85u;
    return x ^ x >> 16;
}

// the tensor that workgroup `group` works on
__device__ __forceinline__ int tensor_of(const Tensor *t, int count, uint32_t group)
{
    int low = 0, high = count;  // low's first <= group < high's
    while (high - low > 1) {
        const int middle = (low + high) / 2;
        if ((t[middle].first & 0x7fffffffu) <= group)
            low = middle;
        else
            high = middle;
    }
    return low;
}

template <typename T> struct Values {
    T v[PER];
};
// values at .. at + 7, as far as they are there; `whole`: all of them, at a vector's alignment
template <typename T> __device__ __forceinline__ Values<T> load(const T *p, uint32_t at, uint32_t n, bool whole)
{
    Values<T> r;
    if (whole) {
        __builtin_memcpy(&r, __builtin_assume_aligned(p + at, sizeof(r) < 16 ? sizeof(r) : 16), sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) r.v[i] = at + i < n ? p[at + i] : (T)0;
    }
    return r;
}
template <typename T> __device__ __forceinline__ void store(T *p, uint32_t at, uint32_t n, bool whole, const Values<T> &r)
{
    if (whole) {
        __builtin_memcpy(__builtin_assume_aligned(p + at, sizeof(r) < 16 ? sizeof(r) : 16), &r, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (at + i < n) p[at + i] = r.v[i];
    }
}

__device__ __forceinline__ double power64(int e) { return __builtin_bit_cast(double, (uint64_t)(e + 1023) << 52); }
__device__ __forceinline__ int exponent64(double v) { return (int)(__builtin_bit_cast(uint64_t, v) >> 52 & 0x7ff) - 1023; }
__device__ __forceinline__ float scale_value(uint8_t byte)
{
    return byte ? __builtin_bit_cast(float, (uint32_t)byte << 23) : __builtin_bit_cast(float, 0x00400000u);
}

// largest of the four lanes that hold a block of 32
__device__ __forceinline__ int block_max(int v)
{
    v = max(v, __shfl_xor(v, 1, 64));
    return max(v, __shfl_xor(v, 2, 64));
}

constexpr int LOWEST = -120;  // exponent of a scale

// |y| 2^-e, to 3 bits behind its leading one from exponent `least` on, down or up as the dither (in 2^-16) says
__device__ __forceinline__ float rounded(double y, int e, int least, uint32_t dither)
{
    const int q = max(exponent64(y) - e, least) - 3;
    const double steps = floor(y * power64(-e - q) + (double)dither * (1.0 / 65536));
    return (float)steps * __builtin_bit_cast(float, (uint32_t)(q + 127) << 23);
}

// e5m3 from what `rounded` gives
__device__ __forceinline__ uint8_t e5m3(float v) { return (uint8_t)(__builtin_bit_cast(uint16_t, (half_t)v) >> 7); }
__device__ __forceinline__ float from_e5m3(uint8_t code) { return (float)__builtin_bit_cast(half_t, (uint16_t)(code << 7)); }
__device__ __forceinline__ float from_e4m3(uint8_t code) { return __builtin_amdgcn_cvt_f32_fp8(code, 0); }

// A block's new moments as codes, and its scale; every lane of the four has eight of its values.
__device__ __forceinline__ uint8_t encode_m(const double (&m)[PER], const uint32_t (&h)[PER], Values<uint8_t> &code)
{
    int top = -1023;
#pragma unroll
    for (int i = 0; i < PER; ++i) top = max(top, fabs(m[i]) <= FLT_MAX ? exponent64(m[i]) : -1023);
    const int e = max(block_max(top) - 7, LOWEST);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const bool finite = fabs(m[i]) <= FLT_MAX;
        const float v = copysignf(finite ? rounded(fabs(m[i]), e, -6, h[i] & 0xffff) : 0.f, (float)m[i]);
        code.v[i] = finite ? (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) : 0x7f;
    }
    return (uint8_t)(e + 127);
}
__device__ __forceinline__ uint8_t encode_v(const double (&v)[PER], const uint32_t (&h)[PER], Values<uint8_t> &code)
{
    int top = -1023;
#pragma unroll
    for (int i = 0; i < PER; ++i) top = max(top, v[i] <= FLT_MAX ? exponent64(v[i]) : -1023);
    const int e = max(block_max(top) - 14, LOWEST);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const bool finite = v[i] <= FLT_MAX;
        const uint8_t c = finite ? e5m3(rounded(v[i], e, -14, h[i] >> 16)) : v[i] > 0 ? 0xf8 : 0xfc;  // (infinity, NaN)
        code.v[i] = c == 0 && v[i] > 0 ? 1 : c;
    }
    return (uint8_t)(e + 127);
}

template <typename T, int BITS, bool MASTER> __global__ __launch_bounds__(THREADS) void ks_adamw_kernel(Args a)
{
#pragma clang fp contract(off)
    __shared__ float of_step[2];
    const int which = tensor_of(a.t, a.count, blockIdx.x);
    const Tensor &t = a.t[which];
    const bool aligned = t.first >> 31;
    const uint32_t n = t.n, start = (blockIdx.x - (t.first & 0x7fffffffu)) * (uint32_t)CHUNK;
    int64_t step = a.step;
    float rate = a.rate, root = a.root;
    if (a.device_step) {
        step = *a.device_step;
        if (threadIdx.x == 0) {
            const double at = step < 1 ? 1.0 : (double)step;
            of_step[0] = (float)((double)a.lr / (1.0 - pow(a.beta1, at)));
            of_step[1] = (float)(1.0 / sqrt(1.0 - pow(a.beta2, at)));
        }
        __syncthreads();
        rate = of_step[0];
        root = of_step[1];
    }
    const uint32_t key = mix(mix(a.seed + (uint32_t)which) + (uint32_t)step);
    const double beta1 = a.beta1, beta2 = a.beta2, other1 = 1.0 - beta1, other2 = 1.0 - beta2;
    for (uint32_t at = start + threadIdx.x * PER; at < start + CHUNK; at += THREADS * PER) {
        // (the lanes of a block of 32 stay together: those behind the end hold zeros)
        if ((at & ~31u) >= n) break;
        const bool whole = aligned && at + PER <= n;
        const Values<T> g = load((const T *)t.g, at, n, whole);
        Values<T> w = load((const T *)t.w, at, n, whole);
        Values<float> master;
        if constexpr (MASTER) master = load((const float *)t.master, at, n, whole);
        float m_new[PER], v_new[PER];
        if constexpr (BITS == 32) {
            Values<float> m = load((const float *)t.m, at, n, whole), v = load((const float *)t.v, at, n, whole);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float x = (float)g.v[i] * (float)a.scale;
                m.v[i] = m_new[i] = (float)beta1 * m.v[i] + (float)other1 * x;
                v.v[i] = v_new[i] = (float)beta2 * v.v[i] + (float)other2 * (x * x);
            }
            store((float *)t.m, at, n, whole, m);
            store((float *)t.v, at, n, whole, v);
        } else {
            const uint32_t blocks = (n + 31) / 32, block = at / 32;
            Values<uint8_t> cm = load((const uint8_t *)t.m, at, n, whole), cv = load((const uint8_t *)t.v, at, n, whole);
            const float sm = scale_value(t.scales[block]), sv = scale_value(t.scales[blocks + block]);
            double m[PER], v[PER];
            uint32_t h[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const double x = (double)(float)g.v[i] * a.scale;
                m[i] = (double)(from_e4m3(cm.v[i]) * sm) * beta1 + x * other1;
                v[i] = (double)(from_e5m3(cv.v[i]) * sv) * beta2 + x * x * other2;
                m_new[i] = (float)m[i];
                v_new[i] = (float)v[i];
                h[i] = mix(at + i ^ key);
            }
            const uint8_t em = encode_m(m, h, cm), ev = encode_v(v, h, cv);
            store((uint8_t *)t.m, at, n, whole, cm);
            store((uint8_t *)t.v, at, n, whole, cv);
            if ((at & 31) == 0) {
                t.scales[block] = em;
                t.scales[blocks + block] = ev;
            }
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            float old = (float)w.v[i];
            if constexpr (MASTER) old = a.follow && (T)master.v[i] != w.v[i] ? old : master.v[i];
            const float next = a.keep * old - rate * (m_new[i] / (sqrtf(v_new[i]) * root + a.eps));
            if constexpr (MASTER) master.v[i] = next;
            w.v[i] = (T)next;
        }
        if constexpr (MASTER) store(t.master, at, n, whole, master);
        store((T *)t.w, at, n, whole, w);
    }
}

// What 8-bit moments stand for (w, master: where m and v go, as fp32).
__global__ __launch_bounds__(THREADS) void ks_adamw_moments_kernel(Args a)
{
    const Tensor &t = a.t[tensor_of(a.t, a.count, blockIdx.x)];
    const bool aligned = t.first >> 31;
    const uint32_t n = t.n, start = (blockIdx.x - (t.first & 0x7fffffffu)) * (uint32_t)CHUNK, blocks = (n + 31) / 32;
    for (uint32_t at = start + threadIdx.x * PER; at < start + CHUNK && at < n; at += THREADS * PER) {
        const bool whole = aligned && at + PER <= n;
        const Values<uint8_t> cm = load((const uint8_t *)t.m, at, n, whole), cv = load((const uint8_t *)t.v, at, n, whole);
        const float sm = scale_value(t.scales[at / 32]), sv = scale_value(t.scales[blocks + at / 32]);
        Values<float> m, v;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            m.v[i] = from_e4m3(cm.v[i]) * sm;
            v.v[i] = from_e5m3(cv.v[i]) * sv;
        }
        store((float *)t.w, at, n, whole, m);
        store(t.master, at, n, whole, v);
    }
}

struct Range {
    uintptr_t from, to;
    bool written;
};
// whether something that is written overlaps anything else
bool any_alias(std::vector<Range> &r)
{
    std::sort(r.begin(), r.end(), [](const Range &x, const Range &y) { return x.from < y.from; });
    uintptr_t seen = 0, written = 0;
    for (const Range &x : r) {
        if (x.from < (x.written ? seen : written)) return true;
        seen = std::max(seen, x.to);
        if (x.written) written = std::max(written, x.to);
    }
    return false;
}
void add(std::vector<Range> &r, const void *p, int64_t bytes, bool written)
{
    if (p && bytes > 0) r.push_back(Range{(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, written});
}

template <typename F> int in_tables(Args &a, const Tensor *all, int n, F launch)
{
    uint32_t groups = 0;
    int first = 0;
    const uint32_t seed = a.seed;
    a.count = 0;
    for (int i = 0; i <= n; ++i) {
        const uint32_t more = i < n ? (all[i].n + CHUNK - 1) / CHUNK : 0;
        // (a table's workgroups are counted in 31 bits)
        if (a.count > 0 && (i == n || a.count == MOST || (uint64_t)groups + more > 0x7fffffffu)) {
            a.seed = seed + (uint32_t)first;
            launch(groups);
            if (hipGetLastError() != hipSuccess) return KSMM_ERR_LAUNCH;
            groups = 0;
            a.count = 0;
        }
        if (i == n) break;
        if (a.count == 0) first = i;
        Tensor &t = a.t[a.count++] = all[i];
        t.first |= groups;
        groups += more;
    }
    return KSMM_OK;
}

bool aligned(const void *p, int to) { return ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace

}  // namespace ksmm

using namespace ksmm;

extern "C" {

int ksmm_adamw_update(const ksmm_adamw_desc *desc, const ksmm_adamw_tensor *tensors, int count, int dtype, void *stream)
{
    if (!desc || (count > 0 && !tensors)) return KSMM_ERR_NULL_POINTER;
    if (count < 0) return KSMM_ERR_BAD_BATCH;
    if (dtype != KSMM_F32 && dtype != KSMM_F16) return KSMM_ERR_BAD_DTYPE;
    if (desc->bits != 8 && desc->bits != 32) return KSMM_ERR_BAD_DTYPE;
    const double betas[] = {desc->beta1, desc->beta2}, rates[] = {desc->lr, desc->eps, desc->weight_decay, desc->grad_scale};
    for (double b : betas)
        if (!(b >= 0.0 && b < 1.0)) return KSMM_ERR_BAD_ALGO;
    for (double r : rates)
        if (!std::isfinite(r)) return KSMM_ERR_BAD_ALGO;
    if (!desc->device_step && desc->step < 1) return KSMM_ERR_BAD_ALGO;
    const int64_t size = (int64_t)dtype_size(dtype);
    const bool small = desc->bits == 8;
    try {
        std::vector<Tensor> all;
        std::vector<Range> ranges;
        all.reserve(count);
        ranges.reserve(6 * (size_t)count + 1);
        add(ranges, desc->device_step, 8, false);
        bool master = false, any = false;
        for (int i = 0; i < count; ++i) {
            const ksmm_adamw_tensor &t = tensors[i];
            if (t.n < 0) return KSMM_ERR_BAD_BATCH;
            if (t.n > 0x7fffffffLL - CHUNK) return KSMM_ERR_TOO_LARGE;
            if (t.n > 0) {  // (pointers of empty tensors say nothing)
                if (!any) master = t.master != nullptr;
                any = true;
                if ((t.master != nullptr) != master) return KSMM_ERR_NULL_POINTER;
                if (!t.weight || !t.grad || !t.m || !t.v || (small && !t.scales)) return KSMM_ERR_NULL_POINTER;
            }
            const int64_t state = small ? t.n : 4 * t.n;
            add(ranges, t.weight, size * t.n, true);
            add(ranges, t.grad, size * t.n, false);
            add(ranges, t.master, 4 * t.n, true);
            add(ranges, t.m, state, true);
            add(ranges, t.v, state, true);
            if (small) add(ranges, t.scales, 2 * ((t.n + 31) / 32), true);
            const bool vectors = aligned(t.weight, 16) && aligned(t.grad, 16) && aligned(t.master, 16) && aligned(t.m, small ? 8 : 16) && aligned(t.v, small ? 8 : 16);
            all.push_back(Tensor{t.weight, t.grad, t.master, t.m, t.v, (uint8_t *)t.scales, (uint32_t)t.n, vectors ? 0x80000000u : 0u});
        }
        if (any_alias(ranges)) return KSMM_ERR_ALIAS;
        Args a{};
        const double at = (double)desc->step;
        a.seed = desc->seed;
        a.follow = desc->follow;
        a.keep = (float)(1.0 - desc->lr * desc->weight_decay);
        a.lr = (float)desc->lr;
        a.rate = desc->device_step ? 0.f : (float)(desc->lr / (1.0 - std::pow(desc->beta1, at)));
        a.root = desc->device_step ? 0.f : (float)(1.0 / std::sqrt(1.0 - std::pow(desc->beta2, at)));
        a.eps = (float)desc->eps;
        a.beta1 = desc->beta1;
        a.beta2 = desc->beta2;
        a.scale = desc->grad_scale;
        a.step = desc->step;
        a.device_step = desc->device_step;
        hipStream_t s = (hipStream_t)stream;
        auto run = [&](auto kernel) {
            return in_tables(a, all.data(), count, [&](uint32_t groups) {
                if (groups > 0) hipLaunchKernelGGL(kernel, dim3(groups), dim3(THREADS), 0, s, a);
            });
        };
        if (dtype == KSMM_F32) {
            if (master) return small ? run(&ks_adamw_kernel<float, 8, true>) : run(&ks_adamw_kernel<float, 32, true>);
            return small ? run(&ks_adamw_kernel<float, 8, false>) : run(&ks_adamw_kernel<float, 32, false>);
        }
        if (master) return small ? run(&ks_adamw_kernel<half_t, 8, true>) : run(&ks_adamw_kernel<half_t, 32, true>);
        return small ? run(&ks_adamw_kernel<half_t, 8, false>) : run(&ks_adamw_kernel<half_t, 32, false>);
    } catch (...) {  // (no memory for the tables)
        return KSMM_ERR_TOO_LARGE;
    }
}

int ksmm_adamw_moments(const ksmm_adamw_moment *tensors, int count, void *stream)
{
    if (count > 0 && !tensors) return KSMM_ERR_NULL_POINTER;
    if (count < 0) return KSMM_ERR_BAD_BATCH;
    try {
        std::vector<Tensor> all;
        std::vector<Range> ranges;
        all.reserve(count);
        ranges.reserve(5 * (size_t)count);
        for (int i = 0; i < count; ++i) {
            const ksmm_adamw_moment &t = tensors[i];
            if (t.n < 0) return KSMM_ERR_BAD_BATCH;
            if (t.n > 0x7fffffffLL - CHUNK) return KSMM_ERR_TOO_LARGE;
            if (t.n > 0 && (!t.m || !t.v || !t.scales || !t.m_out || !t.v_out)) return KSMM_ERR_NULL_POINTER;
            add(ranges, t.m, t.n, false);
            add(ranges, t.v, t.n, false);
            add(ranges, t.scales, 2 * ((t.n + 31) / 32), false);
            add(ranges, t.m_out, 4 * t.n, true);
            add(ranges, t.v_out, 4 * t.n, true);
            const bool vectors = aligned(t.m, 8) && aligned(t.v, 8) && aligned(t.m_out, 16) && aligned(t.v_out, 16);
            all.push_back(Tensor{t.m_out, nullptr, t.v_out, (void *)t.m, (void *)t.v, (uint8_t *)t.scales, (uint32_t)t.n, vectors ? 0x80000000u : 0u});
        }
        if (any_alias(ranges)) return KSMM_ERR_ALIAS;
        Args a{};
        return in_tables(a, all.data(), count, [&](uint32_t groups) {
            if (groups > 0) hipLaunchKernelGGL(ks_adamw_moments_kernel, dim3(groups), dim3(THREADS), 0, (hipStream_t)stream, a);
        });
    } catch (...) {
        return KSMM_ERR_TOO_LARGE;
    }
}

}  // extern "C"
