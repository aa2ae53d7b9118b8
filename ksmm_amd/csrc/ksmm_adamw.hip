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
// What bounds it: HBM, 16 bytes a weight in fp16 with 8-bit moments and fp32 weights behind them, 28 in fp32.  10.9 million values of 72
// tensors in fp32: 306 MB in 61 us, 5.0 TB/s; 14.4 million with 8-bit moments: 257 MB in 64, 4 TB/s, of which the vector ALU is
// busy for half (64-bit moments, codes); what they stand for 23 us.  A value costs one read and one write of each tensor whatever
// the order, so that all there is to choose is how many are on their way: four a thread, vectors of 4 to 16
// bytes (eight: 65 us for 61, the same for 64, 25 for 23).
#include "ksmm_common.h"
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>
#include <vector>

namespace ksmm {

namespace {

constexpr int PER = 4;                    // values a thread takes at a time

struct Tensor {
    void *w;
    const void *g;
    float *master;
    void *m, *v;
    uint8_t *scales;  // m's, then v's
    uint32_t n, first;  // values, and the first workgroup; first's highest bit: every pointer allows vectors
};
// The tensors of a launch are a kernel argument, of 4 KB at most: without pointers that are not there more of them fit.
template <bool MASTER, bool SCALES> struct Entry {
    const void *p[4 + MASTER + SCALES];
    uint32_t n, first;
    static constexpr bool HAS_MASTER = MASTER, HAS_SCALES = SCALES;
    __host__ __device__ void set(const Tensor &t)
    {
        p[0] = t.w;
        p[1] = t.g;
        p[2] = t.m;
        p[3] = t.v;
        if constexpr (MASTER) p[4] = t.master;
        if constexpr (SCALES) p[4 + MASTER] = t.scales;
        n = t.n;
        first = t.first;
    }
    __device__ Tensor get() const
    {
        Tensor t{(void *)p[0], p[1], nullptr, (void *)p[2], (void *)p[3], nullptr, n, first};
        if constexpr (MASTER) t.master = (float *)p[4];
        if constexpr (SCALES) t.scales = (uint8_t *)p[4 + MASTER];
        return t;
    }
};
struct Common {
    int count;
    uint32_t chunk;  // values a workgroup takes: 256 threads' once (8-bit moments: twice), or where that makes few, of 64 threads
    uint32_t seed;  // the first tensor's
    int follow;
    float keep, rate, root, eps;  // rate, root: of the step, or (with `device_step`) to be found from it
    double lr, beta1, beta2, scale;
    int64_t step;
    const int64_t *device_step;
};
template <typename E> struct Args : Common {
    static constexpr int MOST = (int)((4096 - sizeof(Common)) / sizeof(E)) < 128 ? (int)((4096 - sizeof(Common)) / sizeof(E)) : 128;
    E t[MOST];
};

__host__ __device__ __forceinline__ uint32_t mix(uint32_t x)
{
    x = (x ^ x >> 16) * 0x6A09E667u;  // 2^32 times the fractions of sqrt(2) and sqrt(3)
    x = (x ^ x >> 15) * 0xBB67AE85u;
    return x ^ x >> 16;
}

// the tensor that workgroup `group` works on: of all that begin at it or before, the last (every lane looks at two)
template <typename E> __device__ __forceinline__ int tensor_of(const Args<E> &a, uint32_t group)
{
    const int lane = threadIdx.x & 63;
    auto before = [&](int i) { return __popcll(__ballot(i < a.count && (a.t[i].first & 0x7fffffffu) <= group)); };
    return before(lane) + (a.count > 64 ? before(lane + 64) : 0) - 1;
}

template <typename T> struct Values {
    T v[PER];
};
// values at .. at + 3, as far as they are there; `whole`: all of them, at a vector's alignment
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

__device__ __forceinline__ int exponent64(double v) { return (int)(__builtin_bit_cast(uint64_t, v) >> 52 & 0x7ff) - 1023; }
__device__ __forceinline__ float scale_value(uint8_t byte)
{
    return byte ? __builtin_bit_cast(float, (uint32_t)byte << 23) : __builtin_bit_cast(float, 0x00400000u);
}

// largest of the eight lanes that hold a block of 32
__device__ __forceinline__ int block_max(int v)
{
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true));  // lanes 1 0 3 2
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true));  // 2 3 0 1
    return max(v, __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true));  // 7 6 5 4 3 2 1 0: the other four's
}

constexpr int LOWEST = -120;  // exponent of a scale

// y 2^-e (y >= 0, its exponent given) to 3 bits behind its leading one from exponent `least` on, down or up as the dither (in 2^-16)
// says, as the code of an 8-bit number: steps of its exponent E are 8 to 16 (below, of `least`, 0 to 8), and (E - least) 8 + steps
// carries into the exponent by itself.
__device__ __forceinline__ uint32_t rounded(double y, int exponent, int e, int least, uint32_t dither)
{
    const int E = max(exponent - e, least);
    const double steps = fma((double)dither, 1.0 / 65536, __builtin_ldexp(y, 3 - e - E));
    uint32_t code = (uint32_t)(E - least) * 8 + (uint32_t)steps;
    asm("" : "+v"(code));  // (found for every value, and not behind a branch on whether it is finite)
    return code;
}

__device__ __forceinline__ float from_e5m3(uint8_t code) { return (float)__builtin_bit_cast(half_t, (uint16_t)(code << 7)); }
__device__ __forceinline__ float from_e4m3(uint8_t code) { return __builtin_amdgcn_cvt_f32_fp8(code, 0); }

// A block's new moments as codes, and its scale; every lane of the eight has four of its values.  What is 2^128 or more, or NaN, is not
// counted among the largest.
__device__ __forceinline__ uint8_t encode_m(const double (&m)[PER], const uint32_t (&h)[PER], Values<uint8_t> &code)
{
    int top = -1023, at[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        at[i] = exponent64(m[i]);
        top = max(top, at[i] < 128 ? at[i] : -1023);
    }
    const int e = max(block_max(top) - 7, LOWEST);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const uint32_t sign = (uint32_t)(__builtin_bit_cast(uint64_t, m[i]) >> 63) << 7;
        const uint32_t c = rounded(fabs(m[i]), at[i], e, -6, h[i] & 0xffff) | sign;
        code.v[i] = (uint8_t)(at[i] < 128 ? c : 0x7f);  // (NaN)
    }
    return (uint8_t)(e + 127);
}
__device__ __forceinline__ uint8_t encode_v(const double (&v)[PER], const uint32_t (&h)[PER], Values<uint8_t> &code)
{
    int top = -1023, at[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        at[i] = exponent64(v[i]);
        top = max(top, at[i] < 128 ? at[i] : -1023);
    }
    const int e = max(block_max(top) - 14, LOWEST);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const uint32_t c = rounded(v[i], at[i], e, -14, h[i] >> 16), least = v[i] > 0 ? 1 : 0;
        code.v[i] = (uint8_t)(at[i] < 128 ? max(c, least) : v[i] > 0 ? 0xf8 : 0xfc);  // (infinity, NaN)
    }
    return (uint8_t)(e + 127);
}

// sqrt and quotient, good to a few 2^-24 of the value: the correctly rounded ones take 25 instructions more a value.  The instruction
// takes what is subnormal as zero, so that small values are moved up before it.
__device__ __forceinline__ float root_of(float v)
{
    const bool small = v < 0x1p-96f;
    const float r = __builtin_amdgcn_sqrtf(small ? v * 0x1p96f : v);
    return small ? r * 0x1p-48f : r;
}

template <typename T, int BITS, bool MASTER> __global__ __launch_bounds__(256) void ks_adamw_kernel(Args<Entry<MASTER, BITS == 8>> a)
{
#pragma clang fp contract(off)
    __shared__ float of_step[2];
    const int which = tensor_of(a, blockIdx.x);
    const Tensor t = a.t[which].get();
    const bool aligned = t.first >> 31;
    const uint32_t n = t.n, start = (blockIdx.x - (t.first & 0x7fffffffu)) * a.chunk;
    int64_t step = a.step;
    float rate = a.rate, root = a.root;
    if (a.device_step) {
        step = *a.device_step;
        if (threadIdx.x == 0) {
            const double at = step < 1 ? 1.0 : (double)step;
            of_step[0] = (float)(a.lr / (1.0 - pow(a.beta1, at)));
            of_step[1] = (float)(1.0 / sqrt(1.0 - pow(a.beta2, at)));
        }
        __syncthreads();
        rate = of_step[0];
        root = of_step[1];
    }
    const uint32_t key = mix(mix(a.seed + (uint32_t)which) + (uint32_t)step);
    const double beta1 = a.beta1, beta2 = a.beta2, other1 = 1.0 - beta1, other2 = 1.0 - beta2;
    for (uint32_t at = start + threadIdx.x * PER; at < start + a.chunk; at += blockDim.x * PER) {
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
            const float next = a.keep * old - rate * (m_new[i] * __builtin_amdgcn_rcpf(root_of(v_new[i]) * root + a.eps));
            if constexpr (MASTER) master.v[i] = next;
            w.v[i] = (T)next;
        }
        if constexpr (MASTER) store(t.master, at, n, whole, master);
        store((T *)t.w, at, n, whole, w);
    }
}

// What 8-bit moments stand for (w, master: where m and v go, as fp32).
__global__ __launch_bounds__(256) void ks_adamw_moments_kernel(Args<Entry<true, true>> a)
{
    const Tensor t = a.t[tensor_of(a, blockIdx.x)].get();
    const bool aligned = t.first >> 31;
    const uint32_t n = t.n, start = (blockIdx.x - (t.first & 0x7fffffffu)) * a.chunk, blocks = (n + 31) / 32;
    for (uint32_t at = start + threadIdx.x * PER; at < start + a.chunk && at < n; at += blockDim.x * PER) {
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

template <typename E, typename F> int in_tables(const Common &common, const Tensor *all, int n, F launch)
{
    Args<E> a;
    (Common &)a = common;
    uint32_t groups = 0;
    int first = 0;
    const uint32_t seed = a.seed;
    int64_t values = 0;
    for (int i = 0; i < n; ++i) values += all[i].n;
    // (172 thousand 8-bit values of 25 tensors: 10.6 us in workgroups of 256 threads)
    const int threads = values < 1 << 20 ? 64 : 256;
    // (28 bytes a value: 61 us once, 62.6 twice, 67 four times; 8-bit moments 95, 90.5 and 95 with the launch that gives them back)
    a.chunk = threads * PER * (threads == 256 && E::HAS_SCALES ? 2 : 1);
    a.count = 0;
    for (int i = 0; i <= n; ++i) {
        const uint32_t more = i < n ? (all[i].n + a.chunk - 1) / a.chunk : 0;
        if (a.count > 0 && (i == n || a.count == Args<E>::MOST || (int64_t)groups + more > THREADS_MOST / threads)) {
            a.seed = seed + (uint32_t)first;
            if (groups > 0) {
                const int rc = launch(a, groups, threads);
                if (rc != KSMM_OK) return rc;
            }
            groups = 0;
            a.count = 0;
        }
        if (i == n) break;
        if (a.count == 0) first = i;
        Tensor t = all[i];
        t.first |= groups;
        a.t[a.count++].set(t);
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
    if (desc->eps != 0.0 && std::fabs(desc->eps) < FLT_MIN) return KSMM_ERR_BAD_ALGO;  // (0 / eps is 0: its reciprocal has to be a number)
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
            if (t.n > 0x7fffffffLL - 8192) return KSMM_ERR_TOO_LARGE;
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
            const bool vectors = aligned(t.weight, PER * (int)size) && aligned(t.grad, PER * (int)size) && aligned(t.master, PER * 4) && aligned(t.m, small ? PER : PER * 4) &&
                                 aligned(t.v, small ? PER : PER * 4);
            all.push_back(Tensor{t.weight, t.grad, t.master, t.m, t.v, (uint8_t *)t.scales, (uint32_t)t.n, vectors ? 0x80000000u : 0u});
        }
        if (any_alias(ranges)) return KSMM_ERR_ALIAS;
        Common a{};
        const double at = (double)desc->step;
        a.seed = desc->seed;
        a.follow = desc->follow;
        a.keep = (float)(1.0 - desc->lr * desc->weight_decay);
        a.lr = desc->lr;
        a.rate = desc->device_step ? 0.f : (float)(desc->lr / (1.0 - std::pow(desc->beta1, at)));
        a.root = desc->device_step ? 0.f : (float)(1.0 / std::sqrt(1.0 - std::pow(desc->beta2, at)));
        a.eps = (float)desc->eps;
        a.beta1 = desc->beta1;
        a.beta2 = desc->beta2;
        a.scale = desc->grad_scale;
        a.step = desc->step;
        a.device_step = desc->device_step;
        hipStream_t s = (hipStream_t)stream;
        auto run = [&](auto of, auto masters, auto states) {
            typedef decltype(of) T;
            constexpr bool MASTER = decltype(masters)::value, SMALL = decltype(states)::value;
            return in_tables<Entry<MASTER, SMALL>>(a, all.data(), count, [&](const Args<Entry<MASTER, SMALL>> &args, uint32_t groups, int threads) {
                return launch_kernel(&ks_adamw_kernel<T, SMALL ? 8 : 32, MASTER>, groups, threads, 0, s, args);
            });
        };
        auto with = [&](auto of) {
            if (master) return small ? run(of, std::true_type(), std::true_type()) : run(of, std::true_type(), std::false_type());
            return small ? run(of, std::false_type(), std::true_type()) : run(of, std::false_type(), std::false_type());
        };
        return dtype == KSMM_F32 ? with(0.f) : with((half_t)0.f);
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
            if (t.n > 0x7fffffffLL - 8192) return KSMM_ERR_TOO_LARGE;
            if (t.n > 0 && (!t.m || !t.v || !t.scales || !t.m_out || !t.v_out)) return KSMM_ERR_NULL_POINTER;
            add(ranges, t.m, t.n, false);
            add(ranges, t.v, t.n, false);
            add(ranges, t.scales, 2 * ((t.n + 31) / 32), false);
            add(ranges, t.m_out, 4 * t.n, true);
            add(ranges, t.v_out, 4 * t.n, true);
            const bool vectors = aligned(t.m, PER) && aligned(t.v, PER) && aligned(t.m_out, PER * 4) && aligned(t.v_out, PER * 4);
            all.push_back(Tensor{t.m_out, nullptr, t.v_out, (void *)t.m, (void *)t.v, (uint8_t *)t.scales, (uint32_t)t.n, vectors ? 0x80000000u : 0u});
        }
        if (any_alias(ranges)) return KSMM_ERR_ALIAS;
        Common a{};
        return in_tables<Entry<true, true>>(a, all.data(), count, [&](const Args<Entry<true, true>> &args, uint32_t groups, int threads) {
            return launch_kernel(&ks_adamw_moments_kernel, groups, threads, 0, (hipStream_t)stream, args);
        });
    } catch (...) {
        return KSMM_ERR_TOO_LARGE;
    }
}

}  // extern "C"
