// Activations of the gated and of the 4-bit products, and their slopes.
#pragma once
#include <type_traits>

#include "ksmm_common.h"

namespace ksmm {

constexpr float LOG2E = 1.4426950408889634f;

// act(z), and act'(z) where wanted.  fp32: the library's functions; fp16: forms of two or three transcendentals, good to 5e-6
// of the VALUE (half a step of the type is 2.4e-4 of it): below zero activations fade, and what is left of them is multiplied
// by a projection that may be large.
// GELU is z Phi(z), with Phi(-|z|) as e^(-z^2/2) times a polynomial in t = 1 / (1 + p u), u = |z| / sqrt 2.  The form is that of
// Abramowitz & Stegun 7.1.26, whose own five coefficients bound the error of erf and not that of its tail's value (5e-4 of it
// at z = -4, 4e-3 at -6).  The six here, with p = 0.425, are the least-squares fit of e^(u^2) erfc(u) / 2, weighted anew by its own
// error until the largest relative one is least: 1.7e-6 for u up to 5.6.
// FIXED: the same bits in every kernel (else it is the compiler's to contract 1 - tail with the product that tail is, or not).
template <typename T, int ACT, bool SLOPE, bool FIXED = false> __device__ __forceinline__ float activate(float z, float &slope)
{
    if constexpr (ACT == KSMM_ACT_SILU) {
        float s;
        if constexpr (sizeof(T) == 4)
            s = 1.f / (1.f + expf(-z));
        else
            s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * z));
        if constexpr (SLOPE) slope = s * fmaf(z, 1.f - s, 1.f);
        return z * s;
    }
    if constexpr (ACT == KSMM_ACT_GELU) {
        float phi, ex;
        if constexpr (sizeof(T) == 4) {
            phi = 0.5f * erfcf(-0.70710678118654752f * z);
            ex = SLOPE ? expf(-0.5f * z * z) : 0.f;
        } else {
            const float q = fabsf(z) * 0.84932180028801907f;  // u sqrt(log2 e): the exponential is 2^(-q^2)
            const float t = __builtin_amdgcn_rcpf(fmaf(0.3538357097f, q, 1.0f));
            float poly = fmaf(-0.0821466377f, t, 0.2300047798f);
            poly = fmaf(poly, t, -0.0337080860f);
            poly = fmaf(poly, t, 0.1539474561f);
            poly = fmaf(poly, t, 0.1113554886f);
            poly = fmaf(poly, t, 0.1205461711f);
            ex = __builtin_amdgcn_exp2f(-(q * q));
            if constexpr (FIXED) {
                phi = z >= 0.f ? fmaf(-(poly * t), ex, 1.f) : poly * t * ex;
            } else {
                const float tail = poly * t * ex;
                phi = z >= 0.f ? 1.f - tail : tail;
            }
        }
        if constexpr (SLOPE) slope = fmaf(z * 0.39894228040143268f, ex, phi);
        return z * phi;
    }
    if constexpr (SLOPE) slope = 1.f;
    return z;
}

// one branch on the activation: around all of a tile's values, or around the launch
template <typename F> __host__ __device__ __forceinline__ void with_act(int act, F f)
{
    if (act == KSMM_ACT_SILU)
        f(std::integral_constant<int, KSMM_ACT_SILU>());
    else if (act == KSMM_ACT_GELU)
        f(std::integral_constant<int, KSMM_ACT_GELU>());
    else
        f(std::integral_constant<int, KSMM_ACT_NONE>());
}

}  // namespace ksmm
