// Activations of the projections' and the group norm's epilogues, in fp32.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "seedvr2_hip.h"

namespace s2 {

// x / (1 + e^-x), e^-x = 2^(-x log2 e): from the exponential's overflow on the
// quotient is -0, the limit.
__device__ __forceinline__ float silu_f32(float x) {
    return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f));
}

// tanh-GELU: x (1 + tanh u) / 2 = x / (1 + e^-2u), u = sqrt(2 / pi) (x + 0.044715 x^3)
__device__ __forceinline__ float gelu_tanh_f32(float x) {
    constexpr float a = -2.f * 1.4426950408889634f * 0.79788456080286536f;
    const float z = x * fmaf(a * 0.044715f, x * x, a);
    return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z));
}

// erf-GELU, 0.5 x (1 + erf(x / sqrt 2)) = max(x, 0) - |x| Q(|x|) with
// Q(a) = 0.5 erfc(a / sqrt 2): both signs reduce to one fma, and for x < 0
// the result is the product -|x| Q directly, without cancellation.  erfc is
// Abramowitz & Stegun 7.1.26, erfc(z) = (a1 t + ... + a5 t^5) e^(-z^2),
// t = 1 / (1 + p z), |error| <= 1.5e-7; the factor 0.5 is folded into a1..a5
// and e^(-z^2) = 2^(-w^2) with w = z sqrt(log2 e).  (Q as 2^p(a), p a degree-8
// fit of log2 Q, has one transcendental less and took 1854 us for the 720p
// MLP against 1882, but its rms error over |x| <= 0.1 is 3.5 times this one's,
// 1.8e-8 against 5.3e-9, and its relative error over [-8, -6] 5% against 1%.)
__device__ __forceinline__ float gelu(float x) {
    constexpr float kSqrtLog2e = 1.2011224087864498f;
    const float ax = fabsf(x);
    const float w = ax * (0.70710678118654752f * kSqrtLog2e);
    const float t = __builtin_amdgcn_rcpf(fmaf(w, 0.3275911f / kSqrtLog2e, 1.f));
    const float poly =
        t * (0.5f * 0.254829592f +
             t * (0.5f * -0.284496736f +
                  t * (0.5f * 1.421413741f + t * (0.5f * -1.453152027f + t * (0.5f * 1.061405429f)))));
    const float q = poly * __builtin_amdgcn_exp2f(-w * w);   // Q(|x|)
    // +inf meets q = 0 as the largest finite value, and stays; -inf gives -inf * 0, NaN,
    // as the product 0.5 x (1 + erf) does
    return fmaf(-fabsf(fminf(x, __FLT_MAX__)), q, fmaxf(x, 0.f));
}

// The same for fp32 results, to a few of their steps relative to the value: gelu() above
// is off by up to 0.75e-7 |x|, 4e-4 of the value at -4 and 4e-3 at -6, which is at most
// about half a step of 16-bit results.  e^(a^2 / 2) Q(a) is smooth, a polynomial in t = 1 / (1 + 0.35 a),
// fitted by least squares reweighted to even out the relative error, 5e-8 at most over
// [0, 15] (from 14.2 on Q is below fp32's range).  8000 x 2560 by 2560 x 2560 with fp32
// results 168 us (165 by gelu(), 187 by the library's erfcf); for 16-bit ones, 21664 x
// 2560 by 10240 x 2560 938 (915 by gelu()) and the norm of 4 x 921600 x 128 544 (510).
__device__ __forceinline__ float gelu_fp32(float x) {
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(x), 0.35f, 1.f));
    float p = -0.0291635804f;
    p = fmaf(p, t, 0.144059241f);
    p = fmaf(p, t, -0.255898863f);
    p = fmaf(p, t, 0.159389779f);
    p = fmaf(p, t, -0.0232618768f);
    p = fmaf(p, t, 0.105574057f);
    p = fmaf(p, t, 0.11981567f);
    p = fmaf(p, t, 0.139864311f);
    p = fmaf(p, t, 0.139621258f);
    const float q = p * t * __builtin_amdgcn_exp2f(x * x * (-0.5f * 1.4426950408889634f));   // Q(|x|)
    return fmaf(-fabsf(fminf(x, __FLT_MAX__)), q, fmaxf(x, 0.f));   // (infinities as in gelu)
}

// FP32: of a result that keeps 32 bits
template <bool FP32>
__device__ __forceinline__ float activate(float x, int act) {
    if (act == S2_ACT_SILU) return silu_f32(x);
    if (act == S2_ACT_GELU) return FP32 ? gelu_fp32(x) : gelu(x);
    if (act == S2_ACT_GELU_TANH) return gelu_tanh_f32(x);
    return x;
}

// f(std::integral_constant<int, act>): one branch around a loop, instead of branches
// at each of its values, whose code a short kernel would spend its time fetching
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
    if (act == S2_ACT_NONE)
        f(std::integral_constant<int, S2_ACT_NONE>{});
    else if (act == S2_ACT_GELU)
        f(std::integral_constant<int, S2_ACT_GELU>{});
    else if (act == S2_ACT_SILU)
        f(std::integral_constant<int, S2_ACT_SILU>{});
    else
        f(std::integral_constant<int, S2_ACT_GELU_TANH>{});
}

}  // namespace s2
