// The activations of a gated product and their slopes, in fp32.
#pragma once

#include "device_common.hpp"
#include "launch.hpp"

namespace cuvit::device {

using detail::Gate;

/// 1 / (1 + exp(-x)), 0 and 1 at the ends: exp2 and the reciprocal on the
/// transcendental unit, each within a unit in the last place. exp2's argument is
/// rounded to fp32 as well, which far below zero, where the result is about exp(x), is
/// |x| / 2 units of it: at -20 1e-6 of a sigmoid of 2e-9, so not worth a second product.
__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.0F + __builtin_amdgcn_exp2f(x * -1.44269504088896341F));
}

/// The tanh form of GELU as x sigmoid(2 u), since (1 + tanh u) / 2 = sigmoid(2 u),
/// with 2 u = 2 sqrt(2 / pi) (x + 0.044715 x^3).
__device__ __forceinline__ float gelu_tanh_argument(float x) {
    return x * fmaf(x * x, 0.07135481627260025F, 1.5957691216057308F);
}

template <Gate G> __device__ __forceinline__ float gate_value(float x) {
    if constexpr (G == Gate::kSilu) {
        return x * sigmoid(x);
    } else if constexpr (G == Gate::kGelu) {
        return gelu(x);
    } else {
        return x * sigmoid(gelu_tanh_argument(x));
    }
}

/// gate_value and its slope together; @p Fine takes the erf form's Phi from erfcf,
/// which fp32 results can tell from gelu's (4e-7 of it).
template <Gate G, bool Fine> __device__ __forceinline__ float gate_value(float x, float& slope) {
    if constexpr (G == Gate::kSilu) {
        const float s = sigmoid(x);
        slope = s * fmaf(x, 1.0F - s, 1.0F);
        return x * s;
    } else if constexpr (G == Gate::kGelu) {
        // Phi(x) + x phi(x).
        const float phi = 0.3989422804014327F * __builtin_amdgcn_exp2f(x * x * -0.72134752044448170F);
        const float cumulative = Fine ? 0.5F * erfcf(x * -0.70710678118654752F) : gelu<true>(x);
        slope = fmaf(x, phi, cumulative);
        return x * cumulative;
    } else {
        const float s = sigmoid(gelu_tanh_argument(x));
        // (Held finite: s (1 - s) is 0 long before, and 0 times infinity would be NaN.)
        const float argument_slope = fmaf(fminf(x * x, 1.0e30F), 0.21406444881780075F, 1.5957691216057308F);
        slope = fmaf(x * s * (1.0F - s), argument_slope, s);
        return x * s;
    }
}

} // namespace cuvit::device
