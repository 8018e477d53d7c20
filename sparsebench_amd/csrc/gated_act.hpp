// The activations of the gated experts, H = a(G) U, and their slopes.
//
//   SB_ACT_SILU  a(g) = g s,       a'(g) = s (1 + g (1 - s)),  s = 1 / (1 + e^-g)
//   SB_ACT_GELU  a(g) = g Phi(g),  a'(g) = Phi(g) + g phi(g)   (the erf form)
//
// In fp32. s is one exp2 and one reciprocal (each to 1 ulp); Phi comes from
// the erfc of gelu_erf_fast (to 1.5e-7), and phi(g) = e^(-g^2 / 2) / sqrt(2 pi)
// from the exp2 that it computes anyway.
#pragma once

#include "gelu.hpp"

namespace sb {

struct ActSlope {
  float value, slope;
};

template <int ACT>
__device__ __forceinline__ float gated_act(float g) {
  if constexpr (ACT == SB_ACT_SILU) return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g));
  else return gelu_erf_fast(g);
}

template <int ACT>
__device__ __forceinline__ ActSlope gated_act_slope(float g) {
  if constexpr (ACT == SB_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g));
    return {g * s, s * fmaf(g, 1.0f - s, 1.0f)};
  } else {
    // As gelu_erf_fast: a = |g| sqrt(log2(e) / 2), e2 = 2^(-a^2) = e^(-g^2 / 2),
    // q t e2 = erfc(|g| / sqrt 2) / (2 sqrt(log2(e) / 2)).
    const float a = fabsf(g) * 0.8493218002880191f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.2727374808792225f, a, 1.0f));
    float q = fmaf(0.6248546950284685f, t, -0.8554778804142388f);
    q = fmaf(q, t, 0.8367933923973075f);
    q = fmaf(q, t, -0.1674846541696695f);
    q = fmaf(q, t, 0.1500194578271646f);
    const float e2 = __builtin_amdgcn_exp2f(-(a * a));
    const float tail = q * t * e2 * 0.8493218002880191f;  // Phi(-|g|)
    const float cdf = g < 0.0f ? tail : 1.0f - tail;
    return {g * cdf, fmaf(g * 0.3989422804014327f, e2, cdf)};
  }
}

}  // namespace sb
