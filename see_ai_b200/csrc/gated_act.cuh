// The activations of the gated block and their slopes, through the hardware's exponential and reciprocal, as products of factors
// that keep their own relative accuracy: what is small far from zero is as good as what is large.  The exponential of e is
// off by at most 7 |e| 2^-24, and 2^-22 beside that: 2^-17 of GELU where f16's range ends (g = -5.2), 2^-14.7 where bf16's does
// (g = -10), in either type a thirtieth of half a step.  (SiLU's slope takes 1 - s as it stands, a rounding of s.)  A sigmoid below
// 2^-126 is zero.  A value that is not finite stays visible (ReLU keeps a NaN too).
#ifndef SEE_CUDA_GATED_ACT_CUH_
#define SEE_CUDA_GATED_ACT_CUH_

#include "act_expr.cuh"

namespace see::k {

// 1 / (1 + e^-x)
__device__ __forceinline__ float FastSigmoid(float x) { return RcpApprox(1.0f + Ex2Approx(x * -1.4426950408889634f)); }

// GELU as g s, s = 1 / (1 + E), E = e^-2u, u = c (g + a g^3).  (The plans' g - g r, with r = 1 - s, cancels below zero: tenths of a percent off at
// g = -4, nothing left from -5.2 on.)  Its slope is s + g s (1 - s) 2u', and 1 - s is E s.
__device__ __forceinline__ float GeluExponential(float g, float g2) {
  return Ex2Approx(g * __fmaf_rn(g2, kGeluExprC * kGeluExprA, kGeluExprC) * -kTwoLog2E);
}
__device__ __forceinline__ float GatedGelu(float g) { return g * RcpApprox(1.0f + GeluExponential(g, g * g)); }
__device__ __forceinline__ void GatedGeluAndSlope(float g, float& value, float& slope) {
  const float g2 = g * g, e = GeluExponential(g, g2), s = RcpApprox(1.0f + e);
  value = g * s;
  const float both = e * s * s;   // s (1 - s); at either end 0, or infinity times 0
  slope = s + (both > 0.0f ? g * both * __fmaf_rn(g2, 6.0f * kGeluExprC * kGeluExprA, 2.0f * kGeluExprC) : 0.0f);
}

template <int kAct> __device__ __forceinline__ float GatedAct(float g) {
  if constexpr (kAct == kActRelu) return g <= 0.0f ? 0.0f : g;
  if constexpr (kAct == kActGelu) return GatedGelu(g);
  return g * FastSigmoid(g);
}
template <int kAct> __device__ __forceinline__ void GatedActAndSlope(float g, float& value, float& slope) {
  if constexpr (kAct == kActRelu) {
    value = g <= 0.0f ? 0.0f : g;
    slope = g > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (kAct == kActGelu) {
    GatedGeluAndSlope(g, value, slope);
  } else {
    const float s = FastSigmoid(g);
    value = g * s;
    slope = s * (1.0f + g * (1.0f - s));
  }
}

}  // namespace see::k

#endif  // SEE_CUDA_GATED_ACT_CUH_
