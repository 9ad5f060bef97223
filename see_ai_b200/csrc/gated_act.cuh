// The activations of the gated block and their slopes, through the hardware's exponential and reciprocal: relative errors of
// a few 2^-22, below the steps of the 16-bit results.  A value that is not finite stays visible (ReLU keeps a NaN too).
#ifndef SEE_CUDA_GATED_ACT_CUH_
#define SEE_CUDA_GATED_ACT_CUH_

#include "act_expr.cuh"

namespace see::k {

// 1 / (1 + e^-x)
__device__ __forceinline__ float FastSigmoid(float x) { return RcpApprox(1.0f + Ex2Approx(x * -1.4426950408889634f)); }

template <int kAct> __device__ __forceinline__ float GatedAct(float g) {
  if constexpr (kAct == kActRelu) return g <= 0.0f ? 0.0f : g;
  if constexpr (kAct == kActGelu) return GeluExpr(g);
  return g * FastSigmoid(g);
}
template <int kAct> __device__ __forceinline__ void GatedActAndSlope(float g, float& value, float& slope) {
  if constexpr (kAct == kActRelu) {
    value = g <= 0.0f ? 0.0f : g;
    slope = g > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (kAct == kActGelu) {
    value = GeluExpr(g);
    slope = GeluGrad(1.0f, g);
  } else {
    const float s = FastSigmoid(g);
    value = g * s;
    slope = s * (1.0f + g * (1.0f - s));
  }
}

}  // namespace see::k

#endif  // SEE_CUDA_GATED_ACT_CUH_
