// qg_act.cuh -- activations of the fused GEMM epilogue and their derivatives.
//
// All of them are built on the logistic function p(v) = 1 / (1 + exp(-v)):
//   silu(z)  = z p(z),                 silu'(z) = p (1 + z (1 - p))
//   gelu(z)  = z p(v), v = 2 sqrt(2/pi) (z + 0.044715 z^3)   (the tanh form:
//              (1 + tanh(v/2)) / 2 = p(v), without its cancellation at z < 0)
//   gelu'(z) = p (1 + z (1 - p) v'(z))
//   swiglu(g, u) = silu(g) u
// exp and the quotient are CUDA's fast forms (2 ulp each); the denominators lie
// in [1, inf], where an infinite one gives 0 as the limit does.
#pragma once
#include <cuda_runtime.h>

namespace qg {

enum : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActSwiglu = 4 };

// Columns of a gate block; its factors are the kGateCols columns after it.
constexpr int kGateCols = 128;

constexpr float kGeluC = 1.5957691216057308f;   // 2 sqrt(2 / pi)
constexpr float kGeluC3 = 0.07135481282636f;    // 0.044715 * kGeluC

__device__ __forceinline__ float over_one_plus_exp(float num, float v) {
  return __fdividef(num, 1.0f + __expf(-v));
}

__device__ __forceinline__ float gelu_arg(float z) { return z * fmaf(kGeluC3, z * z, kGeluC); }

template <int kAct>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (kAct == kActRelu) return z > 0.0f ? z : (z == z ? 0.0f : z);
  if constexpr (kAct == kActSilu) return over_one_plus_exp(z, z);
  if constexpr (kAct == kActGelu) return over_one_plus_exp(z, gelu_arg(z));
  return z;
}

template <int kAct>
__device__ __forceinline__ float act_slope(float z) {
  // Beyond +-128 every slope is 0 or 1 to fp32; the bound keeps 0 * inf out.
  z = fabsf(z) > 128.0f ? copysignf(128.0f, z) : z;
  if constexpr (kAct == kActRelu) return z > 0.0f ? 1.0f : 0.0f;
  if constexpr (kAct == kActSilu) {
    const float p = over_one_plus_exp(1.0f, z);
    return p * fmaf(z, 1.0f - p, 1.0f);
  }
  if constexpr (kAct == kActGelu) {
    const float p = over_one_plus_exp(1.0f, gelu_arg(z));
    return p * fmaf(z * (1.0f - p), fmaf(3.0f * kGeluC3, z * z, kGeluC), 1.0f);
  }
  return 1.0f;
}

}  // namespace qg
