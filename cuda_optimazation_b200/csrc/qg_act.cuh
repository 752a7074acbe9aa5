// qg_act.cuh -- activations of the fused GEMM epilogue and their derivatives.
//
// All of them are built on the logistic function p(v) = 1 / (1 + exp(-v)):
//   silu(z)  = z p(z),                 silu'(z) = p (1 + z (1 - p))
//   gelu(z)  = z p(v), v = 2 sqrt(2/pi) (z + 0.044715 z^3)   (the tanh form:
//              (1 + tanh(v/2)) / 2 = p(v), without its cancellation at z < 0)
//   gelu'(z) = p (1 + z (1 - p) v'(z))
//   swiglu(g, u) = silu(g) u
// exp2 and the reciprocal are the hardware's approximations (good to about
// 2^-22 and 1 ulp); the denominators lie in [1, inf], where an infinite one
// gives 0 as the limit does.
#pragma once
#include <cuda_runtime.h>

#include "qg_codec.cuh"

namespace qg {

enum : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActSwiglu = 4 };

// Columns of a gate block; its factors are the kGateCols columns after it.
constexpr int kGateCols = 128;

constexpr float kGeluC = 1.5957691216057308f;   // 2 sqrt(2 / pi)
constexpr float kGeluC3 = 0.07135481282636f;    // 0.044715 * kGeluC

__device__ __forceinline__ float logistic(float v) {
  float e, p;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(1.0f + e));
  return p;
}

__device__ __forceinline__ float gelu_arg(float z) { return z * fmaf(kGeluC3, z * z, kGeluC); }

template <int kAct>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (kAct == kActRelu) return z > 0.0f ? z : (z == z ? 0.0f : z);
  if constexpr (kAct == kActSilu) return z * logistic(z);
  if constexpr (kAct == kActGelu) return z * logistic(gelu_arg(z));
  return z;
}

// d act'(z) of relu at two values: 0 at z <= 0 whatever d is there (a product with the
// slope would make a NaN of an infinite d), NaN where z is.
__device__ __forceinline__ float relu_grad(float d, float z) {
  return z > 0.0f ? d : (z <= 0.0f ? 0.0f : z);
}
__device__ __forceinline__ float2 relu_grad2(float2 d, float2 z) {
  return make_float2(relu_grad(d.x, z.x), relu_grad(d.y, z.y));
}

// The slopes of silu and gelu at two values.  Beyond +-128 every one is 0 or 1 to fp32; that bound
// keeps 0 * inf out (and NaN in).  Pairs take half the instructions of the
// polynomial: backward of 8192 x 14336 gelu 152.9 us one by one, 136.6 in pairs.
__device__ __forceinline__ float bounded(float z) {
  asm("min.NaN.f32 %0, %0, 0f43000000;\n\tmax.NaN.f32 %0, %0, 0fC3000000;" : "+f"(z));
  return z;
}
template <int kAct>
__device__ __forceinline__ float2 act_slope2(float2 z) {
  static_assert(kAct == kActSilu || kAct == kActGelu, "the others need no slope");
  const float2 one = both(1.0f);
  z = make_float2(bounded(z.x), bounded(z.y));
  if constexpr (kAct == kActSilu) {
    const float2 p = make_float2(logistic(z.x), logistic(z.y));
    return mul2(p, fma2(z, fma2(p, both(-1.0f), one), one));
  }
  const float2 zz = mul2(z, z);
  const float2 v = mul2(z, fma2(both(kGeluC3), zz, both(kGeluC)));
  const float2 p = make_float2(logistic(v.x), logistic(v.y));
  const float2 dv = fma2(both(3.0f * kGeluC3), zz, both(kGeluC));
  return mul2(p, fma2(mul2(z, fma2(p, both(-1.0f), one)), dv, one));
}

// Two gates g, factors u and output gradients d at a time:
// dg = d u silu'(g), du = d silu(g).
__device__ __forceinline__ void gated_grad2(float2 d, float2 g, float2 u, float2& dg, float2& du) {
  const float2 p = make_float2(logistic(g.x), logistic(g.y));
  const float2 gp = mul2(g, p);
  const float2 slope = fma2(gp, fma2(p, both(-1.0f), both(1.0f)), p);
  dg = mul2(mul2(d, u), slope);
  du = mul2(d, gp);
}

}  // namespace qg
