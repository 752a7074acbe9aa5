// rmsnorm.cu -- RMS norm with the residual's addition and MXFP8 output, and
// its gradient.
//
// Forward, per row of k values:   h = x + residual,
//   rstd = (mean h^2 + eps)^-1/2,  y = h * rstd * w,
// written as the MXFP8 operand that the next block-scaled product reads
// (qg_quantize_mxfp8's rule on y, one ue8m0 scale per 32 values), h in x's
// type and rstd in fp32.  The sum and the statistics are fp32; h is rounded
// once, for the store, and y is formed from the unrounded h.
//
// Backward (the quantisation passed straight through), with xh = h * rstd and
// g = dy * w:   dx = rstd (g - xh mean(g xh)) + dres,   dw = sum_rows dy xh.
//
// Both are bound by HBM: 7 bytes an element forward (bf16 with a residual), 8
// backward.  A row lives in its CTA's registers between the reduction and the
// output, so every byte crosses HBM once.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "qg_codec.cuh"
#include "qg_gemm.h"

namespace qg {

namespace {

// Eight consecutive values as fp32 (16 bytes of bf16 or 32 of fp32).  kOnce: a
// row's own values, read once (streaming, and coherent: an output may be an
// input's own buffer); otherwise the weight, which every row reads again.
template <bool kBf16, bool kOnce = true>
__device__ __forceinline__ void load8(const void* base, int64_t elem, float (&v)[8]) {
  if constexpr (kBf16) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(base) + elem);
    const uint4 a = kOnce ? __ldcs(p) : __ldg(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + elem);
    const float4 a = kOnce ? __ldcs(p) : __ldg(p), b = kOnce ? __ldcs(p + 1) : __ldg(p + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
}

template <bool kBf16>
__device__ __forceinline__ void store8(void* base, int64_t elem, const float (&v)[8]) {
  if constexpr (kBf16) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(base) + elem) =
        make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + elem);
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// Sum over the CTA in a fixed order; every thread gets it.  `red` holds one
// float per warp and is free again after the next call's first barrier.
__device__ __forceinline__ float cta_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One CTA per row; thread t owns the 8-value vectors t, t + blockDim, ...
// (kVec of them at most), so four neighbouring lanes hold one 32-value MX
// block and sixteen one 4-byte word of scales.
template <bool kBf16, bool kWBf16, int kVec>
__global__ void __launch_bounds__(512) rmsnorm_mxfp8_kernel(const RmsNormParams p) {
  __shared__ float red[32];
  const int64_t row = blockIdx.x;
  const int nvec = static_cast<int>(p.k / 8);
  float h[kVec][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nvec) {
      load8<kBf16>(p.x, row * p.ldx + v * 8, h[i]);
      if (p.residual) {
        float r[8];
        load8<kBf16>(p.residual, row * p.ldr + v * 8, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] += r[j];
      }
      if (p.h) store8<kBf16>(p.h, row * p.ldh + v * 8, h[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(h[i][j], h[i][j], ss);
    }
  }
  ss = cta_sum(ss, red);
  const float rstd = rsqrtf(ss / static_cast<float>(p.k) + p.eps);
  if (threadIdx.x == 0 && p.rstd) p.rstd[row] = rstd;
  const int lane = threadIdx.x & 31;
  const int64_t sfk = p.k / 32;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    const bool in = v < nvec;
    float y[8];
    float amax = 0.0f;
    if (in) {
      float w[8];
      load8<kWBf16, false>(p.weight, v * 8, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = h[i][j] * rstd * w[j];
        amax = fmaxf(amax, fabsf(y[j]));
      }
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    float mul;
    const uint32_t code = mxfp8_scale_code(amax, mul);  // 0 beyond the row: padding
    if (in)
      *reinterpret_cast<uint2*>(p.q + row * p.k + v * 8) =
          make_uint2(cvt_e4m3x4(y[0] * mul, y[1] * mul, y[2] * mul, y[3] * mul),
                     cvt_e4m3x4(y[4] * mul, y[5] * mul, y[6] * mul, y[7] * mul));
    if (p.layout == 0) {
      if (in && (lane & 3) == 0) p.sf[row * sfk + v / 4] = static_cast<uint8_t>(code);
    } else {
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        word |= __shfl_sync(0xffffffffu, code, (lane & 16) + 4 * j) << (8 * j);
      if ((lane & 15) == 0 && in)
        *reinterpret_cast<uint32_t*>(
            p.sf + mma_scale_offset(row, v / 4, p.row_blocks, p.sf_blocks, p.layout)) = word;
    }
  }
  // The scale words of the rows that fill the last 128-row chunk read as 0;
  // the CTAs share them out.
  if (p.layout != 0) {
    const int64_t pad = (p.row_blocks * 128 - p.rows) * p.sf_blocks;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < pad;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
      const int64_t r = p.rows + i / p.sf_blocks, c = i % p.sf_blocks;
      *reinterpret_cast<uint32_t*>(
          p.sf + mma_scale_offset(r, 4 * c, p.row_blocks, p.sf_blocks, p.layout)) = 0u;
    }
  }
}

// CTA b takes rows b, b + grid, ...; each thread owns the same columns of all
// of them, so its share of dw stays in registers and is written once, to row b
// of the partial sums.
template <bool kBf16, bool kWBf16, int kVec>
__global__ void __launch_bounds__(512) rmsnorm_backward_kernel(const RmsNormBwdParams p) {
  __shared__ float red[32];
  const int nvec = static_cast<int>(p.k / 8);
  const float inv_k = 1.0f / static_cast<float>(p.k);
  float dw[kVec][8];
#pragma unroll
  for (int i = 0; i < kVec; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = 0.0f;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float rstd = __ldg(p.rstd + row);
    float g[kVec][8], xh[kVec][8];
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nvec) {
        float w[8];
        load8<kBf16>(p.dy, row * p.lddy + v * 8, g[i]);
        load8<kBf16>(p.h, row * p.ldh + v * 8, xh[i]);
        load8<kWBf16, false>(p.weight, v * 8, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          xh[i][j] *= rstd;
          dw[i][j] = fmaf(g[i][j], xh[i][j], dw[i][j]);
          g[i][j] *= w[j];
          dot = fmaf(g[i][j], xh[i][j], dot);
        }
      }
    }
    const float c = cta_sum(dot, red) * inv_k;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nvec) {
        float d[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = rstd * fmaf(-xh[i][j], c, g[i][j]);
        if (p.dres) {
          float r[8];
          load8<kBf16>(p.dres, row * p.lddres + v * 8, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) d[j] += r[j];
        }
        store8<kBf16>(p.dx, row * p.lddx + v * 8, d);
      }
    }
  }
  if (p.dw_part) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nvec) store8<false>(p.dw_part, blockIdx.x * p.k + v * 8, dw[i]);
    }
  }
}

// out[c] = sum over `parts` rows of part[.][c], in a fixed order: eight threads
// of a column sum every eighth row and are joined in shared memory.
__global__ void __launch_bounds__(256) column_sum_kernel(const float* part, int parts, int64_t k,
                                                         float* out) {
  __shared__ float sum[8][32];
  const int64_t c = blockIdx.x * 32ll + threadIdx.x;
  float s = 0.0f;
  if (c < k)
    for (int r = threadIdx.y; r < parts; r += 8) s += part[r * k + c];
  sum[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < k) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += sum[i][threadIdx.x];
    out[c] = s;
  }
}

// Threads per CTA and vectors per thread of a row of k values: whole warps,
// at most 512 threads until a thread would hold more than eight vectors.
struct RowShape {
  int threads, vec;
};
RowShape row_shape(int64_t k) {
  const int64_t nvec = k / 8;
  RowShape s{};
  for (s.vec = 1; s.vec < 8 && nvec > 512 * s.vec; s.vec *= 2) {
  }
  s.threads = static_cast<int>((nvec + s.vec - 1) / s.vec + 31) / 32 * 32;
  return s;
}

template <bool kBf16, bool kWBf16>
void launch_norm(const RmsNormParams& p, RowShape s, cudaStream_t stream) {
  const int grid = static_cast<int>(p.rows);
  if (s.vec == 1) rmsnorm_mxfp8_kernel<kBf16, kWBf16, 1><<<grid, s.threads, 0, stream>>>(p);
  else if (s.vec == 2) rmsnorm_mxfp8_kernel<kBf16, kWBf16, 2><<<grid, s.threads, 0, stream>>>(p);
  else if (s.vec == 4) rmsnorm_mxfp8_kernel<kBf16, kWBf16, 4><<<grid, s.threads, 0, stream>>>(p);
  else rmsnorm_mxfp8_kernel<kBf16, kWBf16, 8><<<grid, s.threads, 0, stream>>>(p);
}

template <bool kBf16, bool kWBf16>
void launch_norm_bwd(const RmsNormBwdParams& p, RowShape s, int grid, cudaStream_t stream) {
  if (s.vec == 1) rmsnorm_backward_kernel<kBf16, kWBf16, 1><<<grid, s.threads, 0, stream>>>(p);
  else if (s.vec == 2) rmsnorm_backward_kernel<kBf16, kWBf16, 2><<<grid, s.threads, 0, stream>>>(p);
  else if (s.vec == 4) rmsnorm_backward_kernel<kBf16, kWBf16, 4><<<grid, s.threads, 0, stream>>>(p);
  else rmsnorm_backward_kernel<kBf16, kWBf16, 8><<<grid, s.threads, 0, stream>>>(p);
}

}  // namespace

cudaError_t launch_rmsnorm_mxfp8(const RmsNormParams& p, bool bf16, bool w_bf16,
                                 cudaStream_t stream) {
  const RowShape s = row_shape(p.k);
  if (bf16) w_bf16 ? launch_norm<true, true>(p, s, stream) : launch_norm<true, false>(p, s, stream);
  else w_bf16 ? launch_norm<false, true>(p, s, stream) : launch_norm<false, false>(p, s, stream);
  return cudaGetLastError();
}

int rmsnorm_backward_parts(int64_t rows) {
  const int64_t most = 2ll * num_sms();
  return static_cast<int>(rows < most ? rows : most);
}

cudaError_t launch_rmsnorm_backward(const RmsNormBwdParams& p, bool bf16, bool w_bf16, float* dw,
                                    cudaStream_t stream) {
  const RowShape s = row_shape(p.k);
  const int grid = rmsnorm_backward_parts(p.rows);
  if (bf16)
    w_bf16 ? launch_norm_bwd<true, true>(p, s, grid, stream)
           : launch_norm_bwd<true, false>(p, s, grid, stream);
  else
    w_bf16 ? launch_norm_bwd<false, true>(p, s, grid, stream)
           : launch_norm_bwd<false, false>(p, s, grid, stream);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !dw) return e;
  return launch_column_sum(p.dw_part, grid, p.k, dw, stream);
}

cudaError_t launch_column_sum(const float* part, int parts, int64_t k, float* out,
                              cudaStream_t stream) {
  column_sum_kernel<<<static_cast<int>((k + 31) / 32), dim3(32, 8), 0, stream>>>(part, parts, k,
                                                                                out);
  return cudaGetLastError();
}

}  // namespace qg
