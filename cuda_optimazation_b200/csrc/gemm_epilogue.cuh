// gemm_epilogue.cuh -- the fused epilogue of the block-scaled GEMM, on 32
// consecutive columns of one output row held by one thread:
//   z = alpha acc + bias,  y = act(z) (or silu(gate) * factor),  out = y + residual,
// out in fp32, bf16 or MXFP8, and optionally z itself as an MXFP8 checkpoint.
// All of it is fp32; each output is rounded once, at its store.  A thread's
// 32 columns are one MX block, so its amax needs no other lane.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "qg_act.cuh"
#include "qg_codec.cuh"
#include "qg_gemm.h"

namespace qg {

// z of columns [col0, col0 + 32); lane j of the warp fetches bias[col0 + j]
// for all of them.
__device__ __forceinline__ void epi_affine(const EpiParams& e, const uint32_t (&acc)[32],
                                           float alpha, int col0, int n, int lane,
                                           float (&z)[32]) {
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    const float2 t = mul2(make_float2(__uint_as_float(acc[j]), __uint_as_float(acc[j + 1])),
                          both(alpha));
    z[j] = t.x;
    z[j + 1] = t.y;
  }
  if (e.bias) {
    float b = 0.0f;
    if (col0 + lane < n)
      b = e.bias_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(e.bias)[col0 + lane])
                      : static_cast<const float*>(e.bias)[col0 + lane];
#pragma unroll
    for (int j = 0; j < 32; ++j) z[j] += __shfl_sync(0xffffffffu, b, j);
  }
}

template <int kAct>
__device__ __forceinline__ void epi_act_all(float (&z)[32]) {
#pragma unroll
  for (int j = 0; j < 32; ++j) z[j] = act_fwd<kAct>(z[j]);
}

__device__ __forceinline__ void epi_act(int act, float (&z)[32]) {
  if (act == kActRelu) epi_act_all<kActRelu>(z);
  else if (act == kActSilu) epi_act_all<kActSilu>(z);
  else if (act == kActGelu) epi_act_all<kActGelu>(z);
}

// One MX block of an MXFP8 matrix with n columns: 32 value bytes and its scale.
// Rows and columns of the last scale chunks that lie beyond the matrix get
// code 0.
__device__ __forceinline__ void epi_store_mx(const float (&v)[32], uint8_t* q, uint8_t* sf,
                                             int layout, int row_blocks, int sf_blocks, int row,
                                             int col0, int m, int n) {
  const bool in = row < m && col0 < n;
  uint32_t code = 0;
  if (in) {
    float amax = 0.0f, mul;
#pragma unroll
    for (int j = 0; j < 32; j += 2) amax = max3_abs(amax, v[j], v[j + 1]);
    code = mxfp8_scale_code(amax, mul);
    uint4* dst = reinterpret_cast<uint4*>(q + static_cast<int64_t>(row) * n + col0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 16 * h + 4 * i;
        const float2 a = mul2(make_float2(v[j], v[j + 1]), both(mul));
        const float2 b = mul2(make_float2(v[j + 2], v[j + 3]), both(mul));
        w[i] = cvt_e4m3x4(a.x, a.y, b.x, b.y);
      }
      dst[h] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (layout == 0) {
    if (in) sf[static_cast<int64_t>(row) * (n / 32) + col0 / 32] = static_cast<uint8_t>(code);
  } else if (row < row_blocks * 128 && col0 / 32 < sf_blocks * 4) {
    sf[mma_scale_offset(row, col0 / 32, row_blocks, sf_blocks, layout)] =
        static_cast<uint8_t>(code);
  }
}

// y += residual (n: the output's columns).
__device__ __forceinline__ void epi_residual(const EpiParams& e, float (&y)[32], int row, int col0,
                                             int m, int n) {
  const bool full = col0 + 32 <= n;
  if (e.res && row < m && col0 < n) {
    const int64_t at = row * e.ldr + col0;
    if (e.res_bf16) {
      const __nv_bfloat16* r = static_cast<const __nv_bfloat16*>(e.res) + at;
      if (full && e.res_vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 a = __ldg(reinterpret_cast<const uint4*>(r) + i);
          const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            y[8 * i + 2 * j] += __uint_as_float(w[j] << 16);
            y[8 * i + 2 * j + 1] += __uint_as_float(w[j] & 0xffff0000u);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (col0 + j < n) y[j] += __bfloat162float(r[j]);
      }
    } else {
      const float* r = static_cast<const float*>(e.res) + at;
      if (full && e.res_vec) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 a = __ldg(reinterpret_cast<const float4*>(r) + i);
          y[4 * i] += a.x;
          y[4 * i + 1] += a.y;
          y[4 * i + 2] += a.z;
          y[4 * i + 3] += a.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (col0 + j < n) y[j] += r[j];
      }
    }
  }
}

// 32 values as 16 words of bf16.
__device__ __forceinline__ void epi_pack(const float (&y)[32], uint32_t (&w)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
}

// The output, straight to global memory.
__device__ __forceinline__ void epi_store(const EpiParams& e, const float (&y)[32], int row,
                                          int col0, int m, int n) {
  const bool in = row < m && col0 < n;
  const bool full = col0 + 32 <= n;
  if (e.out_kind == kEpiMxfp8) {
    epi_store_mx(y, static_cast<uint8_t*>(e.out), e.out_sf, e.out_layout, e.row_blocks,
                 e.out_sf_blocks, row, col0, m, n);
  } else if (in) {
    const int64_t at = row * e.ldc + col0;
    if (e.out_kind == kEpiBf16) {
      __nv_bfloat16* c = static_cast<__nv_bfloat16*>(e.out) + at;
      if (full && e.out_vec) {
        uint32_t w[16];
        epi_pack(y, w);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          reinterpret_cast<uint4*>(c)[i] =
              make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (col0 + j < n) c[j] = __float2bfloat16_rn(y[j]);
      }
    } else {
      float* c = static_cast<float*>(e.out) + at;
      if (full && e.out_vec) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          reinterpret_cast<float4*>(c)[i] =
              make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (col0 + j < n) c[j] = y[j];
      }
    }
  }
}

__device__ __forceinline__ void epi_checkpoint(const EpiParams& e, const float (&z)[32], int row,
                                               int col0, int m, int n) {
  if (e.z_q)
    epi_store_mx(z, e.z_q, e.z_sf, e.z_layout, e.row_blocks, e.z_sf_blocks, row, col0, m, n);
}

}  // namespace qg
