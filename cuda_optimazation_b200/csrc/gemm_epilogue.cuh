// gemm_epilogue.cuh -- the fused epilogue of the block-scaled GEMM, on 32
// consecutive columns of one output row held by one thread:
//   z = alpha acc + bias,  y = act(z) (or silu(gate) * factor),  out = y + residual,
// out in fp32, bf16 or MXFP8, and optionally z itself as an MXFP8 checkpoint.
// All of it is fp32; each output is rounded once, at its store.  A thread's
// 32 columns are one MX block, so its amax needs no other lane.  In the pair kernel
// it overlaps the next tile's products: 4096 x 28672 x 4096 gated with MXFP8 output and
// checkpoint takes 374-390 us, the plain GEMM of that shape with bf16 output 366-371.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "qg_act.cuh"
#include "qg_codec.cuh"
#include "qg_gemm.h"

namespace qg {

// bias[col] (0 without one, or beyond it).
__device__ __forceinline__ float epi_bias(const EpiParams& e, int col, int n) {
  if (!e.bias || col >= n) return 0.0f;
  return e.bias_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(e.bias)[col])
                     : static_cast<const float*>(e.bias)[col];
}

// z = alpha acc + bias of 32 columns, in place; lane j of the warp holds the
// bias of column j for all of them.
__device__ __forceinline__ void epi_affine(const EpiParams& e, float (&z)[32], float alpha,
                                           float bias) {
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    const float2 t = mul2(make_float2(z[j], z[j + 1]), both(alpha));
    z[j] = t.x;
    z[j + 1] = t.y;
  }
  if (e.bias) {
#pragma unroll
    for (int j = 0; j < 32; ++j) z[j] += __shfl_sync(0xffffffffu, bias, j);
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

// One MX block of an MXFP8 matrix with n columns: its scale goes to `sf`, its 32
// value bytes to w.  Rows and columns of the last scale chunks that lie beyond
// the matrix get code 0.
__device__ __forceinline__ void epi_quantise(const float (&v)[32], uint8_t* sf, int layout,
                                             int row_blocks, int sf_blocks, int row, int col0,
                                             int m, int n, uint32_t (&w)[8]) {
  const bool in = row < m && col0 < n;
  float amax = 0.0f, mul;
#pragma unroll
  for (int j = 0; j < 32; j += 2) amax = max3_abs(amax, v[j], v[j + 1]);
  const uint32_t code = mxfp8_scale_code(in ? amax : 0.0f, mul);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 a = mul2(make_float2(v[4 * i], v[4 * i + 1]), both(mul));
    const float2 b = mul2(make_float2(v[4 * i + 2], v[4 * i + 3]), both(mul));
    w[i] = cvt_e4m3x4(a.x, a.y, b.x, b.y);
  }
  if (layout == 0) {
    if (in) sf[static_cast<int64_t>(row) * (n / 32) + col0 / 32] = static_cast<uint8_t>(code);
  } else if (row < row_blocks * 128 && col0 / 32 < sf_blocks * 4) {
    sf[mma_scale_offset(row, col0 / 32, row_blocks, sf_blocks, layout)] =
        static_cast<uint8_t>(code);
  }
}

// The residual of 32 columns of a row of 16-byte aligned rows, fetched ahead of its
// use.
struct EpiResidual {
  uint4 v[8];
};
__device__ __forceinline__ void epi_fetch_residual(const EpiParams& e, EpiResidual& r, int row,
                                                   int col0, int m, int n) {
  if (!e.res || row >= m || col0 + 32 > n) return;
  const uint8_t* at =
      static_cast<const uint8_t*>(e.res) + (row * e.ldr + col0) * (e.res_bf16 ? 2 : 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = __ldg(reinterpret_cast<const uint4*>(at) + i);
  if (!e.res_bf16) {
#pragma unroll
    for (int i = 4; i < 8; ++i) r.v[i] = __ldg(reinterpret_cast<const uint4*>(at) + i);
  }
}
__device__ __forceinline__ void epi_add_residual(const EpiParams& e, const EpiResidual& r,
                                                 float (&y)[32], int row, int col0, int m, int n) {
  if (!e.res || row >= m || col0 >= n) return;
  if (col0 + 32 > n) {  // the last columns of a row
    const int64_t at = row * e.ldr + col0;
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (col0 + j < n)
        y[j] += e.res_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(e.res)[at + j])
                           : static_cast<const float*>(e.res)[at + j];
  } else if (e.res_bf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w[4] = {r.v[i].x, r.v[i].y, r.v[i].z, r.v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[8 * i + 2 * j] += __uint_as_float(w[j] << 16);
        y[8 * i + 2 * j + 1] += __uint_as_float(w[j] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[4 * i] += __uint_as_float(r.v[i].x);
      y[4 * i + 1] += __uint_as_float(r.v[i].y);
      y[4 * i + 2] += __uint_as_float(r.v[i].z);
      y[4 * i + 3] += __uint_as_float(r.v[i].w);
    }
  }
}

// The same for rows that start anywhere: the warp fetches its 32 rows at once, a
// lane a column, and turns them in 4 KB of its shared memory.  Places beyond the
// matrix read its last row or column (and are never stored): no load is
// conditional, so that none waits for another.  bf16 arrives as raw bits.
__device__ __forceinline__ void epi_fetch_rows(const EpiParams& e, uint32_t (&v)[32], int row0,
                                               int col0, int m, int n) {
  if (!e.res) return;
  const int col = min(col0 + static_cast<int>(threadIdx.x & 31), n - 1);
  if (e.res_bf16) {
    const uint16_t* at = static_cast<const uint16_t*>(e.res) + col;
#pragma unroll
    for (int r = 0; r < 32; ++r) v[r] = at[min(row0 + r, m - 1) * e.ldr];
  } else {
    const uint32_t* at = static_cast<const uint32_t*>(e.res) + col;
#pragma unroll
    for (int r = 0; r < 32; ++r) v[r] = at[min(row0 + r, m - 1) * e.ldr];
  }
}
__device__ __forceinline__ void epi_add_rows(const EpiParams& e, const uint32_t (&v)[32],
                                             float (&y)[32], float* turn) {
  if (!e.res) return;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int r = 0; r < 32; ++r)
    turn[r * 32 + (lane ^ r)] = __uint_as_float(e.res_bf16 ? v[r] << 16 : v[r]);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 32; ++j) y[j] += turn[lane * 32 + (j ^ lane)];
  __syncwarp();
}

// 32 values as 16 words of bf16.
__device__ __forceinline__ void epi_pack(const float (&y)[32], uint32_t (&w)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
}

// Output rows that TMA cannot store (not 16-byte aligned): turned in the warp's
// shared memory, then stored one by one, a lane a column.
__device__ __forceinline__ void epi_store_turned(const EpiParams& e, const float (&y)[32], int row,
                                                 int col0, int m, int n, float* turn) {
  const int lane = threadIdx.x & 31, row0 = row - lane;
#pragma unroll
  for (int j = 0; j < 32; ++j) turn[lane * 32 + (j ^ lane)] = y[j];
  __syncwarp();
  const bool in = col0 + lane < n;
  const int64_t first = row0 * e.ldc + col0 + lane;
  if (e.out_kind == kEpiBf16) {
    __nv_bfloat16* at = static_cast<__nv_bfloat16*>(e.out) + first;
#pragma unroll
    for (int r = 0; r < 32; ++r)
      if (in && row0 + r < m) at[r * e.ldc] = __float2bfloat16_rn(turn[r * 32 + (lane ^ r)]);
  } else {
    float* at = static_cast<float*>(e.out) + first;
#pragma unroll
    for (int r = 0; r < 32; ++r)
      if (in && row0 + r < m) at[r * e.ldc] = turn[r * 32 + (lane ^ r)];
  }
  __syncwarp();
}

}  // namespace qg
