// act_backward.cu -- 8-bit activation checkpoints in the backward pass: the
// gradient of an activation from the MXFP8 checkpoint of its input, quantised
// for both of the products that follow, and an MXFP8 matrix turned for the
// weight gradient.
//
// With z the checkpoint's value and d the gradient of the activation's output:
//   dz = d act'(z), or for gate and factor columns (g, u) of the gated form
//   dg = d u silu'(g),  du = d silu(g).
// dz (fp32, never stored) is written twice: as MXFP8 along n (the A operand of
// the input gradient, K = n) and, turned, as MXFP8 along m (the A operand of
// the weight gradient, K = m filled up to a multiple of 32 with zeros), each
// with the block scales of its own direction; its column sums are dbias.
//
// Bound by HBM: 1 + 2 x 33/32 bytes an element of z, and d's.  A CTA owns 128 rows x
// 128 columns (the gated form: 128 gate columns and their 128 factors), which is
// exactly one 512-byte scale chunk of each output.  Warp w takes columns
// [32 w, 32 w + 32) in four steps of 32 rows; of such a 32 x 32 block a lane
// holds 4 consecutive rows x 8 consecutive columns, so that row blocks are
// joined over 4 lanes, column blocks over the 8 others, a lane's bytes of a row
// are 8 neighbours and those of a column 4, and no value passes through
// shared memory.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "qg_act.cuh"
#include "qg_codec.cuh"
#include "qg_gemm.h"

namespace qg {

namespace {

constexpr int kTile = 128;  // rows, and columns of a set, of a CTA

template <bool kBf16>
__device__ __forceinline__ void load_grad8(const void* base, int64_t elem, float (&v)[8]) {
  if constexpr (kBf16) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(
        static_cast<const __nv_bfloat16*>(base) + elem));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + elem);
    const float4 a = __ldg(p), b = __ldg(p + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
}

// Eight consecutive values of an MXFP8 matrix of row length n.
__device__ __forceinline__ void load_mx8(const uint8_t* q, const uint8_t* sf, int layout,
                                         int64_t row, int64_t col, int64_t n, int64_t row_blocks,
                                         int64_t sf_blocks, float (&v)[8]) {
  const uint2 w = __ldg(reinterpret_cast<const uint2*>(q + row * n + col));
  const int64_t so = layout == 0
                         ? row * (n / 32) + col / 32
                         : mma_scale_offset(row, col / 32, row_blocks, sf_blocks, layout);
  const float s = e8m0_decode(__ldg(sf + so));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = e4m3x2_decode((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
    v[2 * i] = f.x * s;
    v[2 * i + 1] = f.y * s;
  }
}

// kAct < 0: z itself (the transposition).
template <int kAct, bool kBf16>
__global__ void __launch_bounds__(128) act_backward_kernel(const ActBackwardParams p) {
  constexpr int kSets = kAct == kActSwiglu ? 2 : 1;
  __shared__ uint4 row_sf[kSets][32], col_sf[kSets][32];  // one 512-byte chunk each
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rg = lane >> 2, cg = lane & 3;
  const int64_t col_tiles = (p.n + kSets * kTile - 1) / (kSets * kTile);
  const int64_t tm = blockIdx.x / col_tiles, tc = blockIdx.x % col_tiles;
  const int64_t m0 = tm * kTile;
  // This lane's first column of z (of the gate set) and of dout.
  const int64_t zc = tc * kSets * kTile + warp * 32 + cg * 8;
  const int64_t dc = tc * kTile + warp * 32 + cg * 8;
  const int64_t row_blocks = (p.m + 127) / 128, n_blocks = (p.n + 127) / 128;
  const int64_t sf_blocks = (p.n / 32 + 3) / 4, t_blocks = (p.mt / 32 + 3) / 4;
  for (int i = threadIdx.x; i < kSets * 32; i += blockDim.x) {
    row_sf[i / 32][i % 32] = make_uint4(0, 0, 0, 0);
    col_sf[i / 32][i % 32] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  float sum[kSets][8];
#pragma unroll
  for (int s = 0; s < kSets; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[s][j] = 0.0f;
  if (zc < p.n) {  // p.n is a multiple of 32: a warp is in or out as a whole
    for (int rb = 0; rb < 4 && m0 + rb * 32 < p.m; ++rb) {
      float v[kSets][4][8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t row = m0 + rb * 32 + rg * 4 + i;
        if (row < p.m) {
          float d[8];
          if constexpr (kAct >= 0) load_grad8<kBf16>(p.dout, row * p.ldd + dc, d);
          if constexpr (kAct == kActNone) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[0][i][j] = d[j];
          } else {
            load_mx8(p.z_q, p.z_sf, p.z_layout, row, zc, p.n, row_blocks, sf_blocks, v[0][i]);
            if constexpr (kAct == kActSwiglu) {
              load_mx8(p.z_q, p.z_sf, p.z_layout, row, zc + kTile, p.n, row_blocks, sf_blocks,
                       v[1][i]);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float g = v[0][i][j], u = v[1][i][j];
                v[0][i][j] = d[j] * u * act_slope<kActSilu>(g);
                v[1][i][j] = d[j] * act_fwd<kActSilu>(g);
              }
            } else if constexpr (kAct > 0) {
#pragma unroll
              for (int j = 0; j < 8; ++j) v[0][i][j] = d[j] * act_slope<kAct>(v[0][i][j]);
            }
          }
        } else {
#pragma unroll
          for (int s = 0; s < kSets; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[s][i][j] = 0.0f;
        }
      }
#pragma unroll
      for (int s = 0; s < kSets; ++s) {
        if constexpr (kAct >= 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(v[s][i][j]));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            float mul;
            const uint32_t code = mxfp8_scale_code(amax, mul);
            const int64_t row = m0 + rb * 32 + rg * 4 + i;
            if (row < p.m)
              *reinterpret_cast<uint2*>(p.dz_q + row * p.n + zc + s * kTile) = make_uint2(
                  cvt_e4m3x4(v[s][i][0] * mul, v[s][i][1] * mul, v[s][i][2] * mul,
                             v[s][i][3] * mul),
                  cvt_e4m3x4(v[s][i][4] * mul, v[s][i][5] * mul, v[s][i][6] * mul,
                             v[s][i][7] * mul));
            if (cg == 0)
              reinterpret_cast<uint8_t*>(row_sf[s])[(rg * 4 + i) * 16 + rb * 4 + warp] =
                  static_cast<uint8_t>(code);
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float amax = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(v[s][i][j]));
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 4));
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 8));
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 16));
          float mul;
          const uint32_t code = mxfp8_scale_code(amax, mul);
          *reinterpret_cast<uint32_t*>(p.dzt_q + (zc + s * kTile + j) * p.mt + m0 + rb * 32 +
                                       rg * 4) =
              cvt_e4m3x4(v[s][0][j] * mul, v[s][1][j] * mul, v[s][2][j] * mul, v[s][3][j] * mul);
          if (rg == j)
            reinterpret_cast<uint8_t*>(col_sf[s])[(cg * 8 + j) * 16 + warp * 4 + rb] =
                static_cast<uint8_t>(code);
          if constexpr (kAct >= 0)
            sum[s][j] += (v[s][0][j] + v[s][1][j]) + (v[s][2][j] + v[s][3][j]);
        }
      }
    }
    if constexpr (kAct >= 0) {
      if (p.dbias_part) {
#pragma unroll
        for (int s = 0; s < kSets; ++s) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            sum[s][j] += __shfl_xor_sync(0xffffffffu, sum[s][j], 4);
            sum[s][j] += __shfl_xor_sync(0xffffffffu, sum[s][j], 8);
            sum[s][j] += __shfl_xor_sync(0xffffffffu, sum[s][j], 16);
            if (rg == j) p.dbias_part[tm * p.n + zc + s * kTile + j] = sum[s][j];
          }
        }
      }
    }
  }
  __syncthreads();
  // Whole chunks: what lies beyond the matrix reads as zero scales.
  if (warp < kSets) {
    const int64_t br = tm, bs = tc * kSets + warp;
    const int64_t chunk = p.out_layout == 1 ? bs * row_blocks + br : br * sf_blocks + bs;
    if constexpr (kAct >= 0)
      reinterpret_cast<uint4*>(p.dz_sf + chunk * 512)[lane] = row_sf[warp][lane];
  } else if (warp >= 2 && warp < 2 + kSets) {
    const int64_t br = tc * kSets + warp - 2, bs = tm;
    const int64_t chunk = p.out_layout == 1 ? bs * n_blocks + br : br * t_blocks + bs;
    reinterpret_cast<uint4*>(p.dzt_sf + chunk * 512)[lane] = col_sf[warp - 2][lane];
  }
}

template <int kAct>
void launch_act(const ActBackwardParams& p, bool bf16, int grid, cudaStream_t stream) {
  if (bf16) act_backward_kernel<kAct, true><<<grid, 128, 0, stream>>>(p);
  else act_backward_kernel<kAct, false><<<grid, 128, 0, stream>>>(p);
}

int act_grid(const ActBackwardParams& p, int sets) {
  return static_cast<int>(((p.m + kTile - 1) / kTile) *
                          ((p.n + sets * kTile - 1) / (sets * kTile)));
}

}  // namespace

cudaError_t launch_act_backward(const ActBackwardParams& p, int act, bool bf16,
                                cudaStream_t stream) {
  const int grid = act_grid(p, act == kActSwiglu ? 2 : 1);
  switch (act) {
    case kActNone: launch_act<kActNone>(p, bf16, grid, stream); break;
    case kActRelu: launch_act<kActRelu>(p, bf16, grid, stream); break;
    case kActSilu: launch_act<kActSilu>(p, bf16, grid, stream); break;
    case kActGelu: launch_act<kActGelu>(p, bf16, grid, stream); break;
    case kActSwiglu: launch_act<kActSwiglu>(p, bf16, grid, stream); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

cudaError_t launch_transpose_mxfp8(const ActBackwardParams& p, cudaStream_t stream) {
  act_backward_kernel<-1, false><<<act_grid(p, 1), 128, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace qg
