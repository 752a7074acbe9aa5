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
// Bytes: 1 + 2 x 33/32 an element of z, and d's.  A CTA owns 128 rows x 128
// columns (the gated form: 128 gate columns and their 128 factors), which is
// exactly one 512-byte scale chunk of each output.  A warp takes 32 x 32 blocks;
// of such a block a lane holds 4 consecutive rows x 8 consecutive columns, so
// that row blocks are joined over 4 lanes, column blocks over the 8 others, a
// lane's bytes of a row are 8 neighbours and those of a column 4, and no value
// passes through shared memory.
//
// What bounds it is the instruction rate as much as HBM, so the work per element
// is kept down: fp32 pairs in one instruction (f32x2), and block scales from the
// upper halves of the peaks' fp32 patterns, two peaks to a register -- a scale
// needs the exponent of its peak only, and the upper halves order as the
// peaks do.
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

// Eight consecutive values of an MXFP8 row with scale s.
__device__ __forceinline__ void load_mx8(const uint8_t* q, float s, float2 (&v)[4]) {
  const uint2 w = __ldg(reinterpret_cast<const uint2*>(q));
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = mul2(e4m3x2_decode((i < 2 ? w.x : w.y) >> (16 * (i & 1))), both(s));
}

// Larger of two pairs of 16-bit unsigned values.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }

// Upper halves of two non-negative floats' patterns: b's in the high half.
__device__ __forceinline__ uint32_t upper2(float a, float b) {
  return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
}
// Two peaks' upper halves -> their scale codes times 128 (one per half).
__device__ __forceinline__ uint32_t codes_x128(uint32_t peaks) {
  return max_u16x2(peaks & 0x7f807f80u, 0x04000400u) - 0x04000400u;
}
// Upper halves of the two reciprocal scales 2^(127 - code): (254 - code) << 7.
__device__ __forceinline__ uint32_t reciprocals(uint32_t codes128) {
  return 0x7f007f00u - codes128;
}
__device__ __forceinline__ float lower_half(uint32_t r) { return __uint_as_float(r << 16); }
__device__ __forceinline__ float upper_half(uint32_t r) {
  return __uint_as_float(r & 0xffff0000u);
}

// kAct < 0: z itself (the transposition).  kGroups: 32-row groups of the tile
// that are worked on at once, by four warps each.
template <int kAct, bool kBf16, int kGroups>
__global__ void __launch_bounds__(128 * kGroups) act_backward_kernel(const ActBackwardParams p) {
  constexpr int kSets = kAct == kActSwiglu ? 2 : 1;
  constexpr bool kGrad = kAct >= 0, kZ = kAct != kActNone;
  __shared__ uint4 row_sf[kSets][32], col_sf[kSets][32], z_sf[kSets][32];  // 512-byte chunks
  __shared__ float part[kGroups > 1 ? kGroups : 1][kSets * kTile];
  const int warp = (threadIdx.x >> 5) & 3, group = threadIdx.x >> 7, lane = threadIdx.x & 31;
  const int rg = lane >> 2, cg = lane & 3;
  const int col_tiles = static_cast<int>((p.n + kSets * kTile - 1) / (kSets * kTile));
  const int tm = static_cast<int>(blockIdx.x) / col_tiles;
  const int tc = static_cast<int>(blockIdx.x) % col_tiles;
  const int64_t m0 = static_cast<int64_t>(tm) * kTile;
  const int rows = static_cast<int>(p.m - m0 < kTile ? p.m - m0 : kTile);
  // This lane's first column of z (of the gate set) and of dout.
  const int64_t zc = static_cast<int64_t>(tc) * kSets * kTile + warp * 32 + cg * 8;
  const int64_t dc = static_cast<int64_t>(tc) * kTile + warp * 32 + cg * 8;
  const int64_t row_blocks = (p.m + 127) / 128, n_blocks = (p.n + 127) / 128;
  const int64_t sf_blocks = (p.n / 32 + 3) / 4, t_blocks = (p.mt / 32 + 3) / 4;
  if (threadIdx.x < kSets * 32) {
    const int s = threadIdx.x / 32, i = threadIdx.x % 32;
    row_sf[s][i] = make_uint4(0, 0, 0, 0);
    col_sf[s][i] = make_uint4(0, 0, 0, 0);
    if constexpr (kZ) {
      if (p.z_layout != 0) {
        const int64_t bs = static_cast<int64_t>(tc) * kSets + s;
        const int64_t chunk = p.z_layout == 1 ? bs * row_blocks + tm : tm * sf_blocks + bs;
        z_sf[s][i] = __ldg(reinterpret_cast<const uint4*>(p.z_sf + chunk * 512) + i);
      }
    }
  }
  if constexpr (kZ) {
    if (p.z_layout == 0) {
      for (int i = threadIdx.x; i < kSets * kTile * 4; i += 128 * kGroups) {
        const int s = i / (kTile * 4), r = i / 4 % kTile, c = i % 4;
        const int64_t sc = (static_cast<int64_t>(tc) * kSets + s) * 4 + c;
        if (r < rows && sc < p.n / 32)
          reinterpret_cast<uint8_t*>(z_sf[s])[(r & 31) * 16 + (r >> 5) * 4 + c] =
              __ldg(p.z_sf + (m0 + r) * (p.n / 32) + sc);
      }
    }
  }
  __syncthreads();
  float2 sum[kSets][4];
#pragma unroll
  for (int s = 0; s < kSets; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[s][j] = make_float2(0.0f, 0.0f);
  if (zc < p.n) {  // p.n is a multiple of 32: a warp is in or out as a whole
    for (int rb = group; rb * 32 < rows; rb += kGroups) {
      const int r0 = rb * 32 + rg * 4;  // this lane's first row of the tile
      const uint8_t* zq = kZ ? p.z_q + (m0 + r0) * p.n + zc : nullptr;
      const int64_t de = (m0 + r0) * p.ldd + dc;
      float2 v[kSets][4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (r0 + i < rows) {
          float2 d[4];
          if constexpr (kGrad) {
            float f[8];
            load_grad8<kBf16>(p.dout, de + i * p.ldd, f);
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = make_float2(f[2 * j], f[2 * j + 1]);
          }
          if constexpr (kZ) {
#pragma unroll
            for (int s = 0; s < kSets; ++s)
              load_mx8(zq + i * p.n + s * kTile,
                       e8m0_decode(reinterpret_cast<const uint8_t*>(
                           z_sf[s])[(rg * 4 + i) * 16 + rb * 4 + warp]),
                       v[s][i]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (kAct == kActSwiglu)
              gated_grad2(d[j], v[0][i][j], v[1][i][j], v[0][i][j], v[1][i][j]);
            else if constexpr (kAct == kActNone)
              v[0][i][j] = d[j];
            else if constexpr (kAct > 0)
              v[0][i][j] = mul2(d[j], make_float2(act_slope<kAct>(v[0][i][j].x),
                                                  act_slope<kAct>(v[0][i][j].y)));
          }
        } else {
#pragma unroll
          for (int s = 0; s < kSets; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[s][i][j] = make_float2(0.0f, 0.0f);
        }
      }
#pragma unroll
      for (int s = 0; s < kSets; ++s) {
        float2 (&x)[4][4] = v[s];
        if constexpr (kGrad) {
          // Along the rows: 8 values here, the block's others in 3 neighbours.
          float peak[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            peak[i] = fmaxf(fabsf(x[i][0].x), fabsf(x[i][0].y));
#pragma unroll
            for (int j = 1; j < 4; ++j)
              peak[i] = fmaxf(fmaxf(peak[i], fabsf(x[i][j].x)), fabsf(x[i][j].y));
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t t = upper2(peak[2 * h], peak[2 * h + 1]);
            t = max_u16x2(t, __shfl_xor_sync(0xffffffffu, t, 1));
            t = max_u16x2(t, __shfl_xor_sync(0xffffffffu, t, 2));
            const uint32_t c = codes_x128(t), r = reciprocals(c);
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              const int i = 2 * h + o;
              const float2 mul = both(o ? upper_half(r) : lower_half(r));
              uint32_t w[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float2 a = mul2(x[i][2 * e], mul), b = mul2(x[i][2 * e + 1], mul);
                w[e] = cvt_e4m3x4(a.x, a.y, b.x, b.y);
              }
              if (r0 + i < rows)
                *reinterpret_cast<uint2*>(p.dz_q + (m0 + r0 + i) * p.n + zc + s * kTile) =
                    make_uint2(w[0], w[1]);
            }
            if (cg == 0) {
              uint8_t* to = reinterpret_cast<uint8_t*>(row_sf[s]) + (rg * 4 + 2 * h) * 16 +
                            rb * 4 + warp;
              to[0] = static_cast<uint8_t>(c >> 7);
              to[16] = static_cast<uint8_t>(c >> 23);
            }
          }
        }
        // Along the columns: 4 values here, the block's others in the 7 lanes
        // with the same cg.  The eight columns' peaks are halved twice among
        // them (lanes with bit 4 set keep columns 4..7, and so on), so that a
        // lane finds the codes of two columns and fetches the others'.
        uint32_t t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = fmaxf(fmaxf(fabsf(x[0][j].x), fabsf(x[1][j].x)),
                                fmaxf(fabsf(x[2][j].x), fabsf(x[3][j].x)));
          const float b = fmaxf(fmaxf(fabsf(x[0][j].y), fabsf(x[1][j].y)),
                                fmaxf(fabsf(x[2][j].y), fabsf(x[3][j].y)));
          t[j] = upper2(a, b);
        }
        const bool b4 = lane & 16, b3 = lane & 8;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t other = __shfl_xor_sync(0xffffffffu, b4 ? t[j] : t[j + 2], 16);
          t[j] = max_u16x2(b4 ? t[j + 2] : t[j], other);
        }
        t[0] = max_u16x2(b3 ? t[1] : t[0],
                         __shfl_xor_sync(0xffffffffu, b3 ? t[0] : t[1], 8));
        t[0] = max_u16x2(t[0], __shfl_xor_sync(0xffffffffu, t[0], 4));
        // Lane bits 4, 3: this lane's pair of columns is 2 * (2 b4 + b3).
        const uint32_t c = codes_x128(t[0]), r = reciprocals(c);
        if ((lane & 4) == 0) {
          uint8_t* to = reinterpret_cast<uint8_t*>(col_sf[s]) +
                        (cg * 8 + (lane >> 3) * 2) * 16 + warp * 4 + rb;
          to[0] = static_cast<uint8_t>(c >> 7);
          to[16] = static_cast<uint8_t>(c >> 23);
        }
        uint8_t* tq = p.dzt_q + (zc + s * kTile) * p.mt + m0 + r0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t rj = __shfl_sync(0xffffffffu, r, cg + 8 * j);
          const float2 mul = make_float2(lower_half(rj), upper_half(rj));
          float2 y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = mul2(x[i][j], mul);
          *reinterpret_cast<uint32_t*>(tq) = cvt_e4m3x4(y[0].x, y[1].x, y[2].x, y[3].x);
          *reinterpret_cast<uint32_t*>(tq + p.mt) = cvt_e4m3x4(y[0].y, y[1].y, y[2].y, y[3].y);
          tq += 2 * p.mt;
          if constexpr (kGrad)
            sum[s][j] = add2(sum[s][j], add2(add2(x[0][j], x[1][j]), add2(x[2][j], x[3][j])));
        }
      }
    }
    if constexpr (kGrad) {
      if (p.dbias_part) {
#pragma unroll
        for (int s = 0; s < kSets; ++s) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float2 t = sum[s][j];
#pragma unroll
            for (int o = 4; o <= 16; o *= 2)
              t = add2(t, make_float2(__shfl_xor_sync(0xffffffffu, t.x, o),
                                      __shfl_xor_sync(0xffffffffu, t.y, o)));
            if (rg == j) {
              float* to = kGroups > 1 ? &part[group][s * kTile + warp * 32 + cg * 8 + 2 * j]
                                      : p.dbias_part + tm * p.n + zc + s * kTile + 2 * j;
              to[0] = t.x;
              to[1] = t.y;
            }
          }
        }
      }
    }
  }
  __syncthreads();
  // Whole chunks: what lies beyond the matrix reads as zero scales.
  if (threadIdx.x < 128) {
    if (warp < kSets) {
      const int64_t bs = static_cast<int64_t>(tc) * kSets + warp;
      const int64_t chunk = p.out_layout == 1 ? bs * row_blocks + tm : tm * sf_blocks + bs;
      if constexpr (kGrad)
        reinterpret_cast<uint4*>(p.dz_sf + chunk * 512)[lane] = row_sf[warp][lane];
    } else if (warp >= 2 && warp < 2 + kSets) {
      const int64_t br = static_cast<int64_t>(tc) * kSets + warp - 2;
      const int64_t chunk = p.out_layout == 1 ? tm * n_blocks + br : br * t_blocks + tm;
      reinterpret_cast<uint4*>(p.dzt_sf + chunk * 512)[lane] = col_sf[warp - 2][lane];
    }
  }
  if constexpr (kGrad && kGroups > 1) {
    const int64_t col = static_cast<int64_t>(tc) * kSets * kTile + threadIdx.x;
    if (p.dbias_part && threadIdx.x < kSets * kTile && col < p.n) {
      float t = part[0][threadIdx.x];
      for (int g = 1; g < kGroups && g * 32 < rows; ++g) t += part[g][threadIdx.x];
      p.dbias_part[tm * p.n + col] = t;
    }
  }
}

// Few tiles: all four row groups of a tile at once, for latency; enough tiles to
// fill the SMs with 128-thread CTAs several times: one group after the other.
constexpr int kGroupsSmall = 4;
bool small_grid(int grid) { return grid < 4 * num_sms(); }

template <int kAct>
void launch_act(const ActBackwardParams& p, bool bf16, int grid, cudaStream_t stream) {
  if (small_grid(grid)) {
    if (bf16) act_backward_kernel<kAct, true, kGroupsSmall><<<grid, 512, 0, stream>>>(p);
    else act_backward_kernel<kAct, false, kGroupsSmall><<<grid, 512, 0, stream>>>(p);
  } else {
    if (bf16) act_backward_kernel<kAct, true, 1><<<grid, 128, 0, stream>>>(p);
    else act_backward_kernel<kAct, false, 1><<<grid, 128, 0, stream>>>(p);
  }
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
  const int grid = act_grid(p, 1);
  if (small_grid(grid))
    act_backward_kernel<-1, false, kGroupsSmall><<<grid, 512, 0, stream>>>(p);
  else
    act_backward_kernel<-1, false, 1><<<grid, 128, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace qg
