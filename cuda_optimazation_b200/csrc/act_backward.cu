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
// lane's bytes of a row are 8 neighbours and those of a column 4, and no result
// passes through shared memory.
//
// Issue slots are 66 % busy (gated) and DRAM 50 %: neither is full, and with 16 warps an
// SM latency counts as well.  So the work per element is kept down: fp32 pairs in one
// instruction (f32x2), and block scales from the upper halves of the peaks' fp32
// patterns, two peaks to a register -- a scale needs the exponent of its peak only, and
// the upper halves order as the peaks do.
//
// Measured: 4096 x 28672 gated, bf16, 106 us (4.5 TB/s; 73 M warp instructions); 8192 x
// 14336 gelu 137 us bf16, relu 106, silu fp32 134 (6.2 TB/s); 1024 x 8192 gelu bf16 17;
// 333 x 4128 gelu fp32 7.1; transposition of 16384 x 8192 49.7 us (5.6 TB/s; 58 while lanes
// fetched 8 bytes of 8 rows: the L1's data stage was the limit).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "qg_act.cuh"
#include "qg_codec.cuh"
#include "qg_gemm.h"
#include "qg_ptx.cuh"

namespace qg {

namespace {

constexpr int kTile = 128;  // rows, and columns of a set, of a CTA

// Staging (cp.async).
__device__ __forceinline__ void stage_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int kLeft>
__device__ __forceinline__ void stage_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// Eight gradients: 16 bytes of bf16, or two 16-byte pieces of fp32, `second` apart.
template <bool kBf16>
__device__ __forceinline__ void read_grad8(uint32_t at, int second, float2 (&v)[4]) {
  const uint4 a = lds128_at(at);
  if constexpr (kBf16) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  } else {
    const uint4 b = lds128_at(at + second);
    v[0] = make_float2(__uint_as_float(a.x), __uint_as_float(a.y));
    v[1] = make_float2(__uint_as_float(a.z), __uint_as_float(a.w));
    v[2] = make_float2(__uint_as_float(b.x), __uint_as_float(b.y));
    v[3] = make_float2(__uint_as_float(b.z), __uint_as_float(b.w));
  }
}

// Eight values of an MXFP8 row with scale s.
__device__ __forceinline__ void read_mx8(uint32_t at, float s, float2 (&v)[4]) {
  const uint2 w = lds64_at(at);
  e4m3x4_decode(w.x, v[0], v[1]);
  e4m3x4_decode(w.y, v[2], v[3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = mul2(v[i], both(s));
}

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

// Bytes of a staged 32-row group: the gradient's rows and each set's of z.
template <int kAct, bool kBf16>
constexpr int staged_bytes() {
  return 32 * ((kAct >= 0 ? (kBf16 ? 256 : 512) : 0) +
               128 * (kAct == kActNone ? 0 : kAct == kActSwiglu ? 2 : 1));
}

// kAct < 0: z itself (the transposition).  kGroups: 32-row groups of the tile
// that are worked on at once, by four warps each.
template <int kAct, bool kBf16, int kGroups>
__global__ void __launch_bounds__(128 * kGroups, kGroups == 1 && kAct == kActSwiglu ? 4 : 0)
    act_backward_kernel(const ActBackwardParams p) {
  constexpr int kSets = kAct == kActSwiglu ? 2 : 1;
  constexpr bool kGrad = kAct >= 0, kZ = kAct != kActNone;
  // Rows are staged in whole lines (32-byte pieces of eight rows cost the L1 four
  // times as much).  One group after the other: of the transposition 32 rows by each
  // warp, whose blocks then lie side by side, else 32 rows by the CTA at a time.
  constexpr bool kLines = !kGrad && kGroups == 1, kShared = kGrad && kGroups == 1;
  extern __shared__ __align__(16) uint8_t staged[];
  __shared__ uint4 row_sf[kSets][32], col_sf[kSets][32];  // 512-byte chunks
  __shared__ float4 z_scale[kSets][4][4][8];               // [row group][warp][row / 4]
  __shared__ float part[kGroups > 1 ? kGroups : 1][kSets * kTile];
  const int warp = (threadIdx.x >> 5) & 3, group = threadIdx.x >> 7, lane = threadIdx.x & 31;
  const int rg = lane >> 2, cg = lane & 3;
  const int col_tiles = static_cast<int>((p.n + kSets * kTile - 1) / (kSets * kTile));
  const int row_tiles = static_cast<int>((p.m + kTile - 1) / kTile);
  // All groups at once: the row tiles of a column tile are neighbours, and one
  // cluster where p.cluster_rows says so.
  const int tm = static_cast<int>(kGroups > 1 ? blockIdx.x % row_tiles : blockIdx.x / col_tiles);
  const int tc = static_cast<int>(kGroups > 1 ? blockIdx.x / row_tiles : blockIdx.x % col_tiles);
  const int64_t m0 = static_cast<int64_t>(tm) * kTile;
  const int rows = static_cast<int>(p.m - m0 < kTile ? p.m - m0 : kTile);
  // This lane's first column of z (of the gate set).
  const int64_t zc =
      static_cast<int64_t>(tc) * kSets * kTile + (kLines ? 0 : warp * 32) + cg * 8;
  // p.n is a multiple of 32: a warp is in or out as a whole.
  const bool active = kLines ? warp * 32 < rows : zc < p.n;
  const int64_t row_blocks = (p.m + 127) / 128, n_blocks = (p.n + 127) / 128;
  const int64_t sf_blocks = (p.n / 32 + 3) / 4, t_blocks = (p.mt / 32 + 3) / 4;
  const int64_t d_step = p.ldd * (kBf16 ? 2 : 4);
  const uint32_t stage_line = smem_u32(staged) + (warp * 32 + rg * 4) * 128 + cg * 8;
  // Whole lines, of 32 rows: the gradient's, then each set of z.  Row 4 a + b's
  // 16-byte piece c lies at place c ^ x(a), so that what a part of a warp reads at
  // once (8 bytes of 4 rows, or 16 of 2, 4 apart) lies in all banks.
  constexpr int kGradRow = kBf16 ? 256 : 512, kGradPieces = kGradRow / 16;
  constexpr int kZAt = kGrad ? 32 * kGradRow : 0;
  constexpr int kSlotBytes = staged_bytes<kAct, kBf16>();
  const uint32_t line_d =
      smem_u32(staged) + rg * 4 * kGradRow +
      (kBf16 ? (warp * 4 + cg) ^ 4 * (rg & 1) : (warp * 8 + cg * 2) ^ (rg & 1)) * 16;
  const uint32_t line_z = smem_u32(staged) + kZAt + rg * 4 * 128 +
                          ((warp * 2 + (cg >> 1)) ^ 2 * (rg & 3)) * 16 + (cg & 1) * 8;
  // 32 rows, copied by the 128 threads that work on them, into slot rb (all groups at
  // once) or rb % 2.
  auto fetch_lines = [&](int rb) {
    const uint32_t to = smem_u32(staged) + (kGroups > 1 ? rb : rb & 1) * kSlotBytes;
    const int t = threadIdx.x & 127;
    if constexpr (kGrad) {
      constexpr int kRows = 128 / kGradPieces;  // of a pass
      const int piece = t % kGradPieces, row = t / kGradPieces;
      const int64_t col = static_cast<int64_t>(tc) * kTile + piece * (kBf16 ? 8 : 4);
      const uint8_t* from = static_cast<const uint8_t*>(p.dout) +
                            (m0 + rb * 32 + row) * d_step + col * (kBf16 ? 2 : 4);
      if (col < p.n / kSets) {
#pragma unroll
        for (int k = 0; k < 32 / kRows; ++k) {
          const int place = piece ^ (kBf16 ? row & 4 : k & 1);
          if (rb * 32 + row + k * kRows < rows)
            copy_async_at(to + (row + k * kRows) * kGradRow + place * 16, from);
          from += kRows * d_step;
        }
      }
    }
    if constexpr (kZ) {
      const int piece = t & 7, row = t >> 3;
      const int64_t col = static_cast<int64_t>(tc) * kSets * kTile + piece * 16;
      const uint8_t* from = p.z_q + (m0 + rb * 32 + row) * p.n + col;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (rb * 32 + row + k * 16 < rows) {
#pragma unroll
          for (int s = 0; s < kSets; ++s)
            if (col + s * kTile < p.n)
              copy_async_at(to + kZAt + s * 4096 + (row + k * 16) * 128 +
                                    (piece ^ 2 * warp) * 16,
                                from + s * kTile);
        }
        from += 16 * p.n;
      }
    }
    stage_commit();
  };
  // Scales first: the CTA's barrier waits for them.
  uint32_t zw[4] = {0, 0, 0, 0};
  if (kZ && threadIdx.x < kSets * 32) {
    // Row i's 16 bytes of the chunk: scales of rows i, i + 32, i + 64, i + 96.
    const int i = threadIdx.x % 32;
    const int64_t bs = static_cast<int64_t>(tc) * kSets + threadIdx.x / 32;
    if (p.z_layout != 0) {
      const int64_t chunk = p.z_layout == 1 ? bs * row_blocks + tm : tm * sf_blocks + bs;
      const uint4 c = __ldg(reinterpret_cast<const uint4*>(p.z_sf + chunk * 512) + i);
      zw[0] = c.x; zw[1] = c.y; zw[2] = c.z; zw[3] = c.w;
    } else {
      for (int r = 0; r < 4; ++r)
        for (int c = 0; c < 4; ++c)
          if (r * 32 + i < rows && bs * 4 + c < p.n / 32)
            zw[r] |= static_cast<uint32_t>(
                         __ldg(p.z_sf + (m0 + r * 32 + i) * (p.n / 32) + bs * 4 + c))
                     << (8 * c);
    }
  }
  if constexpr (kLines) {
    const int piece = lane & 7, row = warp * 32 + (lane >> 3);
    const uint8_t* from = p.z_q + (m0 + row) * p.n + tc * kTile + piece * 16;
    if (static_cast<int64_t>(tc) * kTile + piece * 16 < p.n) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (row + i * 4 < rows)
          copy_async_at(smem_u32(staged) + (row + i * 4) * 128 + (piece ^ 2 * (i & 3)) * 16,
                            from);
        from += 4 * p.n;
      }
    }
    stage_commit();
  } else {
    fetch_lines(group);
  }
  if (threadIdx.x < kSets * 32) {
    const int s = threadIdx.x / 32, i = threadIdx.x % 32;
    row_sf[s][i] = make_uint4(0, 0, 0, 0);
    col_sf[s][i] = make_uint4(0, 0, 0, 0);
    if constexpr (kZ) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          reinterpret_cast<float*>(z_scale[s][r][c])[i] = e8m0_decode(zw[r] >> (8 * c) & 0xffu);
    }
  }
  if constexpr (kGroups > 1) stage_wait<0>();
  __syncthreads();
  float2 sum[kSets][4];
#pragma unroll
  for (int s = 0; s < kSets; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[s][j] = make_float2(0.0f, 0.0f);
  if (active || kShared) {
    uint8_t* row_out = p.dz_q + (m0 + group * 32 + rg * 4) * p.n + zc;
    uint8_t* col_out = p.dzt_q + zc * p.mt + m0 + (kLines ? warp : group) * 32 + rg * 4;
    if constexpr (kLines) {
      stage_wait<0>();
      __syncwarp();
    }
    const int64_t end = kLines ? p.n - static_cast<int64_t>(tc) * kTile : rows;
#pragma unroll 1
    for (int it = group; it * 32 < end && (!kLines || it < 4); it += kGroups) {
      const int rb = kLines ? warp : it, cb = kLines ? it : warp;  // block row and column
      const int r0 = rb * 32 + rg * 4;  // this lane's first row of the tile
      const int slot = kGroups > 1 ? rb : rb & 1;
      if constexpr (kShared) {
        stage_wait<0>();
        __syncthreads();  // these rows have come, and the rows before them been read
        if ((it + 1) * 32 < rows) fetch_lines(it + 1);
        if (!active) continue;
      }
      float2 v[kSets][4][4];
      float zs[kSets][4];
      if constexpr (kZ) {
#pragma unroll
        for (int s = 0; s < kSets; ++s) {
          const float4 f = z_scale[s][rb][cb][rg];
          zs[s][0] = f.x; zs[s][1] = f.y; zs[s][2] = f.z; zs[s][3] = f.w;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (r0 + i < rows) {
          float2 d[4];
          if constexpr (kGrad)
            read_grad8<kBf16>(line_d + slot * kSlotBytes + i * kGradRow, rg & 1 ? -16 : 16, d);
          if constexpr (kZ) {
#pragma unroll
            for (int s = 0; s < kSets; ++s)
              read_mx8(kLines ? stage_line + i * 128 + (cb * 32 ^ (rg & 3) * 32)
                              : line_z + slot * kSlotBytes + s * 4096 + i * 128,
                       zs[s][i], v[s][i]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (kAct == kActSwiglu)
              gated_grad2(d[j], v[0][i][j], v[1][i][j], v[0][i][j], v[1][i][j]);
            else if constexpr (kAct == kActNone)
              v[0][i][j] = d[j];
            else if constexpr (kAct == kActRelu)
              v[0][i][j] = relu_grad2(d[j], v[0][i][j]);
            else if constexpr (kAct > 0)
              v[0][i][j] = mul2(d[j], act_slope2<kAct>(v[0][i][j]));
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
            peak[i] = max3_abs(x[i][0].x, x[i][0].y, x[i][1].x);
            peak[i] = max3_abs(peak[i], x[i][1].y, x[i][2].x);
            peak[i] = max3_abs(peak[i], x[i][2].y, x[i][3].x);
            peak[i] = max3_abs(peak[i], x[i][3].y, 0.0f);
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
                *reinterpret_cast<uint2*>(row_out + i * p.n + s * kTile) =
                    make_uint2(w[0], w[1]);
            }
            if (cg == 0) {
              uint8_t* to = reinterpret_cast<uint8_t*>(row_sf[s]) + (rg * 4 + 2 * h) * 16 +
                            rb * 4 + cb;
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
          const float a = max3_abs(x[0][j].x, x[1][j].x, x[2][j].x);
          const float b = max3_abs(x[0][j].y, x[1][j].y, x[2][j].y);
          t[j] = upper2(max3_abs(a, x[3][j].x, 0.0f), max3_abs(b, x[3][j].y, 0.0f));
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
                        (cg * 8 + (lane >> 3) * 2) * 16 + cb * 4 + rb;
          to[0] = static_cast<uint8_t>(c >> 7);
          to[16] = static_cast<uint8_t>(c >> 23);
        }
        uint8_t* tq = col_out + s * kTile * p.mt;
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
      row_out += 32 * p.n;
      col_out += kLines ? 32 * p.mt : 32;
    }
    if constexpr (kGrad) {
      if (p.dbias_part && active) {
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
    if (p.dbias_part) {
      const int64_t col = static_cast<int64_t>(tc) * kSets * kTile + threadIdx.x;
      const bool in = threadIdx.x < kSets * kTile && col < p.n;
      float t = 0.0f;
      if (in)
        for (int g = 0; g < kGroups && g * 32 < rows; ++g) t += part[g][threadIdx.x];
      if (!p.cluster_rows) {
        if (in) p.dbias_part[tm * p.n + col] = t;
      } else {
        // The column tile's row tiles are this cluster: the first sums them up.
        if (in) part[0][threadIdx.x] = t;
        cluster_sync();
        if (tm == 0 && in) {
          for (int r = 1; r < row_tiles; ++r)
            t += ld_cluster_f32(
                mapa_shared(smem_u32(&part[0][threadIdx.x]), static_cast<uint32_t>(r)));
          p.dbias_part[col] = t;
        }
        cluster_sync();  // the others' shared memory has been read
      }
    }
  }
}

// One round of tiles: all four row groups of a tile at once, for latency.  Such a CTA
// fills an SM (the transposition's half of one), so more tiles than that would take a
// second round: 128-thread CTAs then, one group after the other.  Measured, us at once /
// in turn: gelu bf16 of 64 tiles 6.5 / 9.0, 148 9.5 / 10.9, 152 13.8 / 12.0, 512 36.7 /
// 17.0; transposition of 128 tiles 3.3 / 3.9, 288 5.0 / 5.3, 304 6.8 / 5.4.
constexpr int kGroupsSmall = 4;
bool small_grid(int64_t grid, int ctas_per_sm) { return grid <= ctas_per_sm * num_sms(); }
// Row tiles that a cluster may join (the portable size).
constexpr int kClusterRows = 8;
// Tiles of which the clusters of `rows` CTAs, one an SM, find a place at once: of 148
// SMs 148 in clusters of 2, 130 to 135 of 3 to 6, 105 of 7 and 120 of 8.
int64_t cluster_tiles(int64_t rows) {
  return num_sms() * (rows <= 2 ? 100 : rows <= 6 ? 87 : 70) / 100;
}

template <int kAct, bool kBf16, int kGroups>
cudaError_t launch_one(const ActBackwardParams& p, int grid, cudaStream_t stream) {
  constexpr int kSmem = kAct < 0 ? kTile * kTile
                                 : staged_bytes<kAct, kBf16>() * (kGroups > 1 ? kGroups : 2);
  auto kernel = act_backward_kernel<kAct, kBf16, kGroups>;
  static bool done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
    return cudaErrorInvalidDevice;
  if (!done[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    done[dev] = true;
  }
  if (p.cluster_rows) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(128 * kGroups);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>((p.m + kTile - 1) / kTile);
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
  }
  kernel<<<grid, 128 * kGroups, kSmem, stream>>>(p);
  return cudaGetLastError();
}

template <int kAct, bool kBf16>
cudaError_t launch_act(const ActBackwardParams& p, int grid, cudaStream_t stream) {
  return small_grid(grid, kAct < 0 ? 2 : 1)
             ? launch_one<kAct, kBf16, kGroupsSmall>(p, grid, stream)
             : launch_one<kAct, kBf16, 1>(p, grid, stream);
}

int64_t act_grid(int64_t m, int64_t n, int sets) {
  return ((m + kTile - 1) / kTile) * ((n + sets * kTile - 1) / (sets * kTile));
}

}  // namespace

// Joining saves the second launch where every cluster finds a place (us with / without:
// 256 x 4096 gelu 6.5 / 7.3, 1024 x 1024 7.1 / 7.7, 512 x 4096 7.3 / 8.5), and costs a
// round where one does not (512 x 4608 13.6 / 9.0, 1024 x 2048 13.8 / 8.7).
bool act_backward_joins(int64_t m, int64_t n, int act) {
  const int64_t parts = (m + kTile - 1) / kTile;
  return parts == 1 || (parts <= kClusterRows &&
                        act_grid(m, n, act == kActSwiglu ? 2 : 1) <= cluster_tiles(parts));
}

cudaError_t launch_act_backward(const ActBackwardParams& in, int act, bool bf16,
                                cudaStream_t stream) {
  ActBackwardParams p = in;
  p.cluster_rows = p.dbias_part && p.m > kTile && act_backward_joins(p.m, p.n, act);
  const int grid = static_cast<int>(act_grid(p.m, p.n, act == kActSwiglu ? 2 : 1));
#define QG_ACT_CASE(a) \
  case a:              \
    return bf16 ? launch_act<a, true>(p, grid, stream) : launch_act<a, false>(p, grid, stream);
  switch (act) {
    QG_ACT_CASE(kActNone)
    QG_ACT_CASE(kActRelu)
    QG_ACT_CASE(kActSilu)
    QG_ACT_CASE(kActGelu)
    QG_ACT_CASE(kActSwiglu)
    default: return cudaErrorInvalidValue;
  }
#undef QG_ACT_CASE
}

cudaError_t launch_transpose_mxfp8(const ActBackwardParams& p, cudaStream_t stream) {
  return launch_act<-1, false>(p, static_cast<int>(act_grid(p.m, p.n, 1)), stream);
}

}  // namespace qg
