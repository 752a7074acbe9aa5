// gemm_fused_rows.cu -- the fused-epilogue block-scaled GEMM for few rows
// (m <= 128: single tokens, decoding batches).
//
// The product is bound by streaming the weights B [n][k] once, so they are the
// MMA's M side: D[128 weight rows][kN activation rows] in TMEM, one weight tile
// (the gated form: the 128 gate rows and their 128 factor rows) per cluster.  The
// clusters' CTAs split K, as many as keep every SM streaming (one CTA an SM, or two
// for long shares where their accumulators and rings fit): a CTA's ring holds
// ~100 KB, twice what HBM's latency asks of an SM.  The partial sums meet in
// the cluster's shared memory, where every CTA sums and finishes its share
// of the rows in a fixed order: no workspace, no atomics, one launch.
//
// Scales reach TMEM by tcgen05.cp: its fixed cost per 512-byte chunk, which the
// large-m kernel avoids, hides behind the weight stream here.
//
// The epilogue runs across lanes (four columns each): a warp has a row of the
// tile, eight lanes an MX block of it.
//
// Roles (8 warps): warp 0 TMA producer, warp 1 MMA issuer (and TMEM owner),
// warps 2..5 read the accumulator (one TMEM lane quadrant each); all eight finish
// rows.  Every mbarrier wait is bounded (qg_ptx.cuh), so the cluster's barriers are reached.
//
// Measured (MXFP8): one token, 2 x 14336 x 4096 gated, 21.2 us (5.7 TB/s), x 8192
// 37.5 (6.45 TB/s, the rate of a copy); 64 x 4096 x 14336 16.5 us, of which about 6
// are start, exchange and end.  NVFP4 16 x 28672 x 8192 24.8 us.  Against the pair kernel:
// at the rule that chooses between them, in capi.cu.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "gemm_epilogue.cuh"
#include "qg_codec.cuh"
#include "qg_gemm.h"
#include "qg_ptx.cuh"

namespace qg {

namespace {

constexpr int kPrefetch = 4;  // K blocks of weights prefetched into L2 before the wait
constexpr int kMaxRanks = 8;  // CTAs per cluster (the portable size)
constexpr int kRowsFmtMxfp8 = 0, kRowsFmtNvfp4 = 1, kRowsFmtMxfp4 = 2;

constexpr int pow2_at_least(int v) {
  int p = 32;
  while (p < v) p *= 2;
  return p;
}

template <int kFmt, int kN, bool kGated>
struct RowsCfg {
  static constexpr int kSets = kGated ? 2 : 1;
  static constexpr int kChunks = kFmt == kRowsFmtNvfp4 ? 4 : (kFmt == kRowsFmtMxfp4 ? 2 : 1);
  static constexpr int kWBytes = kSets * 128 * 128;
  static constexpr int kXBytes = kN * 128;
  static constexpr int kSfwBytes = kSets * kChunks * 512;
  static constexpr int kSfxBytes = kChunks * 512;
  static constexpr int kTx = kWBytes + kXBytes + kSfwBytes + kSfxBytes;
  static constexpr int kStageBytes = (kTx + 1023) / 1024 * 1024;
  static constexpr int kSfCols = (kSets + 1) * kChunks * 4;  // scale columns of a stage
  static constexpr int kAccCols = kSets * kN;
  // Two CTAs an SM if both fit its 512 TMEM columns (more CTAs than TMEM for
  // them would wait for one another inside their clusters).
  static constexpr int kExtra = 256 + 1024;  // barriers, alignment
  static constexpr int kStagesTwo = (228 * 1024 / 2 - 1024 - kExtra) / kStageBytes;
  static constexpr bool kTwo = kAccCols + kStagesTwo * kSfCols <= 256;
  static constexpr int kStagesOne =
      (216 * 1024) / kStageBytes < (512 - kAccCols) / kSfCols ? (216 * 1024) / kStageBytes
                                                              : (512 - kAccCols) / kSfCols;
  static constexpr int kStages = kTwo ? kStagesTwo : kStagesOne;
  static_assert(kStages >= 2, "ring");
  static constexpr int kTmemCols = pow2_at_least(kAccCols + kStages * kSfCols);
  // The partial sums are exchanged through the ring's memory.
  static_assert(kSets * kN * 512 <= kStages * kStageBytes, "exchange buffer");
  static constexpr int kSmemBytes = kStages * kStageBytes + kExtra;
  // Never three CTAs on an SM, whose TMEM would not do.
  static_assert(3 * (kSmemBytes + 1024) > 228 * 1024 && kTmemCols <= (kTwo ? 256 : 512),
                "residency");
  static constexpr int kPerSm = kTwo ? 2 : 1;
};

__device__ __forceinline__ uint32_t cluster_nctas() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}

// Four consecutive columns a lane: their bytes of an MXFP8 row and, from every
// eighth lane, the scale of its 32-column block.  `in`: the block lies in the matrix.
__device__ __forceinline__ void lane_store_mx(const float (&v)[4], bool in, uint8_t* q, uint8_t* sf,
                                              int layout, int sf_blocks, int row, int col, int n,
                                              int lane) {
  float peak = in ? max3_abs(max3_abs(v[0], v[1], v[2]), v[3], 0.0f) : 0.0f;
#pragma unroll
  for (int o = 1; o <= 4; o *= 2) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, o));
  float mul;
  const uint32_t code = mxfp8_scale_code(peak, mul);
  if (in)
    *reinterpret_cast<uint32_t*>(q + static_cast<int64_t>(row) * n + col) =
        cvt_e4m3x4(v[0] * mul, v[1] * mul, v[2] * mul, v[3] * mul);
  if ((lane & 7) == 0) {
    const int sc = col / 32;
    if (layout == 0) {
      if (in) sf[static_cast<int64_t>(row) * (n / 32) + sc] = static_cast<uint8_t>(code);
    } else if (sc < sf_blocks * 4) {  // rows fit one 128-row block: both MMA orders agree
      sf[mma_scale_offset(row, sc, 1, sf_blocks, layout)] = static_cast<uint8_t>(code);
    }
  }
}

// Zero scales of rows [m, 128) in the chunk of columns [col0, col0 + 128).
__device__ __forceinline__ void pad_rows(uint8_t* sf, int layout, int sf_blocks, int col0, int m) {
  const int w = threadIdx.x;
  if (layout == 0 || w >= 128 || (w >> 2) + (w & 3) * 32 < m || col0 / 128 >= sf_blocks) return;
  reinterpret_cast<uint32_t*>(sf + mma_scale_offset(0, col0 / 32, 1, sf_blocks, layout))[w] = 0u;
}

template <int kFmt, int kN, bool kGated>
__global__ void __launch_bounds__(256, RowsCfg<kFmt, kN, kGated>::kPerSm)
    gemm_fused_rows_kernel(const __grid_constant__ GemmParams p) {
  using Cfg = RowsCfg<kFmt, kN, kGated>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + Cfg::kStages * Cfg::kStageBytes);
  uint64_t* empty_bar = full_bar + Cfg::kStages;
  uint64_t* acc_full = empty_bar + Cfg::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  static_assert(16 * Cfg::kStages + 16 <= 256, "barrier space");

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = static_cast<int>(cluster_ctarank()), ranks = static_cast<int>(cluster_nctas());
  const int tile = static_cast<int>(cluster_id_x());
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.num_k_blocks) * rank / ranks);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.num_k_blocks) * (rank + 1) / ranks);

  const int col0 = tile * Cfg::kSets * 128;  // first column of z
  // One stage's loads (the producer thread).
  auto load_stage = [&](int stage, int kb, uint64_t pol_w, uint64_t pol_x) {
    uint8_t* sw = smem + stage * Cfg::kStageBytes;
    uint8_t* sx = sw + Cfg::kWBytes;
    uint8_t* ssw = sx + Cfg::kXBytes;
    uint8_t* ssx = ssw + Cfg::kSfwBytes;
    mbar_arrive_expect_tx(&full_bar[stage], Cfg::kTx);
    tma_load_2d(sw, &p.tm_a, &full_bar[stage], kb * 128, col0, pol_w);
    tma_load_3d(ssw, &p.tm_sfa, &full_bar[stage], 0, col0 / 128, kb * Cfg::kChunks, pol_w);
    tma_load_2d(sx, &p.tm_b, &full_bar[stage], kb * 128, 0, pol_x);
    tma_load_3d(ssx, &p.tm_sfb, &full_bar[stage], 0, 0, kb * Cfg::kChunks, pol_x);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0u;
    fence_barrier_init();
    // While the stream's previous kernel ends: this CTA's first weights into L2
    // (which stays coherent, should that kernel be writing them).
    for (int kb = kb0; kb < kb1 && kb < kb0 + kPrefetch; ++kb) {
      tma_prefetch_l2_2d(&p.tm_a, kb * 128, col0);
      tma_prefetch_l2_3d(&p.tm_sfa, 0, col0 / 128, kb * Cfg::kChunks);
    }
    griddep_wait();
    // The first stages need no one's leave: on their way before the TMEM
    // allocation and the CTA's barrier.
    const uint64_t pol_w = l2_policy_evict_first(), pol_x = l2_policy_evict_last();
    for (int s = 0; s < Cfg::kStages && kb0 + s < kb1; ++s) load_stage(s, kb0 + s, pol_w, pol_x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  griddep_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA
    if (lane == 0) {
      const uint64_t pol_w = l2_policy_evict_first(), pol_x = l2_policy_evict_last();
      // Stages loaded above: round 0, parity 0.
      const int early = kb1 - kb0 < Cfg::kStages ? kb1 - kb0 : Cfg::kStages;
      uint32_t issued_mask = (1u << early) - 1u, issued_parity = 0, phase = 1;
      int stage = 0;
      bool ok = true;
      for (int kb = kb0 + Cfg::kStages; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1u, p.timeout_ns, abort_flag, p.status,
                               kDevTimeoutProducer)) {
          ok = false;
          break;
        }
        load_stage(stage, kb, pol_w, pol_x);
        issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
        if (++stage == Cfg::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      griddep_launch_dependents();  // all loads are on their way
      if (!ok) {
        uint32_t dummy = 0;
        for (int s = 0; s < Cfg::kStages; ++s)
          if (issued_mask & (1u << s))
            mbar_wait_bounded(&full_bar[s], (issued_parity >> s) & 1u, p.timeout_ns, &dummy,
                              nullptr, 0);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA
    if (lane == 0) {
      const uint32_t idesc_base =
          kFmt == kRowsFmtMxfp8
              ? make_idesc_block_scaled(128, kN, 0u, 1u, 0u, 0u)
              : make_idesc_block_scaled(128, kN, 1u, kFmt == kRowsFmtMxfp4 ? 1u : 0u, 0u, 0u);
      int stage = 0;
      uint32_t phase = 0, acc = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&full_bar[stage], phase, p.timeout_ns, abort_flag, p.status,
                               kDevTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint8_t* sw = smem + stage * Cfg::kStageBytes;
        uint8_t* ssw = sw + Cfg::kWBytes + Cfg::kXBytes;
        uint8_t* ssx = ssw + Cfg::kSfwBytes;
        const uint32_t sfx_col = tmem_base + Cfg::kAccCols + stage * Cfg::kSfCols;
        const uint32_t sfw_col = sfx_col + Cfg::kChunks * 4;
#pragma unroll
        for (int c = 0; c < Cfg::kChunks; ++c) {
          tmem_cp_32x128b_warpx4(sfx_col + c * 4,
                                 make_smem_desc(smem_u32(ssx + c * 512), 0, 128, kSwizzleNone));
#pragma unroll
          for (int s = 0; s < Cfg::kSets; ++s)
            tmem_cp_32x128b_warpx4(
                sfw_col + (s * Cfg::kChunks + c) * 4,
                make_smem_desc(smem_u32(ssw + (c * Cfg::kSets + s) * 512), 0, 128, kSwizzleNone));
        }
        const uint64_t xdesc = make_smem_desc(smem_u32(sw + Cfg::kWBytes), 16, 1024, kSwizzle128B);
#pragma unroll
        for (int s = 0; s < Cfg::kSets; ++s) {
          const uint64_t wdesc = make_smem_desc(smem_u32(sw + s * 16384), 16, 1024, kSwizzle128B);
          const uint32_t d = tmem_base + s * kN;
          const uint32_t sfw = sfw_col + s * Cfg::kChunks * 4;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint64_t koff = static_cast<uint64_t>(j * 2);  // +32 B of K
            const uint32_t on = acc | (j > 0 ? 1u : 0u);
            if (kFmt == kRowsFmtMxfp8) {
              const uint32_t id = idesc_base | (static_cast<uint32_t>(j) << 29) |
                                  (static_cast<uint32_t>(j) << 4);
              mma_mxf8f6f4(d, wdesc + koff, xdesc + koff, id, sfw, sfx_col, on);
            } else if (kFmt == kRowsFmtMxfp4) {
              const uint32_t sid = static_cast<uint32_t>((j & 1) * 2);
              mma_mxf4(d, wdesc + koff, xdesc + koff, idesc_base | (sid << 29) | (sid << 4),
                       sfw + (j / 2) * 4, sfx_col + (j / 2) * 4, on);
            } else {
              mma_mxf4nvf4(d, wdesc + koff, xdesc + koff, idesc_base, sfw + j * 4,
                           sfx_col + j * 4, on);
            }
          }
        }
        acc = 1u;
        tc_commit(&empty_bar[stage]);
        if (++stage == Cfg::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      tc_commit(acc_full);
      if (!ok) {
        // Let the MMAs that were issued finish before the roles meet.
        uint32_t dummy = 0;
        mbar_wait_bounded(acc_full, 0, p.timeout_ns, &dummy, nullptr, 0);
      }
    }
  }

  // ------------------------------------------------------------------ epilogue
  float alpha = 1.0f;
  if (p.a_ts) alpha *= *p.a_ts;
  if (p.b_ts) alpha *= *p.b_ts;
  const EpiParams& e = p.epi;
  // In the last step a warp finishes a row at a time, four columns a lane.
  const int f = lane * 4;
  const int n_out = kGated ? p.n / 2 : p.n;
  const int out_col = (kGated ? tile * 128 : col0) + f;
  const bool in_z = col0 + f < p.n;  // gated: n is a multiple of 256, so both sets are in
  float bias[Cfg::kSets][4];
#pragma unroll
  for (int s = 0; s < Cfg::kSets; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) bias[s][j] = epi_bias(e, col0 + s * 128 + f + j, p.n);
  float* part = reinterpret_cast<float*>(smem);  // [set][row][128]
  const uint32_t part_addr = smem_u32(part);
  bool ok = true;
  if (warp >= 2 && warp <= 5) {
    if (lane == 0)
      ok = mbar_wait_bounded<false, 32>(acc_full, 0, p.timeout_ns, abort_flag, p.status,
                                        kDevTimeoutEpilogue);
    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
    if (ok) mbar_try_wait(acc_full, 0);
    tc_fence_after();
  }
  if (warp >= 2 && warp <= 5 && ok) {
    const int quad = warp % 4;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
#pragma unroll 1
    for (int s = 0; s < Cfg::kSets; ++s) {
#pragma unroll 1
      for (int c = 0; c < p.m; c += 16) {
        uint32_t r[16];
        __syncwarp();
        tmem_ld_32x32b_x16(t_row + s * kN + c, r);
        tmem_wait_ld();
        float* to = part + (s * kN + c) * 128 + quad * 32 + lane;
#pragma unroll
        for (int j = 0; j < 16; ++j) to[j * 128] = __uint_as_float(r[j]);
      }
    }
  }
  __syncwarp();
  cluster_sync();  // every CTA's partial sums are in place
  // A warp finishes every (8 ranks)-th row, kTogether rows at a time: all their remote
  // loads and residuals are in flight at once.
  constexpr int kTogether = kGated ? 1 : 2;
  for (int i0 = rank * 8 + warp; i0 < p.m; i0 += 8 * ranks * kTogether) {
    float z[kTogether][Cfg::kSets][4];
    uint32_t res[kTogether][4];  // raw; beyond the matrix its last row or columns
    if (e.res) {
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        const int64_t at = min(i0 + u * 8 * ranks, p.m - 1) * e.ldr;
        if (e.res_vec && n_out % 4 == 0) {
          const int64_t c = at + min(out_col, n_out - 4);
          if (e.res_bf16) {
            const uint2 r = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(e.res) + c);
            res[u][0] = r.x << 16; res[u][1] = r.x & 0xffff0000u;
            res[u][2] = r.y << 16; res[u][3] = r.y & 0xffff0000u;
          } else {
            const uint4 r = *reinterpret_cast<const uint4*>(static_cast<const uint32_t*>(e.res) + c);
            res[u][0] = r.x; res[u][1] = r.y; res[u][2] = r.z; res[u][3] = r.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int64_t c = at + min(out_col + j, n_out - 1);
            if (e.res_bf16) res[u][j] = static_cast<uint32_t>(static_cast<const uint16_t*>(e.res)[c]) << 16;
            else res[u][j] = static_cast<const uint32_t*>(e.res)[c];
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      // Only what this lane goes on to store is read: a store waits for its values, so
      // every remote read has ended when the warp reaches the closing barrier, after
      // which the read CTA may be gone.
      const int i = i0 + u * 8 * ranks;
      const bool on = i < p.m && in_z;
#pragma unroll
      for (int s = 0; s < Cfg::kSets; ++s) {
        float4 v[kMaxRanks];
        const uint32_t at = part_addr + ((s * kN + i) * 128 + f) * 4;
#pragma unroll
        for (int r = 0; r < kMaxRanks; ++r)
          v[r] = on && r < ranks ? ld_cluster_f32x4(mapa_shared(at, static_cast<uint32_t>(r)))
                                 : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int r = 1; r < kMaxRanks; ++r) {
          v[0].x += v[r].x;
          v[0].y += v[r].y;
          v[0].z += v[r].z;
          v[0].w += v[r].w;
        }
        z[u][s][0] = v[0].x; z[u][s][1] = v[0].y; z[u][s][2] = v[0].z; z[u][s][3] = v[0].w;
      }
    }
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      const int i = i0 + u * 8 * ranks;
      if (i >= p.m) break;
      const int row = i;
#pragma unroll
      for (int s = 0; s < Cfg::kSets; ++s) {
#pragma unroll
        for (int j = 0; j < 4; ++j) z[u][s][j] = z[u][s][j] * alpha + bias[s][j];
        if (e.z_q)
          lane_store_mx(z[u][s], in_z, e.z_q, e.z_sf, e.z_layout, e.z_sf_blocks, row,
                        col0 + s * 128 + f, p.n, lane);
      }
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (kGated) {
          y[j] = act_fwd<kActSilu>(z[u][0][j]) * z[u][1][j];
        } else {
          y[j] = z[u][0][j];
          if (e.act == kActRelu) y[j] = act_fwd<kActRelu>(y[j]);
          else if (e.act == kActSilu) y[j] = act_fwd<kActSilu>(y[j]);
          else if (e.act == kActGelu) y[j] = act_fwd<kActGelu>(y[j]);
        }
        if (e.res) y[j] += __uint_as_float(res[u][j]);
      }
      if (e.out_kind == kEpiMxfp8) {
        lane_store_mx(y, in_z, static_cast<uint8_t*>(e.out), e.out_sf, e.out_layout,
                      e.out_sf_blocks, row, out_col, n_out, lane);
      } else {
        const int64_t at = row * e.ldc + out_col;
        const bool whole = e.out_vec && out_col + 4 <= n_out;
        if (e.out_kind == kEpiBf16) {
          __nv_bfloat16* c = static_cast<__nv_bfloat16*>(e.out) + at;
          if (whole) {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(y[0], y[1]);
            const __nv_bfloat162 hi = __floats2bfloat162_rn(y[2], y[3]);
            *reinterpret_cast<uint2*>(c) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&lo),
                           *reinterpret_cast<const uint32_t*>(&hi));
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (out_col + j < n_out) c[j] = __float2bfloat16_rn(y[j]);
          }
        } else {
          float* c = static_cast<float*>(e.out) + at;
          if (whole) {
            *reinterpret_cast<float4*>(c) = make_float4(y[0], y[1], y[2], y[3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (out_col + j < n_out) c[j] = y[j];
          }
        }
      }
    }
  }
  cluster_sync_relaxed();  // the sums have been read: their CTA may exit
  if (rank == 0) {
    if (e.out_kind == kEpiMxfp8)
      pad_rows(e.out_sf, e.out_layout, e.out_sf_blocks, out_col - f, p.m);
    if (e.z_q) {
#pragma unroll
      for (int s = 0; s < Cfg::kSets; ++s)
        pad_rows(e.z_sf, e.z_layout, e.z_sf_blocks, col0 + s * 128, p.m);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

template <int kFmt, int kN, bool kGated>
cudaError_t launch_rows(const GemmParams& p, cudaStream_t stream) {
  using Cfg = RowsCfg<kFmt, kN, kGated>;
  auto kernel = gemm_fused_rows_kernel<kFmt, kN, kGated>;
  // Clusters of each size that find a place on the device at once.
  static int places[kMaxDevices][kMaxRanks + 1] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
    return cudaErrorInvalidDevice;
  if (!places[dev][1]) {
    cudaError_t err =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes);
    if (err != cudaSuccess) return err;
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                               cudaSharedmemCarveoutMaxShared);
    if (err != cudaSuccess) return err;
    for (int c = kMaxRanks; c >= 2; --c) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(static_cast<unsigned>(c));
      cfg.blockDim = dim3(256);
      cfg.dynamicSmemBytes = Cfg::kSmemBytes;
      cudaLaunchAttribute attr{};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = static_cast<unsigned>(c);
      attr.val.clusterDim.y = 1;
      attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      err = cudaOccupancyMaxActiveClusters(&places[dev][c], kernel, &cfg);
      if (err != cudaSuccess) return err;
    }
    places[dev][1] = num_sms();
  }
  // As many CTAs to a cluster as let every tile's find its place at once, with at
  // least two K blocks each: one CTA an SM (which is what the runtime counts of
  // CTAs that use TMEM), or, where that leaves each more than kN / 2 blocks, two.  The
  // exchange costs every CTA kN x 512 bytes of remote reads: 64 x 4096 x 2048 takes
  // 6.8 us with 128 CTAs and 9.2 with 192, x 28672 27.1 and 26.5; one token, 2 x 14336
  // x 4096 gated, 23.8 with 112 and 21.2 with 224.  (A second round costs more than
  // either: 64 x 4736 x 14336 in 37 clusters of 8 26.8 us, of 6 17.8.)
  const int tiles = p.num_n_tiles;
  auto most = [&](int per_sm) {
    int c = kMaxRanks;
    while (c > 1 && (tiles > per_sm * places[dev][c] || p.num_k_blocks < 2 * c)) --c;
    return c;
  };
  int c = most(1);
  if (Cfg::kPerSm == 2 && p.num_k_blocks > c * kN / 2) c = most(2);
  return launch_overlapped(kernel, dim3(static_cast<unsigned>(tiles) * c), dim3(256),
                           Cfg::kSmemBytes, stream, c, p);
}

template <int kFmt, bool kGated>
cudaError_t launch_rows_n(const GemmParams& p, cudaStream_t stream) {
  switch (rows_mma_n(p.m)) {
    case 16: return launch_rows<kFmt, 16, kGated>(p, stream);
    case 32: return launch_rows<kFmt, 32, kGated>(p, stream);
    case 64: return launch_rows<kFmt, 64, kGated>(p, stream);
    default: return launch_rows<kFmt, 128, kGated>(p, stream);
  }
}

}  // namespace

int rows_mma_n(int64_t m) { return m <= 16 ? 16 : (m <= 32 ? 32 : (m <= 64 ? 64 : 128)); }

cudaError_t launch_gemm_fused_rows(const GemmParams& p, int fmt, cudaStream_t stream) {
  const bool gated = p.epi.act == kActSwiglu;
  if (fmt == kRowsFmtNvfp4)
    return gated ? launch_rows_n<kRowsFmtNvfp4, true>(p, stream)
                 : launch_rows_n<kRowsFmtNvfp4, false>(p, stream);
  if (fmt == kRowsFmtMxfp4)
    return gated ? launch_rows_n<kRowsFmtMxfp4, true>(p, stream)
                 : launch_rows_n<kRowsFmtMxfp4, false>(p, stream);
  return gated ? launch_rows_n<kRowsFmtMxfp8, true>(p, stream)
               : launch_rows_n<kRowsFmtMxfp8, false>(p, stream);
}

}  // namespace qg
