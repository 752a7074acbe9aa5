// qg_gemm.h -- internal launch interface between the C-ABI host code and
// the kernels.  Not part of the public ABI (include/qgemm.h is).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace qg {

// Launch with programmatic stream serialization: the grid may start while the
// stream's previous one is ending (its CTAs past griddep_launch_dependents), so
// the kernel calls griddep_wait before it reads or writes global memory.
// `cluster`: CTAs of a cluster along x.
template <typename... P>
cudaError_t launch_overlapped(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem,
                              cudaStream_t stream, int cluster, P... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Devices a process may drive (per-device launch state is kept in arrays).
constexpr int kMaxDevices = 64;

// Diagnostic switches, fixed when the library is compiled (-DQG_DIAG_FLAGS=...
// through QG_EXTRA_NVCC); shipped builds have none and the branches vanish.
// Results are wrong by design when any of bits 0-3, 7, 8, 11 is set:
// bit 0 skips the scale staging, bit 1 the MMAs, bit 2 the TMA loads (pair /
// solo kernels), bit 3 the epilogue stores, bit 7 the pair kernel's B loads,
// bit 8 its SFB loads, bit 11 all its scale loads and their shared memory.
// Bit 6 makes the decode GEMM's CTA (kDiag >> 16) and its quantiser kernels
// write %globaltimer stamps of their roles, and every decode GEMM CTA its
// start, end and epilogue milestones (into an unused partial slice); bit 9
// makes the pair kernel's first pair stamp its roles into C.  Used to
// attribute kernel time to its parts.
#ifndef QG_DIAG_FLAGS
#define QG_DIAG_FLAGS 0u
#endif
constexpr uint32_t kDiag = QG_DIAG_FLAGS;

// Fused epilogue of the GEMM (gemm_epilogue.cuh): out = act(alpha A B^T + bias)
// + residual.  The output has n columns, n / 2 for the gated activation.
enum : int { kEpiF32 = 0, kEpiBf16 = 1, kEpiMxfp8 = 2 };
struct EpiParams {
  int act;          // kAct* (qg_act.cuh)
  int bias_bf16;
  const void* bias;  // [n], may be null
  const void* res;   // residual, may be null
  int64_t ldr;
  int res_bf16, res_vec;  // *_vec: 16-byte accesses are legal for every full 32-column run
  int out_kind, out_vec;
  void* out;        // fp32 / bf16 rows with stride ldc, or e4m3 values, dense
  int64_t ldc;
  uint8_t* out_sf;
  int out_layout;
  int row_blocks;   // 128-row blocks of the output and the checkpoint
  int out_sf_blocks, z_sf_blocks;
  uint8_t* z_q;     // MXFP8 checkpoint of z = alpha A B^T + bias, may be null
  uint8_t* z_sf;
  int z_layout;
};

struct GemmParams {
  CUtensorMap tm_a;    // uint8 [rows][K bytes], box 128 B x kBM, SWIZZLE_128B
  CUtensorMap tm_b;    // uint8 [rows][K bytes], box 128 B x kBN, SWIZZLE_128B
  CUtensorMap tm_sfa;  // uint32 [scale_blocks][row_blocks][128], box (128, kBM/128, chunks)
  CUtensorMap tm_sfb;
  // bf16 C through TMA stores (pair kernel): box 64 x 32, SWIZZLE_128B.
  // n_out destinations receive the same tile: this GPU's C, or for the
  // fused column-parallel gather every rank's C (peer buffers mapped with
  // CUDA IPC).  n_out == 0: direct stores to c.
  static constexpr int kMaxOut = 8;
  CUtensorMap tm_out[kMaxOut];
  int n_out;
  void* c;
  int64_t ldc;  // elements
  int m, n, k;
  int num_m_tiles, num_n_tiles, num_k_blocks;
  int vec_ok;  // 16-byte vector stores are legal for every full 32-column run
  const float* a_ts;
  const float* b_ts;
  // NVFP4 output (requantising epilogue, pair kernel): values [m][n/2] and
  // one e4m3 scale per 16 columns in layout rq_layout (REF_LINEAR or an MMA
  // order with rq_row_blocks x rq_sf_blocks chunks), decoded with the tensor
  // scale *rq_ts; the output's amax is max-reduced into *rq_amax (optional).
  uint8_t* rq_q;
  uint8_t* rq_sf;
  const float* rq_ts;
  uint32_t* rq_amax;
  int rq_layout;
  int rq_row_blocks, rq_sf_blocks;
  uint32_t* status;
  uint64_t timeout_ns;
  EpiParams epi;  // out_kind 4..7 of launch_gemm_pair, launch_gemm_fused_rows
};

// Decode-shaped NVFP4 GEMM (gemm_skinny.cu): weights W [n][k] on the MMA's M
// side, activations X [m][k] (m <= 128) on its N side, stream-K over
// (weight tile, K block) units.  The activations are quantised by two small
// kernels launched ahead of it (launch_skinny_quant) with programmatic
// dependent launch, so the GEMM streams weights meanwhile.  A tile split
// between CTAs is summed by the last contributor to finish it (per-tile
// counters), in a fixed order, from per-CTA partial slices; whole tiles are
// written straight to C.
struct SkinnyParams {
  CUtensorMap tm_w;    // uint8 [n][k/2], box 128 B x 128 rows, SWIZZLE_128B
  CUtensorMap tm_x;    // uint8 [m][k/2] (the quantised xq), box 128 B x mma_n rows
  CUtensorMap tm_sfw;  // uint32 chunks, box (128, 1, 4)
  CUtensorMap tm_sfx;
  const void* x;       // activations, fp32 or bf16 [m][k]
  int x_bf16;
  uint8_t* xq;         // quantised activations [m][k/2]
  uint8_t* xsf;        // their scales, MMA layout
  float* x_ts;         // their tensor scale
  float* amax_part;    // [quantiser grid] per-CTA amax
  float* part;         // [grid][2][m][128] fp32 partial tiles
  uint32_t* cnt;       // [num_tiles][4] tile arrival counters, zeroed by the quantiser
  void* c;
  int64_t ldc;
  const float* w_ts;   // weight tensor scale (may be null)
  int out_bf16;
  int vec_ok;          // C rows start 16-byte aligned (16-byte stores legal)
  int m, n, k;
  int num_tiles, num_k_blocks;  // tiles of SkinnyShape::tile_rows, K blocks per stage
  int slices;                    // partial slices per CTA (2 per 128-row half)
  int num_counters;              // words of cnt the quantiser zeroes
  uint32_t* status;
  uint64_t timeout_ns;
};
// Tile geometry of the decode GEMM for m activation rows.
struct SkinnyShape {
  int tile_rows;      // weight rows per tile (128, or 256 as two halves)
  int stage_k_bytes;  // K bytes per stage (256 or 128)
  int sf_chunks;      // 64-K scale chunks per stage
  int halves;         // 128-row halves per tile
};
SkinnyShape skinny_shape(int64_t m);
cudaError_t launch_gemm_skinny(const SkinnyParams& p, int grid, cudaStream_t stream);
// Decode GEMM on CTA pairs (gemm_skinny_pair.cu), MMA N = 64 or 128: one whole
// skinny_pair_tile_rows()-row weight tile per pair (grid = 2 x tiles); tm_x
// has a box of mma_n / 2 rows (each CTA loads half of the activation rows).
cudaError_t launch_gemm_skinny_pair(const SkinnyParams& p, int grid, cudaStream_t stream);
int skinny_pair_tile_rows();
int skinny_quant_grid(int64_t xblocks, int sms);
cudaError_t launch_skinny_quant(const SkinnyParams& p, int grid, cudaStream_t stream);
int skinny_max_ctas();
int skinny_mma_n(int64_t m);

cudaError_t launch_gemm_blockscaled(const GemmParams& p, bool fp4, bool out_bf16, int grid,
                                    cudaStream_t stream);
// fmt: 0 MXFP8, 1 NVFP4, 2 MXFP4.  out_kind: 0 fp32 C, 1 bf16 C, 2 NVFP4
// output (rq_* fields; NVFP4 only), 3 bf16 C through TMA stores (n_out > 0)
// with eight epilogue warps, 4 the fused epilogue (epi), 5 its gated form, 6 and 7
// these two for rows that do not start on 16 bytes.
cudaError_t launch_gemm_pair(const GemmParams& p, int fmt, int out_kind, int grid,
                             cudaStream_t stream);
int pair_sf_chunks_per_stage(int fmt);
// The fused-epilogue GEMM for m <= 128 rows (gemm_fused_rows.cu): tm_a / tm_sfa
// are the weights B (box 128 rows, 256 for the gated activation), tm_b /
// tm_sfb the rows A (box rows_mma_n(m)); num_n_tiles tiles of the weights' boxes.
cudaError_t launch_gemm_fused_rows(const GemmParams& p, int fmt, cudaStream_t stream);
int rows_mma_n(int64_t m);
cudaError_t launch_gemm_solo(const GemmParams& p, bool fp4, bool out_bf16, int grid,
                             cudaStream_t stream);
int pair_tile_m();
int pair_tile_n();
int gemm_tile_m();
int gemm_tile_n();
int gemm_stage_k_bytes();
int gemm_sf_chunks_per_stage(bool fp4);

// Quantizer launches (quantize.cu).
cudaError_t launch_amax(const void* x, bool bf16, int64_t n, uint32_t* amax_bits,
                        cudaStream_t stream);
cudaError_t launch_quantize_nvfp4(const void* x, bool bf16, int64_t rows, int64_t k, int layout,
                                  uint8_t* q, uint8_t* sf, float* ts, const uint32_t* amax_bits,
                                  cudaStream_t stream);
cudaError_t launch_quantize_mxfp8(const void* x, bool bf16, int64_t rows, int64_t k, int layout,
                                  uint8_t* q, uint8_t* sf, cudaStream_t stream);
cudaError_t launch_quantize_mxfp4(const void* x, bool bf16, int64_t rows, int64_t k, int layout,
                                  uint8_t* q, uint8_t* sf, cudaStream_t stream);
cudaError_t launch_repack_nvfp4(const uint8_t* sq, const uint8_t* ssf, int src_layout,
                                uint8_t* dq, uint8_t* dsf, int dst_layout, int64_t rows,
                                int64_t k, cudaStream_t stream);
cudaError_t launch_repack_mx(bool fp4, const uint8_t* sq, const uint8_t* ssf, int src_layout,
                             uint8_t* dq, uint8_t* dsf, int dst_layout, int64_t rows, int64_t k,
                             cudaStream_t stream);
cudaError_t launch_e2m1_cvt_selftest(unsigned long long* out, cudaStream_t stream);
cudaError_t launch_wait_timeout_selftest(uint64_t timeout_ns, uint32_t* status,
                                         cudaStream_t stream);

// RMS norm with residual addition and MXFP8 output, and its gradient
// (rmsnorm.cu).  Strides in elements; k a multiple of 32, at most kMaxNormK.
constexpr int64_t kMaxNormK = 32768;
struct RmsNormParams {
  const void* x;
  const void* residual;  // may be null: h = x
  const void* weight;
  void* h;               // may be null
  float* rstd;           // may be null
  uint8_t* q;            // [rows][k]
  uint8_t* sf;
  int64_t ldx, ldr, ldh;
  int64_t rows, k;
  int64_t row_blocks, sf_blocks;
  int layout;
  float eps;
};
struct RmsNormBwdParams {
  const void* dy;
  const void* h;
  const void* weight;
  const void* dres;  // may be null
  const float* rstd;
  void* dx;
  float* dw_part;    // [rmsnorm_backward_parts(rows, k)][k] at most
  float* dw;         // [k]; null: not wanted
  int64_t lddy, ldh, lddres, lddx;
  int64_t rows, k;
};
cudaError_t launch_rmsnorm_mxfp8(const RmsNormParams& p, bool bf16, bool w_bf16,
                                 cudaStream_t stream);
// Rows of partial sums; 0 where the kernel writes dw itself.
int rmsnorm_backward_parts(int64_t rows, int64_t k);
cudaError_t launch_rmsnorm_backward(const RmsNormBwdParams& p, bool bf16, bool w_bf16,
                                    cudaStream_t stream);
// out[c] = sum over r < parts of part[r][c], in a fixed order.
cudaError_t launch_column_sum(const float* part, int parts, int64_t k, float* out,
                              cudaStream_t stream);

// Backward of an activation from its MXFP8 checkpoint, and the transposition of
// an MXFP8 matrix (act_backward.cu).
struct ActBackwardParams {
  const void* dout;      // [m][n], or [m][n / 2] for the gated activation
  int64_t ldd;
  const uint8_t* z_q;    // [m][n]; unused for act none: dz = dout
  const uint8_t* z_sf;
  int z_layout;
  int64_t m, n;
  uint8_t* dz_q;         // [m][n] (unused by the transposition)
  uint8_t* dz_sf;
  uint8_t* dzt_q;        // [n][mt]
  uint8_t* dzt_sf;
  int64_t mt;            // m rounded up to 32
  int out_layout;
  float* dbias_part;     // [ceil(m / 128)][n], or dbias itself where
                         // act_backward_joins(); null: no dbias
  int cluster_rows;      // set by the launch: a column tile's CTAs are one cluster
};
// Whether the kernel finishes dbias by itself (one row tile, or a cluster's).
bool act_backward_joins(int64_t m, int64_t n, int act);
cudaError_t launch_act_backward(const ActBackwardParams& p, int act, bool bf16,
                                cudaStream_t stream);
// dzt = z turned (dout, dz and dbias unused).
cudaError_t launch_transpose_mxfp8(const ActBackwardParams& p, cudaStream_t stream);

int num_sms();

}  // namespace qg
