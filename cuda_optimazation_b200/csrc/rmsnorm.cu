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
// backward, every byte crossing once.  A row belongs to a group of threads;
// thread t of it owns the 8-value vectors t, t + group, ... (kVec at most), so
// four neighbouring lanes hold one 32-value MX block and sixteen one 4-byte
// word of scales.
//
// Many rows (ring kernels): CTAs stay on their SM and every thread copies its
// own vectors of the next rows into shared memory ahead of time (cp.async, two
// or three rows deep), so the bytes in flight do not depend on registers or
// on where a CTA stands between its two barriers.  A thread reads back only
// what it copied itself, so the ring needs no barrier.  Elsewhere (few rows, rows too
// long for the ring, most fp32 rows): one CTA per row, values straight to registers;
// the rules stand at the launches with what was measured on both sides.
//
// Measured, of the 6.51 TB/s that a copy reaches here: forward, 16384 x 8192 bf16 with
// a residual, 152 us (6.2 TB/s); backward with dres 171 us (6.3 TB/s).  One row of
// 8192: 2.5 us; backward of 333 x 5152 fp32 8.2 us.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "qg_codec.cuh"
#include "qg_gemm.h"
#include "qg_ptx.cuh"

namespace qg {

namespace {

// Eight consecutive values as four fp32 pairs.
struct Vec8 {
  float2 v[4];
};

// Raw storage of eight consecutive values: 16 bytes of bf16 or 32 of fp32.
template <bool kBf16>
struct Raw8 {
  static constexpr int kChunks = kBf16 ? 1 : 2;
  uint4 c[kChunks];
  __device__ __forceinline__ Vec8 decode() const {
    Vec8 r;
    const uint32_t* w = &c[0].x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kBf16)
        r.v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      else
        r.v[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    }
    return r;
  }
};

template <bool kBf16>
constexpr int kElem = kBf16 ? 2 : 4;

// A row's own values, read once (streaming, and coherent: an output may be an
// input's own buffer).
template <bool kBf16>
__device__ __forceinline__ Raw8<kBf16> load_once(const void* base, int64_t elem) {
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) +
                                                  elem * kElem<kBf16>);
  Raw8<kBf16> r;
#pragma unroll
  for (int i = 0; i < Raw8<kBf16>::kChunks; ++i) r.c[i] = __ldcs(p + i);
  return r;
}

// The weight, which every row reads again.
template <bool kBf16>
__device__ __forceinline__ Raw8<kBf16> load_kept(const void* base, int64_t elem) {
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) +
                                                  elem * kElem<kBf16>);
  Raw8<kBf16> r;
#pragma unroll
  for (int i = 0; i < Raw8<kBf16>::kChunks; ++i) r.c[i] = __ldg(p + i);
  return r;
}

// bf16 rows by streaming stores, as the values below: left to L2's own order the forward
// pass over 16384 x 8192 took 168 us at full clocks and 157 under the power cap, streamed
// 152 and 161.  fp32 by plain ones: dw's shares, some in shared memory, are stored here too
// and read again at once.
template <bool kBf16>
__device__ __forceinline__ void store8(void* base, int64_t elem, const Vec8& x) {
  uint4* p = reinterpret_cast<uint4*>(static_cast<uint8_t*>(base) + elem * kElem<kBf16>);
  if constexpr (kBf16) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(x.v[i].x, x.v[i].y);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    __stcs(p, make_uint4(w[0], w[1], w[2], w[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      p[i] = make_uint4(__float_as_uint(x.v[2 * i].x), __float_as_uint(x.v[2 * i].y),
                        __float_as_uint(x.v[2 * i + 1].x), __float_as_uint(x.v[2 * i + 1].y));
  }
}

template <bool kBf16>
__device__ __forceinline__ const uint8_t* at_row(const void* base, int64_t row, int64_t ld) {
  return static_cast<const uint8_t*>(base) + row * ld * kElem<kBf16>;
}
// One input's row in a ring slot: 16-byte chunks, the first chunks of all
// vectors and then (fp32) the second ones, so that a warp's accesses are
// contiguous.  `at`: 32-bit shared-memory address; `second`: bytes from a vector's
// first chunk to its second.
template <bool kBf16>
__device__ __forceinline__ void ring_copy(uint32_t at, const uint8_t* from, uint32_t second) {
#pragma unroll
  for (int i = 0; i < Raw8<kBf16>::kChunks; ++i) copy_async_at(at + i * second, from + 16 * i);
}
template <bool kBf16>
__device__ __forceinline__ Raw8<kBf16> ring_read(uint32_t at, uint32_t second) {
  Raw8<kBf16> r;
#pragma unroll
  for (int i = 0; i < Raw8<kBf16>::kChunks; ++i) r.c[i] = lds128_at(at + i * second);
  return r;
}
__device__ __forceinline__ void ring_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int kLeft>
__device__ __forceinline__ void ring_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// Sum over the row's threads (blockDim.x of them: one warp, or the whole CTA) in
// a fixed order; every thread gets it.
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  __syncthreads();  // the previous sum's reads of red
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ void add_to(Vec8& a, const Vec8& b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) a.v[i] = add2(a.v[i], b.v[i]);
}
__device__ __forceinline__ void add_squares(float2& s, const Vec8& h) {
#pragma unroll
  for (int i = 0; i < 4; ++i) s = fma2(h.v[i], h.v[i], s);
}

// Where a row's scale words go: `at` for its first four blocks, `step` bytes
// further for each four more (the MMA layouts).
struct ScaleRow {
  uint8_t* at;
  int64_t step;
};
__device__ __forceinline__ ScaleRow scale_row(const RmsNormParams& p, int64_t row) {
  const int64_t in_chunk = (row & 31) * 16 + (row >> 5 & 3) * 4, br = row >> 7;
  if (p.layout == 1) return {p.sf + br * 512 + in_chunk, p.row_blocks * 512};
  if (p.layout == 2) return {p.sf + br * p.sf_blocks * 512 + in_chunk, 512};
  return {p.sf + row * (p.k / 32), 0};
}

// t = h * w of one vector (y without rstd) and the peak |t| of its MX block.
// Formed before the row's sum is known, so that little is left after it; the
// peak of y is the peak of t times rstd (rounding is monotonic).  Every lane of
// the warp takes part; a lane beyond the row brings zeros.
__device__ __forceinline__ float weighted(const Vec8& h, const Vec8& w, Vec8& t) {
#pragma unroll
  for (int i = 0; i < 4; ++i) t.v[i] = mul2(h.v[i], w.v[i]);
  float peak = max3_abs(t.v[0].x, t.v[0].y, t.v[1].x);
  peak = max3_abs(peak, t.v[1].y, t.v[2].x);
  peak = max3_abs(peak, t.v[2].y, t.v[3].x);
  return max3_abs(peak, t.v[3].y, 0.0f);
}
__device__ __forceinline__ float block_peak(float peak) {
  peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
  return fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
}

// y = t * rstd of vector v, quantised and stored (q: the row's values).
__device__ __forceinline__ void store_y(const RmsNormParams& p, uint8_t* q, const ScaleRow& sr,
                                        int v, bool in, const Vec8& t, float peak, float rstd,
                                        int lane) {
  float mul;
  const uint32_t code = mxfp8_scale_code(fmaxf(peak * rstd, 0.0f), mul);  // 0 beyond the row: padding
  if (in) {
    // Two products: rstd * mul may overflow where t is 0.
    float2 y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = mul2(mul2(t.v[i], both(rstd)), both(mul));
    __stcs(reinterpret_cast<uint2*>(q + v * 8),
           make_uint2(cvt_e4m3x4(y[0].x, y[0].y, y[1].x, y[1].y),
                      cvt_e4m3x4(y[2].x, y[2].y, y[3].x, y[3].y)));
  }
  if (p.layout == 0) {
    if (in && (lane & 3) == 0) sr.at[v / 4] = static_cast<uint8_t>(code);
  } else {
    // Codes of the word's four blocks, joined over lanes 0, 4, 8, 12 of 16.
    uint32_t word = code | __shfl_down_sync(0xffffffffu, code, 4) << 8;
    word |= __shfl_down_sync(0xffffffffu, word, 8) << 16;
    if (in && (lane & 15) == 0)
      *reinterpret_cast<uint32_t*>(sr.at + (v / 16) * sr.step) = word;
  }
}

// The scale words of the rows that fill the last 128-row chunks read as zero:
// threads `first`, first + step, ... write them, neighbours neighbouring words.
__device__ __forceinline__ void pad_scales(const RmsNormParams& p, int first, int step) {
  if (p.layout == 0) return;
  const int used = static_cast<int>(p.rows - (p.row_blocks - 1) * 128);
  if (used == 128) return;
  const int words = static_cast<int>(p.sf_blocks) * 128;
  for (int i = first; i < words; i += step) {
    const int bs = i >> 7, w = i & 127;
    if ((w >> 2) + (w & 3) * 32 < used) continue;
    const int64_t chunk = p.layout == 1 ? bs * p.row_blocks + p.row_blocks - 1
                                        : (p.row_blocks - 1) * p.sf_blocks + bs;
    reinterpret_cast<uint32_t*>(p.sf + chunk * 512)[w] = 0u;
  }
}

// ------------------------------------------------------------------ forward
// One CTA per row; CTAs past the rows write the padding.
template <bool kBf16, bool kWBf16, int kVec>
__global__ void __launch_bounds__(1024) rmsnorm_direct_kernel(const RmsNormParams p) {
  __shared__ float red[32];
  const int64_t row = blockIdx.x;
  griddep_launch_dependents();
  griddep_wait();
  if (row >= p.rows) {
    const int pads = static_cast<int>(gridDim.x - p.rows);
    pad_scales(p, static_cast<int>(row - p.rows) * blockDim.x + threadIdx.x, pads * blockDim.x);
    return;
  }
  const int nvec = static_cast<int>(p.k / 8);
  Vec8 t[kVec];
  float peak[kVec];
  float2 ss = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    peak[i] = 0.0f;
    if (v < nvec) {
      Vec8 h = load_once<kBf16>(p.x, row * p.ldx + v * 8).decode();
      const Vec8 w = load_kept<kWBf16>(p.weight, v * 8).decode();
      if (p.residual) add_to(h, load_once<kBf16>(p.residual, row * p.ldr + v * 8).decode());
      if (p.h) store8<kBf16>(p.h, row * p.ldh + v * 8, h);
      add_squares(ss, h);
      peak[i] = weighted(h, w, t[i]);
    }
    peak[i] = block_peak(peak[i]);
  }
  const float rstd = rsqrtf(row_sum(ss.x + ss.y, red) / static_cast<float>(p.k) + p.eps);
  if (threadIdx.x == 0 && p.rstd) p.rstd[row] = rstd;
  const ScaleRow sr = scale_row(p, row);
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    store_y(p, p.q + row * p.k, sr, v, v < nvec, t[i], peak[i], rstd, threadIdx.x & 31);
  }
}

// blockDim (group, rows at a time).
template <bool kBf16, bool kWBf16, int kVec, int kStages>
__global__ void __launch_bounds__(512) rmsnorm_ring_kernel(const RmsNormParams p) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[32];
  const int nvec = static_cast<int>(p.k / 8);
  const int row_bytes = static_cast<int>(p.k) * kElem<kBf16>;
  const int slot_bytes = p.residual ? 2 * row_bytes : row_bytes;
  const bool add = p.residual != nullptr, keep = p.h != nullptr;
  const uint32_t second = nvec * 16, hop = blockDim.x * 16;  // from vector to vector of a thread
  const uint32_t mine = smem_u32(ring) + threadIdx.y * kStages * slot_bytes + threadIdx.x * 16;
  const uint32_t end = mine + kStages * slot_bytes;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
  const int mine_vecs =  // of this thread
      (nvec - static_cast<int>(threadIdx.x) + static_cast<int>(blockDim.x) - 1) /
      static_cast<int>(blockDim.x);
  const uint32_t reach = blockDim.x * 8 * kElem<kBf16>;
  const uint8_t* x_next = at_row<kBf16>(p.x, first, p.ldx) + threadIdx.x * 8 * kElem<kBf16>;
  const uint8_t* r_next = at_row<kBf16>(p.residual, first, p.ldr) + threadIdx.x * 8 * kElem<kBf16>;
  const int64_t x_step = step * p.ldx * kElem<kBf16>, r_step = step * p.ldr * kElem<kBf16>;
  // Starts copying row `row`, and moves on by `step` rows.
  auto fetch = [&](int64_t row, uint32_t slot) {
    if (row < p.rows) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if (i < mine_vecs) {
          ring_copy<kBf16>(slot + i * hop, x_next + i * reach, second);
          if (add) ring_copy<kBf16>(slot + row_bytes + i * hop, r_next + i * reach, second);
        }
      }
    }
    x_next += x_step;
    r_next += r_step;
    ring_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s) fetch(first + s * step, mine + s * slot_bytes);
  Raw8<kWBf16> w[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nvec) w[i] = load_kept<kWBf16>(p.weight, v * 8);
  }
  const float inv_k = 1.0f / static_cast<float>(p.k);
  uint32_t slot = mine;
  uint8_t* q = p.q + first * p.k;
  uint8_t* h_out = static_cast<uint8_t*>(p.h) + first * p.ldh * kElem<kBf16>;
  for (int64_t row = first; row < p.rows; row += step) {
    ring_wait<kStages - 1>();
    Vec8 t[kVec];
    float peak[kVec];
    float2 ss = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      peak[i] = 0.0f;
      if (i < mine_vecs) {
        Vec8 h = ring_read<kBf16>(slot + i * hop, second).decode();
        if (add) add_to(h, ring_read<kBf16>(slot + row_bytes + i * hop, second).decode());
        if (keep) store8<kBf16>(h_out, (threadIdx.x + i * blockDim.x) * 8, h);
        add_squares(ss, h);
        peak[i] = weighted(h, w[i].decode(), t[i]);
      }
      peak[i] = block_peak(peak[i]);
    }
    fetch(row + kStages * step, slot);
    slot += slot_bytes;
    if (slot == end) slot = mine;
    const float rstd = rsqrtf(fmaf(row_sum(ss.x + ss.y, red), inv_k, p.eps));
    if (threadIdx.x == 0 && p.rstd) p.rstd[row] = rstd;
    const ScaleRow sr = scale_row(p, row);
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      store_y(p, q, sr, threadIdx.x + i * blockDim.x, i < mine_vecs, t[i], peak[i], rstd,
              threadIdx.x & 31);
    q += step * p.k;
    h_out += step * p.ldh * kElem<kBf16>;
  }
  ring_wait<0>();
  const int t = threadIdx.y * blockDim.x + threadIdx.x, n = blockDim.x * blockDim.y;
  pad_scales(p, static_cast<int>(blockIdx.x) * n + t, static_cast<int>(gridDim.x) * n);
}

// ------------------------------------------------------------------ backward
// dot += g xh and dw += dy xh of one vector.
template <bool kWBf16>
__device__ __forceinline__ float bwd_dot(const Vec8& dy, const Vec8& h, const Vec8& w, float rstd,
                                         Vec8& dw) {
  float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 t = mul2(dy.v[j], mul2(h.v[j], both(rstd)));
    dw.v[j] = add2(dw.v[j], t);
    s = fma2(t, w.v[j], s);
  }
  return s.x + s.y;
}

// dx of one vector: rstd (dy w - xh c) + dres.
__device__ __forceinline__ Vec8 bwd_dx(const Vec8& dy, const Vec8& h, const Vec8& w, float rstd,
                                       float c) {
  Vec8 d;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    d.v[j] = mul2(both(rstd), fma2(mul2(h.v[j], both(rstd)), both(-c), mul2(dy.v[j], w.v[j])));
  return d;
}

// dw of 128 bytes' worth of columns by one CTA of 16 warps: eight lanes span the
// columns (16 bytes each), the warp's four such groups and the warps take the
// rows in turn; the sums are joined in a fixed order.
template <bool kBf16>
__device__ __forceinline__ void column_dw(const RmsNormBwdParams& p, int64_t col0) {
  constexpr int kPairs = kBf16 ? 4 : 2;  // column pairs of a lane
  __shared__ float2 sums[16][8][kPairs];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t col = col0 + (lane & 7) * 2 * kPairs;
  float2 s[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) s[i] = make_float2(0.0f, 0.0f);
  if (col < p.k) {
    const uint8_t* dy = static_cast<const uint8_t*>(p.dy) + col * kElem<kBf16>;
    const uint8_t* h = static_cast<const uint8_t*>(p.h) + col * kElem<kBf16>;
#pragma unroll 4
    for (int row = warp * 4 + (lane >> 3); row < static_cast<int>(p.rows); row += 64) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(dy + row * p.lddy * kElem<kBf16>));
      const uint4 b = __ldg(reinterpret_cast<const uint4*>(h + row * p.ldh * kElem<kBf16>));
      const float2 r = both(__ldg(p.rstd + row));
      const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        if constexpr (kBf16)
          s[i] = fma2(make_float2(__uint_as_float(x[i] << 16), __uint_as_float(x[i] & 0xffff0000u)),
                      mul2(make_float2(__uint_as_float(y[i] << 16),
                                       __uint_as_float(y[i] & 0xffff0000u)), r), s[i]);
        else
          s[i] = fma2(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])),
                      mul2(make_float2(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1])),
                           r), s[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
#pragma unroll
    for (int o = 8; o <= 16; o *= 2)
      s[i] = add2(s[i], make_float2(__shfl_xor_sync(0xffffffffu, s[i].x, o),
                                    __shfl_xor_sync(0xffffffffu, s[i].y, o)));
    if (lane < 8) sums[warp][lane][i] = s[i];
  }
  __syncthreads();
  if (warp == 0 && lane < 8 && col < p.k) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      for (int w = 1; w < 16; ++w) s[i] = add2(s[i], sums[w][lane][i]);
      p.dw[col + 2 * i] = s[i].x;
      p.dw[col + 2 * i + 1] = s[i].y;
    }
  }
}

// kColumns (few rows): the first CTAs take the columns of dw, which need no row's
// sum, the others one row each: dy and h are read twice, the second time mostly
// from L2 where they fit it, and nothing is left to join.  dx may not be dy then.
// Otherwise CTA b takes rows b, b + grid, ...; each thread owns the same columns
// of all of them, so its share of dw stays in registers and is written once, to
// row b of the partial sums.
template <bool kBf16, bool kWBf16, int kVec, bool kColumns>
__global__ void __launch_bounds__(512, kColumns && kVec <= 2 ? 2 : 1)
    rmsnorm_backward_direct_kernel(const RmsNormBwdParams p) {
  __shared__ float red[32];
  griddep_launch_dependents();
  griddep_wait();
  if constexpr (kColumns) {
    if (blockIdx.x + p.rows < gridDim.x) {
      column_dw<kBf16>(p, static_cast<int64_t>(blockIdx.x) * (128 / kElem<kBf16>));
      return;
    }
  }
  const int64_t first = kColumns ? blockIdx.x + p.rows - gridDim.x : blockIdx.x;
  const int nvec = static_cast<int>(p.k / 8);
  const float inv_k = 1.0f / static_cast<float>(p.k);
  Vec8 dw[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) dw[i].v[j] = make_float2(0.0f, 0.0f);
  for (int64_t row = first; row < p.rows; row += gridDim.x) {
    const float rstd = __ldg(p.rstd + row);
    Raw8<kBf16> dy[kVec], h[kVec];
    Raw8<kWBf16> w[kVec];
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nvec) {
        dy[i] = load_once<kBf16>(p.dy, row * p.lddy + v * 8);
        h[i] = load_once<kBf16>(p.h, row * p.ldh + v * 8);
        w[i] = load_kept<kWBf16>(p.weight, v * 8);
        dot += bwd_dot<kWBf16>(dy[i].decode(), h[i].decode(), w[i].decode(), rstd, dw[i]);
      }
    }
    const float c = row_sum(dot, red) * inv_k;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nvec) {
        // By columns two CTAs share an SM's registers: w once more, from L1.
        if (kColumns) w[i] = load_kept<kWBf16>(p.weight, v * 8);
        Vec8 d = bwd_dx(dy[i].decode(), h[i].decode(), w[i].decode(), rstd, c);
        if (p.dres) add_to(d, load_once<kBf16>(p.dres, row * p.lddres + v * 8).decode());
        store8<kBf16>(p.dx, row * p.lddx + v * 8, d);
      }
    }
    if constexpr (kColumns) return;
  }
  if (!kColumns && p.dw) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nvec) store8<false>(p.dw_part, blockIdx.x * p.k + v * 8, dw[i]);
    }
  }
}

// blockDim (group, rows at a time).  dy and h are read from the ring twice
// instead of being held over the reduction.
template <bool kBf16, bool kWBf16, int kVec, int kStages>
__global__ void __launch_bounds__(512) rmsnorm_backward_ring_kernel(const RmsNormBwdParams p) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[32];
  const int nvec = static_cast<int>(p.k / 8);
  const float inv_k = 1.0f / static_cast<float>(p.k);
  const int row_bytes = static_cast<int>(p.k) * kElem<kBf16>;
  const int slot_bytes = p.dres ? 3 * row_bytes : 2 * row_bytes;
  const bool add = p.dres != nullptr;
  const uint32_t second = nvec * 16, hop = blockDim.x * 16;
  const uint32_t mine = smem_u32(ring) + threadIdx.y * kStages * slot_bytes + threadIdx.x * 16;
  const uint32_t end = mine + kStages * slot_bytes;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
  const int mine_vecs =
      (nvec - static_cast<int>(threadIdx.x) + static_cast<int>(blockDim.x) - 1) /
      static_cast<int>(blockDim.x);
  const uint32_t reach = blockDim.x * 8 * kElem<kBf16>, lead = threadIdx.x * 8 * kElem<kBf16>;
  const uint8_t* dy_next = at_row<kBf16>(p.dy, first, p.lddy) + lead;
  const uint8_t* h_next = at_row<kBf16>(p.h, first, p.ldh) + lead;
  const uint8_t* r_next = at_row<kBf16>(p.dres, first, p.lddres) + lead;
  const int64_t dy_step = step * p.lddy * kElem<kBf16>, h_step = step * p.ldh * kElem<kBf16>,
                r_step = step * p.lddres * kElem<kBf16>;
  auto fetch = [&](int64_t row, uint32_t slot) {
    if (row < p.rows) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if (i < mine_vecs) {
          const uint32_t at = slot + i * hop;
          ring_copy<kBf16>(at, dy_next + i * reach, second);
          ring_copy<kBf16>(at + row_bytes, h_next + i * reach, second);
          if (add) ring_copy<kBf16>(at + 2 * row_bytes, r_next + i * reach, second);
        }
      }
    }
    dy_next += dy_step;
    h_next += h_step;
    r_next += r_step;
    ring_commit();
  };
  Vec8 dw[kVec];
  Raw8<kWBf16> w[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) dw[i].v[j] = make_float2(0.0f, 0.0f);
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nvec) w[i] = load_kept<kWBf16>(p.weight, v * 8);
  }
#pragma unroll
  for (int s = 0; s < kStages; ++s) fetch(first + s * step, mine + s * slot_bytes);
  uint32_t slot = mine;
  uint8_t* out = static_cast<uint8_t*>(p.dx) + first * p.lddx * kElem<kBf16>;
  for (int64_t row = first; row < p.rows; row += step) {
    const float rstd = __ldg(p.rstd + row);
    ring_wait<kStages - 1>();
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      if (i < mine_vecs)
        dot += bwd_dot<kWBf16>(ring_read<kBf16>(slot + i * hop, second).decode(),
                               ring_read<kBf16>(slot + row_bytes + i * hop, second).decode(),
                               w[i].decode(), rstd, dw[i]);
    }
    const float c = row_sum(dot, red) * inv_k;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      if (i < mine_vecs) {
        const uint32_t at = slot + i * hop;
        Vec8 d = bwd_dx(ring_read<kBf16>(at, second).decode(),
                        ring_read<kBf16>(at + row_bytes, second).decode(), w[i].decode(), rstd, c);
        if (add) add_to(d, ring_read<kBf16>(at + 2 * row_bytes, second).decode());
        store8<kBf16>(out, (threadIdx.x + i * blockDim.x) * 8, d);
      }
    }
    fetch(row + kStages * step, slot);
    slot += slot_bytes;
    if (slot == end) slot = mine;
    out += step * p.lddx * kElem<kBf16>;
  }
  ring_wait<0>();
  if (!p.dw) return;
  if (blockDim.y == 1) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nvec) store8<false>(p.dw_part, blockIdx.x * p.k + v * 8, dw[i]);
    }
    return;
  }
  // The CTA's row groups, joined in order through the ring's memory.
  __syncthreads();
  float* sums = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nvec) store8<false>(sums, threadIdx.y * p.k + v * 8, dw[i]);
  }
  __syncthreads();
  for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < p.k; c += blockDim.x * blockDim.y) {
    float s = sums[c];
    for (int y = 1; y < static_cast<int>(blockDim.y); ++y) s += sums[y * p.k + c];
    p.dw_part[blockIdx.x * p.k + c] = s;
  }
}

// out[c] = sum over `parts` rows of part[.][c], in a fixed order: 32 threads of
// a column sum every 32nd row and are joined in shared memory.
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* part, int parts, int64_t k,
                                                          float* out) {
  __shared__ float sum[32][33];
  const int64_t c = blockIdx.x * 32ll + threadIdx.x;
  float s = 0.0f;
  if (c < k)
    for (int r = threadIdx.y; r < parts; r += 32) s += part[r * k + c];
  sum[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = sum[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int64_t oc = blockIdx.x * 32ll + threadIdx.y;
  if (threadIdx.x == 0 && oc < k) out[oc] = s;
}

// ------------------------------------------------------------------ shapes
constexpr int kRingSmem = 220 * 1024;  // shared memory of an SM that rings may take
constexpr int kRingVec = 4;            // vectors of a row per thread

// Ring kernels: rows of at most kRingVec x 512 vectors, one warp per row and
// eight rows per CTA up to 1024 values.  Three slots a row group where two
// such CTAs fit an SM, else two; none (stages 0) where a CTA does not fit or
// the rows do not go `rounds` times round the resident CTAs.
struct RingShape {
  int group = 0, rows = 0, stages = 0, smem = 0, grid = 0;
};
RingShape ring_shape(int64_t rows, int64_t k, int64_t slot_bytes, int rounds) {
  RingShape s;
  const int64_t nvec = k / 8;
  if (nvec > 512 * kRingVec) return s;
  s.group = static_cast<int>((nvec + kRingVec - 1) / kRingVec + 31) / 32 * 32;
  s.rows = s.group == 32 ? 8 : 1;
  const int64_t slots = slot_bytes * s.rows;
  const int stages = 2 * (3 * slots + 1024) <= kRingSmem ? 3 : 2;
  if (stages * slots > kRingSmem) return s;
  int64_t ctas = kRingSmem / (stages * slots + 1024);
  if (ctas < 1) ctas = 1;
  if (ctas > 512 / (s.group * s.rows)) ctas = 512 / (s.group * s.rows);  // 128 registers
  s.grid = static_cast<int>(ctas * num_sms());
  if (rows < static_cast<int64_t>(rounds) * s.grid * s.rows) return s;
  s.stages = stages;
  s.smem = static_cast<int>(stages * slots);
  return s;
}

// Direct kernels: whole warps, as many threads as the row has vectors, up to
// `most`.
struct RowShape {
  int threads, vec;
};
RowShape row_shape(int64_t k, int most) {
  const int64_t nvec = k / 8;
  RowShape s{};
  for (s.vec = 1; s.vec < 8 && nvec > static_cast<int64_t>(most) * s.vec; s.vec *= 2) {
  }
  s.threads = static_cast<int>((nvec + s.vec - 1) / s.vec + 31) / 32 * 32;
  return s;
}

template <auto kKernel, typename P>
cudaError_t launch_ring(const P& p, const RingShape& s, cudaStream_t stream) {
  static bool done[kMaxDevices] = {};  // of this kernel
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
    return cudaErrorInvalidDevice;
  if (!done[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem);
    if (e != cudaSuccess) return e;
    done[dev] = true;
  }
  kKernel<<<s.grid, dim3(s.group, s.rows), s.smem, stream>>>(p);
  return cudaGetLastError();
}

// Where the ring is ahead of one CTA a row.  Measured, us ring / direct, with a residual:
// bf16 4800 x 128 6.0 / 5.6, 7200 x 256 7.4 / 8.3, 9600 x 512 12.1 / 10.7, 16384 x 512
// 15.8 / 17.9, 32768 x 1024 42.1 / 40.4; 16384 x 2048 41.2 / 41.0, 4800 x 4096 27.5 /
// 25.6, 9600 x 4096 46.4 / 49.3, 1200 x 8192 18.8 / 15.7, 4800 x 8192 46.9 / 53.2, 1200 x
// 16384 28.3 / 39.8; fp32 9600 x 128 10.1 / 10.7, 9600 x 256 13.0 / 10.8, 16384 x 4096
// 221 / 129, 2400 x 12288 98 / 73: such rows take twice the ring for the same arithmetic,
// and too few threads are left to keep up.
bool forward_ring(int64_t rows, int64_t k, int64_t slot_bytes, bool bf16) {
  if (k <= 1024) return slot_bytes <= 2048 && rows >= 6144 && rows >= 8 * slot_bytes;
  return bf16 && (k > 12288 || rows * k * k >= 1ll << 37);
}

template <bool kBf16, bool kWBf16>
cudaError_t launch_norm(const RmsNormParams& p, cudaStream_t stream) {
  const int64_t slot = p.k * kElem<kBf16> * (p.residual ? 2 : 1);
  if (forward_ring(p.rows, p.k, slot, kBf16)) {
    const RingShape r = ring_shape(p.rows, p.k, slot, 2);  // (one round prefetches nothing)
    if (r.stages == 3)
      return launch_ring<rmsnorm_ring_kernel<kBf16, kWBf16, kRingVec, 3>>(p, r, stream);
    if constexpr (kBf16) {  // (fp32: short rows alone, of which three stages fit)
      if (r.stages == 2)
        return launch_ring<rmsnorm_ring_kernel<kBf16, kWBf16, kRingVec, 2>>(p, r, stream);
    }
  }
  const RowShape s = row_shape(p.k, 1024);
  // Padding words of the last chunks, four per thread.
  int pads = 0;
  if (p.layout != 0 && p.rows % 128 != 0)
    pads = static_cast<int>((p.sf_blocks * 128 + 4 * s.threads - 1) / (4 * s.threads));
  const int grid = static_cast<int>(p.rows) + pads;
  auto kernel = s.vec == 1   ? rmsnorm_direct_kernel<kBf16, kWBf16, 1>
                : s.vec == 2 ? rmsnorm_direct_kernel<kBf16, kWBf16, 2>
                             : rmsnorm_direct_kernel<kBf16, kWBf16, 4>;
  return launch_overlapped(kernel, dim3(grid), dim3(s.threads), 0, stream, 1, p);
}

int backward_direct_grid(int64_t rows) {
  const int64_t most = 2ll * num_sms();
  return static_cast<int>(rows < most ? rows : most);
}

// Which gradient kernel; measured, us, with dres.
// By columns (see the direct kernel) up to 512 rows; against partial sums bf16 1 x 8192
// 3.1 / 5.3, 512 x 1024 3.7 / 5.5, 512 x 4096 7.1 / 11.7, 290 x 16384 18.5 / 22.9, 512 x
// 32768 57.5 / 70.1, against the ring fp32 384 x 8192 14.9 / 22.5, 384 x 9376 22.8 / 24.9,
// bf16 512 x 8192 12.2 / 15.2, but 384 x 16384 25.6 / 21.1.  Beyond 512 rows it depends on
// k: 2000 x 32 8.8 / 7.3, 2000 x 1024 13.8 / 14.4, 4000 x 1024 25.9 / 24.6.
// The ring against the direct kernel: bf16 2400 x 256 6.6 / 10.0, 1400 x 1280 10.9 / 12.2,
// 520 x 6144 13.7 / 23.2, 4800 x 8192 58.7 / 107.7, in between from two rounds on (800 x
// 2048 10.7 / 9.3, 1480 x 2048 12.9 / 13.1); fp32 2400 x 512 12.4 / 17.1, 3600 x 768 19.6 /
// 24.8, 2400 x 1024 19.9 / 19.0, 4800 x 1024 28.5 / 32.3, 4800 x 1536 40.2 / 35.7, 4800 x
// 8192 193 / 137, where two CTAs an SM find their rings (4096 is a direct thread's second
// vector) 2400 x 4096 47 / 42, 4608 53 / 60, 5120 69 / 62, without dres 9600 x 2560 78 /
// 63, 9600 x 4096 120 / 134, 9600 x 7168 203 / 224, 4800 x 8192 138 / 129, and where a
// direct thread would hold four vectors 4800 x 9376 184 / 236.
struct BackwardPlan {
  RingShape ring;  // stages 0: none
  bool columns = false;
  int parts = 0;  // rows of partial sums of dw
};
BackwardPlan backward_plan(int64_t rows, int64_t k, int elem, int inputs) {
  BackwardPlan p;
  p.columns = rows <= 512;
  if (p.columns && (elem == 4 || k <= 8192)) return p;
  const bool f32_too = k <= 768 || (k <= 1280 && rows >= 2560) || k > 8192 ||
                       (inputs == 2 ? k >= 3104 && k <= 7168 : k > 4096 && k <= 4608);
  if (elem == 2 || f32_too)
    p.ring = ring_shape(rows, k, k * elem * inputs,
                        k <= 1536 || (k >= 3104 && k <= 8192) ? 1 : 2);
  if (p.ring.stages) p.columns = false;
  if (!p.columns) p.parts = p.ring.stages ? p.ring.grid : backward_direct_grid(rows);
  return p;
}

template <bool kBf16, bool kWBf16, bool kColumns>
cudaError_t launch_bwd_direct(const RmsNormBwdParams& p, int grid, cudaStream_t stream) {
  RowShape s = row_shape(p.k, 512);
  if (kColumns) s.threads = 512;
  auto kernel = rmsnorm_backward_direct_kernel<kBf16, kWBf16, 8, kColumns>;
  if (s.vec == 1) kernel = rmsnorm_backward_direct_kernel<kBf16, kWBf16, 1, kColumns>;
  if constexpr (!kBf16 || kColumns) {  // (bf16 rows of these widths take the ring)
    if (s.vec == 2) kernel = rmsnorm_backward_direct_kernel<kBf16, kWBf16, 2, kColumns>;
    if (s.vec == 4) kernel = rmsnorm_backward_direct_kernel<kBf16, kWBf16, 4, kColumns>;
  }
  return launch_overlapped(kernel, dim3(grid), dim3(s.threads), 0, stream, 1, p);
}

template <bool kBf16, bool kWBf16>
cudaError_t launch_norm_bwd(const RmsNormBwdParams& p, cudaStream_t stream) {
  const BackwardPlan plan = backward_plan(p.rows, p.k, kElem<kBf16>, p.dres ? 3 : 2);
  const RingShape& r = plan.ring;
  if (plan.columns) {
    const int64_t per = 128 / kElem<kBf16>, columns = p.dw ? (p.k + per - 1) / per : 0;
    return launch_bwd_direct<kBf16, kWBf16, true>(p, static_cast<int>(p.rows + columns), stream);
  }
  const cudaError_t e =
      r.stages == 3
          ? launch_ring<rmsnorm_backward_ring_kernel<kBf16, kWBf16, kRingVec, 3>>(p, r, stream)
      : r.stages == 2
          ? launch_ring<rmsnorm_backward_ring_kernel<kBf16, kWBf16, kRingVec, 2>>(p, r, stream)
          : launch_bwd_direct<kBf16, kWBf16, false>(p, plan.parts, stream);
  if (e != cudaSuccess || !p.dw) return e;
  return launch_column_sum(p.dw_part, plan.parts, p.k, p.dw, stream);
}

}  // namespace

cudaError_t launch_rmsnorm_mxfp8(const RmsNormParams& p, bool bf16, bool w_bf16,
                                 cudaStream_t stream) {
  if (bf16)
    return w_bf16 ? launch_norm<true, true>(p, stream) : launch_norm<true, false>(p, stream);
  return w_bf16 ? launch_norm<false, true>(p, stream) : launch_norm<false, false>(p, stream);
}

int rmsnorm_backward_parts(int64_t rows, int64_t k) {
  int most = 0;
  for (int inputs = 2; inputs <= 3; ++inputs)
    for (int elem = 2; elem <= 4; elem += 2) {
      const int parts = backward_plan(rows, k, elem, inputs).parts;
      if (parts > most) most = parts;
    }
  return most;
}

cudaError_t launch_rmsnorm_backward(const RmsNormBwdParams& p, bool bf16, bool w_bf16,
                                    cudaStream_t stream) {
  if (bf16)
    return w_bf16 ? launch_norm_bwd<true, true>(p, stream)
                  : launch_norm_bwd<true, false>(p, stream);
  return w_bf16 ? launch_norm_bwd<false, true>(p, stream)
                : launch_norm_bwd<false, false>(p, stream);
}

cudaError_t launch_column_sum(const float* part, int parts, int64_t k, float* out,
                              cudaStream_t stream) {
  column_sum_kernel<<<static_cast<unsigned>((k + 31) / 32), dim3(32, 32), 0, stream>>>(part, parts,
                                                                                     k, out);
  return cudaGetLastError();
}

}  // namespace qg
