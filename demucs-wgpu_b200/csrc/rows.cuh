// Layer norm and 8-bit quantisation of rows (dmx_layer_norm,
// dmx_quantize_rows, dmx_layer_norm_quantize).
//
//   mean = sum x / C,  var = sum (x - mean)^2 / C,  rstd = 1 / sqrt(var + eps)
//   y = (x - mean) rstd weight + bias
//   scale = max |y| / 127,  q = rint(y / scale)
//
// The variance is taken about the mean (not as a difference of squares), so a
// row whose mean is large against its spread keeps its digits. A row holding
// an infinity or a NaN gets a non-finite scale and q = 0, so every product
// with it is NaN; an all-zero row gets scale 0 and q = 0.
//
// Bound by HBM: a row is read once, held in registers through its two or three
// reductions, and written once. Rows of up to 1024 columns belong to a warp
// (or half or a quarter of one), so nothing waits on other warps and dozens of
// rows per SM are in flight; up to 16384 columns to a block of as many threads
// as 16 values each take; longer rows are re-read (from L2) for each
// reduction.
#pragma once

#include <algorithm>

#include "ops.h"
#include "ops_common.cuh"

namespace dmx {

enum { ROWS_NORM = 0, ROWS_NORM_QUANTIZE = 1, ROWS_QUANTIZE = 2 };

// q = rint(v / scale) of a correctly rounded quotient. v times the rounded
// reciprocal is within 127 * 3 * 2^-24 < 1e-4 of it, so only a product that
// near a tie needs the division; a subnormal scale, whose reciprocal can
// overflow, always takes it.
struct Quantizer {
  float scale, inv;
  bool usable, divide;
  DMX_DEVICE explicit Quantizer(uint32_t top_bits) {
    scale = __fdiv_rn(__uint_as_float(top_bits), 127.f);
    usable = scale > 0.f && scale < INFINITY;
    divide = scale < 1.17549435e-38f;
    inv = usable && !divide ? __frcp_rn(scale) : 0.f;
  }
  DMX_DEVICE int operator()(float v) const {
    if (!usable) return 0;
    const float t = v * inv;
    float q = rintf(t);
    if (divide || fabsf(fabsf(t - q) - 0.5f) < 1e-4f) q = rintf(__fdiv_rn(v, scale));
    return (int)fminf(fmaxf(q, -127.f), 127.f);
  }
  DMX_DEVICE void store(int8_t* row, const Pieces& p, bool vec8, int j, const float* v) const {
    if (vec8 && p.vec && p.whole(j)) {
      uint32_t w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[h] = ((uint32_t)(*this)(v[4 * h]) & 255u) | (((uint32_t)(*this)(v[4 * h + 1]) & 255u) << 8) |
               (((uint32_t)(*this)(v[4 * h + 2]) & 255u) << 16) | ((uint32_t)(*this)(v[4 * h + 3]) << 24);
      *reinterpret_cast<uint2*>(row + p.col(j, 0)) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (p.has(j, e)) row[p.col(j, e)] = (int8_t)(*this)(v[e]);
    }
  }
};

// Reductions over the threads of one row: LANES neighbouring lanes, or (0) a block.
template <int LANES>
struct RowSum {
  DMX_DEVICE float sum(float v, float*) const {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  DMX_DEVICE uint32_t max(uint32_t v, uint32_t*) const {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = ::max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
};
template <>
struct RowSum<0> {
  // `sh` is not in use for anything else until the block's next barrier
  DMX_DEVICE float sum(float v, float* sh) const {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = blockDim.x / 32, lane = threadIdx.x & 31;
    return warp_sum(lane < warps ? sh[lane] : 0.f);
  }
  DMX_DEVICE uint32_t max(uint32_t v, uint32_t* sh) const {
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = blockDim.x / 32, lane = threadIdx.x & 31;
    return __reduce_max_sync(0xffffffffu, lane < warps ? sh[lane] : 0u);
  }
};

// One row held in NV pieces per thread.
template <typename XT, int MODE, int LANES, int NV>
DMX_DEVICE void row_in_registers(const RowArgs& a, int64_t row, bool live, const Pieces& p,
                                 bool q_vec, float (*sh)[32]) {
  const RowSum<LANES> over;
  const XT* x = static_cast<const XT*>(a.x) + row * a.x_ld;
  float v[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) p.load(x, j, v[j]);
  if (MODE != ROWS_QUANTIZE) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[j][e];
    const float mean = over.sum(s, sh[0]) / (float)a.cols;
    s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool whole = p.whole(j);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[j][e] = whole || p.has(j, e) ? v[j][e] - mean : 0.f;
        s = fmaf(v[j][e], v[j][e], s);
      }
    }
    const float rstd = 1.f / sqrtf(over.sum(s, sh[1]) / (float)a.cols + a.eps);
    if (p.t == 0 && live) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] *= rstd;
      if (a.weight) {
        p.load(a.weight, a.param_type, j, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] *= w[e];
      }
      if (a.bias) {
        p.load(a.bias, a.param_type, j, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] += w[e];
      }
    }
  } else if (a.col_scale) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float w[8];
      p.load(a.col_scale, j, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] *= w[e];
    }
  }
  if (MODE == ROWS_NORM) {
    if (!live) return;
#pragma unroll
    for (int j = 0; j < NV; ++j) p.store(a.y, a.y_type, row * a.y_ld, j, v[j]);
    return;
  }
  // a NaN's bits are above infinity's, so it is kept by the maximum; past the
  // row's end a NaN mean or rstd must not count
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const bool whole = p.whole(j);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (whole || p.has(j, e)) top = ::max(top, __float_as_uint(fabsf(v[j][e])));
  }
  const Quantizer quant(over.max(top, reinterpret_cast<uint32_t*>(sh[2])));
  if (!live) return;
  if (p.t == 0) a.scale[row] = quant.scale;
#pragma unroll
  for (int j = 0; j < NV; ++j) quant.store(a.q + row * a.q_ld, p, q_vec, j, v[j]);
}

constexpr int kRowsThreads = 256;

template <typename XT, int MODE, int LANES, int NV>
__global__ void __launch_bounds__(kRowsThreads) rows_warp_kernel(const RowArgs a, int vec, bool q_vec) {
  const int64_t at = (int64_t)blockIdx.x * (kRowsThreads / LANES) + threadIdx.x / LANES;
  // lanes without a row of their own follow the last one's, for the shuffles
  const bool live = at < a.rows;
  const Pieces p = {(int)(threadIdx.x % LANES), LANES, a.cols, vec};
  row_in_registers<XT, MODE, LANES, NV>(a, live ? at : a.rows - 1, live, p, q_vec, nullptr);
}

template <typename XT, int MODE, int NV>
__global__ void __launch_bounds__(1024) rows_block_kernel(const RowArgs a, int vec, bool q_vec) {
  __shared__ float sh[3][32];
  const Pieces p = {(int)threadIdx.x, (int)blockDim.x, a.cols, vec};
  row_in_registers<XT, MODE, 0, NV>(a, blockIdx.x, true, p, q_vec, sh);
}

// Rows too long for registers: one block re-reads its row for each reduction.
template <typename XT, int MODE>
__global__ void __launch_bounds__(1024) rows_long_kernel(const RowArgs a, int vec, bool q_vec) {
  __shared__ float sh[3][32];
  const RowSum<0> over;
  const Pieces p = {(int)threadIdx.x, (int)blockDim.x, a.cols, vec};
  const int pieces = (a.cols - 1) / ((int)blockDim.x * 8) + 1;
  const int64_t row = blockIdx.x;
  const XT* x = static_cast<const XT*>(a.x) + row * a.x_ld;
  float v[8], w[8], mean = 0.f, rstd = 1.f;
  if (MODE != ROWS_QUANTIZE) {
    float s = 0.f;
    for (int j = 0; j < pieces; ++j) {
      p.load(x, j, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[e];
    }
    mean = over.sum(s, sh[0]) / (float)a.cols;
    s = 0.f;
    for (int j = 0; j < pieces; ++j) {
      p.load(x, j, v, mean);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(v[e] - mean, v[e] - mean, s);
    }
    rstd = 1.f / sqrtf(over.sum(s, sh[1]) / (float)a.cols + a.eps);
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
  auto values = [&](int j) {
    p.load(x, j, v);
    if (MODE != ROWS_QUANTIZE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (v[e] - mean) * rstd;
      if (a.weight) {
        p.load(a.weight, a.param_type, j, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= w[e];
      }
      if (a.bias) {
        p.load(a.bias, a.param_type, j, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += w[e];
      }
    } else if (a.col_scale) {
      p.load(a.col_scale, j, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= w[e];
    }
  };
  if (MODE == ROWS_NORM) {
    for (int j = 0; j < pieces; ++j) {
      values(j);
      p.store(a.y, a.y_type, row * a.y_ld, j, v);
    }
    return;
  }
  uint32_t top = 0;
  for (int j = 0; j < pieces; ++j) {
    values(j);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (p.has(j, e)) top = ::max(top, __float_as_uint(fabsf(v[e])));
  }
  const Quantizer quant(over.max(top, reinterpret_cast<uint32_t*>(sh[2])));
  if (threadIdx.x == 0) a.scale[row] = quant.scale;
  for (int j = 0; j < pieces; ++j) {
    values(j);
    quant.store(a.q + row * a.q_ld, p, q_vec, j, v);
  }
}

template <typename XT, int MODE, int LANES, int NV>
void launch_rows_warp(const RowArgs& a, int vec, bool q_vec, cudaStream_t s) {
  constexpr int per = kRowsThreads / LANES;
  rows_warp_kernel<XT, MODE, LANES, NV>
      <<<(unsigned)((a.rows + per - 1) / per), kRowsThreads, 0, s>>>(a, vec, q_vec);
}

template <typename XT, int MODE>
void launch_rows_mode(const RowArgs& a, int vec, bool q_vec, cudaStream_t s) {
  if (a.cols <= 64) return launch_rows_warp<XT, MODE, 8, 1>(a, vec, q_vec, s);
  if (a.cols <= 128) return launch_rows_warp<XT, MODE, 16, 1>(a, vec, q_vec, s);
  if (a.cols <= 256) return launch_rows_warp<XT, MODE, 32, 1>(a, vec, q_vec, s);
  if (a.cols <= 512) return launch_rows_warp<XT, MODE, 32, 2>(a, vec, q_vec, s);
  if (a.cols <= 1024) return launch_rows_warp<XT, MODE, 32, 4>(a, vec, q_vec, s);
  const unsigned rows = (unsigned)a.rows;
  if (a.cols > 16384) {
    rows_long_kernel<XT, MODE><<<rows, 1024, 0, s>>>(a, vec, q_vec);
    return;
  }
  const int threads = ((a.cols + 15) / 16 + 31) / 32 * 32;
  rows_block_kernel<XT, MODE, 2><<<rows, threads, 0, s>>>(a, vec, q_vec);
}

template <typename XT>
void launch_rows_typed(const RowArgs& a, cudaStream_t s) {
  int vec = vec_of(a.x, a.x_ld, sizeof(XT));
  auto narrow = [&vec](int other) { vec = std::min(vec, other); };
  if (a.norm) {
    narrow(vec_of(a.weight, 0, type_size(a.param_type)));
    narrow(vec_of(a.bias, 0, type_size(a.param_type)));
  }
  if (a.y) {
    narrow(vec_of(a.y, a.y_ld, type_size(a.y_type)));
    return launch_rows_mode<XT, ROWS_NORM>(a, vec, false, s);
  }
  narrow(vec_of(a.col_scale, 0, 4));
  const bool q_vec = reinterpret_cast<uintptr_t>(a.q) % 8 == 0 && a.q_ld % 8 == 0;
  if (a.norm) launch_rows_mode<XT, ROWS_NORM_QUANTIZE>(a, vec, q_vec, s);
  else launch_rows_mode<XT, ROWS_QUANTIZE>(a, vec, q_vec, s);
}

}  // namespace dmx
