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
// reductions, and written once. Rows of up to 1024 columns (2048 of 16 bits)
// belong to a warp (or half or a quarter of one), which waits for no other;
// up to 16384 columns to a block; longer rows are re-read (from L2) for each
// reduction. 16-bit rows are held as they lie and unpacked in every pass: one
// more instruction per value and pass, half the registers, and so twice the
// rows in flight. Measured: norm 60000 x 1024 f32 78 us (6330 GB/s), 112896 x
// 512 f32 -> bf16 62 us (5610), 112896 x 512 bf16 56 us (4120: by issue slots);
// quantise 112896 x 2048 bf16 145 us (4790); norm of 1 x 512 1.8 us.
#pragma once

#include <algorithm>

#include "ops.h"
#include "ops_common.cuh"

namespace dmx {

enum { ROWS_NORM = 0, ROWS_NORM_QUANTIZE = 1, ROWS_QUANTIZE = 2 };

// max(|a|, |b|, |c|); a NaN among them comes out as a NaN
DMX_DEVICE float max3_abs(float a, float b, float c) {
  float m;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}

// q = rint(v / scale) of the correctly rounded quotient: t = v * inv with inv the
// correctly rounded reciprocal, then one step t + (v - t scale) inv with fused
// products, which rounds as the quotient does (Markstein 1990) unless the
// scale's significand is all ones or the remainder underflows; rows with such
// a scale divide. Every value goes this way: ties are no rarity among 16-bit
// inputs, whose quotients have few digits, and a branch for values near one
// took most pieces (112896 x 2048 bf16: 235 us against 145). The integer is
// read off the sum with 1.5 * 2^23, whose last place is 1; the conversion
// instructions share the special-function unit, which two of them per value
// kept busy for longer than the row's memory traffic (316 us).
struct Quantizer {
  float scale, inv;
  bool usable, divide;
  DMX_DEVICE explicit Quantizer(uint32_t top_bits) {
    scale = __fdiv_rn(__uint_as_float(top_bits), 127.f);
    usable = scale > 0.f && scale < INFINITY;
    // |t| >= 1/4 (less rounds to 0): the remainder's last place is 2^-26 of the scale's
    divide = scale < 0x1p-100f || (__float_as_uint(scale) & 0x7fffffu) == 0x7fffffu;
    inv = usable && !divide ? __frcp_rn(scale) : 0.f;
  }
  // eight integers as bytes
  DMX_DEVICE uint2 operator()(const float* v) const {
    if (!usable) return make_uint2(0, 0);
    uint32_t q[8];
    if (!divide) {
      const float2 inv2 = make_float2(inv, inv), minus = make_float2(-scale, -scale),
                   up = make_float2(12582912.f, 12582912.f);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float2 x = make_float2(v[e], v[e + 1]);
        float2 t = __fmul2_rn(x, inv2);
        t = __ffma2_rn(__ffma2_rn(t, minus, x), inv2, t);
        t = __fadd2_rn(t, up);
        q[e] = __float_as_uint(t.x);
        q[e + 1] = __float_as_uint(t.y);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        q[e] = (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(v[e], scale)), -127.f), 127.f);
    }
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[h] = __byte_perm(__byte_perm(q[4 * h], q[4 * h + 1], 0x0040),
                         __byte_perm(q[4 * h + 2], q[4 * h + 3], 0x0040), 0x5410);
    return make_uint2(w[0], w[1]);
  }
  template <bool VEC>
  DMX_DEVICE void store(int8_t* row, const Pieces<VEC>& p, bool q_vec, int j, const float* v) const {
    const uint2 w = (*this)(v);
    if (VEC && q_vec && p.whole(j)) {
      *reinterpret_cast<uint2*>(row + p.col(j, 0)) = w;
    } else if (p.ragged() || !q_vec) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (p.has(j, e)) row[p.col(j, e)] = (int8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
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

// Piece j's values past the row's end become 0.
template <bool VEC>
DMX_DEVICE void mask8(const Pieces<VEC>& p, int j, float* v) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = p.has(j, e) ? v[e] : 0.f;
}

constexpr int kRowsThreads = 256;

// One row held in NV pieces per thread; PT is the parameters' type. Without
// `live` the lanes only take part in the shuffles.
template <typename XT, typename PT, int MODE, int LANES, int NV, bool SHIFT, bool VEC>
DMX_DEVICE void row_in_registers(const RowArgs& a, int64_t row, bool live, const Pieces<VEC>& p,
                                 bool q_vec, float (*sh)[32], float* cross) {
  const RowSum<LANES> over;
  const auto weight = array_of(a.weight, a.param_type, PT());
  const auto bias = array_of(a.bias, a.param_type, PT());
  uint32_t raw[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const XT* x = static_cast<const XT*>(a.x) + row * a.x_ld;
    if constexpr (SHIFT) p.fetch_shifted(x, j, raw[j]);
    else p.fetch(x, j, raw[j]);
  }
  auto get = [&](int j, float* v) { Pieces<VEC>::template unpack<XT>(raw[j], v); };
  float v[8];
  if (MODE == ROWS_QUANTIZE) {
    auto value = [&](int j) {
      get(j, v);
      if (a.col_scale) {
        float w[8];
        p.load(a.col_scale, j, w);
        times8(v, w);
      }
    };
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      value(j);
#pragma unroll
      for (int e = 0; e < 8; e += 2) top = max3_abs(top, v[e], v[e + 1]);
    }
    const Quantizer quant(over.max(__float_as_uint(top), reinterpret_cast<uint32_t*>(sh[2])));
    if (!live) return;
    if (p.t == 0) a.scale[row] = quant.scale;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      value(j);
      quant.store(a.q + row * a.q_ld, p, q_vec, j, v);
    }
    return;
  }
  // the forms for a few rows, where a load's latency counts, fetch the
  // parameters with the row
  constexpr bool kEarly = NV == 1 || (LANES == 32 && NV == 2);
  constexpr int kHold = kEarly ? NV : 1;
  uint32_t wr[kHold][8], br[kHold][8];
  if (kEarly) {
    if (weight)
#pragma unroll
      for (int j = 0; j < kHold; ++j) p.fetch(weight, j, wr[j]);
    if (bias)
#pragma unroll
      for (int j = 0; j < kHold; ++j) p.fetch(bias, j, br[j]);
  }
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    get(j, v);
#pragma unroll
    for (int e = 0; e < 8; e += 2) s = __fadd2_rn(s, make_float2(v[e], v[e + 1]));
  }
  const float mean = over.sum(s.x + s.y, sh[0]) / (float)a.cols;
  s = make_float2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    get(j, v);
    centre8(v, mean);
    if (p.ragged()) mask8(p, j, v);
    float2 t = s;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float2 d = make_float2(v[e], v[e + 1]);
      t = __ffma2_rn(d, d, t);
    }
    // a piece past the row's end holds -mean: left out whole, as cheaper than masked
    const bool in = p.has(j, 0);
    s = make_float2(in ? t.x : s.x, in ? t.y : s.y);
  }
  const float rstd = 1.f / sqrtf(over.sum(s.x + s.y, sh[1]) / (float)a.cols + a.eps);
  if (p.t == 0 && live) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  auto value = [&](int j, float* v) {
    get(j, v);
    centre8(v, mean);
    scale8(v, rstd);
    float w[8];
    if (weight) {
      if (!kEarly) p.fetch(weight, j, wr[0]);
      Pieces<VEC>::template unpack<PT>(wr[kEarly ? j : 0], w);
      times8(v, w);
    }
    if (bias) {
      if (!kEarly) p.fetch(bias, j, br[0]);
      Pieces<VEC>::template unpack<PT>(br[kEarly ? j : 0], w);
      plus8(v, w);
    }
  };
  if (MODE == ROWS_NORM) {
    if constexpr (SHIFT) {
      constexpr int kLanes = LANES ? LANES : 32;
      const int64_t row0 = LANES ? (int64_t)blockIdx.x * (kRowsThreads / kLanes) + threadIdx.x / 32 * (32 / kLanes) : row;
      with_type(a.y_type, [&](auto type) {
        using T = decltype(type);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          value(j, v);
          store_crossed<kLanes>(reinterpret_cast<T*>(cross + threadIdx.x / 32 * 256), v,
                                static_cast<T*>(a.y), a.y_ld, row0, LANES ? a.rows : row + 1,
                                (j * p.threads + p.t / kLanes * kLanes) * 8, a.cols);
        }
      });
      return;
    }
    if (!live) return;
    with_type(a.y_type, [&](auto type) {
      auto* y = static_cast<decltype(type)*>(a.y) + row * a.y_ld;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        value(j, v);
        p.store(y, j, v);
      }
    });
    return;
  }
  float y[NV][8], top = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    value(j, y[j]);
    if (p.ragged()) mask8(p, j, y[j]);
    float t = top;
#pragma unroll
    for (int e = 0; e < 8; e += 2) t = max3_abs(t, y[j][e], y[j][e + 1]);
    top = p.has(j, 0) ? t : top;
  }
  const Quantizer quant(over.max(__float_as_uint(top), reinterpret_cast<uint32_t*>(sh[2])));
  if (!live) return;
  if (p.t == 0) a.scale[row] = quant.scale;
#pragma unroll
  for (int j = 0; j < NV; ++j) quant.store(a.q + row * a.q_ld, p, q_vec, j, y[j]);
}

constexpr unsigned kOneRound = 2 * 148;  // blocks that surely run at once

template <typename XT, typename PT, int MODE, int LANES, int NV, int VEC>
__global__ void __launch_bounds__(kRowsThreads, NV == 8 ? 3 : 1)
    rows_warp_kernel(const __grid_constant__ RowArgs a, bool wide, bool q_vec) {
  let_next_kernel_begin();
  after_earlier_kernels();
  constexpr int per = kRowsThreads / LANES;
  const int64_t at = (int64_t)blockIdx.x * per + threadIdx.x / LANES;
  const bool live = at < a.rows;
  // lanes without a row hold nothing
  const Pieces<VEC != BY_ELEMENT> p = {(int)(threadIdx.x % LANES), LANES, live ? a.cols : 0, wide};
  __shared__ float cross[VEC == BY_SHIFT && MODE == ROWS_NORM ? kRowsThreads * 8 : 1];
  row_in_registers<XT, PT, MODE, LANES, NV, VEC == BY_SHIFT>(a, live ? at : 0, live, p, q_vec, nullptr, cross);
}

template <typename XT, typename PT, int MODE, int NV, int VEC>
__global__ void __launch_bounds__(NV == 4 ? 512 : 1024)
    rows_block_kernel(const __grid_constant__ RowArgs a, bool wide, bool q_vec) {
  let_next_kernel_begin();
  after_earlier_kernels();
  __shared__ float sh[3][32];
  constexpr int kMost = NV == 4 ? 512 : 1024;
  __shared__ float cross[VEC == BY_SHIFT && MODE == ROWS_NORM ? kMost * 8 : 1];
  const Pieces<VEC != BY_ELEMENT> p = {(int)threadIdx.x, (int)blockDim.x, a.cols, wide};
  row_in_registers<XT, PT, MODE, 0, NV, VEC == BY_SHIFT>(a, blockIdx.x, true, p, q_vec, sh, cross);
}

// Rows too long for registers: one block re-reads its row for each reduction.
template <typename XT, typename PT, int MODE, int VEC>
__global__ void __launch_bounds__(1024)
    rows_long_kernel(const __grid_constant__ RowArgs a, bool wide, bool q_vec) {
  let_next_kernel_begin();
  after_earlier_kernels();
  __shared__ float sh[3][32];
  const RowSum<0> over;
  const Pieces<VEC != BY_ELEMENT> p = {(int)threadIdx.x, (int)blockDim.x, a.cols, wide};
  const int pieces = (a.cols - 1) / ((int)blockDim.x * 8) + 1;
  const int64_t row = blockIdx.x;
  const XT* x = static_cast<const XT*>(a.x) + row * a.x_ld;
  const auto weight = array_of(a.weight, a.param_type, PT());
  const auto bias = array_of(a.bias, a.param_type, PT());
  float v[8], w[8], mean = 0.f, rstd = 1.f;
  auto load = [&](int j) {
    uint32_t raw[8];
    if constexpr (VEC == BY_SHIFT) p.fetch_shifted(x, j, raw);
    else p.fetch(x, j, raw);
    p.template unpack<XT>(raw, v);
  };
  if (MODE != ROWS_QUANTIZE) {
    float s = 0.f;
    for (int j = 0; j < pieces; ++j) {
      load(j);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[e];
    }
    mean = over.sum(s, sh[0]) / (float)a.cols;
    s = 0.f;
    for (int j = 0; j < pieces; ++j) {
      load(j);
      centre8(v, mean);
      mask8(p, j, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(v[e], v[e], s);
    }
    rstd = 1.f / sqrtf(over.sum(s, sh[1]) / (float)a.cols + a.eps);
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
  auto value = [&](int j) {
    load(j);
    if (MODE != ROWS_QUANTIZE) {
      centre8(v, mean);
      scale8(v, rstd);
      uint32_t raw[8];
      if (weight) {
        p.fetch(weight, j, raw);
        Pieces<VEC != BY_ELEMENT>::template unpack<PT>(raw, w);
        times8(v, w);
      }
      if (bias) {
        p.fetch(bias, j, raw);
        Pieces<VEC != BY_ELEMENT>::template unpack<PT>(raw, w);
        plus8(v, w);
      }
    } else if (a.col_scale) {
      p.load(a.col_scale, j, w);
      times8(v, w);
    }
  };
  if (MODE == ROWS_NORM) {
    __shared__ float cross[VEC == BY_SHIFT && MODE == ROWS_NORM ? 1024 * 8 : 1];
    with_type(a.y_type, [&](auto type) {
      using T = decltype(type);
      for (int j = 0; j < pieces; ++j) {
        value(j);
        if constexpr (VEC == BY_SHIFT)
          store_crossed<32>(reinterpret_cast<T*>(cross + threadIdx.x / 32 * 256), v,
                            static_cast<T*>(a.y), a.y_ld, row, row + 1,
                            (j * p.threads + p.t / 32 * 32) * 8, a.cols);
        else
          p.store(static_cast<T*>(a.y) + row * a.y_ld, j, v);
      }
    });
    return;
  }
  float top = 0.f;
  for (int j = 0; j < pieces; ++j) {
    value(j);
    mask8(p, j, v);
#pragma unroll
    for (int e = 0; e < 8; e += 2) top = max3_abs(top, v[e], v[e + 1]);
  }
  const Quantizer quant(over.max(__float_as_uint(top), reinterpret_cast<uint32_t*>(sh[2])));
  if (threadIdx.x == 0) a.scale[row] = quant.scale;
  for (int j = 0; j < pieces; ++j) {
    value(j);
    quant.store(a.q + row * a.q_ld, p, q_vec, j, v);
  }
}

template <typename XT, typename PT, int MODE, int LANES, int NV, int VEC>
void launch_rows_warp(const RowArgs& a, bool wide, bool q_vec, cudaStream_t s) {
  constexpr int per = kRowsThreads / LANES;
  const unsigned grid = (unsigned)((a.rows + per - 1) / per);
  launch_chained(rows_warp_kernel<XT, PT, MODE, LANES, NV, VEC>, grid, kRowsThreads, 0, s,
                 grid <= kOneRound, 1, a, wide, q_vec);
}

template <typename XT, typename PT, int MODE, int NV, int VEC>
void launch_rows_block(const RowArgs& a, bool wide, bool q_vec, cudaStream_t s) {
  const int threads = ((a.cols + NV * 8 - 1) / (NV * 8) + 31) / 32 * 32;
  launch_chained(rows_block_kernel<XT, PT, MODE, NV, VEC>, dim3((unsigned)a.rows), threads, 0, s,
                 a.rows <= kOneRound, 1, a, wide, q_vec);
}

template <typename XT, typename PT, int MODE, int VEC>
void launch_rows_mode(const RowArgs& a, bool wide, bool q_vec, cudaStream_t s) {
  // few rows: more threads to a row, for the shortest chain (2688x512 f32 normed
  // and quantised: 5.5 us by 16 lanes with 4 pieces)
  if (a.rows <= 32 * sm_count()) {
    if (a.cols > 128 && a.cols <= 256) return launch_rows_warp<XT, PT, MODE, 32, 1, VEC>(a, wide, q_vec, s);
    if (a.cols > 256 && a.cols <= 512) return launch_rows_warp<XT, PT, MODE, 32, 2, VEC>(a, wide, q_vec, s);
  }
  if (a.cols > 512 && a.cols <= 8192 && a.rows <= (VEC == BY_ELEMENT ? 8 : 2) * sm_count())
    return launch_rows_block<XT, PT, MODE, 1, VEC>(a, wide, q_vec, s);
  if (a.cols <= 64) return launch_rows_warp<XT, PT, MODE, 8, 1, VEC>(a, wide, q_vec, s);
  if (a.cols <= 128) return launch_rows_warp<XT, PT, MODE, 8, 2, VEC>(a, wide, q_vec, s);
  if (a.cols <= 256) return launch_rows_warp<XT, PT, MODE, 8, 4, VEC>(a, wide, q_vec, s);
  if (a.cols <= 512) return launch_rows_warp<XT, PT, MODE, 16, 4, VEC>(a, wide, q_vec, s);
  if (a.cols <= 1024) return launch_rows_warp<XT, PT, MODE, 32, 4, VEC>(a, wide, q_vec, s);
  if constexpr (sizeof(XT) == 2 && MODE != ROWS_NORM_QUANTIZE && VEC != BY_ELEMENT)
    if (a.cols <= 2048) return launch_rows_warp<XT, PT, MODE, 32, 8, VEC>(a, wide, q_vec, s);
  constexpr int kBlock = sizeof(XT) == 2 && VEC != BY_ELEMENT ? 4 : 2;
  if (a.cols <= 16384) return launch_rows_block<XT, PT, MODE, kBlock, VEC>(a, wide, q_vec, s);
  launch_chained(rows_long_kernel<XT, PT, MODE, VEC>, dim3((unsigned)a.rows), 1024, 0, s,
                 a.rows <= kOneRound, 1, a, wide, q_vec);
}

// MODE on rows of XT; parameters of type f32 or XT are read by vectors, others by elements.
template <typename XT, int MODE>
void launch_rows_typed(const RowArgs& a, cudaStream_t s) {
  int vec = VEC_32;  // of the parameters
  auto narrow = [&vec](const void* p, int64_t ld, int bytes) {
    vec = std::min(vec, vec_of(p, ld, bytes));
  };
  if (MODE == ROWS_QUANTIZE) {
    narrow(a.col_scale, 0, 4);
  } else {
    narrow(a.weight, 0, type_size(a.param_type));
    narrow(a.bias, 0, type_size(a.param_type));
  }
  int row_vec = vec_of(a.x, a.x_ld, sizeof(XT));
  if (MODE == ROWS_NORM) row_vec = std::min(row_vec, vec_of(a.y, a.y_ld, type_size(a.y_type)));
  const bool wide = std::min(vec, row_vec) == VEC_32, q_vec = vec_of(a.q, a.q_ld, 1) != VEC_NONE;
  const bool params = a.weight || a.bias;
  const bool as_f32 = MODE == ROWS_QUANTIZE || !params || a.param_type == DMX_TYPE_F32;
  const bool as_xt = params && a.param_type == type_code(XT());
  if (vec == VEC_NONE || !(as_f32 || as_xt))
    return launch_rows_mode<XT, Any, MODE, BY_ELEMENT>(a, false, q_vec, s);
  if (row_vec == VEC_NONE) {
    // rows start off 16 bytes, as those of an odd length do: x's units are
    // shifted into place, a norm's outputs cross between lanes
    if (as_f32) launch_rows_mode<XT, float, MODE, BY_SHIFT>(a, vec == VEC_32, q_vec, s);
    else launch_rows_mode<XT, XT, MODE, BY_SHIFT>(a, vec == VEC_32, q_vec, s);
    return;
  }
  if (as_f32) launch_rows_mode<XT, float, MODE, BY_VECTOR>(a, wide, q_vec, s);
  else launch_rows_mode<XT, XT, MODE, BY_VECTOR>(a, wide, q_vec, s);
}

}  // namespace dmx
