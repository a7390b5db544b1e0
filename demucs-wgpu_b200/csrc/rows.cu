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
#include "ops.h"
#include "ops_common.cuh"

namespace dmx {

namespace {

constexpr int kThreads = 256;

DMX_DEVICE float block_sum(float v, float* sh) {
  v = warp_sum(v);
  __syncthreads();  // the last sum in `sh` has been read
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < kThreads / 32; ++i) t += sh[i];
  return t;
}
// Maximum of non-negative floats given as their bits: a NaN's are above infinity's.
DMX_DEVICE uint32_t block_max(uint32_t v, uint32_t* sh) {
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t t = 0;
  for (int i = 0; i < kThreads / 32; ++i) t = max(t, sh[i]);
  return t;
}

__global__ void __launch_bounds__(kThreads) rows_kernel(const RowArgs a) {
  __shared__ float shf[kThreads / 32];
  __shared__ uint32_t shu[kThreads / 32];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t x0 = row * a.x_ld;
    float mean = 0.f, rstd = 1.f;
    if (a.norm) {
      float s = 0.f;
      for (int c = threadIdx.x; c < a.cols; c += kThreads) s += load_as_f32(a.x, a.x_type, x0 + c);
      mean = block_sum(s, shf) / (float)a.cols;
      float v = 0.f;
      for (int c = threadIdx.x; c < a.cols; c += kThreads) {
        const float d = load_as_f32(a.x, a.x_type, x0 + c) - mean;
        v = fmaf(d, d, v);
      }
      rstd = 1.f / sqrtf(block_sum(v, shf) / (float)a.cols + a.eps);
      if (threadIdx.x == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
      }
    }
    auto value = [&](int c) {
      float v = load_as_f32(a.x, a.x_type, x0 + c);
      if (a.norm) {
        v = (v - mean) * rstd;
        if (a.weight) v *= load_as_f32(a.weight, a.param_type, c);
        if (a.bias) v += load_as_f32(a.bias, a.param_type, c);
      } else if (a.col_scale) {
        v *= a.col_scale[c];
      }
      return v;
    };
    if (a.y) {
      for (int c = threadIdx.x; c < a.cols; c += kThreads)
        store_from_f32(a.y, a.y_type, row * a.y_ld + c, value(c));
      continue;
    }
    uint32_t top = 0;
    for (int c = threadIdx.x; c < a.cols; c += kThreads)
      top = max(top, __float_as_uint(fabsf(value(c))));
    const float scale = __fdiv_rn(__uint_as_float(block_max(top, shu)), 127.f);
    const bool usable = scale > 0.f && scale < INFINITY;
    if (threadIdx.x == 0) a.scale[row] = scale;
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
      const float t = usable ? rintf(__fdiv_rn(value(c), scale)) : 0.f;
      a.q[row * a.q_ld + c] = (int8_t)(int)fminf(fmaxf(t, -127.f), 127.f);
    }
  }
}

}  // namespace

void launch_rows(const RowArgs& a, cudaStream_t s) {
  const unsigned grid = (unsigned)(a.rows < (1 << 20) ? a.rows : (1 << 20));
  rows_kernel<<<grid, kThreads, 0, s>>>(a);
}

}  // namespace dmx
