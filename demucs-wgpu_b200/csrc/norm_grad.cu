// Backward pass of the layer norm (dmx_layer_norm_backward).
//
//   h = (x - mean) rstd,  g = dy weight
//   dx = rstd (g - sum g / C - h sum(g h) / C)
//   dweight = sum over rows of dy h,  dbias = sum over rows of dy
//
// The column sums are taken per block of rows into partial sums, which a
// second kernel adds in a fixed order: no atomics, so a gradient is the same
// from call to call.
#include <algorithm>

#include "ops.h"
#include "ops_common.cuh"

namespace dmx {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxParts = 296;

int64_t parts_of(int64_t rows) { return std::min<int64_t>((rows + 31) / 32, kMaxParts); }

__global__ void __launch_bounds__(kThreads) norm_grad_rows_kernel(const NormGradArgs a) {
  __shared__ float sh[2][kThreads / 32];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
      const float h = (load_as_f32(a.x, a.x_type, row * a.x_ld + c) - mean) * rstd;
      float g = load_as_f32(a.dy, a.dy_type, row * a.dy_ld + c);
      if (a.weight) g *= load_as_f32(a.weight, a.param_type, c);
      s1 += g;
      s2 = fmaf(g, h, s2);
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
      sh[0][threadIdx.x >> 5] = s1;
      sh[1][threadIdx.x >> 5] = s2;
    }
    __syncthreads();
    s1 = s2 = 0.f;
    for (int i = 0; i < kThreads / 32; ++i) {
      s1 += sh[0][i];
      s2 += sh[1][i];
    }
    s1 /= (float)a.cols;
    s2 /= (float)a.cols;
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
      const float h = (load_as_f32(a.x, a.x_type, row * a.x_ld + c) - mean) * rstd;
      float g = load_as_f32(a.dy, a.dy_type, row * a.dy_ld + c);
      if (a.weight) g *= load_as_f32(a.weight, a.param_type, c);
      store_from_f32(a.dx, a.x_type, row * a.dx_ld + c, rstd * (g - s1 - h * s2));
    }
  }
}

// Block (column strip, part): sums of its rows.
__global__ void __launch_bounds__(kThreads) norm_grad_cols_kernel(const NormGradArgs a, int parts) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.cols) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += parts) {
    const float h = (load_as_f32(a.x, a.x_type, row * a.x_ld + c) - a.mean[row]) * a.rstd[row];
    const float d = load_as_f32(a.dy, a.dy_type, row * a.dy_ld + c);
    dw = fmaf(d, h, dw);
    db += d;
  }
  a.partials[((int64_t)blockIdx.y * 2) * a.cols + c] = dw;
  a.partials[((int64_t)blockIdx.y * 2 + 1) * a.cols + c] = db;
}

__global__ void __launch_bounds__(kThreads) norm_grad_join_kernel(const NormGradArgs a, int parts) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.cols) return;
  float dw = 0.f, db = 0.f;
  for (int p = 0; p < parts; ++p) {
    dw += a.partials[((int64_t)p * 2) * a.cols + c];
    db += a.partials[((int64_t)p * 2 + 1) * a.cols + c];
  }
  if (a.dweight) a.dweight[c] = dw;
  if (a.dbias) a.dbias[c] = db;
}

}  // namespace

size_t norm_grad_workspace(int64_t rows, int64_t cols) {
  return (size_t)parts_of(rows) * 2 * (size_t)cols * sizeof(float);
}

void launch_norm_grad(const NormGradArgs& a, cudaStream_t s) {
  const int parts = (int)parts_of(a.rows);
  const unsigned strips = (unsigned)((a.cols + kThreads - 1) / kThreads);
  if (a.dweight || a.dbias) {  // first: dx may be written over x or dy
    if (parts > 0) norm_grad_cols_kernel<<<dim3(strips, parts), kThreads, 0, s>>>(a, parts);
    norm_grad_join_kernel<<<strips, kThreads, 0, s>>>(a, parts);
  }
  if (a.dx && a.rows > 0)
    norm_grad_rows_kernel<<<(unsigned)std::min<int64_t>(a.rows, 1 << 20), kThreads, 0, s>>>(a);
}

}  // namespace dmx
