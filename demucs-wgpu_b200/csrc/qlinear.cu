// The 8-bit linear layer (dmx_quantized_linear):
//
//   out[m][n] = act(acc[m][n] x_scale[m] w_scale[n] + bias[n]) + residual[m][n]
//   acc[m][n] = sum_k x[m][k] w[n][k], exact in 32-bit integers
//
// Rows of x and w start on 16-byte boundaries, so both are read 16 bytes at a
// time; the bytes past column k of a row are never used.
#include "ops.h"
#include "ops_common.cuh"

namespace dmx {

namespace {

// Bytes k0 .. k0 + 15 of a row of `k` values, the ones past its end as zero.
DMX_DEVICE int4 row16(const int8_t* row, int k0, int k) {
  int4 v = make_int4(0, 0, 0, 0);
  if (k0 >= k) return v;
  v = *reinterpret_cast<const int4*>(row + k0);
  const int left = k - k0;
  if (left < 16) {
    int* w = reinterpret_cast<int*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int bytes = min(max(left - 4 * i, 0), 4);
      w[i] = bytes == 4 ? w[i] : (w[i] & ((1 << (8 * bytes)) - 1));
    }
  }
  return v;
}

DMX_DEVICE void finish(const LinearArgs& a, int64_t m, int n, int acc) {
  float v = (float)acc * (a.x_scale ? a.x_scale[m] : 1.f) * (a.w_scale ? a.w_scale[n] : 1.f);
  if (a.bias) v += a.bias[n];
  if (a.gelu) v = gelu(v);
  if (a.residual) v += load_as_f32(a.residual, a.out_type, m * a.residual_ld + n);
  store_from_f32(a.out, a.out_type, m * a.out_ld + n, v);
}

constexpr int kTile = 64;

// 64 x 64 outputs per block, 4 x 4 per thread, four products per dp4a.
__global__ void __launch_bounds__(256) linear_tile_kernel(const LinearArgs a, int64_t mtiles) {
  __shared__ int4 xs[kTile][5], ws[kTile][5];  // 64 bytes of k per row, padded
  const int n0 = blockIdx.x * kTile, tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  for (int64_t mt = blockIdx.y; mt < mtiles; mt += gridDim.y) {
    const int64_t m0 = mt * kTile;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < a.k; k0 += 64) {
      const int r = tid / 4, c = tid % 4;
      __syncthreads();
      xs[r][c] = m0 + r < a.rows ? row16(a.x + (m0 + r) * a.x_ld, k0 + 16 * c, a.k) : make_int4(0, 0, 0, 0);
      ws[r][c] = n0 + r < a.n ? row16(a.w + (int64_t)(n0 + r) * a.w_ld, k0 + 16 * c, a.k) : make_int4(0, 0, 0, 0);
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        int4 xv[4], wv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          xv[i] = xs[ty * 4 + i][q];
          wv[i] = ws[tx + 16 * i][q];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc[i][j] = __dp4a(xv[i].x, wv[j].x, acc[i][j]);
            acc[i][j] = __dp4a(xv[i].y, wv[j].y, acc[i][j]);
            acc[i][j] = __dp4a(xv[i].z, wv[j].z, acc[i][j]);
            acc[i][j] = __dp4a(xv[i].w, wv[j].w, acc[i][j]);
          }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (m0 + ty * 4 + i < a.rows && n0 + tx + 16 * j < a.n)
          finish(a, m0 + ty * 4 + i, n0 + tx + 16 * j, acc[i][j]);
  }
}

}  // namespace

bool launch_quantized_linear(const LinearArgs& a, cudaStream_t s) {
  const int64_t mtiles = (a.rows + kTile - 1) / kTile;
  const dim3 grid((unsigned)((a.n + kTile - 1) / kTile), (unsigned)(mtiles < 65535 ? mtiles : 65535));
  linear_tile_kernel<<<grid, 256, 0, s>>>(a, mtiles);
  return true;
}

}  // namespace dmx
