// Backward pass of the layer norm (dmx_layer_norm_backward).
//
//   h = (x - mean) rstd,  g = dy weight
//   dx = rstd (g - sum g / C - h sum(g h) / C)
//   dweight = sum over rows of dy h,  dbias = sum over rows of dy
//
// Bound by HBM: x and dy are read once and dx written once. A block walks rows
// a grid apart; each thread keeps the same columns in every row, so the column
// sums stay with it (in registers, or in shared memory for long rows) and
// leave once, as one partial sum per block and column. A second kernel adds
// the blocks' sums in a fixed order: no atomics, a gradient is the same from
// call to call. Rows of up to 1024 columns belong to a warp (or half or a
// quarter of one); longer ones to a group of up to 1024 threads, which copies
// the rows to come into shared memory while it works on one (each thread what
// it will read itself, so nothing waits on the others for that). Rows longer
// than that are swept twice, for dx and for the column sums, re-read from L2.
// Measured: 112896 x 512 f32 with bf16 gradients 95 us (6070 GB/s), 28000 x 2048
// bf16 82 us (4180), 4095 x 8195 bf16 66 us (3050: the block-wide reductions of
// each row), 20000 x 5001 bf16 off 16 bytes 290 us (2070; 312 with
// an f32 weight).
#pragma once

#include <algorithm>

#include "ops.h"
#include "ops_common.cuh"

namespace dmx {

// Values of piece j of dy, x and the weight to g = dy w and h.
template <typename XT, typename DT, typename PT, bool VEC>
struct GradPiece {
  float d[8], h[8], g[8];
  DMX_DEVICE void unpack(const uint32_t* draw, const uint32_t* xraw, const uint32_t* wraw, bool weight,
                         float mean, float rstd) {
    Pieces<VEC>::template unpack<DT>(draw, d);
    Pieces<VEC>::template unpack<XT>(xraw, h);
    centre8(h, mean);
    scale8(h, rstd);
    if (weight) {
      Pieces<VEC>::template unpack<PT>(wraw, g);
      times8(g, d);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = d[e];
    }
  }
};

DMX_DEVICE float2 dot_sums(const float* g, const float* h, float2 s) {
  // (sum g, sum g h) over eight values
  float2 a = make_float2(0.f, 0.f), b = a;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 g2 = make_float2(g[e], g[e + 1]);
    a = __fadd2_rn(a, g2);
    b = __ffma2_rn(g2, make_float2(h[e], h[e + 1]), b);
  }
  return make_float2(s.x + (a.x + a.y), s.y + (b.x + b.y));
}
// v = rstd (g - m1 - h m2)
DMX_DEVICE void dx8(const float* g, const float* h, float m1, float m2, float rstd, float* v) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 h2 = make_float2(h[e], h[e + 1]);
    float2 t = __fadd2_rn(make_float2(g[e], g[e + 1]), make_float2(-m1, -m1));
    t = __ffma2_rn(h2, make_float2(-m2, -m2), t);
    t = __fmul2_rn(t, make_float2(rstd, rstd));
    v[e] = t.x;
    v[e + 1] = t.y;
  }
}
DMX_DEVICE void gather8(float* w, float* b, const float* d, const float* h) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 d2 = make_float2(d[e], d[e + 1]);
    const float2 r = __ffma2_rn(d2, make_float2(h[e], h[e + 1]), make_float2(w[e], w[e + 1]));
    const float2 s = __fadd2_rn(make_float2(b[e], b[e + 1]), d2);
    w[e] = r.x;
    w[e + 1] = r.y;
    b[e] = s.x;
    b[e + 1] = s.y;
  }
}

// Sums of (a, b) over the threads of one row.
template <int LANES>
DMX_DEVICE float2 lanes_sum2(float2 v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  return v;
}

constexpr int kGradThreads = 256;

// Rows of up to LANES * NV * 8 columns, LANES lanes each.
template <typename XT, typename DT, typename PT, int LANES, int NV, bool VEC>
__global__ void __launch_bounds__(kGradThreads, NV == 4 ? 1 : 2)
    norm_grad_warp_kernel(const __grid_constant__ NormGradArgs a, bool wide) {
  let_next_kernel_begin();
  after_earlier_kernels();
  constexpr int per = kGradThreads / LANES, kCols = LANES * NV * 8;
  __shared__ float sums[per][kCols];
  const Pieces<VEC> p = {(int)(threadIdx.x % LANES), LANES, a.cols, wide};
  const XT* x = static_cast<const XT*>(a.x);
  const DT* dy = static_cast<const DT*>(a.dy);
  const auto weight = array_of(a.weight, a.param_type, PT());
  uint32_t wraw[NV][8], xraw[NV][8], draw[NV][8];
  float dw[NV][8], db[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (weight) p.fetch(weight, j, wraw[j]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[j][e] = db[j][e] = 0.f;
  }
  const int64_t step = (int64_t)gridDim.x * per;
  int64_t row = (int64_t)blockIdx.x * per + threadIdx.x / LANES;
  float mean = 0.f, rstd = 0.f;
  // a row past the last one is zeros: it adds nothing and only takes part in the shuffles
  auto fetch = [&](int64_t r) {
    const bool live = r < a.rows;
    const Pieces<VEC> q = {p.t, LANES, live ? a.cols : 0, wide};
    const int64_t at = live ? r : 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      q.fetch(x + at * a.x_ld, j, xraw[j]);
      q.fetch(dy + at * a.dy_ld, j, draw[j]);
    }
    mean = live ? a.mean[at] : 0.f;
    rstd = live ? a.rstd[at] : 0.f;
  };
  const int64_t passes = (a.rows + step - 1) / step;
  for (int64_t pass = 0; pass < passes; ++pass, row += step) {
    fetch(row);
    GradPiece<XT, DT, PT, VEC> q[NV];
    float2 s = make_float2(0.f, 0.f);
    const float row_mean = mean, row_rstd = rstd;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      q[j].unpack(draw[j], xraw[j], wraw[j], a.weight != nullptr, row_mean, row_rstd);
      s = dot_sums(q[j].g, q[j].h, s);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) gather8(dw[j], db[j], q[j].d, q[j].h);
    if (!a.dx) continue;
    s = lanes_sum2<LANES>(s);
    if (row >= a.rows) continue;
    const float m1 = s.x / (float)a.cols, m2 = s.y / (float)a.cols;
    XT* dx = static_cast<XT*>(a.dx) + row * a.dx_ld;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float v[8];
      dx8(q[j].g, q[j].h, m1, m2, row_rstd, v);
      p.store(dx, j, v);
    }
  }
  if (!a.partials) return;
  // the block's row groups added in their order
  float* out = a.partials + (int64_t)blockIdx.x * 2 * grad_pitch(a.cols);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    // one block's sums are the gradients themselves
    float* to = gridDim.x > 1 ? out + half * grad_pitch(a.cols) : half ? a.dbias : a.dweight;
    if (!to) continue;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        sums[threadIdx.x / LANES][p.col(j, e)] = half ? db[j][e] : dw[j][e];
    __syncthreads();
    for (int c = threadIdx.x; c < a.cols; c += kGradThreads) {
      float t = 0.f;
#pragma unroll
      for (int g = 0; g < per; ++g) t += sums[g][c];
      to[c] = t;
    }
  }
}

// `bytes` (0..16, the rest as zeros) of 16 from global to this thread's shared
// memory. With a clobber: what lay there before is read by plain loads, which
// the compiler could otherwise move below the copy that overwrites it.
DMX_DEVICE void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Rows of up to blockDim.x * 16 columns, a group of blockDim.x threads each, R
// rows at a time (their reductions share their latency); blockDim.y groups to
// a block. Shared memory, all of it each thread's own and laid out with the
// thread innermost: the column sums, (dw, db) of two columns to 16 bytes, and,
// BY_VECTOR, the `ahead` >= R rows to come. BY_SHIFT, rows that start off 16
// bytes: read by shifted vectors, dx written across lanes.
template <typename XT, typename DT, typename PT, int VEC, int THREADS, int R>
__global__ void __launch_bounds__(THREADS)
    norm_grad_block_kernel(const __grid_constant__ NormGradArgs a, bool wide, int ahead) {
  let_next_kernel_begin();
  after_earlier_kernels();
  constexpr int NV = 2, kXUnits = sizeof(XT) / 2, kDUnits = sizeof(DT) / 2;  // of 16 bytes per piece
  constexpr int kStage = NV * (kXUnits + kDUnits);
  extern __shared__ float4 own[];
  __shared__ float2 sh[2][R][32];
  __shared__ float cross[VEC == BY_SHIFT ? THREADS * 8 : 1];
  const int n = blockDim.x * blockDim.y, id = threadIdx.y * blockDim.x + threadIdx.x;
  const Pieces<VEC != BY_ELEMENT> p = {(int)threadIdx.x, (int)blockDim.x, a.cols, wide};
  const XT* x = static_cast<const XT*>(a.x);
  const DT* dy = static_cast<const DT*>(a.dy);
  const auto weight = array_of(a.weight, a.param_type, PT());
  const int lane = id & 31, warp = id >> 5, warps = blockDim.x / 32;
#pragma unroll
  for (int i = 0; i < NV * 4; ++i) own[i * n + id] = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4* ring = own + NV * 4 * n + id;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  const int64_t first = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  // this thread's units of a row: where they start (bytes) and how much of them exists
  int x_from[NV * kXUnits], x_bytes[NV * kXUnits], d_from[NV * kDUnits], d_bytes[NV * kDUnits];
  auto units = [&](int size, int per, int* from, int* bytes) {
#pragma unroll
    for (int i = 0; i < NV * per; ++i) {
      const int at = p.col(i / per, 0) * size + i % per * 16;
      bytes[i] = min(max(a.cols * size - at, 0), 16);
      from[i] = bytes[i] ? at : 0;
    }
  };
  units(sizeof(XT), kXUnits, x_from, x_bytes);
  units(sizeof(DT), kDUnits, d_from, d_bytes);
  // the copies of one row into stage s of the ring; an empty group past the end
  auto copy_row = [&](int64_t row, int s) {
    if (row < a.rows) {
      const uint32_t at = ring_at + (uint32_t)(s * kStage * n) * 16;
      const char* xs = reinterpret_cast<const char*>(x + row * a.x_ld);
      const char* ds = reinterpret_cast<const char*>(dy + row * a.dy_ld);
#pragma unroll
      for (int i = 0; i < NV * kXUnits; ++i) copy16(at + (uint32_t)(i * n) * 16, xs + x_from[i], x_bytes[i]);
#pragma unroll
      for (int i = 0; i < NV * kDUnits; ++i)
        copy16(at + (uint32_t)((NV * kXUnits + i) * n) * 16, ds + d_from[i], d_bytes[i]);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (VEC == BY_VECTOR)
    for (int s = 0; s < ahead; ++s) copy_row(first + s * step, s);
  uint32_t wraw[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (weight) p.fetch(weight, j, wraw[j]);
  int turn = 0, stage = 0;
  // a row past the last one is zeros and adds nothing
  float mean_next[R], rstd_next[R];
  auto fetch_stats = [&](int64_t row0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = row0 + r * step < a.rows;
      mean_next[r] = live ? a.mean[row0 + r * step] : 0.f;
      rstd_next[r] = live ? a.rstd[row0 + r * step] : 0.f;
    }
  };
  fetch_stats(first);
  for (int64_t row0 = first; row0 < a.rows; row0 += R * step, turn ^= 1) {
    uint32_t xraw[R][NV][8], draw[R][NV][8];
    float mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = mean_next[r];
      rstd[r] = rstd_next[r];
    }
    fetch_stats(row0 + R * step);
    // every row's copies are a group: the oldest R of `ahead` have landed
    if (VEC == BY_VECTOR) {
      if (ahead == R) asm volatile("cp.async.wait_group 0;" ::: "memory");
      else if (ahead == R + 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
      else if (ahead == R + 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
      else asm volatile("cp.async.wait_group 3;" ::: "memory");
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r * step;
      const bool live = R == 1 || row < a.rows;
      if (VEC == BY_VECTOR) {
        const float4* from = ring + stage * kStage * n;
        const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
          for (int u = 0; u < kXUnits; ++u)
            *reinterpret_cast<float4*>(&xraw[r][j][4 * u]) = live ? from[(j * kXUnits + u) * n] : none;
#pragma unroll
          for (int u = 0; u < kDUnits; ++u)
            *reinterpret_cast<float4*>(&draw[r][j][4 * u]) =
                live ? from[(NV * kXUnits + j * kDUnits + u) * n] : none;
        }
        copy_row(row + ahead * step, stage);
        stage = stage + 1 == ahead ? 0 : stage + 1;
      } else {
        const Pieces<VEC != BY_ELEMENT> q = {p.t, p.threads, live ? a.cols : 0, wide};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if constexpr (VEC == BY_SHIFT) {
            q.fetch_shifted(x + row * a.x_ld, j, xraw[r][j]);
            q.fetch_shifted(dy + row * a.dy_ld, j, draw[r][j]);
          } else {
            q.fetch(x + row * a.x_ld, j, xraw[r][j]);
            q.fetch(dy + row * a.dy_ld, j, draw[r][j]);
          }
        }
      }
    }
    float2 s[R];
    GradPiece<XT, DT, PT, VEC != BY_ELEMENT> q;
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float dw[8] = {}, db[8] = {};
#pragma unroll
      for (int r = 0; r < R; ++r) {
        q.unpack(draw[r][j], xraw[r][j], wraw[j], a.weight != nullptr, mean[r], rstd[r]);
        s[r] = dot_sums(q.g, q.h, s[r]);
        gather8(dw, db, q.d, q.h);
      }
      if (a.partials)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float4* o = &own[(j * 4 + i) * n + id];
          const float4 t = *o;
          *o = make_float4(t.x + dw[2 * i], t.y + db[2 * i], t.z + dw[2 * i + 1], t.w + db[2 * i + 1]);
        }
    }
    if (!a.dx) continue;
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = lanes_sum2<32>(s[r]);
    // two buffers in turn: the last rows' may still be read
    if (lane == 0)
#pragma unroll
      for (int r = 0; r < R; ++r) sh[turn][r][warp] = s[r];
    asm volatile("bar.sync %0, %1;" ::"r"(threadIdx.y + 1), "r"(blockDim.x) : "memory");
#pragma unroll
    for (int r = 0; r < R; ++r)
      s[r] = lanes_sum2<32>(lane < warps ? sh[turn][r][threadIdx.y * warps + lane]
                                         : make_float2(0.f, 0.f));
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r * step;
      if (R > 1 && row >= a.rows) break;
      const float m1 = s[r].x / (float)a.cols, m2 = s[r].y / (float)a.cols;
      XT* dx = static_cast<XT*>(a.dx) + row * a.dx_ld;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float v[8];
        q.unpack(draw[r][j], xraw[r][j], wraw[j], a.weight != nullptr, mean[r], rstd[r]);
        dx8(q.g, q.h, m1, m2, rstd[r], v);
        if constexpr (VEC == BY_SHIFT)
          store_crossed<32>(reinterpret_cast<XT*>(cross + id / 32 * 256), v, static_cast<XT*>(a.dx),
                            a.dx_ld, row, row + 1, (j * p.threads + p.t / 32 * 32) * 8, a.cols);
        else
          p.store(dx, j, v);
      }
    }
  }
  if (!a.partials) return;
  __syncthreads();
  if (threadIdx.y != 0) return;
  // the block's groups added in their order
  const int pitch = grad_pitch(a.cols);
  float* out = a.partials + (int64_t)blockIdx.x * 2 * pitch;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float dw[8], db[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float4 t = own[(j * 4 + i) * n + id];
      for (int g = 1; g < (int)blockDim.y; ++g) {
        const float4 u = own[(j * 4 + i) * n + g * blockDim.x + threadIdx.x];
        t = make_float4(t.x + u.x, t.y + u.y, t.z + u.z, t.w + u.w);
      }
      dw[2 * i] = t.x;
      db[2 * i] = t.y;
      dw[2 * i + 1] = t.z;
      db[2 * i + 1] = t.w;
    }
    p.store(out, j, dw);
    p.store(out + pitch, j, db);
  }
}

// Rows too long for a block's registers: dx, re-reading the row.
template <typename XT, typename DT, typename PT, bool VEC>
__global__ void __launch_bounds__(1024)
    norm_grad_long_kernel(const __grid_constant__ NormGradArgs a, bool wide) {
  let_next_kernel_begin();
  after_earlier_kernels();
  __shared__ float2 sh[2][32];
  const Pieces<VEC> p = {(int)threadIdx.x, (int)blockDim.x, a.cols, wide};
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x / 32;
  const int pieces = (a.cols - 1) / ((int)blockDim.x * 8) + 1;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const XT* x = static_cast<const XT*>(a.x) + row * a.x_ld;
    const DT* dy = static_cast<const DT*>(a.dy) + row * a.dy_ld;
    XT* dx = static_cast<XT*>(a.dx) + row * a.dx_ld;
    const float mean = a.mean[row], rstd = a.rstd[row];
    GradPiece<XT, DT, PT, VEC> q;
    auto piece = [&](int j) {
      uint32_t xraw[8], draw[8], wraw[8];
      p.fetch(x, j, xraw);
      p.fetch(dy, j, draw);
      if (a.weight) p.fetch(array_of(a.weight, a.param_type, PT()), j, wraw);
      q.unpack(draw, xraw, wraw, a.weight != nullptr, mean, rstd);
    };
    float2 s = make_float2(0.f, 0.f);
    for (int j = 0; j < pieces; ++j) {
      piece(j);
      s = dot_sums(q.g, q.h, s);
    }
    s = lanes_sum2<32>(s);
    if (lane == 0) sh[turn][warp] = s;
    __syncthreads();
    s = lanes_sum2<32>(lane < warps ? sh[turn][lane] : make_float2(0.f, 0.f));
    const float m1 = s.x / (float)a.cols, m2 = s.y / (float)a.cols;
    for (int j = 0; j < pieces; ++j) {
      piece(j);
      float v[8];
      dx8(q.g, q.h, m1, m2, rstd, v);
      p.store(dx, j, v);
    }
  }
}

// The column sums of such rows: block (strip of 8 columns per thread, part).
template <typename XT, typename DT, bool VEC>
__global__ void __launch_bounds__(kGradThreads)
    norm_grad_columns_kernel(const __grid_constant__ NormGradArgs a, bool wide) {
  let_next_kernel_begin();
  after_earlier_kernels();
  const int pieces = (a.cols - 1) / (kGradThreads * 8) + 1, j = blockIdx.x;
  const Pieces<VEC> p = {(int)threadIdx.x, kGradThreads, a.cols, wide};
  if (j >= pieces || !p.has(j, 0)) return;
  float dw[8] = {}, db[8] = {};
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float d[8], h[8];
    p.load(static_cast<const XT*>(a.x) + row * a.x_ld, j, h);
    p.load(static_cast<const DT*>(a.dy) + row * a.dy_ld, j, d);
    centre8(h, a.mean[row]);
    scale8(h, a.rstd[row]);
    gather8(dw, db, d, h);
  }
  const int pitch = grad_pitch(a.cols);
  float* out = a.partials + (int64_t)blockIdx.y * 2 * pitch;
  p.store(out, j, dw);
  p.store(out + pitch, j, db);
}

template <typename XT, typename DT, typename PT, int VEC, int THREADS, int R>
void launch_norm_grad_block(const NormGradArgs& a, int parts, dim3 block, size_t smem, bool wide,
                            int ahead, cudaStream_t s) {
  auto kernel = norm_grad_block_kernel<XT, DT, PT, VEC, THREADS, R>;
  static PerDevice configured;
  configured.once([&] {
    check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    (VEC == BY_SHIFT ? 128 : 220) * 1024));
  });
  launch_chained(kernel, parts, block, smem, s, true, 1, a, wide, ahead);
}

// Long rows that start off 16 bytes, the weight and the partial sums on them.
template <typename XT, typename DT, typename PT>
void launch_norm_grad_shift(const NormGradArgs& a, int parts, bool wide, cudaStream_t s) {
  const int threads = grad_group_threads(a.cols), groups = grad_groups(a.cols);
  launch_norm_grad_block<XT, DT, PT, BY_SHIFT, 1024, 1>(a, parts, dim3(threads, groups),
                                                        (size_t)threads * groups * 128, wide, 0, s);
}

// What norm_grad.cu decides: parts (blocks whose partial sums are joined).
template <typename XT, typename DT, typename PT, bool VEC>
void launch_norm_grad_vec(const NormGradArgs& a, int parts, bool wide, cudaStream_t s) {
  if (a.cols <= 64)
    launch_chained(norm_grad_warp_kernel<XT, DT, PT, 8, 1, VEC>, parts, kGradThreads, 0, s, true, 1, a, wide);
  else if (a.cols <= 128)
    launch_chained(norm_grad_warp_kernel<XT, DT, PT, 8, 2, VEC>, parts, kGradThreads, 0, s, true, 1, a, wide);
  else if (a.cols <= 256)
    launch_chained(norm_grad_warp_kernel<XT, DT, PT, 16, 2, VEC>, parts, kGradThreads, 0, s, true, 1, a, wide);
  else if (a.cols <= 512)
    launch_chained(norm_grad_warp_kernel<XT, DT, PT, 32, 2, VEC>, parts, kGradThreads, 0, s, true, 1, a, wide);
  else if (a.cols <= 1024)
    launch_chained(norm_grad_warp_kernel<XT, DT, PT, 32, 4, VEC>, parts, kGradThreads, 0, s, true, 1, a, wide);
  else if (a.cols <= kGradBlockCols) {
    const int threads = grad_group_threads(a.cols), groups = grad_groups(a.cols);
    // shared memory per thread: its sums, and the rows to come
    const int own = 128, stage = 16 * (sizeof(XT) + sizeof(DT));
    const int most = 220 * 1024 / (threads * groups);
    const int ahead = VEC ? std::min(4, (most - own) / stage) : 0;
    const dim3 block(threads, groups);
    const size_t smem = (size_t)threads * groups * (own + ahead * stage);
    // Built for the registers that a block's threads leave each of them. Up to 512
    // threads (8192 columns) 128, two rows at a time (28000 x 2048 bf16: 82 us, one
    // at a time 94; 7000 x 8192 f32 181 and 195). Up to 640 (10240 columns) 96, one
    // row at a time; with the 64 of 1024 threads values spill: 4000 x 9216 bf16 65
    // us against 114, 3000 x 10240 f32 with bf16 gradients 87 against 148. Longer
    // rows have the 64 all the same (3000 x 12288 bf16 92 us).
    if constexpr (!VEC)
      launch_norm_grad_block<XT, DT, PT, BY_ELEMENT, 1024, 1>(a, parts, block, smem, wide, ahead, s);
    else if (ahead < 1)  // no room to copy ahead: rows go by elements (2500 x 16384 f32: 199 us)
      launch_norm_grad_block<XT, DT, Any, BY_ELEMENT, 1024, 1>(a, parts, block, smem, wide, ahead, s);
    else if (threads * groups <= 512 && ahead >= 2)
      launch_norm_grad_block<XT, DT, PT, BY_VECTOR, 512, 2>(a, parts, block, smem, wide, ahead, s);
    else if (threads * groups <= 640)
      launch_norm_grad_block<XT, DT, PT, BY_VECTOR, 640, 1>(a, parts, block, smem, wide, ahead, s);
    else
      launch_norm_grad_block<XT, DT, PT, BY_VECTOR, 1024, 1>(a, parts, block, smem, wide, ahead, s);
  } else {
    const unsigned strips = (unsigned)((a.cols - 1) / (kGradThreads * 8) + 1);
    // first: dx may be written over x or dy
    if (a.partials)
      launch_chained(norm_grad_columns_kernel<XT, DT, VEC>, dim3(strips, parts), kGradThreads, 0, s, true, 1, a,
                     wide);
    if (a.dx)
      launch_chained(norm_grad_long_kernel<XT, DT, PT, VEC>,
                     dim3((unsigned)std::min<int64_t>(a.rows, 1 << 20)), 1024, 0, s, true, 1, a, wide);
  }
}

// The weight is read by vectors if its type is f32 or XT, else by elements.
template <typename XT, typename DT>
void launch_norm_grad_typed(const NormGradArgs& a, int parts, int how, bool wide, cudaStream_t s) {
  const int type = a.weight ? a.param_type : DMX_TYPE_F32;
  const bool as_f32 = type == DMX_TYPE_F32, as_xt = type == type_code(XT());
  if (how == BY_VECTOR && as_f32) launch_norm_grad_vec<XT, DT, float, true>(a, parts, wide, s);
  else if (how == BY_VECTOR && as_xt) launch_norm_grad_vec<XT, DT, XT, true>(a, parts, wide, s);
  else if (how == BY_SHIFT && as_f32) launch_norm_grad_shift<XT, DT, float>(a, parts, wide, s);
  else if (how == BY_SHIFT && as_xt) launch_norm_grad_shift<XT, DT, XT>(a, parts, wide, s);
  else launch_norm_grad_vec<XT, DT, Any, false>(a, parts, false, s);
}

}  // namespace dmx
