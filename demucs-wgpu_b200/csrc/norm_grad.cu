// Entry of the layer norm's backward pass (norm_grad.cuh): how many blocks
// walk the rows, and the join of their column sums.
#include <algorithm>

#include "dmx.h"
#include "ops.h"
#include "ops_common.cuh"

namespace dmx {

#define DMX_GRAD_UNIT(x) void launch_norm_grad_##x(const NormGradArgs& a, int parts, int how, bool wide, cudaStream_t s);
DMX_GRAD_UNIT(f32_f32)
DMX_GRAD_UNIT(f32_f16)
DMX_GRAD_UNIT(f32_bf16)
DMX_GRAD_UNIT(f16_f32)
DMX_GRAD_UNIT(f16_f16)
DMX_GRAD_UNIT(f16_bf16)
DMX_GRAD_UNIT(bf16_f32)
DMX_GRAD_UNIT(bf16_f16)
DMX_GRAD_UNIT(bf16_bf16)
#undef DMX_GRAD_UNIT

namespace {

// Most blocks that walk the rows: as many as a B200 holds at once, so that they
// end together. Two per SM; where groups of threads hold a row, one whose rows
// to come fill the SM's shared memory, or, for rows that do not start on 16
// bytes, what the 64 registers of its threads leave room for: one to three
// (20000 x 3001 bf16: 188 us with the two that fit, 249 with three). Constants, so that
// a sum does not depend on the device.
int64_t most_parts(int64_t cols, bool vec) {
  if (cols <= 1024 || cols > kGradBlockCols) return 2 * 148;
  return vec ? 148 : 148 * (1024 / (grad_group_threads((int)cols) * grad_groups((int)cols)));
}

// What a block takes in one turn, in units of which the rows make this many.
int64_t units_of(int64_t rows, int64_t cols) {
  const int64_t each = cols <= 128 ? 32 : cols <= 256 ? 16 : cols <= 1024 ? 8
                       : cols <= kGradBlockCols ? grad_groups((int)cols) : 1;
  return (rows + each - 1) / each;
}

// As many blocks as give each the same number of turns.
int parts_of(int64_t rows, int64_t cols, bool vec) {
  const int64_t most = most_parts(cols, vec);
  const int64_t units = units_of(rows, cols), turns = (units + most - 1) / most;
  return turns ? (int)((units + turns - 1) / turns) : 0;
}

// 32 columns per block; each of its 32 warps adds a share of the parts, whose
// sums are joined in order.
__global__ void __launch_bounds__(1024)
    norm_grad_join_kernel(const float* partials, int parts, int cols, float* dweight, float* dbias) {
  let_next_kernel_begin();
  after_earlier_kernels();
  __shared__ float sh[2][32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  const int64_t pitch = grad_pitch(cols);
  float w = 0.f, b = 0.f;
  if (c < cols)
#pragma unroll 5
    for (int p = warp; p < parts; p += 32) {
      w += partials[2 * p * pitch + c];
      b += partials[(2 * p + 1) * pitch + c];
    }
  sh[0][warp][lane] = w;
  sh[1][warp][lane] = b;
  __syncthreads();
  const int mine = blockIdx.x * 32 + warp;  // this warp's column
  w = warp_sum(sh[0][lane][warp]);
  b = warp_sum(sh[1][lane][warp]);
  if (lane != 0 || mine >= cols) return;
  if (dweight) dweight[mine] = w;
  if (dbias) dbias[mine] = b;
}

}  // namespace

// Enough for fewer rows too, which may take more blocks (of fewer turns each).
size_t norm_grad_workspace(int64_t rows, int64_t cols) {
  const int64_t parts = std::min(units_of(rows, cols), std::max(most_parts(cols, true), most_parts(cols, false)));
  return (size_t)parts * 2 * (size_t)grad_pitch((int)cols) * sizeof(float);
}

void launch_norm_grad(const NormGradArgs& args, cudaStream_t s) {
  NormGradArgs a = args;
  const bool sums = a.dweight || a.dbias;
  if (!sums) a.partials = nullptr;
  int row_vec = std::min(vec_of(a.x, a.x_ld, type_size(a.x_type)), vec_of(a.dy, a.dy_ld, type_size(a.dy_type)));
  if (a.dx) row_vec = std::min(row_vec, vec_of(a.dx, a.dx_ld, type_size(a.x_type)));
  int vec = vec_of(a.weight, 0, type_size(a.param_type));
  // partial sums of longer rows are stored by pieces too
  if (a.partials && a.cols > 1024) vec = std::min(vec, vec_of(a.partials, grad_pitch(a.cols), 4));
  const bool wide = std::min(vec, row_vec) == VEC_32;
  int how = vec == VEC_NONE || row_vec == VEC_NONE ? BY_ELEMENT : BY_VECTOR;
  if (vec != VEC_NONE && row_vec == VEC_NONE && a.cols > 1024 && a.cols <= kGradBlockCols) how = BY_SHIFT;
  const int parts = parts_of(a.rows, a.cols, how == BY_VECTOR);
  if (parts > 0 && (sums || a.dx)) {
    using Launch = void (*)(const NormGradArgs&, int, int, bool, cudaStream_t);
    // by dmx_type of x and of dy: F32, F16, BF16
    static const Launch launch[3][3] = {
        {launch_norm_grad_f32_f32, launch_norm_grad_f32_f16, launch_norm_grad_f32_bf16},
        {launch_norm_grad_f16_f32, launch_norm_grad_f16_f16, launch_norm_grad_f16_bf16},
        {launch_norm_grad_bf16_f32, launch_norm_grad_bf16_f16, launch_norm_grad_bf16_bf16}};
    launch[a.x_type][a.dy_type](a, parts, how, how == BY_SHIFT ? vec == VEC_32 : wide, s);
  }
  if (sums && !(parts == 1 && a.cols <= 1024))
    launch_chained(norm_grad_join_kernel, (a.cols + 31) / 32, 1024, 0, s, true, 1, a.partials, parts, a.cols,
                   a.dweight, a.dbias);
}

}  // namespace dmx
