// Launchers of the public operators (include/dmx.h): layer norm, its backward
// pass, the row quantiser and the 8-bit linear layer. Arguments are checked
// by ops.cu before they get here.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dmx {

// SMs of the current device.
int sm_count();

// Throws (an Error that the entry points turn into a status) if a CUDA call of
// an operator failed, and takes its error off the thread's last one. Statuses
// are asked where they arise: the last error may be one that the caller's own
// calls left, which is neither the operator's nor its to clear.
void check_cuda(cudaError_t e);

// One pass over rows: optionally the layer norm, then either a store (y) or
// the 8-bit quantisation (q, scale).
struct RowArgs {
  const void* x = nullptr;
  int x_type = 0;
  int64_t x_ld = 0;
  bool norm = false;
  const void* weight = nullptr;  // norm: may be null (1)
  const void* bias = nullptr;    // norm: may be null (0)
  int param_type = 0;
  float eps = 0.f;
  int64_t rows = 0;
  int cols = 0;
  float* mean = nullptr;  // norm: may be null
  float* rstd = nullptr;  // norm: may be null
  void* y = nullptr;      // null: quantise
  int y_type = 0;
  int64_t y_ld = 0;
  const float* col_scale = nullptr;  // quantise without norm: may be null (1)
  int8_t* q = nullptr;
  int64_t q_ld = 0;
  float* scale = nullptr;
};
void launch_rows(const RowArgs& a, cudaStream_t s);

struct NormGradArgs {
  const void* dy = nullptr;
  int dy_type = 0;
  int64_t dy_ld = 0;
  const void* x = nullptr;
  int x_type = 0;
  int64_t x_ld = 0;
  const void* weight = nullptr;  // may be null (1)
  int param_type = 0;
  const float* mean = nullptr;
  const float* rstd = nullptr;
  int64_t rows = 0;
  int cols = 0;
  void* dx = nullptr;  // x_type; may be null
  int64_t dx_ld = 0;
  float* dweight = nullptr;  // may be null
  float* dbias = nullptr;    // may be null
  float* partials = nullptr;
};
constexpr int kGradBlockCols = 16384;  // longest row that a group of threads holds
// Threads of such a group (16 columns each), and groups in a block of about 512.
inline int grad_group_threads(int cols) { return (cols + 511) / 512 * 32; }
inline int grad_groups(int cols) {
  const int threads = grad_group_threads(cols);
  return threads >= 512 ? 1 : 512 / threads;
}
// Pitch of the partial column sums: whole 32-byte pieces.
__host__ __device__ inline int grad_pitch(int cols) { return (cols + 7) / 8 * 8; }
size_t norm_grad_workspace(int64_t rows, int64_t cols);
void launch_norm_grad(const NormGradArgs& a, cudaStream_t s);

struct LinearArgs {
  const int8_t* x = nullptr;
  int64_t x_ld = 0;
  const float* x_scale = nullptr;  // may be null (1)
  const int8_t* w = nullptr;
  int64_t w_ld = 0;
  const float* w_scale = nullptr;  // may be null (1)
  const float* bias = nullptr;     // may be null (0)
  int64_t rows = 0;
  int n = 0, k = 0;
  bool gelu = false;
  const void* residual = nullptr;  // out's type; may be null, may be out
  int64_t residual_ld = 0;
  void* out = nullptr;
  int out_type = 0;
  int64_t out_ld = 0;
  int* err = nullptr;  // device flag raised by a wait that gave up
};
// false: a tensor map could not be encoded (nothing was launched)
bool launch_quantized_linear(const LinearArgs& a, cudaStream_t s);

}  // namespace dmx
