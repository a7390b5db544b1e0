// Entry of the row kernels (rows.cuh): a translation unit per input type, and
// per parameter type of the layer norm.
#include "dmx.h"
#include "ops.h"

namespace dmx {

#define DMX_ROWS_UNIT(x) void launch_rows_##x(const RowArgs& a, cudaStream_t s);
DMX_ROWS_UNIT(quantize_f32)
DMX_ROWS_UNIT(quantize_f16)
DMX_ROWS_UNIT(quantize_bf16)
DMX_ROWS_UNIT(norm_f32_f32)
DMX_ROWS_UNIT(norm_f32_f16)
DMX_ROWS_UNIT(norm_f32_bf16)
DMX_ROWS_UNIT(norm_f16_f32)
DMX_ROWS_UNIT(norm_f16_f16)
DMX_ROWS_UNIT(norm_f16_bf16)
DMX_ROWS_UNIT(norm_bf16_f32)
DMX_ROWS_UNIT(norm_bf16_f16)
DMX_ROWS_UNIT(norm_bf16_bf16)
#undef DMX_ROWS_UNIT

void launch_rows(const RowArgs& a, cudaStream_t s) {
  using Launch = void (*)(const RowArgs&, cudaStream_t);
  // by dmx_type: F32, F16, BF16
  static const Launch quantize[3] = {launch_rows_quantize_f32, launch_rows_quantize_f16,
                                     launch_rows_quantize_bf16};
  static const Launch norm[3][3] = {
      {launch_rows_norm_f32_f32, launch_rows_norm_f32_f16, launch_rows_norm_f32_bf16},
      {launch_rows_norm_f16_f32, launch_rows_norm_f16_f16, launch_rows_norm_f16_bf16},
      {launch_rows_norm_bf16_f32, launch_rows_norm_bf16_f16, launch_rows_norm_bf16_bf16}};
  if (!a.norm) quantize[a.x_type](a, s);
  else norm[a.x_type][a.weight || a.bias ? a.param_type : a.x_type](a, s);
}

}  // namespace dmx
