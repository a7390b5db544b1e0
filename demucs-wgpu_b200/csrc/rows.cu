// Entry of the row kernels (rows.cuh): a translation unit per operator and input type.
#include "dmx.h"
#include "ops.h"

namespace dmx {

#define DMX_ROWS_UNITS(op)                                   \
  void launch_rows_##op##_f32(const RowArgs& a, cudaStream_t s); \
  void launch_rows_##op##_f16(const RowArgs& a, cudaStream_t s); \
  void launch_rows_##op##_bf16(const RowArgs& a, cudaStream_t s);
DMX_ROWS_UNITS(quantize)
DMX_ROWS_UNITS(norm)
DMX_ROWS_UNITS(norm_quantize)
#undef DMX_ROWS_UNITS

void launch_rows(const RowArgs& a, cudaStream_t s) {
  using Launch = void (*)(const RowArgs&, cudaStream_t);
  // by dmx_type of x: F32, F16, BF16
  static const Launch quantize[3] = {launch_rows_quantize_f32, launch_rows_quantize_f16,
                                     launch_rows_quantize_bf16};
  static const Launch norm[3] = {launch_rows_norm_f32, launch_rows_norm_f16, launch_rows_norm_bf16};
  static const Launch both[3] = {launch_rows_norm_quantize_f32, launch_rows_norm_quantize_f16,
                                 launch_rows_norm_quantize_bf16};
  (a.y ? norm : a.norm ? both : quantize)[a.x_type](a, s);
}

}  // namespace dmx
