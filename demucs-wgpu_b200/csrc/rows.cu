// Entry of the row kernels (rows.cuh): one translation unit per input type.
#include "dmx.h"
#include "ops.h"

namespace dmx {

void launch_rows_f32(const RowArgs& a, cudaStream_t s);
void launch_rows_f16(const RowArgs& a, cudaStream_t s);
void launch_rows_bf16(const RowArgs& a, cudaStream_t s);

void launch_rows(const RowArgs& a, cudaStream_t s) {
  if (a.x_type == DMX_TYPE_F32) launch_rows_f32(a, s);
  else if (a.x_type == DMX_TYPE_F16) launch_rows_f16(a, s);
  else launch_rows_bf16(a, s);
}

}  // namespace dmx
