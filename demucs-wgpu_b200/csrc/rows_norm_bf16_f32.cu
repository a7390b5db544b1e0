// The layer norm's row kernels (rows.cuh) on bf16 rows with f32 parameters.
#include "rows.cuh"

namespace dmx {

void launch_rows_norm_bf16_f32(const RowArgs& a, cudaStream_t s) { launch_rows_norm<__nv_bfloat16, float>(a, s); }

}  // namespace dmx
