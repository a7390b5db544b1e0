// The layer norm's row kernels (rows.cuh) on bf16 rows with bf16 parameters.
#include "rows.cuh"

namespace dmx {

void launch_rows_norm_bf16_bf16(const RowArgs& a, cudaStream_t s) { launch_rows_norm<__nv_bfloat16, __nv_bfloat16>(a, s); }

}  // namespace dmx
