// The row kernels (rows.cuh) of the layer norm on bf16 rows.
#include "rows.cuh"

namespace dmx {

void launch_rows_norm_bf16(const RowArgs& a, cudaStream_t s) { launch_rows_typed<__nv_bfloat16, ROWS_NORM>(a, s); }

}  // namespace dmx
