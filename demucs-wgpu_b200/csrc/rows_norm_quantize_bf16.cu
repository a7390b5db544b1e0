// The row kernels (rows.cuh) of the layer norm with the quantiser on bf16 rows.
#include "rows.cuh"

namespace dmx {

void launch_rows_norm_quantize_bf16(const RowArgs& a, cudaStream_t s) { launch_rows_typed<__nv_bfloat16, ROWS_NORM_QUANTIZE>(a, s); }

}  // namespace dmx
