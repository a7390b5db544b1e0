// The row kernels (rows.cuh) of the layer norm on f16 rows.
#include "rows.cuh"

namespace dmx {

void launch_rows_norm_f16(const RowArgs& a, cudaStream_t s) { launch_rows_typed<__half, ROWS_NORM>(a, s); }

}  // namespace dmx
