// The row kernels (rows.cuh) of the layer norm on f32 rows.
#include "rows.cuh"

namespace dmx {

void launch_rows_norm_f32(const RowArgs& a, cudaStream_t s) { launch_rows_typed<float, ROWS_NORM>(a, s); }

}  // namespace dmx
