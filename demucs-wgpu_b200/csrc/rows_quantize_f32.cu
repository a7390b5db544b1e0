// The row kernels (rows.cuh) of the quantiser on f32 rows.
#include "rows.cuh"

namespace dmx {

void launch_rows_quantize_f32(const RowArgs& a, cudaStream_t s) { launch_rows_typed<float, ROWS_QUANTIZE>(a, s); }

}  // namespace dmx
