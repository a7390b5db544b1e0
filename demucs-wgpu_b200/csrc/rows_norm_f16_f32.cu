// The layer norm's row kernels (rows.cuh) on f16 rows with f32 parameters.
#include "rows.cuh"

namespace dmx {

void launch_rows_norm_f16_f32(const RowArgs& a, cudaStream_t s) { launch_rows_norm<__half, float>(a, s); }

}  // namespace dmx
