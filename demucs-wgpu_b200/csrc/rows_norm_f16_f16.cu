// The layer norm's row kernels (rows.cuh) on f16 rows with f16 parameters.
#include "rows.cuh"

namespace dmx {

void launch_rows_norm_f16_f16(const RowArgs& a, cudaStream_t s) { launch_rows_norm<__half, __half>(a, s); }

}  // namespace dmx
