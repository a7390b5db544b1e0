// The row kernels (rows.cuh) of the quantiser on f16 rows.
#include "rows.cuh"

namespace dmx {

void launch_rows_quantize_f16(const RowArgs& a, cudaStream_t s) { launch_rows_typed<__half, ROWS_QUANTIZE>(a, s); }

}  // namespace dmx
