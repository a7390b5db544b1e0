// The row kernels (rows.cuh) on f16 inputs.
#include "rows.cuh"

namespace dmx {

void launch_rows_f16(const RowArgs& a, cudaStream_t s) { launch_rows_typed<__half>(a, s); }

}  // namespace dmx
