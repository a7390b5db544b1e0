// The row kernels (rows.cuh) on f32 inputs.
#include "rows.cuh"

namespace dmx {

void launch_rows_f32(const RowArgs& a, cudaStream_t s) { launch_rows_typed<float>(a, s); }

}  // namespace dmx
