// The row kernels (rows.cuh) on bf16 inputs.
#include "rows.cuh"

namespace dmx {

void launch_rows_bf16(const RowArgs& a, cudaStream_t s) { launch_rows_typed<__nv_bfloat16>(a, s); }

}  // namespace dmx
