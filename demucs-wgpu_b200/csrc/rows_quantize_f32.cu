// The quantiser's row kernels (rows.cuh) on f32 rows.
#include "rows.cuh"

namespace dmx {

void launch_rows_quantize_f32(const RowArgs& a, cudaStream_t s) {
  const int vec = std::min(vec_of(a.x, a.x_ld, sizeof(float)), vec_of(a.col_scale, 0, 4));
  launch_rows_vec<float, float, ROWS_QUANTIZE>(a, vec, vec_of(a.q, a.q_ld, 1) != VEC_NONE, s);
}

}  // namespace dmx
