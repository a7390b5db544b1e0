// The layer norm's backward pass (norm_grad.cuh) on f32 rows with f32 gradients.
#include "norm_grad.cuh"

namespace dmx {

void launch_norm_grad_f32_f32(const NormGradArgs& a, int parts, int vec,
                             cudaStream_t s) {
  const int type = a.weight ? a.param_type : DMX_TYPE_F32;
  if (type == DMX_TYPE_F32) launch_norm_grad_typed<float, float, float>(a, parts, vec, s);
  else if (type == DMX_TYPE_F16) launch_norm_grad_typed<float, float, __half>(a, parts, vec, s);
  else launch_norm_grad_typed<float, float, __nv_bfloat16>(a, parts, vec, s);
}

}  // namespace dmx
