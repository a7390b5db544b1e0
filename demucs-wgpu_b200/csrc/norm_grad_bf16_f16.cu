// The layer norm's backward pass (norm_grad.cuh) on bf16 rows with f16 gradients.
#include "norm_grad.cuh"

namespace dmx {

void launch_norm_grad_bf16_f16(const NormGradArgs& a, int parts, int vec,
                             cudaStream_t s) {
  const int type = a.weight ? a.param_type : DMX_TYPE_F32;
  if (type == DMX_TYPE_F32) launch_norm_grad_typed<__nv_bfloat16, __half, float>(a, parts, vec, s);
  else if (type == DMX_TYPE_F16) launch_norm_grad_typed<__nv_bfloat16, __half, __half>(a, parts, vec, s);
  else launch_norm_grad_typed<__nv_bfloat16, __half, __nv_bfloat16>(a, parts, vec, s);
}

}  // namespace dmx
