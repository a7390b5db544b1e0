// The layer norm's backward pass (norm_grad.cuh) on bf16 rows with bf16 gradients.
#include "norm_grad.cuh"

namespace dmx {

void launch_norm_grad_bf16_bf16(const NormGradArgs& a, int parts, int vec,
                             cudaStream_t s) {
  const int type = a.weight ? a.param_type : DMX_TYPE_F32;
  if (type == DMX_TYPE_F32) launch_norm_grad_typed<__nv_bfloat16, __nv_bfloat16, float>(a, parts, vec, s);
  else if (type == DMX_TYPE_F16) launch_norm_grad_typed<__nv_bfloat16, __nv_bfloat16, __half>(a, parts, vec, s);
  else launch_norm_grad_typed<__nv_bfloat16, __nv_bfloat16, __nv_bfloat16>(a, parts, vec, s);
}

}  // namespace dmx
