// The layer norm's backward pass (norm_grad.cuh) on bf16 rows with f16 gradients.
#include "norm_grad.cuh"

namespace dmx {

void launch_norm_grad_bf16_f16(const NormGradArgs& a, int parts, int how, bool wide, cudaStream_t s) {
  launch_norm_grad_typed<__nv_bfloat16, __half>(a, parts, how, wide, s);
}

}  // namespace dmx
