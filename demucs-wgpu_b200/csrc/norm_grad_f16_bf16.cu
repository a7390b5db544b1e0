// The layer norm's backward pass (norm_grad.cuh) on f16 rows with bf16 gradients.
#include "norm_grad.cuh"

namespace dmx {

void launch_norm_grad_f16_bf16(const NormGradArgs& a, int parts, int how, bool wide, cudaStream_t s) {
  launch_norm_grad_typed<__half, __nv_bfloat16>(a, parts, how, wide, s);
}

}  // namespace dmx
