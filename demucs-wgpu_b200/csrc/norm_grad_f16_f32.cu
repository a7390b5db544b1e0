// The layer norm's backward pass (norm_grad.cuh) on f16 rows with f32 gradients.
#include "norm_grad.cuh"

namespace dmx {

void launch_norm_grad_f16_f32(const NormGradArgs& a, int parts, int how, bool wide, cudaStream_t s) {
  launch_norm_grad_typed<__half, float>(a, parts, how, wide, s);
}

}  // namespace dmx
