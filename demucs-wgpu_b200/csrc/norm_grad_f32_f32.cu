// The layer norm's backward pass (norm_grad.cuh) on f32 rows with f32 gradients.
#include "norm_grad.cuh"

namespace dmx {

void launch_norm_grad_f32_f32(const NormGradArgs& a, int parts, int how, bool wide, cudaStream_t s) {
  launch_norm_grad_typed<float, float>(a, parts, how, wide, s);
}

}  // namespace dmx
