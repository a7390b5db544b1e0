// Element types of the public operators: loads to f32 and roundings from it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "dmx.h"

namespace dmx {

DMX_DEVICE float to_f32(float v) { return v; }
DMX_DEVICE float to_f32(__half v) { return __half2float(v); }
DMX_DEVICE float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
DMX_DEVICE T from_f32(float v);
template <>
DMX_DEVICE float from_f32<float>(float v) { return v; }
template <>
DMX_DEVICE __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
DMX_DEVICE __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// One element of an array whose type is known only at run time (uniform over the launch).
DMX_DEVICE float load_as_f32(const void* p, int type, int64_t i) {
  if (type == DMX_TYPE_F32) return static_cast<const float*>(p)[i];
  if (type == DMX_TYPE_F16) return to_f32(static_cast<const __half*>(p)[i]);
  return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
}
DMX_DEVICE void store_from_f32(void* p, int type, int64_t i, float v) {
  if (type == DMX_TYPE_F32) static_cast<float*>(p)[i] = v;
  else if (type == DMX_TYPE_F16) static_cast<__half*>(p)[i] = from_f32<__half>(v);
  else static_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v);
}

}  // namespace dmx
