// Element types of the public operators: loads to f32 and roundings from it,
// one value or eight neighbours at a time.
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

// Eight neighbours at a 16-byte boundary; `wide` (uniform): f32 ones at a
// 32-byte boundary, in one access. Loads are not through the read-only path: an
// operator may write its output over its input.
DMX_DEVICE void load8(const float* p, float* v, bool wide) {
  if (wide) return ld_global8(p, v);
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
DMX_DEVICE void load8(const __half* p, float* v, bool) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
DMX_DEVICE void load8(const __nv_bfloat16* p, float* v, bool) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
DMX_DEVICE void store8(float* p, const float* v, bool wide) {
  if (wide) return st_global8(p, v);
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
DMX_DEVICE void store8(__half* p, const float* v, bool) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
DMX_DEVICE void store8(__nv_bfloat16* p, const float* v, bool) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
// How the rows and vectors of a launch may be accessed.
enum { VEC_NONE = 0, VEC_16 = 1, VEC_32 = 2 };  // by elements; from 16-byte, from 32-byte boundaries

// A row is held by `threads` threads in pieces of eight values. Piece j of
// thread t is, if every row and vector starts on 16 bytes (`vec`), the eight
// neighbours from column (j threads + t) 8 on; else the eight columns
// (j 8 + e) threads + t, so that a warp's one-element accesses are neighbours.
struct Pieces {
  int t, threads, cols, vec;
  DMX_DEVICE int col(int j, int e) const {
    return vec ? (j * threads + t) * 8 + e : (j * 8 + e) * threads + t;
  }
  // all eight columns of piece j exist
  DMX_DEVICE bool whole(int j) const { return col(j, 7) < cols; }
  DMX_DEVICE bool has(int j, int e) const { return col(j, e) < cols; }

  // columns past the row's end come as `fill`
  template <typename T>
  DMX_DEVICE void load(const T* p, int j, float* v, float fill = 0.f) const {
    if (vec && whole(j)) {
      load8(p + col(j, 0), v, vec == VEC_32);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = has(j, e) ? to_f32(p[col(j, e)]) : fill;
    }
  }
  template <typename T>
  DMX_DEVICE void store(T* p, int j, const float* v) const {
    if (vec && whole(j)) {
      store8(p + col(j, 0), v, vec == VEC_32);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (has(j, e)) p[col(j, e)] = from_f32<T>(v[e]);
    }
  }
  // the same for a type known only at run time (uniform over the launch)
  DMX_DEVICE void load(const void* p, int type, int j, float* v) const {
    if (type == DMX_TYPE_F32) load(static_cast<const float*>(p), j, v);
    else if (type == DMX_TYPE_F16) load(static_cast<const __half*>(p), j, v);
    else load(static_cast<const __nv_bfloat16*>(p), j, v);
  }
  DMX_DEVICE void store(void* p, int type, int64_t row0, int j, const float* v) const {
    if (type == DMX_TYPE_F32) store(static_cast<float*>(p) + row0, j, v);
    else if (type == DMX_TYPE_F16) store(static_cast<__half*>(p) + row0, j, v);
    else store(static_cast<__nv_bfloat16*>(p) + row0, j, v);
  }
};

// The widest access that suits rows of `ld` elements of `bytes` bytes from p
// on (ld 0: a vector): 16-bit elements need 16 bytes for eight, f32 ones 32.
inline int vec_of(const void* p, int64_t ld, int bytes) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * bytes);
  return at % 16 ? VEC_NONE : at % 32 && bytes == 4 ? VEC_16 : VEC_32;
}
inline int type_size(int type) { return type == DMX_TYPE_F32 ? 4 : 2; }

}  // namespace dmx
