// Element types of the public operators: loads to f32 and roundings from it,
// one value or eight neighbours at a time.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "dmx.h"
#include "ops.h"

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

// 16- and 32-byte accesses in inline PTX, so that a branch on a type known
// only at run time stays a branch: the compiler would otherwise run all three
// types' loads and conversions under predicates (twice the instructions of a
// bf16 row's arithmetic). Not through the read-only path: an operator may
// write its output over its input. No "memory" clobber, which made the
// compiler fetch the launch's arguments anew after every access; the volatile
// ones keep their order among themselves, and every thread stores only what
// it has loaded.
DMX_DEVICE void ld_words4(const void* p, uint32_t* w) {
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "l"(p));
}
DMX_DEVICE void ld_words8(const void* p, uint32_t* w) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]),
                 "=r"(w[7])
               : "l"(p));
}
DMX_DEVICE void st_words4(void* p, const uint32_t* w) {
  asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]));
}
DMX_DEVICE void st_words8(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]),
               "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]));
}

// One element of a cut piece: in PTX too, so that these rare ones are branched over.
DMX_DEVICE uint32_t ld_bits(const float* p) {
  uint32_t w;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(w) : "l"(p));
  return w;
}
DMX_DEVICE uint32_t ld_bits(const __half* p) {
  uint16_t w;
  asm volatile("ld.global.u16 %0, [%1];" : "=h"(w) : "l"(p));
  return w;
}
DMX_DEVICE uint32_t ld_bits(const __nv_bfloat16* p) {
  return ld_bits(reinterpret_cast<const __half*>(p));
}
DMX_DEVICE void st_value(float* p, float v) { asm volatile("st.global.f32 [%0], %1;" ::"l"(p), "f"(v)); }
DMX_DEVICE void st_value(__half* p, __half v) {
  asm volatile("st.global.u16 [%0], %1;" ::"l"(p), "h"(__half_as_ushort(v)));
}
DMX_DEVICE void st_value(__nv_bfloat16* p, __nv_bfloat16 v) {
  asm volatile("st.global.u16 [%0], %1;" ::"l"(p), "h"(__bfloat16_as_ushort(v)));
}

// Eight neighbours at a 16-byte boundary as they lie in memory (f32: 8 words,
// 16-bit types: 4); `wide` (uniform): f32 ones at a 32-byte boundary, in one access.
DMX_DEVICE void fetch8(const float* p, uint32_t* w, bool wide) {
  if (wide) return ld_words8(p, w);
  ld_words4(p, w);
  ld_words4(p + 4, w + 4);
}
DMX_DEVICE void fetch8(const __half* p, uint32_t* w, bool) { ld_words4(p, w); }
DMX_DEVICE void fetch8(const __nv_bfloat16* p, uint32_t* w, bool) { ld_words4(p, w); }

DMX_DEVICE void unpack8(const uint32_t* w, float* v, float) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}
DMX_DEVICE void unpack8(const uint32_t* w, float* v, __half) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
DMX_DEVICE void unpack8(const uint32_t* w, float* v, __nv_bfloat16) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
// one element in a word of its own
DMX_DEVICE uint32_t bits_of(float v) { return __float_as_uint(v); }
DMX_DEVICE uint32_t bits_of(__half v) { return __half_as_ushort(v); }
DMX_DEVICE uint32_t bits_of(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
DMX_DEVICE float from_bits(uint32_t w, float) { return __uint_as_float(w); }
DMX_DEVICE float from_bits(uint32_t w, __half) { return __half2float(__ushort_as_half((unsigned short)w)); }
DMX_DEVICE float from_bits(uint32_t w, __nv_bfloat16) { return __uint_as_float(w << 16); }

// two values in one word, the first in its low half
DMX_DEVICE uint32_t pack2(float lo, float hi, __half) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
DMX_DEVICE uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
DMX_DEVICE void store8(float* p, const float* v, bool wide) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
  if (wide) return st_words8(p, w);
  st_words4(p, w);
  st_words4(p + 4, w + 4);
}
template <typename T>
DMX_DEVICE void store8(T* p, const float* v, bool) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2(v[2 * i], v[2 * i + 1], T());
  st_words4(p, w);
}

// Four neighbours at a boundary of four elements.
DMX_DEVICE float4 load4(const float* p) {
  uint32_t w[4];
  ld_words4(p, w);
  return make_float4(__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]),
                     __uint_as_float(w[3]));
}
template <typename T>
DMX_DEVICE float4 load4(const T* p) {
  uint32_t w[4] = {0, 0, 0, 0};
  asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  float v[8];
  unpack8(w, v, T());
  return make_float4(v[0], v[1], v[2], v[3]);
}
DMX_DEVICE void store4(float* p, float4 v) {
  const uint32_t w[4] = {__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z),
                         __float_as_uint(v.w)};
  st_words4(p, w);
}
template <typename T>
DMX_DEVICE void store4(T* p, float4 v) {
  asm volatile("st.global.v2.b32 [%0], {%1, %2};" ::"l"(p), "r"(pack2(v.x, v.y, T())),
               "r"(pack2(v.z, v.w, T())));
}

// Eight values, two to an instruction.
DMX_DEVICE void scale8(float* v, float w) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 r = __fmul2_rn(make_float2(v[e], v[e + 1]), make_float2(w, w));
    v[e] = r.x;
    v[e + 1] = r.y;
  }
}
DMX_DEVICE void times8(float* v, const float* w) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 r = __fmul2_rn(make_float2(v[e], v[e + 1]), make_float2(w[e], w[e + 1]));
    v[e] = r.x;
    v[e + 1] = r.y;
  }
}
DMX_DEVICE void plus8(float* v, const float* w) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 r = __fadd2_rn(make_float2(v[e], v[e + 1]), make_float2(w[e], w[e + 1]));
    v[e] = r.x;
    v[e + 1] = r.y;
  }
}
DMX_DEVICE void centre8(float* v, float mean) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 r = __fadd2_rn(make_float2(v[e], v[e + 1]), make_float2(-mean, -mean));
    v[e] = r.x;
    v[e + 1] = r.y;
  }
}

// How a kernel reads its rows: element by element, by vectors, or (rows that
// start off 16 bytes) by vectors shifted into place.
enum { BY_ELEMENT = 0, BY_VECTOR = 1, BY_SHIFT = 2 };

// How the rows and vectors of a launch may be accessed.
enum { VEC_NONE = 0, VEC_16 = 1, VEC_32 = 2 };  // by elements; from 16-byte, from 32-byte boundaries

// An array whose type is known only at run time (uniform over the launch), and
// the tag that stands for its type in templates. Kernels without vector
// accesses take parameters this way: a third of the instantiations.
struct Any {};
struct AnyArray {
  const void* p;
  int type;
  DMX_DEVICE explicit operator bool() const { return p != nullptr; }
};
template <typename T>
DMX_DEVICE const T* array_of(const void* p, int, T) { return static_cast<const T*>(p); }
DMX_DEVICE AnyArray array_of(const void* p, int type, Any) { return {p, type}; }

// f(T()) for the element type that `type` names (uniform over the launch)
template <typename F>
DMX_DEVICE void with_type(int type, F&& f) {
  if (type == DMX_TYPE_F32) f(float());
  else if (type == DMX_TYPE_F16) f(__half());
  else f(__nv_bfloat16());
}
DMX_DEVICE float from_bits(uint32_t w, Any) { return __uint_as_float(w); }

// A row is held by `threads` threads in pieces of eight values. Piece j of
// thread t is, if every row and vector starts on 16 bytes (VEC), the eight
// neighbours from column (j threads + t) 8 on; else the eight columns
// (j 8 + e) threads + t, so that a warp's one-element accesses are neighbours.
template <bool VEC>
struct Pieces {
  int t, threads, cols;
  bool wide;  // VEC: 32-byte boundaries too
  DMX_DEVICE int col(int j, int e) const {
    return VEC ? (j * threads + t) * 8 + e : (j * 8 + e) * threads + t;
  }
  // all eight columns of piece j exist
  DMX_DEVICE bool whole(int j) const { return col(j, 7) < cols; }
  DMX_DEVICE bool has(int j, int e) const { return col(j, e) < cols; }
  // Some piece of the row (uniform) or piece j may hold only some of its
  // columns: with VEC, in rows whose length is no multiple of eight.
  DMX_DEVICE bool ragged() const { return !VEC || (cols & 7); }
  DMX_DEVICE bool cut(int j) const { return has(j, 0) && !whole(j); }

  // Piece j of a row as it lies in memory (VEC: words of the packed values;
  // else one value a word). Columns past the row's end come as 0.
  template <typename T>
  DMX_DEVICE void fetch(const T* p, int j, uint32_t* w) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 0;
    if (!VEC) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (has(j, e)) w[e] = bits_of(p[col(j, e)]);
    } else if (whole(j)) {
      fetch8(p + col(j, 0), w, wide);
    } else if (cut(j)) {
      constexpr int kPer = 4 / sizeof(T);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (has(j, e)) w[e / kPer] |= ld_bits(p + col(j, e)) << (e % kPer * 16);
    }
  }
  // The same (VEC) of a row that starts anywhere: the 16-byte units around the
  // piece, shifted by the row's offset in them. A unit that sticks out of the
  // row is put together from the row's own elements.
  template <typename T>
  DMX_DEVICE void fetch_shifted(const T* p, int j, uint32_t* w) const {
    constexpr int kSize = sizeof(T), kUnit = 16 / kSize, kUnits = 8 / kUnit + 1, kWords = 4 * kUnits;
    uint32_t u[kWords + 1];
    const int off = (int)(reinterpret_cast<uintptr_t>(p) & 15);  // uniform over the row
    const int from = col(j, 0) - off / kSize;                    // first element of the first unit
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int c = from + k * kUnit;
      if (c >= 0 && c + kUnit <= cols) {
        ld_words4(p + c, u + 4 * k);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) u[4 * k + i] = 0;
        if (c + kUnit > 0 && c < cols) {
#pragma unroll
          for (int i = 0; i < kUnit; ++i)
            if (c + i >= 0 && c + i < cols)
              u[4 * k + i * kSize / 4] |= ld_bits(p + c + i) << (i * kSize % 4 * 8);
        }
      }
    }
    u[kWords] = 0;
    const bool two = off & 8, one = off & 4;
#pragma unroll
    for (int i = 0; i + 2 <= kWords; ++i) u[i] = two ? u[i + 2] : u[i];
#pragma unroll
    for (int i = 0; i + 1 <= kWords - 2; ++i) u[i] = one ? u[i + 1] : u[i];
    const int bits = (off & 3) * 8;
#pragma unroll
    for (int i = 0; i < 2 * kSize; ++i) w[i] = kSize == 4 ? u[i] : __funnelshift_r(u[i], u[i + 1], bits);
  }
  DMX_DEVICE void fetch(AnyArray p, int j, uint32_t* w) const {  // without VEC
    with_type(p.type, [&](auto type) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        w[e] = has(j, e) ? __float_as_uint(to_f32(static_cast<const decltype(type)*>(p.p)[col(j, e)]))
                         : 0;
    });
  }
  template <typename T>
  DMX_DEVICE static void unpack(const uint32_t* w, float* v) {
    if constexpr (VEC) {
      unpack8(w, v, T());
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = from_bits(w[e], T());
    }
  }
  template <typename T>
  DMX_DEVICE void load(const T* p, int j, float* v) const {
    uint32_t w[8];
    fetch(p, j, w);
    unpack<T>(w, v);
  }
  template <typename T>
  DMX_DEVICE void store(T* p, int j, const float* v) const {
    if (VEC && whole(j)) {
      store8(p + col(j, 0), v, wide);
    } else if (!VEC || cut(j)) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (has(j, e)) st_value(p + col(j, e), from_f32<T>(v[e]));
    }
  }
};

// Eight values of each lane to rows that start anywhere: through `buf` (1 KB, a
// warp's own), so that a warp's one-element stores are neighbours. LANES lanes
// share a row, whose columns from `col0` on are the first one's; `row0` is the
// warp's first row. Every lane takes part.
template <int LANES, typename T>
DMX_DEVICE void store_crossed(T* buf, const float* v, T* out, int64_t ld, int64_t row0, int64_t rows,
                              int col0, int cols) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int e = 0; e < 8; ++e) buf[lane * 8 + e] = from_f32<T>(v[e]);
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int at = e * 32 + lane, c = col0 + at % (LANES * 8);
    const int64_t row = row0 + at / (LANES * 8);
    if (row < rows && c < cols) out[row * ld + c] = buf[at];
  }
  __syncwarp();
}

// The operators' kernels are launched so that one may begin while the kernel
// before it in the stream still runs (programmatic dependent launch): its
// blocks set themselves up, then wait here for that kernel's end. Nothing that
// a kernel before could have written, and nothing at all is written, before
// after_earlier_kernels() (prefetches into L2 excepted, which fetch no value).
DMX_DEVICE void let_next_kernel_begin() { asm volatile("griddepcontrol.launch_dependents;"); }
DMX_DEVICE void after_earlier_kernels() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// `early` false: the kernel begins after the one before it. That is for kernels
// of many rounds of short blocks: the first ones, waiting beside the kernel
// before, would keep the SMs at its division of shared memory and L1 for as
// long as blocks follow one another without a gap (after the linear's tiles,
// which leave L1 28 KB: 112896x2048 quantised in 164 us against 145).
template <typename... P, typename... A>
void launch_chained(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, bool early,
                    unsigned cluster, A&&... args) {
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = early;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim = {cluster, 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  check_cuda(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
}

// The widest access that suits rows of `ld` elements of `bytes` bytes from p
// on (ld 0: a vector): 16-bit elements need 16 bytes for eight, f32 ones 32.
inline int vec_of(const void* p, int64_t ld, int bytes) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * bytes);
  return at % 16 ? VEC_NONE : at % 32 && bytes == 4 ? VEC_16 : VEC_32;
}
constexpr int type_code(float) { return DMX_TYPE_F32; }
constexpr int type_code(__half) { return DMX_TYPE_F16; }
constexpr int type_code(__nv_bfloat16) { return DMX_TYPE_BF16; }
inline int type_size(int type) { return type == DMX_TYPE_F32 ? 4 : 2; }

}  // namespace dmx
