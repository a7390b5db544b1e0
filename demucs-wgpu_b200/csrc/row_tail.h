// The end of a row of bytes, read without a byte past it (host and device).
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define DMX_BOTH __host__ __device__ __forceinline__
#else
#define DMX_BOTH inline
#endif

namespace dmx {

// The `left` (1..15) bytes from the 16-byte boundary p on, then zeros, as four
// words. Read in pieces of 8, 4, 2 and 1 bytes, each at a multiple of its size:
// a buffer may end with its last row's last value.
DMX_BOTH void read_tail16(const void* p, int left, uint32_t* w) {
  const char* at = static_cast<const char*>(p);
  uint64_t lo = 0, rest = 0;
  int shift = 0;
  if (left & 8) {
    lo = *reinterpret_cast<const uint64_t*>(at);
    at += 8;
  }
  if (left & 4) {
    rest = *reinterpret_cast<const uint32_t*>(at);
    at += 4;
    shift = 32;
  }
  if (left & 2) {
    rest |= static_cast<uint64_t>(*reinterpret_cast<const uint16_t*>(at)) << shift;
    at += 2;
    shift += 16;
  }
  if (left & 1) rest |= static_cast<uint64_t>(*reinterpret_cast<const uint8_t*>(at)) << shift;
  const uint64_t hi = left & 8 ? rest : 0;
  lo = left & 8 ? lo : rest;
  w[0] = static_cast<uint32_t>(lo);
  w[1] = static_cast<uint32_t>(lo >> 32);
  w[2] = static_cast<uint32_t>(hi);
  w[3] = static_cast<uint32_t>(hi >> 32);
}

}  // namespace dmx
