// The 8-bit linear layer (dmx_quantized_linear):
//
//   out[m][n] = act(acc[m][n] x_scale[m] w_scale[n] + bias[n]) + residual[m][n]
//   acc[m][n] = sum_k x[m][k] w[n][k], exact in 32-bit integers
//
// Three kernels, all on the same operands (rows on 16-byte boundaries, the
// bytes past column k of a row never used):
//  * linear_gemv_kernel: up to 8 rows, dp4a on weights streamed once;
//  * linear_few_kernel: up to 128 rows, tcgen05 with the weights as the
//    128-row operand, k split over a thread-block cluster;
//  * linear_tile_kernel: more rows, persistent tcgen05 tiles of 128 x BN.
#include <algorithm>

#include "ops.h"
#include "ops_common.cuh"
#include "tc_common.cuh"

namespace dmx {

namespace {

constexpr int kBlockK = 128;  // bytes of k per pipeline stage: one 128-byte swizzled row

// D (+)= A B^T on signed 8-bit integers (K = 32 per instruction), 32-bit integer accumulator.
DMX_DEVICE void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
// s32 accumulator, s8 operands, both K-major, 128 x n
constexpr uint32_t i8_idesc(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

template <typename OT, bool GELU>
DMX_DEVICE float activate(float v) {
  return GELU ? gelu(v) : v;
}

// One output from its exact sum: scales in the order row, channel, then the
// bias in the same rounding as the last product.
template <typename OT, bool GELU>
DMX_DEVICE float linear_value(int acc, float xs, float ws, float b) {
  return activate<OT, GELU>(fmaf((float)acc * xs, ws, b));
}

template <typename OT>
DMX_DEVICE void store_out(const LinearArgs& a, int64_t m, int n, float v) {
  if (a.residual)
    v += to_f32(static_cast<const OT*>(a.residual)[m * a.residual_ld + n]);
  static_cast<OT*>(a.out)[m * a.out_ld + n] = from_f32<OT>(v);
}

// ---------------------------------------------------------------------------
// up to 8 rows
// ---------------------------------------------------------------------------

// Bytes k0 .. k0 + 15 of a row of `k` values, the ones past its end as zero.
DMX_DEVICE int4 row16(const int8_t* row, int k0, int k) {
  int4 v = make_int4(0, 0, 0, 0);
  if (k0 >= k) return v;
  v = __ldg(reinterpret_cast<const int4*>(row + k0));
  const int left = k - k0;
  if (left < 16) {
    int* w = reinterpret_cast<int*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int bytes = min(max(left - 4 * i, 0), 4);
      w[i] = bytes == 4 ? w[i] : (w[i] & ((1 << (8 * bytes)) - 1));
    }
  }
  return v;
}
DMX_DEVICE int dot16(int4 x, int4 w, int acc) {
  acc = __dp4a(x.x, w.x, acc);
  acc = __dp4a(x.y, w.y, acc);
  acc = __dp4a(x.z, w.z, acc);
  return __dp4a(x.w, w.w, acc);
}

constexpr int kGemvThreads = 256;

// A warp takes C channels and every `kw`-th 512-byte piece of k; the `kw`
// warps of one channel group (8 / kw groups per block) are summed through
// shared memory. x (at most 8 rows) stays in L1.
template <int M, int C, typename OT, bool GELU>
__global__ void __launch_bounds__(kGemvThreads) linear_gemv_kernel(const LinearArgs a, int kw) {
  __shared__ int part[kGemvThreads / 32][M * C];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int groups = (kGemvThreads / 32) / kw, group = warp / kw, kpart = warp % kw;
  const int n0 = (blockIdx.x * groups + group) * C;
  int acc[M][C];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int c = 0; c < C; ++c) acc[m][c] = 0;
  if (n0 < a.n) {
#pragma unroll 2
    for (int k0 = kpart * 512 + lane * 16; k0 < a.k; k0 += kw * 512) {
      int4 w[C], x[M];
#pragma unroll
      for (int c = 0; c < C; ++c)
        w[c] = row16(a.w + (int64_t)min(n0 + c, a.n - 1) * a.w_ld, k0, a.k);
#pragma unroll
      for (int m = 0; m < M; ++m)
        x[m] = row16(a.x + min((int64_t)m, a.rows - 1) * a.x_ld, k0, a.k);
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[m][c] = dot16(x[m], w[c], acc[m][c]);
    }
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int t = __reduce_add_sync(0xffffffffu, acc[m][c]);
      if (lane == 0) part[warp][m * C + c] = t;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < groups * M * C; i += kGemvThreads) {
    const int g = i / (M * C), e = i % (M * C), m = e / C;
    const int n = (blockIdx.x * groups + g) * C + e % C;
    if (n >= a.n || m >= a.rows) continue;
    int t = 0;
    for (int p = 0; p < kw; ++p) t += part[g * kw + p][e];
    store_out<OT>(a, m, n,
                  linear_value<OT, GELU>(t, a.x_scale ? a.x_scale[m] : 1.f,
                                         a.w_scale ? a.w_scale[n] : 1.f, a.bias ? a.bias[n] : 0.f));
  }
}

// ---------------------------------------------------------------------------
// tcgen05: what both kernels share
// ---------------------------------------------------------------------------

struct Pipe {
  uint64_t *full, *empty;
};

// After a wait gave up: nothing this CTA started may still write its shared
// memory or read it when it exits. Waits (bounded) for the loads issued last
// into each stage.
template <int STAGES>
DMX_DEVICE void drain_loads(const Pipe& p, uint32_t issued, int* err) {
  for (uint32_t it = issued > STAGES ? issued - STAGES : 0; it < issued; ++it)
    mbar_wait(&p.full[it % STAGES], (it / STAGES) & 1, err, 14);
}
// The same for the MMAs issued so far.
DMX_DEVICE void drain_mmas(uint64_t* bar, int* err) {
  umma_commit(bar);
  mbar_wait(bar, 0, err, 15);
}

DMX_DEVICE void tmem_alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_u32(slot)),
               "r"(cols));
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
DMX_DEVICE void tmem_free(uint32_t tmem, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols));
}
DMX_DEVICE void tc_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
DMX_DEVICE void tc_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Every thread of the cluster: shared-memory writes before it are seen after it.
DMX_DEVICE void cluster_sync() {
  asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}

// The MMAs of one landed stage: `left` bytes of k, 32 per instruction (the
// rest of a last stage was filled with zeros).
template <int N>
DMX_DEVICE void mma_stage(uint32_t d, uint32_t a_addr, uint32_t b_addr, int left, bool first) {
#pragma unroll
  for (int j = 0; j < kBlockK / 32; ++j)
    if (j * 32 < left)
      umma_i8(d, umma_desc_k(a_addr + j * 32, 128), umma_desc_k(b_addr + j * 32, 128), i8_idesc(N),
              !(first && j == 0));
}

// ---------------------------------------------------------------------------
// up to 128 rows: out^T tile of 128 channels x BT rows per cluster
// ---------------------------------------------------------------------------

constexpr int kFewThreads = 192;  // warp 0 TMA, warp 1 MMA, warps 2-5 read the accumulator

template <int BT, int STAGES>
struct FewSmem {
  static constexpr int A = 128 * kBlockK, B = BT * kBlockK, STAGE = A + B;
  // the partial sums [BT][128] reuse the stages
  static constexpr int RING = STAGES * STAGE > BT * 512 ? STAGES * STAGE : BT * 512;
  static constexpr int TOTAL = RING + 1024 + 256;
  static constexpr uint32_t COLS = BT < 32 ? 32 : BT;
};

template <int BT, int STAGES, typename OT, bool GELU>
__global__ void __launch_bounds__(kFewThreads)
    linear_few_kernel(const __grid_constant__ CUtensorMap tm_w,
                      const __grid_constant__ CUtensorMap tm_x, const LinearArgs a, int splits) {
  using S = FewSmem<BT, STAGES>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Pipe pipe;
  pipe.full = reinterpret_cast<uint64_t*>(smem + S::RING);
  pipe.empty = pipe.full + STAGES;
  uint64_t* done = pipe.empty + STAGES;
  uint64_t* drain = done + 1;
  uint32_t* slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int split = blockIdx.x % splits, n0 = (blockIdx.x / splits) * 128, m0 = blockIdx.y * BT;
  const int blocks = (a.k + kBlockK - 1) / kBlockK;
  const int lo = (int)((int64_t)blocks * split / splits);
  const int hi = (int)((int64_t)blocks * (split + 1) / splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&pipe.full[s], 1);
      mbar_init(&pipe.empty[s], 1);
    }
    mbar_init(done, 1);
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(slot, S::COLS);
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  const uint32_t tmem = *slot;

  if (warp == 0 && lane == 0) {
    uint32_t it = 0;
    for (int kb = lo; kb < hi; ++kb, ++it) {
      const int s = it % STAGES;
      if (!mbar_wait(&pipe.empty[s], ((it / STAGES) & 1) ^ 1, a.err, 11)) break;
      unsigned char* dst = smem + s * S::STAGE;
      mbar_expect_tx(&pipe.full[s], S::STAGE);
      tma_load_2d(dst, &tm_w, &pipe.full[s], kb * kBlockK, n0);
      tma_load_2d(dst + S::A, &tm_x, &pipe.full[s], kb * kBlockK, m0);
    }
    if (it < (uint32_t)(hi - lo)) drain_loads<STAGES>(pipe, it, a.err);
  } else if (warp == 1 && lane == 0) {
    uint32_t it = 0;
    for (int kb = lo; kb < hi; ++kb, ++it) {
      const int s = it % STAGES;
      if (!mbar_wait(&pipe.full[s], (it / STAGES) & 1, a.err, 12)) break;
      tc_after_sync();
      const uint32_t addr = smem_u32(smem + s * S::STAGE);
      mma_stage<BT>(tmem, addr, addr + S::A, a.k - kb * kBlockK, kb == lo);
      umma_commit(&pipe.empty[s]);
    }
    if (it < (uint32_t)(hi - lo)) drain_mmas(drain, a.err);
    else umma_commit(done);
  }
  __syncwarp();
  int* part = reinterpret_cast<int*>(smem);  // [BT][128]
  if (warp >= 2) {
    // lane = channel, column = row of x: [row][channel] is written without bank conflicts
    const int q = warp % 4;
    // the lanes may end a wait that gave up apart
    const bool ok = __all_sync(0xffffffffu, mbar_wait(done, 0, a.err, 13));
    tc_after_sync();
    const uint32_t base = tmem + ((uint32_t)(q * 32) << 16);
    if (ok) {
#pragma unroll
      for (int c = 0; c < BT; c += 16) {
        uint32_t r[16];
        tmem_ld16_nw(base + c, r);
        tmem_ld_wait<16>(r);
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(c + i) * 128 + q * 32 + lane] = (int)r[i];
      }
    }
    tc_before_sync();
  }
  if (splits > 1) cluster_sync();
  else __syncthreads();
  // each CTA of the cluster finishes its share of the rows
  const int rows = (int)min((int64_t)BT, a.rows - m0), cols = min(128, a.n - n0);
  for (int i = threadIdx.x; i < rows * 128; i += kFewThreads) {
    const int m = i / 128, c = i % 128;
    if (m % splits != split || c >= cols) continue;
    int acc = 0;
    if (splits > 1) {
      const uint32_t at = smem_u32(part + m * 128 + c);
      for (int p = 0; p < splits; ++p) {
        uint32_t peer;
        int v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(p));
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(peer) : "memory");
        acc += v;
      }
    } else {
      acc = part[m * 128 + c];
    }
    const int n = n0 + c;
    const int64_t row = m0 + m;
    store_out<OT>(a, row, n,
                  linear_value<OT, GELU>(acc, a.x_scale ? a.x_scale[row] : 1.f,
                                         a.w_scale ? a.w_scale[n] : 1.f, a.bias ? a.bias[n] : 0.f));
  }
  // a peer may still be reading this CTA's partial sums
  if (splits > 1) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_after_sync();
    tmem_free(tmem, S::COLS);
  }
}

// ---------------------------------------------------------------------------
// more rows: persistent 128 x BN tiles
// ---------------------------------------------------------------------------

constexpr int kTileThreads = 320;  // warp 0 TMA, warp 1 MMA, warps 2-9 epilogue
constexpr int kEpiThreads = 256;
constexpr int kGroupRows = 8;  // row tiles per group of the tile order

template <int BN>
struct TileSmem {
  static constexpr int A = 128 * kBlockK, B = BN * kBlockK, STAGE = A + B;
  static constexpr int STAGES = 192 * 1024 / STAGE;
  static constexpr int COLUMN = 2 * BN * 8;             // two tiles' (w_scale, bias) pairs
  static constexpr int TURN = (kEpiThreads / 32) * 32 * 17 * 4;  // epilogue warps' transposes
  static constexpr int TOTAL = STAGES * STAGE + COLUMN + TURN + 1024 + 256;
  static constexpr uint32_t COLS = 2 * BN;
};

// Tile t of the order: groups of kGroupRows row tiles, row tile fastest, so
// the CTAs at work together share both operands' tiles in L2.
DMX_DEVICE void tile_at(int64_t t, int64_t mtiles, int ntiles, int64_t& m0, int& n_tile) {
  const int64_t per = (int64_t)kGroupRows * ntiles, g = t / per;
  const int64_t in_group = t - g * per;
  const int high = (int)min((int64_t)kGroupRows, mtiles - g * kGroupRows);
  n_tile = (int)(in_group / high);
  m0 = (g * kGroupRows + in_group % high) * 128;
}

template <typename OT>
struct Pack;  // 16 values of a row as 32-byte accesses
template <>
struct Pack<float> {
  static DMX_DEVICE void store(float* p, const float* v) {
    st_global8(p, v);
    st_global8(p + 8, v + 8);
  }
  static DMX_DEVICE void load(const float* p, float* v) {
    ld_global8(p, v);
    ld_global8(p + 8, v + 8);
  }
};
template <>
struct Pack<__half> {
  static DMX_DEVICE void store(__half* p, const float* v) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    st_global8(reinterpret_cast<uint32_t*>(p), w);
  }
  static DMX_DEVICE void load(const __half* p, float* v) {
    float w[8];
    ld_global8(reinterpret_cast<const float*>(p), w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = __float_as_uint(w[i]);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};
template <>
struct Pack<__nv_bfloat16> {
  static DMX_DEVICE void store(__nv_bfloat16* p, const float* v) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    st_global8(reinterpret_cast<uint32_t*>(p), w);
  }
  static DMX_DEVICE void load(const __nv_bfloat16* p, float* v) {
    float w[8];
    ld_global8(reinterpret_cast<const float*>(p), w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = __float_as_uint(w[i]);
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};

template <int BN, typename OT, bool GELU>
__global__ void __launch_bounds__(kTileThreads, 1)
    linear_tile_kernel(const __grid_constant__ CUtensorMap tm_x,
                       const __grid_constant__ CUtensorMap tm_w, const LinearArgs a,
                       int64_t mtiles, int ntiles, int wide) {
  using S = TileSmem<BN>;
  constexpr int STAGES = S::STAGES;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float2* column = reinterpret_cast<float2*>(smem + STAGES * S::STAGE);  // [2][BN]
  float* turn = reinterpret_cast<float*>(smem + STAGES * S::STAGE + S::COLUMN);
  Pipe pipe;
  pipe.full = reinterpret_cast<uint64_t*>(smem + STAGES * S::STAGE + S::COLUMN + S::TURN);
  pipe.empty = pipe.full + STAGES;
  uint64_t* acc_full = pipe.empty + STAGES;  // [2]
  uint64_t* acc_empty = acc_full + 2;        // [2]
  uint64_t* drain = acc_empty + 2;
  uint32_t* slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&pipe.full[s], 1);
      mbar_init(&pipe.empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kEpiThreads);
    }
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(slot, S::COLS);
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  const uint32_t tmem = *slot;
  const int64_t total = mtiles * ntiles;
  const int blocks = (a.k + kBlockK - 1) / kBlockK;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int64_t t = blockIdx.x; t < total && ok; t += gridDim.x) {
        int64_t m0;
        int nt;
        tile_at(t, mtiles, ntiles, m0, nt);
        for (int kb = 0; kb < blocks; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&pipe.empty[s], ((it / STAGES) & 1) ^ 1, a.err, 21)) {
            ok = false;
            break;
          }
          unsigned char* dst = smem + s * S::STAGE;
          mbar_expect_tx(&pipe.full[s], S::STAGE);
          tma_load_2d(dst, &tm_x, &pipe.full[s], kb * kBlockK, (int)m0);
          tma_load_2d(dst + S::A, &tm_w, &pipe.full[s], kb * kBlockK, nt * BN);
        }
      }
      if (!ok) drain_loads<STAGES>(pipe, it, a.err);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t it = 0;
      int tl = 0;
      bool ok = true;
      for (int64_t t = blockIdx.x; t < total && ok; t += gridDim.x, ++tl) {
        const int acc = tl & 1;
        if (!mbar_wait(&acc_empty[acc], ((tl >> 1) & 1) ^ 1, a.err, 22)) {
          ok = false;
          break;
        }
        tc_after_sync();
        const uint32_t d = tmem + (uint32_t)(acc * BN);
        for (int kb = 0; kb < blocks; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&pipe.full[s], (it / STAGES) & 1, a.err, 23)) {
            ok = false;
            break;
          }
          tc_after_sync();
          const uint32_t addr = smem_u32(smem + s * S::STAGE);
          mma_stage<BN>(d, addr, addr + S::A, a.k - kb * kBlockK, kb == 0);
          umma_commit(&pipe.empty[s]);
        }
        if (ok) umma_commit(&acc_full[acc]);
      }
      if (!ok) drain_mmas(drain, a.err);
    }
  } else {
    // two warps per quarter of the accumulator's lanes (rows); half hh takes
    // the 32-column chunks 64 j + 32 hh
    const int e = threadIdx.x - 64, quarter = warp % 4, hh = (warp - 2) / 4;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    float* mine = turn + (warp - 2) * 32 * 17;
    bool ok = true;
    int tl = 0;
    for (int64_t t = blockIdx.x; t < total; t += gridDim.x, ++tl) {
      int64_t m0;
      int nt;
      tile_at(t, mtiles, ntiles, m0, nt);
      const int n0 = nt * BN, acc = tl & 1;
      float2* col = column + acc * BN;
      // this tile's channel scales and biases; the other buffer is still read
      for (int c = e; c < BN; c += kEpiThreads) {
        const int n = n0 + c;
        col[c] = make_float2(n < a.n && a.w_scale ? a.w_scale[n] : 1.f,
                             n < a.n && a.bias ? a.bias[n] : 0.f);
      }
      const int64_t m = m0 + quarter * 32 + lane;
      const float xs = m < a.rows && a.x_scale ? a.x_scale[m] : 1.f;
      asm volatile("bar.sync 1, %0;" ::"n"(kEpiThreads) : "memory");
      if (ok && !mbar_wait(&acc_full[acc], (tl >> 1) & 1, a.err, 24)) ok = false;
      // the lanes may end a wait that gave up apart
      ok = __all_sync(0xffffffffu, ok);
      tc_after_sync();
      if (ok) {
#pragma unroll 1
        for (int c0 = hh * 32; c0 < BN && n0 + c0 < a.n; c0 += 64) {
          uint32_t r[32];
          tmem_ld32_nw(tmem + lanes + (uint32_t)(acc * BN + c0), r);
          tmem_ld_wait<32>(r);
#pragma unroll
          for (int h = 0; h < 32; h += 16) {
            const int n = n0 + c0 + h;
            if (n >= a.n) break;
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float4 sb = *reinterpret_cast<const float4*>(col + c0 + h + i);
              v[i] = linear_value<OT, GELU>((int)r[h + i], xs, sb.x, sb.y);
              v[i + 1] = linear_value<OT, GELU>((int)r[h + i + 1], xs, sb.z, sb.w);
            }
            if (wide && n + 16 <= a.n) {
              if (m < a.rows) {
                if (a.residual) {
                  float q[16];
                  Pack<OT>::load(static_cast<const OT*>(a.residual) + m * a.residual_ld + n, q);
#pragma unroll
                  for (int i = 0; i < 16; ++i) v[i] += q[i];
                }
                Pack<OT>::store(static_cast<OT*>(a.out) + m * a.out_ld + n, v);
              }
            } else {
              // rows that do not start on 32 bytes: turned in shared memory, so
              // that a store covers neighbouring columns of two rows
#pragma unroll
              for (int i = 0; i < 16; ++i) mine[lane * 17 + i] = v[i];
              __syncwarp();
              const int c = lane & 15;
              for (int i = lane >> 4; i < 32; i += 2) {
                const int64_t row = m0 + quarter * 32 + i;
                if (row < a.rows && n + c < a.n) store_out<OT>(a, row, n + c, mine[i * 17 + c]);
              }
              __syncwarp();
            }
          }
        }
      }
      tc_before_sync();
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&acc_empty[acc]))
                   : "memory");
    }
  }
  tc_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_after_sync();
    tmem_free(tmem, S::COLS);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// int8 rows: a box of 128 bytes of k by `high` rows; reads past either end give zeros
bool row_map(CUtensorMap* map, const int8_t* p, int64_t rows, int k, int64_t ld, int high) {
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  const cuuint64_t str[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {kBlockK, (cuuint32_t)high};
  return make_tensor_map(map, p, 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B, nullptr,
                         CU_TENSOR_MAP_DATA_TYPE_UINT8);
}

template <int M, int C, typename OT, bool GELU>
void launch_gemv(const LinearArgs& a, cudaStream_t s) {
  // warps along k: enough blocks for two per SM, at least 1 KB of k per warp
  int kw = 1;
  while (kw < 8 && a.k >= kw * 2048 && (int64_t)a.n * kw < 2ll * 8 * C * sm_count()) kw *= 2;
  const int per = 8 / kw * C;
  linear_gemv_kernel<M, C, OT, GELU><<<(a.n + per - 1) / per, kGemvThreads, 0, s>>>(a, kw);
}

template <int BT, int STAGES, typename OT, bool GELU>
bool launch_few(const LinearArgs& a, cudaStream_t s) {
  CUtensorMap tw, tx;
  if (!row_map(&tw, a.w, a.n, a.k, a.w_ld, 128) || !row_map(&tx, a.x, a.rows, a.k, a.x_ld, BT))
    return false;
  using S = FewSmem<BT, STAGES>;
  auto kernel = linear_few_kernel<BT, STAGES, OT, GELU>;
  static PerDevice once;
  if (once.first()) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL);
  const int64_t tiles = (a.n + 127) / 128;
  const int mtiles = (int)((a.rows + BT - 1) / BT);
  const int blocks = (a.k + kBlockK - 1) / kBlockK;
  int splits = 1;
  while (splits < 8 && blocks >= splits * 4 && tiles * mtiles * splits * 2 <= 2 * sm_count()) splits *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * splits), (unsigned)mtiles);
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = S::TOTAL;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)splits, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, tw, tx, a, splits);
  return true;
}

template <int BN, typename OT, bool GELU>
bool launch_tile(const LinearArgs& a, cudaStream_t s) {
  CUtensorMap tw, tx;
  if (!row_map(&tx, a.x, a.rows, a.k, a.x_ld, 128) || !row_map(&tw, a.w, a.n, a.k, a.w_ld, BN))
    return false;
  using S = TileSmem<BN>;
  auto kernel = linear_tile_kernel<BN, OT, GELU>;
  static PerDevice once;
  if (once.first()) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL);
  const int64_t mtiles = (a.rows + 127) / 128;
  const int ntiles = (a.n + BN - 1) / BN;
  const size_t pitch = sizeof(OT);
  const bool wide = reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.out_ld * pitch % 32 == 0 &&
                    (!a.residual || (reinterpret_cast<uintptr_t>(a.residual) % 32 == 0 &&
                                     a.residual_ld * pitch % 32 == 0));
  const unsigned grid = (unsigned)std::min<int64_t>(mtiles * ntiles, sm_count());
  kernel<<<grid, kTileThreads, S::TOTAL, s>>>(tx, tw, a, mtiles, ntiles, wide ? 1 : 0);
  return true;
}

template <typename OT, bool GELU>
bool launch_typed(const LinearArgs& a, cudaStream_t s) {
  if (a.rows <= 8) {
    if (a.rows == 1) launch_gemv<1, 4, OT, GELU>(a, s);
    else if (a.rows == 2) launch_gemv<2, 4, OT, GELU>(a, s);
    else if (a.rows <= 4) launch_gemv<4, 4, OT, GELU>(a, s);
    else launch_gemv<8, 2, OT, GELU>(a, s);
    return true;
  }
  if (a.rows <= 128) {
    if (a.rows <= 16) return launch_few<16, 5, OT, GELU>(a, s);
    if (a.rows <= 32) return launch_few<32, 5, OT, GELU>(a, s);
    if (a.rows <= 64) return launch_few<64, 4, OT, GELU>(a, s);
    return launch_few<128, 3, OT, GELU>(a, s);
  }
  // the widest tile that still gives every SM one
  const int64_t mtiles = (a.rows + 127) / 128;
  if (mtiles * ((a.n + 255) / 256) >= sm_count()) return launch_tile<256, OT, GELU>(a, s);
  if (mtiles * ((a.n + 127) / 128) >= sm_count()) return launch_tile<128, OT, GELU>(a, s);
  return launch_tile<64, OT, GELU>(a, s);
}

}  // namespace

bool launch_quantized_linear(const LinearArgs& a, cudaStream_t s) {
  switch (a.out_type * 2 + (a.gelu ? 1 : 0)) {
    case 0: return launch_typed<float, false>(a, s);
    case 1: return launch_typed<float, true>(a, s);
    case 2: return launch_typed<__half, false>(a, s);
    case 3: return launch_typed<__half, true>(a, s);
    case 4: return launch_typed<__nv_bfloat16, false>(a, s);
    default: return launch_typed<__nv_bfloat16, true>(a, s);
  }
}

}  // namespace dmx
