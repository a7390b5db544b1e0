// The 8-bit linear layer (dmx_quantized_linear):
//
//   out[m][n] = act(acc[m][n] x_scale[m] w_scale[n] + bias[n]) + residual[m][n]
//   acc[m][n] = sum_k x[m][k] w[n][k], exact in 32-bit integers
//
// Three kernels, all on the same operands (rows on 16-byte boundaries, the
// bytes past column k of a row never used):
//  * linear_gemv_kernel: up to 8 rows and not too many weights, dp4a on weights
//    streamed once;
//  * linear_few_kernel: up to 128 rows and long k, tcgen05 with the weights as
//    the 128-row operand, k split over a thread-block cluster;
//  * linear_tile_kernel: the rest, persistent tcgen05 tiles.
// The first two are bound by the weights' bytes (1 x 8192 -> 8192: 14.3 us, 4.7
// TB/s), the last by the tensor core where k is long (8192^3: 356 us, 3.09
// POP/s) and by its epilogue or HBM where it is short (112896 x 512 -> 2048 to
// bf16: 150 us; with GELU 212).
#include <algorithm>

#include "ops.h"
#include "ops_common.cuh"
#include "row_tail.h"
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
// The same by a pair of CTAs: rows 0..127 of D and A in the first's memory,
// 128..255 in the second's, B's rows in halves likewise.
DMX_DEVICE void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
// s32 accumulator, s8 operands, both K-major, m x n
constexpr uint32_t i8_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// max that keeps a NaN
DMX_DEVICE float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// GELU of 2 P values: z (1 + erf(z / sqrt 2)) / 2 = max(z, 0) + n E(n) with
// n = -|z| and E(n) = erfc(-n / sqrt 2) / 2 = exp(-n^2 / 2) R(n). R is smooth (a
// scaled complementary error function). This polynomial of degree 10 was found
// by linear programming on 1200 Chebyshev points of [-4, 0]: the least largest
// error of exp(-n^2 / 2) R(n), in units of 1 or, where that is less, of 10^5 E,
// with R(0) = 1/2 and the coefficients rounded to f32 one after the other from
// the highest, the rest fitted anew each time. So rounded, it is off by at most
// 5.1e-8 there, and by 1.5e-3 of E. Below -4 n stays while the exponential goes
// on with z: n R(n) is within 4.7 % of its limit -1 / sqrt(2 pi) already, so the
// tail keeps that relative error down to where f32 ends, and nothing overflows.
// Measured over [-14, 14]: at most 1.4e-7 |z| off, and 2.3 % of the value at
// -5.5 (the form by erff: 1.1e-7 |z|, and 57 %). -infinity gives 0, a NaN stays
// one. One special-function operation and paired FMAs a value; each step for
// all the pairs before the next, so that a coefficient is set up once.
template <int P>
DMX_DEVICE void gelu_pairs(float2* z) {
  constexpr float kR[11] = {0.5f,           0.39893952f,    0.249949172f,    0.132658452f,
                            0.061487034f,   0.0247497074f,  0.00828321464f,  0.00213995879f,
                            0.000386984466f, 4.25554099e-05f, 2.10910139e-06f};
  float2 n[P], r[P], e[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    n[i] = make_float2(max_nan(-fabsf(z[i].x), -4.f), max_nan(-fabsf(z[i].y), -4.f));
    r[i] = make_float2(kR[10], kR[10]);
  }
#pragma unroll
  for (int k = 9; k >= 0; --k)
#pragma unroll
    for (int i = 0; i < P; ++i) r[i] = __ffma2_rn(r[i], n[i], make_float2(kR[k], kR[k]));
  // exp(-z^2 / 2) = 2^(-z^2 log2(e) / 2)
#pragma unroll
  for (int i = 0; i < P; ++i)
    e[i] = __fmul2_rn(__fmul2_rn(z[i], z[i]), make_float2(-0.72134752f, -0.72134752f));
#pragma unroll
  for (int i = 0; i < P; ++i) {
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e[i].x) : "f"(e[i].x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e[i].y) : "f"(e[i].y));
  }
#pragma unroll
  for (int i = 0; i < P; ++i)
    z[i] = __ffma2_rn(n[i], __fmul2_rn(r[i], e[i]),
                      make_float2(fmaxf(z[i].x, 0.f), fmaxf(z[i].y, 0.f)));
}

// Outputs of one row from their exact sums: scales in the order row, channel,
// then the bias in the same rounding as the last product.
DMX_DEVICE float2 scaled2(int acc0, int acc1, float xs, float2 ws, float2 b) {
  return __ffma2_rn(__fmul2_rn(make_float2((float)acc0, (float)acc1), make_float2(xs, xs)), ws, b);
}
template <bool GELU>
DMX_DEVICE float linear_value(int acc, float xs, float ws, float b) {
  float2 v = scaled2(acc, acc, xs, make_float2(ws, ws), make_float2(b, b));
  if (GELU) gelu_pairs<1>(&v);
  return v.x;
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

// 16 bytes of a row (not by the read-only path: what a kernel before writes is
// written while this one, begun early, already runs).
DMX_DEVICE int4 row16(const int8_t* p) { return *reinterpret_cast<const int4*>(p); }
// The last `left` (1..15) bytes of a row and zeros.
DMX_DEVICE int4 row_end16(const int8_t* p, int left) {
  uint32_t w[4];
  read_tail16(p, left, w);
  return make_int4((int)w[0], (int)w[1], (int)w[2], (int)w[3]);
}
DMX_DEVICE int dot16(int4 x, int4 w, int acc) {
  acc = __dp4a(x.x, w.x, acc);
  acc = __dp4a(x.y, w.y, acc);
  acc = __dp4a(x.z, w.z, acc);
  return __dp4a(x.w, w.w, acc);
}

DMX_DEVICE void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

constexpr int kGemvThreads = 256;

// A warp takes C channels and every `kw`-th 512-byte piece of k; the `kw`
// warps of one channel group (8 / kw groups per block) are summed through
// shared memory. x (at most 8 rows) stays in L1. Held to registers with which
// four (three) blocks share an SM: 2 x 2048 -> 8192, whose 512 blocks then run
// at once, takes 3.6 us, by three of them at a time 5.0.
template <int M, int C, typename OT, bool GELU>
__global__ void __launch_bounds__(kGemvThreads, M <= 2 ? 4 : 3)
    linear_gemv_kernel(const __grid_constant__ LinearArgs a, int kw) {
  __shared__ int part[kGemvThreads / 32][M * C];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int groups = (kGemvThreads / 32) / kw, group = warp / kw, kpart = warp % kw;
  const int n0 = (blockIdx.x * groups + group) * C;
  let_next_kernel_begin();
  // the first weights start towards L2 while the tokens are still being made
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int k0 = (kpart * 32 + lane) * 128;
    if (n0 + c < a.n && k0 < a.k) prefetch_l2(a.w + (int64_t)(n0 + c) * a.w_ld + k0);
  }
  after_earlier_kernels();
  int acc[M][C];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int c = 0; c < C; ++c) acc[m][c] = 0;
  if (n0 < a.n) {
    auto w_row = [&](int c) { return a.w + (int64_t)min(n0 + c, a.n - 1) * a.w_ld; };
    auto x_row = [&](int m) { return a.x + min((int64_t)m, a.rows - 1) * a.x_ld; };
    int4 w[C], x[M];
    auto dots = [&] {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[m][c] = dot16(x[m], w[c], acc[m][c]);
    };
    int k0 = kpart * 512 + lane * 16;
#pragma unroll 2
    for (; k0 + 16 <= a.k; k0 += kw * 512) {
#pragma unroll
      for (int c = 0; c < C; ++c) w[c] = row16(w_row(c) + k0);
#pragma unroll
      for (int m = 0; m < M; ++m) x[m] = row16(x_row(m) + k0);
      dots();
    }
    if (k0 < a.k) {  // the lane whose bytes the row's end cuts
#pragma unroll
      for (int c = 0; c < C; ++c) w[c] = row_end16(w_row(c) + k0, a.k - k0);
#pragma unroll
      for (int m = 0; m < M; ++m) x[m] = row_end16(x_row(m) + k0, a.k - k0);
      dots();
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
                  linear_value<GELU>(t, a.x_scale ? a.x_scale[m] : 1.f,
                                         a.w_scale ? a.w_scale[n] : 1.f, a.bias ? a.bias[n] : 0.f));
  }
}

// ---------------------------------------------------------------------------
// tcgen05: what both kernels share
// ---------------------------------------------------------------------------

struct Pipe {
  uint64_t *full, *empty;
};

// What a kernel's warps leave for its end: whether a wait gave up, and how many
// stages each CTA began to load (a pair's: at the first, where they count).
struct Ending {
  uint32_t gave_up, issued[2];
};
// A barrier of both CTAs of a pair gets an arrival once the pair's MMAs so far are done.
DMX_DEVICE void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
template <bool PAIR>
DMX_DEVICE void commit(uint64_t* bar) {
  if (PAIR) umma_commit_pair(bar);
  else umma_commit(bar);
}
// Shared memory of CTA `rank` of the cluster at this CTA's address p.
DMX_DEVICE uint32_t of_rank(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
DMX_DEVICE void st_cluster(uint32_t at, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
DMX_DEVICE int4 ld_cluster(uint32_t at) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(at)
               : "memory");
  return v;
}
// Relaxed: what it announces, reads of tensor memory, is ordered by the
// tcgen05 fence before it; a release would wait for the thread's stores to
// global memory (112896x128->2048: 173 us against 131).
DMX_DEVICE void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A tile into this CTA's memory, its bytes counted at the first CTA's barrier.
DMX_DEVICE void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}

template <bool PAIR>
DMX_DEVICE void tmem_alloc(uint32_t* slot, uint32_t cols) {
  if (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(slot)),
                 "r"(cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(slot)),
                 "r"(cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
}
template <bool PAIR>
DMX_DEVICE void tmem_free(uint32_t tmem, uint32_t cols) {
  if (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols));
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols));
}
DMX_DEVICE bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}
// A bounded wait of a whole warp, whose lanes may end one that gives up apart.
DMX_DEVICE bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code));
}
// The same, a wait that gives up noted at every CTA that shares its loads and MMAs.
template <bool PAIR>
DMX_DEVICE bool noted_wait(uint64_t* bar, uint32_t parity, int* err, int code, Ending* end) {
  if (warp_wait(bar, parity, err, code)) return true;
  if (PAIR) {
    st_cluster(of_rank(&end->gave_up, 0), 1);
    st_cluster(of_rank(&end->gave_up, 1), 1);
  } else {
    *reinterpret_cast<volatile uint32_t*>(&end->gave_up) = 1;
  }
  return false;
}
// After a wait gave up, between two barriers of the CTAs that share its loads
// and MMAs: what was begun is waited for, so that nothing writes shared memory,
// or reads it or tensor memory, once they are another kernel's. These waits are
// bounded too, but look past the raised flag, which is no reason to leave now.
// For the CTA that issues the MMAs, whose elected lane of warp 1 did.
template <int STAGES, bool PAIR>
DMX_DEVICE void settle(const Pipe& pipe, const Ending& end, uint64_t* drain, uint32_t stage_bytes,
                       bool elected) {
  if (threadIdx.x < 32) {
    const uint32_t mine = end.issued[0], other = PAIR ? end.issued[1] : mine, last = max(mine, other);
    for (uint32_t it = last > STAGES ? last - STAGES : 0; it < last; ++it) {
      uint64_t* bar = &pipe.full[it % STAGES];
      if (elected) {
        if (it >= mine) mbar_expect_tx(bar, stage_bytes);  // only the other CTA's bytes come
        if (it >= other)                                   // its bytes never come
          asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                       "r"(stage_bytes)
                       : "memory");
      }
      __syncwarp();
      mbar_wait(bar, (it / STAGES) & 1, nullptr, 0);
    }
  } else if (threadIdx.x < 64 && elected) {
    commit<PAIR>(drain);
    mbar_wait(drain, 0, nullptr, 0);
  }
}
DMX_DEVICE void tc_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
DMX_DEVICE void tc_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

DMX_DEVICE void tma_prefetch_2d(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(c0),
               "r"(c1)
               : "memory");
}
// Every thread of the cluster: shared-memory writes before it are seen after it.
DMX_DEVICE void cluster_sync() {
  asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}

// The MMAs of one landed stage: `left` bytes of k, 32 per instruction (the
// rest of a last stage was filled with zeros).
template <int N, bool PAIR>
DMX_DEVICE void mma_stage(uint32_t d, uint32_t a_addr, uint32_t b_addr, int left, bool first) {
#pragma unroll
  for (int j = 0; j < kBlockK / 32; ++j)
    if (j * 32 < left) {
      const uint64_t ad = umma_desc_k(a_addr + j * 32, 128), bd = umma_desc_k(b_addr + j * 32, 128);
      if (PAIR) umma_i8_pair(d, ad, bd, i8_idesc(256, N), !(first && j == 0));
      else umma_i8(d, ad, bd, i8_idesc(128, N), !(first && j == 0));
    }
}

// ---------------------------------------------------------------------------
// up to 128 rows: out^T tile of 128 channels x BT rows per cluster
// ---------------------------------------------------------------------------

constexpr int kFewThreads = 512;  // warp 0 TMA, warp 1 MMA, warps 2-5 read the accumulator; all finish

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
                      const __grid_constant__ CUtensorMap tm_x,
                      const __grid_constant__ LinearArgs a, int splits, int wide) {
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
  Ending* end = reinterpret_cast<Ending*>(slot + 1);

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
    *end = {};
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc<false>(slot, S::COLS);
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  const uint32_t tmem = *slot;

  const bool elected = elect_one();
  const uint32_t count = (uint32_t)(hi - lo);
  let_next_kernel_begin();
  if (warp == 0 && elected)
    for (int kb = lo; kb < min(hi, lo + STAGES); ++kb) tma_prefetch_2d(&tm_w, kb * kBlockK, n0);
  after_earlier_kernels();
  if (warp == 0) {
    uint32_t it = 0;
    for (int kb = lo; kb < hi; ++kb, ++it) {
      const uint32_t s = it % STAGES;
      if (!noted_wait<false>(&pipe.empty[s], ((it / STAGES) & 1) ^ 1, a.err, 11, end)) break;
      if (elected) {
        unsigned char* dst = smem + s * S::STAGE;
        mbar_expect_tx(&pipe.full[s], S::STAGE);
        tma_load_2d(dst, &tm_w, &pipe.full[s], kb * kBlockK, n0);
        tma_load_2d(dst + S::A, &tm_x, &pipe.full[s], kb * kBlockK, m0);
      }
    }
    if (elected) end->issued[0] = it;
  } else if (warp == 1) {
    uint32_t it = 0;
    for (int kb = lo; kb < hi; ++kb, ++it) {
      const uint32_t s = it % STAGES;
      if (!noted_wait<false>(&pipe.full[s], (it / STAGES) & 1, a.err, 12, end)) break;
      tc_after_sync();
      if (elected) {
        const uint32_t addr = smem_u32(smem + s * S::STAGE);
        mma_stage<BT, false>(tmem, addr, addr + S::A, a.k - kb * kBlockK, kb == lo);
        umma_commit(&pipe.empty[s]);
      }
    }
    if (elected && it == count) umma_commit(done);
  }
  __syncwarp();
  int* part = reinterpret_cast<int*>(smem);  // [BT][128]
  if (warp >= 2 && warp < 6) {
    // lane = channel, column = row of x: [row][channel] is written without bank conflicts
    const int q = warp % 4;
    const bool ok = noted_wait<false>(done, 0, a.err, 13, end);
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
  if (end->gave_up) settle<STAGES, false>(pipe, *end, drain, S::STAGE, elected);
  // each CTA of the cluster finishes its share of the rows, a warp a row and a
  // lane four channels of it
  const int rows = (int)min((int64_t)BT, a.rows - m0), n = n0 + 4 * lane;
  if (n < a.n) {
    float ws[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ws[i] = n + i < a.n && a.w_scale ? a.w_scale[n + i] : 1.f;
      b[i] = n + i < a.n && a.bias ? a.bias[n + i] : 0.f;
    }
    for (int m = split + warp * splits; m < rows; m += kFewThreads / 32 * splits) {
      const int4* at = reinterpret_cast<const int4*>(part + m * 128) + lane;
      int4 acc = splits > 1 ? make_int4(0, 0, 0, 0) : *at;
      if (splits > 1) {
        int4 v[8];
#pragma unroll
        for (int p = 0; p < 8; ++p)
          if (p < splits) v[p] = ld_cluster(of_rank(at, p));
#pragma unroll
        for (int p = 0; p < 8; ++p)
          if (p < splits)
            acc = make_int4(acc.x + v[p].x, acc.y + v[p].y, acc.z + v[p].z, acc.w + v[p].w);
      }
      const int64_t row = m0 + m;
      const float xs = a.x_scale ? a.x_scale[row] : 1.f;
      float2 y[2] = {scaled2(acc.x, acc.y, xs, make_float2(ws[0], ws[1]), make_float2(b[0], b[1])),
                     scaled2(acc.z, acc.w, xs, make_float2(ws[2], ws[3]), make_float2(b[2], b[3]))};
      if (GELU) gelu_pairs<2>(y);
      if (wide && n + 4 <= a.n) {
        float4 f = make_float4(y[0].x, y[0].y, y[1].x, y[1].y);
        if (a.residual) {
          const float4 r = load4(static_cast<const OT*>(a.residual) + row * a.residual_ld + n);
          f = make_float4(f.x + r.x, f.y + r.y, f.z + r.z, f.w + r.w);
        }
        store4(static_cast<OT*>(a.out) + row * a.out_ld + n, f);
      } else {
        const float f[4] = {y[0].x, y[0].y, y[1].x, y[1].y};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < a.n) store_out<OT>(a, row, n + i, f[i]);
      }
    }
  }
  // a peer may still be reading this CTA's partial sums
  if (splits > 1) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_after_sync();
    tmem_free<false>(tmem, S::COLS);
  }
}

// ---------------------------------------------------------------------------
// more rows: persistent 128 x BN tiles
// ---------------------------------------------------------------------------

constexpr int kGroupRows = 8;  // row tiles per group of the tile order

// Warp 0 issues TMA, warp 1 the MMAs, the other 16 are the epilogue: four, one
// per quarter of the accumulator's lanes, for each quarter of the columns. Tiles of 256
// columns are worked on by a pair of CTAs, 128 rows each, which halves what
// each of them loads of w: with a CTA alone, its shared memory took in 48 KB
// and gave out as much for every 512 cycles of the tensor core, more than L2
// delivers (8192^3: 421 us).
template <int BN>
struct Tile {
  static constexpr bool PAIR = BN == 256;
  static constexpr int ROWS = PAIR ? 256 : 128;
  static constexpr int EPI_WARPS = 16, THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int WIDTH = BN / 4;  // an epilogue warp's columns
  static constexpr int A = 128 * kBlockK, B = BN * kBlockK / (PAIR ? 2 : 1), STAGE = A + B;
  static constexpr int TURN = EPI_WARPS * 4096;       // epilogue warps' outputs on their way
  static constexpr int COLUMN = EPI_WARPS * WIDTH * 8;  // their channel scales and biases
  static constexpr int STAGES = (227 * 1024 - TURN - COLUMN - 1024 - 256) / STAGE;
  static constexpr int TOTAL = STAGES * STAGE + TURN + COLUMN + 1024 + 256;
  static constexpr uint32_t COLS = 2 * BN;
};

// Tile t of the order: groups of kGroupRows row tiles, row tile fastest, so
// the CTAs at work together share both operands' tiles in L2.
struct TileOrder {
  uint32_t mtiles, ntiles, total;
  DMX_DEVICE void at(uint32_t t, uint32_t& m_tile, uint32_t& n_tile) const {
    const uint32_t per = kGroupRows * ntiles, g = t / per, in_group = t - g * per;
    const uint32_t high = min((uint32_t)kGroupRows, mtiles - g * kGroupRows);
    n_tile = in_group / high;
    m_tile = g * kGroupRows + in_group % high;
  }
};

// One epilogue warp's 32 rows of a tile, a lane holding a row, to memory by
// whole lines: through 4 KB of shared memory in which the 16-byte units of row
// r are permuted by r % 8, so that neither the rows' writes nor the lines'
// reads meet in a bank. (Stores of 32 bytes to each of 32 rows ran at 2.1 TB/s
// for 16-bit outputs, 2.9 for f32 ones.)
template <typename OT>
struct Lines {
  unsigned char* buf;  // 32 rows of 128 bytes
  int lane;
  DMX_DEVICE void* unit(int row, int u) const { return buf + row * 128 + ((u ^ (row & 7)) << 4); }
  // 8 / 4 values of this lane's row as unit u
  DMX_DEVICE void put_packed(int u, const float2* v) const {
    *reinterpret_cast<uint4*>(unit(lane, u)) =
        make_uint4(pack2(v[0].x, v[0].y, OT()), pack2(v[1].x, v[1].y, OT()),
                   pack2(v[2].x, v[2].y, OT()), pack2(v[3].x, v[3].y, OT()));
  }
  DMX_DEVICE void put_f32(int u, const float2* v) const {
    *reinterpret_cast<float4*>(unit(lane, u)) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
  }
};

// 16 columns of a row of the accumulator, scaled (col: two columns' scales and
// biases to 16 bytes) and activated.
template <bool GELU>
DMX_DEVICE void tile_values(uint32_t tmem_at, const float4* col, float row_scale, float2* v) {
  uint32_t r[16];
  tmem_ld16_nw(tmem_at, r);
  tmem_ld_wait<16>(r);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 q = col[i];
    v[i] = scaled2((int)r[2 * i], (int)r[2 * i + 1], row_scale, make_float2(q.x, q.y),
                   make_float2(q.z, q.w));
  }
  if (GELU) {
    // in halves, for fewer registers at once (112896x512->2048, with a polynomial
    // of degree 11: 224 us against 230)
    gelu_pairs<4>(v);
    gelu_pairs<4>(v + 4);
  }
}

// An epilogue warp's share of a tile: `rows` of its 32 rows exist, from row m0
// and column n0 of the output on.
template <int WIDTH, typename OT, bool GELU>
DMX_DEVICE void tile_share(const LinearArgs& a, const Lines<OT>& lines, uint32_t tmem_at, const float4* col,
                           float row_scale, int64_t m0, int n0, int rows, bool wide) {
  const int lane = lines.lane;
  OT* out = static_cast<OT*>(a.out) + m0 * a.out_ld + n0;
  // unrolled, the GELU's coefficients are set up once; without a GELU the loads of
  // several turns at once only spilled registers (112896x512->2048: 220 us against 150)
  constexpr int kUnroll = GELU ? 4 : 1;
  if constexpr (sizeof(OT) == 2) {
    if (!a.residual) {  // rounded before they cross: all columns in one pass
#pragma unroll kUnroll
      for (int c = 0; c < WIDTH; c += 16) {
        float2 v[8];
        tile_values<GELU>(tmem_at + c, col + c / 2, row_scale, v);
        lines.put_packed(c / 8, v);
        lines.put_packed(c / 8 + 1, v + 4);
      }
      __syncwarp();
      if (wide && n0 + WIDTH <= a.n) {
        constexpr int kUnits = WIDTH / 8;
        OT* at = out + (lane / kUnits) * a.out_ld + (lane % kUnits) * 8;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          const int row = 32 / kUnits * i + lane / kUnits;
          const uint4 w = *reinterpret_cast<const uint4*>(lines.unit(row, lane % kUnits));
          if (row < rows) st_words4(at, reinterpret_cast<const uint32_t*>(&w));
          at += 32 / kUnits * a.out_ld;
        }
      } else {  // rows that do not start on 16 bytes, or end here: by elements
        const int cols = min(WIDTH, a.n - n0);
        for (int row = 0; row < rows; ++row)
          for (int c = lane; c < cols; c += 32)
            out[row * a.out_ld + c] = static_cast<const OT*>(lines.unit(row, c / 8))[c % 8];
      }
      __syncwarp();
      return;
    }
  }
  // as f32, 32 columns to a pass; a residual is added after the crossing
  constexpr int kPass = WIDTH < 32 ? WIDTH : 32, kUnits = kPass / 4;
#pragma unroll 1
  for (int p = 0; p < WIDTH && n0 + p < a.n; p += kPass) {
    const bool whole = wide && n0 + p + kPass <= a.n;
    const OT* residual = static_cast<const OT*>(a.residual) + m0 * a.residual_ld + n0 + p;
    float4 q[kUnits];
    if (whole && a.residual) {  // on its way while the accumulator is read
      const OT* at = residual + (lane / kUnits) * a.residual_ld + (lane % kUnits) * 4;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        if (32 / kUnits * i + lane / kUnits < rows) q[i] = load4(at);
        at += 32 / kUnits * a.residual_ld;
      }
    }
#pragma unroll kUnroll
    for (int c = 0; c < kPass; c += 16) {
      float2 v[8];
      tile_values<GELU>(tmem_at + p + c, col + (p + c) / 2, row_scale, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) lines.put_f32(c / 4 + i, v + 2 * i);
    }
    __syncwarp();
    if (whole) {
      OT* at = out + p + (lane / kUnits) * a.out_ld + (lane % kUnits) * 4;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int row = 32 / kUnits * i + lane / kUnits;
        float4 f = *reinterpret_cast<const float4*>(lines.unit(row, lane % kUnits));
        if (row < rows) {
          if (a.residual) f = make_float4(f.x + q[i].x, f.y + q[i].y, f.z + q[i].z, f.w + q[i].w);
          store4(at, f);
        }
        at += 32 / kUnits * a.out_ld;
      }
    } else {
      const int cols = min(kPass, a.n - n0 - p);
      for (int row = 0; row < rows; ++row)
        for (int c = lane; c < cols; c += 32) {
          float f = static_cast<const float*>(lines.unit(row, c / 4))[c % 4];
          if (a.residual) f += to_f32(residual[row * a.residual_ld + c]);
          out[row * a.out_ld + p + c] = from_f32<OT>(f);
        }
    }
    __syncwarp();
  }
}

template <int BN, typename OT, bool GELU>
__global__ void __launch_bounds__(Tile<BN>::THREADS, 1)
    linear_tile_kernel(const __grid_constant__ CUtensorMap tm_x,
                       const __grid_constant__ CUtensorMap tm_w,
                       const __grid_constant__ LinearArgs a,
                       const __grid_constant__ TileOrder order, int wide) {
  using S = Tile<BN>;
  constexpr int STAGES = S::STAGES;
  constexpr bool PAIR = S::PAIR;
  constexpr int kCtas = PAIR ? 2 : 1;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* turn = smem + STAGES * S::STAGE;
  float4* column = reinterpret_cast<float4*>(turn + S::TURN);
  Pipe pipe;
  pipe.full = reinterpret_cast<uint64_t*>(turn + S::TURN + S::COLUMN);
  pipe.empty = pipe.full + STAGES;
  uint64_t* acc_full = pipe.empty + STAGES;  // [2]
  uint64_t* acc_empty = acc_full + 2;        // [2]
  uint64_t* drain = acc_empty + 2;
  uint32_t* slot = reinterpret_cast<uint32_t*>(drain + 1);
  Ending* end = reinterpret_cast<Ending*>(slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = PAIR ? blockIdx.x % 2 : 0;  // in the pair; the first issues its MMAs
  const uint32_t begin = blockIdx.x / kCtas, step = gridDim.x / kCtas;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&pipe.full[s], 1);
      mbar_init(&pipe.empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kCtas * S::EPI_WARPS);
    }
    mbar_init(drain, 1);
    *end = {};
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc<PAIR>(slot, S::COLS);
  tc_before_sync();
  if (PAIR) cluster_sync();
  else __syncthreads();
  tc_after_sync();
  const uint32_t tmem = *slot;
  const int blocks = (a.k + kBlockK - 1) / kBlockK;

  // Both warps walk their loops whole, one elected lane issuing: the
  // descriptors then live in uniform registers, which is where the tensor core
  // and the copy engine take them from.
  const bool elected = elect_one();
  let_next_kernel_begin();
  after_earlier_kernels();
  if (warp == 0) {
    uint32_t it = 0;
    bool ok = true;
    for (uint32_t t = begin; t < order.total && ok; t += step) {
      uint32_t mt, nt;
      order.at(t, mt, nt);
      const int m0 = (int)(mt * S::ROWS + rank * 128), n0 = (int)(nt * BN + rank * 128);
      for (int kb = 0; kb < blocks; ++kb, ++it) {
        const uint32_t s = it % STAGES;
        ok = noted_wait<PAIR>(&pipe.empty[s], ((it / STAGES) & 1) ^ 1, a.err, 21, end);
        if (!ok) break;
        if (elected) {
          unsigned char* dst = smem + s * S::STAGE;
          // a pair's loads count at the first CTA's barrier, where its MMAs wait
          if (rank == 0) mbar_expect_tx(&pipe.full[s], kCtas * S::STAGE);
          if (PAIR) {
            const uint32_t bar = of_rank(&pipe.full[s], 0);
            tma_load_pair(dst, &tm_x, bar, kb * kBlockK, m0);
            tma_load_pair(dst + S::A, &tm_w, bar, kb * kBlockK, n0);
          } else {
            tma_load_2d(dst, &tm_x, &pipe.full[s], kb * kBlockK, m0);
            tma_load_2d(dst + S::A, &tm_w, &pipe.full[s], kb * kBlockK, n0);
          }
        }
      }
    }
    if (elected) {
      if (PAIR) st_cluster(of_rank(&end->issued[rank], 0), it);
      else end->issued[0] = it;
    }
  } else if (warp == 1) {
    uint32_t it = 0;
    int tl = 0;
    bool ok = true;
    for (uint32_t t = begin; t < order.total && ok && rank == 0; t += step, ++tl) {
      const int acc = tl & 1;
      ok = noted_wait<PAIR>(&acc_empty[acc], ((tl >> 1) & 1) ^ 1, a.err, 22, end);
      if (!ok) break;
      tc_after_sync();
      const uint32_t d = tmem + (uint32_t)(acc * BN);
      for (int kb = 0; kb < blocks; ++kb, ++it) {
        const uint32_t s = it % STAGES;
        ok = noted_wait<PAIR>(&pipe.full[s], (it / STAGES) & 1, a.err, 23, end);
        if (!ok) break;
        tc_after_sync();
        if (elected) {
          const uint32_t addr = smem_u32(smem + s * S::STAGE);
          mma_stage<BN, PAIR>(d, addr, addr + S::A, a.k - kb * kBlockK, kb == 0);
          commit<PAIR>(&pipe.empty[s]);
        }
      }
      if (ok && elected) commit<PAIR>(&acc_full[acc]);
    }
  } else {
    // this warp: rows 32 quarter + lane, columns c_lo .. c_lo + WIDTH - 1 of each tile
    constexpr int WIDTH = S::WIDTH;
    const int quarter = warp % 4, c_lo = (warp - 2) / 4 * WIDTH;
    const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + c_lo;
    const Lines<OT> lines = {turn + (warp - 2) * 4096, lane};
    // its channel scales and biases, two columns to 16 bytes. A tile's are
    // fetched while the tile before it is worked on, each warp its own: no
    // barrier among the epilogue's warps, which so drift apart and share the
    // issue slots with one another's waits.
    float4* col = column + (warp - 2) * (WIDTH / 2);
    float4 sb;
    float xs;
    int64_t m0_next;
    int n0_next;
    auto fetch = [&](uint32_t t) {
      uint32_t mt, nt;
      order.at(t, mt, nt);
      m0_next = (int64_t)mt * S::ROWS + rank * 128 + quarter * 32;
      n0_next = (int)(nt * BN) + c_lo;
      const int n = n0_next + 2 * lane;
      sb = make_float4(1.f, 1.f, 0.f, 0.f);
      if (2 * lane < WIDTH) {
        if (a.w_scale) {
          if (n < a.n) sb.x = a.w_scale[n];
          if (n + 1 < a.n) sb.y = a.w_scale[n + 1];
        }
        if (a.bias) {
          if (n < a.n) sb.z = a.bias[n];
          if (n + 1 < a.n) sb.w = a.bias[n + 1];
        }
      }
      const int64_t m = m0_next + lane;
      xs = m < a.rows && a.x_scale ? a.x_scale[m] : 1.f;
      if (a.residual && m < a.rows) {  // towards L2: this row's share of the residual
        const OT* at = static_cast<const OT*>(a.residual) + m * a.residual_ld + n0_next;
        for (int c = 0; c < WIDTH && n0_next + c < a.n; c += 128 / (int)sizeof(OT)) prefetch_l2(at + c);
      }
    };
    bool ok = true;
    int tl = 0;
    if (begin < order.total) fetch(begin);
    for (uint32_t t = begin; t < order.total; t += step, ++tl) {
      const int64_t m0 = m0_next;
      const int n0 = n0_next, acc = tl & 1;
      const float row_scale = xs;
      __syncwarp();
      if (2 * lane < WIDTH) col[lane] = sb;
      __syncwarp();
      if (t + step < order.total) fetch(t + step);
      ok = ok && noted_wait<PAIR>(&acc_full[acc], (tl >> 1) & 1, a.err, 24, end);
      tc_after_sync();
      if (ok && n0 < a.n)
        tile_share<WIDTH, OT, GELU>(a, lines, from + (uint32_t)(acc * BN), col, row_scale, m0, n0,
                                    (int)min((int64_t)32, a.rows - m0), wide);
      tc_before_sync();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) arrive_at(of_rank(&acc_empty[acc], 0));
        else
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&acc_empty[acc]))
                       : "memory");
      }
    }
  }
  tc_before_sync();
  // a pair's MMAs read both CTAs' memory, and its barriers are the first's
  if (PAIR) cluster_sync();
  else __syncthreads();
  if (end->gave_up) {
    if (rank == 0) settle<STAGES, PAIR>(pipe, *end, drain, S::STAGE, elected);
    if (PAIR) cluster_sync();
    else __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    tc_after_sync();
    tmem_free<PAIR>(tmem, S::COLS);
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
  launch_chained(linear_gemv_kernel<M, C, OT, GELU>, (a.n + per - 1) / per, kGemvThreads, 0, s, true, 1, a, kw);
}

// Whether the rows of out and residual start on 16 bytes.
template <typename OT>
int wide_rows(const LinearArgs& a) {
  const int bytes = sizeof(OT);
  return vec_of(a.out, a.out_ld, bytes) != VEC_NONE &&
         (!a.residual || vec_of(a.residual, a.residual_ld, bytes) != VEC_NONE);
}

template <int BT, int STAGES, typename OT, bool GELU>
bool launch_few(const LinearArgs& a, cudaStream_t s) {
  CUtensorMap tw, tx;
  if (!row_map(&tw, a.w, a.n, a.k, a.w_ld, 128) || !row_map(&tx, a.x, a.rows, a.k, a.x_ld, BT))
    return false;
  using S = FewSmem<BT, STAGES>;
  auto kernel = linear_few_kernel<BT, STAGES, OT, GELU>;
  static PerDevice configured;
  configured.once([&] {
    check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL));
  });
  const int64_t tiles = (a.n + 127) / 128;
  const int mtiles = (int)((a.rows + BT - 1) / BT);
  const int blocks = (a.k + kBlockK - 1) / kBlockK;
  int splits = 1;
  while (splits < 8 && blocks >= splits * 8 && tiles * mtiles * splits * 2 <= 2 * sm_count()) splits *= 2;
  launch_chained(kernel, dim3((unsigned)(tiles * splits), (unsigned)mtiles), kFewThreads, S::TOTAL, s,
                 true, (unsigned)splits, tw, tx, a, splits, wide_rows<OT>(a));
  return true;
}

template <int BN, typename OT, bool GELU>
bool launch_tile(const LinearArgs& a, cudaStream_t s) {
  using S = Tile<BN>;
  constexpr int kCtas = S::PAIR ? 2 : 1;
  CUtensorMap tw, tx;
  if (!row_map(&tx, a.x, a.rows, a.k, a.x_ld, 128) ||
      !row_map(&tw, a.w, a.n, a.k, a.w_ld, BN / kCtas))
    return false;
  auto kernel = linear_tile_kernel<BN, OT, GELU>;
  static PerDevice configured;
  configured.once([&] {
    check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL));
  });
  const int64_t mtiles = (a.rows + S::ROWS - 1) / S::ROWS, ntiles = (a.n + BN - 1) / BN;
  if (mtiles * ntiles > INT32_MAX) return false;  // no memory holds such an output
  const TileOrder order = {(uint32_t)mtiles, (uint32_t)ntiles, (uint32_t)(mtiles * ntiles)};
  const int wide = wide_rows<OT>(a);
  const unsigned grid = (unsigned)(kCtas * std::min<int64_t>(mtiles * ntiles, sm_count() / kCtas));
  launch_chained(kernel, grid, S::THREADS, S::TOTAL, s, true, kCtas, tx, tw, a, order, wide);
  return true;
}

template <typename OT, bool GELU>
bool launch_typed(const LinearArgs& a, cudaStream_t s) {
  // A few rows: dp4a on streamed weights until its multiplications outweigh a
  // tensor core tile's start. us for 8 rows: 512->512 2.3 against 3.8,
  // 4096->4096 8.6 against 6.9; for 4: 4096->4096 5.5 against 7.0, 8192->8192 21.3
  // against 15.0; for one 4096->4096 2.8 against 8.2. One row of more weights:
  // where k is short for a tile (1024->131072 24.8 against 44.8, 2048->40000 17.8
  // against 21.2; 3000->30000 21.0 against 17.3, 8192->28672 44.4 against 40.8) or
  // the channels make too few clusters for the SMs (65536->2048 25.6 against 27.4,
  // 128000->700 25.2 against 35.8; 65536->4096 52.7 against 45.6).
  if (a.rows <= 8 && (a.rows * a.n * a.k <= 1ll << 26 || (a.rows == 1 && (a.k <= 2048 || a.n <= 2048)))) {
    if (a.rows == 1) launch_gemv<1, 4, OT, GELU>(a, s);
    else if (a.rows == 2) launch_gemv<2, 4, OT, GELU>(a, s);
    else if (a.rows <= 4) launch_gemv<4, 4, OT, GELU>(a, s);
    else launch_gemv<8, 2, OT, GELU>(a, s);
    return true;
  }
  // k split over a cluster pays where k is long (17 rows, 2048->512: 4.5 us
  // against 8.0 by tiles; 512->512 5.1 against 3.8) and, past 64 rows, where
  // tiles would leave most SMs idle (128 rows, 2048->512: 6.4 against 8.2;
  // 4096->4096 13.5 against 11.7)
  if (a.k > 1024 && (a.rows <= 64 || (a.rows <= 128 && a.n <= 1024))) {
    if (a.rows <= 16) return launch_few<16, 5, OT, GELU>(a, s);
    if (a.rows <= 32) return launch_few<32, 5, OT, GELU>(a, s);
    if (a.rows <= 64) return launch_few<64, 4, OT, GELU>(a, s);
    return launch_few<128, 3, OT, GELU>(a, s);
  }
  // the tile whose rounds over the SMs take least: a tile costs its columns and
  // about 32 more for its start and end
  const int64_t sms = sm_count();
  auto cost = [&](int rows, int bn) {
    const int64_t tiles = (a.rows + rows - 1) / rows * ((a.n + bn - 1) / bn) * (rows / 128);
    return (tiles + sms - 1) / sms * (bn + 32);
  };
  const int64_t pair = cost(256, 256), half = cost(128, 128), quarter = cost(128, 64);
  if (pair <= half && pair <= quarter) return launch_tile<256, OT, GELU>(a, s);
  if (half <= quarter) return launch_tile<128, OT, GELU>(a, s);
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
