// Gated linear layer:  h = act(x Wg^T + bg) * (x Wu^T + bu)
//   x (T, K), Wg and Wu (F, K), h (T, F), all bf16; fp32 accumulation.
// Backward from dh, with zg, zu the two projections (recomputed, not kept):
//   dg = dh zu act'(zg),  du = dh act(zg),
//   dx = dg Wg + du Wu,   dWg = dg^T x,  dWu = du^T x,  dbg, dbu = column sums.
//
// Four matrix products on one engine (pair_gemm_kernel), all bound by the
// tensor cores at sizes worth speaking of (4 T K F FLOP forward, 12 T K F with
// the gradients against a few bytes for each of T K + 2 F K + T F values):
//   forward    both projections in one tile: of its 256 accumulator columns 128
//              are the gate's and 128 the other's, so the epilogue finds both
//              in its own TMEM lane and h is all that is written;
//   recompute  the same product again with dg and du for an epilogue.  Keeping
//              zg and zu instead would cost 8 bytes of traffic for each pair of
//              values and 4 F bytes a token of memory, and their rounding to
//              bf16 would reach every gradient; at K = 384 (this model family's
//              towers) the second product takes less time than those bytes;
//   dx         one product over the 2 F values of (dg, du) against (Wg; Wu);
//   dW         (dg, du)^T x, split over tokens where the tiles are few; the
//              parts are fp32 and are added in order by a second kernel.
// dg and du are rounded to bf16 between the products (operands of the tensor
// cores): gradients are 2.3e-3 of their norm off where one rounding at the end leaves
// 1.7e-3.  Everything else is rounded once, when it is written.
//
// Engine: clusters of two CTAs (cta_group::2) share a 256 x 256 tile: each
// loads its 128 rows of A and its 128 rows of B (TMA, 128-byte swizzle, no
// multicast; completion on the even CTA's barrier), the even CTA issues
// tcgen05.mma over both, each keeps its 128 x 256 half of the accumulator in
// its own TMEM, double buffered so that the epilogue of one tile runs under the
// products of the next.  Each SM then reads 128 + 128 operand rows for 256 x
// 128 outputs: half the shared-memory traffic of one CTA alone.  Warp roles
// (576 threads): warp 0 TMA, warp 1 MMA, warps 2-17 epilogue.  Waits are bounded.
// Each launch sets its blocks up while the one before it ends, and one kernel adds
// up what is left of both the biases' and the weights' sums: the training pass of
// 8192 x 384 x 1000 took 127 us with five plain launches and two joins, 118 so.
//
// A few tokens (T <= 8) take skinny_kernel instead: bound by reading the
// weights once, a warp to each hidden value, both weight rows in flight.
#include "alloc.h"
#include "sequence_ops.h"
#include "tmap.h"

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>

#include "pair_sm100.cuh"

namespace tgcm {
namespace {

constexpr int kEpilogueWarps = 16;              // four to a scheduler: one warp's epilogue is mostly latency
constexpr int kPairThreads = 64 + 32 * kEpilogueWarps;
constexpr int kOperand = 128 * 128;             // bytes: 128 rows of 64 bf16
constexpr int kPairStage = 2 * kOperand;
constexpr int kWarpStage = 32 * 64;             // bytes: one epilogue warp's 32 x 32 bf16 tile
// Ring stages: kDact gives one up for the tiles of dh, which are on their way while the tile before is worked on.
template <int MODE>
struct PairCfg {
  static constexpr int kStages = MODE == 1 ? 5 : 6;
  static constexpr int kStaging = (MODE == 1 ? 2 : 1) * kEpilogueWarps * kWarpStage;
  static constexpr int kSmem = kStages * kPairStage + kStaging + 256 + 1024;
};
constexpr int kSkinnyTokens = 8;

enum PairMode : int { kFwd = 0, kDact = 1, kDx = 2, kDw = 3 };

struct PairMaps {
  CUtensorMap a[2], b[2];
};

struct PairParams {
  int M, N;                 // rows and columns of the output (kFwd, kDact: N = F)
  int tiles_m, tiles_n;     // 256 rows; 128 (kFwd, kDact) or 256 columns
  int kb;                   // 64-wide blocks of the reduction (kDx: of each half)
  int splits;               // kDw: parts of the reduction
  int act;
  const __nv_bfloat16 *bias_g, *bias_u;
  __nv_bfloat16* out[2];    // kFwd: h; kDact: dg, du; kDx: dx; kDw: dWg, dWu
  long long ld;             // of out
  const __nv_bfloat16* dh;  // kDact
  long long dh_ld;
  float* bias_part;         // kDact: [row groups of 32][2][F] column sums, or null
  float* part;              // kDw with splits > 1: [split][2][M][part_ld]
  long long part_ld;
  int* err;
};

// 1 / (1 + 2^t) of two values: the sigmoid of -t ln 2.  Two special-function
// instructions each, exact to a few units of 1e-7: far below the rounding of
// the bf16 result.  2^t = inf gives 0.
__device__ __forceinline__ float2 sigmoid2(float2 t) {
  const float2 d = add2(make_float2(ex2(t.x), ex2(t.y)), make_float2(1.f, 1.f));
  return make_float2(rcp(d.x), rcp(d.y));
}
__device__ __forceinline__ float2 all2(float v) { return make_float2(v, v); }

// gelu_tanh(z) = z sigmoid(2u) with 2u = c1 z (1 + 0.044715 z^2), c1 = 2 sqrt(2 / pi)
constexpr float kGeluC1 = 1.5957691216057308f, kGeluC3 = 0.044715f;
constexpr float kLog2E = 1.4426950408889634f;

// NaN stays NaN (a maximum would make it 0).
__device__ __forceinline__ float2 relu2(float2 z) { return make_float2(z.x <= 0.f ? 0.f : z.x, z.y <= 0.f ? 0.f : z.y); }

// act(z) of a pair of pre-activations
template <int ACT>
__device__ __forceinline__ float2 act_val2(float2 z) {
  if constexpr (ACT == kActGeluTanh) {
    const float2 k = fma2(mul2(z, z), all2(-kGeluC1 * kGeluC3 * kLog2E), all2(-kGeluC1 * kLog2E));
    return mul2(z, sigmoid2(mul2(k, z)));
  } else if constexpr (ACT == kActSilu) {
    return mul2(z, sigmoid2(mul2(z, all2(-kLog2E))));
  } else if constexpr (ACT == kActRelu) {
    return relu2(z);
  } else if constexpr (ACT == kActGelu) {
    return make_float2(gelu_erf_f(z.x), gelu_erf_f(z.y));
  } else if constexpr (ACT == kActTanh) {
    return make_float2(tanhf(z.x), tanhf(z.y));
  } else {
    return z;
  }
}

// act(z) and act'(z)
template <int ACT>
__device__ __forceinline__ void act_both2(float2 z, float2* a, float2* da) {
  if constexpr (ACT == kActGeluTanh || ACT == kActSilu) {
    float2 s, slope;  // slope: the derivative of the sigmoid's argument
    if constexpr (ACT == kActGeluTanh) {
      const float2 z2 = mul2(z, z);
      const float2 k = fma2(z2, all2(-kGeluC1 * kGeluC3 * kLog2E), all2(-kGeluC1 * kLog2E));
      s = sigmoid2(mul2(k, z));
      slope = fma2(z2, all2(3.f * kGeluC1 * kGeluC3), all2(kGeluC1));
    } else {
      s = sigmoid2(mul2(z, all2(-kLog2E)));
    }
    *a = mul2(z, s);
    float2 t = mul2(*a, fma2(s, all2(-1.f), all2(1.f)));  // z s (1 - s)
    *da = ACT == kActGeluTanh ? fma2(t, slope, s) : add2(t, s);
  } else if constexpr (ACT == kActRelu) {
    *a = relu2(z);
    *da = make_float2(z.x <= 0.f ? 0.f : 1.f, z.y <= 0.f ? 0.f : 1.f);
  } else if constexpr (ACT == kActGelu) {
    const float2 c = make_float2(0.5f * (1.f + erff(z.x * 0.7071067811865476f)),
                                 0.5f * (1.f + erff(z.y * 0.7071067811865476f)));
    const float2 q = mul2(mul2(z, z), all2(-0.5f * kLog2E));
    *a = mul2(z, c);
    *da = fma2(mul2(z, all2(0.3989422804014327f)), make_float2(ex2(q.x), ex2(q.y)), c);
  } else if constexpr (ACT == kActTanh) {
    *a = make_float2(tanhf(z.x), tanhf(z.y));
    *da = fma2(mul2(*a, all2(-1.f)), *a, all2(1.f));
  } else {
    *a = z;
    *da = all2(1.f);
  }
}

// One switch for 16 values, so the epilogue is compiled once, not once an activation.
#define TGCM_GATED_ACTS(CASE) \
  CASE(kActRelu) CASE(kActGelu) CASE(kActGeluTanh) CASE(kActSilu) CASE(kActTanh) CASE(kActNone)

__device__ __forceinline__ float2 pair_at(const uint32_t (&v)[16], int j) {
  return make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1]));
}
__device__ __forceinline__ void pair_to(uint32_t (&v)[16], int j, float2 x) {
  v[j] = __float_as_uint(x.x);
  v[j + 1] = __float_as_uint(x.y);
}
__device__ __forceinline__ float2 bf2(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

__device__ __forceinline__ void gate16(int act, uint32_t (&g)[16], const uint32_t (&u)[16]) {
  switch (act) {
#define TGCM_CASE(A)                                                                                  \
  case A:                                                                                             \
    _Pragma("unroll") for (int j = 0; j < 16; j += 2)                                                 \
        pair_to(g, j, mul2(act_val2<A>(pair_at(g, j)), pair_at(u, j)));                               \
    break;
    TGCM_GATED_ACTS(TGCM_CASE)
#undef TGCM_CASE
  }
}

// (zg, zu, dh) -> (dg, du)
__device__ __forceinline__ void dgate16(int act, uint32_t (&g)[16], uint32_t (&u)[16], const uint32_t (&dh)[8]) {
  switch (act) {
#define TGCM_CASE(A)                                                                                  \
  case A:                                                                                             \
    _Pragma("unroll") for (int j = 0; j < 16; j += 2) {                                               \
      const float2 d = bf2(dh[j >> 1]);                                                               \
      float2 a, da;                                                                                   \
      act_both2<A>(pair_at(g, j), &a, &da);                                                           \
      pair_to(g, j, mul2(mul2(d, pair_at(u, j)), da));                                                \
      pair_to(u, j, mul2(d, a));                                                                      \
    }                                                                                                 \
    break;
    TGCM_GATED_ACTS(TGCM_CASE)
#undef TGCM_CASE
  }
}

__device__ __forceinline__ uint32_t pack2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(a), __uint_as_float(b));
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Epilogue tiles are 32 rows of four 16-byte pieces; piece c of row r sits at
// c ^ (r / 2 & 3), so a lane writing its own row and four lanes reading one row
// both spread over all banks.
__device__ __forceinline__ uint4* piece(uint8_t* stage, int row, int c) {
  return reinterpret_cast<uint4*>(stage + row * 64 + ((c ^ ((row >> 1) & 3)) << 4));
}

// 32 x 32 bf16 tile to global memory, clipped to nrows x ncols: four lanes to a row's 64
// bytes, or, where rows do not start on 16-byte boundaries, one value to a lane and
// a row to an instruction.
__device__ __forceinline__ void tile_out(uint8_t* stage, __nv_bfloat16* g, long long ld, int nrows, int ncols,
                                         int lane) {
  if ((ld & 7) == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0) {
    const int c = lane & 3;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int row = it * 8 + (lane >> 2);
      if (row >= nrows || c * 8 >= ncols) continue;
      const uint4 v = *piece(stage, row, c);
      __nv_bfloat16* dst = g + row * ld + c * 8;
      if (c * 8 + 8 <= ncols) {
        *reinterpret_cast<uint4*>(dst) = v;
      } else {
        const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(&v);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c * 8 + k < ncols) dst[k] = e[k];
      }
    }
  } else if (lane < ncols) {
#pragma unroll 8
    for (int row = 0; row < 32; ++row)
      if (row < nrows)
        g[row * ld + lane] = reinterpret_cast<const __nv_bfloat16*>(piece(stage, row, lane >> 3))[lane & 7];
  }
}

__device__ __forceinline__ void tile_in(uint8_t* stage, const __nv_bfloat16* g, long long ld, int nrows, int ncols,
                                        int lane) {
  if ((ld & 7) == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0) {
    const int c = lane & 3;
    uint4 v[4];
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int row = it * 8 + (lane >> 2);
      v[it] = make_uint4(0, 0, 0, 0);
      if (row >= nrows || c * 8 >= ncols) continue;
      const __nv_bfloat16* src = g + row * ld + c * 8;
      if (c * 8 + 8 <= ncols) {
        v[it] = __ldg(reinterpret_cast<const uint4*>(src));
      } else {
        __nv_bfloat16* e = reinterpret_cast<__nv_bfloat16*>(&v[it]);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c * 8 + k < ncols) e[k] = src[k];
      }
    }
#pragma unroll
    for (int it = 0; it < 4; ++it) *piece(stage, it * 8 + (lane >> 2), c) = v[it];
  } else {
    const unsigned short* src = reinterpret_cast<const unsigned short*>(g);
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += 16) {
      unsigned short v[16];
#pragma unroll
      for (int r = 0; r < 16; ++r)
        v[r] = r0 + r < nrows && lane < ncols ? __ldg(src + (r0 + r) * ld + lane) : static_cast<unsigned short>(0);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        reinterpret_cast<unsigned short*>(piece(stage, r0 + r, lane >> 3))[lane & 7] = v[r];
    }
  }
}

// The same by asynchronous copies; false where rows do not start on 16-byte boundaries.
__device__ __forceinline__ bool tile_in_async(uint8_t* stage, const __nv_bfloat16* g, long long ld, int nrows,
                                              int ncols, int lane) {
  if ((ld & 7) != 0 || (reinterpret_cast<uintptr_t>(g) & 15) != 0) return false;
  const int c = lane & 3;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int row = it * 8 + (lane >> 2);
    const int have = row < nrows ? max(0, min(8, ncols - c * 8)) * 2 : 0;  // bytes; the rest is zeros
    const __nv_bfloat16* src = have > 0 ? g + row * ld + c * 8 : g;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(piece(stage, row, c))),
                 "l"(src), "r"(have)
                 : "memory");
  }
  return true;
}

// 32 x 16 fp32 tile (the same 64-byte rows) to global memory.
__device__ __forceinline__ void tile_out_f32(uint8_t* stage, float* g, long long ld, int nrows, int ncols, int lane) {
  const int c = lane & 3;  // part_ld is a multiple of 4
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int row = it * 8 + (lane >> 2);
    if (row >= nrows || c * 4 >= ncols) continue;
    *reinterpret_cast<uint4*>(g + row * ld + c * 4) = *piece(stage, row, c);
  }
}

// Column sums of a 32 x 16 block held one row to a lane: after the halving
// steps lanes j and j + 16 have the sum of column j.
__device__ __forceinline__ float column_sums(const uint32_t (&v)[16], int lane) {
  float a[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) a[j] = __uint_as_float(v[j]);
#pragma unroll
  for (int n = 8; n >= 1; n >>= 1) {
    const bool up = lane & n;
#pragma unroll
    for (int j = 0; j < n; ++j) {
      const float keep = up ? a[j + n] : a[j], give = up ? a[j] : a[j + n];
      a[j] = keep + __shfl_xor_sync(0xffffffffu, give, n);
    }
  }
  return a[0] + __shfl_xor_sync(0xffffffffu, a[0], 16);
}

__device__ __forceinline__ uint4 pack8(const uint32_t (&v)[16], int j) {
  return make_uint4(pack2(v[j], v[j + 1]), pack2(v[j + 2], v[j + 3]), pack2(v[j + 4], v[j + 5]),
                    pack2(v[j + 6], v[j + 7]));
}

struct PairTile {
  int tm, tn, which, split, kb0, nkb;
};

template <int MODE>
__device__ __forceinline__ PairTile pair_tile(const PairParams& p, int t) {
  PairTile c;
  c.tn = t % p.tiles_n;
  int r = t / p.tiles_n;
  c.tm = r % p.tiles_m;
  r /= p.tiles_m;
  c.which = 0;
  c.split = 0;
  c.kb0 = 0;
  c.nkb = p.kb;
  if constexpr (MODE == kDx) c.nkb = 2 * p.kb;
  if constexpr (MODE == kDw) {
    c.which = r & 1;
    c.split = r >> 1;
    const int per = (p.kb + p.splits - 1) / p.splits;
    c.kb0 = c.split * per;
    c.nkb = max(0, min(per, p.kb - c.kb0));
  }
  return c;
}

template <int MODE>
__device__ __forceinline__ int pair_tiles(const PairParams& p) {
  return p.tiles_m * p.tiles_n * (MODE == kDw ? 2 * p.splits : 1);
}

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    pair_gemm_kernel(const __grid_constant__ PairMaps maps, const __grid_constant__ PairParams p) {
  constexpr bool A_MN = MODE == kDw;
  constexpr bool B_MN = MODE == kDx || MODE == kDw;
  constexpr uint32_t kIdesc = make_idesc(1, A_MN ? 1 : 0, B_MN ? 1 : 0, 256, 256);
  constexpr int kTileN = (MODE == kFwd || MODE == kDact) ? 128 : 256;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kPairStages = PairCfg<MODE>::kStages;
  uint8_t* staging = smem + kPairStages * kPairStage;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(staging + PairCfg<MODE>::kStaging);  // the leader's are used
  uint64_t* empty_bar = full_bar + kPairStages;
  uint64_t* acc_full = empty_bar + kPairStages;   // [2]
  uint64_t* acc_empty = acc_full + 2;             // [2], the leader's are used
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = pair_rank();
  const int n_tiles = pair_tiles<MODE>(p);
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * kEpilogueWarps);  // of both CTAs
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&maps.a[0]);
    tma_prefetch_desc(&maps.b[0]);
  }
  if (warp == 1) pair_tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  pair_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  after_previous();

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (int t = first; t < n_tiles && !*abort_flag; t += step) {
        const PairTile c = pair_tile<MODE>(p, t);
        for (int i = 0; i < c.nkb; ++i, ++it) {
          const int s = it % kPairStages;
          if (!mbar_park(&empty_bar[s], ((it / kPairStages) & 1) ^ 1, p.err, kErrTimeoutEmpty)) {
            *abort_flag = 1;
            break;
          }
          uint8_t* sa = smem + s * kPairStage;
          uint8_t* sb = sa + kOperand;
          const uint32_t bar = leader_addr(&full_bar[s]);
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], 2 * kPairStage);  // both CTAs' bytes
          if constexpr (MODE == kFwd || MODE == kDact) {
            tma_load_2d_pair(sa, &maps.a[0], bar, i * 64, c.tm * 256 + rank * 128);
            // the even CTA brings the gate's rows, the odd one the other projection's
            tma_load_2d_pair(sb, &maps.b[rank], bar, i * 64, c.tn * 128);
          } else if constexpr (MODE == kDx) {
            const int half = i >= p.kb, k0 = (i - half * p.kb) * 64;
            tma_load_2d_pair(sa, &maps.a[half], bar, k0, c.tm * 256 + rank * 128);
            tma_load_2d_pair(sb, &maps.b[half], bar, c.tn * 256 + rank * 128, k0);
            tma_load_2d_pair(sb + kOperand / 2, &maps.b[half], bar, c.tn * 256 + rank * 128 + 64, k0);
          } else {
            const int k0 = (c.kb0 + i) * 64, m0 = c.tm * 256 + rank * 128, n0 = c.tn * 256 + rank * 128;
            tma_load_2d_pair(sa, &maps.a[c.which], bar, m0, k0);
            tma_load_2d_pair(sa + kOperand / 2, &maps.a[c.which], bar, m0 + 64, k0);
            tma_load_2d_pair(sb, &maps.b[0], bar, n0, k0);
            tma_load_2d_pair(sb + kOperand / 2, &maps.b[0], bar, n0 + 64, k0);
          }
        }
      }
      // no load is in flight when the CTA leaves
      if (rank == 0)
        for (int i = max(0, it - kPairStages); i < it; ++i)
          mbar_park(&full_bar[i % kPairStages], (i / kPairStages) & 1, p.err, kErrTimeoutDrain);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // The whole warp keeps step, one lane issues: addresses stay in uniform registers.
      const bool issuer = elect_lane();
      const uint32_t d0 = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t a0 = desc_lo(smem_u32(smem), A_MN ? kOperand / 2 : 16);
      const uint32_t b0 = desc_lo(smem_u32(smem) + kOperand, B_MN ? kOperand / 2 : 16);
      int s = 0, n = 0;
      uint32_t phase = 0;
      bool go = true;
      for (int t = first; t < n_tiles && go; t += step) {
        const PairTile c = pair_tile<MODE>(p, t);
        if (c.nkb == 0) continue;
        const int acc = n & 1;
        go = mbar_park(&acc_empty[acc], ((n >> 1) & 1) ^ 1, p.err, kErrTimeoutEmpty);
        tc_fence_after();
        for (int i = 0; i < c.nkb && go; ++i) {
          go = mbar_park(&full_bar[s], phase, p.err, kErrTimeoutFull);
          tc_fence_after();
          if (go && issuer) {
            const uint32_t ad = a0 + s * (kPairStage >> 4), bd = b0 + s * (kPairStage >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              pair_umma_ss(d0 + acc * 256, ad + (A_MN ? step_mn(k) : step_k(128, k)),
                           bd + (B_MN ? step_mn(k) : step_k(128, k)), kIdesc, (i | k) ? 1u : 0u);
            pair_commit(&empty_bar[s]);
          }
          __syncwarp();
          if (++s == kPairStages) {
            s = 0;
            phase ^= 1;
          }
        }
        go = __all_sync(0xffffffffu, go && !*abort_flag);
        if (issuer) pair_commit(&acc_full[acc]);  // also after a timeout: the epilogue does not wait for nothing
        __syncwarp();
        ++n;
      }
      if (!go) *abort_flag = 1;
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;  // TMEM lanes, quarter of the tile's columns
    uint8_t* stage = staging + (warp - 2) * kWarpStage;
    // kDact: dh of the tile to come, asked for as soon as this tile's du has left its place
    uint8_t* dh_stage = staging + (kEpilogueWarps + warp - 2) * kWarpStage;
    auto fetch_dh = [&](int t) {
      if (t < n_tiles) {
        const PairTile c = pair_tile<MODE>(p, t);
        const int row0 = c.tm * 256 + rank * 128 + q * 32, col0 = c.tn * kTileN + part * (kTileN / 4);
        const int nrows = min(32, p.M - row0), ncols = p.N - col0;
        if (nrows > 0 && ncols > 0) {
          const __nv_bfloat16* src = p.dh + static_cast<long long>(row0) * p.dh_ld + col0;
          if (!tile_in_async(dh_stage, src, p.dh_ld, nrows, ncols, lane))
            tile_in(dh_stage, src, p.dh_ld, nrows, ncols, lane);
        } else {
#pragma unroll
          for (int v = 0; v < 4; ++v) *piece(dh_stage, lane, v) = make_uint4(0, 0, 0, 0);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if constexpr (MODE == kDact) fetch_dh(first);
    int n = 0;
    for (int t = first; t < n_tiles; t += step) {
      const PairTile c = pair_tile<MODE>(p, t);
      const int row0 = c.tm * 256 + rank * 128 + q * 32;
      const int nrows = min(32, p.M - row0);
      const int colw = part * (kTileN / 4);            // this warp's columns of the tile
      const int col0 = c.tn * kTileN + colw;
      uint32_t bias = 0;  // of column col0 + lane: the gate's in the lower half, the other's in the upper
      if constexpr (MODE == kFwd || MODE == kDact) {
        if (p.bias_g != nullptr && col0 + lane < p.N)
          bias = static_cast<uint32_t>(__ldg(reinterpret_cast<const unsigned short*>(p.bias_g) + col0 + lane)) |
                 static_cast<uint32_t>(__ldg(reinterpret_cast<const unsigned short*>(p.bias_u) + col0 + lane)) << 16;
      }
      const int acc = n & 1;
      if (c.nkb > 0) {
        const bool have = mbar_park(&acc_full[acc], (n >> 1) & 1, p.err, kErrTimeoutTmemFull);
        if (__any_sync(0xffffffffu, !have || *abort_flag)) break;
        tc_fence_after();
        ++n;
      }
      if constexpr (MODE == kDact) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();  // every lane's part of dh has landed, and the staging tile has been read
      }
      const uint32_t ta = tmem + acc * 256 + (static_cast<uint32_t>(q * 32) << 16);
      if constexpr (MODE == kFwd || MODE == kDact) {
        // One body for both chunks: unrolled, the recompute's instructions outgrow their cache (8192 tokens,
        // 384 x 1000: 34.7 us with two bodies, 31.5 with one).
#pragma unroll 1
        for (int ch = 0; ch < 2; ++ch) {
          uint32_t g[16], u[16];
          tmem_ld_32x32b_x16(ta + colw + ch * 16, g);
          tmem_ld_32x32b_x16(ta + 128 + colw + ch * 16, u);
          tmem_ld_wait();
          if (p.bias_g != nullptr) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float2 b = bf2(__shfl_sync(0xffffffffu, bias, ch * 16 + j));
              g[j] = __float_as_uint(__uint_as_float(g[j]) + b.x);
              u[j] = __float_as_uint(__uint_as_float(u[j]) + b.y);
            }
          }
          if constexpr (MODE == kFwd) {
            gate16(p.act, g, u);
          } else {
            uint32_t dh[8];
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              const uint4 w = *piece(dh_stage, lane, ch * 2 + v);
              dh[4 * v] = w.x, dh[4 * v + 1] = w.y, dh[4 * v + 2] = w.z, dh[4 * v + 3] = w.w;
            }
            dgate16(p.act, g, u, dh);
            if (p.bias_part != nullptr) {
              const float sg = column_sums(g, lane), su = column_sums(u, lane);
              const int col = col0 + ch * 16 + (lane & 15);
              if (col < p.N)  // the lower half of the warp has the gate's sums to write, the upper the other's
                p.bias_part[(static_cast<long long>(row0 >> 5) * 2 + (lane >> 4)) * p.N + col] = lane < 16 ? sg : su;
            }
            *piece(dh_stage, lane, ch * 2) = pack8(u, 0);  // du takes dh's place
            *piece(dh_stage, lane, ch * 2 + 1) = pack8(u, 8);
          }
          *piece(stage, lane, ch * 2) = pack8(g, 0);
          *piece(stage, lane, ch * 2 + 1) = pack8(g, 8);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(leader_addr(&acc_empty[acc]));
        tile_out(stage, p.out[0] + static_cast<long long>(row0) * p.ld + col0, p.ld, nrows, p.N - col0, lane);
        if constexpr (MODE == kDact) {
          tile_out(dh_stage, p.out[1] + static_cast<long long>(row0) * p.ld + col0, p.ld, nrows, p.N - col0, lane);
          __syncwarp();
          fetch_dh(t + step);
        }
        __syncwarp();
      } else {
        const bool parts = MODE == kDw && p.splits > 1;
        if (parts) {
          float* dst = p.part + (static_cast<long long>(c.split * 2 + c.which) * p.M + row0) * p.part_ld;
#pragma unroll 1
          for (int ch = 0; ch < 4; ++ch) {
            uint32_t v[16];
            tmem_ld_32x32b_x16(ta + colw + ch * 16, v);
            tmem_ld_wait();
            if (c.nkb == 0) {
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = 0u;
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *piece(stage, lane, j) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            __syncwarp();
            const int col = col0 + ch * 16;
            tile_out_f32(stage, dst + col, p.part_ld, nrows, static_cast<int>(p.part_ld) - col, lane);
          }
        } else {
          __nv_bfloat16* dst = p.out[c.which] + static_cast<long long>(row0) * p.ld;
#pragma unroll 1
          for (int c2 = 0; c2 < 2; ++c2) {
            uint32_t v[16], w[16];
            tmem_ld_32x32b_x16(ta + colw + c2 * 32, v);
            tmem_ld_32x32b_x16(ta + colw + c2 * 32 + 16, w);
            tmem_ld_wait();
            __syncwarp();
            *piece(stage, lane, 0) = pack8(v, 0);
            *piece(stage, lane, 1) = pack8(v, 8);
            *piece(stage, lane, 2) = pack8(w, 0);
            *piece(stage, lane, 3) = pack8(w, 8);
            __syncwarp();
            const int col = col0 + c2 * 32;
            tile_out(stage, dst + col, p.ld, nrows, p.N - col, lane);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0 && c.nkb > 0) arrive_cluster(leader_addr(&acc_empty[acc]));
      }
    }
    if constexpr (MODE == kDact) asm volatile("cp.async.wait_group 0;" ::: "memory");
  }

  tc_fence_before();
  __syncthreads();
  pair_sync();
  if (warp == 1) {
    tc_fence_after();
    pair_tmem_dealloc(tmem, 512);
  }
}

// What the products leave to be added up, in order and rounded once: the first blocks take the biases' column
// sums over the row groups (32 columns to a block), the others the parts of dW (four columns to a thread).
struct JoinParams {
  const float* bias_part;  // [groups][2][F]
  const float* part;       // [splits][2][F][part_ld]
  __nv_bfloat16 *bg, *bu, *wg, *wu;
  int F, K, groups, splits, bias_blocks;
  long long part_ld;
};

__global__ void __launch_bounds__(256) join_kernel(const JoinParams p) {
  after_previous();
  if (static_cast<int>(blockIdx.x) < p.bias_blocks) {
    __shared__ float acc[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float a = 0.f;
    if (c < 2 * p.F) {
#pragma unroll 8
      for (int g = warp; g < p.groups; g += 8) a += p.bias_part[static_cast<long long>(g) * 2 * p.F + c];
    }
    acc[warp][lane] = a;
    __syncthreads();
    if (warp == 0 && c < 2 * p.F) {
      float t = 0.f;
      for (int w = 0; w < 8; ++w) t += acc[w][lane];
      (c < p.F ? p.bg[c] : p.bu[c - p.F]) = __float2bfloat16(t);
    }
    return;
  }
  const long long i = (static_cast<long long>(blockIdx.x - p.bias_blocks) * 256 + threadIdx.x) * 4;
  const long long row = i / p.part_ld;
  const int col = static_cast<int>(i - row * p.part_ld);
  if (row >= 2ll * p.F) return;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < p.splits; ++s) {
    const float4 v = *reinterpret_cast<const float4*>(p.part + (s * 2ll * p.F + row) * p.part_ld + col);
    a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
  }
  __nv_bfloat16* o = row < p.F ? p.wg + row * p.K : p.wu + (row - p.F) * p.K;
  const float r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < p.K) o[col + e] = __float2bfloat16(r[e]);
}

// A few tokens: a warp to each hidden value.  x stays in shared memory (bf16);
// a lane reads 16 bytes of both weight rows and meets them with every token.
template <int TT>
__global__ void __launch_bounds__(256) skinny_kernel(const __nv_bfloat16* __restrict__ x, long long x_ld,
                                                    const __nv_bfloat16* __restrict__ wg,
                                                    const __nv_bfloat16* __restrict__ wu, long long w_ld,
                                                    long long u_ld, const __nv_bfloat16* __restrict__ bg,
                                                    const __nv_bfloat16* __restrict__ bu,
                                                    __nv_bfloat16* __restrict__ h, int T, int K, int F, int act) {
  const int lane = threadIdx.x & 31;
  const int f = (blockIdx.x * 256 + threadIdx.x) >> 5;
  if (f >= F) return;
  float ag[TT], au[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) ag[t] = au[t] = 0.f;
  const __nv_bfloat16* g = wg + f * w_ld;
  const __nv_bfloat16* u = wu + f * u_ld;
#pragma unroll 4
  for (int k = lane * 8; k < K; k += 256) {
    const uint4 gv = __ldg(reinterpret_cast<const uint4*>(g + k)), uv = __ldg(reinterpret_cast<const uint4*>(u + k));
    const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w}, uw[4] = {uv.x, uv.y, uv.z, uv.w};
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      if (t >= T) break;
      const uint4 xv = __ldg(reinterpret_cast<const uint4*>(x + t * x_ld + k));
      const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x0 = __uint_as_float(xw[e] << 16), x1 = __uint_as_float(xw[e] & 0xffff0000u);
        ag[t] = fmaf(x0, __uint_as_float(gw[e] << 16), ag[t]);
        ag[t] = fmaf(x1, __uint_as_float(gw[e] & 0xffff0000u), ag[t]);
        au[t] = fmaf(x0, __uint_as_float(uw[e] << 16), au[t]);
        au[t] = fmaf(x1, __uint_as_float(uw[e] & 0xffff0000u), au[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TT; ++t) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ag[t] += __shfl_xor_sync(0xffffffffu, ag[t], o);
      au[t] += __shfl_xor_sync(0xffffffffu, au[t], o);
    }
  }
  float zg = 0.f, zu = 0.f;  // lane t finishes token t
#pragma unroll
  for (int t = 0; t < TT; ++t)
    if (lane == t) zg = ag[t], zu = au[t];
  if (lane >= T) return;
  if (bg != nullptr) {
    zg += __bfloat162float(bg[f]);
    zu += __bfloat162float(bu[f]);
  }
  float a = zg;
  switch (act) {
#define TGCM_CASE(A) \
  case A: a = act_val2<A>(make_float2(zg, 0.f)).x; break;
    TGCM_GATED_ACTS(TGCM_CASE)
#undef TGCM_CASE
  }
  h[static_cast<long long>(lane) * F + f] = __float2bfloat16(a * zu);
}

// Rows of `from` values (any strides) to rows of `to` values behind one another, zeros behind the end: TMA's
// 16-byte rows for matrices that have none.
__global__ void __launch_bounds__(256) pad_rows_kernel(const __nv_bfloat16* __restrict__ in, long long row_stride,
                                                      long long col_stride, __nv_bfloat16* __restrict__ out, int rows,
                                                      int from, int to) {
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < static_cast<long long>(rows) * to / 8;
       i += static_cast<long long>(gridDim.x) * 256) {
    const int r = static_cast<int>(i / (to / 8)), c = static_cast<int>(i - static_cast<long long>(r) * (to / 8)) * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    __nv_bfloat16* e = reinterpret_cast<__nv_bfloat16*>(&v);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < from) e[k] = in[r * row_stride + (c + k) * col_stride];
    reinterpret_cast<uint4*>(out)[i] = v;
  }
}

// Rows of 64 (K-major operands: 128 of them; MN-major ones: 64 steps of the reduction).
CUtensorMap matrix_map(const at::Tensor& t, uint32_t box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(t.size(1)), static_cast<uint64_t>(t.size(0))};
  const uint64_t strides[1] = {static_cast<uint64_t>(t.size(0) > 1 ? t.stride(0) : (t.size(1) + 7) / 8 * 8) * 2};
  const uint32_t box[2] = {64, box_rows};
  return tmap_bf16<2>(t.data_ptr(), dims, strides, box);
}

// CTA pairs that run at once: a GPC with an odd number of free SMs leaves one idle,
// and a pair that has to wait for another to end would double the time.
int resident_pairs() {
  static int pairs[64] = {0};
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 64 && pairs[dev] > 0) return pairs[dev];
  auto kern = pair_gemm_kernel<kFwd>;
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg<kFwd>::kSmem));
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(sms / 2 * 2);
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = PairCfg<kFwd>::kSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  C10_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
  TORCH_CHECK(n >= 1, "gated_linear: no room for a pair of CTAs on this device");
  if (dev < 64) pairs[dev] = n;
  return n;
}

// A launch whose blocks may be set up while the kernel before it ends (see after_previous).
template <class... P, class... A>
void launch_after(void (*kern)(P...), int blocks, int threads, int smem, cudaStream_t st, const A&... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, args...));
}

template <int MODE>
void launch_pair(const PairMaps& maps, const PairParams& p, int tiles, cudaStream_t st) {
  auto kern = pair_gemm_kernel<MODE>;
  static bool set[64] = {false};  // the attribute is per device and per kernel
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev >= 64 || !set[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg<MODE>::kSmem));
    if (dev < 64) set[dev] = true;
  }
  launch_after(kern, 2 * std::max(1, std::min(tiles, resident_pairs())), kPairThreads, PairCfg<MODE>::kSmem, st, maps, p);
}

int ceil_div(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }

// TMA rows: unit inner stride, 16-byte row pitch and base.
bool tma_ok(const at::Tensor& t) {
  return t.stride(1) == 1 && (t.size(0) == 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1))) &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && t.size(1) % 8 == 0;
}

// A copy with the inner extent padded to a multiple of 8 with zeros, where TMA cannot read the tensor as it is.
at::Tensor tma_rows(const at::Tensor& t) {
  if (tma_ok(t)) return t;
  const int64_t w = (t.size(1) + 7) / 8 * 8;
  auto c = out_empty({t.size(0), w}, t.options());
  const int64_t blocks = std::min<int64_t>((t.size(0) * w / 8 + 255) / 256, 148 * 8);
  if (blocks > 0) {
    pad_rows_kernel<<<static_cast<unsigned>(blocks), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
        reinterpret_cast<const __nv_bfloat16*>(t.data_ptr()), t.stride(0), t.stride(1),
        reinterpret_cast<__nv_bfloat16*>(c.data_ptr()), static_cast<int>(t.size(0)), static_cast<int>(t.size(1)),
        static_cast<int>(w));
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return c;
}

void check_gated(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const c10::optional<at::Tensor>& bg,
                 const c10::optional<at::Tensor>& bu, int64_t act) {
  for (const auto* t : {&x, &wg, &wu})
    TORCH_CHECK(t->is_cuda() && t->device() == x.device() && t->dim() == 2 && t->scalar_type() == at::kBFloat16,
                "gated_linear: bf16 CUDA matrices of one device expected");
  TORCH_CHECK(wg.sizes() == wu.sizes() && wg.size(1) == x.size(1),
              "gated_linear: both weights must be (hidden, features) and match x");
  TORCH_CHECK(x.size(1) >= 1 && wg.size(0) >= 1, "gated_linear: empty weights");
  TORCH_CHECK(x.size(0) < (1ll << 31) - 256 && x.size(1) < (1ll << 31) - 256 && wg.size(0) < (1ll << 30),
              "gated_linear: sizes beyond 2^31");
  const bool a = bg.has_value() && bg->defined(), b = bu.has_value() && bu->defined();
  TORCH_CHECK(a == b, "gated_linear: both biases or none");
  if (a)
    for (const auto& t : {*bg, *bu})
      TORCH_CHECK(t.device() == x.device() && t.scalar_type() == at::kBFloat16 && t.is_contiguous() &&
                      t.numel() == wg.size(0),
                  "gated_linear: biases must be contiguous bf16 vectors of the hidden size");
  TORCH_CHECK(act >= kActNone && act <= kActTanh, "gated_linear: unknown activation");
}

const __nv_bfloat16* bf16_or_null(const c10::optional<at::Tensor>& t) {
  return t.has_value() && t->defined() ? reinterpret_cast<const __nv_bfloat16*>(t->data_ptr()) : nullptr;
}
__nv_bfloat16* bf16_ptr(const at::Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); }

}  // namespace

at::Tensor gated_rows(const at::Tensor& t) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && t.scalar_type() == at::kBFloat16,
              "gated_linear: bf16 CUDA matrices of one device expected");
  c10::cuda::CUDAGuard guard(t.device());
  return tma_rows(t);
}

at::Tensor gated_fwd(const at::Tensor& x_in, const at::Tensor& wg_in, const at::Tensor& wu_in,
                     const c10::optional<at::Tensor>& bg, const c10::optional<at::Tensor>& bu, int64_t act,
                     const c10::optional<at::Tensor>& err) {
  check_gated(x_in, wg_in, wu_in, bg, bu, act);
  c10::cuda::CUDAGuard guard(x_in.device());
  const int64_t T = x_in.size(0), F = wg_in.size(0);
  auto h = out_empty({T, F}, x_in.options());
  if (T == 0) return h;
  const at::Tensor x = tma_rows(x_in), wg = tma_rows(wg_in), wu = tma_rows(wu_in);
  const int64_t K = x.size(1);
  auto st = at::cuda::getCurrentCUDAStream();
  if (T <= kSkinnyTokens) {
    const dim3 grid(ceil_div(F, 8));
    auto run = [&](auto tt) {
      skinny_kernel<decltype(tt)::value><<<grid, 256, 0, st>>>(
          bf16_ptr(x), x.stride(0), bf16_ptr(wg), bf16_ptr(wu), wg.stride(0), wu.stride(0), bf16_or_null(bg),
          bf16_or_null(bu), bf16_ptr(h), static_cast<int>(T), static_cast<int>(K), static_cast<int>(F),
          static_cast<int>(act));
    };
    if (T == 1)
      run(std::integral_constant<int, 1>());
    else if (T == 2)
      run(std::integral_constant<int, 2>());
    else if (T <= 4)
      run(std::integral_constant<int, 4>());
    else
      run(std::integral_constant<int, 8>());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    return h;
  }
  PairMaps maps;
  maps.a[0] = maps.a[1] = matrix_map(x, 128);
  maps.b[0] = matrix_map(wg, 128);
  maps.b[1] = matrix_map(wu, 128);
  PairParams p{};
  p.M = static_cast<int>(T), p.N = static_cast<int>(F);
  p.tiles_m = ceil_div(T, 256), p.tiles_n = ceil_div(F, 128), p.kb = ceil_div(K, 64), p.splits = 1;
  p.act = static_cast<int>(act);
  p.bias_g = bf16_or_null(bg), p.bias_u = bf16_or_null(bu);
  p.out[0] = bf16_ptr(h);
  p.ld = F;
  p.err = err.has_value() && err->defined() ? err->data_ptr<int>() : nullptr;
  launch_pair<kFwd>(maps, p, p.tiles_m * p.tiles_n, st);
  return h;
}

// dx, dWg, dWu, dbg, dbu; the ones not asked for are undefined.  x and the weights may be padded (gated_rows): the
// first `features` columns count.
std::vector<at::Tensor> gated_bwd(const at::Tensor& dh_in, const at::Tensor& x_in, const at::Tensor& wg_in,
                                  const at::Tensor& wu_in, const c10::optional<at::Tensor>& bg,
                                  const c10::optional<at::Tensor>& bu, int64_t act, int64_t features, bool need_x, bool need_w,
                                  bool need_b, const c10::optional<at::Tensor>& err) {
  check_gated(x_in, wg_in, wu_in, bg, bu, act);
  const int64_t T = x_in.size(0), F = wg_in.size(0), K0 = features;
  TORCH_CHECK(K0 >= 1 && K0 <= x_in.size(1), "gated_linear backward: features beyond x's rows");
  TORCH_CHECK(dh_in.dim() == 2 && dh_in.size(0) == T && dh_in.size(1) == F && dh_in.device() == x_in.device() &&
                  dh_in.scalar_type() == at::kBFloat16 && (F == 1 || dh_in.stride(1) == 1),
              "gated_linear backward: the gradient must be bf16 (tokens, hidden) with contiguous rows");
  c10::cuda::CUDAGuard guard(x_in.device());
  need_b = need_b && bg.has_value() && bg->defined();
  auto opt = x_in.options();
  auto dx = need_x ? out_empty({T, K0}, opt) : at::Tensor();
  auto dwg = need_w ? out_empty({F, K0}, opt) : at::Tensor(), dwu = need_w ? out_empty({F, K0}, opt) : at::Tensor();
  auto dbg = need_b ? out_empty({F}, opt) : at::Tensor(), dbu = need_b ? out_empty({F}, opt) : at::Tensor();
  auto result = [&] {
    return std::vector<at::Tensor>{dx, dwg, dwu, dbg, dbu};
  };
  if (T == 0) {
    for (auto* t : {&dwg, &dwu, &dbg, &dbu})
      if (t->defined()) t->zero_();
    return result();
  }
  const at::Tensor x = tma_rows(x_in), wg = tma_rows(wg_in), wu = tma_rows(wu_in);
  const int64_t K = x.size(1), Fp = (F + 7) / 8 * 8;
  auto st = at::cuda::getCurrentCUDAStream();
  int* flag = err.has_value() && err->defined() ? err->data_ptr<int>() : nullptr;
  auto dgu = out_empty({2, T, Fp}, opt);
  const at::Tensor dg = dgu[0].narrow(1, 0, F), du = dgu[1].narrow(1, 0, F);
  at::Tensor bias_part, part;
  JoinParams join{};
  join.F = static_cast<int>(F), join.K = static_cast<int>(K0), join.part_ld = 4;
  const int groups = ceil_div(T, 256) * 8;
  {
    PairMaps maps;
    maps.a[0] = maps.a[1] = matrix_map(x, 128);
    maps.b[0] = matrix_map(wg, 128);
    maps.b[1] = matrix_map(wu, 128);
    PairParams p{};
    p.M = static_cast<int>(T), p.N = static_cast<int>(F);
    p.tiles_m = ceil_div(T, 256), p.tiles_n = ceil_div(F, 128), p.kb = ceil_div(K, 64), p.splits = 1;
    p.act = static_cast<int>(act);
    p.bias_g = bf16_or_null(bg), p.bias_u = bf16_or_null(bu);
    p.out[0] = bf16_ptr(dg), p.out[1] = bf16_ptr(du);
    p.ld = Fp;
    p.dh = bf16_ptr(dh_in);
    p.dh_ld = T > 1 ? dh_in.stride(0) : F;
    if (need_b) {
      bias_part = out_empty({groups, 2, F}, opt.dtype(at::kFloat));
      join.bias_part = p.bias_part = bias_part.data_ptr<float>();
      join.bg = bf16_ptr(dbg), join.bu = bf16_ptr(dbu);
      join.groups = groups, join.bias_blocks = ceil_div(2 * F, 32);
    }
    p.err = flag;
    launch_pair<kDact>(maps, p, p.tiles_m * p.tiles_n, st);
  }
  if (need_x) {
    PairMaps maps;
    maps.a[0] = matrix_map(dg, 128);
    maps.a[1] = matrix_map(du, 128);
    maps.b[0] = matrix_map(wg, 64);
    maps.b[1] = matrix_map(wu, 64);
    PairParams p{};
    p.M = static_cast<int>(T), p.N = static_cast<int>(K0);
    p.tiles_m = ceil_div(T, 256), p.tiles_n = ceil_div(K0, 256), p.kb = ceil_div(F, 64), p.splits = 1;
    p.out[0] = bf16_ptr(dx);
    p.ld = K0;
    p.err = flag;
    launch_pair<kDx>(maps, p, p.tiles_m * p.tiles_n, st);
  }
  if (need_w) {
    PairMaps maps;
    maps.a[0] = matrix_map(dg, 64);
    maps.a[1] = matrix_map(du, 64);
    maps.b[0] = maps.b[1] = matrix_map(x, 64);
    PairParams p{};
    p.M = static_cast<int>(F), p.N = static_cast<int>(K0);
    p.tiles_m = ceil_div(F, 256), p.tiles_n = ceil_div(K0, 256), p.kb = ceil_div(T, 64);
    // Parts of the reduction, by their estimated time: the slowest pair's steps of 0.27 us (512 cycles of
    // products), and for more than one part 3 us and the parts' way to memory and back at 5 TB/s.  F = 1000,
    // K = 384, T = 8192 gets four parts (20 us and 3 us to join them); 4096, 1024, 16384 one (204 us; four parts
    // took 186 us and 27 us to join).
    const int pairs = resident_pairs();
    const int64_t tiles = 2ll * p.tiles_m * p.tiles_n;
    const double bytes = 2.0 * F * K0 * 8;
    double best = 0;
    p.splits = 1;
    for (int s = 1; s <= 32 && (s == 1 || p.kb / s >= 8); ++s) {
      const double cost = 0.27 * ((tiles * s + pairs - 1) / pairs) * ceil_div(p.kb, s) + (s > 1 ? 3 + s * bytes / 5e6 : 0);
      if (s == 1 || cost < best) best = cost, p.splits = s;
    }
    p.out[0] = bf16_ptr(dwg), p.out[1] = bf16_ptr(dwu);
    p.ld = K0;
    p.err = flag;
    if (p.splits > 1) {
      p.part_ld = (K0 + 3) / 4 * 4;
      part = out_empty({p.splits, 2, F, p.part_ld}, opt.dtype(at::kFloat));
      p.part = part.data_ptr<float>();
      join.part = p.part, join.part_ld = p.part_ld, join.splits = p.splits;
      join.wg = bf16_ptr(dwg), join.wu = bf16_ptr(dwu);
    }
    launch_pair<kDw>(maps, p, static_cast<int>(tiles * p.splits), st);
  }
  const int join_blocks = join.bias_blocks + (join.splits > 1 ? ceil_div(2 * F * join.part_ld / 4, 256) : 0);
  if (join_blocks > 0) launch_after(join_kernel, join_blocks, 256, 0, st, join);
  return result();
}

}  // namespace tgcm
