// Window attention with sinks on the tensor cores: bf16, head sizes that are
// multiples of 8 up to 128 (formulas in window_attention.cu).
//
// Three kernels: forward, dq (with delta), dk and dv.  Each gives a CTA 128
// rows of one head (queries; keys for dk and dv) and walks the tiles of the
// other side that are in sight of them: a run of tiles through the window,
// and the sinks.  Warp 0 feeds a ring of shared-memory slots by TMA, one
// thread of warp 1 issues tcgen05.mma, warps 2-5 own one row to a thread and
// do the softmax arithmetic on accumulators read from TMEM; the weights and
// their gradients are the A operand of the next product as bf16, from TMEM
// (forward) or shared memory (backward, where TMEM is full).  That rounding is the
// price of these products: results are 2.0e-3 (o) and 2.4e-3 (gradients) of their
// norm off where one rounding at the end leaves 1.7e-3; a second product with what the
// rounding left over would double the products of P and dS.  Nothing of the
// size of the score matrix leaves the SM.
//
// What bounds them: 128 x 64 scores are 8192 exponentials, 512 cycles of the
// SM's 16 a cycle, against 256 cycles of products at D = 64, but a tile's way
// through wait, accumulator read, maximum, exponentials and write-back takes one
// CTA 1400 cycles (2950 in dk/dv).  So two CTAs share an SM (tiles sized for half of
// its TMEM and shared memory), and the next tile's scores are made while this
// one's are worked on.  Only at D = 128 do dk and dv need all of TMEM.
// Measured on 2 x 8192 tokens, 16 + 4 heads of 64, window 512, 4 sinks: forward 97
// us (112 with what the backward needs), dq 142 us, dk/dv 183 us.  Eight softmax warps instead of four, smaller TMEM
// shares for three or four CTAs, and weights kept in TMEM in the backward were
// each tried and took as long or longer.
//   D <= 64:  forward 64-key tiles (2 x S, under P, 64, O 64 columns),
//             dq 64-key tiles (S, dP, dQ 64 each),
//             dk/dv 64-query tiles (S, dP, dV, dK 64 each)
//   D <= 128: forward 64-key tiles (2 x S, under P, 64, O 128),
//             dq 64-key tiles (S 64, dP 64, dQ 128),
//             dk/dv 64-query tiles (2 x (S, dP 64), dV, dK 128)
// A head narrower than its tile is filled with zeros by TMA; products run over
// the columns that are there, rounded up to 16.
//
// The forward keeps a running maximum that is only raised (and O rescaled)
// when a row exceeds it by 2^8: the weights stay below 256 and the sums are
// fp32, so nothing is lost.  dq and dk/dv recompute the weights from lse; they
// are separate kernels, at the price of two more products, so that every sum
// has one owner: no atomics, the same bits every time, and shared key heads are
// summed over their query heads in the accumulator.  The sinks are seen by
// every query, so their gradients would be one CTA's work over the whole
// sequence: the queries outside the sink tile's own window are split over
// extra CTAs whose fp32 parts are added in order by a small kernel.
#include "alloc.h"
#include "tmap.h"

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>

#include <algorithm>

#include "pair_sm100.cuh"
#include "window_attention.h"

namespace tgcm {
namespace {

constexpr int kAttnThreads = 192;
constexpr int kAtom = 128;  // bytes of a swizzled row: 64 bf16

struct AttnMaps {
  CUtensorMap q, k, v, g;
};

// ── instructions ───────────────────────────────────────────────────────────
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Largest of three, NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^t of two values on the FMA pipe: t = n + f with |f| <= 1/2 (n by adding and
// taking away 1.5 * 2^23), a cubic for 2^f (least largest relative error on the
// interval, 7.5e-5: a twentieth of a bf16 weight's rounding), n into the
// exponent.  t below -126 gives 2^-126, and so does NaN: nothing beside a row's
// largest weight, and rows that have none are set to zero at the end.
__device__ __forceinline__ float2 ex2_poly2(float2 t) {
  t.x = fmaxf(t.x, -126.f);
  t.y = fmaxf(t.y, -126.f);
  const float2 shift = make_float2(12582912.f, 12582912.f), back = make_float2(-12582912.f, -12582912.f);
  const float2 z = add2(t, shift);
  const float2 n = add2(z, back);
  const float2 f = fma2(n, make_float2(-1.f, -1.f), t);
  float2 v = fma2(f, make_float2(0.05517166853f, 0.05517166853f), make_float2(0.24261112511f, 0.24261112511f));
  v = fma2(v, f, make_float2(0.69326096773f, 0.69326096773f));
  v = fma2(v, f, make_float2(0.99992805719f, 0.99992805719f));
  v.x = __int_as_float(__float_as_int(v.x) + (__float_as_int(z.x) << 23));
  v.y = __int_as_float(__float_as_int(v.y) + (__float_as_int(z.y) << 23));
  return v;
}

__device__ __forceinline__ uint32_t pack_f2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// c plus the two bf16 values of w.
__device__ __forceinline__ float2 add_packed(float2 c, uint32_t w) {
  float2 d;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "add.rn.f32.bf16 %0, l, %3;\n\tadd.rn.f32.bf16 %1, h, %4;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "r"(w), "f"(c.x), "f"(c.y));
  return d;
}

__device__ __forceinline__ void load_row32(uint32_t taddr, float* s) {
  uint32_t r[32];
  tmem_ld_32x32b_x32(taddr, r);
#pragma unroll
  for (int i = 0; i < 32; ++i) s[i] = __uint_as_float(r[i]);
}

// Bounded wait of a whole warp: false in all lanes when one gave up.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  return __all_sync(0xffffffffu, mbar_park(bar, parity, err, code));
}

// One row of D <= 64 * A values in bf16 from this thread to the staging tile
// (atoms of 128 rows), then 32 rows of the warp to global memory, eight lanes
// to a row's 128 bytes.
__device__ __forceinline__ uint4* stage_piece(uint8_t* stage, int atom, int row, int c) {
  return reinterpret_cast<uint4*>(stage + atom * (128 * kAtom) + row * kAtom + ((c ^ (row & 7)) << 4));
}
template <int DP>
__device__ __forceinline__ void store_rows(uint8_t* stage, __nv_bfloat16* dst, long long row_stride, int D, int row0,
                                           int lo, int hi, int lane) {
#pragma unroll
  for (int a = 0; a < DP / 64; ++a)
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int row = row0 + it * 4 + (lane >> 3), d = a * 64 + (lane & 7) * 8;
      if (row >= lo && row < hi && d < D)
        *reinterpret_cast<uint4*>(dst + row * row_stride + d) = *stage_piece(stage, a, row, lane & 7);
    }
}
// TMEM columns [col, col + DP) of this thread's row, times f, to the staging tile; with REST what these values
// times `exact` have beyond their rounded products with f.
template <int DP, bool REST = false>
__device__ __forceinline__ void stage_row(uint8_t* stage, uint32_t taddr, bool have, float f, int row,
                                          float exact = 0.f) {
#pragma unroll
  for (int c = 0; c < DP / 32; ++c) {
    float v[32];
    if (have) {
      load_row32(taddr + c * 32, v);
      tmem_ld_wait();
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float x = v[i] * f;
      v[i] = REST ? v[i] * exact - __bfloat162float(__float2bfloat16(x)) : x;
    }
#pragma unroll
    for (int p = 0; p < 4; ++p)
      *stage_piece(stage, c >> 1, row, (c & 1) * 4 + p) =
          make_uint4(pack_f2(v[8 * p], v[8 * p + 1]), pack_f2(v[8 * p + 2], v[8 * p + 3]),
                     pack_f2(v[8 * p + 4], v[8 * p + 5]), pack_f2(v[8 * p + 6], v[8 * p + 7]));
  }
}

// Key tiles of the queries [i0, i0 + 128): tiles of the sinks below the window's
// first key, then tiles through the window (and up to the last sink).
struct KeyTiles {
  int sink_end, lo, hi, n_sink, n;  // keys [0, sink_end) and [lo, hi); tiles
};
template <int KT>
__device__ __forceinline__ KeyTiles key_tiles(const WinParams& p, int L, int i0) {
  KeyTiles t;
  const int last = min(i0 + 128, p.S) - 1;
  t.lo = max(0, i0 - (p.window - 1));
  t.hi = min(L, p.causal ? last + 1 : max(last + p.window, p.sinks));  // not causal: sinks may lie ahead
  t.sink_end = min(min(p.sinks, t.lo), L);
  t.n_sink = (t.sink_end + KT - 1) / KT;
  t.n = t.n_sink + (t.hi > t.lo ? (t.hi - t.lo + KT - 1) / KT : 0);
  return t;
}
// First key of tile j and its columns, rounded up to 16.
template <int KT>
__device__ __forceinline__ void key_tile(const KeyTiles& t, int j, int* j0, int* cols) {
  const bool sink = j < t.n_sink;
  *j0 = sink ? j * KT : t.lo + (j - t.n_sink) * KT;
  *cols = min(KT, ((sink ? t.sink_end : t.hi) - *j0 + 15) & ~15);
}

// What query i sees of a key tile starting at j0: bit c of the pair of words for column c.
struct Sight {
  uint32_t w[2];
};
__device__ __forceinline__ unsigned long long bits_below(int x) {
  return x <= 0 ? 0ull : (x >= 64 ? ~0ull : (1ull << x) - 1);
}
__device__ __forceinline__ Sight words(unsigned long long m) {
  Sight s;
  s.w[0] = static_cast<uint32_t>(m);
  s.w[1] = static_cast<uint32_t>(m >> 32);
  return s;
}
__device__ __forceinline__ Sight sight_of(const WinParams& p, const KeyTiles& t, int L, int i, int j, int j0) {
  // sinks below the window of every query of the tile: none is ahead of a query
  if (j < t.n_sink) return words(bits_below(t.sink_end - j0));
  const int a = i - (p.window - 1), b = min(L, p.causal ? i + 1 : i + p.window);
  const int c = min(min(p.sinks, L), p.causal ? i + 1 : L);
  return words((bits_below(b - j0) & ~bits_below(a - j0)) | bits_below(c - j0));
}

// Zeroes the rows [first, n) of a tile of `rows` rows: keys behind the end may
// hold NaN, which a weight of zero would not remove from a product.
template <int DP>
__device__ __forceinline__ void clear_rows(uint8_t* tile, int rows, int first, int n, int thread) {
  const int pieces = (n - first) * 8;
#pragma unroll
  for (int a = 0; a < DP / 64; ++a)
    for (int e = thread; e < pieces; e += 128)
      *reinterpret_cast<uint4*>(tile + a * rows * kAtom + first * kAtom + e * 16) = make_uint4(0, 0, 0, 0);
  fence_async_smem();
}

// ── forward ────────────────────────────────────────────────────────────────
template <int DP>
struct FwdCfg {
  static constexpr int KT = 64;
  static constexpr int kBufs = 2;   // score tiles: one is made while the other is worked on
  static constexpr int kSlots = 4;
  static constexpr int kSlot = KT * DP * 2;
  static constexpr int kQ = 128 * DP * 2;
  static constexpr int kSmem = kQ + kSlots * kSlot + 256 + 1024;
  static constexpr uint32_t kO = kBufs * 64;                // TMEM columns: the scores first, P over them
};

// TRAIN: leaves o_rest for the backward pass.  delta = dO . O has to be the mean of dP under weights that add up
// to one, or a weight near 1 brings its own rounding (2^-9 of dP) into a difference that is far smaller; so O for delta
// is divided by the sum of the rounded weights, which were multiplied with V, and o by that of the exact ones, as without.
template <int DP, bool TRAIN>
__global__ void __launch_bounds__(kAttnThreads, 2)
    win_fwd_sm100(const __grid_constant__ AttnMaps maps, const __grid_constant__ WinParams p, int* err) {
  using C = FwdCfg<DP>;
  constexpr int KT = C::KT;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + C::kQ;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + C::kSlots * C::kSlot);
  uint64_t* empty = full + C::kSlots;
  uint64_t* q_full = empty + C::kSlots;
  // Of each buffer its own: with one barrier for both, the scores (or weights) of
  // tile j + 1 could complete a second phase before anyone had looked at tile j's.
  uint64_t* s_full = q_full + 1;
  uint64_t* p_full = s_full + C::kBufs;
  uint64_t* pv_done = p_full + C::kBufs;  // of a tile
  uint64_t* all_done = pv_done + 1;  // of the last one
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(all_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i0 = blockIdx.x * 128, h = blockIdx.y, b = blockIdx.z, hk = h / (p.H / p.Hk);
  const int L = win_length(p, b);
  const KeyTiles kt = key_tiles<KT>(p, L, i0);
  const int kd = (p.D + 15) / 16;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 1);
    for (int i = 0; i < C::kBufs; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    mbar_init(pv_done, 1);
    mbar_init(all_done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0 && kt.n > 0) {
      mbar_arrive_expect_tx(q_full, C::kQ);
#pragma unroll
      for (int a = 0; a < DP / 64; ++a) tma_load_4d(smem + a * 128 * kAtom, &maps.q, q_full, a * 64, i0, h, b);
      int it = 0;
      bool go = true;
      for (int j = 0; j < kt.n && go; ++j) {
        int j0, cols;
        key_tile<KT>(kt, j, &j0, &cols);
        for (int kv = 0; kv < 2; ++kv, ++it) {
          const int s = it % C::kSlots;
          if (!mbar_park(&empty[s], ((it / C::kSlots) & 1) ^ 1, err, kErrTimeoutEmpty) || *abort_flag) {
            *abort_flag = 1;
            go = false;
            break;
          }
          mbar_arrive_expect_tx(&full[s], C::kSlot);
#pragma unroll
          for (int a = 0; a < DP / 64; ++a)
            tma_load_4d(ring + s * C::kSlot + a * KT * kAtom, kv ? &maps.v : &maps.k, &full[s], a * 64, j0, hk, b);
        }
      }
      mbar_park(q_full, 0, err, kErrTimeoutDrain);
      for (int i = max(0, it - C::kSlots); i < it; ++i)
        mbar_park(&full[i % C::kSlots], (i / C::kSlots) & 1, err, kErrTimeoutDrain);
    }
  } else if (warp == 1) {
    if (kt.n > 0) {
      // The whole warp keeps step, one lane issues: addresses stay in uniform registers.
      const bool issuer = elect_lane();
      const uint32_t idesc_s = make_idesc(1, 0, 0, 128, 0), idesc_o = make_idesc(1, 0, 1, 128, 16 * kd);
      const uint32_t d0 = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t q0 = desc_lo(smem_u32(smem)), k0 = desc_lo(smem_u32(ring)), v0 = desc_lo(smem_u32(ring), KT * kAtom);
      // S = Q K^T, once the product that read the weights of this buffer is over
      auto scores = [&](int j) {
        const int it = 2 * j, s = it % C::kSlots;
        int j0, cols;
        key_tile<KT>(kt, j, &j0, &cols);
        if (!warp_wait(&full[s], (it / C::kSlots) & 1, err, kErrTimeoutFull)) return false;
        if (j >= C::kBufs && !warp_wait(pv_done, (j - C::kBufs) & 1, err, kErrTimeoutEmpty)) return false;
        tc_fence_after();
        if (issuer) {
          const uint32_t buf = d0 + (j % C::kBufs) * 64, id = idesc_s | ((cols >> 3) << 17);
          const uint32_t ks = k0 + s * (C::kSlot >> 4);
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
            if (k < kd) umma_ss(buf, q0 + step_k(128, k), ks + step_k(KT, k), id, k ? 1u : 0u);
          tc_commit(&empty[s]);
          tc_commit(&s_full[j % C::kBufs]);
        }
        __syncwarp();
        return true;
      };
      bool go = warp_wait(q_full, 0, err, kErrTimeoutFull) && scores(0);
      for (int j = 0; j < kt.n && go; ++j) {
        if (j + 1 < kt.n && !(go = scores(j + 1))) break;
        const int it = 2 * j + 1, s = it % C::kSlots;
        int j0, cols;
        key_tile<KT>(kt, j, &j0, &cols);
        go = warp_wait(&full[s], (it / C::kSlots) & 1, err, kErrTimeoutFull) &&
             warp_wait(&p_full[j % C::kBufs], (j / C::kBufs) & 1, err, kErrTimeoutFull);
        if (!go) break;
        tc_fence_after();
        if (issuer) {
          const uint32_t vs = v0 + s * (C::kSlot >> 4), pa = d0 + (j % C::kBufs) * 64;
#pragma unroll
          for (int k = 0; k < KT / 16; ++k)  // O += P V
            if (k * 16 < cols) umma_ts(d0 + C::kO, pa + k * 8, vs + step_mn(k), idesc_o, (j | k) ? 1u : 0u);
          tc_commit(&empty[s]);
          tc_commit(pv_done);
          if (j + 1 == kt.n) tc_commit(all_done);
        }
        __syncwarp();
      }
      if (!go) *abort_flag = 1;
    }
  } else {
    const int q4 = warp & 3, row = q4 * 32 + lane, i = i0 + row;
    const uint32_t lanes = static_cast<uint32_t>(q4 * 32) << 16;
    const float c = p.scale * kLog2e;
    const int w0 = i0 + q4 * 32, w1 = w0 + 31;  // this warp's queries
    float m = -INFINITY;                        // in the scaled base-2 domain
    float2 l2 = make_float2(0.f, 0.f), r2 = l2;  // sums of the weights, and of the rounded ones
    bool ok = true;
    // tiles that all of this warp's queries see whole
    const int from = kt.n_sink + max(0, w1 - p.window + 1 - kt.lo + KT - 1) / KT;
    const int room = min(L, p.causal ? w0 + 1 : w0 + p.window) - kt.lo;
    const int to = room < KT ? 0 : kt.n_sink + room / KT;
    for (int j = 0; j < kt.n; ++j) {
      int j0, cols;
      key_tile<KT>(kt, j, &j0, &cols);
      const uint32_t buf = tmem + lanes + (j % C::kBufs) * 64;
      const bool whole = j >= from && j < to;
      if (!(ok = warp_wait(&s_full[j % C::kBufs], (j / C::kBufs) & 1, err, kErrTimeoutTmemFull))) break;
      tc_fence_after();
      float s[KT];
      load_row32(buf, s);
      load_row32(buf + 32, s + 32);  // a narrow tile's columns behind its end are out of sight
      tmem_ld_wait();
      if (!whole) {
        const Sight si = sight_of(p, kt, L, i, j, j0);
#pragma unroll
        for (int e = 0; e < KT; ++e) s[e] = (si.w[e >> 5] & (1u << (e & 31))) ? s[e] : -INFINITY;
      }
      float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < KT; e += 8)
#pragma unroll
        for (int u = 0; u < 4; ++u) t4[u] = max_nan(t4[u], s[e + u], s[e + u + 4]);
      float mx = max_nan(max_nan(t4[0], t4[1], t4[2]), t4[3], t4[3]) * c;
      mx = mx < INFINITY ? mx : NAN;  // a score that is NaN or infinite makes the row NaN, as its softmax is
      float f = 1.f;
      bool raise = false;
      if (m == -INFINITY) {
        m = mx;
      } else if (!(mx <= m + 8.f)) {
        f = ex2(m - mx);
        m = mx;
        l2 = mul2(l2, make_float2(f, f));
        if constexpr (TRAIN) r2 = mul2(r2, make_float2(f, f));
        raise = true;
      }
      const float base = m == -INFINITY ? 0.f : m;
      const float2 c2 = make_float2(c, c), b2 = make_float2(-base, -base);
      uint32_t pk[KT / 2];
      if (whole) {
        // Three of eight pairs of exponentials on the FMA pipe: the special-function
        // unit's 4 a cycle and scheduler are what the others wait for.
#pragma unroll
        for (int e = 0; e < KT; e += 2) {
          float2 w = fma2(make_float2(s[e], s[e + 1]), c2, b2);
          if ((e / 2) % 8 == 1 || (e / 2) % 8 == 4 || (e / 2) % 8 == 6) {
            w = ex2_poly2(w);
          } else {
            w.x = ex2(w.x);
            w.y = ex2(w.y);
          }
          l2 = add2(l2, w);
          pk[e / 2] = pack_f2(w.x, w.y);
          if constexpr (TRAIN) r2 = add_packed(r2, pk[e / 2]);
        }
      } else {
#pragma unroll
        for (int half = 0; half < 2; ++half)
          if (half * 32 < cols) {
#pragma unroll
            for (int e = half * 32; e < half * 32 + 32; e += 2) {
              float2 w = fma2(make_float2(s[e], s[e + 1]), c2, b2);
              w.x = ex2(w.x);
              w.y = ex2(w.y);
              l2 = add2(l2, w);
              pk[e / 2] = pack_f2(w.x, w.y);
              if constexpr (TRAIN) r2 = add_packed(r2, pk[e / 2]);
            }
          }
      }
      if (j > 0 && __any_sync(0xffffffffu, raise)) {
        // S_j was made after the product of tile j - 2: only that of j - 1 can be under way
        if (!(ok = warp_wait(pv_done, (j - 1) & 1, err, kErrTimeoutTmemFull))) break;
        tc_fence_after();
#pragma unroll 1
        for (int ch = 0; ch < DP / 16; ++ch) {
          uint32_t o[16];
          tmem_ld_32x32b_x16(tmem + C::kO + lanes + ch * 16, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmem_st_32x32b_x16(tmem + C::kO + lanes + ch * 16, o);
        }
      }
      if (cols > 32)
        tmem_st_32x32b_x32(buf, pk);
      else
        tmem_st_32x32b_x16(buf, pk);
      if (j0 + cols > L) {
        const int it = 2 * j + 1, sl = it % C::kSlots;
        if (!(ok = warp_wait(&full[sl], (it / C::kSlots) & 1, err, kErrTimeoutFull))) break;
        clear_rows<DP>(ring + sl * C::kSlot, KT, max(0, L - j0), cols, threadIdx.x - 64);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[j % C::kBufs]);
    }
    // not on pv_done: the tile before the last may still be under way, and its phase looks like the last one's
    if (ok && kt.n > 0) ok = warp_wait(all_done, 0, err, kErrTimeoutTmemFull);
    tc_fence_after();
    if (!ok) {
      *abort_flag = 1;
    } else {
      // Every score minus infinity: no weight (the polynomial's least value is not zero), as if nothing were in sight.
      // A row that met NaN has a sum of NaN, whatever its maximum became afterwards.
      const float sum = l2.x + l2.y;
      const bool none = m == -INFINITY && sum == sum;
      const float l = none ? 0.f : sum;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      // every product has read the queries: their tile is the staging tile now
      stage_row<DP>(smem, tmem + C::kO + lanes, kt.n > 0, inv, row);
      __syncwarp();
      const long long at = ((static_cast<long long>(b) * p.S + i0) * p.H + h) * p.D, stride = static_cast<long long>(p.H) * p.D;
      store_rows<DP>(smem, static_cast<__nv_bfloat16*>(p.o) + at, stride, p.D, q4 * 32, 0, p.S - i0, lane);
      if constexpr (TRAIN) {
        const float r = none ? 0.f : r2.x + r2.y;
        __syncwarp();  // the staging rows have been read
        stage_row<DP, true>(smem, tmem + C::kO + lanes, kt.n > 0, inv, row, r > 0.f ? 1.f / r : (r == 0.f ? 0.f : r));
        __syncwarp();
        store_rows<DP>(smem, static_cast<__nv_bfloat16*>(p.o_rest) + at, stride, p.D, q4 * 32, 0, p.S - i0, lane);
      }
      if (i < p.S)
        p.lse[(static_cast<long long>(b) * p.H + h) * p.S + i] = l == 0.f ? INFINITY : m + log2f(l);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// ── dq and delta ───────────────────────────────────────────────────────────
template <int DP>
struct DqCfg {
  static constexpr int KT = 64;
  static constexpr int kSlots = DP == 64 ? 4 : 2;
  // With one pair of slots the next tile's keys arrive only after the product that reads this tile's.
  static constexpr bool kEarly = kSlots == 4;
  static constexpr int kSlot = KT * DP * 2;
  static constexpr int kQ = 128 * DP * 2;
  static constexpr int kDs = 128 * KT * 2;                // dS as the A operand of dQ += dS K
  static constexpr int kSmem = 2 * kQ + kDs + kSlots * kSlot + 256;
  static constexpr uint32_t kDp = 64, kDq = 128;          // TMEM columns: S at 0
};

template <int DP>
__global__ void __launch_bounds__(kAttnThreads, 2)
    win_dq_sm100(const __grid_constant__ AttnMaps maps, const __grid_constant__ WinParams p, int* err) {
  using C = DqCfg<DP>;
  constexpr int KT = C::KT;
  extern __shared__ __align__(1024) uint8_t smem[];  // no slack to align it in: two CTAs fill the SM at D = 128
  if (smem_u32(smem) & 1023u) {
    record_error(err, kErrBounds);
    return;
  }
  uint8_t* ds_tile = smem + 2 * C::kQ;  // queries, dO, dS, then the ring
  uint8_t* ring = ds_tile + C::kDs;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + C::kSlots * C::kSlot);
  uint64_t* empty = full + C::kSlots;
  uint64_t* q_full = empty + C::kSlots;
  uint64_t* s_full = q_full + 1;   // S and dP
  uint64_t* s_empty = s_full + 1;
  uint64_t* ds_full = s_empty + 1;
  uint64_t* dq_done = ds_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dq_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i0 = blockIdx.x * 128, h = blockIdx.y, b = blockIdx.z, hk = h / (p.H / p.Hk);
  const int L = win_length(p, b);
  const KeyTiles kt = key_tiles<KT>(p, L, i0);
  const int kd = (p.D + 15) / 16;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(s_full, 1);
    mbar_init(s_empty, 4);
    mbar_init(ds_full, 4);
    mbar_init(dq_done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0 && kt.n > 0) {
      mbar_arrive_expect_tx(q_full, 2 * C::kQ);
#pragma unroll
      for (int a = 0; a < DP / 64; ++a) {
        tma_load_4d(smem + a * 128 * kAtom, &maps.q, q_full, a * 64, i0, h, b);
        tma_load_4d(smem + C::kQ + a * 128 * kAtom, &maps.g, q_full, a * 64, i0, h, b);
      }
      int it = 0;
      bool go = true;
      for (int j = 0; j < kt.n && go; ++j) {
        int j0, cols;
        key_tile<KT>(kt, j, &j0, &cols);
        for (int kv = 0; kv < 2; ++kv, ++it) {
          const int s = it % C::kSlots;
          if (!mbar_park(&empty[s], ((it / C::kSlots) & 1) ^ 1, err, kErrTimeoutEmpty) || *abort_flag) {
            *abort_flag = 1;
            go = false;
            break;
          }
          mbar_arrive_expect_tx(&full[s], C::kSlot);
#pragma unroll
          for (int a = 0; a < DP / 64; ++a)
            tma_load_4d(ring + s * C::kSlot + a * KT * kAtom, kv ? &maps.v : &maps.k, &full[s], a * 64, j0, hk, b);
        }
      }
      mbar_park(q_full, 0, err, kErrTimeoutDrain);
      for (int i = max(0, it - C::kSlots); i < it; ++i)
        mbar_park(&full[i % C::kSlots], (i / C::kSlots) & 1, err, kErrTimeoutDrain);
    }
  } else if (warp == 1) {
    if (kt.n > 0) {
      const bool issuer = elect_lane();
      const uint32_t idesc_s = make_idesc(1, 0, 0, 128, 0), idesc_q = make_idesc(1, 0, 1, 128, 16 * kd);
      const uint32_t d0 = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t q0 = desc_lo(smem_u32(smem)), g0 = desc_lo(smem_u32(smem) + C::kQ);
      const uint32_t a0 = desc_lo(smem_u32(ds_tile));
      const uint32_t k0 = desc_lo(smem_u32(ring)), t0 = desc_lo(smem_u32(ring), KT * kAtom);
      auto scores = [&](int j) {  // S = Q K^T, dP = dO V^T
        int j0, cols;
        key_tile<KT>(kt, j, &j0, &cols);
        const uint32_t id = idesc_s | ((cols >> 3) << 17);
        const int ik = 2 * j, iv = ik + 1, s = ik % C::kSlots, sv = iv % C::kSlots;
        if (j > 0 && !warp_wait(s_empty, (j - 1) & 1, err, kErrTimeoutEmpty)) return false;
        if (!warp_wait(&full[s], (ik / C::kSlots) & 1, err, kErrTimeoutFull)) return false;
        if (!warp_wait(&full[sv], (iv / C::kSlots) & 1, err, kErrTimeoutFull)) return false;
        tc_fence_after();
        if (issuer) {
          const uint32_t ks = k0 + s * (C::kSlot >> 4), vs = k0 + sv * (C::kSlot >> 4);
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
            if (k < kd) umma_ss(d0, q0 + step_k(128, k), ks + step_k(KT, k), id, k ? 1u : 0u);
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
            if (k < kd) umma_ss(d0 + C::kDp, g0 + step_k(128, k), vs + step_k(KT, k), id, k ? 1u : 0u);
          tc_commit(&empty[sv]);
          tc_commit(s_full);
        }
        __syncwarp();
        return true;
      };
      bool go = warp_wait(q_full, 0, err, kErrTimeoutFull) && scores(0);
      for (int j = 0; j < kt.n && go; ++j) {
        if (C::kEarly && j + 1 < kt.n && !(go = scores(j + 1))) break;
        int j0, cols;
        key_tile<KT>(kt, j, &j0, &cols);
        const int s = (2 * j) % C::kSlots;
        if (!(go = warp_wait(ds_full, j & 1, err, kErrTimeoutFull))) break;
        tc_fence_after();
        if (issuer) {
          const uint32_t ks = t0 + s * (C::kSlot >> 4);
#pragma unroll
          for (int k = 0; k < KT / 16; ++k)  // dQ += dS K
            if (k * 16 < cols) umma_ss(d0 + C::kDq, a0 + step_k(128, k), ks + step_mn(k), idesc_q, (j | k) ? 1u : 0u);
          tc_commit(&empty[s]);
          tc_commit(dq_done);
        }
        __syncwarp();
        if (!C::kEarly && j + 1 < kt.n) go = scores(j + 1);
      }
      if (!go) *abort_flag = 1;
    }
  } else {
    const int q4 = warp & 3, row = q4 * 32 + lane, i = i0 + row;
    const uint32_t lanes = static_cast<uint32_t>(q4 * 32) << 16;
    const float c = p.scale * kLog2e;
    const int w0 = i0 + q4 * 32, w1 = w0 + 31;
    const long long srow = (static_cast<long long>(b) * p.H + h) * p.S + i;
    float delta = 0.f, lse = INFINITY;
    if (i < p.S) {
      lse = p.lse[srow];
      const long long orow = ((static_cast<long long>(b) * p.S + i) * p.H + h) * p.D;
      const uint4* o = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.o) + orow);
      const uint4* rest = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.o_rest) + orow);
      const uint4* g = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.dout) + b * p.g_sb +
                                                      i * p.g_ss + h * p.g_sh);
#pragma unroll 4
      for (int d = 0; d < p.D / 8; ++d) {
        const uint4 x = o[d], z = rest[d], y = g[d];
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, zs[4] = {z.x, z.y, z.z, z.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          delta = fmaf(__uint_as_float(xs[e] << 16) + __uint_as_float(zs[e] << 16), __uint_as_float(ys[e] << 16), delta);
          delta = fmaf(__uint_as_float(xs[e] & 0xffff0000u) + __uint_as_float(zs[e] & 0xffff0000u),
                       __uint_as_float(ys[e] & 0xffff0000u), delta);
        }
      }
      p.delta[srow] = delta;
    }
    const float2 c2 = make_float2(c, c), lse2 = make_float2(-lse, -lse), delta2 = make_float2(-delta, -delta);
    const bool alone = win_alone(p, L, i);  // never a row that sees a tile whole
    // tiles that all of this warp's queries see whole
    const int from = kt.n_sink + max(0, w1 - p.window + 1 - kt.lo + KT - 1) / KT;
    const int room = min(L, p.causal ? w0 + 1 : w0 + p.window) - kt.lo;
    const int to = room < KT ? 0 : kt.n_sink + room / KT;
    bool ok = true;
    for (int j = 0; j < kt.n; ++j) {
      int j0, cols;
      key_tile<KT>(kt, j, &j0, &cols);
      if (!(ok = warp_wait(s_full, j & 1, err, kErrTimeoutTmemFull))) break;
      tc_fence_after();
      // The whole row at once, so that the next tile's scores are made under this one's arithmetic.
      float s[KT], dp[KT];
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // a narrow tile's columns behind its end are out of sight
        load_row32(tmem + lanes + half * 32, s + half * 32);
        load_row32(tmem + C::kDp + lanes + half * 32, dp + half * 32);
      }
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_empty);
      const bool whole = j >= from && j < to;
      if (kt.n == 1) {
        // The row's few keys are all here: delta from the weights themselves, without the forward's rounding of them
        // to bf16, which is seen when a row has two or three keys (dq and dk off by 2.7 against 2.4e-3).
        const Sight si = whole ? words(~0ull) : sight_of(p, kt, L, i, j, j0);
        delta = 0.f;
#pragma unroll
        for (int e = 0; e < KT; ++e) {
          const bool on = si.w[e >> 5] & (1u << (e & 31));
          s[e] = on ? ex2(fmaf(s[e], c, -lse)) : 0.f;
          dp[e] = on ? dp[e] : 0.f;
          delta = fmaf(s[e], dp[e], delta);
        }
        if (i < p.S) p.delta[srow] = delta;
#pragma unroll
        for (int e = 0; e < KT; ++e) s[e] *= alone ? 0.f : dp[e] - delta;
      } else {
#pragma unroll
        for (int e = 0; e < KT; e += 2) {
          float2 w = fma2(make_float2(s[e], s[e + 1]), c2, lse2);
          w.x = ex2(w.x);
          w.y = ex2(w.y);
          w = mul2(w, add2(make_float2(dp[e], dp[e + 1]), delta2));
          s[e] = w.x;
          s[e + 1] = w.y;
        }
        if (!whole) {
          const Sight si = sight_of(p, kt, L, i, j, j0);
#pragma unroll
          for (int e = 0; e < KT; ++e) s[e] = (si.w[e >> 5] & (1u << (e & 31))) ? s[e] : 0.f;
          if (alone) {
#pragma unroll
            for (int e = 0; e < KT; ++e) s[e] *= 0.f;
          }
        }
      }
      if (j > 0) {  // the product before has read dS
        if (!(ok = warp_wait(dq_done, (j - 1) & 1, err, kErrTimeoutTmemFull))) break;
      }
#pragma unroll
      for (int c8 = 0; c8 < KT / 8; ++c8)
        *stage_piece(ds_tile, 0, row, c8) =
            make_uint4(pack_f2(s[8 * c8], s[8 * c8 + 1]), pack_f2(s[8 * c8 + 2], s[8 * c8 + 3]),
                       pack_f2(s[8 * c8 + 4], s[8 * c8 + 5]), pack_f2(s[8 * c8 + 6], s[8 * c8 + 7]));
      if (j0 + cols > L)  // K has arrived: S was made from it
        clear_rows<DP>(ring + ((2 * j) % C::kSlots) * C::kSlot, KT, max(0, L - j0), cols, threadIdx.x - 64);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    if (ok && kt.n > 0) ok = warp_wait(dq_done, (kt.n - 1) & 1, err, kErrTimeoutTmemFull);
    tc_fence_after();
    if (!ok) {
      *abort_flag = 1;
    } else {
      stage_row<DP>(smem, tmem + C::kDq + lanes, kt.n > 0, p.scale, row);
      __syncwarp();
      __nv_bfloat16* dq = static_cast<__nv_bfloat16*>(p.dq) +
                          ((static_cast<long long>(b) * p.S + i0) * p.H + h) * p.D;
      store_rows<DP>(smem, dq, static_cast<long long>(p.H) * p.D, p.D, q4 * 32, 0, p.S - i0, lane);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// ── dk and dv ──────────────────────────────────────────────────────────────
template <int DP>
struct DkvCfg {
  static constexpr int QT = 64;
  static constexpr int kBufs = DP == 64 ? 1 : 2;  // score tiles in TMEM
  static constexpr int kSlots = 4;
  static constexpr int kSlot = QT * DP * 2;
  static constexpr int kK = 128 * DP * 2;
  static constexpr int kP = 128 * QT * 2;             // P^T, and dS^T, as A operands of dV += P^T dO, dK += dS^T Q
  static constexpr int kSmem = 2 * kK + 2 * kP + kSlots * kSlot + 2 * 2 * QT * 4 + 256 + 1024;
  static constexpr uint32_t kCols = DP == 64 ? 256 : 512;
  static constexpr uint32_t kDv = kBufs * 128, kDk = kDv + DP;  // S at 0, dP at 64 of each buffer
  static constexpr int kPerSm = DP == 64 ? 2 : 1;
};

// Parts of the sinks' gradients: [B][Hk][sink tile][1 + extra][dk, dv][rows][D] fp32.
struct SinkParts {
  float* part;
  int tiles, extra, rows;  // sink tiles, extra CTAs for each, rows kept of a tile (at most 128)
};

template <int DP>
__global__ void __launch_bounds__(kAttnThreads, DkvCfg<DP>::kPerSm)
    win_dkv_sm100(const __grid_constant__ AttnMaps maps, const __grid_constant__ WinParams p, const SinkParts sp,
                  int* err) {
  using C = DkvCfg<DP>;
  constexpr int QT = C::QT;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* p_tile = smem + 2 * C::kK;  // keys, values, P, dS, then the ring
  uint8_t* ds_tile = p_tile + C::kP;
  uint8_t* ring = ds_tile + C::kP;
  float* stat = reinterpret_cast<float*>(ring + C::kSlots * C::kSlot);  // [2][-lse, -delta][QT], one for each dO slot
  uint64_t* full = reinterpret_cast<uint64_t*>(stat + 4 * QT);
  uint64_t* empty = full + C::kSlots;
  uint64_t* k_full = empty + C::kSlots;
  uint64_t* s_full = k_full + 1;             // S and dP; of each buffer its own, as in the forward
  uint64_t* s_empty = s_full + C::kBufs;
  uint64_t* ds_full = s_empty + C::kBufs;    // P and dS
  uint64_t* d_done = ds_full + 1;            // dV and dK of an iteration
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(d_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = blockIdx.y, b = blockIdx.z, group = p.H / p.Hk;
  // the first CTAs of a head are the extra ones of its sink tiles
  const int n_extra = sp.tiles * sp.extra;
  const bool extra = static_cast<int>(blockIdx.x) < n_extra;
  const int tile = extra ? blockIdx.x / sp.extra : blockIdx.x - n_extra;
  const int j0 = tile * 128;
  const int L = win_length(p, b);
  const int kd = (p.D + 15) / 16;
  // Queries of the tile's window, [lo, hi), are the tile's own; of what is left,
  // [0, lo) (not causal) and [hi, S), each extra CTA takes a run of query tiles.
  const int lo = p.causal ? j0 : max(0, j0 - (p.window - 1));
  const int hi = min(p.S, j0 + 127 + p.window);
  const int before = p.causal ? 0 : (lo + QT - 1) / QT, after = (p.S - hi + QT - 1) / QT;
  int n, first = 0;  // iterations: query tiles x heads of the group
  int span;          // query tiles of one head
  if (extra) {
    span = before + after;
    const int all = span * group, per = (all + sp.extra - 1) / sp.extra;
    first = min(all, static_cast<int>(blockIdx.x - tile * sp.extra) * per);
    n = min(all, first + per) - first;
  } else {
    span = (hi - lo + QT - 1) / QT;
    n = span * group;
  }
  if (j0 >= L) n = 0;
  // The iterations in order: head, first query, and where that run of queries ends.
  struct Walk {
    int h, t;
  };
  Walk walk{hk * group + (span > 0 ? first / span : 0), span > 0 ? first % span : 0};
  auto next_tile = [&](int* h, int* i0, int* end) {
    *h = walk.h;
    const int t = walk.t;
    if (!extra) {
      *i0 = lo + t * QT;
      *end = hi;
    } else if (t < before) {
      *i0 = t * QT;
      *end = lo;
    } else {
      *i0 = hi + (t - before) * QT;
      *end = p.S;
    }
    if (++walk.t == span) {
      walk.t = 0;
      ++walk.h;
    }
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(&full[s], (s & 1) ? 33 : 1);  // dO's slots also wait for their rows' lse and delta
      mbar_init(&empty[s], 1);
    }
    mbar_init(k_full, 1);
    for (int i = 0; i < C::kBufs; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 4);
    }
    mbar_init(ds_full, 4);
    mbar_init(d_done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (n > 0) {
      if (lane == 0) {
        mbar_arrive_expect_tx(k_full, 2 * C::kK);
#pragma unroll
        for (int a = 0; a < DP / 64; ++a)
#pragma unroll
          for (int r = 0; r < 2; ++r) {  // the keys' map has boxes of 64 rows
            tma_load_4d(smem + (a * 128 + r * 64) * kAtom, &maps.k, k_full, a * 64, j0 + r * 64, hk, b);
            tma_load_4d(smem + C::kK + (a * 128 + r * 64) * kAtom, &maps.v, k_full, a * 64, j0 + r * 64, hk, b);
          }
      }
      int it = 0;
      bool go = true;
      for (int t = 0; t < n && go; ++t) {
        int h, i0, end;
        next_tile(&h, &i0, &end);
        // -lse and -delta of the tile's queries, two of each to a lane; -inf makes a weight of zero
        const float* ls = p.lse + (static_cast<long long>(b) * p.H + h) * p.S;
        const float* de = p.delta + (static_cast<long long>(b) * p.H + h) * p.S;
        float v[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int i = i0 + lane + 32 * u;
          v[u] = i < end ? -ls[i] : -INFINITY;
          v[2 + u] = i < end ? -de[i] : 0.f;
        }
        for (int qg = 0; qg < 2; ++qg, ++it) {
          const int s = it % C::kSlots;
          go = warp_wait(&empty[s], ((it / C::kSlots) & 1) ^ 1, err, kErrTimeoutEmpty) && !*abort_flag;
          go = __all_sync(0xffffffffu, go);
          if (!go) {
            *abort_flag = 1;
            break;
          }
          if (qg) {
            float* st = stat + (t & 1) * 2 * QT;
            st[lane] = v[0], st[lane + 32] = v[1], st[QT + lane] = v[2], st[QT + lane + 32] = v[3];
            mbar_arrive(&full[s]);
          }
          if (lane == 0) {
            mbar_arrive_expect_tx(&full[s], C::kSlot);
#pragma unroll
            for (int a = 0; a < DP / 64; ++a)
              tma_load_4d(ring + s * C::kSlot + a * QT * kAtom, qg ? &maps.g : &maps.q, &full[s], a * 64, i0, h, b);
          }
          __syncwarp();
        }
      }
      mbar_park(k_full, 0, err, kErrTimeoutDrain);
      for (int i = max(0, it - C::kSlots); i < it; ++i)
        mbar_park(&full[i % C::kSlots], (i / C::kSlots) & 1, err, kErrTimeoutDrain);
    }
  } else if (warp == 1) {
    if (n > 0) {
      const bool issuer = elect_lane();
      const uint32_t idesc_s = make_idesc(1, 0, 0, 128, QT), idesc_d = make_idesc(1, 0, 1, 128, 16 * kd);
      const uint32_t d0 = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t k0 = desc_lo(smem_u32(smem)), v0 = desc_lo(smem_u32(smem) + C::kK);
      const uint32_t q0 = desc_lo(smem_u32(ring)), t0 = desc_lo(smem_u32(ring), QT * kAtom);
      const uint32_t p0 = desc_lo(smem_u32(p_tile)), ds0 = desc_lo(smem_u32(ds_tile));
      // S^T = K Q^T and dP^T = V dO^T, once the buffer has been read
      auto scores = [&](int t) {
        const int iq = 2 * t, ig = iq + 1, s = iq % C::kSlots, sg = ig % C::kSlots;
        if (t >= C::kBufs &&
            !warp_wait(&s_empty[t % C::kBufs], (t / C::kBufs - 1) & 1, err, kErrTimeoutEmpty)) return false;
        if (!warp_wait(&full[s], (iq / C::kSlots) & 1, err, kErrTimeoutFull)) return false;
        if (!warp_wait(&full[sg], (ig / C::kSlots) & 1, err, kErrTimeoutFull)) return false;
        tc_fence_after();
        if (issuer) {
          const uint32_t buf = d0 + (t % C::kBufs) * 128;
          const uint32_t qs = q0 + s * (C::kSlot >> 4), gs = q0 + sg * (C::kSlot >> 4);
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
            if (k < kd) umma_ss(buf, k0 + step_k(128, k), qs + step_k(QT, k), idesc_s, k ? 1u : 0u);
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
            if (k < kd) umma_ss(buf + 64, v0 + step_k(128, k), gs + step_k(QT, k), idesc_s, k ? 1u : 0u);
          tc_commit(&s_full[t % C::kBufs]);
        }
        __syncwarp();
        return true;
      };
      bool go = warp_wait(k_full, 0, err, kErrTimeoutFull) && scores(0);
      for (int t = 0; t < n && go; ++t) {
        if (t + 1 < n && !(go = scores(t + 1))) break;
        if (!(go = warp_wait(ds_full, t & 1, err, kErrTimeoutFull))) break;
        tc_fence_after();
        const int s = (2 * t) % C::kSlots, sg = (2 * t + 1) % C::kSlots;
        if (issuer) {
          const uint32_t qs = t0 + s * (C::kSlot >> 4), gs = t0 + sg * (C::kSlot >> 4);
#pragma unroll
          for (int k = 0; k < QT / 16; ++k)  // dV += P^T dO
            umma_ss(d0 + C::kDv, p0 + step_k(128, k), gs + step_mn(k), idesc_d, (t | k) ? 1u : 0u);
          tc_commit(&empty[sg]);
#pragma unroll
          for (int k = 0; k < QT / 16; ++k)  // dK += dS^T Q
            umma_ss(d0 + C::kDk, ds0 + step_k(128, k), qs + step_mn(k), idesc_d, (t | k) ? 1u : 0u);
          tc_commit(&empty[s]);
          tc_commit(d_done);
        }
        __syncwarp();
      }
      if (!go) *abort_flag = 1;
    }
  } else {
    const int q4 = warp & 3, row = q4 * 32 + lane, j = j0 + row;
    const uint32_t lanes = static_cast<uint32_t>(q4 * 32) << 16;
    const float c = p.scale * kLog2e;
    const int w0 = j0 + q4 * 32, w1 = w0 + 31;
    // an extra CTA's rows behind the sinks are nobody's: their warps only keep step
    const bool idle = extra && w0 >= p.sinks;
    const bool sink = j < p.sinks, valid = j < L;
    const bool part_rows = sp.extra > 0 && tile < sp.tiles;
    const float2 c2 = make_float2(c, c);
    bool ok = true;
    for (int t = 0; t < n; ++t) {
      int h, i0, end;
      next_tile(&h, &i0, &end);
      const float* st = stat + (t & 1) * 2 * QT;
      const int ig = 2 * t + 1;
      ok = warp_wait(&s_full[t % C::kBufs], (t / C::kBufs) & 1, err, kErrTimeoutTmemFull) &&
           warp_wait(&full[ig % C::kSlots], (ig / C::kSlots) & 1, err, kErrTimeoutFull);
      if (!ok) break;
      tc_fence_after();
      const uint32_t buf = tmem + lanes + (t % C::kBufs) * 128;
      // The whole row at once, so that the next tile's scores are made under this one's arithmetic.
      float s[QT], dp[QT];
      if (!idle) {
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
          load_row32(buf + ch * 32, s + ch * 32);
          load_row32(buf + 64 + ch * 32, dp + ch * 32);
        }
        tmem_ld_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_empty[t % C::kBufs]);
      // the products before have read P and dS
      if (t > 0 && !(ok = warp_wait(d_done, (t - 1) & 1, err, kErrTimeoutTmemFull))) break;
      if (!idle) {
#pragma unroll
        for (int e = 0; e < QT; e += 4) {
          const float4 ls = *reinterpret_cast<const float4*>(st + e);
          const float4 de = *reinterpret_cast<const float4*>(st + QT + e);
          const float2 lv[2] = {make_float2(ls.x, ls.y), make_float2(ls.z, ls.w)};
          const float2 dv[2] = {make_float2(de.x, de.y), make_float2(de.z, de.w)};
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float2 w = fma2(make_float2(s[e + 2 * u], s[e + 2 * u + 1]), c2, lv[u]);
            w.x = ex2(w.x);
            w.y = ex2(w.y);
            const float2 g = mul2(w, add2(make_float2(dp[e + 2 * u], dp[e + 2 * u + 1]), dv[u]));
            s[e + 2 * u] = w.x, s[e + 2 * u + 1] = w.y;
            dp[e + 2 * u] = g.x, dp[e + 2 * u + 1] = g.y;
          }
        }
        const bool whole = !extra && w1 < L && i0 >= (p.causal ? w1 : w1 - (p.window - 1)) &&
                           i0 + QT <= w0 + p.window;
        if (!whole) {
          // queries [qa, qb) of the tile see this thread's key
          int qa, qb;
          if (extra) {
            qa = 0;
            qb = sink && valid ? QT : 0;
          } else {
            qa = (p.causal ? j : (sink ? i0 : j - (p.window - 1))) - i0;
            qb = valid ? (sink ? QT : j + p.window - i0) : 0;
          }
          const Sight seen = words(bits_below(qb) & ~bits_below(qa));
          // queries whose only key this is: the first one, ones behind the last key, or all of a window of one
          if (i0 == 0 || i0 + QT > L || p.window == 1) {
            Sight alone;
            alone.w[0] = __ballot_sync(0xffffffffu, win_alone(p, L, i0 + lane));
            alone.w[1] = __ballot_sync(0xffffffffu, win_alone(p, L, i0 + 32 + lane));
#pragma unroll
            for (int e = 0; e < QT; ++e)
              if (alone.w[e >> 5] & (1u << (e & 31))) dp[e] *= 0.f;
          }
#pragma unroll
          for (int e = 0; e < QT; ++e) {
            const bool on = seen.w[e >> 5] & (1u << (e & 31));
            s[e] = on ? s[e] : 0.f;
            dp[e] = on ? dp[e] : 0.f;
          }
        }
#pragma unroll
        for (int c8 = 0; c8 < QT / 8; ++c8) {
          const int e = 8 * c8;
          *stage_piece(p_tile, 0, row, c8) = make_uint4(pack_f2(s[e], s[e + 1]), pack_f2(s[e + 2], s[e + 3]),
                                                        pack_f2(s[e + 4], s[e + 5]), pack_f2(s[e + 6], s[e + 7]));
          *stage_piece(ds_tile, 0, row, c8) = make_uint4(pack_f2(dp[e], dp[e + 1]), pack_f2(dp[e + 2], dp[e + 3]),
                                                         pack_f2(dp[e + 4], dp[e + 5]), pack_f2(dp[e + 6], dp[e + 7]));
        }
        fence_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    if (ok && n > 0) ok = warp_wait(d_done, (n - 1) & 1, err, kErrTimeoutTmemFull);
    tc_fence_after();
    if (!ok) {
      *abort_flag = 1;
    } else {
      const uint32_t tk = tmem + lanes + C::kDk, tv = tmem + lanes + C::kDv;
      if (part_rows && w0 < p.sinks) {  // the sinks' rows, in fp32
        const int slot = extra ? 1 + static_cast<int>(blockIdx.x) - tile * sp.extra : 0;
        float* dst = sp.part + ((((static_cast<long long>(b) * p.Hk + hk) * sp.tiles + tile) * (1 + sp.extra) + slot) *
                                    2 * sp.rows + row) * p.D;
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
#pragma unroll 1
          for (int ch = 0; ch < DP / 32; ++ch) {
            float v[32];
            if (n > 0) {
              load_row32((kv ? tv : tk) + ch * 32, v);
              tmem_ld_wait();
            }
            if (!sink) continue;
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              if (ch * 32 + e >= p.D) break;
              const float f = kv ? 1.f : p.scale;
              *reinterpret_cast<float4*>(dst + static_cast<long long>(kv) * sp.rows * p.D + ch * 32 + e) =
                  n > 0 ? make_float4(v[e] * f, v[e + 1] * f, v[e + 2] * f, v[e + 3] * f)
                        : make_float4(0.f, 0.f, 0.f, 0.f);
            }
          }
        }
      }
      if (!extra) {
        const int from = part_rows ? min(128, max(0, p.sinks - j0)) : 0;
        const long long stride = static_cast<long long>(p.Hk) * p.D;
        const long long at = ((static_cast<long long>(b) * p.S + j0) * p.Hk + hk) * p.D;
        // every product has read the keys and values: their tiles are the staging tiles now
        stage_row<DP>(smem, tk, n > 0, p.scale, row);
        stage_row<DP>(smem + C::kK, tv, n > 0, 1.f, row);
        __syncwarp();
        store_rows<DP>(smem, static_cast<__nv_bfloat16*>(p.dk) + at, stride, p.D, q4 * 32, from, p.S - j0, lane);
        store_rows<DP>(smem + C::kK, static_cast<__nv_bfloat16*>(p.dv) + at, stride, p.D, q4 * 32, from, p.S - j0,
                       lane);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kCols);
  }
}

// dk and dv of the sinks from their parts, added in order.
__global__ void __launch_bounds__(128) join_sinks_kernel(const WinParams p, const SinkParts sp) {
  const int j = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const int tile = j / 128, row = j % 128;
  const long long step = 2ll * sp.rows * p.D;
  const float* src = sp.part + ((static_cast<long long>(b) * p.Hk + hk) * sp.tiles + tile) * (1 + sp.extra) * step +
                     static_cast<long long>(row) * p.D;
  const long long at = ((static_cast<long long>(b) * p.S + j) * p.Hk + hk) * p.D;
  for (int e = threadIdx.x; e < 2 * p.D; e += 128) {
    const int kv = e / p.D, d = e - kv * p.D;
    float a = 0.f;
    for (int s = 0; s <= sp.extra; ++s) a += src[s * step + static_cast<long long>(kv) * sp.rows * p.D + d];
    static_cast<__nv_bfloat16*>(kv ? p.dv : p.dk)[at + d] = __float2bfloat16(a);
  }
}

// ── host ───────────────────────────────────────────────────────────────────
CUtensorMap head_map(const void* ptr, int D, int S, int H, int B, long long ss, long long sh, long long sb, int rows) {
  // a dimension of one element may carry any stride: give it a valid one
  const uint64_t row = static_cast<uint64_t>((D + 7) / 8 * 8) * 2;
  const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(S), static_cast<uint64_t>(H),
                            static_cast<uint64_t>(B)};
  const uint64_t strides[3] = {S > 1 ? static_cast<uint64_t>(ss) * 2 : row, H > 1 ? static_cast<uint64_t>(sh) * 2 : row,
                               B > 1 ? static_cast<uint64_t>(sb) * 2 : row};
  const uint32_t box[4] = {64, static_cast<uint32_t>(rows), 1, 1};
  return tmap_bf16<4>(ptr, dims, strides, box);
}

bool tma_heads(const void* ptr, int S, int H, int B, long long ss, long long sh, long long sb) {
  auto ok = [](int n, long long s) { return n <= 1 || (s > 0 && s % 8 == 0); };
  return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && ok(S, ss) && ok(H, sh) && ok(B, sb);
}

template <typename K>
void allow_smem(K kern, int bytes, bool (&set)[64]) {
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 64 && set[dev]) return;
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) set[dev] = true;
}

AttnMaps maps_of(const WinParams& p, int q_rows, int k_rows) {
  AttnMaps m;
  m.q = head_map(p.q, p.D, p.S, p.H, p.B, p.q_ss, p.q_sh, p.q_sb, q_rows);
  m.k = head_map(p.k, p.D, p.S, p.Hk, p.B, p.k_ss, p.k_sh, p.k_sb, k_rows);
  m.v = head_map(p.v, p.D, p.S, p.Hk, p.B, p.v_ss, p.v_sh, p.v_sb, k_rows);
  m.g = p.dout ? head_map(p.dout, p.D, p.S, p.H, p.B, p.g_ss, p.g_sh, p.g_sb, q_rows) : m.q;
  return m;
}

template <int DP, bool TRAIN>
void fwd(const WinParams& p, cudaStream_t st, int* err) {
  using C = FwdCfg<DP>;
  static bool set[64] = {false};
  allow_smem(win_fwd_sm100<DP, TRAIN>, C::kSmem, set);
  win_fwd_sm100<DP, TRAIN><<<dim3((p.S + 127) / 128, p.H, p.B), kAttnThreads, C::kSmem, st>>>(maps_of(p, 128, C::KT), p, err);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <int DP>
void bwd(const WinParams& p, cudaStream_t st, int* err) {
  {
    using C = DqCfg<DP>;
    static bool set[64] = {false};
    allow_smem(win_dq_sm100<DP>, C::kSmem, set);
    win_dq_sm100<DP><<<dim3((p.S + 127) / 128, p.H, p.B), kAttnThreads, C::kSmem, st>>>(maps_of(p, 128, C::KT), p, err);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  using C = DkvCfg<DP>;
  static bool set[64] = {false};
  allow_smem(win_dkv_sm100<DP>, C::kSmem, set);
  SinkParts sp{};
  at::Tensor part;
  const int k_tiles = (p.S + 127) / 128;
  // Queries that the sinks' own tiles leave over, in CTAs of an ordinary tile's size.
  const int own = 127 + p.window + (p.causal ? 0 : p.window);
  const int sink_tiles = (p.sinks + 127) / 128;
  if (p.sinks > 0 && (p.S > 127 + p.window || (!p.causal && (sink_tiles - 1) * 128 > p.window - 1))) {
    sp.tiles = sink_tiles;
    sp.rows = std::min(p.sinks, 128);
    sp.extra = static_cast<int>(std::max(1ll, (p.S - 127ll - p.window + own - 1) / own));
    // Not one more than the last round of resident CTAs has room for, unless that is less than half of them: 12
    // extra CTAs for each of 8 heads on top of 512 start a third round (225 us), 10 fit into the second
    // (190 us).
    const long long heads = static_cast<long long>(p.B) * p.Hk;
    const long long resident = static_cast<long long>(at::cuda::getCurrentDeviceProperties()->multiProcessorCount) *
                               C::kPerSm;
    const long long own_ctas = heads * k_tiles, rounds = (own_ctas + resident - 1) / resident;
    const long long room = (rounds * resident - own_ctas) / (heads * sink_tiles);
    if (room < sp.extra && 2 * room >= sp.extra) sp.extra = static_cast<int>(room);
    sp.extra = std::min(sp.extra, std::max(1, 512 / sink_tiles));  // bounds the parts
    part = out_empty({p.B, p.Hk, sp.tiles, 1 + sp.extra, 2, sp.rows, p.D},
                     at::TensorOptions().dtype(at::kFloat).device(at::kCUDA, at::cuda::current_device()));
    sp.part = part.data_ptr<float>();
  }
  win_dkv_sm100<DP><<<dim3(k_tiles + sp.tiles * sp.extra, p.Hk, p.B), kAttnThreads, C::kSmem, st>>>(
      maps_of(p, C::QT, 64), p, sp, err);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (sp.extra > 0) {
    join_sinks_kernel<<<dim3(p.sinks, p.Hk, p.B), 128, 0, st>>>(p, sp);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
}

}  // namespace

// bf16 operands that TMA can read in place; a positive scale (the running
// maximum is taken before scaling).
bool window_sm100_takes(const WinParams& p, bool bf16) {
  return bf16 && p.D % 8 == 0 && p.scale > 0.f && reinterpret_cast<uintptr_t>(p.o) % 16 == 0 && tma_heads(p.q, p.S, p.H, p.B, p.q_ss, p.q_sh, p.q_sb) &&
         tma_heads(p.k, p.S, p.Hk, p.B, p.k_ss, p.k_sh, p.k_sb) &&
         tma_heads(p.v, p.S, p.Hk, p.B, p.v_ss, p.v_sh, p.v_sb) &&
         (!p.dout || tma_heads(p.dout, p.S, p.H, p.B, p.g_ss, p.g_sh, p.g_sb));
}

void window_sm100_fwd(const WinParams& p, cudaStream_t st, int* err) {
  const bool train = p.o_rest != nullptr;
  if (p.D <= 64)
    train ? fwd<64, true>(p, st, err) : fwd<64, false>(p, st, err);
  else
    train ? fwd<128, true>(p, st, err) : fwd<128, false>(p, st, err);
}

void window_sm100_bwd(const WinParams& p, cudaStream_t st, int* err) {
  if (p.D <= 64)
    bwd<64>(p, st, err);
  else
    bwd<128>(p, st, err);
}

}  // namespace tgcm
