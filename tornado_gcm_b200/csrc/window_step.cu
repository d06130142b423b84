// One new token of every sequence: its key and value are put in the cache and
// its query attends to what the cache then holds.
//
// The cache keeps the first `sinks` tokens and the last `window` others:
// token t lives in slot t while t < sinks + window and in slot
// sinks + (t - sinks) mod window from then on, so a new token overwrites the
// one that leaves its window and every occupied slot is in sight.  The order
// of the slots does not matter to a softmax.
//
// Bound by reading the cache once: 2 D values for each slot and key head
// against 4 D FLOP per query head; the query heads that share a key head are
// scored together while its rows are on the SM.  bf16 rows go through warp matrix
// instructions (step_mma_kernel); fp32 ones, and head sizes off 8, through
// step_kernel: a group of LPK lanes covers a slot's row with one 16-byte vector
// each, a warp reads 32 / LPK rows of K and of V per load, kUnroll of them in
// flight, and each lane group keeps its own running maximum, sum and output,
// rescaled once for kUnroll rows.  The slots of a sequence are split
// over a cluster of up to 8 blocks, because batch x key heads alone leave SMs
// idle; the blocks leave their statistics in shared memory and each combines
// its part of the outputs through distributed shared memory: one launch, no
// workspace, and a fixed order of the sums.
#include "alloc.h"
#include "sequence_ops.h"

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "common.cuh"
#include "window_attention.h"

namespace tgcm {
namespace {

constexpr int kStepThreads = 128;
constexpr int kStepWarps = kStepThreads / 32;
constexpr int kUnroll = 4;
constexpr int kMaxSplits = 8;  // portable cluster size

struct StepParams {
  const void *q, *k, *v;   // (B, H, D), (B, Hk, D): unit stride along D
  long long q_sb, q_sh, k_sb, k_sh, v_sb, v_sh;
  void *kc, *vc;           // (B, cap, Hk, D)
  long long kc_sb, kc_ss, kc_sh, vc_sb, vc_ss, vc_sh;
  const int* lengths;      // tokens before the new one; negative: the sequence takes no part
  void* o;                 // (B, H, D) contiguous
  int H, Hk, D, cap, sinks, heads_per_block, head_blocks;
  float scale;
  bool vec;                // every row is a run of whole 16-byte vectors
};

template <typename T, int V>
__device__ __forceinline__ uint4 load_vec(const T* row, int d0, int D, bool on, bool vec) {
  if (!on) return make_uint4(0, 0, 0, 0);
  if (vec) return *reinterpret_cast<const uint4*>(row + d0);
  uint4 u = make_uint4(0, 0, 0, 0);
  T* t = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (d0 + e < D) t[e] = row[d0 + e];
  return u;
}

template <typename T, int V>
__device__ __forceinline__ void widen(const uint4& u, float (&v)[V]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (V == 4) {
      v[i] = __uint_as_float(w[i]);
    } else {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_peer(const float* p, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// Outputs of the cluster's blocks joined: statistics and unnormalised outputs of
// every block lie in its shared memory, each block finishes its share of them.
template <typename T>
__device__ __forceinline__ void join_cluster(const StepParams& p, int b, int h0, int heads, uint32_t rank, int splits,
                                             const float* blk_m, const float* blk_l, const float* blk_o, int o_ld) {
  cluster_sync();
  for (int i = rank * kStepThreads + threadIdx.x; i < heads * p.D; i += splits * kStepThreads) {
    const int g = i / p.D, d = i - g * p.D;
    float mb = -INFINITY;
    for (int r = 0; r < splits; ++r) mb = fmaxf(mb, ld_peer(blk_m + g, r));
    const float base = mb == -INFINITY ? 0.f : mb;
    float a = 0.f, t = 0.f;
    for (int r = 0; r < splits; ++r) {
      const float f = exp2f(ld_peer(blk_m + g, r) - base);
      t = fmaf(ld_peer(blk_l + g, r), f, t);
      a = fmaf(ld_peer(blk_o + g * o_ld + d, r), f, a);
    }
    const float out = t == 0.f ? 0.f : a / t;
    T* o = static_cast<T*>(p.o) + (static_cast<long long>(b) * p.H + h0 + g) * p.D + d;
    if constexpr (std::is_same<T, float>::value)
      *o = out;
    else
      *o = __float2bfloat16(out);
  }
  cluster_sync();  // nobody leaves while its shared memory is read
}

// What a block works on.
struct StepShare {
  int hk, hb, b, h0, heads, slot, s0, s1;
};
__device__ __forceinline__ StepShare step_share(const StepParams& p, uint32_t rank, int splits) {
  StepShare w;
  w.hk = blockIdx.y / p.head_blocks, w.hb = blockIdx.y % p.head_blocks, w.b = blockIdx.z;
  const int group = p.H / p.Hk;
  w.h0 = w.hk * group + w.hb * p.heads_per_block;
  w.heads = min(p.heads_per_block, (w.hk + 1) * group - w.h0);
  const int at = p.lengths[w.b];
  const int seen = at < 0 ? 0 : (at < p.cap ? at + 1 : p.cap);
  const int window = p.cap - p.sinks;
  w.slot = at < 0 ? -1 : (at < p.cap ? at : p.sinks + (at - p.sinks) % window);
  const int per = (seen + splits - 1) / splits;
  w.s0 = min(seen, static_cast<int>(rank) * per), w.s1 = min(seen, w.s0 + per);
  return w;
}

// The new token goes to its slot.  Whoever meets that slot reads the inputs
// instead, so this write races with no read.
template <typename T>
__device__ __forceinline__ void put_token(const StepParams& p, const StepShare& w, const T* kn, const T* vn, T* kc,
                                          T* vc) {
  if (w.hb == 0 && w.slot >= w.s0 && w.slot < w.s1)
    for (int d = threadIdx.x; d < p.D; d += kStepThreads) {
      kc[w.slot * p.kc_ss + d] = kn[d];
      vc[w.slot * p.vc_ss + d] = vn[d];
    }
}

// ── bf16, D a multiple of 8: warp matrix instructions ──────────────────────
// A warp takes 16 slots at a time: S (16 heads x 16 slots) = q K^T and
// O (16 heads x D) += P V, up to 8 of the 16 head rows in use.  One token's few
// query heads cannot fill a tcgen05 tile (128 rows), and the kernel is bound by
// the cache's bytes; the warp instructions take a fifth of the issue slots that
// fp32 arithmetic on the same rows took (256 sequences of up to 1464 slots,
// 16 + 4 heads of 64: 113 us before).  Slots arrive by 16-byte asynchronous copies
// into the warp's own ring of kStages groups (two: more blocks to an SM do better than
// deeper rings, 59 us against 62 with three and 71 with four); rows are padded by 16 bytes so
// that the eight rows of a matrix load lie in different banks.  P enters the
// second product as two bf16 terms (value and remainder): its rounding would
// otherwise be as large as the output's own.  Heads are filled up to 16 with zeros.
constexpr int kStages = 2;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;  // 0: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void ldm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// C (16 x 8) += A (16 x 16) B (16 x 8); rows 8-15 of A are zero.
__device__ __forceinline__ void mma_8rows(float (&c)[4], uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, {%0, %1, %2, "
      "%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(0u), "r"(a2), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int ND>
struct MmaStep {
  static constexpr int kRow = ND * 32 + 16;            // bytes of a padded row
  static constexpr int kGroup = 2 * 16 * kRow;         // K and V of 16 slots
  static constexpr int kWarp = kStages * kGroup;
  static constexpr int kOut = (kStepWarps + 1) * 8 * ND * 16 * 4;  // outputs of the warps and of the block, over the rings
  static constexpr int kSmem = kStepWarps * kWarp > kOut ? kStepWarps * kWarp : kOut;
};

template <int ND>
__global__ void __launch_bounds__(kStepThreads) step_mma_kernel(const __grid_constant__ StepParams p) {
  using C = MmaStep<ND>;
  using T = __nv_bfloat16;
  constexpr int D = ND * 16;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float sm_m[kStepWarps][8], sm_l[kStepWarps][8], blk_m[8], blk_l[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t rank = cluster_rank();
  const int splits = gridDim.x;
  const StepShare w = step_share(p, rank, splits);
  const T* kn = static_cast<const T*>(p.k) + w.b * p.k_sb + w.hk * p.k_sh;
  const T* vn = static_cast<const T*>(p.v) + w.b * p.v_sb + w.hk * p.v_sh;
  T* kc = static_cast<T*>(p.kc) + w.b * p.kc_sb + w.hk * p.kc_sh;
  T* vc = static_cast<T*>(p.vc) + w.b * p.vc_sb + w.hk * p.vc_sh;
  put_token<T>(p, w, kn, vn, kc, vc);

  const uint32_t my = smem_u32(ring) + warp * C::kWarp;
  const int groups = w.s1 > w.s0 + warp * 16 ? (w.s1 - w.s0 - warp * 16 + kStepWarps * 16 - 1) / (kStepWarps * 16) : 0;
  auto fetch = [&](int i) {  // group i of this warp; an empty commit behind the last one keeps the count
    if (i < groups) {
      const int j0 = w.s0 + (warp + i * kStepWarps) * 16;
      const uint32_t dst = my + (i % kStages) * C::kGroup;
#pragma unroll
      for (int e = lane; e < 16 * 2 * ND; e += 32) {
        const int r = e / (2 * ND), c = e % (2 * ND), j = j0 + r;
        const bool on = j < w.s1 && c * 8 < p.D;
        const int js = on ? j : w.s0;
        const T* ks = js == w.slot ? kn : kc + js * p.kc_ss;
        const T* vs = js == w.slot ? vn : vc + js * p.vc_ss;
        const int d = on ? c * 8 : 0;
        cp_async16(dst + r * C::kRow + c * 16, ks + d, on);
        cp_async16(dst + 16 * C::kRow + r * C::kRow + c * 16, vs + d, on);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);

  uint32_t qa[ND][2];
  {
    const T* qr = static_cast<const T*>(p.q) + w.b * p.q_sb + (w.h0 + (g < w.heads ? g : 0)) * p.q_sh;
#pragma unroll
    for (int s = 0; s < ND; ++s)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        qa[s][u] = g < w.heads && s * 16 + u * 8 < p.D
                       ? *reinterpret_cast<const uint32_t*>(qr + s * 16 + u * 8 + 2 * t) : 0u;
  }
  const float sc = p.scale * kLog2e;
  float o[2 * ND][4];
#pragma unroll
  for (int i = 0; i < 2 * ND; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m = -INFINITY, l = 0.f;  // of head g; l of this lane's slots
  // Lane's row and column of a matrix load: K's four matrices are (slots 0-7, d 0-7), (0-7, 8-15), (8-15, 0-7),
  // (8-15, 8-15); V's, transposed on the way, (slots 0-7, d 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15).
  const uint32_t k_at = ((lane & 7) + ((lane >> 4) << 3)) * C::kRow + ((lane >> 3) & 1) * 16;
  const uint32_t v_at = 16 * C::kRow + ((lane & 7) + (((lane >> 3) & 1) << 3)) * C::kRow + (lane >> 4) * 16;

  for (int i = 0; i < groups; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();  // group i of every lane has landed, and group i - 1 has been read by all
    fetch(i + kStages - 1);
    const uint32_t at = my + (i % kStages) * C::kGroup;
    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < ND; ++s) {
      uint32_t k[4];
      ldm_x4(k, at + k_at + s * 32);
      mma_8rows(s0, qa[s][0], qa[s][1], k[0], k[1]);
      mma_8rows(s1, qa[s][0], qa[s][1], k[2], k[3]);
    }
    const int j = w.s0 + (warp + i * kStepWarps) * 16 + 2 * t;
    float z[4] = {s0[0] * sc, s0[1] * sc, s1[0] * sc, s1[1] * sc};
    if (j + 10 > w.s1) {  // the last group
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j + (e >> 1) * 8 + (e & 1) >= w.s1) z[e] = -INFINITY;
    }
    float mx = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    if (__any_sync(0xffffffffu, mx > m)) {
      const float mn = fmaxf(m, mx);
      const float f = mn == -INFINITY ? 1.f : exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int n = 0; n < 2 * ND; ++n) {
        o[n][0] *= f;
        o[n][1] *= f;
      }
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = exp2f(z[e] - base);
    l += (z[0] + z[1]) + (z[2] + z[3]);
    const uint32_t p0 = pack_pair(z[0], z[1]), p2 = pack_pair(z[2], z[3]);
    const uint32_t r0 = pack_pair(z[0] - __uint_as_float(p0 << 16), z[1] - __uint_as_float(p0 & 0xffff0000u));
    const uint32_t r2 = pack_pair(z[2] - __uint_as_float(p2 << 16), z[3] - __uint_as_float(p2 & 0xffff0000u));
#pragma unroll
    for (int s = 0; s < ND; ++s) {
      uint32_t v[4];
      ldm_x4_t(v, at + v_at + s * 32);
      mma_8rows(o[2 * s], p0, p2, v[0], v[1]);
      mma_8rows(o[2 * s], r0, r2, v[0], v[1]);
      mma_8rows(o[2 * s + 1], p0, p2, v[2], v[3]);
      mma_8rows(o[2 * s + 1], r0, r2, v[2], v[3]);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  if (t == 0) {
    sm_m[warp][g] = m;
    sm_l[warp][g] = l;
  }
  __syncthreads();  // statistics are there, and the rings are free
  float mb = -INFINITY;
#pragma unroll
  for (int v = 0; v < kStepWarps; ++v) mb = fmaxf(mb, sm_m[v][g]);
  const float base = mb == -INFINITY ? 0.f : mb;
  const float f = exp2f(m - base);
  float* outs = reinterpret_cast<float*>(ring);  // [warp][head][D], then the block's [head][D]
#pragma unroll
  for (int n = 0; n < 2 * ND; ++n)
    *reinterpret_cast<float2*>(outs + (warp * 8 + g) * D + n * 8 + 2 * t) = make_float2(o[n][0] * f, o[n][1] * f);
  if (warp == 0 && t == 0) {
    float lb = 0.f;
#pragma unroll
    for (int v = 0; v < kStepWarps; ++v) lb += sm_l[v][g] * exp2f(sm_m[v][g] - base);
    blk_m[g] = mb;
    blk_l[g] = lb;
  }
  __syncthreads();
  float* blk_o = outs + kStepWarps * 8 * D;
  for (int i = threadIdx.x; i < 8 * D; i += kStepThreads) {
    float a = 0.f;
#pragma unroll
    for (int v = 0; v < kStepWarps; ++v) a += outs[v * 8 * D + i];
    blk_o[i] = a;
  }
  join_cluster<T>(p, w.b, w.h0, w.heads, rank, splits, blk_m, blk_l, blk_o, D);
}

// ── any type and head size: fp32 arithmetic ────────────────────────────────
template <typename T, int LPK, int G>
__global__ void __launch_bounds__(kStepThreads) step_kernel(const __grid_constant__ StepParams p) {
  constexpr int V = 16 / sizeof(T);
  constexpr int ROWS = 32 / LPK;             // slots of a warp's load
  constexpr int SETS = kStepWarps * ROWS;    // lane groups of the block
  constexpr int DP = LPK * V;
  __shared__ float sm_m[SETS][G], sm_l[SETS][G];
  __shared__ float sm_acc[kStepWarps][G][DP];
  __shared__ float blk_m[G], blk_l[G], blk_o[G][DP];

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane % LPK, sub = lane / LPK, set = warp * ROWS + sub;
  const int d0 = l * V;
  const bool live = d0 < p.D;
  const uint32_t rank = cluster_rank();
  const int splits = gridDim.x;              // the cluster spans the grid's x
  const StepShare w = step_share(p, rank, splits);
  const int hk = w.hk, b = w.b, h0 = w.h0, heads = w.heads, slot = w.slot, s0 = w.s0, s1 = w.s1;
  const T* kn = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const T* vn = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh;
  T* kc = static_cast<T*>(p.kc) + b * p.kc_sb + hk * p.kc_sh;
  T* vc = static_cast<T*>(p.vc) + b * p.vc_sb + hk * p.vc_sh;
  put_token<T>(p, w, kn, vn, kc, vc);

  float q[G][V], acc[G][V], m[G], z[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const T* qr = static_cast<const T*>(p.q) + b * p.q_sb + (h0 + g) * p.q_sh;
    widen<T, V>(load_vec<T, V>(qr, d0, p.D, live && g < heads, p.vec), q[g]);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      q[g][e] *= p.scale * kLog2e;
      acc[g][e] = 0.f;
    }
    m[g] = -INFINITY;
    z[g] = 0.f;
  }
  for (int j0 = s0 + set; j0 < s1 + set; j0 += SETS * kUnroll) {  // the same count for every group of a warp
    uint4 ku[kUnroll], vu[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int j = j0 + u * SETS;
      const bool on = live && j < s1;
      ku[u] = load_vec<T, V>(j == slot ? kn : kc + j * p.kc_ss, d0, p.D, on, p.vec);
      vu[u] = load_vec<T, V>(j == slot ? vn : vc + j * p.vc_ss, d0, p.D, on, p.vec);
    }
    float s[kUnroll][G];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float kv[V];
      widen<T, V>(ku[u], kv);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float t = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) t = fmaf(q[g][e], kv[e], t);
#pragma unroll
        for (int o = LPK / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        s[u][g] = j0 + u * SETS < s1 ? t : -INFINITY;
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float mn = m[g];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) mn = fmaxf(mn, s[u][g]);
      const float base = mn == -INFINITY ? 0.f : mn;
      const float c = exp2f(m[g] - base);
      m[g] = mn;
      z[g] *= c;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[g][e] *= c;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        s[u][g] = exp2f(s[u][g] - base);
        z[g] += s[u][g];
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float vv[V];
      widen<T, V>(vu[u], vv);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[g][e] = fmaf(s[u][g], vv[e], acc[g][e]);
    }
  }

  // block: statistics of every lane group, then its outputs on one scale
  if (l == 0) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      sm_m[set][g] = m[g];
      sm_l[set][g] = z[g];
    }
  }
  __syncthreads();
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float mb = -INFINITY;
    for (int t = 0; t < SETS; ++t) mb = fmaxf(mb, sm_m[t][g]);
    const float base = mb == -INFINITY ? 0.f : mb;
    const float f = exp2f(m[g] - base);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float a = acc[g][e] * f;
#pragma unroll
      for (int o = LPK; o < 32; o <<= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
      if (sub == 0) sm_acc[warp][g][d0 + e] = a;
    }
    if (threadIdx.x == 0) {
      float lb = 0.f;
      for (int t = 0; t < SETS; ++t) lb += sm_l[t][g] * exp2f(sm_m[t][g] - base);
      blk_m[g] = mb;
      blk_l[g] = lb;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * DP; i += kStepThreads) {
    const int g = i / DP, d = i % DP;
    float a = 0.f;
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) a += sm_acc[w][g][d];
    blk_o[g][d] = a;
  }
  join_cluster<T>(p, b, h0, heads, rank, splits, blk_m, blk_l, &blk_o[0][0], DP);
}

template <typename K>
void launch_cluster(K kern, const StepParams& p, int splits, int B, size_t smem, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(splits, p.Hk * p.head_blocks, B);
  cfg.blockDim = dim3(kStepThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
}

template <typename T, int LPK, int G>
void launch_step(const StepParams& p, int splits, int B, cudaStream_t st) {
  launch_cluster(step_kernel<T, LPK, G>, p, splits, B, 0, st);
}

template <int ND>
void launch_mma(const StepParams& p, int splits, int B, cudaStream_t st) {
  static bool set[64] = {false};
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev >= 64 || !set[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(step_mma_kernel<ND>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        MmaStep<ND>::kSmem));
    if (dev < 64) set[dev] = true;
  }
  launch_cluster(step_mma_kernel<ND>, p, splits, B, MmaStep<ND>::kSmem, st);
}

template <typename T, int LPK>
void by_heads(const StepParams& p, int splits, int B, cudaStream_t st) {
  switch (p.heads_per_block) {
    case 1: launch_step<T, LPK, 1>(p, splits, B, st); break;
    case 2: launch_step<T, LPK, 2>(p, splits, B, st); break;
    default: launch_step<T, LPK, 4>(p, splits, B, st); break;
  }
}

template <typename T>
void by_lanes(const StepParams& p, int splits, int B, cudaStream_t st) {
  const int lanes = (p.D + 16 / static_cast<int>(sizeof(T)) - 1) / (16 / static_cast<int>(sizeof(T)));
  if (lanes <= 2)
    by_heads<T, 2>(p, splits, B, st);
  else if (lanes <= 4)
    by_heads<T, 4>(p, splits, B, st);
  else if (lanes <= 8)
    by_heads<T, 8>(p, splits, B, st);
  else if (lanes <= 16)
    by_heads<T, 16>(p, splits, B, st);
  else
    by_heads<T, 32>(p, splits, B, st);
}

bool rows16(const at::Tensor& t) {
  bool ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) == 1 || (t.stride(i) * t.element_size()) % 16 == 0);
  return ok;
}

}  // namespace

at::Tensor window_attention_step(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor& k_cache,
                                 at::Tensor& v_cache, const at::Tensor& lengths, int64_t sinks, double scale) {
  for (const auto* t : {&q, &k, &v}) {
    TORCH_CHECK(t->is_cuda() && t->device() == q.device() && t->dim() == 3 &&
                    t->scalar_type() == q.scalar_type() &&
                    (t->scalar_type() == at::kBFloat16 || t->scalar_type() == at::kFloat),
                "window_attention_step: q, k and v must be (batch, heads, head_dim) CUDA tensors of one type, bf16 or fp32");
    TORCH_CHECK(t->size(2) == 1 || t->stride(2) == 1, "window_attention_step: head_dim must be contiguous");
  }
  const int64_t B = q.size(0), H = q.size(1), D = q.size(2), Hk = k.size(1);
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == B && k.size(2) == D,
              "window_attention_step: k and v must match q in batch and head_dim");
  TORCH_CHECK(Hk >= 1 && H % Hk == 0, "window_attention_step: the query heads must be a multiple of the key heads");
  TORCH_CHECK(D >= 1 && D <= 128, "window_attention_step: head_dim 1 to 128 expected, got " + std::to_string(D));
  for (const auto* t : {&k_cache, &v_cache}) {
    TORCH_CHECK(t->device() == q.device() && t->scalar_type() == q.scalar_type() && t->dim() == 4 &&
                    t->size(0) == B && t->size(2) == Hk && t->size(3) == D && (D == 1 || t->stride(3) == 1),
                "window_attention_step: the caches must be (batch, sinks + window, key heads, head_dim) of q's type");
    at::assert_no_internal_overlap(*t);  // sequences would overwrite each other's slots
  }
  TORCH_CHECK(k_cache.size(1) == v_cache.size(1), "window_attention_step: the caches differ in slots");
  const int64_t cap = k_cache.size(1);
  TORCH_CHECK(sinks >= 0 && sinks < cap && cap <= (1ll << 30),
              "window_attention_step: sinks must lie between 0 and the cache's slots (at least one slot is the window's)");
  TORCH_CHECK(lengths.device() == q.device() && lengths.scalar_type() == at::kInt && lengths.is_contiguous() &&
                  lengths.dim() == 1 && lengths.size(0) == B,
              "window_attention_step: lengths must be a contiguous int32 vector of one value for each sequence");
  TORCH_CHECK(static_cast<float>(scale) > 0.f && static_cast<float>(scale) < INFINITY,
              "window_attention_step: the scale must be positive and finite");
  TORCH_CHECK(B <= 65535 && H <= 65535, "window_attention_step: batch and heads up to 65535");
  c10::cuda::CUDAGuard guard(q.device());
  auto o = out_empty({B, H, D}, q.options());
  if (o.numel() == 0) return o;
  StepParams p{};
  p.q = q.data_ptr(), p.k = k.data_ptr(), p.v = v.data_ptr();
  p.q_sb = q.stride(0), p.q_sh = q.stride(1);
  p.k_sb = k.stride(0), p.k_sh = k.stride(1);
  p.v_sb = v.stride(0), p.v_sh = v.stride(1);
  p.kc = k_cache.data_ptr(), p.vc = v_cache.data_ptr();
  p.kc_sb = k_cache.stride(0), p.kc_ss = k_cache.stride(1), p.kc_sh = k_cache.stride(2);
  p.vc_sb = v_cache.stride(0), p.vc_ss = v_cache.stride(1), p.vc_sh = v_cache.stride(2);
  p.lengths = lengths.data_ptr<int>();
  p.o = o.data_ptr();
  p.H = static_cast<int>(H), p.Hk = static_cast<int>(Hk), p.D = static_cast<int>(D);
  p.cap = static_cast<int>(cap), p.sinks = static_cast<int>(sinks);
  p.scale = static_cast<float>(scale);
  const int64_t group = H / Hk;
  p.vec = D % (16 / q.element_size()) == 0 && rows16(q) && rows16(k) && rows16(v) && rows16(k_cache) && rows16(v_cache);
  // Rows of whole 16-byte pieces of bf16 go to the matrix instructions, the rest to fp32 arithmetic.
  const bool mma = q.scalar_type() == at::kBFloat16 && p.vec;
  const int64_t most = mma ? 8 : 4;
  p.heads_per_block = static_cast<int>(mma ? std::min(group, most) : (group >= 3 ? 4 : group));
  p.head_blocks = static_cast<int>((group + p.heads_per_block - 1) / p.heads_per_block);
  // Enough blocks to fill the SMs with the last of them short, none with less than 32 slots (64 for the matrix
  // kernel: 16 to a warp).  1024 units of up to 1464 slots: 64 us whole, 59 us in halves, more in quarters.
  const int64_t units = B * Hk * p.head_blocks;
  int splits = 1;
  while (splits < kMaxSplits && units * splits < 148 * 8 && cap / (2 * splits) >= (mma ? 64 : 32)) splits *= 2;
  auto st = at::cuda::getCurrentCUDAStream();
  TORCH_CHECK(p.Hk * static_cast<int64_t>(p.head_blocks) <= 65535, "window_attention_step: too many heads");
  const int nb = static_cast<int>(B);
  if (mma)
    switch ((D + 15) / 16) {
      case 1: launch_mma<1>(p, splits, nb, st); break;
      case 2: launch_mma<2>(p, splits, nb, st); break;
      case 3: launch_mma<3>(p, splits, nb, st); break;
      case 4: launch_mma<4>(p, splits, nb, st); break;
      case 5: launch_mma<5>(p, splits, nb, st); break;
      case 6: launch_mma<6>(p, splits, nb, st); break;
      case 7: launch_mma<7>(p, splits, nb, st); break;
      default: launch_mma<8>(p, splits, nb, st); break;
    }
  else if (q.scalar_type() == at::kBFloat16)
    by_lanes<__nv_bfloat16>(p, splits, nb, st);
  else
    by_lanes<float>(p, splits, nb, st);
  return o;
}

}  // namespace tgcm

TORCH_LIBRARY_FRAGMENT(tgcm, m) {
  m.def("window_attention_step(Tensor q, Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor lengths, "
        "int sinks, float scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(tgcm, CUDA, m) { m.impl("window_attention_step", &tgcm::window_attention_step); }
