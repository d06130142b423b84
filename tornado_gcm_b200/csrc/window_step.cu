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
// against 4 D FLOP per query head.  A group of LPK lanes covers a slot's row
// with one 16-byte vector each, so a warp reads 32 / LPK rows of K and of V
// per load, kUnroll of them in flight; the query heads that share the key
// head (up to kHeads) are all scored against the row while it is in
// registers.  Each lane group keeps its own running maximum, sum and output
// (fp32), rescaled once for kUnroll rows.  The slots of a sequence are split
// over a cluster of up to 8 blocks, because batch x key heads alone leave SMs
// idle; the blocks leave their statistics in shared memory and each combines
// its part of the outputs through distributed shared memory: one launch, no
// workspace, and a fixed order of the sums.
#include "alloc.h"

#include <ATen/ATen.h>
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
  const int hk = blockIdx.y / p.head_blocks, hb = blockIdx.y % p.head_blocks, b = blockIdx.z;
  const int group = p.H / p.Hk;
  const int h0 = hk * group + hb * p.heads_per_block;
  const int heads = min(p.heads_per_block, (hk + 1) * group - h0);
  const int at = p.lengths[b];
  const int seen = at < 0 ? 0 : (at < p.cap ? at + 1 : p.cap);
  const int window = p.cap - p.sinks;
  const int slot = at < 0 ? -1 : (at < p.cap ? at : p.sinks + (at - p.sinks) % window);
  const int per = (seen + splits - 1) / splits;
  const int s0 = min(seen, static_cast<int>(rank) * per), s1 = min(seen, s0 + per);

  const T* kn = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const T* vn = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh;
  T* kc = static_cast<T*>(p.kc) + b * p.kc_sb + hk * p.kc_sh;
  T* vc = static_cast<T*>(p.vc) + b * p.vc_sb + hk * p.vc_sh;
  // The new token is read from the inputs by whoever meets its slot, so the
  // write below races with no read.
  if (hb == 0 && slot >= s0 && slot < s1)
    for (int d = threadIdx.x; d < p.D; d += kStepThreads) {
      kc[slot * p.kc_ss + d] = kn[d];
      vc[slot * p.vc_ss + d] = vn[d];
    }

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
  cluster_sync();
  // cluster: outputs i = rank, rank + splits, ... of this block's heads
  for (int i = rank * kStepThreads + threadIdx.x; i < heads * p.D; i += splits * kStepThreads) {
    const int g = i / p.D, d = i - g * p.D;
    float mb = -INFINITY;
    for (int r = 0; r < splits; ++r) mb = fmaxf(mb, ld_peer(&blk_m[g], r));
    const float base = mb == -INFINITY ? 0.f : mb;
    float a = 0.f, t = 0.f;
    for (int r = 0; r < splits; ++r) {
      const float f = exp2f(ld_peer(&blk_m[g], r) - base);
      t = fmaf(ld_peer(&blk_l[g], r), f, t);
      a = fmaf(ld_peer(&blk_o[g][d], r), f, a);
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

template <typename T, int LPK, int G>
void launch_step(const StepParams& p, int splits, int B, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(splits, p.Hk * p.head_blocks, B);
  cfg.blockDim = dim3(kStepThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, step_kernel<T, LPK, G>, p));
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
  }
  TORCH_CHECK(k_cache.size(1) == v_cache.size(1), "window_attention_step: the caches differ in slots");
  const int64_t cap = k_cache.size(1);
  TORCH_CHECK(sinks >= 0 && sinks < cap && cap <= (1ll << 30),
              "window_attention_step: sinks must lie between 0 and the cache's slots (at least one slot is the window's)");
  TORCH_CHECK(lengths.device() == q.device() && lengths.scalar_type() == at::kInt && lengths.is_contiguous() &&
                  lengths.dim() == 1 && lengths.size(0) == B,
              "window_attention_step: lengths must be a contiguous int32 vector of one value for each sequence");
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
  p.heads_per_block = group >= 4 ? 4 : static_cast<int>(group == 3 ? 4 : group);
  p.head_blocks = static_cast<int>((group + p.heads_per_block - 1) / p.heads_per_block);
  p.vec = D % (16 / q.element_size()) == 0 && rows16(q) && rows16(k) && rows16(v) && rows16(k_cache) && rows16(v_cache);
  // Enough blocks for two waves of resident blocks, none with less than 32 slots.
  const int64_t units = B * Hk * p.head_blocks;
  int splits = 1;
  while (splits < kMaxSplits && units * splits < 148 * 8 && cap / (2 * splits) >= 32) splits *= 2;
  auto st = at::cuda::getCurrentCUDAStream();
  TORCH_CHECK(p.Hk * static_cast<int64_t>(p.head_blocks) <= 65535, "window_attention_step: too many heads");
  if (q.scalar_type() == at::kBFloat16)
    by_lanes<__nv_bfloat16>(p, splits, static_cast<int>(B), st);
  else
    by_lanes<float>(p, splits, static_cast<int>(B), st);
  return o;
}

}  // namespace tgcm

TORCH_LIBRARY_FRAGMENT(tgcm, m) {
  m.def("window_attention_step(Tensor q, Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor lengths, "
        "int sinks, float scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(tgcm, CUDA, m) { m.impl("window_attention_step", &tgcm::window_attention_step); }
