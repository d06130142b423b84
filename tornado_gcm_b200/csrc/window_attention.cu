// Attention in a sliding window with a few first tokens always in sight:
// the CUDA-core kernels (any head size up to 128, bf16 or fp32) and the
// operators' host side.  bf16 problems whose shapes the tensor cores take go
// to window_attention_sm100.cu.
//
// With z_ij = q_i . k_j * scale over the keys in sight of query i:
//   m = max_j z,  l = sum_j exp(z - m),  o_i = sum_j exp(z - m) v_j / l,
//   lse_i = m + log l  (kept in base 2; a row that sees nothing: o = 0, lse = inf).
// Backward, with p_ij = exp(z_ij - lse_i) and delta_i = dO_i . O_i:
//   dv_j = sum_i p_ij dO_i,   ds_ij = p_ij (dO_i . v_j - delta_i) * scale,
//   dq_i = sum_j ds_ij k_j,   dk_j = sum_i ds_ij q_i,
// the sums over i running over every query head that shares the key head.
// delta takes O as it was before its rounding to bf16: dO . v_j - delta is a
// difference of nearly equal numbers where a row has few keys or one weight close
// to 1, and O's rounding alone, 2^-9, would be more than dS's own there.  A forward
// pass that a backward follows keeps the remainder as bf16 beside o (dq off by 2.4
// to 2.8e-3 of its norm for every window and scores up to eight times as large; from
// the rounded O 4.7e-3 at a window of 2 and 1e-2 with such scores, emulated in fp64).
//
// The work of these kernels is fp32 FMAs (2 D per pair and product); they reach
// about a sixth of that rate (2 x 875 tokens, 32 + 8 heads of 40, window 319 to
// both sides: forward 0.66 ms, dq 0.84, dk/dv 1.46), the rest is the latency of a
// step's chain of products, shuffles and exponentials.  Two rows to a thread, for
// half the shared-memory reads, took as long (0.64, 0.84, 1.50).  Four threads
// share a row (query rows forward and for dq, key rows for dk and dv) and hold its
// vectors in registers, float4 pieces dealt out in turn, so a row of the other
// side, staged in shared memory as fp32, is read as four 16-byte broadcasts per
// step.  dk and dv take every query that sees the key in one block: no atomics, so
// gradients have the same bits every time.
#include "alloc.h"
#include "sequence_ops.h"

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "common.cuh"
#include "window_attention.h"

namespace tgcm {

// window_attention_sm100.cu
bool window_sm100_takes(const WinParams& p, bool bf16);
void window_sm100_fwd(const WinParams& p, cudaStream_t st, int* err);
void window_sm100_bwd(const WinParams& p, cudaStream_t st, int* err);

namespace {

constexpr int kRows = 32;                // rows of a block
constexpr int kTile = 32;                // staged rows of the other side
constexpr int kStep = 4;                 // of them in work at once
constexpr int kWinThreads = 4 * kRows;

template <typename T>
__device__ __forceinline__ float ldw(const T* p) {
  if constexpr (std::is_same<T, float>::value)
    return *p;
  else
    return __bfloat162float(*p);
}
template <typename T>
__device__ __forceinline__ void stw(T* p, float v) {
  if constexpr (std::is_same<T, float>::value)
    *p = v;
  else
    *p = __float2bfloat16(v);
}

// The thread's share of one row: float4 pieces part, part + 4, ...
template <typename T, int N>
__device__ __forceinline__ void load_share(const T* row, int D, int part, bool on, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = 4 * (part + 4 * (i / 4)) + i % 4;
    v[i] = (on && d < D) ? ldw(row + d) : 0.f;
  }
}
// Remainders of the same values behind their rounding to T.
template <typename T, int N>
__device__ __forceinline__ void store_rest(T* row, int D, int part, bool on, const float (&v)[N], float f) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = 4 * (part + 4 * (i / 4)) + i % 4;
    const float x = v[i] * f;
    if (on && d < D) stw(row + d, x - __bfloat162float(__float2bfloat16(x)));
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_share(T* row, int D, int part, bool on, const float (&v)[N], float f) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = 4 * (part + 4 * (i / 4)) + i % 4;
    if (on && d < D) stw(row + d, v[i] * f);
  }
}

// Rows [j0, j0 + kTile) below `end` of two tensors into shared memory, zero
// elsewhere; all of a thread's loads are under way before the first is stored.
template <typename T, int DP>
__device__ __forceinline__ void stage_rows(float* sa, const T* a, long long a_stride, float* sb, const T* b,
                                           long long b_stride, int j0, int end, int D, int thread) {
  constexpr int kEach = kTile * DP / kWinThreads, kOnce = kEach <= 16 ? kEach : kEach / 2;
#pragma unroll
  for (int e0 = 0; e0 < kEach; e0 += kOnce) {
    float va[kOnce], vb[kOnce];
#pragma unroll
    for (int e = 0; e < kOnce; ++e) {
      const int at = (e0 + e) * kWinThreads + thread, j = j0 + at / DP, d = at % DP;
      const bool on = j < end && d < D;
      va[e] = on ? ldw(a + j * a_stride + d) : 0.f;
      vb[e] = on ? ldw(b + j * b_stride + d) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < kOnce; ++e) {
      sa[(e0 + e) * kWinThreads + thread] = va[e];
      sb[(e0 + e) * kWinThreads + thread] = vb[e];
    }
  }
}

// Products with kStep staged rows at once: one row's chain of FMAs and shuffles
// is latency from end to end.
template <int N, int DP>
__device__ __forceinline__ void dot_rows(const float (&a)[N], const float* rows, int part, float (&s)[kStep]) {
#pragma unroll
  for (int u = 0; u < kStep; ++u) s[u] = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 4)
#pragma unroll
    for (int u = 0; u < kStep; ++u) {
      const float4 b = *reinterpret_cast<const float4*>(rows + u * DP + 4 * (part + i));
      s[u] = fmaf(a[i], b.x, s[u]);
      s[u] = fmaf(a[i + 1], b.y, s[u]);
      s[u] = fmaf(a[i + 2], b.z, s[u]);
      s[u] = fmaf(a[i + 3], b.w, s[u]);
    }
#pragma unroll
  for (int u = 0; u < kStep; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], 1);
#pragma unroll
  for (int u = 0; u < kStep; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], 2);
}
template <int N>
__device__ __forceinline__ void axpy_share(float (&a)[N], float f, const float* row, int part) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 b = *reinterpret_cast<const float4*>(row + 4 * (part + i));
    a[i] = fmaf(f, b.x, a[i]);
    a[i + 1] = fmaf(f, b.y, a[i + 1]);
    a[i + 2] = fmaf(f, b.z, a[i + 2]);
    a[i + 3] = fmaf(f, b.w, a[i + 3]);
  }
}

// Threads of a block beside its rows: kGroups groups of 128 take the staged tiles
// in turn and join their sums at the end, in order.  (One group alone leaves most
// of a short sequence's time to the latency of tile after tile, and the keys of a
// sink meet every query of the sequence.)
template <int DP>
struct RowShape {
  static constexpr int kGroups = DP <= 32 ? 4 : 2;
  static constexpr int kTileBytes = 2 * kTile * DP * 4 + 3 * kTile * 4;
  static constexpr int kSmem = kGroups * kTileBytes;
};

__device__ __forceinline__ void group_sync(int gid) { asm volatile("bar.sync %0, 128;" ::"r"(gid + 1) : "memory"); }

// Adds up the groups' values of one array in group 0; every thread of the block calls it.
template <int N, int GROUPS>
__device__ __forceinline__ void join_groups(float (&acc)[N], float* smem, int gid, int thread) {
  __syncthreads();
  if (gid > 0) {
#pragma unroll
    for (int e = 0; e < N; ++e) smem[((gid - 1) * N + e) * kWinThreads + thread] = acc[e];
  }
  __syncthreads();
  if (gid == 0) {
#pragma unroll
    for (int o = 1; o < GROUPS; ++o)
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += smem[((o - 1) * N + e) * kWinThreads + thread];
  }
}

// Keys in sight of some query of [i0, i0 + kRows): the sinks below the window's
// first key, [0, sinks), then [lo, hi), in tiles.
struct KeyRun {
  int sinks, lo, hi, sink_tiles, tiles;
  __device__ __forceinline__ KeyRun(const WinParams& p, int L, int i0) {
    const int last = min(i0 + kRows, p.S) - 1;
    lo = max(0, i0 - (p.window - 1));
    hi = min(L, p.causal ? last + 1 : max(last + p.window, p.sinks));
    sinks = min(min(p.sinks, lo), L);
    sink_tiles = (sinks + kTile - 1) / kTile;
    tiles = sink_tiles + (hi > lo ? (hi - lo + kTile - 1) / kTile : 0);
  }
  __device__ __forceinline__ int first(int t) const { return t < sink_tiles ? t * kTile : lo + (t - sink_tiles) * kTile; }
  __device__ __forceinline__ int end(int t) const { return t < sink_tiles ? sinks : hi; }
};

template <typename T, int DP>
__global__ void __launch_bounds__(RowShape<DP>::kGroups* kWinThreads) win_fwd_kernel(const WinParams p) {
  using C = RowShape<DP>;
  constexpr int N = DP / 4;
  extern __shared__ __align__(16) float row_smem[];
  const int gid = threadIdx.x / kWinThreads, thread = threadIdx.x % kWinThreads;
  float* ks = row_smem + gid * (C::kTileBytes / 4);
  float* vs = ks + kTile * DP;
  const int part = thread & 3, r = thread >> 2;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / (p.H / p.Hk);
  const int i0 = blockIdx.x * kRows, i = i0 + r;
  const bool on = i < p.S;
  const int L = win_length(p, b);
  const T* kb = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const T* vb = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh;
  float q[N], acc[N];
  load_share<T, N>(static_cast<const T*>(p.q) + b * p.q_sb + i * p.q_ss + h * p.q_sh, p.D, part, on, q);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    q[e] *= p.scale * kLog2e;
    acc[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const KeyRun run(p, L, i0);
  for (int it = gid; it < run.tiles; it += C::kGroups) {
    const int j0 = run.first(it), end = run.end(it), n = min(kTile, end - j0);
    group_sync(gid);
    stage_rows<T, DP>(ks, kb, p.k_ss, vs, vb, p.v_ss, j0, end, p.D, thread);
    group_sync(gid);
    for (int t = 0; t < n; t += kStep) {
      float z[kStep];
      dot_rows<N, DP>(q, ks + t * DP, part, z);
      float mn = m;
#pragma unroll
      for (int u = 0; u < kStep; ++u) {  // the four threads of a row agree
        z[u] = t + u < n && win_sees(p, L, i, j0 + t + u) ? z[u] : -INFINITY;
        mn = fmaxf(mn, z[u]);
      }
      if (mn > m) {
        const float c = exp2f(m - mn);  // 0 for the row's first key
        l *= c;
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] *= c;
        m = mn;
      }
#pragma unroll
      for (int u = 0; u < kStep; ++u) {
        if (z[u] == -INFINITY) continue;  // also: a value behind the end may be NaN
        const float w = exp2f(z[u] - m);
        l += w;
        axpy_share<N>(acc, w, vs + (t + u) * DP, part);
      }
    }
  }
  // the groups' sums on one scale
  __syncthreads();
  row_smem[threadIdx.x] = m;
  __syncthreads();
  float mb = m;
#pragma unroll
  for (int o = 0; o < C::kGroups; ++o) mb = fmaxf(mb, row_smem[o * kWinThreads + thread]);
  const float f = m == -INFINITY ? 0.f : exp2f(m - mb);
  float ls[1] = {l * f};
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] *= f;
  join_groups<1, C::kGroups>(ls, row_smem, gid, thread);
  join_groups<N, C::kGroups>(acc, row_smem, gid, thread);
  if (gid > 0) return;
  l = ls[0];
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const long long orow = ((static_cast<long long>(b) * p.S + i) * p.H + h) * p.D;
  store_share<T, N>(static_cast<T*>(p.o) + orow, p.D, part, on, acc, inv);
  if constexpr (!std::is_same<T, float>::value)
    if (p.o_rest != nullptr) store_rest<T, N>(static_cast<T*>(p.o_rest) + orow, p.D, part, on, acc, inv);
  if (on && part == 0)
    p.lse[(static_cast<long long>(b) * p.H + h) * p.S + i] = l == 0.f ? INFINITY : mb + log2f(l);
}

// dq and delta; rows are queries.
template <typename T, int DP>
__global__ void __launch_bounds__(RowShape<DP>::kGroups* kWinThreads) win_dq_kernel(const WinParams p) {
  using C = RowShape<DP>;
  constexpr int N = DP / 4;
  extern __shared__ __align__(16) float row_smem[];
  const int gid = threadIdx.x / kWinThreads, thread = threadIdx.x % kWinThreads;
  float* ks = row_smem + gid * (C::kTileBytes / 4);
  float* vs = ks + kTile * DP;
  const int part = thread & 3, r = thread >> 2;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / (p.H / p.Hk);
  const int i0 = blockIdx.x * kRows, i = i0 + r;
  const bool on = i < p.S;
  const int L = win_length(p, b);
  const T* kb = static_cast<const T*>(p.k) + b * p.k_sb + hk * p.k_sh;
  const T* vb = static_cast<const T*>(p.v) + b * p.v_sb + hk * p.v_sh;
  const long long orow = ((static_cast<long long>(b) * p.S + i) * p.H + h) * p.D;
  const long long srow = (static_cast<long long>(b) * p.H + h) * p.S + i;
  float q[N], g[N], acc[N];
  load_share<T, N>(static_cast<const T*>(p.q) + b * p.q_sb + i * p.q_ss + h * p.q_sh, p.D, part, on, q);
  load_share<T, N>(static_cast<const T*>(p.dout) + b * p.g_sb + i * p.g_ss + h * p.g_sh, p.D, part, on, g);
  load_share<T, N>(static_cast<const T*>(p.o) + orow, p.D, part, on, acc);
  float delta = 0.f;
  if constexpr (!std::is_same<T, float>::value) {
    float rest[N];
    load_share<T, N>(static_cast<const T*>(p.o_rest) + orow, p.D, part, on, rest);
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] += rest[e];
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    delta = fmaf(g[e], acc[e], delta);
    q[e] *= p.scale * kLog2e;
    acc[e] = 0.f;
  }
  delta += __shfl_xor_sync(0xffffffffu, delta, 1);
  delta += __shfl_xor_sync(0xffffffffu, delta, 2);
  const float lse = on ? p.lse[srow] : INFINITY;
  const float gate = win_alone(p, L, i) ? 0.f : 1.f;
  if (on && part == 0 && gid == 0) p.delta[srow] = delta;
  const KeyRun run(p, L, i0);
  for (int it = gid; it < run.tiles; it += C::kGroups) {
    const int j0 = run.first(it), end = run.end(it), n = min(kTile, end - j0);
    group_sync(gid);
    stage_rows<T, DP>(ks, kb, p.k_ss, vs, vb, p.v_ss, j0, end, p.D, thread);
    group_sync(gid);
    for (int t = 0; t < n; t += kStep) {
      float z[kStep], dp[kStep];
      dot_rows<N, DP>(q, ks + t * DP, part, z);
      dot_rows<N, DP>(g, vs + t * DP, part, dp);
#pragma unroll
      for (int u = 0; u < kStep; ++u)
        if (t + u < n && win_sees(p, L, i, j0 + t + u))
          axpy_share<N>(acc, exp2f(z[u] - lse) * (dp[u] - delta) * gate, ks + (t + u) * DP, part);
    }
  }
  join_groups<N, C::kGroups>(acc, row_smem, gid, thread);
  if (gid > 0) return;
  store_share<T, N>(static_cast<T*>(p.dq) + orow, p.D, part, on, acc, p.scale);
}

// dk and dv; rows are keys, the staged side the queries of each head that shares them.
template <typename T, int DP>
__global__ void __launch_bounds__(RowShape<DP>::kGroups* kWinThreads) win_dkv_kernel(const WinParams p) {
  using C = RowShape<DP>;
  constexpr int N = DP / 4;
  extern __shared__ __align__(16) float row_smem[];
  const int gid = threadIdx.x / kWinThreads, thread = threadIdx.x % kWinThreads;
  float* qs = row_smem + gid * (C::kTileBytes / 4);
  float *gs = qs + kTile * DP, *ls = gs + kTile * DP, *ds = ls + kTile, *gate = ds + kTile;
  const int part = thread & 3, r = thread >> 2;
  const int hk = blockIdx.y, b = blockIdx.z, group = p.H / p.Hk;
  const int j0 = blockIdx.x * kRows, j = j0 + r;
  const int L = win_length(p, b);
  const bool on = j < L;
  float k[N], v[N], dk[N], dv[N];
  load_share<T, N>(static_cast<const T*>(p.k) + b * p.k_sb + j * p.k_ss + hk * p.k_sh, p.D, part, on, k);
  load_share<T, N>(static_cast<const T*>(p.v) + b * p.v_sb + j * p.v_ss + hk * p.v_sh, p.D, part, on, v);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    k[e] *= p.scale * kLog2e;
    dk[e] = dv[e] = 0.f;
  }
  const bool sink = j0 < p.sinks;
  const int lo = p.causal ? j0 : (sink ? 0 : max(0, j0 - (p.window - 1)));
  const int hi = j0 >= L ? 0
                         : (sink ? p.S
                                 : static_cast<int>(min(static_cast<long long>(p.S),
                                                        static_cast<long long>(j0) + kRows - 1 + p.window)));
  const int tiles = hi > lo ? (hi - lo + kTile - 1) / kTile : 0;
  for (int it = gid; it < tiles * group; it += C::kGroups) {
    const int h = hk * group + it / tiles, i0 = lo + (it % tiles) * kTile;
    const T* qb = static_cast<const T*>(p.q) + b * p.q_sb + h * p.q_sh;
    const T* gb = static_cast<const T*>(p.dout) + b * p.g_sb + h * p.g_sh;
    const long long srow = (static_cast<long long>(b) * p.H + h) * p.S;
    const int n = min(kTile, hi - i0);
    group_sync(gid);
    stage_rows<T, DP>(qs, qb, p.q_ss, gs, gb, p.g_ss, i0, hi, p.D, thread);
    if (thread < n) {
      ls[thread] = p.lse[srow + i0 + thread];
      ds[thread] = p.delta[srow + i0 + thread];
      gate[thread] = win_alone(p, L, i0 + thread) ? 0.f : 1.f;
    }
    group_sync(gid);
    for (int t = 0; t < n; t += kStep) {
      float z[kStep], dp[kStep];
      dot_rows<N, DP>(k, qs + t * DP, part, z);
      dot_rows<N, DP>(v, gs + t * DP, part, dp);
#pragma unroll
      for (int u = 0; u < kStep; ++u)
        if (t + u < n && win_sees(p, L, i0 + t + u, j)) {
          const float w = exp2f(z[u] - ls[t + u]);
          axpy_share<N>(dv, w, gs + (t + u) * DP, part);
          axpy_share<N>(dk, w * (dp[u] - ds[t + u]) * gate[t + u], qs + (t + u) * DP, part);
        }
    }
  }
  join_groups<N, C::kGroups>(dk, row_smem, gid, thread);
  join_groups<N, C::kGroups>(dv, row_smem, gid, thread);
  if (gid > 0) return;
  const bool in = j < p.S;
  const long long row = ((static_cast<long long>(b) * p.S + j) * p.Hk + hk) * p.D;
  store_share<T, N>(static_cast<T*>(p.dk) + row, p.D, part, in, dk, p.scale);
  store_share<T, N>(static_cast<T*>(p.dv) + row, p.D, part, in, dv, 1.f);
}

template <int DP, typename K>
void launch_rows(K kern, const WinParams& p, int heads, cudaStream_t st) {
  using C = RowShape<DP>;
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
  kern<<<dim3((p.S + kRows - 1) / kRows, heads, p.B), C::kGroups * kWinThreads, C::kSmem, st>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// Padded head sizes.  96 beside 128: 16 heads of 80 take 2.34 ms in rows of 96 and 3.00 in rows of 128 (2 x 875
// tokens, training); rows of 48 were slower than rows of 64 (forward 0.80 against 0.66 ms for heads of 40).
template <typename F>
void by_dim(int D, F&& f) {
  if (D <= 16)
    f(std::integral_constant<int, 16>());
  else if (D <= 32)
    f(std::integral_constant<int, 32>());
  else if (D <= 64)
    f(std::integral_constant<int, 64>());
  else if (D <= 96)
    f(std::integral_constant<int, 96>());
  else
    f(std::integral_constant<int, 128>());
}

void check_qkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t window, int64_t sinks) {
  for (const auto* t : {&q, &k, &v}) {
    TORCH_CHECK(t->is_cuda() && t->device() == q.device(), "window_attention: CUDA tensors of one device expected");
    TORCH_CHECK(t->dim() == 4, "window_attention: (batch, sequence, heads, head_dim) tensors expected");
    TORCH_CHECK(t->scalar_type() == q.scalar_type() &&
                    (t->scalar_type() == at::kBFloat16 || t->scalar_type() == at::kFloat),
                "window_attention: q, k and v share one type, bf16 or fp32");
    TORCH_CHECK(t->size(3) == 1 || t->stride(3) == 1, "window_attention: head_dim must be contiguous");
  }
  TORCH_CHECK(k.sizes() == v.sizes(), "window_attention: k and v differ in shape");
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3),
              "window_attention: q and k differ in batch, sequence or head_dim");
  TORCH_CHECK(k.size(2) >= 1 && q.size(2) % k.size(2) == 0,
              "window_attention: the query heads must be a multiple of the key heads");
  TORCH_CHECK(q.size(3) >= 1 && q.size(3) <= 128, "window_attention: head_dim 1 to 128 expected, got " + std::to_string(q.size(3)));
  TORCH_CHECK(window >= 1, "window_attention: the window must hold at least the token itself, got " + std::to_string(window));
  TORCH_CHECK(sinks >= 0, "window_attention: sinks must not be negative, got " + std::to_string(sinks));
  TORCH_CHECK(q.size(0) <= 65535 && q.size(2) <= 65535 && q.size(1) <= (1ll << 30),
              "window_attention: batch and heads up to 65535, sequences up to 2^30");
}

WinParams params_of(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t window, int64_t sinks,
                    bool causal, const c10::optional<at::Tensor>& lengths, double scale) {
  check_qkv(q, k, v, window, sinks);
  WinParams p{};
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.q_sb = q.stride(0), p.q_ss = q.stride(1), p.q_sh = q.stride(2);
  p.k_sb = k.stride(0), p.k_ss = k.stride(1), p.k_sh = k.stride(2);
  p.v_sb = v.stride(0), p.v_ss = v.stride(1), p.v_sh = v.stride(2);
  p.B = static_cast<int>(q.size(0));
  p.S = static_cast<int>(q.size(1));
  p.H = static_cast<int>(q.size(2));
  p.Hk = static_cast<int>(k.size(2));
  p.D = static_cast<int>(q.size(3));
  p.window = static_cast<int>(std::min<int64_t>(window, 1ll << 30));
  p.sinks = static_cast<int>(std::min<int64_t>(sinks, p.S));
  p.causal = causal;
  p.scale = static_cast<float>(scale);
  TORCH_CHECK(p.scale > 0.f && p.scale < INFINITY, "window_attention: the scale must be positive and finite");
  if (lengths.has_value() && lengths->defined()) {
    TORCH_CHECK(lengths->device() == q.device() && lengths->scalar_type() == at::kInt && lengths->is_contiguous() &&
                    lengths->dim() == 1 && lengths->size(0) == q.size(0),
                "window_attention: lengths must be a contiguous int32 vector of one value for each sequence");
    p.lengths = lengths->data_ptr<int>();
  }
  return p;
}

int* flag_of(const c10::optional<at::Tensor>& err) {
  return err.has_value() && err->defined() ? err->data_ptr<int>() : nullptr;
}

}  // namespace

std::vector<at::Tensor> window_attention_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                             int64_t window, int64_t sinks, bool causal,
                                             const c10::optional<at::Tensor>& lengths, double scale, bool train,
                                             const c10::optional<at::Tensor>& err) {
  WinParams p = params_of(q, k, v, window, sinks, causal, lengths, scale);
  c10::cuda::CUDAGuard guard(q.device());
  const bool bf16 = q.scalar_type() == at::kBFloat16;
  auto o = out_empty(q.sizes(), q.options());
  auto rest = train && bf16 ? out_empty(q.sizes(), q.options()) : at::Tensor();
  auto lse = out_empty({p.B, p.H, p.S}, q.options().dtype(at::kFloat));
  if (o.numel() == 0) return {o, lse, rest};
  p.o = o.data_ptr();
  p.o_rest = rest.defined() ? rest.data_ptr() : nullptr;
  p.lse = lse.data_ptr<float>();
  auto st = at::cuda::getCurrentCUDAStream();
  if (window_sm100_takes(p, bf16)) {
    window_sm100_fwd(p, st, flag_of(err));
    return {o, lse, rest};
  }
  by_dim(p.D, [&](auto dc) {
    constexpr int DP = decltype(dc)::value;
    if (bf16)
      launch_rows<DP>(win_fwd_kernel<__nv_bfloat16, DP>, p, p.H, st);
    else
      launch_rows<DP>(win_fwd_kernel<float, DP>, p, p.H, st);
  });
  return {o, lse, rest};
}

std::vector<at::Tensor> window_attention_bwd(const at::Tensor& dout, const at::Tensor& q, const at::Tensor& k,
                                             const at::Tensor& v, const at::Tensor& o, const at::Tensor& o_rest,
                                             const at::Tensor& lse, int64_t window, int64_t sinks, bool causal,
                                             const c10::optional<at::Tensor>& lengths, double scale,
                                             const c10::optional<at::Tensor>& err) {
  WinParams p = params_of(q, k, v, window, sinks, causal, lengths, scale);
  TORCH_CHECK(dout.sizes() == q.sizes() && dout.scalar_type() == q.scalar_type() && dout.device() == q.device() &&
                  (dout.size(3) == 1 || dout.stride(3) == 1),
              "window_attention backward: the gradient must match q, contiguous along head_dim");
  TORCH_CHECK(o.sizes() == q.sizes() && o.is_contiguous() && o.scalar_type() == q.scalar_type() &&
                  lse.is_contiguous() && lse.scalar_type() == at::kFloat &&
                  lse.numel() == q.size(0) * q.size(1) * q.size(2),
              "window_attention backward: o and lse must be the forward's");
  const bool bf16 = q.scalar_type() == at::kBFloat16;
  TORCH_CHECK(!bf16 || (o_rest.defined() && o_rest.sizes() == q.sizes() && o_rest.is_contiguous() &&
                        o_rest.scalar_type() == at::kBFloat16),
              "window_attention backward: the forward must have kept o's remainder");
  c10::cuda::CUDAGuard guard(q.device());
  auto dq = out_empty(q.sizes(), q.options()), dk = out_empty(k.sizes(), k.options()),
       dv = out_empty(v.sizes(), v.options());
  if (q.numel() == 0) return {dq, dk.zero_(), dv.zero_()};
  auto delta = out_empty({p.B, p.H, p.S}, lse.options());
  p.o = o.data_ptr();
  p.o_rest = bf16 ? o_rest.data_ptr() : nullptr;
  p.lse = lse.data_ptr<float>();
  p.dout = dout.data_ptr();
  p.g_sb = dout.stride(0), p.g_ss = dout.stride(1), p.g_sh = dout.stride(2);
  p.delta = delta.data_ptr<float>();
  p.dq = dq.data_ptr();
  p.dk = dk.data_ptr();
  p.dv = dv.data_ptr();
  auto st = at::cuda::getCurrentCUDAStream();
  if (window_sm100_takes(p, bf16)) {
    window_sm100_bwd(p, st, flag_of(err));
    return {dq, dk, dv};
  }
  by_dim(p.D, [&](auto dc) {
    constexpr int DP = decltype(dc)::value;
    if (bf16) {
      launch_rows<DP>(win_dq_kernel<__nv_bfloat16, DP>, p, p.H, st);
      launch_rows<DP>(win_dkv_kernel<__nv_bfloat16, DP>, p, p.Hk, st);
    } else {
      launch_rows<DP>(win_dq_kernel<float, DP>, p, p.H, st);
      launch_rows<DP>(win_dkv_kernel<float, DP>, p, p.Hk, st);
    }
  });
  return {dq, dk, dv};
}

}  // namespace tgcm
