// Shared declarations of the window-attention kernels.
//
// Query i and key j of one sequence with L valid keys see each other when
//   j < L,  j <= i (causal),  and  |i - j| < window  or  j < sinks.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace tgcm {

constexpr float kLog2e = 1.4426950408889634f;

struct WinParams {
  const void *q, *k, *v;         // (B, S, heads, D), unit stride along D
  long long q_sb, q_ss, q_sh;    // element strides
  long long k_sb, k_ss, k_sh;
  long long v_sb, v_ss, v_sh;
  void* o;                       // (B, S, H, D) contiguous
  void* o_rest;                  // bf16, o's shape: what o lacks of O after its rounding; null unless a backward follows
  float* lse;                    // (B, H, S): log2 of the softmax sum, +inf for rows that see nothing
  // backward
  const void* dout;              // (B, S, H, D), unit stride along D
  long long g_sb, g_ss, g_sh;
  float* delta;                  // (B, H, S): sum_d dO O, with O = o + o_rest
  void *dq, *dk, *dv;            // contiguous, shapes of q, k, v
  const int* lengths;            // (B,) or null
  int B, S, H, Hk, D;
  int window, sinks, causal;
  float scale;
};

#ifdef __CUDACC__
__device__ __forceinline__ int win_length(const WinParams& p, int b) {
  if (p.lengths == nullptr) return p.S;
  const int l = p.lengths[b];
  return l < 0 ? 0 : (l > p.S ? p.S : l);
}

__device__ __forceinline__ bool win_sees(const WinParams& p, int L, int i, int j) {
  const int far = i - j;
  return j < L && !(p.causal && far < 0) && (j < p.sinks || (far < p.window && -far < p.window));
}

// Whether query i sees exactly one key.  Its weight is 1 whatever its score, so its ds is zero; from dP - delta,
// sums of the same values in two orders, it would be what their roundings differ by.
__device__ __forceinline__ bool win_alone(const WinParams& p, int L, int i) {
  const int lo = max(0, i - (p.window - 1)), hi = min(L, p.causal ? i + 1 : i + p.window);
  const int sinks = min(min(p.sinks, L), p.causal ? i + 1 : L);
  return sinks + max(0, hi - max(lo, sinks)) == 1;
}
#endif

}  // namespace tgcm
