// Norm of every query and key head followed by the rotation of its first R
// values, in one pass, and the adjoint with the norm's parameter gradients.
//
// One head row x of D values (statistics in fp32):
//   layer:  xh = (x - mean) r,  r = (var + eps)^-1/2       y = xh * w + b
//   rms:    xh = x r,           r = (mean(x^2) + eps)^-1/2  y = xh * w
//   none:   y = x
// then pairs (a, b) = (i, i + R/2), or (2i, 2i + 1) interleaved, turn by the
// angle of the row's position:  (a cos - b sin, b cos + a sin).
// The adjoint turns dy back, g = R(-angle) dy, adds dw += g xh and db += g, and
//   dx = r (g w - mean(g w) [layer only] - xh mean(g w xh)).
//
// Both directions are bound by the bytes of the heads (a few dozen FLOP per
// value).  A warp owns tokens: a row is covered by LPR lanes with one 16-byte
// vector each (LPR = D / vector, rounded up to a power of two), so 32 / LPR
// heads of the token are in work at once; each lane reads the token's cosines
// and sines once and keeps them in registers over the token's heads — the
// table is fp32 and would otherwise be four times the traffic of bf16 heads.
// Partners of the half layout live R/2 values away: when R/2 is a multiple of
// the vector they are the same element of another lane (a shuffle); the
// interleaved partners are neighbours in the lane's own vector.  Rows that
// break those rules (odd strides, R/2 off the vector) take the row kernel, one
// warp to a row through shared memory.
// Parameter gradients: a lane sees the same D positions in every row, so it
// sums them in registers; blocks leave one partial each and a second kernel
// adds the partials in order (no atomics).
#include "alloc.h"
#include "sequence_ops.h"

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <array>
#include <string>

#include "common.cuh"

namespace tgcm {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotWarps = kRotThreads / 32;
constexpr int kRotMaxDim = 256;
constexpr int kRotBatch = 2;  // heads that a lane group asks for at once
// Resident blocks of an SM: more of them spill (8192 x 2 tokens, 16 + 4 heads of 64: forward 28 us with 3, 36 us
// with 4; adjoint 47 us with 2, 54 us with 3; 30 and 49 us since values outside the rotation are left alone).
constexpr int kRotFwdBlocks = 3, kRotBwdBlocks = 2;

enum NormKind : int { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };

// One of the two inputs (queries or keys).
struct HeadSet {
  const void* x;           // (B, S, H, D), unit stride along D
  long long sb, ss, sh;    // element strides
  const void* dy;          // adjoint: (B, S, H, D)
  long long gb, gs, gh;
  void* y;                 // (B, S, H, D) contiguous: the result, or dx
  const float* w;
  const float* b;
  float* dparam;           // adjoint: [blocks][2][D] partial sums of dw, db (or null)
  int H;
  int block0, blocks;      // the blocks that work on this set
};

struct RotParams {
  HeadSet set[2];
  int S, D, R;
  long long tokens;        // B * S
  const float2* table;     // (rows, R/2) cos, sin
  int table_rows;
  const void* pos;         // int32 or int64 (B, S) or (S,), or null
  long long pos_sb, pos_ss;
  int pos64;
  int norm, interleaved;
  float eps;
  int* err;
};

template <typename T>
__device__ __forceinline__ float ldv(const T* p) {
  if constexpr (std::is_same<T, float>::value)
    return *p;
  else
    return __bfloat162float(*p);
}
template <typename T>
__device__ __forceinline__ void stv(T* p, float v) {
  if constexpr (std::is_same<T, float>::value)
    *p = v;
  else
    *p = __float2bfloat16(v);
}

template <typename T>
struct HVec {
  static constexpr int n = 16 / sizeof(T);
};

template <typename T>
__device__ __forceinline__ void unpack16(const uint4& u, float (&v)[HVec<T>::n]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      v[i] = __uint_as_float(w[i]);
    } else {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&v)[HVec<T>::n]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      w[i] = __float_as_uint(v[i]);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Row of the table for token (b, s); a position outside it is reported and clamped.
__device__ __forceinline__ int table_row(const RotParams& p, int b, int s) {
  long long at = s;
  if (p.pos != nullptr) {
    const long long o = b * p.pos_sb + s * p.pos_ss;
    at = p.pos64 ? static_cast<const long long*>(p.pos)[o] : static_cast<const int*>(p.pos)[o];
  }
  if (at < 0 || at >= p.table_rows) {
    record_error(p.err, kErrBounds);
    at = at < 0 ? 0 : p.table_rows - 1;
  }
  return static_cast<int>(at);
}

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// Turns the lane's vector.  Half layout: element e of lanes [0, R/2/V) pairs
// with element e of the lane R/2/V further; cs holds this element's pair.  The
// lane's first `turned` elements take part (half layout: all or none); the others
// stay as they are, infinities and NaN among them.
template <int V>
__device__ __forceinline__ void turn(float (&v)[V], const float (&c)[V], const float (&s)[V], bool inter, int partner,
                                     int turned) {
  if (inter) {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float a = v[e], b = v[e + 1];
      if (e < turned) {
        v[e] = a * c[e] - b * s[e];
        v[e + 1] = b * c[e] + a * s[e];
      }
    }
  } else {  // s carries the sign: -sin for first halves, +sin for second ones
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float o = __shfl_sync(0xffffffffu, v[e], partner);
      if (turned > 0) v[e] = v[e] * c[e] + o * s[e];
    }
  }
}

// Vector kernel.  BWD: the adjoint.  A block's warps take tokens of one set
// (blockIdx.x), strided by the set's blocks.
template <typename T, int LPR, bool BWD>
__global__ void __launch_bounds__(kRotThreads, BWD ? kRotBwdBlocks : kRotFwdBlocks) rot_vec_kernel(const __grid_constant__ RotParams p) {
  constexpr int V = HVec<T>::n;
  constexpr int ROWS = 32 / LPR;
  constexpr int kBatch = kRotBatch;
  __shared__ __align__(16) float sw[LPR * V], sb[LPR * V];  // scale and shift: registers are warps here
  const HeadSet& hs = p.set[blockIdx.x >= p.set[1].block0];
  const int block = blockIdx.x - hs.block0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane % LPR, sub = lane / LPR;
  const int d0 = l * V;
  const bool live = d0 < p.D;
  const float inv_d = 1.f / static_cast<float>(p.D);
  for (int d = threadIdx.x; d < LPR * V; d += kRotThreads) {
    sw[d] = (d < p.D && hs.w) ? hs.w[d] : 1.f;
    sb[d] = (d < p.D && hs.b) ? hs.b[d] : 0.f;
  }
  __syncthreads();
  float dw[V], db[V];
#pragma unroll
  for (int e = 0; e < V; ++e) dw[e] = db[e] = 0.f;
  // partner lane and pair index of the half layout
  const int half = p.R / 2;
  const int hl = half / V;
  const bool first = live && d0 < half, second = live && d0 >= half && d0 < p.R;
  const int partner = p.interleaved ? lane : (first ? lane + hl : (second ? lane - hl : lane));
  const int turned = live ? min(V, max(0, p.R - d0)) : 0;
  const int H = hs.H;
  const int step = hs.blocks * kRotWarps, tokens = static_cast<int>(p.tokens);
  int t = block * kRotWarps + warp;
  int b = t / p.S, s = t - b * p.S;
  int at = p.R && t < tokens ? table_row(p, b, s) : 0;  // asked for one token ahead
  for (; t < tokens; t += step) {
    const T* xt = static_cast<const T*>(hs.x) + b * hs.sb + s * hs.ss + d0;
    const T* gt = BWD ? static_cast<const T*>(hs.dy) + b * hs.gb + s * hs.gs + d0 : nullptr;
    T* yt = static_cast<T*>(hs.y) + static_cast<long long>(t) * H * p.D + d0;
    // kBatch heads of every lane group are asked for at once, the first ones before the table's row
    uint4 xu[kBatch], gu[kBatch];
    auto fetch = [&](int h0) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int h = h0 + u * ROWS + sub;
        const bool on = live && h < H;
        xu[u] = make_uint4(0, 0, 0, 0);
        if (on && (!BWD || p.norm != kNormNone)) xu[u] = __ldg(reinterpret_cast<const uint4*>(xt + h * hs.sh));
        if (BWD) {
          gu[u] = make_uint4(0, 0, 0, 0);
          if (on) gu[u] = __ldg(reinterpret_cast<const uint4*>(gt + h * hs.gh));
        }
      }
    };
    fetch(0);
    const int b_next = (t + step) / p.S, s_next = t + step - b_next * p.S;
    const int at_next = p.R && t + step < tokens ? table_row(p, b_next, s_next) : 0;
    float c[V], sn[V];
#pragma unroll
    for (int e = 0; e < V; ++e) c[e] = 1.f, sn[e] = 0.f;
    if (turned > 0) {
      const float2* row = p.table + static_cast<long long>(at) * half;
      const float dir = BWD ? -1.f : 1.f;
      if (p.interleaved) {
#pragma unroll
        for (int e = 0; e < V; e += 2)
          if (d0 + e < p.R) {
            const float2 cs = __ldg(row + (d0 + e) / 2);
            c[e] = cs.x;
            sn[e] = dir * cs.y;
          }
      } else {
        // half is a multiple of V here, so the row and its pieces lie on 16-byte boundaries
        const float4* cs4 = reinterpret_cast<const float4*>(row + (first ? d0 : d0 - half));
        const float sign = first ? -dir : dir;
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float4 cs = __ldg(cs4 + e / 2);
          c[e] = cs.x, c[e + 1] = cs.z;
          sn[e] = sign * cs.y, sn[e + 1] = sign * cs.w;
        }
      }
    }
    for (int h0 = 0; h0 < H; h0 += ROWS * kBatch) {
      if (h0 > 0) fetch(h0);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (h0 + u * ROWS >= H) break;
        const int h = h0 + u * ROWS + sub;
        const bool on = live && h < H;
        float x[V];
        unpack16<T>(xu[u], x);
        float r = 1.f;
        if (p.norm == kNormLayer) {
          float m = 0.f;
#pragma unroll
          for (int e = 0; e < V; ++e) m += x[e];
          m = row_sum<LPR>(m) * inv_d;
#pragma unroll
          for (int e = 0; e < V; ++e) x[e] = live ? x[e] - m : 0.f;  // absent lanes stay out of the variance
        }
        if (p.norm != kNormNone) {
          float q = 0.f;
#pragma unroll
          for (int e = 0; e < V; ++e) q = fmaf(x[e], x[e], q);
          q = row_sum<LPR>(q);
          // a lane group without a head takes part in the shuffles alone: 1 / sqrt(eps) of an eps of zero would put
          // 0 * inf into the parameter sums
          r = h < H ? rsqrtf(q * inv_d + p.eps) : 0.f;
        }
        if (!BWD) {
#pragma unroll
          for (int e = 0; e < V; ++e) x[e] = fmaf(x[e] * r, sw[d0 + e], sb[d0 + e]);
          turn<V>(x, c, sn, p.interleaved, partner, turned);
          if (on) *reinterpret_cast<uint4*>(yt + h * p.D) = pack16<T>(x);
        } else {
          float g[V];
          unpack16<T>(gu[u], g);
          turn<V>(g, c, sn, p.interleaved, partner, turned);
          if (p.norm != kNormNone) {
            float m1 = 0.f, m2 = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
              x[e] *= r;
              dw[e] = fmaf(g[e], x[e], dw[e]);
              db[e] += g[e];
              g[e] *= sw[d0 + e];
              m1 += g[e];
              m2 = fmaf(g[e], x[e], m2);
            }
            m2 = row_sum<LPR>(m2) * inv_d;
            m1 = p.norm == kNormLayer ? row_sum<LPR>(m1) * inv_d : 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) g[e] = r * (g[e] - m1 - x[e] * m2);
          }
          if (on) *reinterpret_cast<uint4*>(yt + h * p.D) = pack16<T>(g);
        }
      }
    }
    b = b_next, s = s_next, at = at_next;
  }
  if (BWD && hs.dparam != nullptr) {  // the block's sums: rows of a warp, then the warps, in order
    __shared__ float part[kRotWarps][2][LPR * V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1) {
        dw[e] += __shfl_xor_sync(0xffffffffu, dw[e], o);
        db[e] += __shfl_xor_sync(0xffffffffu, db[e], o);
      }
      if (sub == 0) {
        part[warp][0][d0 + e] = dw[e];
        part[warp][1][d0 + e] = db[e];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.D; i += kRotThreads) {
      const int k = i / p.D, d = i - k * p.D;
      float a = 0.f;
      for (int q = 0; q < kRotWarps; ++q) a += part[q][k][d];
      hs.dparam[(static_cast<long long>(block) * 2 + k) * p.D + d] = a;
    }
  }
}

// Row kernel: any strides, any R.  One warp to a row, the row in shared memory.
template <typename T, bool BWD>
__global__ void __launch_bounds__(kRotThreads) rot_row_kernel(const __grid_constant__ RotParams p) {
  constexpr int E = kRotMaxDim / 32;
  __shared__ float rowbuf[kRotWarps][kRotMaxDim];
  __shared__ float part[kRotWarps][2][kRotMaxDim];
  const HeadSet& hs = p.set[blockIdx.x >= p.set[1].block0];
  const int block = blockIdx.x - hs.block0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* buf = rowbuf[warp];
  const int D = p.D, half = p.R / 2;
  const float inv_d = 1.f / static_cast<float>(D);
  float dw[E], db[E];
#pragma unroll
  for (int j = 0; j < E; ++j) dw[j] = db[j] = 0.f;
  const long long rows = p.tokens * hs.H;
  for (long long row = static_cast<long long>(block) * kRotWarps + warp; row < rows;
       row += static_cast<long long>(hs.blocks) * kRotWarps) {
    const long long t = row / hs.H;
    const int h = static_cast<int>(row - t * hs.H);
    const int b = static_cast<int>(t / p.S), s = static_cast<int>(t - static_cast<long long>(b) * p.S);
    const T* xr = static_cast<const T*>(hs.x) + b * hs.sb + s * hs.ss + h * hs.sh;
    const T* gr = BWD ? static_cast<const T*>(hs.dy) + b * hs.gb + s * hs.gs + h * hs.gh : nullptr;
    T* yr = static_cast<T*>(hs.y) + row * D;
    const float2* cs = p.R ? p.table + static_cast<long long>(table_row(p, b, s)) * half : nullptr;
    float x[E], g[E];
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int d = lane + 32 * j;
      x[j] = d < D ? ldv(xr + d) : 0.f;
      m += x[j];
    }
    float r = 1.f;
    if (p.norm == kNormLayer) {
      m = row_sum<32>(m) * inv_d;
#pragma unroll
      for (int j = 0; j < E; ++j) x[j] = lane + 32 * j < D ? x[j] - m : 0.f;
    }
    if (p.norm != kNormNone) {
      float q = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) q = fmaf(x[j], x[j], q);
      r = rsqrtf(row_sum<32>(q) * inv_d + p.eps);
    }
    __syncwarp();  // the buffer's last readers are done
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int d = lane + 32 * j;
      if (d >= D) continue;
      x[j] *= r;
      buf[d] = BWD ? ldv(gr + d) : fmaf(x[j], hs.w ? hs.w[d] : 1.f, hs.b ? hs.b[d] : 0.f);
    }
    __syncwarp();
    float m1 = 0.f, m2 = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int d = lane + 32 * j;
      g[j] = 0.f;
      if (d >= D) continue;
      float v = buf[d];
      if (d < p.R) {
        const int i = p.interleaved ? d / 2 : (d < half ? d : d - half);
        const bool a = p.interleaved ? (d & 1) == 0 : d < half;
        const int o = p.interleaved ? (a ? d + 1 : d - 1) : (a ? d + half : d - half);
        const float2 c = __ldg(cs + i);
        const float sn = (a ? -c.y : c.y) * (BWD ? -1.f : 1.f);
        v = v * c.x + buf[o] * sn;
      }
      if (!BWD) {
        stv(yr + d, v);
      } else {
        dw[j] = fmaf(v, x[j], dw[j]);
        db[j] += v;
        g[j] = v * (hs.w ? hs.w[d] : 1.f);
        m1 += g[j];
        m2 = fmaf(g[j], x[j], m2);
      }
    }
    if (BWD) {
      if (p.norm != kNormNone) {
        m2 = row_sum<32>(m2) * inv_d;
        m1 = p.norm == kNormLayer ? row_sum<32>(m1) * inv_d : 0.f;
      }
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int d = lane + 32 * j;
        if (d < D) stv(yr + d, p.norm == kNormNone ? g[j] : r * (g[j] - m1 - x[j] * m2));
      }
    }
  }
  if (BWD && hs.dparam != nullptr) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      part[warp][0][lane + 32 * j] = dw[j];
      part[warp][1][lane + 32 * j] = db[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += kRotThreads) {
      const int k = i / D, d = i - k * D;
      float a = 0.f;
      for (int q = 0; q < kRotWarps; ++q) a += part[q][k][d];
      hs.dparam[(static_cast<long long>(block) * 2 + k) * D + d] = a;
    }
  }
}

struct ParamGrads {
  float* out[2][2];      // q, k: dw, db, or null
  const float* part[2];
  int blocks[2];
};

// Sums of the blocks' partials, in order: one block of 8 warps for 32 columns of
// (set, dw or db), the blocks dealt to the warps in turn.
__global__ void __launch_bounds__(256) rot_param_kernel(const ParamGrads g, int D) {
  __shared__ float acc[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int set = blockIdx.z, k = blockIdx.y, d = blockIdx.x * 32 + lane;
  float* out = g.out[set][k];
  if (out == nullptr) return;
  const float* src = g.part[set] + k * D + d;
  const int blocks = g.blocks[set];
  float a = 0.f;
  if (d < D) {
#pragma unroll 8
    for (int b = warp; b < blocks; b += 8) a += src[static_cast<long long>(b) * 2 * D];
  }
  acc[warp][lane] = a;
  __syncthreads();
  if (warp == 0 && d < D) {
    float t = 0.f;
    for (int w = 0; w < 8; ++w) t += acc[w][lane];
    out[d] = t;
  }
}

// Lanes to a row in the vector kernel.
int row_lanes(int D, int vec) {
  int l = 2;
  while (l < 32 && l * vec < D) l *= 2;
  return l;
}

template <typename T, bool BWD>
void launch_rot(const RotParams& p, bool vec, cudaStream_t st) {
  const int grid = p.set[0].blocks + p.set[1].blocks;
  if (!vec) {
    rot_row_kernel<T, BWD><<<grid, kRotThreads, 0, st>>>(p);
  } else {
    switch (row_lanes(p.D, HVec<T>::n)) {
      case 2: rot_vec_kernel<T, 2, BWD><<<grid, kRotThreads, 0, st>>>(p); break;
      case 4: rot_vec_kernel<T, 4, BWD><<<grid, kRotThreads, 0, st>>>(p); break;
      case 8: rot_vec_kernel<T, 8, BWD><<<grid, kRotThreads, 0, st>>>(p); break;
      case 16: rot_vec_kernel<T, 16, BWD><<<grid, kRotThreads, 0, st>>>(p); break;
      default: rot_vec_kernel<T, 32, BWD><<<grid, kRotThreads, 0, st>>>(p); break;
    }
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

bool aligned16(const at::Tensor& t) {
  const int64_t e = t.element_size();
  bool ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) == 1 || (t.stride(i) * e) % 16 == 0);
  return ok;
}

void check_heads(const at::Tensor& t, const at::Tensor& q, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == q.device(), std::string("qk_norm_rotary: ") + name + " must be a CUDA tensor beside q");
  TORCH_CHECK(t.dim() == 4, std::string("qk_norm_rotary: ") + name + " must be (batch, sequence, heads, head_dim)");
  TORCH_CHECK(t.scalar_type() == q.scalar_type() &&
                  (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat),
              std::string("qk_norm_rotary: ") + name + " must have q's type, bf16 or fp32");
  TORCH_CHECK(t.size(0) == q.size(0) && t.size(1) == q.size(1) && t.size(3) == q.size(3),
              std::string("qk_norm_rotary: ") + name + " does not match q in batch, sequence or head_dim");
  TORCH_CHECK(t.size(3) == 1 || t.stride(3) == 1, std::string("qk_norm_rotary: ") + name + " must be contiguous along head_dim");
}

const float* param(const c10::optional<at::Tensor>& t, const at::Tensor& q, const char* name) {
  if (!t.has_value() || !t->defined()) return nullptr;
  TORCH_CHECK(t->device() == q.device() && t->scalar_type() == at::kFloat && t->is_contiguous() &&
                  t->numel() == q.size(3),
              std::string("qk_norm_rotary: ") + name + " must be a contiguous fp32 vector of head_dim values");
  return t->data_ptr<float>();
}

struct Prepared {
  RotParams p;
  bool vec;
};

Prepared prepare(const at::Tensor& q, const at::Tensor& k, const c10::optional<at::Tensor>& table,
                 const c10::optional<at::Tensor>& positions, const c10::optional<at::Tensor>& qw,
                 const c10::optional<at::Tensor>& kw, const c10::optional<at::Tensor>& qb,
                 const c10::optional<at::Tensor>& kb, int64_t norm, bool interleaved, double eps,
                 const c10::optional<at::Tensor>& err) {
  TORCH_CHECK(q.dim() == 4, "qk_norm_rotary: q must be (batch, sequence, heads, head_dim)");
  check_heads(q, q, "q");
  check_heads(k, q, "k");
  TORCH_CHECK(norm >= kNormNone && norm <= kNormLayer, "qk_norm_rotary: unknown norm");
  const int64_t D = q.size(3);
  TORCH_CHECK(D >= 1 && D <= kRotMaxDim, "qk_norm_rotary: head_dim 1 to 256 expected, got " + std::to_string(D));
  TORCH_CHECK(q.size(1) < (1ll << 31) && q.size(2) < (1 << 20) && k.size(2) < (1 << 20),
              "qk_norm_rotary: sequence or head count too large");
  TORCH_CHECK(q.size(0) * q.size(1) < (1ll << 31) - (1 << 20), "qk_norm_rotary: 2^31 tokens or more");
  Prepared r{};
  RotParams& p = r.p;
  p.S = static_cast<int>(q.size(1));
  p.D = static_cast<int>(D);
  p.tokens = q.size(0) * q.size(1);
  p.norm = static_cast<int>(norm);
  p.interleaved = interleaved;
  p.eps = static_cast<float>(eps);
  if (table.has_value() && table->defined()) {
    TORCH_CHECK(table->device() == q.device() && table->scalar_type() == at::kFloat && table->is_contiguous() &&
                    table->dim() == 3 && table->size(2) == 2 && 2 * table->size(1) <= D &&
                    reinterpret_cast<uintptr_t>(table->data_ptr()) % 8 == 0,
                "qk_norm_rotary: table must be contiguous fp32 (positions, rotary_dim / 2, 2) with rotary_dim <= head_dim");
    p.table = reinterpret_cast<const float2*>(table->data_ptr<float>());
    p.R = static_cast<int>(2 * table->size(1));
    p.table_rows = static_cast<int>(std::min<int64_t>(table->size(0), (1ll << 31) - 1));
    TORCH_CHECK(p.R == 0 || p.table_rows > 0, "qk_norm_rotary: empty table");
    TORCH_CHECK(p.R == 0 || (positions.has_value() && positions->defined()) || q.size(1) <= table->size(0),
                "qk_norm_rotary: the table has " + std::to_string(table->size(0)) + " positions, the sequence " +
                    std::to_string(q.size(1)));
  }
  if (positions.has_value() && positions->defined()) {
    const auto& t = *positions;
    TORCH_CHECK(t.device() == q.device() && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong),
                "qk_norm_rotary: positions must be int32 or int64 beside q");
    const bool two = t.dim() == 2;
    TORCH_CHECK((two && t.size(0) == q.size(0) && t.size(1) == q.size(1)) || (t.dim() == 1 && t.size(0) == q.size(1)),
                "qk_norm_rotary: positions must be (batch, sequence) or (sequence,)");
    p.pos = t.data_ptr();
    p.pos64 = t.scalar_type() == at::kLong;
    p.pos_sb = two ? t.stride(0) : 0;
    p.pos_ss = t.stride(t.dim() - 1);
  }
  if (err.has_value() && err->defined()) p.err = err->data_ptr<int>();
  const at::Tensor* xs[2] = {&q, &k};
  const float* ws[2] = {param(qw, q, "q_weight"), param(kw, q, "k_weight")};
  const float* bs[2] = {param(qb, q, "q_bias"), param(kb, q, "k_bias")};
  r.vec = true;
  const int V = q.scalar_type() == at::kBFloat16 ? 8 : 4;
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& x = *xs[i];
    p.set[i].x = x.data_ptr();
    p.set[i].sb = x.stride(0);
    p.set[i].ss = x.stride(1);
    p.set[i].sh = x.stride(2);
    p.set[i].H = static_cast<int>(x.size(2));
    p.set[i].w = ws[i];
    p.set[i].b = bs[i];
    r.vec = r.vec && aligned16(x);
  }
  r.vec = r.vec && reinterpret_cast<uintptr_t>(p.table) % 16 == 0 && D % V == 0 && (interleaved || (p.R / 2) % V == 0) && D / V <= 32;
  return r;
}

// The SMs' resident blocks shared out by what a token of the set takes (a trip to
// memory for each batch of heads); a warp takes at least one token (in the row
// kernel one row).
void share_blocks(Prepared& r, bool bwd, int lane_groups) {
  const int resident = at::cuda::getCurrentDeviceProperties()->multiProcessorCount * (r.vec ? (bwd ? kRotBwdBlocks : kRotFwdBlocks) : 8);
  int trips[2];
  for (int i = 0; i < 2; ++i)
    trips[i] = r.vec ? (r.p.set[i].H + lane_groups * kRotBatch - 1) / (lane_groups * kRotBatch) : r.p.set[i].H;
  for (int i = 0; i < 2; ++i) {
    HeadSet& s = r.p.set[i];
    const long long units = r.vec ? r.p.tokens : r.p.tokens * s.H;
    const long long share = static_cast<long long>(resident) * trips[i] / std::max(1, trips[0] + trips[1]);
    s.blocks = static_cast<int>(std::max<long long>(1, std::min((units + kRotWarps - 1) / kRotWarps, share)));
  }
  r.p.set[0].block0 = 0;
  r.p.set[1].block0 = r.p.set[0].blocks;
}

}  // namespace

std::vector<at::Tensor> qk_norm_rotary_fwd(const at::Tensor& q, const at::Tensor& k,
                                           const c10::optional<at::Tensor>& table,
                                           const c10::optional<at::Tensor>& positions,
                                           const c10::optional<at::Tensor>& qw, const c10::optional<at::Tensor>& kw,
                                           const c10::optional<at::Tensor>& qb, const c10::optional<at::Tensor>& kb,
                                           int64_t norm, bool interleaved, double eps,
                                           const c10::optional<at::Tensor>& err) {
  auto r = prepare(q, k, table, positions, qw, kw, qb, kb, norm, interleaved, eps, err);
  c10::cuda::CUDAGuard guard(q.device());
  auto yq = out_empty(q.sizes(), q.options()), yk = out_empty(k.sizes(), k.options());
  if (r.p.tokens == 0) return {yq, yk};
  r.p.set[0].y = yq.data_ptr();
  r.p.set[1].y = yk.data_ptr();
  share_blocks(r, false, 32 / row_lanes(r.p.D, 16 / static_cast<int>(q.element_size())));
  auto st = at::cuda::getCurrentCUDAStream();
  if (q.scalar_type() == at::kBFloat16)
    launch_rot<__nv_bfloat16, false>(r.p, r.vec, st);
  else
    launch_rot<float, false>(r.p, r.vec, st);
  return {yq, yk};
}

// Returns dq, dk, dq_weight, dk_weight, dq_bias, dk_bias; the last four are undefined unless asked for.
std::vector<at::Tensor> qk_norm_rotary_bwd(const at::Tensor& dyq, const at::Tensor& dyk, const at::Tensor& q,
                                           const at::Tensor& k, const c10::optional<at::Tensor>& table,
                                           const c10::optional<at::Tensor>& positions,
                                           const c10::optional<at::Tensor>& qw, const c10::optional<at::Tensor>& kw,
                                           int64_t norm, bool interleaved, double eps, std::array<bool, 4> need,
                                           const c10::optional<at::Tensor>& err) {
  auto r = prepare(q, k, table, positions, qw, kw, c10::nullopt, c10::nullopt, norm, interleaved, eps, err);
  c10::cuda::CUDAGuard guard(q.device());
  const at::Tensor* gs[2] = {&dyq, &dyk};
  const at::Tensor* xs[2] = {&q, &k};
  for (int i = 0; i < 2; ++i) {
    check_heads(*gs[i], q, i ? "the gradient of k" : "the gradient of q");
    TORCH_CHECK(gs[i]->size(2) == xs[i]->size(2), "qk_norm_rotary: a gradient has another number of heads");
    r.p.set[i].dy = gs[i]->data_ptr();
    r.p.set[i].gb = gs[i]->stride(0);
    r.p.set[i].gs = gs[i]->stride(1);
    r.p.set[i].gh = gs[i]->stride(2);
    r.vec = r.vec && aligned16(*gs[i]);
  }
  const int64_t D = q.size(3);
  std::vector<at::Tensor> out(6);
  out[0] = out_empty(q.sizes(), q.options());
  out[1] = out_empty(k.sizes(), k.options());
  ParamGrads pg{};
  bool params = false;
  for (int i = 0; i < 4; ++i) {
    if (!need[i]) continue;
    params = true;
    out[2 + i] = out_empty({D}, q.options().dtype(at::kFloat));
    pg.out[i & 1][i >> 1] = out[2 + i].data_ptr<float>();
  }
  if (r.p.tokens == 0) {
    for (int i = 2; i < 6; ++i)
      if (out[i].defined()) out[i].zero_();
    return out;
  }
  r.p.set[0].y = out[0].data_ptr();
  r.p.set[1].y = out[1].data_ptr();
  share_blocks(r, true, 32 / row_lanes(r.p.D, 16 / static_cast<int>(q.element_size())));
  at::Tensor part;
  if (params) {
    part = out_empty({r.p.set[0].blocks + r.p.set[1].blocks, 2, D}, q.options().dtype(at::kFloat));
    for (int i = 0; i < 2; ++i) {
      r.p.set[i].dparam = part.data_ptr<float>() + static_cast<int64_t>(r.p.set[i].block0) * 2 * D;
      pg.part[i] = r.p.set[i].dparam;
      pg.blocks[i] = r.p.set[i].blocks;
    }
  }
  auto st = at::cuda::getCurrentCUDAStream();
  if (q.scalar_type() == at::kBFloat16)
    launch_rot<__nv_bfloat16, true>(r.p, r.vec, st);
  else
    launch_rot<float, true>(r.p, r.vec, st);
  if (params) {
    rot_param_kernel<<<dim3(static_cast<unsigned>((D + 31) / 32), 2, 2), 256, 0, st>>>(pg, static_cast<int>(D));
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return out;
}

}  // namespace tgcm
