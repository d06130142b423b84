// Global norm of a list of gradients, and clipping by it.
//
//   norm = sqrt( sum_t sum_i g_t[i]^2 ),   out_t[i] = g_t[i] * min(1, max_norm / (norm + 1e-6))
//
// The norm needs every gradient before the first one can be scaled, so the
// list is read twice: once for the sum of squares, once to write the result.
// Bytes bound both passes.  What keeps the second read cheap is L2: pass 2
// walks the chunks from the last to the first, so the tail of the list that
// pass 1 read last is still there; a list below L2's size comes from DRAM once.
//
// The tensors' addresses travel in the kernel's parameters (no table in
// device memory, no copy, so a call can be captured in a graph as it is).  A
// block takes chunks of kChunk elements, strided by the grid; a chunk never
// spans two tensors and is found by bisection in the list of first chunks.
//
// The squares of one 16-byte vector are added in fp32 (relative error of such a
// sum below 5e-7), the vectors' sums in fp64.  No square overflows or vanishes (in
// fp32 they would above 1.8e19 and below 1e-23, which a diverging or a nearly
// converged model reaches): a vector whose sum leaves [1e-30, 1e37], one of zeros
// among them, is done over in fp64.  Converting every value
// would bound the bf16 pass: the unit converts 16 values a cycle and SM, and DRAM
// brings 12 (800 MB: 146 us so).
// Every block of pass 2 adds the partial sums of pass 1 in one fixed order
// itself, so no counter, no atomic and no second barrier is needed and two
// calls give the same bits.
#include "alloc.h"
#include "sequence_ops.h"

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <algorithm>
#include <cstring>
#include <string>
#include <vector>

#include "common.cuh"

namespace tgcm {
namespace {

constexpr int kNormThreads = 256;
constexpr int kChunk = 16384;       // elements; 64 KB of fp32
constexpr int kMaxPartials = 1184;  // blocks of pass 1: eight for each of 148 SMs

enum ElemKind : int { kF32 = 0, kBF16 = 1, kF64 = 2 };

template <int N>
struct TensorList {
  const void* in[N];
  void* out[N];
  long long n[N];
  int first[N + 1];            // first chunk of tensor t; first[count] = chunks
  unsigned char kind_in[N], kind_out[N];
  int count;
};

template <typename T>
struct Vec16 {
  static constexpr int n = 16 / sizeof(T);
  T v[n];
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ double to_f(double x) { return x; }

template <typename T>
__device__ __forceinline__ Vec16<T> ld16(const T* p) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  return *reinterpret_cast<const Vec16<T>*>(&u);
}

// Sum of squares of n elements at p, over the block's threads.
template <typename T>
__device__ __forceinline__ double sum_squares(const T* p, int n) {
  double acc = 0.0;
  auto add = [&acc](T x) {
    const double d = static_cast<double>(to_f(x));
    acc = fma(d, d, acc);
  };
  auto add16 = [&](const Vec16<T>& a) {
    if constexpr (!std::is_same<T, double>::value) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < Vec16<T>::n; ++e) {
        const float f = to_f(a.v[e]);
        s = fmaf(f, f, s);
      }
      if (s >= 1e-30f && s <= 1e37f) {
        acc += static_cast<double>(s);
        return;
      }
    }
#pragma unroll
    for (int e = 0; e < Vec16<T>::n; ++e) add(a.v[e]);
  };
  // elements in front of the first 16-byte boundary
  const int mis = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(T));
  const int head = mis < n ? mis : n;
  if (static_cast<int>(threadIdx.x) < head) add(p[threadIdx.x]);
  p += head;
  n -= head;
  constexpr int V = Vec16<T>::n;
  const int nv = n / V;
  int i = threadIdx.x;
  for (; i + 3 * kNormThreads < nv; i += 4 * kNormThreads) {  // four loads in flight
    Vec16<T> a[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) a[u] = ld16(p + static_cast<long long>(i + u * kNormThreads) * V);
#pragma unroll
    for (int u = 0; u < 4; ++u) add16(a[u]);
  }
  for (; i < nv; i += kNormThreads) {
    add16(ld16(p + static_cast<long long>(i) * V));
  }
  for (int j = nv * V + threadIdx.x; j < n; j += kNormThreads) add(p[j]);
  return acc;
}

// Sum over the block, in every thread (fixed order).
__device__ __forceinline__ double block_sum(double x) {
  __shared__ double part[kNormThreads / 32];
  __shared__ double total;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < kNormThreads / 32; ++w) t += part[w];
    total = t;
  }
  __syncthreads();
  return total;
}

template <int N>
__device__ __forceinline__ int tensor_of(const TensorList<N>& l, int c) {
  int lo = 0, hi = l.count;  // first[lo] <= c < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (l.first[mid] <= c)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <int N>
__global__ void __launch_bounds__(kNormThreads) squares_kernel(const __grid_constant__ TensorList<N> l,
                                                              double* __restrict__ partials) {
  double acc = 0.0;
  const int chunks = l.first[l.count];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = tensor_of(l, c);
    const long long at = static_cast<long long>(c - l.first[t]) * kChunk;
    const long long left = l.n[t] - at;
    const int n = left < kChunk ? static_cast<int>(left) : kChunk;
    if (l.kind_in[t] == kF32)
      acc += sum_squares(static_cast<const float*>(l.in[t]) + at, n);
    else if (l.kind_in[t] == kBF16)
      acc += sum_squares(static_cast<const __nv_bfloat16*>(l.in[t]) + at, n);
    else
      acc += sum_squares(static_cast<const double*>(l.in[t]) + at, n);
  }
  acc = block_sum(acc);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

template <typename To, typename C>
__device__ __forceinline__ To scaled(C x, C coef) {
  if constexpr (std::is_same<To, __nv_bfloat16>::value)
    return __float2bfloat16(static_cast<float>(x * coef));
  else
    return static_cast<To>(x * coef);
}

// Values of a vector access: sized so that the wider of the two sides moves 16
// bytes a lane.  (16-byte loads of bf16 with two 16-byte fp32 stores would leave
// every store half of each 32-byte sector: 510 us against 403 for 800 MB in.)
template <typename Ti, typename To>
__device__ __forceinline__ void scale_chunk(const Ti* in, To* out, int n, float coef_f) {
  using C = typename std::conditional<std::is_same<Ti, double>::value, double, float>::type;
  const C coef = static_cast<C>(coef_f);
  constexpr int V = 16 / (sizeof(Ti) > sizeof(To) ? sizeof(Ti) : sizeof(To));
  constexpr int U = 8;  // accesses in flight
  struct alignas(V * sizeof(Ti)) In { Ti v[V]; };
  struct alignas(V * sizeof(To)) Out { To v[V]; };
  int done = 0;
  if (reinterpret_cast<uintptr_t>(in) % sizeof(In) == 0 && reinterpret_cast<uintptr_t>(out) % sizeof(Out) == 0) {
    const In* vi = reinterpret_cast<const In*>(in);
    Out* vo = reinterpret_cast<Out*>(out);
    const int nv = n / V;
    auto put = [&](int at, const In& a) {
      Out r;
#pragma unroll
      for (int e = 0; e < V; ++e) r.v[e] = scaled<To, C>(to_f(a.v[e]), coef);
      vo[at] = r;
    };
    int i = threadIdx.x;
    for (; i + (U - 1) * kNormThreads < nv; i += U * kNormThreads) {
      In a[U];
#pragma unroll
      for (int u = 0; u < U; ++u) a[u] = vi[i + u * kNormThreads];
#pragma unroll
      for (int u = 0; u < U; ++u) put(i + u * kNormThreads, a[u]);
    }
    for (; i < nv; i += kNormThreads) put(i, vi[i]);
    done = nv * V;
  }
  // What is left, or all of it where the two sides are not aligned to each other (views of a flat buffer behind
  // a tensor of odd size): single values, every warp access still one run of memory.
  constexpr int S = 16;
  int j = done + threadIdx.x;
  for (; j + (S - 1) * kNormThreads < n; j += S * kNormThreads) {
    Ti a[S];
#pragma unroll
    for (int u = 0; u < S; ++u) a[u] = in[j + u * kNormThreads];
#pragma unroll
    for (int u = 0; u < S; ++u) out[j + u * kNormThreads] = scaled<To, C>(to_f(a[u]), coef);
  }
  for (; j < n; j += kNormThreads) out[j] = scaled<To, C>(to_f(in[j]), coef);
}

// Pass 2.  Block 0 of the last launch writes the norm; with `in_place` and a
// coefficient of one nothing is read or written (the product would be the same).
template <int N>
__global__ void __launch_bounds__(kNormThreads) clip_kernel(const __grid_constant__ TensorList<N> l,
                                                           const double* __restrict__ partials, int n_partials,
                                                           float max_norm, float* __restrict__ norm_out,
                                                           bool in_place) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n_partials; i += kNormThreads) s += partials[i];
  const float norm = static_cast<float>(sqrt(block_sum(s)));
  if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  float coef = max_norm / (norm + 1e-6f);
  if (coef > 1.f) coef = 1.f;  // NaN stays NaN
  if (in_place && coef == 1.f) return;
  const int chunks = l.first[l.count];
  for (int r = blockIdx.x; r < chunks; r += gridDim.x) {
    const int c = chunks - 1 - r;
    const int t = tensor_of(l, c);
    const long long at = static_cast<long long>(c - l.first[t]) * kChunk;
    const long long left = l.n[t] - at;
    const int n = left < kChunk ? static_cast<int>(left) : kChunk;
    const int ki = l.kind_in[t], ko = l.kind_out[t];
    if (ki == kF32) {
      if (ko == kF32)
        scale_chunk(static_cast<const float*>(l.in[t]) + at, static_cast<float*>(l.out[t]) + at, n, coef);
      else
        scale_chunk(static_cast<const float*>(l.in[t]) + at, static_cast<__nv_bfloat16*>(l.out[t]) + at, n, coef);
    } else if (ki == kBF16) {
      if (ko == kF32)
        scale_chunk(static_cast<const __nv_bfloat16*>(l.in[t]) + at, static_cast<float*>(l.out[t]) + at, n, coef);
      else
        scale_chunk(static_cast<const __nv_bfloat16*>(l.in[t]) + at, static_cast<__nv_bfloat16*>(l.out[t]) + at, n,
                    coef);
    } else {
      scale_chunk(static_cast<const double*>(l.in[t]) + at, static_cast<double*>(l.out[t]) + at, n, coef);
    }
  }
}

int elem_kind(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return kF32;
    case at::kBFloat16: return kBF16;
    case at::kDouble: return kF64;
    default: TORCH_CHECK(false, std::string("clip_grad_norm: fp32, bf16 or fp64 gradients expected, got ") + c10::toString(t.scalar_type()));
  }
}

template <int N, typename F>
void for_lists(const std::vector<at::Tensor>& in, const std::vector<at::Tensor>& out, F&& launch) {
  TensorList<N> l;
  size_t i = 0;
  while (i < in.size()) {
    l.count = 0;
    long long chunks = 0;
    for (; i < in.size() && l.count < N; ++i) {
      const long long n = in[i].numel();
      if (n == 0) continue;
      const long long c = (n + kChunk - 1) / kChunk;
      if (chunks + c > 0x3fffffffll) break;
      l.in[l.count] = in[i].data_ptr();
      l.out[l.count] = out.empty() ? nullptr : out[i].data_ptr();
      l.n[l.count] = n;
      l.kind_in[l.count] = static_cast<unsigned char>(elem_kind(in[i]));
      l.kind_out[l.count] = out.empty() ? 0 : static_cast<unsigned char>(elem_kind(out[i]));
      l.first[l.count] = static_cast<int>(chunks);
      chunks += c;
      ++l.count;
    }
    l.first[l.count] = static_cast<int>(chunks);
    if (l.count) launch(l, static_cast<int>(std::min<long long>(chunks, kMaxPartials)), i >= in.size());
  }
}

// out empty: the norm alone.
template <int N>
void run_clip(const std::vector<at::Tensor>& in, const std::vector<at::Tensor>& out, float max_norm, bool in_place,
              at::Tensor& norm, cudaStream_t st) {
  std::vector<int> blocks;
  for_lists<N>(in, {}, [&](const TensorList<N>&, int b, bool) { blocks.push_back(b); });
  int total = 0;
  for (int b : blocks) total += b;
  if (total == 0) {
    norm.zero_();
    return;
  }
  auto partials = out_empty({total}, norm.options().dtype(at::kDouble));
  double* pp = partials.data_ptr<double>();
  int done = 0;
  for_lists<N>(in, {}, [&](const TensorList<N>& l, int b, bool) {
    squares_kernel<N><<<b, kNormThreads, 0, st>>>(l, pp + done);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    done += b;
  });
  if (out.empty()) {
    TensorList<1> none{};
    clip_kernel<1><<<1, kNormThreads, 0, st>>>(none, pp, total, max_norm, norm.data_ptr<float>(), true);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    return;
  }
  bool first = true;
  for_lists<N>(in, out, [&](const TensorList<N>& l, int b, bool) {
    clip_kernel<N><<<b, kNormThreads, 0, st>>>(l, pp, total, max_norm, first ? norm.data_ptr<float>() : nullptr,
                                               in_place);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    first = false;
  });
}

// Short lists travel in 4 KB of parameters, long ones in 30 KB (a launch copies them all).
void dispatch_clip(const std::vector<at::Tensor>& in, const std::vector<at::Tensor>& out, float max_norm,
                   bool in_place, at::Tensor& norm) {
  auto st = at::cuda::getCurrentCUDAStream();
  if (in.size() <= 120)
    run_clip<120>(in, out, max_norm, in_place, norm, st);
  else
    run_clip<960>(in, out, max_norm, in_place, norm, st);
}

// Each tensor as one run of memory: itself, or a contiguous copy of a strided one.
std::vector<at::Tensor> dense_list(at::TensorList ts, const char* what) {
  TORCH_CHECK(!ts.empty(), "clip_grad_norm: empty list");
  std::vector<at::Tensor> v;
  v.reserve(ts.size());
  const auto dev = ts[0].device();
  for (const auto& t : ts) {
    if (!(t.is_cuda() && t.device() == dev))
      TORCH_CHECK(false, std::string("clip_grad_norm: ") + what + " must be CUDA tensors of one device");
    elem_kind(t);
    v.push_back(t.is_contiguous() ? t : t.contiguous());
  }
  return v;
}

}  // namespace

at::Tensor grad_norm(at::TensorList grads) {
  const auto in = dense_list(grads, "gradients");
  c10::cuda::CUDAGuard guard(grads[0].device());
  auto norm = out_empty({}, grads[0].options().dtype(at::kFloat));
  dispatch_clip(in, {}, 0.f, true, norm);
  return norm;
}

// An empty `out`: in place.
at::Tensor clip_grad_norm(at::TensorList grads, at::TensorList out, double max_norm) {
  const at::TensorList to = out.empty() ? grads : out;
  TORCH_CHECK(grads.size() == to.size(), "clip_grad_norm: one output for each gradient expected");
  const auto in = dense_list(grads, "gradients");
  std::vector<at::Tensor> dst;
  dst.reserve(to.size());
  bool in_place = true, strided = false;
  for (size_t i = 0; i < grads.size(); ++i) {
    const auto &g = grads[i], &o = to[i];
    if (!(g.device() == o.device() && g.sizes() == o.sizes()))
      TORCH_CHECK(false, "clip_grad_norm: output " + std::to_string(i) +
                             " has another shape or device than its gradient");
    const int ki = elem_kind(g), ko = elem_kind(o);
    TORCH_CHECK((ki == kF64) == (ko == kF64), "clip_grad_norm: fp64 gradients have fp64 outputs");
    const bool whole = o.is_contiguous();
    strided = strided || !whole;
    dst.push_back(whole ? o : at::empty(o.sizes(), o.options()));
    in_place = in_place && ((whole && in[i].data_ptr() == o.data_ptr() && ki == ko) || g.numel() == 0);
  }
  c10::cuda::CUDAGuard guard(grads[0].device());
  auto norm = out_empty({}, grads[0].options().dtype(at::kFloat));
  dispatch_clip(in, dst, static_cast<float>(max_norm), in_place, norm);
  if (strided)
    for (size_t i = 0; i < dst.size(); ++i)
      if (!to[i].is_contiguous()) to[i].copy_(dst[i]);
  return norm;
}

}  // namespace tgcm

TORCH_LIBRARY_FRAGMENT(tgcm, m) {
  m.def("grad_norm(Tensor[] grads) -> Tensor");
  m.def("clip_grad_norm(Tensor[] grads, Tensor(a!)[] out, float max_norm) -> Tensor");
}

TORCH_LIBRARY_IMPL(tgcm, CUDA, m) {
  m.impl("grad_norm", &tgcm::grad_norm);
  m.impl("clip_grad_norm", &tgcm::clip_grad_norm);
}
