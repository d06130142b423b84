// Tensor maps of 2-D to 4-D bf16 tensors with 128-byte swizzled boxes.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <c10/util/Exception.h>

#include <cstdint>
#include <mutex>
#include <string>

namespace tgcm {

using TmapEncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline TmapEncodeFn tmap_encode_fn() {
  static TmapEncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q);
    if (e == cudaSuccess && q == cudaDriverEntryPointSuccess) fn = reinterpret_cast<TmapEncodeFn>(ptr);
  });
  TORCH_CHECK(fn != nullptr, "tgcm: cuTensorMapEncodeTiled entry point unavailable");
  return fn;
}

// dims innermost first; strides in bytes for dims 1, 2, ...; the box's inner extent is 64 elements.
// Reads outside the tensor give zeros.
template <int RANK>
inline CUtensorMap tmap_bf16(const void* ptr, const uint64_t (&dims)[RANK], const uint64_t (&strides)[RANK - 1],
                             const uint32_t (&box)[RANK]) {
  TORCH_CHECK(reinterpret_cast<uint64_t>(ptr) % 16 == 0, "tgcm: TMA base address not 16-byte aligned");
  cuuint64_t d[RANK], s[RANK - 1];
  cuuint32_t b[RANK], one[RANK];
  for (int i = 0; i < RANK; ++i) {
    d[i] = dims[i];
    b[i] = box[i];
    one[i] = 1;
    if (i + 1 < RANK) {
      s[i] = strides[i];
      TORCH_CHECK(strides[i] % 16 == 0, "tgcm: TMA strides must be multiples of 16 bytes");
    }
  }
  // The driver call needs a current context, which a thread that has only used
  // the runtime's allocator (autograd's worker threads) may not have yet.
  static thread_local int ready_device = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev != ready_device && cudaSetDevice(dev) == cudaSuccess) ready_device = dev;
  CUtensorMap map;
  const CUresult r = tmap_encode_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, RANK, const_cast<void*>(ptr), d, s, b,
                                      one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "tgcm: cuTensorMapEncodeTiled failed with code " + std::to_string(static_cast<int>(r)));
  return map;
}

}  // namespace tgcm
