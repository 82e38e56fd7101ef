// Tensor maps of byte arrays, for the TMA copies of the decode-step kernels.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>

namespace sharq {

using EncodeTensorMap = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                     const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                     CUtensorMapFloatOOBfill);

inline EncodeTensorMap encode_tensor_map() {
  static EncodeTensorMap fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTensorMap>(ptr);
  });
  return fn;
}

// `rank` (at most 5) dimensions of bytes, strides of all but the first; what lies outside is read as 0.
inline bool make_tensor_map(CUtensorMap *map, int rank, const void *base, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box,
                            CUtensorMapSwizzle swizzle) {
  const EncodeTensorMap fn = encode_tensor_map();
  const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
  return fn != nullptr && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, (cuuint32_t)rank, const_cast<void *>(base), dims, strides, box, steps,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace sharq
