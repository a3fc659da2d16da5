// tma_encode.cpp — host-side construction of tiled TMA descriptors.
#include "tma_encode.h"

#include <cudaTypedefs.h>

namespace ndl {

static PFN_cuTensorMapEncodeTiled_v12000 find_encode() {
  void *p = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
      q == cudaDriverEntryPointSuccess)
    return (PFN_cuTensorMapEncodeTiled_v12000)p;
  return nullptr;
}

cudaError_t tma_map_tiled(CUtensorMap *map, CUtensorMapDataType type, int rank, const void *base, const uint64_t *dims,
                          const uint64_t *strides, const uint32_t *box) {
  static const PFN_cuTensorMapEncodeTiled_v12000 encode = find_encode();
  if (!encode) return cudaErrorNotSupported;
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  cuuint64_t d[5], s[4];
  cuuint32_t b[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = dims[i];
    b[i] = box[i];
    if (i + 1 < rank) s[i] = strides[i];
  }
  const CUresult r = encode(map, type, (cuuint32_t)rank, const_cast<void *>(base), d, s, b, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

}  // namespace ndl
