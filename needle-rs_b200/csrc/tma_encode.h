// tma_encode.h — host-side construction of tiled TMA descriptors.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ndl {

// Descriptor of a `rank`-dimensional tensor (innermost dimension first;
// strides in bytes of dimensions 1..rank-1) loaded in boxes of `box` elements
// with the 128-byte swizzle; what lies outside the extents reads as zero.
cudaError_t tma_map_tiled(CUtensorMap *map, CUtensorMapDataType type, int rank, const void *base, const uint64_t *dims,
                          const uint64_t *strides, const uint32_t *box);

}  // namespace ndl
