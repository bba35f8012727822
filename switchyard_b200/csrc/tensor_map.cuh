// Tensor maps for the tiled TMA loads: row-major [rows, cols] matrices, 128-byte swizzle.
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace sy {

// Box: box_cols elements (128 bytes) x box_rows. Out-of-range elements read as zero.
int tensor_map_2d(CUtensorMap* map, CUtensorMapDataType type, int elem_bytes, const void* base, uint64_t rows, uint64_t cols,
                  int box_rows, int box_cols);

}  // namespace sy
