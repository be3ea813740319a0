// linear4.hpp -- products with a matrix in 4 bits and group scales.
#pragma once

#include "common.hpp"
#include "kv4.hpp"

namespace msim {

// The matrix [n, k] as the product reads it: tiles of 16 rows x 128 columns,
// each 1 KiB in lane order (rows and columns past the end hold zeros), and per
// tile the scales of its groups.
struct Linear4Matrix {
  const uint8_t* codes;    // [n tiles][k tiles][64 lanes][16 bytes]
  const uint16_t* scales;  // bfloat16 [n tiles][k tiles][4][groups of a tile][4 rows]
  const float* bias;       // [n] or nullptr
  int32_t n, k, group;
};

__host__ __device__ inline int64_t linear4_tiles(int64_t n, int64_t k) { return ((n + 15) / 16) * ((k + 127) / 128); }

hipError_t launch_linear4_layout(const uint8_t* codes, const uint16_t* scales, int64_t n, int64_t k, int group,
                                 uint8_t* out_codes, uint16_t* out_scales, hipStream_t stream);
hipError_t launch_linear4(const Linear4Matrix& w, const void* x, int64_t rows, int64_t x_row_stride, Kv4Type type,
                          void* out, int64_t out_row_stride, int num_cus, hipStream_t stream);

}  // namespace msim
