// rotary.hpp -- queries and keys turned by their positions.
#pragma once

#include "kv4.hpp"

namespace msim {

struct RotaryPlan {
  const uint64_t* turns;  // [pairs]: turns per position, in 2^-64
  const int32_t* axes;    // [pairs]: which positions a pair goes by
  int32_t pairs, dim;     // the first 2 pairs dims of dim are turned
  int32_t num_axes;
  bool adjacent;  // pairs (2 i, 2 i + 1); else (i, i + pairs)
};

struct RotaryRows {  // queries or keys, in and out
  const void* in;
  void* out;
  int64_t in_row_stride, in_head_stride, out_row_stride, out_head_stride;  // in elements
  int32_t heads;
};

hipError_t launch_rotary(const RotaryPlan& plan, const RotaryRows rows[2], int64_t num_rows, const int32_t* positions,
                         int64_t axis_stride, Kv4Type type, hipStream_t stream);

}  // namespace msim
