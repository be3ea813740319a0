// capi_linear4.cpp -- C ABI of products with a 4-bit matrix (linear4.hip).
#include <climits>

#include "capi_internal.hpp"
#include "linear4.hpp"

using namespace msim;

namespace {

constexpr int64_t kMaxSide = int64_t{1} << 24;  // keeps tile numbers and launches within their types

void check_shape(int64_t n, int64_t k, int64_t group) {
  if (group != 32 && group != 64 && group != 128) throw InvalidArgument("group_size must be 32, 64 or 128");
  if (n < 1 || k < 1) throw InvalidArgument("the matrix must have rows and columns");
  if (k % group != 0) throw InvalidArgument("columns must be a multiple of group_size");
  if (n > kMaxSide || k > kMaxSide) throw NotSupported("at most 2^24 rows or columns");
}

}  // namespace

extern "C" int msim_linear4_layout_bytes(int64_t n, int64_t k, int64_t group, uint64_t* codes_bytes,
                                         uint64_t* scales_bytes) {
  return guarded([&] {
    check_shape(n, k, group);
    if (codes_bytes == nullptr || scales_bytes == nullptr) throw InvalidArgument("outputs must not be NULL");
    *codes_bytes = (uint64_t)linear4_tiles(n, k) * 1024;
    *scales_bytes = (uint64_t)linear4_tiles(n, k) * 16 * (128 / group) * sizeof(uint16_t);
  });
}

extern "C" int msim_linear4_layout_async(const uint8_t* codes, const uint16_t* scales, int64_t n, int64_t k,
                                         int64_t group, uint8_t* out_codes, uint16_t* out_scales, void* stream) {
  return guarded([&] {
    check_shape(n, k, group);
    if (!codes || !scales || !out_codes || !out_scales) throw InvalidArgument("matrix pointers must not be NULL");
    if (reinterpret_cast<uintptr_t>(codes) % 4 != 0 || reinterpret_cast<uintptr_t>(out_codes) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(out_scales) % 16 != 0)
      throw InvalidArgument("codes must be 4-byte aligned, the laid-out matrix 16-byte aligned");
    check_hip(launch_linear4_layout(codes, scales, n, k, (int)group, out_codes, out_scales, as_stream(stream)),
              "launch matrix layout kernel");
  });
}

extern "C" int msim_linear4_async(const uint8_t* codes, const uint16_t* scales, int64_t n, int64_t k, int64_t group,
                                  const float* bias, const void* x, int64_t rows, int64_t x_row_stride, int type,
                                  void* out, int64_t out_row_stride, void* stream) {
  return guarded([&] {
    check_shape(n, k, group);
    if (type != MSIM_F32 && type != MSIM_F16 && type != MSIM_BF16)
      throw InvalidArgument("type must be MSIM_F32, MSIM_F16 or MSIM_BF16");
    if (rows < 0) throw InvalidArgument("rows must not be negative");
    if (rows > (int64_t{1} << 20)) throw NotSupported("at most 2^20 rows");
    if (rows == 0) return;
    if (!codes || !scales || !x || !out) throw InvalidArgument("matrix, input and output must not be NULL");
    const size_t size = type == MSIM_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || reinterpret_cast<uintptr_t>(scales) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(x) % size != 0 || reinterpret_cast<uintptr_t>(out) % size != 0)
      throw InvalidArgument("the laid-out matrix must be 16-byte aligned, x and out aligned to their type");
    const Linear4Matrix w{codes, scales, bias, (int32_t)n, (int32_t)k, (int32_t)group};
    check_hip(launch_linear4(w, x, rows, x_row_stride, static_cast<Kv4Type>(type), out, out_row_stride,
                             device_cu_count(), as_stream(stream)),
              "launch 4-bit product kernel");
  });
}
