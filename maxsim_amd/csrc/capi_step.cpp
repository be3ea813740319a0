// capi_step.cpp -- C ABI of what surrounds the 4-bit cache in a decoding step: pages
// (pages.hip) and rotary positions (rotary.hip).
#include <climits>

#include "capi_internal.hpp"
#include "pages.hpp"
#include "rotary.hpp"

using namespace msim;

namespace {

constexpr int64_t kMaxRows = int64_t{1} << 26;
constexpr int64_t kMaxRotaryRows = int64_t{1} << 25;  // a wave's threads per row, within the grid limits
constexpr int64_t kMostKeys = INT_MAX - 4096;         // of a sequence, as the cache's calls take them

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace

extern "C" int msim_pages_update_async(int32_t* page_table, int32_t* lengths, int32_t* free_pages, int32_t* free_count,
                                       int64_t batch, int64_t max_pages, int64_t num_pages, int64_t page_size,
                                       const int32_t* new_tokens, const int32_t* cut, int64_t rows, int32_t* offsets,
                                       int32_t* positions, int64_t* slots, void* stream) {
  return guarded([&] {
    if (page_size < 16 || page_size > 65536 || (page_size & (page_size - 1)) != 0)
      throw InvalidArgument("page_size must be a power of two from 16 to 65536");
    if (num_pages < 1 || num_pages > INT_MAX) throw InvalidArgument("num_pages must be positive");
    if (batch < 0 || max_pages < 0 || rows < 0) throw InvalidArgument("batch, max_pages and rows must not be negative");
    const int page_shift = __builtin_ctzll((unsigned long long)page_size);
    if (max_pages > kMostKeys >> page_shift)
      throw NotSupported("a page table holds sequences of less than 2^31 - 4096 tokens");
    if (rows > kMaxRows || batch > kMaxRows) throw NotSupported("a call takes at most 2^26 rows and sequences");
    if (batch * max_pages > INT_MAX) throw NotSupported("a page table has less than 2^31 entries");
    if (!free_pages || !free_count || !offsets || (rows > 0 && (!positions || !slots)) ||
        (batch > 0 && (!lengths || (max_pages > 0 && !page_table))))
      throw InvalidArgument("the pages' state and the outputs must not be NULL");
    const PagesState state{page_table,         lengths,           free_pages, free_count, (int32_t)batch,
                           (int32_t)max_pages, (int32_t)num_pages, page_shift};
    const PagesUpdate update{new_tokens, cut, (int32_t)rows, offsets, positions, slots};
    check_hip(launch_pages_update(state, update, as_stream(stream)), "launch page kernels");
  });
}

extern "C" int msim_rotary_async(const uint64_t* turns, const int32_t* axes, int64_t pairs, int64_t dim,
                                 int64_t num_axes, int adjacent, const int32_t* positions, int64_t axis_stride,
                                 int64_t rows, int type, const void* q, int64_t q_row_stride, int64_t q_head_stride,
                                 int64_t heads, void* q_out, int64_t q_out_row_stride, int64_t q_out_head_stride,
                                 const void* k, int64_t k_row_stride, int64_t k_head_stride, int64_t kv_heads,
                                 void* k_out, int64_t k_out_row_stride, int64_t k_out_head_stride, void* stream) {
  return guarded([&] {
    if (type != MSIM_F32 && type != MSIM_F16 && type != MSIM_BF16)
      throw InvalidArgument("type must be MSIM_F32, MSIM_F16 or MSIM_BF16");
    if (pairs < 1 || 2 * pairs > dim) throw InvalidArgument("rotary dims must be between 2 and the head's");
    if (dim > 256) throw NotSupported("at most 256 dims of a head");  // a wave holds a head
    if (num_axes < 1 || num_axes > pairs) throw InvalidArgument("axes must be between 1 and the number of pairs");
    if (rows < 0 || heads < 0 || kv_heads < 0) throw InvalidArgument("rows and heads must not be negative");
    if (rows > kMaxRotaryRows || heads > 65536 || kv_heads > 65536)
      throw NotSupported("at most 2^25 rows and 2^16 heads");
    if (rows == 0 || heads + kv_heads == 0) return;
    if (!turns || !axes || !positions) throw InvalidArgument("frequencies, axes and positions must not be NULL");
    const size_t size = type == MSIM_F32 ? 4 : 2;
    const RotaryRows both[2] = {
        {q, q_out, q_row_stride, q_head_stride, q_out_row_stride, q_out_head_stride, (int32_t)heads},
        {k, k_out, k_row_stride, k_head_stride, k_out_row_stride, k_out_head_stride, (int32_t)kv_heads}};
    for (const RotaryRows& r : both) {
      if (r.heads == 0) continue;
      if (!r.in || !r.out) throw InvalidArgument("q, k and their outputs must not be NULL");
      if (!aligned(r.in, size) || !aligned(r.out, size))
        throw InvalidArgument("q, k and their outputs must be aligned to their type");
    }
    const RotaryPlan plan{turns, axes, (int32_t)pairs, (int32_t)dim, (int32_t)num_axes, adjacent != 0};
    check_hip(launch_rotary(plan, both, rows, positions, axis_stride, static_cast<Kv4Type>(type), as_stream(stream)),
              "launch rotary kernel");
  });
}
