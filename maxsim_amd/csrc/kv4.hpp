// kv4.hpp -- the paged 4-bit key/value cache as its kernels see it.
//
// A pool of pages; page p holds, for every key/value head h, page_size rows of
// dim / 2 bytes (two's complement nibbles, even dim low) and as many single
// precision scales.  Sequence b of a batch is the row b of a page table and a
// length.  The rows a call works on (new tokens, queries, rows to read) are
// packed: rows [offsets[b], offsets[b + 1]) belong to sequence b and are its
// last ones (one row per sequence without offsets).
//
// Table, lengths and offsets lie in device memory, unseen by the host, so the
// kernels hold every index within its array: lengths are cut to the table,
// rows to the row count, and a page number outside the pool is a hole that is
// not written, reads back as zeros and takes no attention.
#pragma once

#include "common.hpp"

namespace msim {

enum Kv4Type { kKv4F32 = 0, kKv4F16 = 1, kKv4BF16 = 2 };

struct Kv4Pool {
  uint8_t* codes[2];  // keys, values: [num_pages, kv_heads, page_size, dim / 2]
  float* scales[2];   // [num_pages, kv_heads, page_size]
  int32_t num_pages;
  int32_t page_shift;  // log2(page_size)
  int32_t kv_heads;
  int32_t dim;
};

struct Kv4Batch {
  const int32_t* table;    // [batch, max_pages]
  const int32_t* lengths;  // [batch]
  const int32_t* offsets;  // [batch + 1] or nullptr: one row per sequence
  int32_t batch;
  int32_t max_pages;
  int32_t rows;
};

struct Kv4Rows {  // rows of keys or values in a program's memory
  void* ptr;
  int64_t row_stride, head_stride;  // in elements
};


__device__ __forceinline__ int kv4_length(const Kv4Pool& pool, const Kv4Batch& batch, int b) {
  const int64_t most = (int64_t)batch.max_pages << pool.page_shift;
  const int n = as_constant(batch.lengths)[b];
  return n < 0 ? 0 : ((int64_t)n > most ? (int)most : n);
}

// First row of sequence b (b up to batch): never past the row count.
__device__ __forceinline__ int kv4_first_row(const Kv4Batch& batch, int b) {
  if (batch.offsets == nullptr) return min(b, batch.rows);
  const int v = as_constant(batch.offsets)[b];
  return v < 0 ? 0 : min(v, batch.rows);
}

// The sequence that `row` belongs to, by a wave together: each step reads 64
// offsets and keeps one 64th of the range.  -1 where there is none.
__device__ __forceinline__ int kv4_find_sequence(const Kv4Batch& batch, int row) {
  if (batch.offsets == nullptr) return row < batch.batch ? row : -1;
  int lo = 0, n = batch.batch;
  while (true) {
    const int step = (n + 63) / 64;
    const int i = lo + lane_id() * step;
    const bool below = lane_id() * step < n && batch.offsets[i] <= row;
    const int count = __popcll(__ballot(below));
    if (count == 0) return -1;
    lo += (count - 1) * step;
    n = min(step, n - (count - 1) * step);
    if (step == 1) return row < kv4_first_row(batch, lo + 1) ? lo : -1;
  }
}

// The same by one lane alone, from a sequence at or before the row's.
__device__ __forceinline__ int kv4_find_sequence_from(const Kv4Batch& batch, int row, int from) {
  int lo = from, hi = batch.batch;  // offsets[lo] <= row < offsets[hi], for ordered offsets
  if (lo >= hi || batch.offsets[lo] > row) return -1;
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (batch.offsets[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  return row < kv4_first_row(batch, lo + 1) ? lo : -1;
}

// Page and slot of a row; false where it has none.
struct Kv4Slot {
  int32_t page, slot;
};
__device__ __forceinline__ bool kv4_slot(const Kv4Pool& pool, const Kv4Batch& batch, int b, int row, Kv4Slot& out) {
  const int pos = kv4_length(pool, batch, b) - (kv4_first_row(batch, b + 1) - row);
  if (pos < 0) return false;  // more rows than the sequence holds
  out.page = batch.table[(int64_t)b * batch.max_pages + (pos >> pool.page_shift)];
  out.slot = pos & ((1 << pool.page_shift) - 1);
  return (uint32_t)out.page < (uint32_t)pool.num_pages;
}

// Index of a row of the pool.
__device__ __forceinline__ int64_t kv4_pool_row(const Kv4Pool& pool, int page, int head, int slot) {
  return (((int64_t)page * pool.kv_heads + head) << pool.page_shift) + slot;
}

hipError_t launch_kv4_append(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4Rows rows[2], Kv4Type type,
                             hipStream_t stream);
hipError_t launch_kv4_read(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4Rows rows[2], Kv4Type type,
                           hipStream_t stream);

// Of each sequence's rows those of the list kept [batch, width] stay, in its order; lengths
// [batch] are written.
hipError_t launch_kv4_keep(const Kv4Pool& pool, const Kv4Batch& batch, const int32_t* kept, int width, int32_t* lengths,
                           hipStream_t stream);

// ---------------------------------------------------------------- attention

struct Kv4AttendArgs {
  const void* q;
  int64_t q_row_stride, q_head_stride;  // elements
  void* out;
  int64_t out_row_stride, out_head_stride;
  float* lse;           // [rows, heads] or nullptr
  const uint8_t* mask;  // [rows, mask_width] or nullptr; 0 hides a key
  int64_t mask_row_stride;
  int64_t mask_width;
  int32_t q_wide, out_wide;  // rows of every head start on 16 bytes (out: on 4 elements)
  int32_t heads;
  int32_t causal;
  int32_t window;  // keys at p - window + 1 .. p; INT32_MAX: all
  int32_t sinks;   // and those below, whatever the window
  // [rows] or nullptr: the row of its sequence's that a row comes after (an earlier one;
  // any other number: the last token before them). It sees the tokens before the
  // sequence's rows, the rows that it comes after, and itself, and its position counts those.
  const int32_t* parents;
  float scale_log2;  // softmax scale * log2(e)
};

// Rows of a sequence in a call with parents, at most: rows of a longer one see nothing.
constexpr int kMostDrafts = 1024;

// Bytes for a call of any type; one with parents does with the lesser of both.
size_t kv4_attend_workspace(const Kv4Pool& pool, const Kv4Batch& batch, int heads, bool parents, int num_cus);
hipError_t launch_kv4_attend(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args, Kv4Type type,
                             void* workspace, size_t workspace_bytes, int num_cus, hipStream_t stream);

}  // namespace msim
