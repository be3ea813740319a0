// pages.hpp -- which pages of a pool the sequences of a batch hold.
#pragma once

#include "kv4.hpp"

namespace msim {

// Sequence b holds the first ceil(lengths[b] / page) pages of its row of the table,
// the first free_count entries of free_pages are a stack of the others.
struct PagesState {
  int32_t* table;    // [batch, max_pages]; -1 behind a sequence's pages
  int32_t* lengths;  // [batch]
  int32_t* free_pages;  // [num_pages]; -1 behind the stack
  int32_t* free_count;  // [1]
  int32_t batch, max_pages, num_pages;
  int32_t page_shift;  // log2(tokens of a page)
};

struct PagesUpdate {
  const int32_t* fresh;  // [batch]: tokens that each sequence gets; nullptr: none
  const int32_t* cut;    // [batch]: tokens that it keeps at most; nullptr: all
  int32_t rows;          // capacity of the next ones
  int32_t* offsets;      // [batch + 1]
  int32_t* positions;    // [rows]; -1 behind the last row
  int64_t* slots;        // [rows]
};

hipError_t launch_pages_update(const PagesState& state, const PagesUpdate& update, hipStream_t stream);

}  // namespace msim
