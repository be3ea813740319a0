// pages.hip -- page tables, row offsets, positions and slots, from how many tokens
// each sequence of a batch keeps and gets.
//
//   kept K = min(length, cut); its pages past ceil(K / page) go onto the stack of
//   free ones, all sequences' together in reverse order, so that the i-th page given
//   back is the i-th one taken again
//   new n: none if K + n passes the table; none from the row on that would be the
//   (rows + 1)-th of the call; none if the pages asked for by this and the earlier
//   sequences are more than the stack holds and it needs one
//   offsets = prefix sums of n; row i of a sequence is at position K + i, slot
//   page * page_size + position % page_size
//
// Scans over the sequences decide who gets what, which one workgroup does: a thread
// per sequence, 1,024 at a time. Pages then change hands one per thread, found by a
// search in the scan. Rows are written by the same launch where there are few, else by
// a second one with a thread per row.
#include "pages.hpp"

namespace msim {

namespace {

constexpr int kThreads = 1024;
constexpr int kFewRows = 4096;

// Scan over the workgroup's threads, of an operation with the neutral element 0;
// `all` is the whole of it. `s` is left in use until the next barrier.
template <typename Op>
__device__ __forceinline__ uint32_t group_scan(uint32_t v, Op op, uint32_t* s, uint32_t& all) {
  const int lane = lane_id(), wave = wave_uniform(threadIdx.x / kWave);
  v = wave_scan(v, op);
  if (lane == kWave - 1) s[wave] = v;
  __syncthreads();
  const uint32_t ends = wave_scan(lane < kThreads / kWave ? s[lane] : 0, op);
  all = __builtin_amdgcn_readlane(ends, kThreads / kWave - 1);
  const uint32_t before = wave > 0 ? __builtin_amdgcn_readlane(ends, wave > 0 ? wave - 1 : 0) : 0;
  return op(before, v);
}

__device__ __forceinline__ uint32_t plus(uint32_t a, uint32_t b) { return a + b; }

// The sequence of a chunk whose part of a scan holds element e: the first of `count`
// ends above it.
__device__ __forceinline__ int holder(const uint32_t* ends, int count, uint32_t e) {
  int lo = 0;
  for (int n = count; n > 1;) {
    const int half = n / 2;
    if (ends[lo + half - 1] <= e) {
      lo += half;
      n -= half;
    } else {
      n = half;
    }
  }
  return lo;
}

struct Sequence {
  int kept, held, stay;  // tokens; pages before and after the cut
};
__device__ __forceinline__ Sequence sequence_of(const PagesState& st, const PagesUpdate& up, int b) {
  Sequence q = {0, 0, 0};
  if (b >= st.batch) return q;
  const int64_t most = (int64_t)st.max_pages << st.page_shift;  // less than 2^31
  const int page = 1 << st.page_shift;
  const int length = (int)min((int64_t)max(st.lengths[b], 0), most);
  q.kept = up.cut == nullptr ? length : min(length, max(up.cut[b], 0));
  q.held = (int)(((int64_t)length + page - 1) >> st.page_shift);
  q.stay = (int)(((int64_t)q.kept + page - 1) >> st.page_shift);
  return q;
}

__global__ __launch_bounds__(kThreads) void pages_update_kernel(PagesState st, PagesUpdate up, bool with_rows) {
  __shared__ uint32_t s_scan[4][kThreads / kWave];
  __shared__ uint32_t s_end[kThreads];   // ends of the sequences' parts of a scan
  __shared__ int s_stay[kThreads], s_kept[kThreads];
  __shared__ uint32_t s_popped;
  const int tid = threadIdx.x, page = 1 << st.page_shift;

  // What comes back.
  uint32_t given_back = 0;
  for (int b = tid; b < st.batch; b += kThreads) {
    const Sequence q = sequence_of(st, up, b);
    given_back += q.held - q.stay;
  }
  uint32_t all_back;
  group_scan(given_back, plus, s_scan[0], all_back);
  const int had = min(max(*st.free_count, 0), st.num_pages);
  // Never past the stack, whatever the lengths and the count were set to.
  all_back = min(all_back, (uint32_t)(st.num_pages - had));
  const uint32_t total = had + all_back;
  if (tid == 0) s_popped = 0;
  uint32_t before = 0;
  for (int c0 = 0; c0 < st.batch && all_back > 0; c0 += kThreads) {
    const Sequence q = sequence_of(st, up, c0 + tid);
    uint32_t all;
    s_end[tid] = group_scan(q.held - q.stay, plus, s_scan[1], all);
    s_stay[tid] = q.stay;
    __syncthreads();
    const int count = min(kThreads, st.batch - c0);
    for (uint32_t e = tid; e < all; e += kThreads) {
      const int i = holder(s_end, count, e);
      int32_t& entry = st.table[(int64_t)(c0 + i) * st.max_pages + s_stay[i] + (e - (i > 0 ? s_end[i - 1] : 0))];
      if (before + e < all_back) st.free_pages[total - 1 - (before + e)] = entry;
      entry = -1;
    }
    before += all;
    __syncthreads();
  }
  __syncthreads();

  // What is given.
  const uint32_t cap = (uint32_t)up.rows + 1;
  auto capped = [cap](uint32_t a, uint32_t b) { return min(a + b, cap); };
  uint32_t asked_rows = 0, asked_pages = 0, rows = 0;
  for (int c0 = 0; c0 < st.batch; c0 += kThreads) {
    const int b = c0 + tid, count = min(kThreads, st.batch - c0);
    const Sequence q = sequence_of(st, up, b);
    int64_t n = b < st.batch && up.fresh != nullptr ? max(up.fresh[b], 0) : 0;
    if (q.kept + n > (int64_t)st.max_pages << st.page_shift) n = 0;
    uint32_t all_rows, all_pages;
    const uint32_t end_row = capped(asked_rows, group_scan((uint32_t)min(n, (int64_t)cap), capped, s_scan[0], all_rows));
    bool refused = n > 0 && end_row == cap;
    if (refused) n = 0;
    const int need = (int)((q.kept + n + page - 1) >> st.page_shift) - q.stay;
    const uint32_t end_page = group_scan(need, plus, s_scan[1], all_pages);
    if (need > 0 && asked_pages + end_page > total) {
      refused = true;
      n = 0;
    }
    uint32_t end = asked_rows == rows ? end_row - asked_rows : 0, all = all_rows;
    if (__syncthreads_or(refused) || asked_rows != rows) end = group_scan((uint32_t)n, plus, s_scan[2], all);
    if (need > 0 && asked_pages + end_page <= total) atomicMax(&s_popped, asked_pages + end_page);
    s_end[tid] = end_page;
    s_stay[tid] = q.stay;
    s_kept[tid] = q.kept;
    if (b < st.batch) {
      up.offsets[b] = (int32_t)(rows + end - (uint32_t)n);
      st.lengths[b] = q.kept + (int)n;
    }
    __syncthreads();
    const uint32_t pops = s_popped > asked_pages ? s_popped - asked_pages : 0;
    for (uint32_t e = tid; e < pops; e += kThreads) {
      const int i = holder(s_end, count, e);
      int32_t& entry = st.free_pages[total - 1 - (asked_pages + e)];
      st.table[(int64_t)(c0 + i) * st.max_pages + s_stay[i] + (e - (i > 0 ? s_end[i - 1] : 0))] = entry;
      entry = -1;
    }
    if (with_rows) {
      __syncthreads();
      s_end[tid] = end;
      __syncthreads();
      for (uint32_t e = tid; e < all; e += kThreads) {
        const int i = holder(s_end, count, e);
        const int pos = s_kept[i] + (int)(e - (i > 0 ? s_end[i - 1] : 0));
        const int entry = st.table[(int64_t)(c0 + i) * st.max_pages + (pos >> st.page_shift)];
        up.positions[rows + e] = pos;
        up.slots[rows + e] =
            (uint32_t)entry < (uint32_t)st.num_pages ? ((int64_t)entry << st.page_shift) + (pos & (page - 1)) : -1;
      }
    }
    asked_rows = capped(asked_rows, all_rows);
    asked_pages += all_pages;
    rows += all;
    __syncthreads();
  }
  if (tid == 0) {
    up.offsets[st.batch] = (int32_t)rows;
    *st.free_count = (int32_t)(total - s_popped);
  }
  if (with_rows)
    for (int r = rows + tid; r < up.rows; r += kThreads) up.positions[r] = -1, up.slots[r] = -1;
}

// A thread per row; a sequence's rows are its last ones.
__global__ __launch_bounds__(256) void pages_rows_kernel(Kv4Batch batch, int page_shift, int num_pages,
                                                         int32_t* __restrict__ positions, int64_t* __restrict__ slots) {
  const int row = blockIdx.x * 256 + threadIdx.x, first = wave_uniform(row);
  int b = kv4_find_sequence(batch, first);
  if (b >= 0 && row >= kv4_first_row(batch, b + 1)) b = kv4_find_sequence_from(batch, row, b);
  if (row >= batch.rows) return;
  int pos = -1;
  int64_t slot = -1;
  if (b >= 0) {
    pos = batch.lengths[b] - (batch.offsets[b + 1] - row);
    const int page = batch.table[(int64_t)b * batch.max_pages + (pos >> page_shift)];
    if ((uint32_t)page < (uint32_t)num_pages) slot = ((int64_t)page << page_shift) + (pos & ((1 << page_shift) - 1));
  }
  positions[row] = pos;
  slots[row] = slot;
}

}  // namespace

hipError_t launch_pages_update(const PagesState& state, const PagesUpdate& update, hipStream_t stream) {
  const bool with_rows = update.rows <= kFewRows;
  pages_update_kernel<<<1, kThreads, 0, stream>>>(state, update, with_rows);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || with_rows) return e;
  const Kv4Batch batch{state.table, state.lengths, update.offsets, state.batch, state.max_pages, update.rows};
  pages_rows_kernel<<<(update.rows + 255) / 256, 256, 0, stream>>>(batch, state.page_shift, state.num_pages,
                                                                  update.positions, update.slots);
  return hipGetLastError();
}

}  // namespace msim
