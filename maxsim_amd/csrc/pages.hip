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
//
// Latency bounds it: loads and scans, pages to the stack, pages from it, rows, with barriers
// between. 64 sequences that give back up to a page and get 8 tokens 4.6 us, 5.2 a call; 48 of 1,000 to
// 20,000 tokens of which a third begin anew (25,000 pages of 16 tokens change hands, 203,000 rows)
// 16.5 and 2.6 to 4.6 us, 20.3 a call. There the one workgroup's accesses, not its searches, are
// what takes the time; several would need a launch more for each barrier.
#include "pages.hpp"

namespace msim {

namespace {

constexpr int kThreads = 1024;
constexpr int kFewRows = 4096;  // of 64 sequences: 7.9 us in one launch, 8.7 for 8,192 in two
constexpr uint32_t kNoCap = ~0u;

// Inclusive scans of N sums over the workgroup's threads, each kept at its cap at most;
// `all` are the whole sums.
template <int N>
struct Scans {
  typedef uint32_t Shared[N][kThreads / kWave];  // in use until the next barrier
  uint32_t upto[N], all[N];

  __device__ __forceinline__ Scans(const uint32_t (&v)[N], const uint32_t (&cap)[N], Shared& s) {
    const int lane = lane_id(), wave = wave_uniform(threadIdx.x / kWave);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      upto[i] = wave_scan(v[i], [&](uint32_t a, uint32_t b) { return min(a + b, cap[i]); });
      if (lane == kWave - 1) s[i][wave] = upto[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t ends = wave_scan(lane < kThreads / kWave ? s[i][lane] : 0,
                                      [&](uint32_t a, uint32_t b) { return min(a + b, cap[i]); });
      all[i] = __builtin_amdgcn_readlane(ends, kThreads / kWave - 1);
      if (wave > 0) upto[i] = min(upto[i] + __builtin_amdgcn_readlane(ends, wave - 1), cap[i]);
    }
  }
};

// The sequences of a chunk whose parts of a scan hold the elements e: the first of
// `count` ends above them.
template <int N>
__device__ __forceinline__ void holders(const uint32_t* ends, int count, const uint32_t (&e)[N], int (&at)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) at[j] = 0;
  for (int n = count; n > 1; n -= n / 2)  // it is one of n from at[j] on
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (ends[at[j] + n / 2 - 1] <= e[j]) at[j] += n / 2;
}

// Elements 0 .. all of a chunk's scan, kAtOnce of a thread side by side: visit(element,
// sequence, its place in the sequence's part) gives what is stored by store(element,
// sequence, place, value). Each element's sequence is searched for.
template <int kAtOnce, typename Visit, typename Store>
__device__ __forceinline__ void by_search(const uint32_t* ends, int count, uint32_t all, Visit visit, Store store) {
  for (uint32_t e0 = 0; e0 < all; e0 += kAtOnce * kThreads) {
    uint32_t e[kAtOnce], place[kAtOnce];
    int at[kAtOnce], value[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) e[j] = min(e0 + j * kThreads + threadIdx.x, all - 1);
    holders(ends, count, e, at);
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      place[j] = e[j] - (at[j] > 0 ? ends[at[j] - 1] : 0);
      value[j] = visit(e[j], at[j], place[j]);
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if (e0 + j * kThreads + threadIdx.x < all) store(e[j], at[j], place[j], value[j]);
  }
}

// One element of a thread where that suffices (64 sequences that get a page or none: 4.6 us,
// with four 7.1), else four (25,000 elements: 16.5 us, with one 21.4; eight, or a wave per sequence
// without a search, 17.6).
template <typename Visit, typename Store>
__device__ __forceinline__ void for_elements(const uint32_t* ends, int count, uint32_t all, Visit visit, Store store) {
  if (all <= kThreads)
    by_search<1>(ends, count, all, visit, store);
  else
    by_search<4>(ends, count, all, visit, store);
}

struct Sequence {
  int kept;          // tokens
  int stay, back;    // pages that it keeps and gives back
  int64_t fresh;     // tokens asked for, within its row of the table
};
__device__ __forceinline__ Sequence sequence_of(const PagesState& st, const PagesUpdate& up, int b) {
  Sequence q = {0, 0, 0, 0};
  if (b >= st.batch) return q;
  const int64_t most = (int64_t)st.max_pages << st.page_shift;  // less than 2^31
  const int page = 1 << st.page_shift;
  const int length = (int)min((int64_t)max(st.lengths[b], 0), most);
  q.kept = up.cut == nullptr ? length : min(length, max(up.cut[b], 0));
  q.stay = (int)(((int64_t)q.kept + page - 1) >> st.page_shift);
  q.back = (int)(((int64_t)length + page - 1) >> st.page_shift) - q.stay;
  q.fresh = up.fresh == nullptr ? 0 : max(up.fresh[b], 0);
  if (q.kept + q.fresh > most) q.fresh = 0;
  return q;
}

__global__ __launch_bounds__(kThreads) void pages_update_kernel(PagesState st, PagesUpdate up, bool with_rows) {
  __shared__ Scans<3>::Shared s_three;
  __shared__ Scans<1>::Shared s_one[4];  // one for each place that scans
  __shared__ uint32_t s_end[kThreads];  // ends of the sequences' parts of a scan
  __shared__ int s_stay[kThreads], s_kept[kThreads];
  __shared__ uint32_t s_popped;
  const int tid = threadIdx.x, page = 1 << st.page_shift;
  const uint32_t cap = (uint32_t)up.rows + 1;
  auto need_of = [&](const Sequence& q, int64_t n) -> int {
    return (int)((q.kept + n + page - 1) >> st.page_shift) - q.stay;
  };
  auto entry_of = [&](int b, int column) -> int32_t& { return st.table[(int64_t)b * st.max_pages + column]; };

  if (tid == 0) s_popped = 0;
  // Scans of the first sequences: pages that come back, rows and pages asked for.
  const int had = min(max(*st.free_count, 0), st.num_pages);
  const Sequence head = sequence_of(st, up, tid);
  const uint32_t head_rows = (uint32_t)min(head.fresh, (int64_t)cap), head_need = (uint32_t)need_of(head, head.fresh);
  const Scans<3> first({(uint32_t)head.back, head_rows, head_need}, {kNoCap, cap, kNoCap}, s_three);

  // What comes back: never past the stack, whatever the lengths and the count were set to.
  uint32_t all_back = first.all[0];
  if (st.batch > kThreads) {
    uint32_t rest = 0;
    for (int b = kThreads + tid; b < st.batch; b += kThreads) rest += sequence_of(st, up, b).back;
    all_back += Scans<1>({rest}, {kNoCap}, s_one[0]).all[0];
  }
  all_back = min(all_back, (uint32_t)(st.num_pages - had));
  const uint32_t total = had + all_back;
  uint32_t before = 0;
  for (int c0 = 0; c0 < st.batch && all_back > 0; c0 += kThreads) {
    uint32_t end = first.upto[0], all = first.all[0];
    int stay = head.stay;
    if (c0 > 0) {
      const Sequence q = sequence_of(st, up, c0 + tid);
      const Scans<1> scan({(uint32_t)q.back}, {kNoCap}, s_one[1]);
      end = scan.upto[0], all = scan.all[0], stay = q.stay;
    }
    s_end[tid] = end;
    s_stay[tid] = stay;
    __syncthreads();
    for_elements(
        s_end, min(kThreads, st.batch - c0), all,
        [&](uint32_t, int i, uint32_t place) { return entry_of(c0 + i, s_stay[i] + place); },
        [&](uint32_t e, int i, uint32_t place, int32_t value) {
          if (before + e < all_back) st.free_pages[total - 1 - (before + e)] = value;
          entry_of(c0 + i, s_stay[i] + place) = -1;
        });
    before += all;
    __syncthreads();
  }

  // What is given.
  uint32_t asked_rows = 0, asked_pages = 0, rows = 0;
  for (int c0 = 0; c0 < st.batch; c0 += kThreads) {
    const int b = c0 + tid, count = min(kThreads, st.batch - c0);
    const Sequence q = c0 == 0 ? head : sequence_of(st, up, b);
    int64_t n = q.fresh;
    uint32_t end_row = first.upto[1], all_rows = first.all[1];
    if (c0 > 0) {
      const Scans<1> scan({(uint32_t)min(n, (int64_t)cap)}, {cap}, s_one[1]);
      end_row = min(asked_rows + scan.upto[0], cap), all_rows = min(asked_rows + scan.all[0], cap);
    }
    // Rows past the capacity: their sequences ask for no pages.
    const bool over = all_rows == cap;
    if (over && end_row == cap) n = 0;
    const int need = need_of(q, n);
    uint32_t end_page = first.upto[2], all_pages = first.all[2];
    if (c0 > 0 || over) {
      const Scans<1> scan({(uint32_t)need}, {kNoCap}, s_one[2]);
      end_page = scan.upto[0], all_pages = scan.all[0];
    }
    const bool given = need > 0 && asked_pages + end_page <= total;
    if (need > 0 && !given) n = 0;
    if (given) atomicMax(&s_popped, asked_pages + end_page);
    // The rows given are those asked for, or else are counted.
    uint32_t end = end_row - asked_rows, all = all_rows - asked_rows;
    if (over || asked_pages + all_pages > total) {
      const Scans<1> scan({(uint32_t)n}, {kNoCap}, s_one[3]);
      end = scan.upto[0], all = scan.all[0];
    }
    s_end[tid] = end_page;
    s_stay[tid] = q.stay;
    s_kept[tid] = q.kept;
    if (b < st.batch) {
      up.offsets[b] = (int32_t)(rows + end - (uint32_t)n);
      st.lengths[b] = q.kept + (int)n;
    }
    __syncthreads();
    const uint32_t pops = s_popped > asked_pages ? s_popped - asked_pages : 0;
    for_elements(
        s_end, count, pops,
        [&](uint32_t e, int, uint32_t) { return st.free_pages[total - 1 - (asked_pages + e)]; },
        [&](uint32_t e, int i, uint32_t place, int32_t value) {
          entry_of(c0 + i, s_stay[i] + place) = value;
          st.free_pages[total - 1 - (asked_pages + e)] = -1;
        });
    if (with_rows) {
      __syncthreads();
      s_end[tid] = end;
      __syncthreads();
      for_elements(
          s_end, count, all,
          [&](uint32_t, int i, uint32_t place) { return entry_of(c0 + i, (s_kept[i] + (int)place) >> st.page_shift); },
          [&](uint32_t e, int i, uint32_t place, int32_t value) {
            const int pos = s_kept[i] + (int)place;
            up.positions[rows + e] = pos;
            up.slots[rows + e] = (uint32_t)value < (uint32_t)st.num_pages
                                     ? ((int64_t)value << st.page_shift) + (pos & (page - 1))
                                     : -1;
          });
    }
    asked_rows = all_rows;
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
