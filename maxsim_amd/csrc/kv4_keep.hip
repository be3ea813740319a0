// kv4_keep.hip -- of the rows that a call of the cache added to each sequence, some
// stay: they move up to the end of what was there before.
//
//   row kept[b, i] of sequence b's new rows becomes its i-th, for i < count; count
//   rows of the list, which ascends, are indices of such rows, and the list ends at the
//   first entry that is none.  The length becomes length - rows + count.
//
// A workgroup has a sequence and a key/value head, and moves so many rows at a time:
// all are read before any is written.  As the list ascends, entry i is i at least, and
// no row is written before it has been read.
//
// Latency bounds it, a chain of four loads (offsets, list, page, row): 2 to 3 us for up to five
// rows of 32 sequences, 8 heads of 128; 4.6 to 5.3 for up to 61 of 64, 10 heads of 96.  Workgroups for
// each side of the rows too would halve what one moves, and double the launch.
#include "kv4.hpp"

namespace msim {

namespace {

constexpr int kThreads = 256;

template <int kDim>
__global__ __launch_bounds__(kThreads) void kv4_keep_kernel(Kv4Pool pool, Kv4Batch batch,
                                                            const int32_t* __restrict__ kept, int width,
                                                            int32_t* __restrict__ lengths) {
  constexpr int kPieces = kDim / 32;  // of 16 bytes in a row's codes
  constexpr int kRows = kThreads / (2 * kPieces);
  const int b = blockIdx.x, head = blockIdx.y, lane = lane_id();
  const int first = kv4_first_row(batch, b), rows = max(0, kv4_first_row(batch, b + 1) - first);
  const int length = kv4_length(pool, batch, b), start = length - rows;
  const int32_t* list = kept + (int64_t)b * width;

  // Every wave counts for itself.
  int count = 0;
  for (int i0 = 0; i0 < width; i0 += kWave) {
    const int i = i0 + lane;
    const int row = i < width ? list[i] : -1, before = i > 0 && i < width ? list[i - 1] : -1;
    const uint64_t ends = __ballot(row <= before || row >= rows);
    count = i0 + (ends != 0 ? __builtin_ctzll(ends) : kWave);
    if (ends != 0) break;
  }
  count = min(count, width);
  if (head == 0 && threadIdx.x == 0) lengths[b] = max(0, start + count);

  const int piece = threadIdx.x % kPieces, side = threadIdx.x / kPieces % 2;
  uint8_t* codes = side ? pool.codes[1] : pool.codes[0];
  float* scales = side ? pool.scales[1] : pool.scales[0];
  const int slot_mask = (1 << pool.page_shift) - 1;
  auto page_of = [&](int pos) -> int {
    return pos >= 0 ? batch.table[(int64_t)b * batch.max_pages + (pos >> pool.page_shift)] : -1;
  };
  for (int i0 = 0; i0 < count; i0 += kRows) {
    const int i = i0 + (int)threadIdx.x / (2 * kPieces);
    const bool have = threadIdx.x < kRows * 2 * kPieces && i < count;
    const int row = have ? list[i] : i, to = start + i, from = start + row;
    v4u words = {0, 0, 0, 0};
    float scale = 1.0f;  // a hole's rows are zeros
    bool moves = false;
    int64_t target = 0;
    if (row != i) {
      const int to_page = page_of(to), from_page = page_of(from);
      moves = (uint32_t)to_page < (uint32_t)pool.num_pages;
      target = kv4_pool_row(pool, moves ? to_page : 0, head, to & slot_mask);
      if ((uint32_t)from_page < (uint32_t)pool.num_pages) {
        const int64_t source = kv4_pool_row(pool, from_page, head, from & slot_mask);
        words = *reinterpret_cast<const v4u*>(codes + source * (kDim / 2) + piece * 16);
        scale = scales[source];
      }
    }
    // The loads are complete before any wave goes on to write.
    use_here(words);
    use_here(scale);
    __syncthreads();
    if (moves) {
      *reinterpret_cast<v4u*>(codes + target * (kDim / 2) + piece * 16) = words;
      if (piece == 0) scales[target] = scale;
    }
  }
}

}  // namespace

hipError_t launch_kv4_keep(const Kv4Pool& pool, const Kv4Batch& batch, const int32_t* kept, int width, int32_t* lengths,
                           hipStream_t stream) {
  if (batch.batch <= 0) return hipSuccess;
  const dim3 grid((unsigned)batch.batch, (unsigned)pool.kv_heads), block(kThreads);
  switch (pool.dim) {
    case 64: kv4_keep_kernel<64><<<grid, block, 0, stream>>>(pool, batch, kept, width, lengths); break;
    case 96: kv4_keep_kernel<96><<<grid, block, 0, stream>>>(pool, batch, kept, width, lengths); break;
    case 128: kv4_keep_kernel<128><<<grid, block, 0, stream>>>(pool, batch, kept, width, lengths); break;
    case 192: kv4_keep_kernel<192><<<grid, block, 0, stream>>>(pool, batch, kept, width, lengths); break;
    case 256: kv4_keep_kernel<256><<<grid, block, 0, stream>>>(pool, batch, kept, width, lengths); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace msim
