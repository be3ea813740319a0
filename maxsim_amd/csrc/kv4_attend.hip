// kv4_attend.hip -- attention of new tokens over the 4-bit key/value cache.
//
//   o = sum_j softmax_j(scale q . k_j) v_j over the keys j that the row sees,
//   k_j = c_j s_j and v_j = d_j t_j with int4 codes c, d and row scales s, t
//
// The query rows of one sequence and key/value head (its new tokens times the
// query heads that share it) are taken 16 or 32 at a time against tiles of 32
// keys.  A tile's scores are S^T = C Q^T and its part of the output is
// O^T = D^T P^T, on v_mfma_f32_16x16x32_f16 and _bf16, so that a lane keeps one query
// row throughout (column lane % 16) and the probabilities leave the first
// product in the registers in which the second one takes them:
//   * a lane's keys of the two 16-key halves, 4 g .. 4 g + 3 and 16 + the same
//     (g = lane / 16), are its eight contraction slots of the second product;
//   * a lane reads a quarter of one key's codes (its dims g dim / 4 ...) and an
//     eighth or a sixteenth of eight value rows; the words of two value rows
//     are merged by halves, so that the pairs a decoded register holds are two
//     keys of one dim.
// Keys' codes become f16 by one bitwise operation per pair (0x6400 | code ^ 8 is
// 1032 + code) and one packed subtraction or multiply-add, exactly; values' codes
// bfloat16 by a conversion each and a merge.  The key scale multiplies the score, the
// value scale the probability; nothing else is dequantised.
//
// Queries are scaled to f16 by a power of two per row, largest entry in
// [2^14, 2^15): bfloat16 entries keep all their bits down to 2^-28 of the
// largest, f16 ones too.  Single precision queries are a sum of two f16: 22 bits of
// entries down to 2^-16 of the largest, 2^-40 of the largest below, which the rounding of
// a score's sum exceeds.  A probability times its value scale is the sum of two bfloat16 (16 bits;
// single precision calls: of three, exactly), at any size that single precision
// has: with one f16 outputs to which only small products contribute lost bits, as
// happens in peaked rows, and f16 results had an error of 2.8e-4 of the norm in
// place of 2.1e-4, the rounding of the result.  The second part costs 3 % at 32
// tokens behind up to 8,000 keys, and nothing at three behind 100,000.  Scores,
// maxima, sums and outputs are single precision.
//
// Bytes bound it: dim + 8 per key and head against 4 dim operations per query
// row.  The keys of a sequence are split among workgroups when there are few
// query rows; each leaves its unnormalised sum and a second launch joins them.
// 32 heads of 128 on 8: three tokens behind 100,000 to 131,072 keys (f16) take
// 89 us, 4.3 TB/s, of which the main launch has 84 and the join 5; 32 behind 100 to
// 8,000 (bfloat16) 43 to 44 us, 3.5 TB/s (38 and 5).
//
// Windows with sinks, trees of drafts: instances of their own (kMore), so that the other
// calls keep their registers. The keys between the sinks and the window are left out of the
// tiles' count. A row of a tree sees, of its sequence's own rows, those whose bits are set in
// its line: a walk over the parents makes it, in LDS, while the first tiles come; a tile of
// 32 keys is a word of it. The walk and its barriers cost 1.5 us at 8 drafts behind 700 keys (in tiles
// of 32 rows 16.1 us against 14.3 for a causal call; of 16, as they have there, 13.9). 32 tokens,
// window 1,024 and 4 sinks 17.5 us (2.1 TB/s of the keys they see); three times three, window
// 16,384 and 300 sinks, pages of 16, 29.2 us; 7 x 27 drafts behind 133 to 3,001 keys, 12 heads
// of 64, single precision 23 us.
#include "kv4_split.hpp"

namespace msim {

namespace {

constexpr int kTileKeys = kKeyAlign;
constexpr int kFewWaves = 4;  // of a workgroup, where a CU has several
constexpr int kStages = 2;  // of a wave's ring: three or four, with as many or fewer waves, gained nothing

// Rings of tiles, and in their place the join of the waves.
constexpr int attend_lds(int dim, int cols, int waves) {
  const int rings = waves * kStages * (32 * dim + 256);
  const int join = 16 * cols * 4 * waves * (2 + dim + 4);
  return rings > join ? rings : join;
}

// Workgroups of 4 waves that a CU holds by their registers.
constexpr int waves_per_simd(Kv4Type type, int dim, int cols) {
  if (dim <= 128 && cols == 1) return 3;
  return type == kKv4F32 && dim > 192 ? 1 : 2;
}
// ------------------------------------------------------------ the main kernel

template <int kDim>
struct Shape {
  static constexpr int kKeyWords = kDim / 32;               // a lane's words of a key: dim / 4 codes
  static constexpr int kValueDims = kDim <= 64 ? 4 : (kDim <= 128 ? 8 : 16);  // a lane's dims of a value row
  static constexpr int kValueLanes = kDim / kValueDims;     // 16, or 12
  static constexpr int kTiles = kValueDims;                 // 16-dim tiles of the output
};

// A tile as it lies in LDS: [keys, values][half][16 rows], then the scales
// [keys, values][half][16].  Rows of a half are kept in the order 0, 4, 8, 12, 1,
// 5, ... so that the four rows that a value read of a wave touches are adjacent
// (no bank conflicts).
template <int kDim>
struct TileLds {
  static constexpr int kHalf = 8 * kDim;
  static constexpr int kScales = 4 * kHalf;
  static constexpr int kBytes = kScales + 256;
  static constexpr int kHalfLoads = (kHalf + 1023) / 1024;
  static constexpr int kLoads = 4 * kHalfLoads + 1;  // of a wave, per tile
};

// Page numbers of a tile's halves (pages hold 16 rows or a multiple, so a half
// lies in one page); -1 past the sequence's end.
struct TilePages {
  int page[2];
};
__device__ __forceinline__ TilePages tile_pages(const Kv4Pool& pool, const Kv4Batch& batch, int seq, int length, int key0) {
  TilePages p;
  const auto* table = as_constant(batch.table) + (int64_t)seq * batch.max_pages;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int key = key0 + 16 * h;
    p.page[h] = key < length ? table[key >> pool.page_shift] : -1;
  }
  return p;
}

// Starts a tile's way to LDS (kLoads loads); holes come from page 0.
template <int kDim>
__device__ __forceinline__ void load_tile(const Kv4Pool& pool, const TilePages& pages, int head, int key0,
                                          uint32_t lds) {
  typedef TileLds<kDim> L;
  constexpr int kChunks = kDim / 32;  // of 16 bytes in a row
  const int lane = lane_id();
  int64_t at[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int page = (uint32_t)pages.page[h] < (uint32_t)pool.num_pages ? pages.page[h] : 0;
    at[h] = kv4_pool_row(pool, page, head, (key0 + 16 * h) & ((1 << pool.page_shift) - 1));
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const v4i rsrc = make_rsrc_words(pool.codes[side] + at[h] * (kDim / 2), L::kHalf);
#pragma unroll
      for (int i = 0; i < L::kHalfLoads; ++i) {
        const int chunk = i * kWave + lane, place = chunk / kChunks;
        const int row = place % 4 * 4 + place / 4;
        if (L::kHalf % 1024 == 0 || chunk < L::kHalf / 16)
          lds_load_b128(rsrc, row * (kDim / 2) + chunk % kChunks * 16, lds + (side * 2 + h) * L::kHalf + i * 1024);
      }
    }
  }
  const float* scales = lane & 32 ? pool.scales[1] : pool.scales[0];
  lds_load_b32_global(scales + (lane & 16 ? at[1] : at[0]) + lane % 16, lds + L::kScales);
}

__device__ __forceinline__ float across_groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float across_groups_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Granules from .. upto of an item.  kCols 16-row column tiles of queries per
// workgroup; its waves take the key tiles in turn.
//
// kMore: calls with sinks or parents. Keys are numbered as TileRange says then, else by
// themselves.
template <Kv4Type T, int kDim, int kCols, bool kMore, int kWaves>
__device__ __forceinline__ void attend_item(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args,
                                            const Split& split, float* __restrict__ partial, const Cursor<kMore>& at,
                                            uint32_t from, uint32_t upto) {
  typedef Shape<kDim> S;
  constexpr int kParts = T == kKv4F32 ? 2 : 1;      // of a query
  constexpr int kProbParts = T == kKv4F32 ? 3 : 2;  // of a probability times its value scale
  constexpr int kRows = 16 * kCols;
  __shared__ __attribute__((aligned(16))) char s_raw[attend_lds(kDim, kCols, kWaves)];
  const int lane = lane_id(), col = lane % 16, g = lane / 16, wave = wave_uniform(threadIdx.x / kWave);
  const SeqWork& u = at.work;
  const uint32_t tile = at.tile;
  const int seq = at.seq, head = at.head;

  // With parents: of each row of the tile the rows that it comes after and itself, as bits
  // of the words of 32 keys from first_word on, and how many it comes after.
  constexpr int kLineWords = kMostDrafts / 32 + 1;  // odd: the lines spread over the banks
  __shared__ uint32_t s_line[kMore ? kRows * kLineWords : 1];
  __shared__ int s_parent[kMore ? kMostDrafts : 1], s_depth[kMore ? kRows : 1];
  const bool tree = kMore && args.parents != nullptr;
  const int start = u.length - u.rows;  // the first row's position
  const int first_word = start & -32, drafts = min(u.rows, kMostDrafts);
  constexpr int kTurns = (kMostDrafts + kWaves * kWave - 1) / (kWaves * kWave);
  int parents[kMore ? kTurns : 1];
  if (tree) {
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int row = i * kWaves * kWave + (int)threadIdx.x;
      if (row < drafts) parents[i] = args.parents[u.first + row];
    }
  }

  // Query rows of this tile: row r is new token r / share, head r % share.
  v8h q[kCols][kParts][S::kKeyWords];
  float factor[kCols];       // of a product with the codes, towards log2 scores
  int see_low[kCols], see_high[kCols];
  const uint8_t* mask[kCols];
  int64_t query[kCols];  // first element of the lane's row; -1: a row of padding
  int all_low = 0, all_high = INT_MAX, any_low = INT_MAX, any_high = 0;
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    const uint32_t r = tile * kRows + 16 * c + col;
    const int token = (int)(r / split.share), sub = (int)(r - token * split.share);
    const bool have = token < u.rows;
    query[c] = have ? (int64_t)(u.first + token) * args.q_row_stride +
                          (int64_t)(head * split.share + sub) * args.q_head_stride
                    : -1;
    const int pos = start + token;
    see_low[c] = !tree && pos >= args.window ? pos - args.window + 1 : 0;
    see_high[c] = args.causal ? max(0, min(u.length, pos + 1)) : u.length;
    if (tree && u.rows > kMostDrafts) see_high[c] = 0;
    mask[c] = nullptr;
    if (args.mask != nullptr) {
      see_high[c] = (int)min((int64_t)see_high[c], args.mask_width);
      mask[c] = args.mask + (have ? (int64_t)(u.first + token) * args.mask_row_stride : 0);
    }
    if (!have) {  // nothing depends on what it sees
      see_low[c] = 0;
      see_high[c] = args.mask != nullptr ? 0 : INT_MAX;
    } else if (kMore ? see_high[c] > 0 : see_high[c] > see_low[c]) {
      any_low = min(any_low, see_low[c]);
      any_high = max(any_high, see_high[c]);
    }
    all_low = max(all_low, see_low[c]);
    all_high = min(all_high, see_high[c]);
  }
  all_low = wave_reduce(all_low, [](int a, int b) { return max(a, b); });
  all_high = wave_reduce(all_high, [](int a, int b) { return min(a, b); });
  any_low = wave_reduce(any_low, [](int a, int b) { return min(a, b); });
  any_high = wave_reduce(any_high, [](int a, int b) { return max(a, b); });
  if (tree) all_high = min(all_high, max(0, start));  // up to where all rows see all that the window leaves
  // This worker's keys of the item, cut to what some row sees.
  const int low = kMore ? 0 : at.range.low;
  auto key_of = [&](int number) -> int { return kMore ? at.range.key_of(number) : number; };
  const int begin = kMore ? (int)(from << split.granule_shift)
                          : max(low + (int)(from << split.granule_shift), min(any_low, u.length) / kTileKeys * kTileKeys);
  const int end = (int)min((int64_t)low + ((int64_t)upto << split.granule_shift),
                           (int64_t)(kMore ? at.range.number_of(any_high) : any_high));

  // A ring of tiles per wave: kStages - 1 of them on their way while one is
  // worked on.
  typedef TileLds<kDim> L;
  constexpr int kStep = kWaves * kTileKeys, kAhead = kStages - 1;
  const int key_first = begin + wave * kTileKeys;
  const int tiles = end > key_first ? (end - key_first + kStep - 1) / kStep : 0;
  const char* ring = s_raw + wave * kStages * L::kBytes;
  const uint32_t ring_lds = lds_address(ring);
  // The lines are needed where the worker comes to the rows' own keys, and for a window.
  const bool lines = tree && end > begin && (end > at.range.number_of(start) || args.window != INT_MAX);
  bool hole[kStages][2];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int key = key_of(key_first + i * kStep);
    const TilePages pages = tile_pages(pool, batch, seq, u.length, key);
    if (kMore && i == 0 && lines) {  // before the tiles, or their arrival is waited for
#pragma unroll
      for (int j = 0; j < kTurns; ++j) {
        const int row = j * kWaves * kWave + (int)threadIdx.x;
        if (row < drafts) s_parent[row] = parents[j];
      }
      for (int j = threadIdx.x; j < kRows * kLineWords; j += kWaves * kWave) s_line[j] = 0;
    }
    if (i < tiles) load_tile<kDim>(pool, pages, head, key, ring_lds + i * L::kBytes);
    hole[i][0] = (uint32_t)pages.page[0] >= (uint32_t)pool.num_pages;
    hole[i][1] = (uint32_t)pages.page[1] >= (uint32_t)pool.num_pages;
  }

  // The lines and the queries, while the first tiles come.
  if (kMore && lines) {
    group_sync_lds();
    if (threadIdx.x < kRows) {
      const int token = (int)((tile * kRows + threadIdx.x) / split.share);
      int depth = 0;
      if (token < drafts) {
        if (args.window != INT_MAX)
          for (int row = row_before(s_parent, token); row >= 0; row = row_before(s_parent, row)) ++depth;
        int back = 0;
        for (int row = token; row >= 0; row = row_before(s_parent, row), ++back) {
          const int at = start + row - first_word;
          if (back < args.window || start + depth - back < args.sinks)
            s_line[threadIdx.x * kLineWords + at / 32] |= 1u << at % 32;
        }
      }
      s_depth[threadIdx.x] = depth;
    }
    group_sync_lds();
    if (args.window != INT_MAX) {
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const int pos = start + s_depth[16 * c + col];
        see_low[c] = query[c] >= 0 && pos >= args.window ? pos - args.window + 1 : 0;
        all_low = max(all_low, see_low[c]);
      }
      all_low = wave_reduce(all_low, [](int a, int b) { return max(a, b); });
    }
  }
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    float x[S::kKeyWords][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < S::kKeyWords; ++i) {
      float y[8];
      load8<T>(args.q, max(query[c], (int64_t)0) + g * (kDim / 4) + i * 8, args.q_wide != 0, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[i][j] = query[c] >= 0 ? y[word_order(j)] : 0.0f;
        top = max(top, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
      }
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    const int shift = query_shift(top);
#pragma unroll
    for (int i = 0; i < S::kKeyWords; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // The factor towards log2 scores is kept positive: maxima are taken before it.
        const float y = ldexpf(args.scale_log2 < 0.0f ? -x[i][j] : x[i][j], shift);
        const _Float16 hi = (_Float16)y;
        q[c][0][i][j] = hi;
        if constexpr (kParts == 2) q[c][1][i][j] = (_Float16)(y - (float)hi);
      }
    factor[c] = score_factor(args.scale_log2, shift);
  }

  float ref[kCols], sum[kCols];
  v4f o[kCols][S::kTiles];
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    ref[c] = kUnset;
    sum[c] = 0.0f;
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t) o[c][t] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
  }

  TilePages pages = tile_pages(pool, batch, seq, u.length, key_of(key_first + kAhead * kStep));
  uint32_t seen[kCols][2];  // mask bytes of the tile's keys of this lane
  auto load_mask = [&](int key0) {
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        seen[c][h] = mask_bytes(mask[c], key0 + 16 * h + 4 * g, see_high[c]);
  };
  if (args.mask != nullptr) load_mask(key_of(key_first));
  int slot = 0, fill = kAhead * L::kBytes;  // offsets in the ring
  for (int n = 0; n < tiles; ++n) {
    const int number = key_first + n * kStep, key0 = key_of(number);
    hole[kAhead][0] = (uint32_t)pages.page[0] >= (uint32_t)pool.num_pages;
    hole[kAhead][1] = (uint32_t)pages.page[1] >= (uint32_t)pool.num_pages;
    if (n + kAhead < tiles) {
      load_tile<kDim>(pool, pages, head, key_of(number + kAhead * kStep), ring_lds + fill);
      vm_wait_lds<kAhead * L::kLoads>();
    } else {
      vm_wait_lds<0>();
    }
    // The page numbers of the tile after that.
    pages = tile_pages(pool, batch, seq, u.length, key_of(number + (kAhead + 1) * kStep));
    const char* now = ring + slot;
    slot = slot + L::kBytes == kStages * L::kBytes ? 0 : slot + L::kBytes;
    fill = fill + L::kBytes == kStages * L::kBytes ? 0 : fill + L::kBytes;

    // Scores of the tile.
    v4f s[kCols][2];
#pragma unroll
    for (int c = 0; c < kCols; ++c) s[c][0] = s[c][1] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t words[S::kKeyWords];
      const int place = col % 4 * 4 + col / 4;
      const uint32_t* src =
          reinterpret_cast<const uint32_t*>(now + h * L::kHalf + place * (kDim / 2) + g * (kDim / 8));
      if constexpr (S::kKeyWords % 4 == 0) {
#pragma unroll
        for (int i = 0; i < S::kKeyWords / 4; ++i) {
          const v4u w = reinterpret_cast<const v4u*>(src)[i];
#pragma unroll
          for (int j = 0; j < 4; ++j) words[4 * i + j] = w[j];
        }
      } else {
#pragma unroll
        for (int i = 0; i < S::kKeyWords; ++i) words[i] = src[i];
      }
#pragma unroll
      for (int i = 0; i < S::kKeyWords; ++i) {
        const v8h a = decode_word(words[i]);
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int p = 0; p < kParts; ++p)
            s[c][h] = mfma(a, q[c][p][i], s[c][h]);
      }
    }
    v4f key_scale[2], value_scale[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const v4f* scales = reinterpret_cast<const v4f*>(now + L::kScales + h * 64);
      key_scale[h] = scales[g];
      value_scale[h] = scales[8 + g] * (1.0f / kValueUnit);
    }
    mfma_results_fence();

    const bool whole = (key0 >= all_low || (kMore && key0 + kTileKeys <= args.sinks)) && key0 + kTileKeys <= all_high &&
                       args.mask == nullptr && !hole[0][0] && !hole[0][1];
    v8b probs[kCols][kProbParts];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      float x[8], vs[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = s[c][i / 4][i % 4] * key_scale[i / 4][i % 4];
        vs[i] = value_scale[i / 4][i % 4];
      }
      if (!whole) {
        // A hidden key takes no part in the maxima, and its probability and
        // value scale are zeros whatever the cache holds there.
        const bool own = tree && key0 >= first_word;  // some keys of the tile are the sequence's rows
        const uint32_t line = own ? s_line[(16 * c + col) * kLineWords + (key0 - first_word) / 32] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int local = 16 * (i / 4) + 4 * g + i % 4, key = key0 + local;
          bool see = key >= see_low[c] || (kMore && key < args.sinks);
          if (own && key >= start) see = (line >> local & 1u) != 0;
          see = see && key < see_high[c] && !hole[0][i / 4];
          if (args.mask != nullptr) see = see && (seen[c][i / 4] >> (8 * (i % 4)) & 0xFFu) != 0;
          x[i] = see ? x[i] : kNegInf;
          vs[i] = see ? vs[i] : 0.0f;
        }
      }
      const float top = max_of(x) * factor[c];
      if (__ballot(top > ref[c] + kTopLimit) != 0) {
        const float now = fmaxf(ref[c], across_groups_max(top));
        const float alpha = exp2_hw(ref[c] - now);
        ref[c] = now;
        sum[c] *= alpha;
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) o[c][t] *= alpha;
      }
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = exp2_hw(__builtin_fmaf(x[i], factor[c], -ref[c]));
        sum[c] += p;
        y[i] = p * vs[i];
      }
      in_parts(y, probs[c]);
    }

    // The tile's part of the output: the codes of two keys side by side.
#pragma unroll
    for (int k = 0; k < (S::kValueDims + 7) / 8; ++k) {
      uint32_t low[4], high[4];
      const int vl = S::kValueLanes == 16 ? col : min(col, S::kValueLanes - 1);
      auto value = [&](int h, int r) -> uint32_t {
        const char* src = now + (2 + h) * L::kHalf + (4 * r + g) * (kDim / 2) + vl * (S::kValueDims / 2) + 4 * k;
        if constexpr (S::kValueDims == 4) return *reinterpret_cast<const uint16_t*>(src);
        return *reinterpret_cast<const uint32_t*>(src);
      };
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint32_t a = value(p / 2, 2 * (p % 2)), b = value(p / 2, 2 * (p % 2) + 1);
        low[p] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        high[p] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      }
#pragma unroll
      for (int half = 0; half < (S::kValueDims >= 8 ? 2 : 1); ++half) {
        v8b pair[4];  // [pair of keys]: four dims of both
#pragma unroll
        for (int p = 0; p < 4; ++p) pair[p] = decode_word_bf16(half ? high[p] : low[p]);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          v8b a;
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            a[2 * p] = pair[p][2 * d];
            a[2 * p + 1] = pair[p][2 * d + 1];
          }
#pragma unroll
          for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int p = 0; p < kProbParts; ++p) {
              v4f& acc = o[c][k * 8 + half * 4 + d];
              acc = mfma(a, probs[c][p], acc);
            }
        }
      }
    }
    if (args.mask != nullptr) load_mask(key_of(number + kStep));
    // All reads of the slot are behind this point: the next turn fills it.
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int t = 0; t < S::kTiles; ++t) asm volatile("" : "+v"(o[c][t]));
#pragma unroll
    for (int i = 0; i < kAhead; ++i) hole[i][0] = hole[i + 1][0], hole[i][1] = hole[i + 1][1];
  }
  mfma_results_fence();

  // The waves' results joined in their order, in LDS.
  float* s_ref = reinterpret_cast<float*>(s_raw);  // [waves][rows]
  float* s_sum = s_ref + kWaves * kRows;           // [waves][rows]
  float* s_o = s_sum + kWaves * kRows;             // [waves][rows][dim + 4]
  constexpr int kPitch = kDim + 4;                 // spreads the rows over the banks
#pragma unroll
  for (int c = 0; c < kCols; ++c) sum[c] = across_groups_sum(sum[c]);
  __syncthreads();  // the rings have been read
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    const int r = wave * kRows + 16 * c + col;
    if (g == 0) s_ref[r] = ref[c], s_sum[r] = sum[c];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * g + i < S::kValueLanes) {
        v4f* dst = reinterpret_cast<v4f*>(s_o + r * kPitch + (4 * g + i) * S::kValueDims);
#pragma unroll
        for (int t = 0; t < S::kTiles / 4; ++t)
          dst[t] = (v4f){o[c][4 * t][i], o[c][4 * t + 1][i], o[c][4 * t + 2][i], o[c][4 * t + 3][i]};
      }
  }
  __syncthreads();
  const bool whole_item = from == 0 && upto == at.range.granules;
  constexpr int kPerRow = kDim / 4;
  for (int i = threadIdx.x; i < kRows * kPerRow; i += kWaves * kWave) {
    const int local = i / kPerRow, d = i % kPerRow * 4;
    const uint32_t r = tile * kRows + local;
    const int token = (int)(r / split.share), sub = (int)(r - token * split.share);
    if (token >= u.rows) continue;
    float all = s_ref[local];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) all = fmaxf(all, s_ref[w * kRows + local]);
    float total = 0.0f;
    v4f sum4 = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float alpha = exp2_hw(s_ref[w * kRows + local] - all);
      total += s_sum[w * kRows + local] * alpha;
      sum4 += *reinterpret_cast<const v4f*>(s_o + (w * kRows + local) * kPitch + d) * alpha;
    }
    if (!whole_item) {
      float* dst = partial_slot(partial, split, kDim, blockIdx.x, from == 0);
      *reinterpret_cast<v4f*>(dst + local * kDim + d) = sum4;
      if (d == 0) {
        dst[kRows * kDim + 2 * local] = all;
        dst[kRows * kDim + 2 * local + 1] = total;
      }
      continue;
    }
    const int qh = head * split.share + sub;
    const int64_t row = u.first + token;
    if (args.lse != nullptr && d == 0)
      args.lse[row * args.heads + qh] = log_sum(all, total);
    sum4 *= output_factor(total);
    store4<T>(args.out, row * args.out_row_stride + (int64_t)qh * args.out_head_stride + d, args.out_wide != 0, sum4);
  }
}

// Worker blockIdx.x's granules, item by item.
template <Kv4Type T, int kDim, int kCols, bool kMore, int kWaves>
__global__ __launch_bounds__(kWaves* kWave, waves_per_simd(T, kDim, kCols)) void kv4_attend_kernel(
    Kv4Pool pool, Kv4Batch batch, Kv4AttendArgs args, Split split, float* __restrict__ partial) {
  if (__builtin_expect(blockIdx.x >= split.workers, 0)) {
    loose_rows<T, kDim>(batch, args, split);
    return;
  }
  Deal deal;
  Cursor<kMore> at;
  if (!find_work<kMore>(pool, batch, args, split, blockIdx.x, at, deal)) {
    note_unfinished(partial, split, kDim, at, 0);
    return;
  }
  uint32_t granule = deal.begin(blockIdx.x);
  const uint32_t last = deal.begin(blockIdx.x + 1);
  int parts = 0;
  while (granule < last && at.seek(pool, batch, args, split, granule)) {
    const uint32_t size = at.range.granules + lead_of<kMore>(split), stop = min(size, last - at.item_at);
    const uint32_t from = at.own(split, granule - at.item_at), upto = at.own(split, stop);
    granule = at.item_at + stop;
    if (kMore && from == upto) continue;
    attend_item<T, kDim, kCols, kMore, kWaves>(pool, batch, args, split, partial, at, from, upto);
    if (from == 0 && upto < at.range.granules)
      parts = (int)(deal.worker_of(at.item_at + size - 1) - blockIdx.x) + 1;
    __syncthreads();
  }
  note_unfinished(partial, split, kDim, at, parts);
}

constexpr int kJoinWaves = 4;

// Joins the parts of split items. Of an item of up to kDirect parts each wave joins a row
// by itself, and a workgroup has four rows of it; of more, each wave adds up every
// kJoinWaves-th part and the waves' sums are joined, and a workgroup has one row. Where many
// workgroups would find nothing to do, fewer count the pieces of work in the list of parts
// and take them in turn (kCounted).
template <Kv4Type T, int kDim, bool kCounted>
__global__ __launch_bounds__(kJoinWaves* kWave) void kv4_join_kernel(Kv4AttendArgs args, Split split, uint32_t rows,
                                                                 float* __restrict__ partial) {
  constexpr int kRegs = (kDim + 63) / 64;
  constexpr int kDirect = kWave / kJoinWaves;
  __shared__ float s_part[kJoinWaves][kDim + 1];
  __shared__ uint32_t s_end[kJoinWaves], s_worker, s_piece;
  __shared__ int s_parts;
  const int wave = wave_uniform(threadIdx.x / kWave), lane = lane_id();
  const Unfinished* items = reinterpret_cast<const Unfinished*>(partial + partial_floats(split, kDim));
  const int* counts = reinterpret_cast<const int*>(items + split.workers);
  auto pieces = [&](int parts) -> uint32_t {
    return parts == 0 ? 0 : (parts <= kDirect ? (rows + kJoinWaves - 1) / kJoinWaves : rows);
  };
  // A thread counts the pieces of kEach workers.
  constexpr uint32_t kEach = kMostWorkers / (kJoinWaves * kWave);
  int have_parts[kEach] = {};
  uint32_t mine = 0, before = 0, all_pieces = 0;
  if constexpr (kCounted) {
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      const uint32_t worker = threadIdx.x * kEach + i;
      have_parts[i] = worker < split.workers ? counts[worker] : 0;
      mine += pieces(have_parts[i]);
    }
    const uint32_t upto = wave_scan(mine);
    if (lane == kWave - 1) s_end[wave] = upto;
    __syncthreads();
    before = upto - mine;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) {
      if (w < wave) before += s_end[w];
      all_pieces += s_end[w];
    }
  }
  // Without counting, workgroup (i, y) has the pieces y, y + gridDim.y, ... of worker i.
  const int own_parts = kCounted ? 0 : counts[blockIdx.x];
  const uint32_t step = kCounted ? gridDim.x : gridDim.y;
  if (!kCounted) all_pieces = pieces(own_parts);
  for (uint32_t work = kCounted ? blockIdx.x : blockIdx.y; work < all_pieces; work += step) {
    if (kCounted && work >= before && work < before + mine) {
      uint32_t piece = work - before;
      bool found = false;
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t n = pieces(have_parts[i]);
        if (!found && piece < n) {
          found = true;
          s_worker = threadIdx.x * kEach + i;
          s_parts = have_parts[i];
          s_piece = piece;
        }
        piece -= found ? 0 : n;
      }
    }
    if (kCounted) __syncthreads();
    const uint32_t first = kCounted ? wave_uniform(s_worker) : blockIdx.x;
    const uint32_t piece = kCounted ? wave_uniform(s_piece) : work;
    const int parts = min(kCounted ? wave_uniform(s_parts) : own_parts, (int)(split.workers - first));
    const Unfinished item = items[first];
    const bool direct = parts <= kDirect;
    const int start = direct ? 0 : wave, stride = direct ? 1 : kJoinWaves;
    const uint32_t local = direct ? piece * kJoinWaves + wave : piece;
    const uint32_t r = (item.tile << split.tile_shift) + local;
    const int token = (int)(r / split.share), qh = item.head * split.share + (int)(r - token * split.share);
    if (kCounted) __syncthreads();  // the next piece may be written
    // Without barriers in them for single waves: a row is a wave's, or all waves agree on it.
    if (local >= rows || token >= item.rows) continue;
    float all = kUnset, total = 0.0f, o[kRegs] = {};
    for (int p0 = 0; p0 < parts; p0 += kWave) {
      const int count = min(kWave, parts - p0);
      auto slot = [&](int p) -> const float* {
        return partial_slot(partial, split, kDim, first + p0 + p, p0 + p == 0);
      };
      const bool have = lane < count;
      const float* sums = slot(have ? lane : 0) + ((int64_t)kDim << split.tile_shift) + 2 * local;
      const float ref = have ? sums[0] : kUnset, share = have ? sums[1] : 0.0f;
      // All loads of the wave's parts go out before the weights are known.
      float part[kDirect][kRegs];
#pragma unroll
      for (int i = 0; i < kDirect; ++i) {
        const int p = i * stride + start;
        if (p >= count) break;
        const float* src = slot(p) + local * kDim;
#pragma unroll
        for (int k = 0; k < kRegs; ++k) part[i][k] = src[min(k * 64 + lane, kDim - 1)];
      }
      const float now = fmaxf(all, wave_reduce(ref, [](float a, float b) { return fmaxf(a, b); }));
      const float old = exp2_hw(all - now), alpha = exp2_hw(ref - now);
      all = now;
      const float weighed = direct || lane % kJoinWaves == wave ? share * alpha : 0.0f;
      total = total * old + wave_reduce(weighed, [](float a, float b) { return a + b; });
#pragma unroll
      for (int k = 0; k < kRegs; ++k) o[k] *= old;
#pragma unroll
      for (int i = 0; i < kDirect; ++i) {
        const int p = i * stride + start;
        if (p >= count) break;
        const float a = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(alpha), p));
#pragma unroll
        for (int k = 0; k < kRegs; ++k) o[k] = __builtin_fmaf(part[i][k], a, o[k]);
      }
    }
    if (!direct) {
#pragma unroll
      for (int k = 0; k < kRegs; ++k)
        if (k * 64 + lane < kDim) s_part[wave][k * 64 + lane] = o[k];
      if (lane == 0) s_part[wave][kDim] = total;
      __syncthreads();
      total = 0.0f;
#pragma unroll
      for (int k = 0; k < kRegs; ++k) o[k] = 0.0f;
#pragma unroll
      for (int w = 0; w < kJoinWaves; ++w) {
        total += s_part[w][kDim];
#pragma unroll
        for (int k = 0; k < kRegs; ++k) o[k] += s_part[w][min(k * 64 + lane, kDim - 1)];
      }
      __syncthreads();
    }
    if (direct || wave == 0) {
      const int64_t row = item.first + token;
      const float inv = output_factor(total);
      if (args.lse != nullptr && lane == 0) args.lse[row * args.heads + qh] = log_sum(all, total);
      const int64_t base = row * args.out_row_stride + (int64_t)qh * args.out_head_stride;
#pragma unroll
      for (int k = 0; k < kRegs; ++k)
        if (k * 64 + lane < kDim) store_out<T>(args.out, base + k * 64 + lane, o[k] * inv);
    }
  }
}

// Column tiles per workgroup: as many as a sequence's rows fill on average (one
// for wide heads, whose outputs take the registers). At 8 sequences of 4,000 keys,
// 32 heads of 128 on 8, two took 30.2 us for 5 tokens each and one 32.0; 32.7 and
// 33.3 for 8; 38.2 and 41.7 for 16.  With sinks or parents split_for takes one for
// shorter work.
int columns_for(const Kv4Pool& pool, const Kv4Batch& batch, int heads) {
  const int64_t rows = (int64_t)batch.rows * (heads / pool.kv_heads) / std::max(1, batch.batch);
  return rows <= 16 || pool.dim > 128 ? 1 : 2;
}

// Workgroups that the CUs hold at once.
uint32_t workers_for(Kv4Type type, int dim, int columns, int num_cus) {
  return std::min<uint32_t>(num_cus * waves_per_simd(type, dim, columns), kMostWorkers);
}

// `args` nullptr: any call with or without parents, of those that need a workspace. `prompts`
// false: not by kv4_prompt.hip.
Split split_for(const Kv4Pool& pool, const Kv4Batch& batch, int heads, Kv4Type type, bool parents,
                const Kv4AttendArgs* args, int num_cus, bool prompts = true) {
  Split s{};
  const bool prompt = prompts && kv4_prompt_takes(pool, batch, heads, type, parents, num_cus);
  if (prompt) {
    s = kv4_prompt_split(num_cus);
  } else {
    const int columns = columns_for(pool, batch, heads);
    s.tile_shift = columns == 2 ? 5 : 4;
    s.workers = workers_for(type, pool.dim, columns, num_cus);
    // A granule each is the shortest way while every CU has one workgroup (one token
    // behind 1,000 keys: 12.2 us against 13.2).
    s.few = num_cus;
  }
  s.share = heads / pool.kv_heads;
  const int64_t longest = (int64_t)batch.max_pages << pool.page_shift;
  s.one_launch = longest <= kShort;
  int64_t whole = kShort;  // keys of a granule that is an item
  const bool more = args != nullptr && (args->sinks > 0 || parents);
  if (more && !prompt) {
    // Of these calls, whose keys a window may count, items stay whole where there are many for
    // their length. A tree's keys are the table's, so the rules hold where tables are as wide as
    // the sequences; behind wider ones trees go the way of longer contexts (8 x 8 drafts behind 1,400
    // keys, table for 131,072 tokens, 23.4 us, trimmed 19.3). 32 heads of 128 on 8, one token of a
    // sequence, by the window:
    //   up to 512 keys always: of 4 sequences 11.6 us against 12.8 split, of 64 14.4 against 21;
    //   a workgroup for each CU, with all the waves it holds, from 7 items for each granule of one,
    //   and 10 where the longest sequence alone bounds them, others being shorter:
    //     1,024 keys of 8 sequences 16.5 against 15.6, of 16 16.5 against 18.2, of 32 17.5 against 23;
    //     2,048 of 16 21.8 against 21.9, of 32 22.6 against 27.7; 4,096 of 32 35 against 41, but of
    //     100 to 4,200 tokens 34.5 against 30; 8 tokens of 32, 2,048, 31 against 45;
    //   their tiles have 16 rows if that gives no more items than CUs, for the more items and waves
    //     (32 rows in brackets): 8 drafts of 8 sequences, 1,400 keys, 19.2 (23.6), of 16 at 500 to
    //     2,000 23.0 (29.7), 64 of one at 1,400 20.4 (24.8); 16 tokens of 8, 2,048, 23.3 (29.6);
    //     8 drafts of 16 behind 100 to 2,500, 3,000 and 3,500 keys, 12.8, 10.7 and 9.1 items for a
    //     granule, 25.4, 29.3 and 31.7 against 28.5, 29.5 and 30.6 split;
    //   16 rows too where every granule, or short item, then has a workgroup at once: 8 drafts of one
    //     sequence, 100 keys, 10.1 (12.3), 400 13.6 (17.2), 700 14.6 (16.7), 3,500 16.6 (17.3), of four
    //     at 1,400 18.6 (19.6);
    //   more items than CUs from 16 on, the usual workgroups: 1,024 of 64 25 against 32, 2,048
    //     38 against 42, 4,096 of 100 to 4,200 tokens 54 against 46.
    int64_t keys = 0, granules = 0, whole_items = 0;
    auto count = [&](uint32_t tile_shift) {
      keys = longest;
      if (args->causal && !parents)
        keys = std::min(keys, (int64_t)args->window + (1 << tile_shift) / s.share + 2 + args->sinks + 2 * kKeyAlign);
      granules = (keys + kGranule - 1) / kGranule;
      const int64_t each = (int64_t)batch.rows * s.share / std::max(1, batch.batch);
      whole_items = ((each + (1 << tile_shift) - 1) >> tile_shift) * batch.batch * pool.kv_heads;
      s.whole_cu = keys > kShort && granules <= 33 && waves_per_simd(type, pool.dim, tile_shift == 5 ? 2 : 1) > 1 &&
                   whole_items <= num_cus && whole_items >= (keys == longest ? 10 : 7) * granules;
      return s.whole_cu;
    };
    const int at_once = workers_for(type, pool.dim, 1, num_cus);
    if (count(4) || (s.tile_shift == 5 && whole_items * (keys <= kShort ? 1 : granules) <= at_once)) {
      s.tile_shift = 4;
      s.workers = at_once;
    } else if (s.tile_shift == 5) {
      count(5);
    }
    if (s.whole_cu) s.workers = num_cus;
    s.one_launch = keys <= kShort || s.whole_cu || (granules <= 17 && whole_items >= 16 * granules);
    while (whole < keys && s.one_launch) whole *= 2;
  }
  // An item costs its worker as much as four granules besides its own (queries, the waves' join):
  // 32 x 16 drafts behind 100 to 4,000 keys take 74 us, dealt out by granules alone 134; 4 x 500
  // tokens behind 100 to 9,000, window 4,096, 221 and 349.
  if (more && !s.one_launch) s.lead = 4;
  if (s.one_launch) s.few = s.workers;
  s.granule_shift = __builtin_ctzll(s.one_launch ? whole : kGranule);
  const int64_t items = (((int64_t)batch.rows * s.share >> s.tile_shift) + batch.batch) * pool.kv_heads;
  while (items * ((longest >> s.granule_shift) + 1 + s.lead) >= (int64_t)1 << 31) ++s.granule_shift;
  return s;
}

// What a call of such a split leaves for the join.
size_t split_bytes(const Split& s, int dim) {
  return s.one_launch ? 0 : partial_floats(s, dim) * sizeof(float) + s.workers * (sizeof(Unfinished) + sizeof(int));
}

template <Kv4Type T, int kDim>
hipError_t launch_join(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args, const Split& split,
                       float* partial, int num_cus, hipStream_t stream) {
  // Without offsets a tile has as many rows as heads share a key/value head.
  const uint32_t rows = std::min(1u << split.tile_shift, batch.offsets == nullptr ? split.share : UINT32_MAX);
  // A few workgroups for each worker, or four for each CU that count the pieces of work. Counting
  // costs 0.7 us (768 workers with 1 row 10.5 us against 11.2, with 6 rows 10.4 against 11.1) and
  // saves workgroups that would find nothing: 512 with 16 rows, 14 items, 18.1 us against 15.7; 512
  // with 32, up to 128 items, 2.5 us; 256 with 32 each of 256, up to 128 items, 5. It saves none
  // where there may be a piece for each (4 x 400 tokens behind 2,100, 32 heads of 128: 141 us, counted
  // 151), and under a window, where fewer items than workers are short and all of them split, few
  // (32 x 5 tokens, window 300: 28.3, counted 29.8). The workgroups of an item are all on one XCD,
  // so few items of a megabyte and more are counted too (8 heads of 256 on 1, single precision, 30,000
  // keys, 2 MB: 31.3, counted 20.0; 12 heads of 64 on 2, 360 kB: 16.5 against 17.2).
  const uint32_t y = std::min(32u, rows);
  const uint64_t groups = (uint64_t)split.workers * y;
  const uint64_t items = (((uint64_t)batch.rows * split.share >> split.tile_shift) + batch.batch) * pool.kv_heads;
  const uint64_t pieces = std::min<uint64_t>(items, split.workers) * ((rows + kJoinWaves - 1) / kJoinWaves);
  const int64_t longest = (int64_t)batch.max_pages << pool.page_shift;
  const int64_t keys = args.causal && args.parents == nullptr ? std::min<int64_t>(longest, args.window) : longest;
  const uint64_t parts =
      std::min<uint64_t>((keys >> split.granule_shift) + 1, split.workers / std::max<uint64_t>(items, 1));
  const bool all_split = args.window != INT_MAX && items < split.workers;
  const dim3 block(kJoinWaves * kWave);
  if ((groups > 6144 && pieces < (all_split ? groups / 12 : groups)) ||
      (items < 8 && parts * rows * kDim * sizeof(float) >= 1 << 20))
    kv4_join_kernel<T, kDim, true><<<dim3(num_cus * 4), block, 0, stream>>>(args, split, rows, partial);
  else
    kv4_join_kernel<T, kDim, false><<<dim3(split.workers, y), block, 0, stream>>>(args, split, rows, partial);
  return hipGetLastError();
}

template <Kv4Type T, int kDim, int kCols>
hipError_t launch_attend(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args, const Split& split,
                         float* partial, hipStream_t stream) {
  const dim3 grid(split.workers + loose_groups(batch));
  auto run = [&](auto more, auto waves) {
    constexpr int kWaves = decltype(waves)::value;
    kv4_attend_kernel<T, kDim, kCols, decltype(more)::value, kWaves>
        <<<grid, dim3(kWaves * kWave), 0, stream>>>(pool, batch, args, split, partial);
  };
  typedef std::integral_constant<int, kFewWaves> Few;
  if (split.whole_cu)
    run(std::true_type{}, std::integral_constant<int, 4 * waves_per_simd(T, kDim, kCols)>{});
  else if (args.sinks > 0 || args.parents != nullptr)
    run(std::true_type{}, Few{});
  else
    run(std::false_type{}, Few{});
  return hipGetLastError();
}

template <Kv4Type T, int kDim>
hipError_t launch_dim(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args, const Split& split,
                      float* partial, int num_cus, hipStream_t stream) {
  hipError_t e = hipErrorInvalidValue;
  if (split.prompt)
    e = launch_kv4_prompt(pool, batch, args, T, split, partial, stream);
  else if (kDim > 128 || split.tile_shift == 4)
    e = launch_attend<T, kDim, 1>(pool, batch, args, split, partial, stream);
  else if constexpr (kDim <= 128)
    e = launch_attend<T, kDim, 2>(pool, batch, args, split, partial, stream);
  if (e != hipSuccess || split.one_launch) return e;
  return launch_join<T, kDim>(pool, batch, args, split, partial, num_cus, stream);
}

template <Kv4Type T>
hipError_t launch_type(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args, const Split& split,
                       float* partial, int num_cus, hipStream_t stream) {
  switch (pool.dim) {
    case 64: return launch_dim<T, 64>(pool, batch, args, split, partial, num_cus, stream);
    case 96: return launch_dim<T, 96>(pool, batch, args, split, partial, num_cus, stream);
    case 128: return launch_dim<T, 128>(pool, batch, args, split, partial, num_cus, stream);
    case 192: return launch_dim<T, 192>(pool, batch, args, split, partial, num_cus, stream);
    case 256: return launch_dim<T, 256>(pool, batch, args, split, partial, num_cus, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

size_t kv4_attend_workspace(const Kv4Pool& pool, const Kv4Batch& batch, int heads, bool parents, int num_cus) {
  size_t bytes = 0;
  for (Kv4Type type : {kKv4F32, kKv4BF16}) {  // f16 splits as bfloat16
    Split s = split_for(pool, batch, heads, type, parents, nullptr, num_cus);
    bytes = std::max(bytes, split_bytes(s, pool.dim));
    if (s.tile_shift != 5) continue;  // else a call may take tiles of 16 rows
    s.tile_shift = 4;
    s.workers = workers_for(type, pool.dim, 1, num_cus);
    bytes = std::max(bytes, split_bytes(s, pool.dim));
  }
  return bytes;
}

hipError_t launch_kv4_attend(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args, Kv4Type type,
                             void* workspace, size_t workspace_bytes, int num_cus, hipStream_t stream) {
  if (batch.rows <= 0) return hipSuccess;
  Split split = split_for(pool, batch, args.heads, type, args.parents != nullptr, &args, num_cus);
  // Trees in tiles of 256 rows may leave larger partial results than other calls of their sizes,
  // whose workspace suffices: with that alone their tiles are smaller.
  if (split_bytes(split, pool.dim) > workspace_bytes)
    split = split_for(pool, batch, args.heads, type, args.parents != nullptr, &args, num_cus, false);
  float* partial = static_cast<float*>(workspace);
  switch (type) {
    case kKv4F32: return launch_type<kKv4F32>(pool, batch, args, split, partial, num_cus, stream);
    case kKv4F16: return launch_type<kKv4F16>(pool, batch, args, split, partial, num_cus, stream);
    case kKv4BF16: return launch_type<kKv4BF16>(pool, batch, args, split, partial, num_cus, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace msim
