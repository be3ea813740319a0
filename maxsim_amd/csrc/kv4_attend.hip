// kv4_attend.hip -- attention of new tokens over the 4-bit key/value cache.
//
//   o = sum_j softmax_j(scale q . k_j) v_j over the keys j that the row sees,
//   k_j = c_j s_j and v_j = d_j t_j with int4 codes c, d and row scales s, t
//
// The query rows of one sequence and key/value head (its new tokens times the
// query heads that share it) are taken 16 to 64 at a time against tiles of 32
// keys.  A tile's scores are S^T = C Q^T and its part of the output is
// O^T = D^T P^T, both on v_mfma_f32_16x16x32_f16, so that a lane keeps one query
// row throughout (column lane % 16) and the probabilities leave the first
// product in the registers in which the second one takes them:
//   * a lane's keys of the two 16-key halves, 4 g .. 4 g + 3 and 16 + the same
//     (g = lane / 16), are its eight contraction slots of the second product;
//   * a lane reads a quarter of one key's codes (its dims g dim / 4 ...) and an
//     eighth or a sixteenth of eight value rows; the words of two value rows
//     are merged by halves, so that the pairs a decoded register holds are two
//     keys of one dim.
// Codes become f16 by one bitwise operation per pair (0x6400 | code ^ 8 is
// 1032 + code, exactly) and one packed subtraction.  The key scale multiplies
// the score, the value scale the probability; nothing else is dequantised.
//
// Queries are scaled to f16 by a power of two per row, largest entry in
// [2^14, 2^15): bfloat16 entries keep all their bits down to 2^-28 of the
// largest, f16 ones too.  Single precision queries are a sum of two f16 (22
// bits).  A probability times its value scale is taken relative to the row's
// largest such product, at 2^13 to 2^15, and rounded to f16: 11 bits down to
// 2^-27 of the largest, fewer below.  Single precision calls take it exactly, as
// three bfloat16 parts.  Scores, maxima, sums and outputs are single precision.
//
// Bytes bound it: dim + 8 per key and head against 4 dim operations per query
// row.  The keys of a sequence are split among workgroups when there are few
// query rows; each leaves its unnormalised sum and a second launch joins them.
#include <cfloat>

#include "codes4.hpp"
#include "kv4.hpp"

namespace msim {

namespace {

constexpr int kTileKeys = 32;
constexpr int kWaves = 4;
constexpr int kMinChunk = 256;  // keys of a split, at least
constexpr float kUnset = -FLT_MAX;
// A row's reference moves when a product passes 2^15 or a probability 2^100, to
// where the largest are 2^13 and 2^90.
constexpr float kProductLimit = 15.0f, kProductGoal = 13.0f, kProbLimit = 100.0f, kProbGoal = 90.0f;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// --------------------------------------------------------------- the split
//
// A unit of work is (sequence, tile of query rows, chunk of keys, head).  The
// chunk length follows from the work there is: all (row tile, key) pairs,
// shared evenly among `target` units.
struct Split {
  int chunk;  // keys
  int seq, first_row, rows, length, low;
  int tile, part, parts;
  int slot;  // of the unit's partial result, if parts > 1
};

struct SplitShape {
  int share;   // query heads per key/value head
  int tile_rows;
  int target;  // units, about
  int slots;
};

struct SeqWork {
  int first, rows, length, low, tiles;
};

__device__ __forceinline__ SeqWork seq_work(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args,
                                            const SplitShape& shape, int b) {
  SeqWork w;
  w.first = kv4_first_row(batch, b);
  w.rows = max(0, kv4_first_row(batch, b + 1) - w.first);
  w.length = kv4_length(pool, batch, b);
  const int64_t low = (int64_t)w.length - w.rows - args.window + 1;  // of the first row
  w.low = low > 0 ? (int)min(low, (int64_t)w.length) / kTileKeys * kTileKeys : 0;
  w.tiles = (int)(((int64_t)w.rows * shape.share + shape.tile_rows - 1) / shape.tile_rows);
  return w;
}

__device__ __forceinline__ int parts_of(const SeqWork& w, int chunk) {
  return max(1, (int)(((int64_t)w.length - w.low + chunk - 1) / chunk));
}

template <typename T>
__device__ __forceinline__ T block_sum(T v, T* lds) {
#pragma unroll
  for (int i = 1; i < kWave; i *= 2) v += __shfl_xor(v, i);
  if (lane_id() == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  T sum = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) sum += lds[i];
  __syncthreads();
  return sum;
}

// The workgroup's unit: the one numbered `unit`, or (unit < 0) sequence `seq`
// with the slot of its first partial result.  False past the last unit.
__device__ __forceinline__ bool find_split(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args,
                                           const SplitShape& shape, int64_t unit, int seq, Split& out) {
  __shared__ int64_t s_sum[kWaves];
  __shared__ int64_t s_scan[kWaves][2];
  __shared__ int s_found[2];
  int64_t pairs = 0;
  for (int b = threadIdx.x; b < batch.batch; b += blockDim.x) {
    const SeqWork w = seq_work(pool, batch, args, shape, b);
    pairs += (int64_t)w.tiles * (w.length - w.low);
  }
  pairs = block_sum(pairs, s_sum);
  const int64_t even = (pairs * pool.kv_heads + shape.target - 1) / shape.target;
  out.chunk = (int)min((int64_t)1 << 30, (max((int64_t)kMinChunk, even) + 127) / 128 * 128);
  if (threadIdx.x == 0) s_found[0] = -1;
  int64_t units = 0, slots = 0;  // before this pass's sequences
  __syncthreads();
  int64_t at = -1, slot_at = 0;
  for (int b0 = 0; b0 < batch.batch; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    int64_t mine = 0, mine_slots = 0;
    if (b < batch.batch) {
      const SeqWork w = seq_work(pool, batch, args, shape, b);
      const int parts = parts_of(w, out.chunk);
      mine = (int64_t)w.tiles * parts;
      mine_slots = parts > 1 ? mine : 0;
    }
    int64_t sum = mine, sum_slots = mine_slots;
#pragma unroll
    for (int i = 1; i < kWave; i *= 2) {
      const int64_t u = __shfl_up(sum, i), s = __shfl_up(sum_slots, i);
      if (lane_id() >= i) sum += u, sum_slots += s;
    }
    if (lane_id() == kWave - 1) s_scan[threadIdx.x / kWave][0] = sum, s_scan[threadIdx.x / kWave][1] = sum_slots;
    __syncthreads();
    int64_t before = units, before_slots = slots;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const int64_t u = s_scan[i][0], s = s_scan[i][1];
      if (i < (int)threadIdx.x / kWave) before += u, before_slots += s;
      units += u, slots += s;
    }
    const int64_t first = before + sum - mine;
    const bool here = b < batch.batch && (unit >= 0 ? first <= unit && unit < first + mine : b == seq);
    if (here) {
      s_found[0] = b;
      s_sum[0] = unit >= 0 ? unit - first : 0;
      s_sum[1] = before_slots + sum_slots - mine_slots;
    }
    __syncthreads();
    if (s_found[0] >= 0) {
      at = s_sum[0], slot_at = s_sum[1];
      break;
    }
  }
  const int b = wave_uniform(s_found[0]);
  if (b < 0) return false;
  const SeqWork w = seq_work(pool, batch, args, shape, b);
  out.seq = b;
  out.first_row = wave_uniform(w.first);
  out.rows = wave_uniform(w.rows);
  out.length = wave_uniform(w.length);
  out.low = wave_uniform(w.low);
  out.parts = wave_uniform(parts_of(w, out.chunk));
  const int local = wave_uniform((int)at);
  out.tile = local / out.parts;
  out.part = local % out.parts;
  out.slot = wave_uniform((int)slot_at) + local;
  return true;
}

// ------------------------------------------------------------ the main kernel

template <int kDim>
struct Shape {
  static constexpr int kKeyWords = kDim / 32;               // a lane's words of a key: dim / 4 codes
  static constexpr int kValueDims = kDim <= 64 ? 4 : (kDim <= 128 ? 8 : 16);  // a lane's dims of a value row
  static constexpr int kValueLanes = kDim / kValueDims;     // 16, or 12
  static constexpr int kTiles = kValueDims;                 // 16-dim tiles of the output
};

template <int kDim>
struct Tile {
  uint32_t key[2][kDim / 32];                                  // [half][word]
  uint32_t value[2][4][Shape<kDim>::kValueDims > 8 ? 2 : 1];   // [half][key][word]
  v4f key_scale[2], value_scale[2];
  bool hole[2];
};

// Eight codes of a word as bfloat16, in the order of decode_word.
__device__ __forceinline__ v8b decode_word_bf16(uint32_t w) {
  return __builtin_bit_cast(v8b, (v4u){pair_bf16(w << 3), pair_bf16(w >> 1), pair_bf16(w >> 5), pair_bf16(w >> 9)});
}

// Eight codes of a word as f16: pairs (code i, code i + 4).
__device__ __forceinline__ v8h decode_word(uint32_t w) {
  const v2h base = {(_Float16)1032.0f, (_Float16)1032.0f};
  const v2h high = {(_Float16)72.0f, (_Float16)72.0f}, sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
  const uint32_t w8 = w >> 8;
  const v2h a = __builtin_bit_cast(v2h, (w & 0x000F000Fu) ^ 0x64086408u) - base;
  const v2h b = __builtin_elementwise_fma(__builtin_bit_cast(v2h, (w & 0x00F000F0u) ^ 0x64806480u), sixteenth, -high);
  const v2h c = __builtin_bit_cast(v2h, (w8 & 0x000F000Fu) ^ 0x64086408u) - base;
  const v2h d = __builtin_elementwise_fma(__builtin_bit_cast(v2h, (w8 & 0x00F000F0u) ^ 0x64806480u), sixteenth, -high);
  return (v8h){a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The order of a word's codes in decode_word's result.
__device__ __forceinline__ constexpr int word_order(int i) { return (i & 1) * 4 + i / 2; }

template <Kv4Type T>
__device__ __forceinline__ float load_query(const void* q, int64_t i) {
  if constexpr (T == kKv4F32) return static_cast<const float*>(q)[i];
  if constexpr (T == kKv4F16) return (float)static_cast<const _Float16*>(q)[i];
  return __uint_as_float((uint32_t) static_cast<const uint16_t*>(q)[i] << 16);
}

template <Kv4Type T>
__device__ __forceinline__ void store_out(void* out, int64_t i, float x) {
  if constexpr (T == kKv4F32) static_cast<float*>(out)[i] = x;
  if constexpr (T == kKv4F16) static_cast<_Float16*>(out)[i] = (_Float16)x;
  if constexpr (T == kKv4BF16) static_cast<__bf16*>(out)[i] = (__bf16)x;
}

template <int kDim>
__device__ __forceinline__ void load_tile(const Kv4Pool& pool, const Kv4Batch& batch, int seq, int length, int head,
                                          int key0, Tile<kDim>& t) {
  typedef Shape<kDim> S;
  const int lane = lane_id(), col = lane % 16, g = lane / 16;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    // Pages hold 16 rows or a multiple, so a half lies in one page.
    const int key = key0 + 16 * h;
    int page = key < length ? as_constant(batch.table)[(int64_t)seq * batch.max_pages + (key >> pool.page_shift)] : -1;
    t.hole[h] = (uint32_t)page >= (uint32_t)pool.num_pages;
    if (t.hole[h]) page = 0;
    const int64_t at = kv4_pool_row(pool, page, head, key & ((1 << pool.page_shift) - 1));
    const uint8_t* keys = pool.codes[0] + at * (kDim / 2);
    const uint8_t* values = pool.codes[1] + at * (kDim / 2);
    const uint32_t* kw = reinterpret_cast<const uint32_t*>(keys + col * (kDim / 2) + g * (kDim / 8));
#pragma unroll
    for (int i = 0; i < S::kKeyWords; ++i) t.key[h][i] = kw[i];
    const int vl = S::kValueLanes == 16 ? col : min(col, S::kValueLanes - 1);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint8_t* row = values + (4 * g + r) * (kDim / 2) + vl * (S::kValueDims / 2);
      if constexpr (S::kValueDims == 4) {
        t.value[h][r][0] = *reinterpret_cast<const uint16_t*>(row);
      } else {
#pragma unroll
        for (int i = 0; i < S::kValueDims / 8; ++i) t.value[h][r][i] = reinterpret_cast<const uint32_t*>(row)[i];
      }
    }
    t.key_scale[h] = *reinterpret_cast<const v4f*>(pool.scales[0] + at + 4 * g);
    t.value_scale[h] = *reinterpret_cast<const v4f*>(pool.scales[1] + at + 4 * g);
  }
}

__device__ __forceinline__ float across_groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float across_groups_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// kCols 16-row column tiles of queries per workgroup; its waves take the key
// tiles in turn.
template <Kv4Type T, int kDim, int kCols>
__global__ __launch_bounds__(kWaves* kWave) void kv4_attend_kernel(Kv4Pool pool, Kv4Batch batch, Kv4AttendArgs args,
                                                                   SplitShape shape, float* __restrict__ partial) {
  typedef Shape<kDim> S;
  constexpr int kParts = T == kKv4F32 ? 2 : 1;      // of a query
  constexpr int kProbParts = T == kKv4F32 ? 3 : 1;  // of a probability
  typedef typename std::conditional<T == kKv4F32, v8b, v8h>::type Prob;
  constexpr int kRows = 16 * kCols;
  extern __shared__ char s_raw[];
  const int lane = lane_id(), col = lane % 16, g = lane / 16, wave = wave_uniform(threadIdx.x / kWave);
  const int head = blockIdx.x % pool.kv_heads;
  Split u;
  if (!find_split(pool, batch, args, shape, blockIdx.x / pool.kv_heads, 0, u)) {
    // Past the last unit, as the last workgroup always is: rows of no sequence
    // come out as rows that see nothing.
    if (blockIdx.x == gridDim.x - 1 && batch.offsets != nullptr) {
      const int first = kv4_first_row(batch, 0), last = kv4_first_row(batch, batch.batch);
      for (int row = 0; row < batch.rows; ++row) {
        if (row >= first && row < last) row = last;
        if (row >= batch.rows) break;
        for (int i = threadIdx.x; i < args.heads * kDim; i += blockDim.x)
          store_out<T>(args.out, row * args.out_row_stride + i / kDim * args.out_head_stride + i % kDim, 0.0f);
        for (int h = threadIdx.x; h < args.heads && args.lse != nullptr; h += blockDim.x)
          args.lse[(int64_t)row * args.heads + h] = kNegInf;
      }
    }
    return;
  }

  // Query rows of this tile: row r is new token r / share, head r % share.
  v8h q[kCols][kParts][S::kKeyWords];
  float factor[kCols];       // of a product with the codes, towards log2 scores
  int see_low[kCols], see_high[kCols];
  const uint8_t* mask[kCols];
  int all_low = 0, all_high = INT_MAX, any_low = INT_MAX, any_high = 0;
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    const int64_t r = (int64_t)u.tile * kRows + 16 * c + col;
    const int token = (int)(r / shape.share), sub = (int)(r % shape.share);
    const bool have = token < u.rows;
    const int64_t base = have ? (int64_t)(u.first_row + token) * args.q_row_stride +
                                    (int64_t)(head * shape.share + sub) * args.q_head_stride
                              : 0;
    float x[S::kKeyWords][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < S::kKeyWords; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[i][j] = have ? load_query<T>(args.q, base + g * (kDim / 4) + i * 8 + word_order(j)) : 0.0f;
        top = max(top, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
      }
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    const int shift = 141 - (int)(top >> 23);  // the largest to [2^14, 2^15)
#pragma unroll
    for (int i = 0; i < S::kKeyWords; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = ldexpf(x[i][j], shift);
        const _Float16 hi = (_Float16)y;
        q[c][0][i][j] = hi;
        if constexpr (kParts == 2) q[c][1][i][j] = (_Float16)(y - (float)hi);
      }
    factor[c] = ldexpf(args.scale_log2, -shift);
    const int pos = u.length - u.rows + token;
    const int64_t low = (int64_t)pos - args.window + 1;
    see_low[c] = low > 0 ? (int)low : 0;
    see_high[c] = args.causal ? max(0, min(u.length, pos + 1)) : u.length;
    mask[c] = nullptr;
    if (args.mask != nullptr) {
      see_high[c] = (int)min((int64_t)see_high[c], args.mask_width);
      mask[c] = args.mask + (have ? (int64_t)(u.first_row + token) * args.mask_row_stride : 0);
    }
    if (!have) {  // a row of padding: nothing depends on what it sees
      see_low[c] = 0;
      see_high[c] = args.mask != nullptr ? 0 : INT_MAX;
    } else if (see_high[c] > see_low[c]) {
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
  // Keys of this unit: its chunk, cut to what some row sees.
  const int64_t chunk_low = u.low + (int64_t)u.part * u.chunk;
  int begin = (int)max(chunk_low, (int64_t)min(any_low, u.length) / kTileKeys * kTileKeys);
  const int end = (int)min(chunk_low + u.chunk, (int64_t)any_high);

  float ref[kCols], sum[kCols];
  v4f o[kCols][S::kTiles];
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    ref[c] = kUnset;
    sum[c] = 0.0f;
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t) o[c][t] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
  }

  int key0 = begin + wave * kTileKeys;
  Tile<kDim> tile;
  if (key0 < end) load_tile<kDim>(pool, batch, u.seq, u.length, head, key0, tile);
  for (; key0 < end; key0 += kWaves * kTileKeys) {
    Tile<kDim> next;
    if (key0 + kWaves * kTileKeys < end)
      load_tile<kDim>(pool, batch, u.seq, u.length, head, key0 + kWaves * kTileKeys, next);

    // Scores of the tile.
    v4f s[kCols][2];
#pragma unroll
    for (int c = 0; c < kCols; ++c) s[c][0] = s[c][1] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < S::kKeyWords; ++i) {
        const v8h a = decode_word(tile.key[h][i]);
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int p = 0; p < kParts; ++p)
            s[c][h] = mfma(a, q[c][p][i], s[c][h]);
      }
    mfma_results_fence();

    const bool whole = key0 >= all_low && key0 + kTileKeys <= all_high && args.mask == nullptr && !tile.hole[0] &&
                       !tile.hole[1];
    Prob probs[kCols][kProbParts];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      float x[8], vs[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = s[c][i / 4][i % 4] * (tile.key_scale[i / 4][i % 4] * factor[c]);
        vs[i] = tile.value_scale[i / 4][i % 4];
      }
      if (!whole) {
        // A hidden key takes no part in the maxima, and its probability and
        // value scale are zeros whatever the cache holds there.
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = key0 + 16 * (i / 4) + 4 * g + i % 4;
          bool see = key >= see_low[c] && key < see_high[c] && !tile.hole[i / 4];
          if (args.mask != nullptr && see) see = mask[c][key] != 0;
          x[i] = see ? x[i] : kNegInf;
          vs[i] = see ? vs[i] : 0.0f;
        }
      }
      float top = kNegInf, most = kNegInf;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        top = fmaxf(top, x[i]);
        most = fmaxf(most, x[i] + __builtin_amdgcn_logf(vs[i]));
      }
      if (__ballot(most > ref[c] + kProductLimit || top > ref[c] + kProbLimit) != 0) {
        const float now = fmaxf(ref[c], fmaxf(across_groups_max(most) - kProductGoal, across_groups_max(top) - kProbGoal));
        const float alpha = exp2_hw(ref[c] - now);
        ref[c] = now;
        sum[c] *= alpha;
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) o[c][t] *= alpha;
      }
      uint32_t product[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = exp2_hw(x[i] - ref[c]);
        sum[c] += p;
        if constexpr (T == kKv4F32)
          product[i] = __float_as_uint(p * vs[i]);
        else
          probs[c][0][i] = (_Float16)(p * vs[i]);
      }
      if constexpr (T == kKv4F32) split3(product, probs[c]);
    }

    // The tile's part of the output: the codes of two keys side by side.
#pragma unroll
    for (int k = 0; k < (S::kValueDims + 7) / 8; ++k) {
      uint32_t low[4], high[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint32_t a = tile.value[p / 2][2 * (p % 2)][k], b = tile.value[p / 2][2 * (p % 2) + 1][k];
        low[p] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        high[p] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      }
#pragma unroll
      for (int half = 0; half < (S::kValueDims >= 8 ? 2 : 1); ++half) {
        Prob pair[4];  // [pair of keys]: four dims of both
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          if constexpr (T == kKv4F32)
            pair[p] = decode_word_bf16(half ? high[p] : low[p]);
          else
            pair[p] = decode_word(half ? high[p] : low[p]);
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          Prob a;
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
    tile = next;
  }
  mfma_results_fence();

  // The waves' results joined in a fixed order: the upper half hands over to
  // the lower one until wave 0 holds the sum.
  float* s_ref = reinterpret_cast<float*>(s_raw);           // [waves][cols][16]
  float* s_sum = s_ref + kWaves * kRows;                    // [waves][cols][16]
  v4f* s_o = reinterpret_cast<v4f*>(s_sum + kWaves * kRows);  // [waves / 2][cols][tiles][64]
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    sum[c] = across_groups_sum(sum[c]);
    if (g == 0) s_ref[wave * kRows + 16 * c + col] = ref[c];
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    float all = s_ref[16 * c + col];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) all = fmaxf(all, s_ref[w * kRows + 16 * c + col]);
    const float alpha = exp2_hw(ref[c] - all);
    ref[c] = all;
    sum[c] *= alpha;
    if (g == 0) s_sum[wave * kRows + 16 * c + col] = sum[c];
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t) o[c][t] *= alpha;
  }
#pragma unroll
  for (int n = kWaves / 2; n >= 1; n /= 2) {
    if (wave >= n && wave < 2 * n) {
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) s_o[(((wave - n) * kCols + c) * S::kTiles + t) * kWave + lane] = o[c][t];
    }
    __syncthreads();
    if (wave < n) {
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) o[c][t] += s_o[((wave * kCols + c) * S::kTiles + t) * kWave + lane];
    }
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    const int64_t r = (int64_t)u.tile * kRows + 16 * c + col;
    const int token = (int)(r / shape.share), sub = (int)(r % shape.share);
    float total = s_sum[16 * c + col];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) total += s_sum[w * kRows + 16 * c + col];
    if (u.parts > 1) {
      const int64_t slot = ((int64_t)u.slot * pool.kv_heads + head);
      if (slot >= shape.slots) continue;
      float* dst = partial + slot * kRows * (kDim + 2) + (16 * c + col) * (kDim + 2);
      if (g == 0) {
        dst[kDim] = ref[c];
        dst[kDim + 1] = total;
      }
#pragma unroll
      for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * g + i < S::kValueLanes) dst[(4 * g + i) * S::kValueDims + t] = o[c][t][i];
      continue;
    }
    if (token >= u.rows) continue;
    const int qh = head * shape.share + sub;
    const int64_t row = u.first_row + token;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if (args.lse != nullptr && g == 0)
      args.lse[row * args.heads + qh] = total == 0.0f ? kNegInf : (ref[c] + __log2f(total)) * 0.69314718055994531f;
    const int64_t base = row * args.out_row_stride + (int64_t)qh * args.out_head_stride;
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * g + i < S::kValueLanes)
          store_out<T>(args.out, base + (4 * g + i) * S::kValueDims + t, o[c][t][i] * inv);
  }
}

// One workgroup per (row of the call, head): joins the parts of a split row.
template <Kv4Type T, int kDim>
__global__ __launch_bounds__(kWaves* kWave) void kv4_join_kernel(Kv4Pool pool, Kv4Batch batch, Kv4AttendArgs args,
                                                                 SplitShape shape, const float* __restrict__ partial) {
  const int row = blockIdx.x;
  const int seq = kv4_find_sequence(batch, row);
  Split u;
  if (seq < 0 || !find_split(pool, batch, args, shape, -1, seq, u)) return;
  if (u.parts <= 1) return;
  const int token = row - u.first_row;
  for (int qh = blockIdx.y * kWaves + threadIdx.x / kWave; qh < args.heads; qh += gridDim.y * kWaves) {
    const int head = qh / shape.share;
    const int64_t r = (int64_t)token * shape.share + qh % shape.share;
    const int64_t slot0 = u.slot + r / shape.tile_rows * u.parts;
    const float* src = partial + r % shape.tile_rows * (kDim + 2);
    const int64_t stride = (int64_t)shape.tile_rows * (kDim + 2);
    float all = kUnset;
    for (int p = lane_id(); p < u.parts; p += kWave) {
      const int64_t slot = (slot0 + p) * pool.kv_heads + head;
      if (slot < shape.slots) all = fmaxf(all, src[slot * stride + kDim]);
    }
    all = wave_reduce(all, [](float a, float b) { return fmaxf(a, b); });
    float total = 0.0f, o[(kDim + 63) / 64] = {};
    for (int p = 0; p < u.parts; ++p) {
      const int64_t slot = (slot0 + p) * pool.kv_heads + head;
      if (slot >= shape.slots) break;
      const float* part = src + slot * stride;
      const float alpha = exp2_hw(part[kDim] - all);
      total += part[kDim + 1] * alpha;
#pragma unroll
      for (int i = 0; i < (kDim + 63) / 64; ++i)
        if (i * 64 + lane_id() < kDim) o[i] += part[i * 64 + lane_id()] * alpha;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if (args.lse != nullptr && lane_id() == 0)
      args.lse[(int64_t)row * args.heads + qh] =
          total == 0.0f ? kNegInf : (all + __log2f(total)) * 0.69314718055994531f;
    const int64_t base = row * args.out_row_stride + (int64_t)qh * args.out_head_stride;
#pragma unroll
    for (int i = 0; i < (kDim + 63) / 64; ++i)
      if (i * 64 + lane_id() < kDim) store_out<T>(args.out, base + i * 64 + lane_id(), o[i] * inv);
  }
}

// Column tiles per workgroup: as many as a sequence's rows fill on average (one
// for wide heads, whose outputs take the registers).
int columns_for(const Kv4Pool& pool, const Kv4Batch& batch, int heads) {
  const int64_t rows = (int64_t)batch.rows * (heads / pool.kv_heads) / std::max(1, batch.batch);
  return rows <= 16 || pool.dim > 128 ? 1 : 2;
}

SplitShape split_shape(const Kv4Pool& pool, const Kv4Batch& batch, int heads, int num_cus) {
  SplitShape s;
  s.share = heads / pool.kv_heads;
  s.tile_rows = 16 * columns_for(pool, batch, heads);
  s.target = 4 * num_cus;
  // A split sequence has more than one chunk, so its last one is less than
  // half of what it adds: units of split sequences number less than twice the
  // target.
  s.slots = 2 * s.target + pool.kv_heads;
  return s;
}

template <Kv4Type T, int kDim, int kCols>
hipError_t launch_attend(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args,
                         const SplitShape& shape, float* partial, hipStream_t stream) {
  const int64_t tiles = ((int64_t)batch.rows * shape.share) / shape.tile_rows + batch.batch;
  const int64_t grid = tiles * pool.kv_heads + shape.target + pool.kv_heads;
  if (grid > (1 << 24)) return hipErrorInvalidValue;
  constexpr int kRows = 16 * kCols;
  const size_t lds = sizeof(float) * (2 * kWaves * kRows + (kWaves / 2) * kRows * 16 * Shape<kDim>::kTiles);
  kv4_attend_kernel<T, kDim, kCols><<<dim3((unsigned)grid), dim3(kWaves * kWave), lds, stream>>>(pool, batch, args,
                                                                                               shape, partial);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  // No sequence is split if none can be longer than the least chunk.
  if (((int64_t)batch.max_pages << pool.page_shift) > kMinChunk) {
    const int by = std::min(8, (args.heads + kWaves - 1) / kWaves);
    kv4_join_kernel<T, kDim><<<dim3((unsigned)batch.rows, (unsigned)by), dim3(kWaves * kWave), 0, stream>>>(
        pool, batch, args, shape, partial);
  }
  return hipGetLastError();
}

template <Kv4Type T, int kDim>
hipError_t launch_dim(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args, const SplitShape& shape,
                      float* partial, hipStream_t stream) {
  if constexpr (kDim <= 128)
    if (shape.tile_rows == 32) return launch_attend<T, kDim, 2>(pool, batch, args, shape, partial, stream);
  return launch_attend<T, kDim, 1>(pool, batch, args, shape, partial, stream);
}

template <Kv4Type T>
hipError_t launch_type(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args, const SplitShape& shape,
                       float* partial, hipStream_t stream) {
  switch (pool.dim) {
    case 64: return launch_dim<T, 64>(pool, batch, args, shape, partial, stream);
    case 96: return launch_dim<T, 96>(pool, batch, args, shape, partial, stream);
    case 128: return launch_dim<T, 128>(pool, batch, args, shape, partial, stream);
    case 192: return launch_dim<T, 192>(pool, batch, args, shape, partial, stream);
    case 256: return launch_dim<T, 256>(pool, batch, args, shape, partial, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

size_t kv4_attend_workspace(const Kv4Pool& pool, const Kv4Batch& batch, int heads, int num_cus) {
  const SplitShape s = split_shape(pool, batch, heads, num_cus);
  return (size_t)s.slots * s.tile_rows * (pool.dim + 2) * sizeof(float);
}

hipError_t launch_kv4_attend(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args, Kv4Type type,
                             void* workspace, int num_cus, hipStream_t stream) {
  if (batch.rows <= 0) return hipSuccess;
  const SplitShape shape = split_shape(pool, batch, args.heads, num_cus);
  float* partial = static_cast<float*>(workspace);
  switch (type) {
    case kKv4F32: return launch_type<kKv4F32>(pool, batch, args, shape, partial, stream);
    case kKv4F16: return launch_type<kKv4F16>(pool, batch, args, shape, partial, stream);
    case kKv4BF16: return launch_type<kKv4BF16>(pool, batch, args, shape, partial, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace msim
