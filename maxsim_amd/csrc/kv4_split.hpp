// kv4_split.hpp -- what the kernels of attention over the 4-bit cache share: how
// work is dealt out, queries read and outputs written.
#pragma once

#include <algorithm>
#include <cfloat>

#include "codes4.hpp"
#include "kv4.hpp"

namespace msim {

constexpr float kUnset = -FLT_MAX;
// A row's reference moves, to its largest score, when a probability passes 2^6 (limits
// up to 2^40 took the same time; 2^2 took 1.5 % more at prompts).
constexpr float kTopLimit = 6.0f;
// Value scales are taken over 2^20 and codes over kCodeUnit, so that the sums of
// probabilities times values stay numbers before they are divided, for 2^18 keys and
// values of any size.  The other end: the 16 bits of a product hold from values of
// 2^-94 up.
constexpr float kValueUnit = 0x1p20f;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// --------------------------------------------------------------- the split
//
// An item is (sequence, tile of query rows, key/value head), a granule 128 of
// the keys that the tile sees.  All granules, in the order of items, are dealt
// out evenly: each worker has a run of them, whatever items they belong to.  An
// item that lies within one worker is finished there; of the others each worker
// leaves a partial result, in its slot 1 if the item begins there, in slot 0 if
// it came in from the worker before (it has at most one of each).
//
// Where the page table has no room for sequences longer than kShort keys a granule is
// kShort: no item is split, and the call is one launch. Another 128 keys cost a workgroup
// about 1 us, the second launch 3 to 4 (one token behind 120 keys 7.3 us against 9.8
// split, behind 391 and 500 the same 10.4; 64 tokens behind 500 17.3 against 22.7).
constexpr int kKeyAlign = 32;  // a tile's first key
constexpr int kGranule = 128;
constexpr int kShort = 4 * kGranule;

// Granules, items and rows are counted in 32 bits: the host refuses calls of 2^30
// rows times heads and doubles the granule where their number could pass 2^31.
struct Split {
  uint32_t share;       // query heads per key/value head
  uint32_t tile_shift;  // log2(query rows of a tile)
  uint32_t workers;     // at most
  uint32_t granule_shift;
  uint32_t few;         // workers may have a single granule while there are no more of them
  uint32_t one_launch;  // no item is split
  uint32_t whole_cu;    // a workgroup has as many waves as a CU holds
  uint32_t prompt;      // kv4_prompt.hip's kernel
  uint32_t lead;        // granules that an item is dealt out as, besides its own
};

constexpr uint32_t kMostWorkers = 1024;

struct SeqWork {
  int first, rows, length;
  uint32_t tiles;
};

__device__ __forceinline__ SeqWork seq_work(const Kv4Pool& pool, const Kv4Batch& batch, const Split& split, int b) {
  SeqWork w;
  w.first = kv4_first_row(batch, b);
  w.rows = max(0, kv4_first_row(batch, b + 1) - w.first);
  w.length = kv4_length(pool, batch, b);
  w.tiles = ((uint32_t)w.rows * split.share + (1u << split.tile_shift) - 1) >> split.tile_shift;
  return w;
}

// The keys that some row of a tile may see, by position alone: low .. high, and of calls
// with sinks `head` more from 0 on (a multiple of kKeyAlign, as low is).
struct TileRange {
  int low, high;
  uint32_t granules;
  int head;

  // The keys of such calls are numbered without the gap between the two.
  __device__ int key_of(int number) const { return number < head ? number : number - head + low; }
  __device__ int number_of(int key) const { return key <= head ? key : max(head, key - low + head); }
};

// kMore: calls with sinks or parents.
template <bool kMore>
__device__ __forceinline__ TileRange tile_range(const Kv4AttendArgs& args, const Split& split, const SeqWork& w,
                                                uint32_t tile) {
  TileRange r;
  r.low = 0;
  r.high = w.length;
  if (args.causal) {
    const uint32_t rows = min((tile + 1) << split.tile_shift, (uint32_t)w.rows * split.share);
    r.high = max(0, min(w.length, w.length - w.rows + (int)((rows - 1) / split.share) + 1));
  }
  // Positions of rows with parents begin anew at each that has none.
  const int row = kMore && args.parents != nullptr ? 0 : (int)((tile << split.tile_shift) / split.share);
  const int first = w.length - w.rows + row;
  if (first >= args.window) r.low = min(w.length, (first - args.window + 1)) / kKeyAlign * kKeyAlign;
  r.head = 0;
  if constexpr (kMore) r.head = min(r.low, (min(args.sinks, w.length) + kKeyAlign - 1) / kKeyAlign * kKeyAlign);
  r.granules =
      max(1u, ((uint32_t)(max(0, r.high - r.low) + r.head) + (1u << split.granule_shift) - 1) >> split.granule_shift);
  return r;
}

// Granules that an item is dealt out as, besides its own.
template <bool kMore>
__device__ __forceinline__ uint32_t lead_of(const Split& split) {
  return kMore ? split.lead : 0;
}

// What tile `tile` of a sequence is dealt out as, for all heads; 0 past the last.
template <bool kMore>
__device__ __forceinline__ uint32_t tile_share(const Kv4Pool& pool, const Kv4AttendArgs& args, const Split& split,
                                               const SeqWork& w, uint32_t tile) {
  if (tile >= w.tiles) return 0;
  return (tile_range<kMore>(args, split, w, tile).granules + lead_of<kMore>(split)) * pool.kv_heads;
}

// `total` granules among `workers`: the first `extra` have one more.
struct Deal {
  uint32_t total, workers, each, extra;
  __device__ uint32_t begin(uint32_t i) const { return i * each + min(i, extra); }
  __device__ uint32_t worker_of(uint32_t granule) const {
    const uint32_t longer = extra * (each + 1);
    return min(workers - 1, granule < longer ? granule / (each + 1) : extra + (granule - longer) / each);
  }
};

// Walks over the items of the call from a sequence's first one on.
template <bool kMore>
struct Cursor {
  int seq = 0;
  uint32_t before = 0;  // granules before the item group (sequence, tile)
  uint32_t tile = 0;
  SeqWork work = {};
  TileRange range = {};

  // The item at hand.
  int head = 0;
  uint32_t item_at = 0;  // where it begins

  // The work of sequence `seq` as lane `lane` has it.
  __device__ __forceinline__ void enter(const Kv4AttendArgs& args, const Split& split, const SeqWork& w, int lane) {
    work.first = __builtin_amdgcn_readlane(w.first, lane);
    work.rows = __builtin_amdgcn_readlane(w.rows, lane);
    work.length = __builtin_amdgcn_readlane(w.length, lane);
    work.tiles = __builtin_amdgcn_readlane(w.tiles, lane);
    tile = 0;
    range = tile_range<kMore>(args, split, work, 0);
  }
  // To the item that holds `granule`; false past the last (offsets out of order).  By a wave
  // together: of a sequence's tiles it looks through 64 at a time (2 x 40 tokens, 20 tiles of 16
  // rows: one after another they cost 1 us more).
  __device__ __forceinline__ bool seek(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args,
                                       const Split& split, uint32_t granule) {
    for (int hops = 0;; ++hops) {
      if (tile < work.tiles) {
        const uint32_t size = (range.granules + lead_of<kMore>(split)) * pool.kv_heads;
        if (granule - before < size) break;
        before += size;
        ++tile;
      }
      while (hops > 0 && tile < work.tiles) {
        const uint32_t mine = tile_share<kMore>(pool, args, split, work, tile + lane_id()), upto = wave_scan(mine);
        const uint64_t beyond = __ballot(granule - before < upto);
        if (beyond != 0) {
          const int at = __builtin_ctzll(beyond);
          before += __builtin_amdgcn_readlane(upto - mine, at);
          tile += at;
          break;
        }
        before += __builtin_amdgcn_readlane(upto, kWave - 1);
        tile = min(tile + kWave, work.tiles);
      }
      if (tile < work.tiles) {
        range = tile_range<kMore>(args, split, work, tile);
      } else {
        if (++seq >= batch.batch) return false;
        enter(args, split, seq_work(pool, batch, split, seq), 0);
      }
    }
    head = wave_uniform((granule - before) / (range.granules + lead_of<kMore>(split)));
    item_at = before + head * (range.granules + lead_of<kMore>(split));
    return true;
  }
  // Of what is dealt out from `from` to `upto` (counted from item_at) the item's own granules.
  __device__ __forceinline__ uint32_t own(const Split& split, uint32_t at) const {
    return min(range.granules, at - min(at, lead_of<kMore>(split)));
  }
};

// By a wave together: the deal, and the cursor on the sequence that holds the first
// granule of worker `worker`.  False if the worker has none.
template <bool kMore>
__device__ __forceinline__ bool find_work(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args,
                                          const Split& split, uint32_t worker, Cursor<kMore>& cursor, Deal& deal) {
  const int lane = lane_id();
  // Where there are few sequences, 2^shift lanes share the tiles of each (2 x 2,048 fp32 tokens,
  // window 1,024: 265 us for 382 with a lane each).
  const int shift = batch.batch <= 1 ? 6 : max(0, __builtin_clz(batch.batch - 1) - 26);
  const int each = kWave >> shift, stripes = 1 << shift, stripe = lane & (stripes - 1);
  auto work_of = [&](int b) -> SeqWork {
    return b < batch.batch ? seq_work(pool, batch, split, b) : SeqWork{0, 0, 0, 0};
  };
  auto granules = [&](const SeqWork& w) -> uint32_t {
    uint32_t sum = 0;
    for (uint32_t t = stripe; t < w.tiles; t += stripes) sum += tile_share<kMore>(pool, args, split, w, t);
    return sum;
  };
  const SeqWork head_work = work_of(lane >> shift);
  const uint32_t head = granules(head_work);
  uint32_t total = head;
  for (int b0 = each; b0 < batch.batch; b0 += each) total += granules(work_of(b0 + (lane >> shift)));
  const uint32_t head_scan = wave_scan(head);
  deal.total = batch.batch <= each ? __builtin_amdgcn_readlane(head_scan, kWave - 1)
                                   : __builtin_amdgcn_readlane(wave_scan(total), kWave - 1);
  deal.workers = min(split.workers, max(max(1u, min(deal.total, split.few)), deal.total / 2));
  deal.each = deal.total / deal.workers;
  deal.extra = deal.total - deal.each * deal.workers;
  if (deal.total == 0 || worker >= deal.workers) return false;
  const uint32_t target = deal.begin(worker);
  uint32_t done = 0;
  for (int b0 = 0; b0 < batch.batch; b0 += each) {
    const SeqWork work = b0 == 0 ? head_work : work_of(b0 + (lane >> shift));
    const uint32_t mine = b0 == 0 ? head : granules(work);
    const uint32_t upto = done + (b0 == 0 ? head_scan : wave_scan(mine));
    const uint64_t beyond = __ballot(target < upto);
    if (beyond != 0) {
      const int at = __builtin_ctzll(beyond) & -stripes;  // the sequence's first lane
      cursor.seq = wave_uniform(b0 + (at >> shift));
      cursor.before = __builtin_amdgcn_readlane(upto - mine, at);
      cursor.enter(args, split, work, at);
      return true;
    }
    done = __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return false;
}

// -------------------------------------------------------- queries and outputs

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

// Eight elements of a query from element i on (16-byte loads if `wide`).
template <Kv4Type T>
__device__ __forceinline__ void load8(const void* q, int64_t i, bool wide, float (&x)[8]) {
  if constexpr (T == kKv4F32) {
    const float* p = static_cast<const float*>(q) + i;
    if (wide) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const v4f v = reinterpret_cast<const v4f*>(p)[k];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * k + j] = v[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = p[j];
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(q) + i;
    uint16_t h[8];
    if (wide) {
      __builtin_memcpy(h, __builtin_assume_aligned(p, 16), 16);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = p[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x[j] = T == kKv4BF16 ? __uint_as_float((uint32_t)h[j] << 16) : (float)__builtin_bit_cast(_Float16, h[j]);
  }
}

template <Kv4Type T>
__device__ __forceinline__ void store_out(void* out, int64_t i, float x) {
  if constexpr (T == kKv4F32) static_cast<float*>(out)[i] = x;
  if constexpr (T == kKv4F16) static_cast<_Float16*>(out)[i] = (_Float16)x;
  if constexpr (T == kKv4BF16) static_cast<__bf16*>(out)[i] = (__bf16)x;
}

// Four elements of an output row (one store if `wide`).
template <Kv4Type T>
__device__ __forceinline__ void store4(void* out, int64_t i, bool wide, v4f x) {
  if (!wide) {
#pragma unroll
    for (int k = 0; k < 4; ++k) store_out<T>(out, i + k, x[k]);
  } else if constexpr (T == kKv4F32) {
    *reinterpret_cast<v4f*>(static_cast<float*>(out) + i) = x;
  } else {
    typedef typename std::conditional<T == kKv4F16, _Float16, __bf16>::type E;
    typedef E v4e __attribute__((ext_vector_type(4)));
    *reinterpret_cast<v4e*>(static_cast<E*>(out) + i) = (v4e){(E)x[0], (E)x[1], (E)x[2], (E)x[3]};
  }
}

// Multiplies a query row to f16's range: the exponent to add (its largest entry
// in [2^14, 2^15), below it from 2^-106 down) from the bits of that entry.
__device__ __forceinline__ int query_shift(uint32_t top) { return min(141 - (int)(top >> 23), 120); }
// What turns its products into log2 scores: above zero, so that a hidden score stays
// minus infinity, and else as small as it is (small queries may meet large keys).
// Scores over it are numbers for keys up to 2^102.
__device__ __forceinline__ float score_factor(float scale_log2, int shift) {
  return fmaxf(ldexpf(fabsf(scale_log2), -shift), 0x1p-149f);
}

// Four bytes of a mask row from key `key` on, none of them at `end` or past it
// (zeros there); the row's address and the key may be odd.
__device__ __forceinline__ uint32_t mask_bytes(const uint8_t* mask, int key, int end) {
  uint32_t m = 0;
  if (key + 4 <= end) {
    __builtin_memcpy(&m, mask + key, 4);
  } else {
    for (int i = 0; i < 4 && key + i < end; ++i) m |= (uint32_t)mask[key + i] << (8 * i);
  }
  return m;
}

// The maximum of 8 or 16 values, three operands at a time.
template <int N>
__device__ __forceinline__ float max_of(const float (&x)[N]) {
  float m = max3_op(x[0], x[1], x[2]);
#pragma unroll
  for (int i = 3; i + 4 <= N; i += 4) m = max5_op(m, x[i], x[i + 1], x[i + 2], x[i + 3]);
  return fmaxf(m, x[N - 1]);
}

// What an output row's sums are multiplied by, and its lse, by the last sums.
__device__ __forceinline__ float output_factor(float total) {
  return total == 0.0f ? 0.0f : kCodeUnit * kValueUnit / total;
}
__device__ __forceinline__ float log_sum(float ref, float total) {
  return total == 0.0f ? kNegInf : (ref + __log2f(total)) * 0.69314718055994531f;
}

// Rows of no sequence come out as rows that see nothing: a padded batch has many.  They
// belong to workgroups of their own behind the workers, one per 64 rows of the call, up
// to 256 (one that did them all held a call of 8 rows behind 3,000 keys and 4,088 loose
// ones, 32 heads of 128, for 4,500 us; these make it 69).
inline uint32_t loose_groups(const Kv4Batch& batch) {
  return batch.offsets == nullptr ? 0 : std::min(std::max(1, batch.rows / 64), 256);
}
template <Kv4Type T, int kDim>
__device__ __forceinline__ void loose_rows(const Kv4Batch& batch, const Kv4AttendArgs& args, const Split& split) {
  const int first = kv4_first_row(batch, 0), last = max(first, kv4_first_row(batch, batch.batch));
  const int step = (int)(gridDim.x - split.workers), count = first + batch.rows - last;
  for (int i = (int)(blockIdx.x - split.workers); i < count; i += step) {
    const int64_t row = i < first ? i : i - first + last;
    for (int j = threadIdx.x; j < args.heads * (kDim / 4); j += blockDim.x)
      store4<T>(args.out, row * args.out_row_stride + j / (kDim / 4) * args.out_head_stride + j % (kDim / 4) * 4,
                args.out_wide != 0, (v4f){0.0f, 0.0f, 0.0f, 0.0f});
    for (int h = threadIdx.x; h < args.heads && args.lse != nullptr; h += blockDim.x)
      args.lse[row * args.heads + h] = kNegInf;
  }
}

// The row that a row with parents comes right after; -1 where it is the context's last.
__device__ __forceinline__ int row_before(const int* parents, int row) {
  const int p = parents[row];
  return (uint32_t)p < (uint32_t)row ? p : -1;
}

// A worker's slot of partial results: [rows][dim], then [rows][reference, sum].
__device__ __forceinline__ float* partial_slot(float* partial, const Split& split, int dim, uint32_t worker, bool begins) {
  return partial + (((int64_t)worker * 2 + begins) << split.tile_shift) * (dim + 2);
}

// Behind the slots, for the join: of each worker the item that it begins and leaves to
// others, and behind those in how many parts the item is (0: no such item).
struct Unfinished {
  int first, rows;  // of its sequence
  uint32_t tile;
  int head;
};
__host__ __device__ inline int64_t partial_floats(const Split& split, int dim) {
  return ((int64_t)split.workers * 2 << split.tile_shift) * (dim + 2);
}
template <bool kMore>
__device__ __forceinline__ void note_unfinished(float* partial, const Split& split, int dim, const Cursor<kMore>& at,
                                                int parts) {
  if (threadIdx.x == 0 && blockIdx.x < split.workers && !split.one_launch) {
    Unfinished* items = reinterpret_cast<Unfinished*>(partial + partial_floats(split, dim));
    if (parts > 0) items[blockIdx.x] = Unfinished{at.work.first, at.work.rows, at.tile, at.head};
    reinterpret_cast<int*>(items + split.workers)[blockIdx.x] = parts;
  }
}

// kv4_prompt.hip: many rows per sequence.
bool kv4_prompt_takes(const Kv4Pool& pool, const Kv4Batch& batch, int heads, Kv4Type type, bool parents, int num_cus);
Split kv4_prompt_split(int num_cus);
hipError_t launch_kv4_prompt(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args, Kv4Type type,
                             const Split& split, float* partial, hipStream_t stream);

}  // namespace msim
