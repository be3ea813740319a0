// kv4_prompt.hip -- attention over the 4-bit cache for many query rows per
// sequence (prompts and their pieces), bfloat16 and f16.
//
// The products are those of kv4_attend.hip, S^T = C Q^T and O^T = D^T P^T, here
// on v_mfma_f32_32x32x16_f16 and _bf16, and operations bound them instead of bytes: 4 dim
// per (row, key).  So the codes are decoded once per workgroup of 256 query rows
// and not once per wave:
//   * eight waves have 32 rows each, in registers, and 128 keys at a time: four
//     waves decode the keys to f16, four the values to bfloat16, into one of two buffers of
//     LDS, while all work on the other; one barrier per 128 keys;
//   * LDS holds the MFMAs' A operands in lane order (16 bytes a lane), so every
//     read of it is contiguous: keys [32 keys][16 dims], values [16 keys][32 dims];
//   * a lane keeps one query row (column lane % 32) and 16 of a tile's 32 keys:
//     8 i + 4 (lane / 32) + j.  The values' contraction slots are numbered the
//     same way, so the probabilities stay in their registers;
//   * row i of a value operand's tile t is dim 8 w + d with 32 t + i = w + d
//     (dim / 8): the lanes that decode one word of codes each then write 16-byte
//     pieces side by side.
// A probability times its value scale is the sum of two bfloat16 (16 bits, at any
// size: the smallest is single precision's). One f16 would do for the larger
// products and take 1010 us where this takes 1220, but outputs to which only
// products below 2^-22 of the row's largest contribute would lose bits, as happens
// in ordinary peaked rows.
// Per (row, key) the scores cost a lane a product with the key scale, half a
// maximum, a fused multiply-add, an exponential (four slots), a sum, a product
// with the value scale and three slots for its parts: 12 issue slots for each of a
// lane's 16 of 32 x 32 scores, 770 clocks, and with the decoding of the codes
// about 900 against the MFMAs' 24 x 32. Two waves per SIMD run one's products
// beside the other's exponentials, which hides only a part: 32 MFMAs of 521 ns
// beside 144 vector operations of 480 ns took 727.
// 2 x 2048 tokens behind up to 15,000, 32 heads of 128 on 8, bfloat16: 0.83 TFLOP
// (4 dim per row and key that it sees) in 1.20 to 1.30 ms, by the card, 0.64 to 0.69
// PFLOP/s.
#include "kv4_split.hpp"

namespace msim {

namespace {

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kPromptWaves = 8;
constexpr int kPromptRows = 32 * kPromptWaves;
constexpr int kKeys = 128;  // of a buffer
__device__ __forceinline__ v16f mfma32(v8h a, v8h b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v16f mfma32(v8b a, v8b b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

template <int kDim>
struct Buffer {
  static constexpr int kKeyBytes = kKeys * kDim * 2;  // [32 keys][16 dims][lane] of 16 bytes
  static constexpr int kScales = 2 * kKeyBytes;       // key scales, value scales, 1 for a hole
  static constexpr int kBytes = kScales + 3 * kKeys * 4;
};

// What a thread brings of the next 128 keys: half a key's codes, or a word of
// eight value rows, and a scale.
template <int kDim>
struct Staged {
  static constexpr int kWords = kDim / 16 > 8 ? kDim / 16 : 8;
  uint32_t words[kWords];
  float scale;
  bool hole;
};

template <int kDim>
__device__ __forceinline__ int staged_key(int thread) {
  if (thread < 256) return thread % kKeys;
  const int kg = (thread - 256) / 16;  // keys 32 s + 16 c + 4 g + {0..3, 8..11}
  return kg / 4 * 32 + kg / 2 % 2 * 16 + kg % 2 * 4;
}

__device__ __forceinline__ int page_of(const Kv4Pool& pool, const Kv4Batch& batch, int seq, int length, int key) {
  return key < length ? batch.table[(int64_t)seq * batch.max_pages + (key >> pool.page_shift)] : -1;
}

template <int kDim>
__device__ __forceinline__ void stage(const Kv4Pool& pool, int page, int head, int key, Staged<kDim>& s) {
  const int thread = threadIdx.x;
  s.hole = (uint32_t)page >= (uint32_t)pool.num_pages;
  const int64_t at = kv4_pool_row(pool, s.hole ? 0 : page, head, key & ((1 << pool.page_shift) - 1));
  if (thread < 256) {
    constexpr int kHalf = kDim / 16;
    const uint32_t* src =
        reinterpret_cast<const uint32_t*>(pool.codes[0] + at * (kDim / 2) + thread / kKeys * (kHalf * 4));
#pragma unroll
    for (int i = 0; i < kHalf; ++i) s.words[i] = src[i];
    s.scale = (thread < kKeys ? pool.scales[0] : pool.scales[1])[at];
  } else {
    const int w = min(thread % 16, kDim / 8 - 1);
    const uint8_t* src = pool.codes[1] + at * (kDim / 2) + w * 4;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      s.words[i] = *reinterpret_cast<const uint32_t*>(src + (i / 4 * 8 + i % 4) * (kDim / 2));
  }
}

template <int kDim>
__device__ __forceinline__ void unstage(const Staged<kDim>& s, char* buffer) {
  typedef Buffer<kDim> B;
  const int thread = threadIdx.x;
  if (thread < 256) {
    constexpr int kHalf = kDim / 16;
    const int key = thread % kKeys;
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      const int word = thread / kKeys * kHalf + i;
      *reinterpret_cast<v8h*>(buffer + (((key / 32) * (kDim / 16) + word / 2) * 64 + word % 2 * 32 + key % 32) * 16) =
          decode_word(s.words[i]);
    }
    float* scales = reinterpret_cast<float*>(buffer + B::kScales);
    scales[thread] = thread < kKeys ? s.scale : s.scale * (1.0f / kValueUnit);
    if (thread < kKeys) scales[2 * kKeys + key] = s.hole ? 1.0f : 0.0f;
  } else if (thread % 16 < kDim / 8) {
    const int w = thread % 16, kg = (thread - 256) / 16;
    char* values = buffer + B::kKeyBytes + kg / 2 * (kDim * 32);  // of 16 keys
    const int g = kg % 2;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      v8b pair[4];  // [pair of keys]: four dims of both
#pragma unroll
      for (int p = 0; p < 4; ++p)
        pair[p] = decode_word_bf16(
            __builtin_amdgcn_perm(s.words[2 * p + 1], s.words[2 * p], half ? 0x07060302u : 0x05040100u));
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        v8b a;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          a[2 * p] = pair[p][2 * d];
          a[2 * p + 1] = pair[p][2 * d + 1];
        }
        const int line = (half * 4 + d) * (kDim / 8) + w;
        *reinterpret_cast<v8b*>(values + (line / 32 * 64 + g * 32 + line % 32) * 16) = a;
      }
    }
  }
}

__device__ __forceinline__ float other_half_max(float v) { return fmaxf(v, __shfl_xor(v, 32)); }

template <Kv4Type T, int kDim>
__device__ __forceinline__ void prompt_item(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args,
                                            const Split& split, float* __restrict__ partial, const Cursor& at,
                                            uint32_t from, uint32_t upto, char* s_raw) {
  typedef Buffer<kDim> B;
  constexpr int kChunks = kDim / 16, kTiles = kDim / 32;
  const int lane = lane_id(), col = lane % 32, g = lane / 32, wave = wave_uniform(threadIdx.x / kWave);
  const SeqWork& u = at.work;

  // The first keys' way to registers.
  const int begin = at.range.low + (int)(from << split.granule_shift);
  const int end = (int)min((int64_t)at.range.low + ((int64_t)upto << split.granule_shift), (int64_t)at.range.high);
  Staged<kDim> staged;
  int key = begin + staged_key<kDim>(threadIdx.x);
  stage<kDim>(pool, page_of(pool, batch, at.seq, u.length, key), at.head, key, staged);

  // This wave's query rows.
  v8h q[kChunks];
  const uint32_t r = (at.tile << split.tile_shift) + wave * 32 + col;
  const int token = (int)(r / split.share), sub = (int)(r - token * split.share);
  const bool have = token < u.rows;
  float factor;
  {
    const int64_t base = have ? (int64_t)(u.first + token) * args.q_row_stride +
                                    (int64_t)(at.head * split.share + sub) * args.q_head_stride
                              : 0;
    typedef typename std::conditional<T == kKv4F16, _Float16, uint16_t>::type E;
    auto value = [](uint32_t word, int i) -> float {
      const uint16_t h = (uint16_t)(word >> (16 * (i & 1)));
      return T == kKv4F16 ? (float)__builtin_bit_cast(_Float16, h) : __uint_as_float((uint32_t)h << 16);
    };
    const E* src = static_cast<const E*>(args.q) + base + g * 8;
    v4u raw[kChunks];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      if (!have) {
        raw[i] = (v4u){0, 0, 0, 0};
      } else if (args.q_wide) {
        raw[i] = *reinterpret_cast<const v4u*>(src + i * 16);
      } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(src + i * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[i][j] = h[2 * j] | (uint32_t)h[2 * j + 1] << 16;
      }
    }
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(value(raw[i][j / 2], j)) & 0x7FFFFFFFu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    const int shift = query_shift(top);
    // The factor towards log2 scores is kept positive: maxima are taken before it.
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = value(raw[i][word_order(j) / 2], word_order(j));
        q[i][j] = (_Float16)ldexpf(args.scale_log2 < 0.0f ? -x : x, shift);
      }
    factor = score_factor(args.scale_log2, shift);
  }
  const int pos = u.length - u.rows + token;
  int see_low = pos >= args.window ? pos - args.window + 1 : 0;
  int see_high = args.causal ? max(0, min(u.length, pos + 1)) : u.length;
  const uint8_t* mask = nullptr;
  if (args.mask != nullptr) {
    see_high = (int)min((int64_t)see_high, args.mask_width);
    mask = args.mask + (have ? (int64_t)(u.first + token) * args.mask_row_stride : 0);
  }
  const bool sees = have && see_high > see_low;
  if (!have) {  // a row of padding: nothing depends on what it sees
    see_low = 0;
    see_high = args.mask != nullptr ? 0 : INT_MAX;
  }
  const int all_low = wave_reduce(see_low, [](int a, int b) { return max(a, b); });
  const int all_high = wave_reduce(see_high, [](int a, int b) { return min(a, b); });
  const int any_low = wave_reduce(sees ? see_low : INT_MAX, [](int a, int b) { return min(a, b); });
  const int any_high = wave_reduce(sees ? see_high : 0, [](int a, int b) { return max(a, b); });

  float ref = kUnset, sum = 0.0f;
  v16f o[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) o[t] = (v16f)(0.0f);

  unstage<kDim>(staged, s_raw);
  key += kKeys;
  int page = page_of(pool, batch, at.seq, u.length, key + kKeys);
  stage<kDim>(pool, page_of(pool, batch, at.seq, u.length, key), at.head, key, staged);
  __syncthreads();
  char* now = s_raw;
  char* other = s_raw + B::kBytes;
  for (int key0 = begin; key0 < end; key0 += kKeys) {
    if (key0 + kKeys < end) {
      unstage<kDim>(staged, other);
      key += kKeys;
      stage<kDim>(pool, page, at.head, key, staged);
      page = page_of(pool, batch, at.seq, u.length, key + kKeys);
    }
    const float* scales = reinterpret_cast<const float*>(now + B::kScales);
    const v8h* keys = reinterpret_cast<const v8h*>(now) + lane;
    const v8b* values = reinterpret_cast<const v8b*>(now + B::kKeyBytes) + lane;
    // The 32-key steps that this wave's rows see something of.
    const int step0 = max(0, any_low - key0) / 32, step1 = min(kKeys, any_high - key0 + 31) / 32;
#pragma unroll 1
    for (int st = step0; st < step1; ++st) {
      const int first = key0 + 32 * st;
      v4f k4[4], v4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        k4[i] = *reinterpret_cast<const v4f*>(scales + 32 * st + 8 * i + 4 * g);
        v4[i] = *reinterpret_cast<const v4f*>(scales + kKeys + 32 * st + 8 * i + 4 * g);
      }
      v16f s = (v16f)(0.0f);
#pragma unroll
      for (int i = 0; i < kChunks; ++i) s = mfma32(keys[(st * kChunks + i) * kWave], q[i], s);
      // The step's values are read beside the products.
      __builtin_amdgcn_sched_barrier(0);
      v8b va[2][kTiles];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t = 0; t < kTiles; ++t) va[c][t] = values[((2 * st + c) * kTiles + t) * kWave];
      mfma_results_fence();
      float x[16], vs[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = s[i] * k4[i / 4][i % 4], vs[i] = v4[i / 4][i % 4];
      if (!(first >= all_low && first + 32 <= all_high && args.mask == nullptr && first + 32 <= u.length) ||
          __ballot(scales[2 * kKeys + 32 * st + col] != 0.0f) != 0) {
        // A hidden key takes no part in the maxima, and its probability and
        // value scale are zeros whatever the cache holds there.
        uint32_t seen[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          seen[i] = args.mask != nullptr ? mask_bytes(mask, first + 8 * i + 4 * g, see_high) : 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int local = 8 * (i / 4) + 4 * g + i % 4, k = first + local;
          const bool see = k >= see_low && k < see_high && scales[2 * kKeys + 32 * st + local] == 0.0f &&
                           (seen[i / 4] >> (8 * (i % 4)) & 0xFFu) != 0;
          x[i] = see ? x[i] : kNegInf;
          vs[i] = see ? vs[i] : 0.0f;
        }
      }
      const float top = max_of(x) * factor;
      if (__ballot(top > ref + kTopLimit) != 0) {
        const float next = fmaxf(ref, other_half_max(top));
        const float alpha = exp2_hw(ref - next);
        ref = next;
        sum *= alpha;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) o[t] *= alpha;
      }
      v8b probs[2][2];
      float more = 0.0f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = exp2_hw(__builtin_fmaf(x[8 * c + i], factor, -ref));
          (i & 1 ? more : sum) += p;
          y[i] = p * vs[8 * c + i];
        }
        in_parts(y, probs[c]);
      }
      sum += more;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int t = 0; t < kTiles; ++t) o[t] = mfma32(va[c][t], probs[c][p], o[t]);
    }
    char* swap = now;
    now = other;
    other = swap;
    __syncthreads();
  }
  mfma_results_fence();

  // Each wave turns its outputs about in LDS and writes its rows.
  constexpr int kPitch = kDim + 4;
  float* mine = reinterpret_cast<float*>(s_raw) + wave * 32 * kPitch;
  int turn = g;
  asm volatile("" : "+v"(turn));  // or 64 addresses are kept from before the loop
  sum += __shfl_xor(sum, 32);
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int line = 32 * t + 8 * (i / 4) + 4 * turn + i % 4;
      mine[col * kPitch + line % (kDim / 8) * 8 + line / (kDim / 8)] = o[t][i];
    }
  wave_sync_lds();
  const bool whole_item = from == 0 && upto == at.range.granules;
  constexpr int kPerRow = kDim / 4;
#pragma unroll 1
  for (int i = lane; i < 32 * kPerRow; i += kWave) {
    const int local = i / kPerRow, d = i % kPerRow * 4;
    const uint32_t row = (at.tile << split.tile_shift) + wave * 32 + local;
    const int tok = (int)(row / split.share), qh = at.head * split.share + (int)(row - tok * split.share);
    const float all = __shfl(ref, local), total = __shfl(sum, local);
    if (tok >= u.rows) continue;
    v4f y = *reinterpret_cast<const v4f*>(mine + local * kPitch + d);
    if (!whole_item) {
      float* dst = partial_slot(partial, split, kDim, blockIdx.x, from == 0);
      *reinterpret_cast<v4f*>(dst + (wave * 32 + local) * kDim + d) = y;
      if (d == 0) {
        dst[kPromptRows * kDim + 2 * (wave * 32 + local)] = all;
        dst[kPromptRows * kDim + 2 * (wave * 32 + local) + 1] = total;
      }
      continue;
    }
    const int64_t out_row = u.first + tok;
    if (args.lse != nullptr && d == 0) args.lse[out_row * args.heads + qh] = log_sum(all, total);
    y *= output_factor(total);
    store4<T>(args.out, out_row * args.out_row_stride + (int64_t)qh * args.out_head_stride + d, args.out_wide != 0, y);
  }
}

template <Kv4Type T, int kDim>
__global__ __launch_bounds__(kPromptWaves* kWave, 2) void kv4_prompt_kernel(Kv4Pool pool, Kv4Batch batch,
                                                                           Kv4AttendArgs args, Split split,
                                                                           float* __restrict__ partial) {
  constexpr int kOutputs = kPromptRows * (kDim + 4) * 4;
  __shared__ __attribute__((aligned(16)))
  char s_raw[2 * Buffer<kDim>::kBytes > kOutputs ? 2 * Buffer<kDim>::kBytes : kOutputs];
  if (__builtin_expect(blockIdx.x >= split.workers, 0)) {
    loose_rows<T, kDim>(batch, args, split);
    return;
  }
  Deal deal;
  Cursor at;
  if (!find_work(pool, batch, args, split, blockIdx.x, at.seq, at.before, deal)) {
    note_unfinished(partial, split, kDim, at, 0);
    return;
  }
  uint32_t granule = deal.begin(blockIdx.x);
  const uint32_t last = deal.begin(blockIdx.x + 1);
  at.enter(pool, batch, args, split);
  int parts = 0;
  while (granule < last && at.seek(pool, batch, args, split, granule)) {
    const uint32_t from = granule - at.item_at, upto = min(at.range.granules, last - at.item_at);
    prompt_item<T, kDim>(pool, batch, args, split, partial, at, from, upto, s_raw);
    granule = at.item_at + upto;
    if (from == 0 && upto < at.range.granules)
      parts = (int)(deal.worker_of(at.item_at + at.range.granules - 1) - blockIdx.x) + 1;
    __syncthreads();
  }
  note_unfinished(partial, split, kDim, at, parts);
}

template <Kv4Type T>
hipError_t launch(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args, const Split& split,
                  float* partial, hipStream_t stream) {
  const dim3 grid(split.workers + loose_groups(batch)), block(kPromptWaves * kWave);
  switch (pool.dim) {
    case 64: kv4_prompt_kernel<T, 64><<<grid, block, 0, stream>>>(pool, batch, args, split, partial); break;
    case 96: kv4_prompt_kernel<T, 96><<<grid, block, 0, stream>>>(pool, batch, args, split, partial); break;
    case 128: kv4_prompt_kernel<T, 128><<<grid, block, 0, stream>>>(pool, batch, args, split, partial); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

bool kv4_prompt_takes(const Kv4Pool& pool, const Kv4Batch& batch, int heads, Kv4Type type) {
  // Two workgroups' rows per sequence and head on average, or one where the items
  // fill half the CUs: fewer leave CUs, or parts of them, without work. Heads of
  // 128, 32 on 8, this kernel against kv4_attend.hip's: 8 x 128 tokens behind 4,000
  // keys 136 us against 151, 8 x 96 129 against 123, 8 x 64 87 against 85, 8 x 32 70
  // against 52; 2 x 128 behind 16,000 135 against 141; 32 x 256 behind 1,000, 8 heads
  // on 8, 71 against 114.
  const int64_t rows = (int64_t)batch.rows * (heads / pool.kv_heads), whole = (int64_t)batch.batch * kPromptRows;
  return type != kKv4F32 && pool.dim <= 128 && batch.offsets != nullptr &&
         (rows >= 2 * whole || (rows >= whole && rows * pool.kv_heads >= 128 * kPromptRows));
}

Split kv4_prompt_split(int num_cus) {
  Split s{};
  s.tile_shift = __builtin_ctz(kPromptRows);
  s.workers = num_cus;  // LDS holds one workgroup per CU
  s.few = 0;
  return s;
}

hipError_t launch_kv4_prompt(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4AttendArgs& args, Kv4Type type,
                             const Split& split, float* partial, hipStream_t stream) {
  return type == kKv4F16 ? launch<kKv4F16>(pool, batch, args, split, partial, stream)
                         : launch<kKv4BF16>(pool, batch, args, split, partial, stream);
}

}  // namespace msim
