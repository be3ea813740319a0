// rotary.hip -- rotary positions of one axis or several.
//
//   a pair (x, y) of a row's head, of frequency f on axis a: angle t = p_a f,
//   (x cos t - y sin t, x sin t + y cos t), rounded once from single precision
//
// The angle is a fraction of a turn in 64-bit fixed point: p times the frequency in
// turns per position, whose product mod 2^64 drops the whole turns, so far positions
// lose nothing (an error of p 2^-65 turns).  Its upper 32 bits, less the nearest
// quarter, are an angle within pi / 4 in single precision, and sine and cosine its
// Taylor polynomials, up to 2^-28.  32 bits place the angle within 2^-30: small ones lose
// relative bits, but a result moves by 2^-30 of its pair, beside the 2^-24 of what is
// added up in single precision.
//
// Bytes bound it: every element is read and written once.  A lane has one group of
// pairs and meets it in every head of a row, so that its angles are computed once.
// 9,216 rows of 32 + 8 heads of 128 in bfloat16, 189 MB: 34 us over and over, 42 with other inputs
// each time (4.5 TB/s); over and over in f32 75 (5.0), in f16 36, adjacent pairs 1 to 3 more.  16
// rows: 4.4 us.  Loads of the first heads before the angles took
// 114 registers, and 44 us.
#include "rotary.hpp"

namespace msim {

namespace {

constexpr int kWavesPerGroup = 4;

template <Kv4Type T>
struct Elem;
template <>
struct Elem<kKv4F32> {
  typedef float type;
  static constexpr int kGroup = 4;  // pairs of a lane: 16 bytes twice
};
template <>
struct Elem<kKv4F16> {
  typedef _Float16 type;
  static constexpr int kGroup = 8;
};
template <>
struct Elem<kKv4BF16> {
  typedef __bf16 type;
  static constexpr int kGroup = 8;
};

// Cosine and sine of u / 2^64 turns.
__device__ __forceinline__ void cos_sin(uint64_t u, float& c, float& s) {
  const uint32_t t = (uint32_t)((u + 0x80000000u) >> 32), quarter = (t + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(t - (quarter << 30)) * (6.283185307179586f * 0x1p-32f), z = x * x;
  float sine = __builtin_fmaf(z, 1.0f / 362880, -1.0f / 5040);
  sine = __builtin_fmaf(z, sine, 1.0f / 120);
  sine = __builtin_fmaf(z, sine, -1.0f / 6);
  sine = __builtin_fmaf(z * x, sine, x);
  float cosine = __builtin_fmaf(z, -1.0f / 3628800, 1.0f / 40320);
  cosine = __builtin_fmaf(z, cosine, -1.0f / 720);
  cosine = __builtin_fmaf(z, cosine, 1.0f / 24);
  cosine = __builtin_fmaf(z, cosine, -0.5f);
  cosine = __builtin_fmaf(z, cosine, 1.0f);
  const float a = quarter & 1 ? sine : cosine, b = quarter & 1 ? cosine : sine;
  c = __uint_as_float(__float_as_uint(a) ^ ((quarter + 1) & 2) << 30);
  s = __uint_as_float(__float_as_uint(b) ^ (quarter & 2) << 30);
}

// A lane's elements of a head: two runs of kGroup, the first at `first`, the second at
// `second`; of runs that end before kGroup (`count`) only those.
template <typename E, int kGroup, bool kWide>
struct Runs {
  E e[2][kGroup];
  __device__ __forceinline__ void load(const E* p, const int (&at)[2], const int (&count)[2]) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if constexpr (kWide) {
        __builtin_memcpy(e[r], __builtin_assume_aligned(p + at[r], 16), 16);
      } else {
#pragma unroll
        for (int i = 0; i < kGroup; ++i) e[r][i] = i < count[r] ? p[at[r] + i] : (E)0.0f;
      }
    }
  }
  __device__ __forceinline__ void store(E* p, const int (&at)[2], const int (&count)[2]) const {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if constexpr (kWide) {
        __builtin_memcpy(__builtin_assume_aligned(p + at[r], 16), e[r], 16);
      } else {
#pragma unroll
        for (int i = 0; i < kGroup; ++i)
          if (i < count[r]) p[at[r] + i] = e[r][i];
      }
    }
  }
};

// Lanes of a head: a group of pairs each, then groups of the dims that are not turned.
// A wave has `split`-th parts of a row's heads.
template <Kv4Type T, bool kAdjacent, bool kWide>
__global__ __launch_bounds__(kWavesPerGroup* kWave) void rotary_kernel(RotaryPlan plan, RotaryRows q, RotaryRows k,
                                                                       int64_t rows,
                                                                       const int32_t* __restrict__ positions,
                                                                       int64_t axis_stride, int split) {
  typedef typename Elem<T>::type E;
  constexpr int kGroup = Elem<T>::kGroup;
  constexpr int kBatch = 4;  // heads of a lane on their way
  const int64_t wave = (int64_t)blockIdx.x * kWavesPerGroup + wave_uniform(threadIdx.x / kWave);
  const int64_t row = wave / split;
  if (row >= rows) return;
  const int part = (int)(wave - row * split), lane = lane_id();
  const int turning = (plan.pairs + kGroup - 1) / kGroup, rest = plan.dim - 2 * plan.pairs;
  const int lanes = turning + (rest + 2 * kGroup - 1) / (2 * kGroup), heads_at_once = kWave / lanes;
  const int group = lane % lanes;
  if (lane >= lanes * heads_at_once) return;

  int at[2], count[2];
  float c[kGroup], s[kGroup];
#pragma unroll
  for (int i = 0; i < kGroup; ++i) c[i] = 1.0f, s[i] = 0.0f;
  const bool turns = group < turning;
  if (turns) {
    const int pair = group * kGroup, have = min(kGroup, plan.pairs - pair);
    at[0] = kAdjacent ? 2 * pair : pair;
    at[1] = kAdjacent ? 2 * pair + kGroup : pair + plan.pairs;
    count[0] = kAdjacent ? min(kGroup, 2 * have) : have;
    count[1] = kAdjacent ? max(0, 2 * have - kGroup) : have;
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      const int p = min(pair + i, plan.pairs - 1);
      const int axis = min(max(plan.axes[p], 0), plan.num_axes - 1);
      cos_sin((uint64_t)(int64_t)positions[axis * axis_stride + row] * plan.turns[p], c[i], s[i]);
    }
  } else {
    const int first = 2 * plan.pairs + (group - turning) * 2 * kGroup;
    at[0] = first;
    at[1] = first + kGroup;
    count[0] = min(kGroup, plan.dim - first);
    count[1] = min(kGroup, max(0, plan.dim - first - kGroup));
  }

  const int heads = q.heads + k.heads, step = split * heads_at_once;
  const E* in[2] = {static_cast<const E*>(q.in) + row * q.in_row_stride,
                    static_cast<const E*>(k.in) + row * k.in_row_stride};
  E* out[2] = {static_cast<E*>(q.out) + row * q.out_row_stride, static_cast<E*>(k.out) + row * k.out_row_stride};
  for (int h0 = part * heads_at_once + lane / lanes; h0 < heads; h0 += kBatch * step) {
    Runs<E, kGroup, kWide> x[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = h0 + i * step;
      if (h >= heads) break;
      x[i].load(h < q.heads ? in[0] + h * q.in_head_stride : in[1] + (h - q.heads) * k.in_head_stride, at, count);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = h0 + i * step;
      if (h >= heads) break;
      if (turns) {
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
          E& first = kAdjacent ? x[i].e[2 * j / kGroup][2 * j % kGroup] : x[i].e[0][j];
          E& second = kAdjacent ? x[i].e[2 * j / kGroup][2 * j % kGroup + 1] : x[i].e[1][j];
          const float a = (float)first, b = (float)second;
          first = (E)__builtin_fmaf(a, c[j], -(b * s[j]));
          second = (E)__builtin_fmaf(a, s[j], b * c[j]);
        }
      }
      x[i].store(h < q.heads ? out[0] + h * q.out_head_stride : out[1] + (h - q.heads) * k.out_head_stride, at, count);
    }
  }
}

template <Kv4Type T>
hipError_t launch_type(const RotaryPlan& plan, const RotaryRows rows[2], int64_t num_rows, const int32_t* positions,
                       int64_t axis_stride, hipStream_t stream) {
  constexpr int kGroup = Elem<T>::kGroup, kSize = 16 / kGroup;
  bool wide = plan.pairs % kGroup == 0 && (plan.dim - 2 * plan.pairs) % (2 * kGroup) == 0;
  for (int i = 0; i < 2; ++i) {
    if (rows[i].heads == 0) continue;
    for (const void* p : {rows[i].in, static_cast<const void*>(rows[i].out)})
      wide = wide && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (int64_t s : {rows[i].in_row_stride, rows[i].in_head_stride, rows[i].out_row_stride, rows[i].out_head_stride})
      wide = wide && s * kSize % 16 == 0;
  }
  const int turning = (plan.pairs + kGroup - 1) / kGroup;
  const int lanes = turning + (plan.dim - 2 * plan.pairs + 2 * kGroup - 1) / (2 * kGroup);
  const int heads = rows[0].heads + rows[1].heads, at_once = kWave / lanes;
  // Waves for a row, while they are fewer than 1,024: more compute angles that one would
  // share (512 rows of 32 + 8 heads 5.6 us, 6.1 with one for each, 8.0 up to 4,096 waves).
  int split = 1;
  while (split * at_once < heads && num_rows * split < 1024) split *= 2;
  const int64_t groups = (num_rows * split + kWavesPerGroup - 1) / kWavesPerGroup;
  const dim3 grid((unsigned)groups), block(kWavesPerGroup * kWave);
  auto run = [&](auto adjacent, auto w) {
    rotary_kernel<T, decltype(adjacent)::value, decltype(w)::value>
        <<<grid, block, 0, stream>>>(plan, rows[0], rows[1], num_rows, positions, axis_stride, split);
  };
  if (plan.adjacent && wide)
    run(std::true_type{}, std::true_type{});
  else if (plan.adjacent)
    run(std::true_type{}, std::false_type{});
  else if (wide)
    run(std::false_type{}, std::true_type{});
  else
    run(std::false_type{}, std::false_type{});
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary(const RotaryPlan& plan, const RotaryRows rows[2], int64_t num_rows, const int32_t* positions,
                         int64_t axis_stride, Kv4Type type, hipStream_t stream) {
  if (num_rows <= 0 || rows[0].heads + rows[1].heads <= 0) return hipSuccess;
  switch (type) {
    case kKv4F32: return launch_type<kKv4F32>(plan, rows, num_rows, positions, axis_stride, stream);
    case kKv4F16: return launch_type<kKv4F16>(plan, rows, num_rows, positions, axis_stride, stream);
    case kKv4BF16: return launch_type<kKv4BF16>(plan, rows, num_rows, positions, axis_stride, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace msim
