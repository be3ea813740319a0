// kv4_rows.hip -- key and value rows into the 4-bit cache, and back.
//
//   append:  s = f32(max|x|) / f32(7) (0 -> 1), c = clip(rint(x / s), -7, 7)
//            as the corpus packer does, the quotient rounded to single precision
//            before rint; a row that holds an infinity or a NaN gets the scale
//            NaN (it reads back as NaN, and so does attention that reaches it)
//   read:    c * s, rounded once to the type asked for
//
// Byte work, bound by HBM: dim * (2 or 4) bytes in and dim / 2 + 4 out per row
// and head, or the reverse.  45,400 rows of 8 heads of 128 in f16, 235 MB: append
// 60 us, 3.9 TB/s, read 38 us, 6.2 TB/s (behind the append, some of it in the
// caches); 87,400 rows in bfloat16, 453 MB: read 88 us, 5.2 TB/s.
#include "kv4.hpp"

namespace msim {

namespace {

template <Kv4Type T>
struct Elem;
template <>
struct Elem<kKv4F32> {
  typedef float type;
};
template <>
struct Elem<kKv4F16> {
  typedef _Float16 type;
};
template <>
struct Elem<kKv4BF16> {
  typedef __bf16 type;
};

// Eight elements as they lie in memory.
template <Kv4Type T>
struct Raw {
  static constexpr int kWords = T == kKv4F32 ? 8 : 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const void* p, bool wide) {
    if (wide) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const v4u a = static_cast<const v4u*>(p)[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[4 * i + j] = a[j];
      }
    } else if constexpr (T == kKv4F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = static_cast<const uint32_t*>(p)[i];
    } else {
      const uint16_t* h = static_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
    }
  }
  // Element i in single precision.
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (T == kKv4F32) {
      return __uint_as_float(w[i]);
    } else if constexpr (T == kKv4BF16) {
      return __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    } else {
      return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i / 2] >> (16 * (i & 1))));
    }
  }
  // Bits of the largest magnitude, in the element's own format (ordered as
  // integers, infinities and NaNs on top).
  __device__ __forceinline__ uint32_t peak() const {
    if constexpr (T == kKv4F32) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
      return m;
    } else {
      typedef uint16_t v2s __attribute__((ext_vector_type(2)));
      v2s m = __builtin_bit_cast(v2s, w[0] & 0x7FFF7FFFu);
#pragma unroll
      for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(v2s, w[i] & 0x7FFF7FFFu));
      return max((uint32_t)m.x, (uint32_t)m.y);
    }
  }
  static constexpr uint32_t kInfinity = T == kKv4F32 ? 0x7F800000u : (T == kKv4BF16 ? 0x7F80u : 0x7C00u);
  static __device__ __forceinline__ float value(uint32_t bits) {
    if constexpr (T == kKv4F32) return __uint_as_float(bits);
    if constexpr (T == kKv4BF16) return __uint_as_float(bits << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  }
};

// Eight single precision values stored in type T, each rounded once.
template <Kv4Type T>
__device__ __forceinline__ void store8(void* p, bool wide, const float (&x)[8]) {
  typedef typename Elem<T>::type E;
  E e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = (E)x[i];
  if (wide) {
    constexpr int kWords = sizeof(E) * 8 / 16;
    v4u w[kWords];
    __builtin_memcpy(w, e, sizeof e);
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<v4u*>(p)[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) static_cast<E*>(p)[i] = e[i];
  }
}

// Lanes that share a row (8 elements each), a power of two.
constexpr int row_lanes(int dim) { return dim <= 64 ? 8 : (dim <= 128 ? 16 : 32); }

// Maximum over the N lanes of a row, by DPP within 16 lanes.
template <int N>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  auto step = [&](auto ctrl) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, decltype(ctrl)::value, 0xF, 0xF, true));
  };
  step(std::integral_constant<int, 0xB1>{});  // quad_perm [1,0,3,2]
  step(std::integral_constant<int, 0x4E>{});  // quad_perm [2,3,0,1]
  if constexpr (N == 8) {
    step(std::integral_constant<int, 0x141>{});  // row_half_mirror
  } else {
    step(std::integral_constant<int, 0x124>{});  // row_ror:4
    step(std::integral_constant<int, 0x128>{});  // row_ror:8
  }
  if constexpr (N == 32) v = max(v, (uint32_t)__shfl_xor((int)v, 16));
  return v;
}

// Slot of row `row` (each group of lanes has its own row; all 64 lanes call).
__device__ __forceinline__ bool row_slot(const Kv4Pool& pool, const Kv4Batch& batch, int row, Kv4Slot& slot) {
  const int first = wave_uniform(row);
  int b = -1;
  if (batch.offsets == nullptr) {
    b = row < min(batch.batch, batch.rows) ? row : -1;
  } else if (first < batch.rows) {
    b = kv4_find_sequence(batch, first);
    // Most waves lie inside one sequence; the others search on, lane by lane.
    if (b >= 0 && row >= kv4_first_row(batch, b + 1)) b = kv4_find_sequence_from(batch, row, b);
    if (b < 0 && row != first) b = kv4_find_sequence_from(batch, row, 0);
  }
  return row < batch.rows && b >= 0 && kv4_slot(pool, batch, b, row, slot);
}

// Codes of a lane's eight elements, element i in nibble i.  x * (1 / s) plus 1.5 *
// 2^23 leaves the code's two's complement nibble in the sum's last bits; where a
// product lies so near the middle between two codes that the correctly rounded
// quotient may round the other way, or s has no normal reciprocal, the wave
// divides.  (Products differ from quotients by less than 2^-20; near the middle is
// 2^-18.)  |x / s| rounds to 7 at most unless s is subnormal.
template <Kv4Type T>
__device__ __forceinline__ uint32_t codes8(const Raw<T>& x, float s) {
  constexpr float kMagic = 12582912.0f;
  const float inv = __builtin_amdgcn_rcpf(s);
  uint32_t t[8];
  float off = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = x[i], sum = __builtin_fmaf(v, inv, kMagic);
    off = fmaxf(off, fabsf(__builtin_fmaf(v, inv, -(sum - kMagic))));
    t[i] = __float_as_uint(sum);
  }
  if (__ballot(off > 0.5f - 0x1p-18f || s < 0x1p-125f) != 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      t[i] = (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -7.0f), 7.0f);
  }
  // Last bytes of the even and of the odd ones, then their nibbles.
  auto bytes = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) -> uint32_t {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u),
                                 0x05040100u);
  };
  const uint32_t even = bytes(t[0], t[2], t[4], t[6]), odd = bytes(t[1], t[3], t[5], t[7]);
  return (even & 0x0F0F0F0Fu) | (odd << 4 & 0xF0F0F0F0u);
}

// A workgroup has 256 / row_lanes rows, of keys (blockIdx.y 0) or values, and
// `heads` of their heads, kBatch at a time: the rows' slots are looked up once,
// and what it touches of the program's memory is contiguous.
constexpr int kBatch = 4;
constexpr int64_t kEnoughGroups = 2048;

template <Kv4Type T, int kDim>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4Pool pool, Kv4Batch batch, Kv4Rows keys, Kv4Rows values,
                                                         int heads, bool wide) {
  typedef typename Elem<T>::type E;
  constexpr int kLanes = row_lanes(kDim), kRows = 256 / kLanes;
  const int part = threadIdx.x % kLanes;
  const int row = blockIdx.x * kRows + threadIdx.x / kLanes;
  const int first = blockIdx.z * heads, last = min(pool.kv_heads, first + heads);
  const Kv4Rows& src = blockIdx.y ? values : keys;
  const bool have = row < batch.rows && part * 8 < kDim;
  const E* from = static_cast<const E*>(src.ptr) + (have ? row * src.row_stride + part * 8 : 0);
  Raw<T> x[kBatch] = {}, next[kBatch] = {};
#pragma unroll
  for (int i = 0; i < kBatch; ++i)
    if (have && first + i < last) x[i].load(from + (first + i) * src.head_stride, wide);
  Kv4Slot slot;
  const bool placed = row_slot(pool, batch, row, slot);
  uint8_t* codes = blockIdx.y ? pool.codes[1] : pool.codes[0];
  float* scales = blockIdx.y ? pool.scales[1] : pool.scales[0];
  for (int h0 = first; h0 < last; h0 += kBatch) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (have && h0 + kBatch + i < last) next[i].load(from + (h0 + kBatch + i) * src.head_stride, wide);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (h0 + i >= last) break;
      uint32_t m = lanes_max<kLanes>(x[i].peak());
      // The bits pass through an empty asm, so that this stays an integer test
      // where the compiler assumes that no value is a NaN.
      asm volatile("" : "+v"(m));
      const bool finite = m < Raw<T>::kInfinity;
      float s = finite ? __fdiv_rn(Raw<T>::value(m), 7.0f) : 1.0f;
      if (s == 0.0f) s = 1.0f;
      const uint32_t w = codes8<T>(x[i], s);
      if (placed && have) {
        const int64_t at = kv4_pool_row(pool, slot.page, h0 + i, slot.slot);
        *reinterpret_cast<uint32_t*>(codes + at * (kDim / 2) + part * 4) = finite ? w : 0;
        if (part == 0) reinterpret_cast<uint32_t*>(scales)[at] = finite ? __float_as_uint(s) : 0x7FC00000u;
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) x[i] = next[i];
  }
}

template <Kv4Type T, int kDim>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Pool pool, Kv4Batch batch, Kv4Rows keys, Kv4Rows values,
                                                       int heads, bool wide) {
  typedef typename Elem<T>::type E;
  constexpr int kLanes = row_lanes(kDim), kRows = 256 / kLanes;
  const int part = threadIdx.x % kLanes;
  const int row = blockIdx.x * kRows + threadIdx.x / kLanes;
  const int first = blockIdx.z * heads, last = min(pool.kv_heads, first + heads);
  const Kv4Rows& dst = blockIdx.y ? values : keys;
  Kv4Slot slot;
  const bool placed = row_slot(pool, batch, row, slot);
  if (row >= batch.rows || part * 8 >= kDim) return;
  const uint8_t* codes = blockIdx.y ? pool.codes[1] : pool.codes[0];
  const float* scales = blockIdx.y ? pool.scales[1] : pool.scales[0];
  E* to = static_cast<E*>(dst.ptr) + row * dst.row_stride + part * 8;
  for (int h0 = first; h0 < last; h0 += kBatch) {
    uint32_t w[kBatch];
    float s[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      w[i] = 0;
      s[i] = 0.0f;
      if (placed && h0 + i < last) {
        const int64_t at = kv4_pool_row(pool, slot.page, h0 + i, slot.slot);
        w[i] = *reinterpret_cast<const uint32_t*>(codes + at * (kDim / 2) + part * 4);
        s[i] = scales[at];
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (h0 + i >= last) break;
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = (float)((int)(w[i] << (28 - 4 * j)) >> 28) * s[i];
      store8<T>(to + (h0 + i) * dst.head_stride, wide, x);
    }
  }
}

// 16-byte accesses: every row of every head starts on 16 bytes.
bool rows_aligned(const Kv4Rows& r, int size) {
  return reinterpret_cast<uintptr_t>(r.ptr) % 16 == 0 && r.row_stride * size % 16 == 0 && r.head_stride * size % 16 == 0;
}

template <Kv4Type T, int kDim>
hipError_t launch_rows(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4Rows rows[2], bool append,
                       hipStream_t stream) {
  constexpr int kRows = 256 / row_lanes(kDim);
  const int size = T == kKv4F32 ? 4 : 2;
  const bool wide = rows_aligned(rows[0], size) && rows_aligned(rows[1], size);
  // All heads in one workgroup, or as few as give every CU some workgroups. 8 heads
  // of 128, append in bfloat16: 512 rows 3.8 us with one each against 7.4 with all,
  // 45,000 rows 78 against 64 (read 58 against 37).
  const int64_t tiles = (batch.rows + kRows - 1) / kRows;
  int heads = pool.kv_heads;
  while (heads > 1 && tiles * 2 * ((pool.kv_heads + heads - 1) / heads) < kEnoughGroups) heads = (heads + 1) / 2;
  const dim3 grid((unsigned)tiles, 2, (unsigned)((pool.kv_heads + heads - 1) / heads));
  if (append)
    kv4_append_kernel<T, kDim><<<grid, dim3(256), 0, stream>>>(pool, batch, rows[0], rows[1], heads, wide);
  else
    kv4_read_kernel<T, kDim><<<grid, dim3(256), 0, stream>>>(pool, batch, rows[0], rows[1], heads, wide);
  return hipGetLastError();
}

template <Kv4Type T>
hipError_t launch_type(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4Rows rows[2], bool append,
                       hipStream_t stream) {
  switch (pool.dim) {
    case 64: return launch_rows<T, 64>(pool, batch, rows, append, stream);
    case 96: return launch_rows<T, 96>(pool, batch, rows, append, stream);
    case 128: return launch_rows<T, 128>(pool, batch, rows, append, stream);
    case 192: return launch_rows<T, 192>(pool, batch, rows, append, stream);
    case 256: return launch_rows<T, 256>(pool, batch, rows, append, stream);
  }
  return hipErrorInvalidValue;
}

hipError_t launch(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4Rows rows[2], Kv4Type type, bool append,
                  hipStream_t stream) {
  if (batch.rows <= 0) return hipSuccess;
  switch (type) {
    case kKv4F32: return launch_type<kKv4F32>(pool, batch, rows, append, stream);
    case kKv4F16: return launch_type<kKv4F16>(pool, batch, rows, append, stream);
    case kKv4BF16: return launch_type<kKv4BF16>(pool, batch, rows, append, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_kv4_append(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4Rows rows[2], Kv4Type type,
                             hipStream_t stream) {
  return launch(pool, batch, rows, type, true, stream);
}

hipError_t launch_kv4_read(const Kv4Pool& pool, const Kv4Batch& batch, const Kv4Rows rows[2], Kv4Type type,
                           hipStream_t stream) {
  return launch(pool, batch, rows, type, false, stream);
}

}  // namespace msim
