// linear4.hip -- y = x W^T for few rows x and a matrix W in 4 bits:
//
//   y_mn = sum over groups G of s_nG (sum_{k in G} x_mk c_nk)  (+ bias_n)
//
// On v_mfma_f32_16x16x32: A is 16 rows of W times 32 columns, B the same
// columns of up to 16 rows of x, so that a lane's accumulators are four rows
// of W (its scales) by one row of x.  A group's sum is a chain of group / 32
// MFMAs; its scales multiply the sum, in single precision, and nothing else is
// dequantised.
//
// Codes in the registers of the MFMA.  A word holds eight columns of a row as
// nibbles, turned left by three bits, and becomes eight exact values:
//   bfloat16 x: turned back, the conversion of four bits to sixteenths and a merge
//     per pair, 14 operations a word.
//   f16 x: bits 3..6 of a half, under a constant exponent, make 136 + code; 136 is
//     subtracted, 11 operations.
//   f32 x: three bfloat16 parts that sum to x exactly; codes under a constant
//     exponent as (24 + code) / 1024, 24 / 1024 subtracted in single precision.
// So every product is exact, and a column whose code is zero adds nothing: with the
// 24 left in the codes and taken off the sum (7 operations) a column of x 1e7 times
// the others left its rounding in results that it has no part in.
//
// Bytes bound it: n k / 2 and the scales, for any number of rows that fits a
// pass (16; 32 in groups of 128 and 16 bits).  Waves of a workgroup take the 128-column tiles of the same rows of W
// in turn and join in LDS in a fixed order.  One row by 4096 x 4096 takes 4.8 us (the
// host side of a call is 4.2); 16 rows by 28672 x 8192 in groups of 64 take 30.2 us,
// 4.2 TB/s, of which the decoding that does not hide costs two.
#include "codes4.hpp"
#include "linear4.hpp"

namespace msim {

namespace {

// One thread per word of the laid-out codes.
__global__ __launch_bounds__(256) void linear4_layout_kernel(const uint8_t* __restrict__ codes,
                                                             const uint16_t* __restrict__ scales, int64_t n,
                                                             int64_t k, int group, uint32_t* __restrict__ out_codes,
                                                             uint16_t* __restrict__ out_scales) {
  const int64_t tiles_k = (k + 127) / 128, words = linear4_tiles(n, k) * 256;
  const int per_tile = 128 / group;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < words; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t tile = i / 256;
    const int lane = (int)(i % 256) / 4, c = (int)(i % 4);
    const int64_t row = tile / tiles_k * 16 + lane % 16, col = tile % tiles_k * 128 + 32 * c + 8 * (lane / 16);
    uint32_t w = 0;
    if (row < n && col < k) {
      const uint32_t src = *reinterpret_cast<const uint32_t*>(codes + row * (k / 2) + col / 2);
#pragma unroll
      for (int j = 0; j < 8; ++j) w |= ((src >> (4 * j)) & 15u) << (4 * (j / 2) + 16 * (j & 1));
    }
    out_codes[i] = w << 3 | w >> 29;
    const int g = (int)(i % 256);
    if (g < 16 * per_tile) {  // [4][per_tile][4 rows]
      const int64_t srow = tile / tiles_k * 16 + g / (4 * per_tile) * 4 + g % 4;
      const int64_t at = tile % tiles_k * per_tile + g / 4 % per_tile;
      out_scales[tile * 16 * per_tile + g] = srow < n && at < k / group ? scales[srow * (k / group) + at] : 0;
    }
  }
}

template <Kv4Type T>
struct Operand {
  typedef v8b type;
  static constexpr int kParts = 1;
};
template <>
struct Operand<kKv4F16> {
  typedef v8h type;
  static constexpr int kParts = 1;
};
template <>
struct Operand<kKv4F32> {
  typedef v8b type;
  static constexpr int kParts = 3;
};

// Eight codes of a word, over code_unit().  Single precision x reach the largest
// numbers, and 128 products with codes of 2^-7 at most stay below them; for bfloat16
// one_result() takes the sums that do not.
constexpr float code_unit(Kv4Type type) { return type == kKv4F16 ? 1.0f : (type == kKv4BF16 ? kCodeUnit : 1024.0f); }
template <Kv4Type T>
__device__ __forceinline__ typename Operand<T>::type decode(uint32_t w) {
  if constexpr (T == kKv4BF16) {
    return decode_word_bf16(__builtin_amdgcn_alignbit(w, w, 3));
  } else {
    const uint32_t p[4] = {w, w >> 4, w >> 8, __builtin_amdgcn_alignbit(w, w, 12)};
    v4u r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = T == kKv4F16 ? pair_f16(p[i]) : pair_bf16(p[i]);
    return __builtin_bit_cast(typename Operand<T>::type, r);
  }
}

// Eight elements of a row of x as they lie in memory.
template <int kWords>
__device__ __forceinline__ void load_x(const void* p, bool wide, uint32_t (&x)[kWords]) {
  if (wide) {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const v4u a = static_cast<const v4u*>(p)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * i + j] = a[j];
    }
  } else if constexpr (kWords == 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<const uint32_t*>(p)[i];
  } else {
    const uint16_t* src = static_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = src[2 * i] | (uint32_t)src[2 * i + 1] << 16;
  }
}

// The same as MFMA operands.
template <Kv4Type T, int kWords>
__device__ __forceinline__ void operands(const uint32_t (&u)[kWords],
                                         typename Operand<T>::type (&x)[Operand<T>::kParts]) {
  if constexpr (T == kKv4F32) {
    split3(u, x);
  } else {
    x[0] = __builtin_bit_cast(typename Operand<T>::type, (v4u){u[0], u[1], u[2], u[3]});
  }
}

// y_mn of a bfloat16 row and row n of W, by one thread, the scales before the sums.
// Sums of products alone pass the largest number where a few x of nearly that size add
// up, whatever their scale leaves of them: results that are no numbers come from here.
// (An exponent less in every code costs 2.6 us of 30 at 16 rows by 28672 x 8192.)
__device__ __forceinline__ float one_result(const Linear4Matrix& w, const uint16_t* x, int n) {
  const int tiles_k = (w.k + 127) / 128, per_tile = 128 / w.group;
  float y = 0.0f;
#pragma unroll 1
  for (int k = 0; k < w.k; k += 8) {
    const int64_t tile = (int64_t)(n / 16) * tiles_k + k / 128;
    const uint32_t turned =
        reinterpret_cast<const uint32_t*>(w.codes)[(tile * kWave + k % 32 / 8 * 16 + n % 16) * 4 + k % 128 / 32];
    const uint32_t word = __builtin_amdgcn_alignbit(turned, turned, 3);
    const float s = __uint_as_float(
        (uint32_t)w.scales[(tile * 4 + n % 16 / 4) * 4 * per_tile + k % 128 / w.group * 4 + n % 4] << 16);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int code = (int)(word << (28 - 4 * (j / 2) - 16 * (j & 1))) >> 28;
      y = __builtin_fmaf(__uint_as_float((uint32_t)x[k + j] << 16), (float)code * s, y);
    }
  }
  return y;
}

// Waves of a workgroup, by their registers.
constexpr int most_waves(Kv4Type type, int groups, int cols, int row_tiles) {
  return type != kKv4F32 && cols == 1 && groups * row_tiles <= 4 ? 16 : 8;
}

// kRowTiles tiles of 16 rows of W, kCols of 16 rows of x per workgroup.
template <Kv4Type T, int kGroups, int kCols, int kRowTiles>
__global__ __launch_bounds__(kWave* most_waves(T, kGroups, kCols, kRowTiles)) void linear4_kernel(Linear4Matrix w, const void* __restrict__ x, int64_t rows,
                                                      int64_t x_row_stride, bool wide, void* __restrict__ out,
                                                      int64_t out_row_stride) {
  constexpr int kParts = Operand<T>::kParts;
  constexpr int kSize = T == kKv4F32 ? 4 : 2;
  typedef uint32_t XTile[4][kCols][T == kKv4F32 ? 8 : 4];
  extern __shared__ float s_acc[];
  const int lane = lane_id(), col = lane % 16, g = lane / 16;
  const int wave = wave_uniform(threadIdx.x / kWave), waves = blockDim.x / kWave;
  const int tiles_k = (w.k + 127) / 128, tiles_n = (w.n + 15) / 16;
  const int n0 = blockIdx.x * kRowTiles;
  const int64_t m0 = (int64_t)blockIdx.y * 16 * kCols;

  auto load_w = [&](int kt, v4u (&codes)[kRowTiles], uint32_t (&scales)[kRowTiles][kGroups * 2]) {
#pragma unroll
    for (int r = 0; r < kRowTiles; ++r) {
      const int64_t tile = (int64_t)min(n0 + r, tiles_n - 1) * tiles_k + kt;
      codes[r] = reinterpret_cast<const v4u*>(w.codes)[tile * kWave + lane];
      const uint32_t* s = reinterpret_cast<const uint32_t*>(w.scales) + (tile * 4 + g) * kGroups * 2;
#pragma unroll
      for (int i = 0; i < kGroups * 2; ++i) scales[r][i] = s[i];
    }
  };
  // Rows past the last are the last one again (their columns of the result are
  // not written), columns past the last the last ones (their codes and scales are
  // zeros).
  const char* xrow[kCols];
#pragma unroll
  for (int j = 0; j < kCols; ++j)
    xrow[j] = static_cast<const char*>(x) + (min(m0 + 16 * j + col, rows - 1) * x_row_stride + 8 * g) * kSize;
  auto load_rows = [&](int kt, XTile& t) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int k = min(kt * 128 + 32 * c, w.k - 32);
#pragma unroll
      for (int j = 0; j < kCols; ++j) load_x(xrow[j] + (int64_t)k * kSize, wide, t[c][j]);
    }
  };

  v4f acc[kRowTiles][kCols];
#pragma unroll
  for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
    for (int j = 0; j < kCols; ++j) acc[r][j] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};

  auto multiply = [&](const v4u (&codes)[kRowTiles], const uint32_t (&scales)[kRowTiles][kGroups * 2],
                      const XTile& t) {
    typename Operand<T>::type b[4][kCols][kParts];
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int j = 0; j < kCols; ++j) operands<T>(t[c][j], b[c][j]);
    // A row tile's sums meet their scales one row tile later, behind the next
    // one's decoding and products: MFMA results are not read right after they are
    // issued.
    v4f sum[2][kGroups][kCols];
    auto scale = [&](int r) {
#pragma unroll
      for (int i = 0; i < kGroups; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t s2 = scales[r][i * 2 + e / 2];
          const float s = __uint_as_float(e & 1 ? s2 & 0xFFFF0000u : s2 << 16);
#pragma unroll
          for (int j = 0; j < kCols; ++j) acc[r][j][e] = __builtin_fmaf(s, sum[r % 2][i][j][e], acc[r][j][e]);
        }
    };
#pragma unroll
    for (int r = 0; r < kRowTiles; ++r) {
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) sum[r % 2][i][j] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = i * 4 / kGroups; c < (i + 1) * 4 / kGroups; ++c) {
          const typename Operand<T>::type a = decode<T>(codes[r][c]);
#pragma unroll
          for (int j = 0; j < kCols; ++j)
#pragma unroll
            for (int p = 0; p < kParts; ++p) sum[r % 2][i][j] = mfma(a, b[c][j][p], sum[r % 2][i][j]);
        }
      }
      if (r == 0) continue;
#pragma unroll
      for (int i = 0; i < kGroups; ++i)
#pragma unroll
        for (int j = 0; j < kCols; ++j) asm volatile("" : "+v"(sum[0][i][j]), "+v"(sum[1][i][j]));
      scale(r - 1);
    }
    mfma_results_fence();
    scale(kRowTiles - 1);
  };

  // The next tile of x is on its way during a tile's products, and the next tiles
  // of W too where the registers hold them.
  constexpr bool kBoth = kRowTiles <= 4 && kGroups * kCols * kRowTiles <= 8;
  v4u codes[kBoth ? 2 : 1][kRowTiles];
  uint32_t scales[kBoth ? 2 : 1][kRowTiles][kGroups * 2];
  XTile xs[2];
  if (wave < tiles_k) {
    load_rows(wave, xs[0]);
    load_w(wave, codes[0], scales[0]);
  }
  for (int k0 = wave; k0 < tiles_k; k0 += 2 * waves) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const int kt = k0 + d * waves;
      if (kt >= tiles_k) break;
      const bool more = kt + waves < tiles_k;
      if (more) load_rows(kt + waves, xs[1 - d]);
      if constexpr (kBoth) {
        if (more) load_w(kt + waves, codes[1 - d], scales[1 - d]);
        multiply(codes[d], scales[d], xs[d]);
      } else {
        multiply(codes[0], scales[0], xs[d]);
        if (more) load_w(kt + waves, codes[0], scales[0]);
      }
    }
  }

  // [wave][row tile][column tile][element][lane]
  constexpr int kPerWave = kRowTiles * kCols * 4 * kWave;
#pragma unroll
  for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
    for (int j = 0; j < kCols; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s_acc[wave * kPerWave + ((r * kCols + j) * 4 + e) * kWave + lane] = acc[r][j][e];
  __syncthreads();
  for (int i = threadIdx.x; i < kPerWave; i += blockDim.x) {
    const int n_in = i % (16 * kRowTiles), m_in = i / (16 * kRowTiles);
    const int r = n_in / 16, e = n_in % 4, l = n_in % 16 / 4 * 16 + m_in % 16, j = m_in / 16;
    const int n = n0 * 16 + n_in;
    const int64_t m = m0 + m_in;
    if (n >= w.n || m >= rows) continue;
    float y = 0.0f;
    for (int v = 0; v < waves; ++v) y += s_acc[v * kPerWave + ((r * kCols + j) * 4 + e) * kWave + l];
    y *= code_unit(T);
    if constexpr (T == kKv4BF16) {
      uint32_t bits = __float_as_uint(y);
      asm volatile("" : "+v"(bits));  // an integer test, where the compiler assumes that there are no NaNs
      if ((bits & 0x7F800000u) == 0x7F800000u)
        y = one_result(w, static_cast<const uint16_t*>(x) + m * x_row_stride, n);
    }
    if (w.bias != nullptr) y += w.bias[n];
    const int64_t at = m * out_row_stride + n;
    if constexpr (T == kKv4F32) static_cast<float*>(out)[at] = y;
    if constexpr (T == kKv4F16) static_cast<_Float16*>(out)[at] = (_Float16)y;
    if constexpr (T == kKv4BF16) static_cast<__bf16*>(out)[at] = (__bf16)y;
  }
}

template <Kv4Type T, int kGroups, int kCols, int kRowTiles>
hipError_t launch_shape(const Linear4Matrix& w, const void* x, int64_t rows, int64_t x_row_stride, void* out,
                        int64_t out_row_stride, int num_cus, hipStream_t stream) {
  const int size = T == kKv4F32 ? 4 : 2;
  const bool wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && x_row_stride * size % 16 == 0;
  const int64_t gx = ((w.n + 15) / 16 + kRowTiles - 1) / kRowTiles, gy = (rows + 16 * kCols - 1) / (16 * kCols);
  if (gy > 65535) return hipErrorInvalidValue;
  // Enough waves for the CUs' latency, within the tiles there are and the LDS
  // that joins them (one row by 4096 x 4096 5.1 us, with four waves 5.8; by 28672 x
  // 8192 27.8 and 32.2; three matrices in turn).
  const int tiles_k = (w.k + 127) / 128;
  int waves = 4;
  while (waves < most_waves(T, kGroups, kCols, kRowTiles) && waves * 2 <= tiles_k && gx * gy * waves < num_cus * 16)
    waves *= 2;
  const size_t lds = sizeof(float) * waves * kRowTiles * kCols * 4 * kWave;
  linear4_kernel<T, kGroups, kCols, kRowTiles><<<dim3((unsigned)gx, (unsigned)gy), dim3(waves * kWave), lds, stream>>>(
      w, x, rows, x_row_stride, wide, out, out_row_stride);
  return hipGetLastError();
}

// Row tiles that the registers hold without spilling.
constexpr int most_row_tiles(Kv4Type type, int groups, int cols) {
  return groups * cols >= 4 || (type == kKv4F32 && groups > 1) ? 4 : 7;
}

template <Kv4Type T, int kGroups, int kCols>
hipError_t launch_columns(const Linear4Matrix& w, const void* x, int64_t rows, int64_t x_row_stride, void* out,
                          int64_t out_row_stride, int num_cus, hipStream_t stream) {
  // Row tiles of a workgroup: the busiest CU has its workgroups' row tiles to do,
  // and with each workgroup the rows of x, whose loads (16 rows apart) cost as
  // much as two row tiles; one row costs half of one. At 4096 x 4096 one tile takes
  // 5.1 us for a row and 7.0 for 16, as many as the registers hold (seven)
  // 12.0 and 15.0; at 28672 x 8192 60 us against 31 for 16 rows.
  const int64_t tiles = (w.n + 15) / 16, columns = (rows + 16 * kCols - 1) / (16 * kCols);
  auto cost = [&](int row_tiles) -> int64_t {
    const int64_t groups = (tiles + row_tiles - 1) / row_tiles * columns;
    return (groups + num_cus - 1) / num_cus * (2 * row_tiles + (rows > 1 ? 4 * kCols : 1));
  };
  constexpr int kMost = most_row_tiles(T, kGroups, kCols);
  int best = 1;
  for (int row_tiles : {2, 4, 7})
    if (row_tiles <= kMost && cost(row_tiles) <= cost(best)) best = row_tiles;
  if constexpr (kMost >= 7)
    if (best == 7)
      return launch_shape<T, kGroups, kCols, 7>(w, x, rows, x_row_stride, out, out_row_stride, num_cus, stream);
  if constexpr (kMost >= 4)
    if (best == 4)
      return launch_shape<T, kGroups, kCols, 4>(w, x, rows, x_row_stride, out, out_row_stride, num_cus, stream);
  if constexpr (kMost >= 2)
    if (best == 2)
      return launch_shape<T, kGroups, kCols, 2>(w, x, rows, x_row_stride, out, out_row_stride, num_cus, stream);
  return launch_shape<T, kGroups, kCols, 1>(w, x, rows, x_row_stride, out, out_row_stride, num_cus, stream);
}

template <Kv4Type T, int kGroups>
hipError_t launch_group(const Linear4Matrix& w, const void* x, int64_t rows, int64_t x_row_stride, void* out,
                        int64_t out_row_stride, int num_cus, hipStream_t stream) {
  // From 17 rows on, two column tiles read and decode W once for both, where the
  // registers leave them as many row tiles: 16-bit x, groups of 128. 32 rows by 28672 x
  // 8192 take 40 us against 54 with one, by 4096 x 4096, which one spreads over more
  // CUs, 10.7 against 9.4. The others lose: by 28672 x 8192 in groups of 32 86 us with
  // two and 76 with one, in single precision 220 to 238 and 97 to 143; groups of 64 tie.
  if constexpr (kGroups == 1 && T != kKv4F32)
    if (rows > 16) return launch_columns<T, kGroups, 2>(w, x, rows, x_row_stride, out, out_row_stride, num_cus, stream);
  return launch_columns<T, kGroups, 1>(w, x, rows, x_row_stride, out, out_row_stride, num_cus, stream);
}

template <Kv4Type T>
hipError_t launch_type(const Linear4Matrix& w, const void* x, int64_t rows, int64_t x_row_stride, void* out,
                       int64_t out_row_stride, int num_cus, hipStream_t stream) {
  switch (w.group) {
    case 32: return launch_group<T, 4>(w, x, rows, x_row_stride, out, out_row_stride, num_cus, stream);
    case 64: return launch_group<T, 2>(w, x, rows, x_row_stride, out, out_row_stride, num_cus, stream);
    case 128: return launch_group<T, 1>(w, x, rows, x_row_stride, out, out_row_stride, num_cus, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_linear4_layout(const uint8_t* codes, const uint16_t* scales, int64_t n, int64_t k, int group,
                                 uint8_t* out_codes, uint16_t* out_scales, hipStream_t stream) {
  const int64_t words = linear4_tiles(n, k) * 256;
  const int64_t blocks = std::min<int64_t>((words + 255) / 256, 65536);
  if (blocks <= 0) return hipSuccess;
  linear4_layout_kernel<<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(
      codes, scales, n, k, group, reinterpret_cast<uint32_t*>(out_codes), out_scales);
  return hipGetLastError();
}

hipError_t launch_linear4(const Linear4Matrix& w, const void* x, int64_t rows, int64_t x_row_stride, Kv4Type type,
                          void* out, int64_t out_row_stride, int num_cus, hipStream_t stream) {
  if (rows <= 0) return hipSuccess;
  switch (type) {
    case kKv4F32: return launch_type<kKv4F32>(w, x, rows, x_row_stride, out, out_row_stride, num_cus, stream);
    case kKv4F16: return launch_type<kKv4F16>(w, x, rows, x_row_stride, out, out_row_stride, num_cus, stream);
    case kKv4BF16: return launch_type<kKv4BF16>(w, x, rows, x_row_stride, out, out_row_stride, num_cus, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace msim
