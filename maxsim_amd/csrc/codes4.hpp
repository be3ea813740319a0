// codes4.hpp -- 4-bit codes and single precision values as operands of
// v_mfma_f32_16x16x32_f16 / _bf16.
#pragma once

#include "common.hpp"

namespace msim {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

__device__ __forceinline__ v4f mfma(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mfma(v8b a, v8b b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// A pair of codes, bits 3..6 of both halves.  Under a constant exponent they are
// 136 + code in f16 and (24 + code) / 1024 in bfloat16 (the sign bit turned); the
// differences, in f16 and in single precision, are exact.
__device__ __forceinline__ uint32_t pair_f16(uint32_t w) {
  const v2h base = {(_Float16)136.0f, (_Float16)136.0f};
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, (w & 0x00780078u) ^ 0x58405840u) - base);
}
__device__ __forceinline__ uint32_t pair_bf16(uint32_t w) {
  const uint32_t r = (w & 0x00780078u) ^ 0x3CC03CC0u;
  const float base = 24.0f / 1024.0f, lo = __uint_as_float(r << 16) - base, hi = __uint_as_float(r & 0xFFFF0000u) - base;
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

// Eight codes of a word over 16 as bfloat16, pairs (code i, code i + 4): the
// conversion of four bits (-8 .. 7 to sixteenths in single precision, a byte's low
// half being any byte of a register) and the upper halves of two.
constexpr float kCodeUnit = 16.0f;
__device__ __forceinline__ v8b decode_word_bf16(uint32_t w) {
  uint32_t odd = w >> 4;
  asm("" : "+v"(odd));  // so that bytes of it are taken, and not others of w by shifts
  auto pair = [](uint32_t x, int byte) -> uint32_t {
    return __builtin_amdgcn_perm(
        __float_as_uint(__builtin_amdgcn_cvt_off_f32_i4(__builtin_amdgcn_ubfe(x, 8 * byte + 16, 8))),
        __float_as_uint(__builtin_amdgcn_cvt_off_f32_i4(__builtin_amdgcn_ubfe(x, 8 * byte, 8))), 0x07060302u);
  };
  return __builtin_bit_cast(v8b, (v4u){pair(w, 0), pair(odd, 0), pair(w, 1), pair(odd, 1)});
}

// Three bfloat16 parts (in the upper halves) that sum to x exactly: the upper
// eight bits of the significand, the next eight, the rest.  An infinity or a
// NaN is its first part alone.
__device__ __forceinline__ void split3(uint32_t x, uint32_t (&part)[3]) {
  const bool special = (x & 0x7F800000u) == 0x7F800000u;
  const uint32_t a = x & 0xFFFF0000u;
  const float r1 = special ? 0.0f : __uint_as_float(x) - __uint_as_float(a);
  const uint32_t b = __float_as_uint(r1) & 0xFFFF0000u;
  part[0] = special && (x & 0x007FFFFFu) ? 0x7FC00000u : a;
  part[1] = b;
  part[2] = __float_as_uint(r1 - __uint_as_float(b));
}

// Eight single precision values as three operands, which sum to them exactly.
__device__ __forceinline__ void split3(const uint32_t (&x)[8], v8b (&out)[3]) {
  v4u parts[3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t lo[3], hi[3];
    split3(x[2 * i], lo);
    split3(x[2 * i + 1], hi);
#pragma unroll
    for (int k = 0; k < 3; ++k) parts[k][i] = __builtin_amdgcn_perm(hi[k], lo[k], 0x07060302u);
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) out[k] = __builtin_bit_cast(v8b, parts[k]);
}

// Eight as two, 16 bits of them: the upper eight bits of the significand, and the
// rest rounded.
__device__ __forceinline__ void in_parts(const float (&x)[8], v8b (&out)[2]) {
  v4u parts[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = __float_as_uint(x[2 * i]), hi = __float_as_uint(x[2 * i + 1]);
    parts[0][i] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
    const float a = x[2 * i] - __uint_as_float(lo & 0xFFFF0000u), b = x[2 * i + 1] - __uint_as_float(hi & 0xFFFF0000u);
    typedef __bf16 v2b __attribute__((ext_vector_type(2)));
    parts[1][i] = __builtin_bit_cast(uint32_t, (v2b){(__bf16)a, (__bf16)b});
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) out[k] = __builtin_bit_cast(v8b, parts[k]);
}
__device__ __forceinline__ void in_parts(const float (&x)[8], v8b (&out)[3]) {
  uint32_t bits[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) bits[i] = __float_as_uint(x[i]);
  split3(bits, out);
}

}  // namespace msim
