// Codes of 8 bits with a scale for each block of 16 tokens and key head, a power of two.
// A code has at most 8 significant bits, so that its value, code times scale, is a bf16
// number: what is read back is what the attention sees, to the bit.  Only e4m3's can pass the
// largest one (255 2^120 is rounded to 256 2^120): their value is that one.
#pragma once

#include "common.hpp"

namespace umic {

constexpr int kBlockTokens = 16;  // that share a scale
constexpr int kLeastExp = -100;   // of a scale

// The checks of a cache that entry points share (cache8.hip); cap: keys that table_w of its
// pages hold.
int check_cache8(const umic_cache8_t* cache, int64_t& cap, int64_t table_w);

template <int FORMAT>
struct Codes;

constexpr float kMost = 0x1.fep127f;      // bf16's largest number
constexpr float kMostScale = 0x1p120f;    // from it on a code's value can pass it
constexpr int kMostBits = (127 + 120) << 23;
// 2^97.  From it on a scale, times a weight of the softmax, can pass what fp32 holds, and so
// can products of codes with elements of q (wide_q).
constexpr int kWideBits = (127 + 97) << 23;

// Two bf16 numbers, infinite ones as the largest.
__device__ __forceinline__ uint32_t at_most(uint32_t w) {
  if ((w & 0x7fffu) == 0x7f80u) w -= 1u;
  if ((w & 0x7fff0000u) == 0x7f800000u) w -= 0x10000u;
  return w;
}
__device__ __forceinline__ u32x2 at_most(u32x2 v) { return u32x2{at_most(v[0]), at_most(v[1])}; }
__device__ __forceinline__ u32x4 at_most(u32x4 v) {
  return u32x4{at_most(v[0]), at_most(v[1]), at_most(v[2]), at_most(v[3])};
}

// Whether one of these bf16 numbers is 2^97 or more, infinite or NaN: the exponents' upper
// three bits, both halves of a word at once.
__device__ __forceinline__ uint32_t wide_q(u32x4 v) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) any |= (v[i] & 0x70007000u) + 0x10001000u;
  return any & 0x80008000u;
}

// Scales are such that a block's largest magnitude is 2^7 to 2^8 codes, below e4m3's
// largest, 448: its bits, but for the three of a code's fraction, are the exponent's.
template <>
struct Codes<UMIC_CODES_E4M3> {
  static constexpr int kTop = 7;
  static constexpr bool kPasses = true;  // values can pass bf16's largest number
  // two bf16 numbers of the low (HI: high) half of w
  template <bool HI>
  static __device__ __forceinline__ uint32_t pair(uint32_t w, float scale = 1.0f) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
  }
  // four codes as four bf16 numbers
  static __device__ __forceinline__ u32x2 four(uint32_t w, float scale = 1.0f) {
    return u32x2{pair<false>(w, scale), pair<true>(w, scale)};
  }
  // codes c of a and c of b side by side, as bf16 numbers
  static __device__ __forceinline__ void turn(uint32_t a, uint32_t b, uint32_t (&o)[4]) {
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x05010400u);
    const uint32_t hi = __builtin_amdgcn_perm(b, a, 0x07030602u);
    o[0] = pair<false>(lo), o[1] = pair<true>(lo);
    o[2] = pair<false>(hi), o[3] = pair<true>(hi);
  }
  // four values, in units of the scale, to the nearest codes
  static __device__ __forceinline__ uint32_t round4(const float* x) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true);
  }
  static __device__ __forceinline__ void values4(uint32_t w, float* x) {
    x[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0), x[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
    x[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2), x[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
  }
};

// A block's largest magnitude is 2^6 to 2^7 codes.  A bf16 number of 8 significant bits
// is then at most 127.5 codes, and rounds to 127 at worst by half a step.
template <>
struct Codes<UMIC_CODES_INT8> {
  static constexpr int kTop = 6;
  static constexpr bool kPasses = false;
  static __device__ __forceinline__ void values4(uint32_t w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  }
  static __device__ __forceinline__ uint32_t halves(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  }
  static __device__ __forceinline__ u32x2 four(uint32_t w, float scale = 1.0f) {
    float x[4];
    values4(w, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= scale;
    return u32x2{halves(x[0], x[1]), halves(x[2], x[3])};
  }
  static __device__ __forceinline__ void turn(uint32_t a, uint32_t b, uint32_t (&o)[4]) {
    float x[4], y[4];
    values4(a, x);
    values4(b, y);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = halves(x[i], y[i]);
  }
  static __device__ __forceinline__ uint32_t round4(const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)  // 1.5 2^23: the sum's last place is 1, its low byte the code
      w[i] = __float_as_uint(__builtin_amdgcn_fmed3f(x[i], -127.0f, 127.0f) + 12582912.0f);
    const uint32_t lo = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(w[3], w[2], 0x0c0c0400u);
    return lo | hi << 16;
  }
};

}  // namespace umic
