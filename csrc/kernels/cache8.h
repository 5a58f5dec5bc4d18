// The paged key / value cache in 8 bits: what its writer (cache8.hip) and the attention off it
// (attn_cache8.hip) share.
//
// Pages [n_blocks, Hkv, BLK, D] of int8 or OCP e4m3 codes; an f32 scale per page and head, of keys and of
// values: an entry stands for code * scale. Both kinds of codes are f16 values exactly (int8: 1024 + (c + 128)
// formed by bytes, less 1152; e4m3: the hardware's conversion), so products run on the f16 MFMAs without
// a rounding of what is cached. A scale under C8_LEAST (a negative one too) counts as C8_LEAST to all that read it.
#pragma once
#include "common.h"

#define C8_INT8 0
#define C8_E4M3 1
#define C8_LEAST 7.888609052210118e-31f           // 2^-100

typedef _Float16 c8_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 c8_h8 __attribute__((ext_vector_type(8)));
typedef unsigned c8_u2 __attribute__((ext_vector_type(2)));
typedef unsigned c8_u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float c8_least(float s) { return s < C8_LEAST ? C8_LEAST : s; }   // NaN stays

// four codes -> four f16
template <int KIND> __device__ __forceinline__ c8_u2 c8_widen(unsigned w) {
  if constexpr (KIND == C8_INT8) {
    const unsigned x = w ^ 0x80808080u;           // c + 128, 0 .. 255
    const c8_h2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
    const c8_h2 lo = __builtin_bit_cast(c8_h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) + off;
    const c8_h2 hi = __builtin_bit_cast(c8_h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) + off;
    return c8_u2{__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi)};
  } else {
    return c8_u2{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))};
  }
}

template <int KIND> __device__ __forceinline__ c8_h8 c8_widen8(unsigned lo, unsigned hi) {
  const c8_u2 a = c8_widen<KIND>(lo), b = c8_widen<KIND>(hi);
  return __builtin_bit_cast(c8_h8, c8_u4{a[0], a[1], b[0], b[1]});
}

// four codes -> four f32
template <int KIND> __device__ __forceinline__ float4v c8_floats(unsigned w) {
  if constexpr (KIND == C8_INT8) {
    return float4v{(float)(int)(signed char)w, (float)(int)(signed char)(w >> 8), (float)(int)(signed char)(w >> 16), (float)((int)w >> 24)};
  } else {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    return float4v{a[0], a[1], b[0], b[1]};
  }
}

// v / s to the nearest code (ties to even), at most the largest one; a quotient that is no number gives the largest
template <int KIND> __device__ __forceinline__ unsigned c8_codes(const float4v& v, float s) {
  constexpr float most = KIND == C8_INT8 ? 127.f : 448.f;
  float4v x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = fmaxf(fminf(v[i] / s, most), -most);
  if constexpr (KIND == C8_INT8) {
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= ((unsigned)(int)rintf(x[i]) & 255u) << (8 * i);
    return w;
  } else {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
  }
}

// the scale of a page whose largest magnitude has the bits `top` (infinities and NaN stay what they are)
template <int KIND> __device__ __forceinline__ unsigned c8_scale(unsigned top) {
  if (top >= 0x7f800000u) return top;
  if constexpr (KIND == C8_INT8) return __float_as_uint(__uint_as_float(top) / 127.f);
  // the power of two at or above a quotient: rows that are rounded again to a larger scale only lose
  // what falls below e4m3's smallest exponent
  else return (__float_as_uint(__uint_as_float(top) / 448.f) + 0x7fffffu) & 0x7f800000u;
}
