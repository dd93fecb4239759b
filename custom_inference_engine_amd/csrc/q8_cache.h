// The 8-bit paged cache: K and V rows in e4m3 with a power-of-two scale for each
// block of 16 tokens, kv head and K / V.
//
// A block is one 16-key tile of one kv head: rows [16 i, 16 i + 16) of a page
// (page_size is a multiple of 16).  Pools are (n_pages, H_kv, page_size, D)
// bytes; scales are (n_pages, H_kv, page_size / 16, 2) fp32, [0] K's and [1] V's,
// each 2^e with -15 <= e <= 8.  A held value is byte * 2^e.
//
// Why powers of two, and that range: a byte's value times 2^e is then always an
// fp16 value — the smallest step is 2^-9 * 2^-15 = 2^-24, fp16's own, and the
// largest value held is 240 * 2^8 = 61440 (larger inputs are limited to it, at
// most 6.2 % off: half an e4m3 step) — so the attention kernels convert tiles to
// exact fp16 operands (one v_cvt_scalef32_pk_f16_fp8 for two values, scale
// included) and lose nothing after the cache's own rounding.  A block whose scale
// grows by 2^n has its rows rounded again; their bytes change exactly (the
// exponent moves) unless they fall under e4m3's smallest normal, 2^-6: then by at
// most half of 2^-9, in the new scale, each time.  Over all growths that is less than
// 2^-9 of the last scale (the halves of steps that double at least: 1/2 + 1/4 + ..).
//
// e of a block is the least with amax <= 448 * 2^e, over the rows written since
// its first row was: writing a block's row 0 starts it anew (its page may have
// been another sequence's), writing any other row keeps the others.  Each value
// is rounded once, to nearest even, from its fp16 input.  NaN is held as NaN and
// does not enter amax.
#pragma once

#include <type_traits>

#include "cie_common.h"

namespace cie {

constexpr int kQ8Block = 16;     // tokens that share a scale
constexpr int kQ8EMin = -15, kQ8EMax = 8;
constexpr uint32_t kQ8Limit = 0x7b80;  // fp16 bits of 61440

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Fp16 magnitudes order as their bits.  q8_raw_max: the largest of eight (NaN the largest of all); where a wave's is
// past the limit (rare) q8_limit8 first brings the values to it, and q8_mag8 leaves NaN out.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t q8_raw_max(const f16x8& x, uint32_t m) {
  const u32x4 w = __builtin_bit_cast(u32x4, x);
  u16x2 t = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fffu);
#pragma unroll
  for (int i = 1; i < 4; ++i) t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
  return max(m, (uint32_t)max(t[0], t[1]));
}
// (by value: a bit cast of a vector's element as an lvalue reads its first one)
__device__ __forceinline__ uint32_t q8_bits(f16 x) { return __builtin_bit_cast(uint16_t, x); }
__device__ __forceinline__ uint32_t q8_mag8(const f16x8& x, uint32_t m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = q8_bits(x[i]) & 0x7fff;
    m = max(m, a > 0x7c00 ? 0 : min(a, kQ8Limit));
  }
  return m;
}
__device__ __forceinline__ void q8_limit8(f16x8& x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t h = q8_bits(x[i]), a = h & 0x7fff;
    x[i] = __builtin_bit_cast(f16, (uint16_t)((a > kQ8Limit && a <= 0x7c00 ? kQ8Limit : a) | (h & 0x8000)));
  }
}

// Least e with amax <= 448 * 2^e (448 = 1.75 * 2^8), from amax's fp16 bits.
__device__ __forceinline__ int q8_exponent(uint32_t mag) {
  const int e = (int)(mag >> 10) - 15 - 8 + ((mag & 0x3ff) > 0x300 ? 1 : 0);
  return max(kQ8EMin, min(kQ8EMax, e));
}

// 2^e as fp32, and the exponent of a stored scale (limited, so that a word that
// no append wrote does no harm).
__device__ __forceinline__ float q8_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ int q8_scale_exponent(float s) {
  const int e = (int)((__float_as_uint(s) >> 23) & 0xff) - 127;
  return max(kQ8EMin, min(kQ8EMax, e));
}

// Eight fp16 values over scale = 2^e, rounded to e4m3 (v_cvt_scalef32_pk_fp8_f16, two values: to nearest even, as one
// rounding of the exact quotient; checked over every fp16 value and scale).  At most 448 where e covers the values.
__device__ __forceinline__ u32x2 q8_round8(const f16x8& x, float scale) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  u32x2 r;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    s16x2 b = {0, 0};
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(b, f16x2{x[4 * w], x[4 * w + 1]}, scale, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(b, f16x2{x[4 * w + 2], x[4 * w + 3]}, scale, true);
    r[w] = __builtin_bit_cast(uint32_t, b);
  }
  return r;
}

// Four e4m3 bytes times 2^-n (n >= 0), rounded again.
__device__ __forceinline__ uint32_t q8_rescale4(uint32_t b, float factor) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)b, false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)b, true);
  const int r = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * factor, lo[1] * factor, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * factor, hi[1] * factor, r, true);
}

// Two bytes of a word (its low or high half) as exact fp16 values.
template <bool HI>
__device__ __forceinline__ f16x2 q8_pair(uint32_t b, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, scale, HI);
}

// Eight consecutive bytes as fp16 values.
__device__ __forceinline__ f16x8 q8_values8(uint32_t lo, uint32_t hi, float scale) {
  const f16x2 a = q8_pair<false>(lo, scale), b = q8_pair<true>(lo, scale);
  const f16x2 c = q8_pair<false>(hi, scale), d = q8_pair<true>(hi, scale);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Over the wave's 64 lanes (every lane active): wave_max's steps on integers.
__device__ __forceinline__ uint32_t q8_wave_mag(uint32_t m) {
  auto ror = [](uint32_t x, auto n) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + decltype(n)::value, 0xf, 0xf, false);
  };
  m = max(m, ror(m, std::integral_constant<int, 8>{}));
  m = max(m, ror(m, std::integral_constant<int, 4>{}));
  m = max(m, ror(m, std::integral_constant<int, 2>{}));
  m = max(m, ror(m, std::integral_constant<int, 1>{}));
  const auto a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  m = max((uint32_t)a[0], (uint32_t)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  return max((uint32_t)b[0], (uint32_t)b[1]);
}

}  // namespace cie
