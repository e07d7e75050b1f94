// Device side of the 8-bit activation format (quant8.h): steps, codes and the
// SiLU of what codes stand for, shared by the elementwise kernels and the
// GEMM epilogues.
#pragma once

#include <stdint.h>

#include "quant8.h"
#include "vec.cuh"

namespace es {

struct Step8 {
  float inv;  // 2^-e, or 0 for a block that holds an infinity or a NaN
  int byte;   // e + 127, or kQuantNan
};

// amax_bits: the largest |x| of the block as fp32 bits (infinities and NaN sort above every finite value).
__device__ __forceinline__ Step8 step8_of(uint32_t amax_bits) {
  int e = static_cast<int>(amax_bits >> 23) - 127 - 6;
  if (e < -126) e = -126;
  float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  if (rintf(__uint_as_float(amax_bits) * inv) > 127.0f) {
    ++e;
    inv *= 0.5f;
  }
  if (amax_bits >= 0x7f800000u) return {0.0f, kQuantNan};
  return {inv, e + 127};
}

// 2^e of an exponent byte; NaN for kQuantNan.
__device__ __forceinline__ float scale8_of(int byte) {
  return byte == kQuantNan ? __uint_as_float(0x7fc00000u) : __uint_as_float(static_cast<uint32_t>(byte) << 23);
}

// The same where nothing clamps what codes stand for: 64 steps of 2^122, the largest there are, would be past 32 bits,
// and are the largest 32-bit value with a step that is one rounding smaller.
constexpr int kTopStep = 122 + 127;
__device__ __forceinline__ float finite_scale8_of(int byte) {
  return byte == kTopStep ? __uint_as_float((static_cast<uint32_t>(byte) << 23) - 1u) : scale8_of(byte);
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t bytes_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// A code, in the low byte.  1.5 2^23 + x 2^-e rounds to the nearest whole number
// (ties to even) in one FMA, whose low byte is the code in two's complement.
constexpr float kCodeMagic = 12582912.0f;

// Four codes of one block in a word.
__device__ __forceinline__ uint32_t codes8_of(float a, float b, float c, float d, const Step8& s) {
  const uint32_t w =
      bytes_of(__float_as_uint(fmaf(a, s.inv, kCodeMagic)), __float_as_uint(fmaf(b, s.inv, kCodeMagic)),
               __float_as_uint(fmaf(c, s.inv, kCodeMagic)), __float_as_uint(fmaf(d, s.inv, kCodeMagic)));
  return s.byte == kQuantNan ? 0u : w;
}

// One code, in the low byte; 0 for an infinity or a NaN, whose block has inv 0 (the maximum drops the NaN).
__device__ __forceinline__ uint32_t code8_of(float x, float inv) {
  return __float_as_uint(fmaxf(fmaf(x, inv, kCodeMagic), 0.0f));
}

// Code i of a word of four: the byte, its sign bit flipped, below 2^23 as a float is code + 128 + 2^23.
__device__ __forceinline__ float code8_at(uint32_t word, int i) {
  const uint32_t f = __byte_perm(word ^ 0x80808080u, 0x4b000000u, 0x7440 | i);
  return __uint_as_float(f) - 8388736.0f;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sigmoids of two values with one reciprocal, s1 = e2' / (e1' e2') with
// e' = 1 + e^-x.  Below -43, where silu is under 10^-17, x is taken as -43: the
// product of the two stays in range.  (A NaN makes both NaN: for what codes stand
// for, where NaN blocks are NaN whole.)  e1, e2: e^-x.  For results of 16 bits.
__device__ __forceinline__ void sigmoid_pair(float& x1, float& x2, float& s1, float& s2, float& e1, float& e2) {
  x1 = max_nan(x1, -43.0f);
  x2 = max_nan(x2, -43.0f);
  e1 = exp2_approx(x1 * -1.4426950408889634f);
  e2 = exp2_approx(x2 * -1.4426950408889634f);
  const float d1 = 1.0f + e1, d2 = 1.0f + e2;
  const float r = __fdividef(1.0f, d1 * d2);
  s1 = r * d2;
  s2 = r * d1;
}
__device__ __forceinline__ void sigmoid_pair(float& x1, float& x2, float& s1, float& s2) {
  float e1, e2;
  sigmoid_pair(x1, x2, s1, s2, e1, e2);
}

// The same of values that may be NaN each by itself.
__device__ __forceinline__ void sigmoid_apart(float& x1, float& x2, float& s1, float& s2) {
  const bool bad1 = x1 != x1, bad2 = x2 != x2;
  if (bad1) x1 = 0.0f;
  if (bad2) x2 = 0.0f;
  sigmoid_pair(x1, x2, s1, s2);
  if (bad1) x1 = __uint_as_float(0x7fc00000u);
  if (bad2) x2 = __uint_as_float(0x7fc00000u);
}

// silu' = s (1 + x (1 - s)) with 1 - s = e^-x s: a difference would leave a rounding of s, which a large x multiplies.
__device__ __forceinline__ float silu_slope(float x, float s, float e) { return s * fmaf(x * e, s, 1.0f); }

}  // namespace es
