// Values to int8 with a scale: what the row quantiser and the append to the int8 cache share.
#pragma once
#include "causal.h"

// the least scale of values that are not all 0: scales of one cache stay within 2^-64 .. 2^121, so that the attention can hold their ratios in 32 bits
constexpr float HXA_Q8_LEAST = 0x1p-64f;

// the scale of values whose largest finite magnitude is top (by the rounded 1 / 127: at most an ulp beside the quotient, without a division)
HXA_DEV float q8_scale(float top) { return top > 0.0f ? fmaxf(top * (1.0f / 127.0f), HXA_Q8_LEAST) : 0.0f; }
// |x|, 0 where it is not finite
HXA_DEV float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.0f;
}
// eight values x inv, rounded to the nearest integer (ties to even) within +-127, as bytes; NaN becomes 0. The sum with 1.5 2^23 rounds, and its
// low byte is the integer's.
HXA_DEV uint2_t q8_pack(const float (&x)[8], float inv) {
  uint32_t b[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    float r = x[e] * inv;
    r = r == r ? r : 0.0f;
    r = fminf(fmaxf(r, -127.0f), 127.0f);
    b[e] = __builtin_bit_cast(uint32_t, r + 12582912.0f);
  }
  auto four = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400), __builtin_amdgcn_perm(b, a, 0x0c0c0400), 0x05040100);
  };
  return (uint2_t){four(b[0], b[1], b[2], b[3]), four(b[4], b[5], b[6], b[7])};
}
