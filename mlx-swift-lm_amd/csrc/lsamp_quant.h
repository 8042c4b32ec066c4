// lsamp_quant.h — a row's values as 8-bit integers of one scale:
//   s = max(max |x| (1 / 127), 2^-126),  q = rint(x / s), the exact quotient.
#ifndef LSAMP_QUANT_H
#define LSAMP_QUANT_H

#include <hip/hip_runtime.h>

#include <stdint.h>

namespace lsamp {

// A row's scale from the largest bit pattern of its magnitudes (a NaN's is above an
// infinity's, that above every number's).
__device__ __forceinline__ uint32_t magnitude(float v) {
  return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
}
__device__ __forceinline__ float row_scale(uint32_t top) {
  return top < 0x7f800000u ? fmaxf(__builtin_bit_cast(float, top) * (1.f / 127.f), 1.17549435e-38f)
                           : NAN;
}

// q of eight values as eight bytes, given 1 / scale (rounded).  q = rint(x / s) by one fma
// with 1.5 2^23, whose sum has q in its last byte: off by one at most, near a tie.  e = x
// - q s is exact (both are multiples of the smaller one's last place); where no |e| of a
// wave reaches half a step the q are right, which is nearly always, and where one does
// they are put right.  Nothing exceeds 127: |x| / s <= 127 (1 + 2^-22).  (A row whose
// scale is NaN: q = 0.)
__device__ __forceinline__ uint64_t quantize8(const float (&x)[8], float scale, float inverse) {
  constexpr float kRound = 12582912.f;
  const float half = 0.5f * scale;
  uint32_t bits[8];
  bool near = false;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float f = fmaf(x[k], inverse, kRound);
    const float e = fmaf(kRound - f, scale, x[k]);
    bits[k] = __builtin_bit_cast(uint32_t, f);
    near |= !(fabsf(e) < half);
  }
  if (__any(near)) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float q = __builtin_bit_cast(float, bits[k]) - kRound;
      const float e = fmaf(-q, scale, x[k]);
      const bool odd = bits[k] & 1;
      if (e > half || (e == half && odd)) ++bits[k];
      if (e < -half || (e == -half && odd)) --bits[k];
      if (scale != scale) bits[k] = 0;
    }
  }
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t a = __builtin_amdgcn_perm(bits[4 * i + 1], bits[4 * i], 0x0c0c0400);
    const uint32_t b = __builtin_amdgcn_perm(bits[4 * i + 3], bits[4 * i + 2], 0x04000c0c);
    w[i] = a | b;
  }
  return (uint64_t)w[1] << 32 | w[0];
}

}  // namespace lsamp

#endif
