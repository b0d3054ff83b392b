// fk_e4m3.h — 8-bit values (e4m3: 448 the largest, no infinity) with scales
// that are powers of two: the smallest, from 2^-126 on, that keeps the largest
// finite magnitude of a block within 448.
#pragma once

#include "fk_common.h"

namespace fk {

typedef short e4m3_short2 __attribute__((ext_vector_type(2)));
typedef float e4m3_float2 __attribute__((ext_vector_type(2)));

// The bits of the largest finite magnitude of eight values; those that are
// not finite are made NaN.  Few wavefronts hold any, so the others do not pay for
// looking at each (5 operations an element fewer: a norm of 8191 x 5000 bf16 took
// 65.3 us so, 67.4 without).
__device__ __forceinline__ uint32_t e4m3_largest(float (&x)[8]) {
  constexpr uint32_t INF = 0x7F800000u;
  uint32_t big = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) big = max(big, __float_as_uint(x[j]) & 0x7FFFFFFFu);
  if (__builtin_amdgcn_ballot_w64(big >= INF)) {
    big = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t u = __float_as_uint(x[j]) & 0x7FFFFFFFu;
      x[j] = u < INF ? x[j] : __builtin_nanf("");
      big = max(big, u < INF ? u : 0u);
    }
  }
  return big;
}

// The scale's biased exponent for a largest magnitude of these bits: m 2^e is
// within 448 = 1.75 2^8 times 2^(e - 8) where m is at most 1.75, which the sum
// carries past otherwise.
__device__ __forceinline__ uint32_t e4m3_exponent(uint32_t big) {
  const uint32_t e = (big + 0x1FFFFFu) >> 23;
  return e > 9u ? e - 8u : 1u;
}
__device__ __forceinline__ float e4m3_scale(uint32_t exponent) { return __uint_as_float(exponent << 23); }

// Four values, finite or NaN, to codes: x / scale to the nearest, halfway cases
// to the even code.
__device__ __forceinline__ uint32_t e4m3_codes(float x0, float x1, float x2, float x3, float scale) {
  e4m3_short2 w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x0, x1, scale, false);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x2, x3, scale, true);
  return __builtin_bit_cast(uint32_t, w);
}

// Four codes' values, over their scale.
__device__ __forceinline__ void e4m3_values(uint32_t w, float (&x)[4]) {
  const e4m3_float2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const e4m3_float2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
}

}  // namespace fk
