// fk_divisor.h — quotients by a whole number that a launch knows: a product's
// high half, a difference and shifts (Granlund and Montgomery, Division by
// Invariant Integers using Multiplication, 1994, figure 4.1), exact for all 32
// bits, in place of the reciprocal and its corrections that a division takes.
#pragma once

#include <stdint.h>

namespace fk {

struct Divisor {
  uint32_t by, mul, shift1, shift2;
};

inline Divisor divisor(uint32_t by) {
  uint32_t l = 0;
  while (l < 32 && 1ull << l < by) l++;
  return {by, (uint32_t)((((1ull << l) - by) << 32) / by + 1), l < 1 ? l : 1u, l < 1 ? 0u : l - 1};
}

__host__ __device__ __forceinline__ uint32_t quotient(uint32_t x, const Divisor &d) {
  const uint32_t t = (uint32_t)((uint64_t)x * d.mul >> 32);
  return (t + ((x - t) >> d.shift1)) >> d.shift2;
}

}  // namespace fk
