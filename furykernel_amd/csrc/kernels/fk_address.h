// fk_address.h — device addresses that a kernel's arguments carry as whole
// numbers, as pointers into global memory: the compiler then takes global
// loads and stores, where a plain pointer would be a flat one (which may mean
// LDS or scratch, and holds up both counters).
#pragma once

#include <stdint.h>

namespace fk {

template <typename T>
using global_ptr = T __attribute__((address_space(1))) *;

template <typename T>
__device__ __forceinline__ global_ptr<T> global_at(uint64_t address) {
  return (global_ptr<T>)address;
}

// A load of what a launch takes once, with ONCE: it leaves the caches to what
// is used again.
template <bool ONCE, typename T>
__device__ __forceinline__ T load_from(global_ptr<const T> p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(p);
  else return *p;
}

}  // namespace fk
