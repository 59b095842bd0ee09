// divide.cuh — division by a number that a launch knows: the host prepares it, the device multiplies.
#pragma once

#include <stdint.h>

namespace up {

// x / d for x below 2^31 by a multiplication (Granlund and Montgomery, "Division by invariant integers using
// multiplication", 1994): with 2^s >= d > 2^(s-1) and m = floor(2^32 (2^s - d) / d) + 1, x / d = (hi(m x) + x) >> s.
struct Divide32 {
  using Int = uint32_t;
  uint32_t d, m, s;
  explicit Divide32(int64_t by = 1) : d((uint32_t)by), s(0) {
    while (((uint64_t)1 << s) < d) ++s;
    m = (uint32_t)(((((uint64_t)1 << s) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return (__umulhi(x, m) + x) >> s; }
};
struct Divide64 {
  using Int = uint64_t;
  uint64_t d;
  explicit Divide64(int64_t by) : d((uint64_t)by) {}
  __device__ __forceinline__ uint64_t operator()(uint64_t x) const { return x / d; }
};

}  // namespace up
