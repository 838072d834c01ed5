// dropout_mask.cuh — the library's counter-based dropout mask.
//
// Element e is kept when the (e mod 4)-th 16-bit slice of splitmix64 of (seed,
// e / 4) is >= p * 65536 (splitmix64: Steele, Lea and Flood, "Fast splittable
// pseudorandom number generators", OOPSLA 2014).  The mask is a function of the
// seed and the element's index alone, so the backward makes it again instead of
// reading it.
#pragma once

#include <cstdint>

namespace fp8b {

__device__ __forceinline__ uint64_t splitmix64(uint64_t z) {
  z += 0x9E3779B97F4A7C15ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}

// Keep mask bits for the 8 elements starting at linear index e0 (e0 % 8 == 0).
__device__ __forceinline__ uint32_t dropout_keep8(uint64_t seed, int64_t e0, uint32_t thresh16) {
  uint32_t keep = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint64_t r = splitmix64(seed ^ (static_cast<uint64_t>(e0 / 4 + h) * 0xD1B54A32D192ED03ull));
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (static_cast<uint32_t>((r >> (16 * k)) & 0xFFFFu) >= thresh16) keep |= 1u << (h * 4 + k);
  }
  return keep;
}

}  // namespace fp8b
