// The 8-bit format of the paged cache: e4m3 codes (OCP: 448 the largest, no
// infinities, 0x7f and 0xff NaN) and the power-of-two scale of a block of them.
// A power of two, because then a code times its scale is exact, and raising a
// block's scale leaves its codes exact too, but for those that end below e4m3's
// smallest normal 2^-6.  (Compiles for the host too, where it is tested.)
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define LC_BOTH __host__ __device__ __forceinline__
#else
#define LC_BOTH inline
#endif

namespace lc {

constexpr uint32_t kScaleMin = 1u << 23;  // bits of 2^-126: the scale of zeros

// Bits of the smallest power of two s >= 2^-126 with amax <= 448 s, from the bits
// of amax >= 0, finite.  448 = 1.75 2^8.
LC_BOTH uint32_t scale_bits(uint32_t amax) {
  const uint32_t e = (amax >> 23) + ((amax & 0x7fffffu) > 0x600000u ? 1u : 0u);
  return e > 9u ? (e - 8u) << 23 : kScaleMin;
}

// Bits of 2^-n for a scale 2^n: exact from 2^-126 (0 would need 2^127 + ..) on.
// n <= 120, as a finite amax gives no larger scale.
LC_BOTH uint32_t inverse_bits(uint32_t scale) { return (254u << 23) - scale; }

// Bits of was / now for scales was <= now: 0 where that is below 2^-126, where
// nothing is left of a code either.
LC_BOTH uint32_t ratio_bits(uint32_t was, uint32_t now) {
  const uint32_t d = now - was;
  return d > (126u << 23) ? 0u : (127u << 23) - d;
}

// The row of the page table that a key is in, and its page; -1: none.
LC_BOTH int page_of(const int32_t* table, int width, int pages, int64_t at) {
  if (at < 0 || at >= width) return -1;
  const int id = table[at];
  return id >= 0 && id < pages ? id : -1;
}

}  // namespace lc
