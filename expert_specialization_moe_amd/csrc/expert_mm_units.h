// How the experts' products divide an expert's rows, and a sum into steps.  Plain arithmetic that also compiles for the host.
//
// An expert may have up to 2^31 - 1 rows: what is rounded up passes 31 bits on the way and is formed without a sign.
#pragma once
#include <stdint.h>

#if defined(__HIP__)
#define ESMOE_MM_UNITS_HD __host__ __device__ __forceinline__
#else
#define ESMOE_MM_UNITS_HD inline
#endif

namespace esmoe {

// Steps of `each` that hold `length`.
ESMOE_MM_UNITS_HD int mm_steps(int length, int each) { return (int)(((uint32_t)length + (uint32_t)(each - 1)) / (uint32_t)each); }

// The rows of an expert in units of at most 256, as equal as sixteens allow: a tile of few rows takes as long as its weights' way from memory,
// a full one hardly longer (32 experts x 356 rows, 4096 x 7168: 256 and 100 rows 667 us, twice 178 650 us).
ESMOE_MM_UNITS_HD uint32_t mm_units(int rows) { return ((uint32_t)rows + 255) / 256; }
ESMOE_MM_UNITS_HD int mm_unit_rows(int rows) {
  const uint32_t units = mm_units(rows);
  return units ? (int)((((uint32_t)rows + units - 1) / units + 15) & ~15u) : 0;
}

}  // namespace esmoe
