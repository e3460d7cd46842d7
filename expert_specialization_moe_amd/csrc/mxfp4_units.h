// The units of a grouped product with 4-bit weights: experts in order, each in tiles of sixteen rows.  Plain arithmetic that also
// compiles for the host.
//
// The counts come from device memory and are not checked there, so they may say that many experts own the same rows: their tiles then
// add up to as much as 2^37.  All sums saturate (which is associative, so a prefix sum in any order of lanes gives the same) and a
// place in them is looked up by the sum before it, which is exact wherever a unit lies behind it: no unit leaves its expert's rows.
#pragma once
#include <stdint.h>

#if defined(__HIP__)
#define ESMOE_UNITS_HD __host__ __device__ __forceinline__
#else
#define ESMOE_UNITS_HD inline
#endif

namespace esmoe {

constexpr int kFp4Rows = 16;

struct Fp4Unit {
  int expert, row0, rows;   // rows 0: no such unit
};

// Rows of an expert that lie in the tensor; 0 where none does.
ESMOE_UNITS_HD int fp4_rows(int m, int off, int total_rows) {
  return off < 0 || off >= total_rows || m < 0 ? 0 : m > total_rows - off ? total_rows - off : m;
}

ESMOE_UNITS_HD uint32_t fp4_tiles(int rows) { return ((uint32_t)rows + (kFp4Rows - 1)) / kFp4Rows; }

ESMOE_UNITS_HD uint32_t sum_or_most(uint32_t a, uint32_t b) { return a + b < a ? 0xffffffffu : a + b; }

// Unit u (counted like `start`, the units before this expert's) of an expert with `rows` rows from `off` on.
ESMOE_UNITS_HD Fp4Unit fp4_unit(int expert, int off, int rows, uint32_t u, uint32_t start) {
  const int tile = (int)(u - start), left = rows - tile * kFp4Rows;
  return {expert, off + tile * kFp4Rows, left < kFp4Rows ? left : kFp4Rows};
}

// Units of a call whose experts own rows of their own, at most: one per expert with rows and one more per full tile.
ESMOE_UNITS_HD long fp4_most_units(int num_experts, int total_rows) {
  return (long)(num_experts < total_rows ? num_experts : total_rows) + total_rows / kFp4Rows;
}

}  // namespace esmoe
