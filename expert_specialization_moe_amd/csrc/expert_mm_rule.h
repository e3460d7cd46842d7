// Which kernel multiplies a call of the experts' products: the large one (expert_mm.hip) or that of few rows (expert_mm_few.hip).  By the call's
// sizes alone, since the rows of each expert stand in device memory.  Plain C++, so that tests can ask it, too.
#pragma once

namespace esmoe {

// kind: 0 forward, 1 forward with SwiGLU, 2 gradient of the rows, 3 gradient of the weights
struct MmTileCount {
  long col_tiles, units;   // of an output's columns; of rows (kind 3: of the weights' rows), at most
};
inline MmTileCount expert_mm_tiles(int kind, int num_experts, int total_rows, int n, int k) {
  const long cols = kind >= 2 ? k : kind == 1 ? n / 2 : n, wide = kind == 1 ? 128 : 256;
  return {(cols + wide - 1) / wide, kind == 3 ? (long)num_experts * ((n + 255) / 256) : total_rows / 256 + (num_experts < total_rows ? num_experts : total_rows)};
}

inline bool expert_mm_takes_few(int kind, int num_experts, int total_rows, int n, int k, int cus) {
  const MmTileCount t = expert_mm_tiles(kind, num_experts, total_rows, n, k);
  // Times are us there and here, bf16, the operands of three to six calls in turn (weights of more than 60 MB come from memory every time).
  // A kernel of its own (expert_mm_few.hip) for few rows: it reads the weights at the memory's rate whatever their number (4096 x 7168, 8 rows each of 8 /
  // 32 experts: 69 / 99, 267 / 274; 7168 x 2048, 256 rows of 30: 139 / 155), but again for every 32 rows (4096 x 7168, 512 / 1024 rows by Zipf over 32
  // experts: 323 / 283, 401 / 301), so up to eight an expert, which leaves popular ones room; or where there is not much to multiply and less than
  // two tiles a CU (8 x 32 rows 73 / 100, one x 1024 175 / 119, and on the line itself one x 512 86 / 112, 8 x 64 113 / 102; 2048 x 1024, 8 x 128 rows
  // 17 / 22, x 256 rows 31 / 25; 2304 x 4096, 512 rows by Zipf over 32 110 / 133).
  // The rows' gradient, whose weight rows it reads in pieces of 128 bytes: only that, and if tiles are not enough for the CUs (8 experts x 64
  // rows, 4096 x 2048: 45 / 62; one x 512 rows, 4096 x 4096: 43 / 70; 32 x 16 rows, 4096 x 2048, 256 tiles: 108 / 86).
  const long experts = num_experts < total_rows ? num_experts : total_rows;
  const bool small = total_rows * t.col_tiles <= 32 * cus && experts * t.col_tiles < (kind <= 1 ? 2 : 1) * cus;
  // The weights' gradient: where a tile for every second CU is all there is, or rows are few enough for the stores alone to count (8 experts x 50 rows, 720 x
  // 520: 5.8 / 8.6; one x 4096 rows, 1024 x 1024: 71 / 75; 3 x 500 rows, 2048 x 2048, 192 tiles: 31 / 24; 32 experts, 4096 x 2048, x 1 row 118 / 125,
  // x 16 rows 135 / 126, x 64 rows 185 / 143).  Neither kernel splits an expert's rows, so a long sum of few tiles leaves most CUs without work.
  return kind <= 1 ? small || total_rows <= 8 * experts : kind == 2 ? small : 2 * t.units * t.col_tiles <= cus || total_rows <= 16 * num_experts;
}

}  // namespace esmoe
