// Grouped products of experts with few rows each (decode, small steps), 16 bits and int8: the sums of expert_mm.hip.
//
// Bound by the weights' way from memory.  An item is 16 to 64 columns (SwiGLU: half of them gate columns, half their up columns) of up to 16 or 32 rows of
// an expert, whose sum the four wavefronts of a workgroup split in steps of 128 bytes dealt in turn.  Weights and rows go from memory straight
// into LDS, rows of 128 bytes whole: loads into registers in the layout of the matrix instruction touch half of sixteen lines each, and few
// lines can be under way (8 experts x 32 rows, 4096 x 7168: 115 us so, 82 through LDS and the caches, 73 past the caches).  A wavefront has a ring
// of steps of its own, as many as LDS holds, whose copies run on across items; it waits for its own copies and reads, and no barrier stands in
// the way.  The four sums are added in LDS, in one order for any number of rows.  An expert's items of the same columns are neighbours on one XCD:
// their weights come from memory once.
// What lies beyond an expert's rows, the columns or the sum's length arrives as zeros without a load.
// One row of each of 8 experts, 4096 x 7168 with SwiGLU, bf16: 68 us (6.9 TB/s of weights), int8 36 us; 32 experts x 8 rows 267 us (7.0 TB/s).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "expert_mm.h"
#include "expert_mm_units.h"
#include "mxfp4_units.h"
#include "swiglu.h"
#include "wave_scan.h"

namespace esmoe {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));

enum { kFewForward = 0, kFewSwiglu = 1, kFewSwigluSave = 2, kFewRowsGrad = 3 };

constexpr int kFewWaves = 4, kFewThreads = 64 * kFewWaves;
constexpr int kFewNowhere = (int)0x80000000u;   // an offset beyond every descriptor

template <int TYPE> struct FewAcc { typedef v4f T; };
template <> struct FewAcc<kMmInt8> { typedef v4i T; };

template <int TYPE>
__device__ __forceinline__ typename FewAcc<TYPE>::T few_product(v4i w, v4i t, typename FewAcc<TYPE>::T c) {
  if constexpr (TYPE == kMmInt8) return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, t, c, 0, 0, 0);
  else if constexpr (TYPE == kMmFp16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, w), __builtin_bit_cast(v8h, t), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w), __builtin_bit_cast(v8bf, t), c, 0, 0, 0);
}

__device__ __forceinline__ int few_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ v4i few_descriptor(const void* p, int bytes) {
  return v4i{few_uniform((int)(uint64_t)p), few_uniform((int)((uint64_t)p >> 32)), few_uniform(bytes > 0 ? bytes : 0), 0x00020000};
}
// 64 x 16 bytes into LDS (a scalar register that a vector instruction wrote is there for a memory instruction five slots on).  STREAM: no cache is to keep it
template <bool STREAM>
__device__ __forceinline__ void few_copy(uint32_t lds, v4i rsrc, int at) {
  if constexpr (STREAM)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds" ::"s"(lds), "v"(at), "s"(rsrc) : "memory");
  else asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(at), "s"(rsrc) : "memory");
}
__device__ __forceinline__ v2i few_half4(v4f v, bool fp16) {
  return fp16 ? __builtin_bit_cast(v2i, __builtin_convertvector(v, v4h)) : __builtin_bit_cast(v2i, __builtin_convertvector(v, v4bf));
}

// The experts' rows, cut at the tensor's, in units of ROWS.
template <int ROWS>
struct FewTable {
  int rows[kMmExperts], off[kMmExperts];
  uint32_t unit_end[kMmExperts];   // running sums of units
  uint32_t units;

  __device__ __forceinline__ void build(const ExpertMmArgs& g) {
    const int lane = threadIdx.x;
    if (lane < 64) {
      uint32_t sum = 0;
      for (int e0 = 0; e0 < g.num_experts; e0 += 64) {
        const int e = e0 + lane, o = e < g.num_experts ? g.expert_offsets[e] : 0;
        const int m = e < g.num_experts ? fp4_rows(g.problem_sizes[e * 3], o, g.total_rows) : 0;
        const uint32_t end = sum_or_most(sum, wave_inclusive_sum_or_most(((uint32_t)m + ROWS - 1) / ROWS));
        if (e < g.num_experts) {
          rows[e] = m;
          off[e] = o;
          unit_end[e] = end;
        }
        sum = (uint32_t)__builtin_amdgcn_readlane((int)end, 63);
      }
      if (lane == 0) {   // no more than experts with rows of their own can have
        const uint32_t most = (uint32_t)(g.total_rows / ROWS) + (uint32_t)(g.num_experts < g.total_rows ? g.num_experts : g.total_rows);
        units = sum < most ? sum : most;
      }
    }
    __syncthreads();
  }
};

// Columns col0 .. + WIDE of up to ROWS rows of an expert; no rows where there is no such item.
struct FewItem {
  int expert, rows, col0;
  long row0;
};
template <int ROWS, int WIDE>
__device__ __forceinline__ FewItem few_item(const FewTable<ROWS>& s, const ExpertMmArgs& g, uint32_t p, uint32_t total, uint32_t col_items) {
  FewItem t = {g.num_experts - 1, 0, 0, 0};
  if (p >= total) return t;
  // the expert whose units' running sum is the first above this unit
  const uint32_t unit = p / col_items;
  const int lane = threadIdx.x & 63;
  uint32_t before = 0, behind = 0;
  for (int e0 = 0; e0 < g.num_experts; e0 += 64) {
    const uint32_t end = e0 + lane < g.num_experts ? s.unit_end[e0 + lane] : 0xffffffffu;
    const unsigned long long past = __ballot(end > unit);
    if (past) {
      const int l = __builtin_ctzll(past);
      if (e0 + l < g.num_experts) t.expert = e0 + l;
      if (l) before = (uint32_t)__builtin_amdgcn_readlane((int)end, l - 1);
      behind = (uint32_t)__builtin_amdgcn_readlane((int)end, l);
      break;
    }
    before = (uint32_t)__builtin_amdgcn_readlane((int)end, 63);
  }
  const uint32_t i = p - before * col_items, units = behind - before, col_item = i / units;
  const int from = (int)(i - col_item * units) * ROWS, left = few_uniform(s.rows[t.expert]) - from;
  t.rows = left < ROWS ? left : ROWS;
  t.row0 = (long)few_uniform(s.off[t.expert]) + from;
  t.col0 = (int)col_item * WIDE;
  return t;
}

template <int NT, int NC, int DEPTH>
struct FewShared {
  static constexpr int kWeights = NC * 2048, kStep = kWeights + NT * 2048;
  uint8_t ring[kFewWaves][DEPTH][kStep];   // a step: sixteen rows of 128 bytes a tile, the weights' tiles first
  v4f sums[kFewWaves][NT * NC][64];        // [row tile * NC + column tile][lane]
  FewTable<NT * 16> table;
};

// NT row tiles x NC column tiles of sixteen (SwiGLU: the second half of the latter are the up columns), the sum over four wavefronts, DEPTH steps of each in LDS.
template <int TYPE, int KIND, int NT, int NC, int DEPTH, bool STREAM>
__global__ void __launch_bounds__(kFewThreads) expert_mm_few_kernel(const ExpertMmArgs g) {
  typedef typename FewAcc<TYPE>::T Acc;
  typedef FewShared<NT, NC, DEPTH> Shared;
  typedef __attribute__((address_space(3))) char* Lds;
  constexpr bool kSw = KIND == kFewSwiglu || KIND == kFewSwigluSave, kGrad = KIND == kFewRowsGrad;
  constexpr int kTiles = kSw ? NC / 2 : NC, kWide = kTiles * 16, kRows = NT * 16, kSize = TYPE == kMmInt8 ? 1 : 2, kCopies = Shared::kStep / 1024;
  static_assert(sizeof(Shared) <= 160 * 1024, "LDS");
  static_assert(!kGrad || NC == 4, "a weight row of a step is 128 bytes");
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 63, wave = few_uniform(tid >> 6), l16 = lane & 15, gq = lane >> 4;
  s.table.build(g);
  const int cols = kSw ? g.n / 2 : kGrad ? g.k : g.n, pitch = (kGrad ? g.n : g.k) * kSize, w_pitch = g.k * kSize;
  const int rounds = (pitch + kFewWaves * 128 - 1) / (kFewWaves * 128);
  const uint32_t col_items = (cols + kWide - 1) / kWide, total = (uint32_t)few_uniform((int)s.table.units) * col_items;
  const MmPlace at = mm_place(total);
  const uint32_t ring = (uint32_t)few_uniform((int)(uint32_t)(uintptr_t)(Lds)(char*)s.ring[wave][0]);

  // A copy is eight rows of 128 bytes.  Rows along the sum: chunk x of row r in slot x ^ (r / 2 % 8), sixteen rows' reads of a chunk fall on different
  // banks.  Weight rows across it (the gradient): pairs of chunks change places by the row's bits 1 and 3, which does the same for the transposing read.
  const int row8 = lane >> 3;
  int chunk[2], w_chunk[2];   // bytes along a row, of even and odd copies
#pragma unroll
  for (int q = 0; q < 2; q++) {
    const int row = q * 8 + row8, x = lane & 7;
    chunk[q] = (x ^ (row >> 1 & 7)) * 16;
    w_chunk[q] = kGrad ? ((x >> 1 ^ ((row >> 1 & 1) | (row >> 3 & 1) << 1)) << 1 | (x & 1)) * 16 : chunk[q];
  }
  // The copies' item and round, ahead of the products'.
  uint32_t copy_p = at.place;
  int copy_round = 0;
  FewItem item = few_item<kRows, kWide>(s.table, g, copy_p, total, col_items);
  auto copy = [&](uint32_t slot) {
    const int step = copy_round * kFewWaves + wave, along = step * 128;
    if constexpr (kGrad) {
      const char* w = (const char*)g.w + ((long)item.expert * g.n + step * 64) * w_pitch + item.col0 * 2;
      const int have = g.n - step * 64 < 64 ? g.n - step * 64 : 64;
      const v4i wd = few_descriptor(w, item.rows && have > 0 ? have * w_pitch - item.col0 * 2 : 0);
#pragma unroll
      for (int q = 0; q < NC * 2; q++) few_copy<STREAM>(few_uniform(ring + slot + q * 1024), wd, w_chunk[q & 1] + (q * 8 + row8) * w_pitch);
    } else {
      const char* w = (const char*)g.w + ((long)item.expert * g.n + item.col0) * w_pitch;
      const int have = cols - item.col0 < kWide ? cols - item.col0 : kWide, len = item.rows ? have * w_pitch : 0;
#pragma unroll
      for (int h = 0; h < (kSw ? 2 : 1); h++) {
        const v4i wd = few_descriptor(w + h * (long)cols * w_pitch, len);
#pragma unroll
        for (int q = 0; q < kTiles * 2; q++) {
          const int x = w_chunk[q & 1] + along;
          few_copy<STREAM>(few_uniform(ring + slot + (h * kTiles * 2 + q) * 1024), wd, x < pitch ? (q * 8 + row8) * w_pitch + x : kFewNowhere);
        }
      }
    }
    const v4i td = few_descriptor((const char*)g.t + item.row0 * pitch, item.rows * pitch);
#pragma unroll
    for (int q = 0; q < NT * 2; q++) {
      const int x = chunk[q & 1] + along;
      few_copy<false>(few_uniform(ring + slot + Shared::kWeights + q * 1024), td, x < pitch ? (q * 8 + row8) * pitch + x : kFewNowhere);
    }
    if (++copy_round == rounds) {
      copy_round = 0;
      copy_p = copy_p < total ? copy_p + at.of : copy_p;
      item = few_item<kRows, kWide>(s.table, g, copy_p, total, col_items);
    }
  };
#pragma unroll
  for (int d = 0; d < DEPTH; d++) copy(d * Shared::kStep);
  uint32_t slot = 0;
  for (uint32_t p = at.place; p < total; p += at.of) {
    const FewItem t = few_item<kRows, kWide>(s.table, g, p, total, col_items);
    Acc c[NT][NC];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
      for (int j = 0; j < NC; j++) c[i][j] = Acc{0, 0, 0, 0};
    for (int r = 0; r < rounds; r++) {
      // (a wavefront reads, and copies into again, what is its own: it waits for its own copies and reads)
      asm volatile("s_waitcnt vmcnt(%0) ; explicit" ::"n"((DEPTH - 1) * kCopies) : "memory");
      v4i tf[NT][2], wf[NC][2];
      const Lds step = (Lds)(uintptr_t)(ring + slot);
      auto along = [&](int row, int ks) { return *(const __attribute__((address_space(3))) v4i*)(step + row * 128 + ((gq + ks * 4) ^ (l16 >> 1)) * 16); };
#pragma unroll
      for (int ks = 0; ks < 2; ks++) {
#pragma unroll
        for (int i = 0; i < NT; i++) tf[i][ks] = along(NC * 16 + i * 16 + l16, ks);
#pragma unroll
        for (int j = 0; j < NC; j++) {
          if constexpr (kGrad) {
            // four lanes read 16 columns of a row, sixteen lanes of four rows, and the hardware hands lane i column i
            typedef __attribute__((address_space(3))) v4s* Lds4;
            const int row = ks * 32 + gq * 8 + (l16 >> 2), f = (row >> 1 & 1) | (row >> 3 & 1) << 1;
            const Lds from = step + row * 128 + (j ^ f) * 32 + (l16 & 3) * 8;   // (row + 4: of the same bits 1 and 3)
            const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)from)),
                      hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)(from + 4 * 128)));
            wf[j][ks] = v4i{lo[0], lo[1], hi[0], hi[1]};
          } else wf[j][ks] = along(j * 16 + l16, ks);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      copy(slot);
      slot = slot == (DEPTH - 1) * Shared::kStep ? 0 : slot + Shared::kStep;
#pragma unroll
      for (int ks = 0; ks < 2; ks++)
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
          for (int j = 0; j < NC; j++) c[i][j] = few_product<TYPE>(wf[j][ks], tf[i][ks], c[i][j]);
    }

    __syncthreads();   // (the sums of the item before have been read)
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
      for (int j = 0; j < NC; j++) s.sums[wave][i * NC + j][lane] = __builtin_bit_cast(v4f, c[i][j]);
    __syncthreads();
    // Outputs: a unit is a tile's lane: row l % 16, columns 4 (l / 16) .. + 4.
    constexpr int kUnits = NT * kTiles;
    const bool fp16 = TYPE == kMmFp16 || (TYPE == kMmInt8 && g.out_fp16);
    auto put = [&](void* out, int width, v2i v, int row, int col) { *(v2i*)((char*)out + ((t.row0 + row) * width + col) * 2) = v; };
#pragma unroll
    for (int u = 0; u < (kUnits + kFewWaves - 1) / kFewWaves; u++) {
      const int tile = wave + u * kFewWaves, row = tile / kTiles * 16 + l16, col = t.col0 + tile % kTiles * 16 + gq * 4;
      if (kUnits % kFewWaves && tile >= kUnits) break;
      if (row >= t.rows || col >= cols) continue;
      v4f sum[kSw ? 2 : 1];
#pragma unroll
      for (int h = 0; h < (kSw ? 2 : 1); h++) {
        const int part = tile / kTiles * NC + h * kTiles + tile % kTiles;
        Acc all = __builtin_bit_cast(Acc, s.sums[0][part][lane]);
#pragma unroll
        for (int w = 1; w < kFewWaves; w++) all += __builtin_bit_cast(Acc, s.sums[w][part][lane]);
        if constexpr (TYPE == kMmInt8) {
          const float sa = g.sa[t.row0 + row];
          const v4f sb = *(const v4f*)(g.sb + (long)t.expert * g.n + h * cols + col);
#pragma unroll
          for (int x = 0; x < 4; x++) sum[h][x] = (float)all[x] * sa * sb[x];
        } else sum[h] = all;
      }
      if constexpr (kSw) {
        v4f y;
#pragma unroll
        for (int x = 0; x < 4; x++) y[x] = swiglu_f32(sum[0][x], sum[1][x]);
        put(g.out, cols, few_half4(y, fp16), row, col);
        if constexpr (KIND == kFewSwigluSave) {
          put(g.gate_up, g.n, few_half4(sum[0], fp16), row, col);
          put(g.gate_up, g.n, few_half4(sum[1], fp16), row, cols + col);
        }
      } else put(g.out, cols, few_half4(sum[0], fp16), row, col);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (nothing may arrive in LDS that is another workgroup's by then)
}

// The weights' gradient where there are few tiles for the large kernel, or next to no rows: out[j, c] = sum_m t[m, j] w[m, c] over an expert's rows.  Bound by the
// stores.  A wavefront has 64 x 64 outputs and a ring of its own, two steps of 32 rows of 64 columns of either operand, as above; both are read
// transposed.  An expert without rows gets zeros.
constexpr int kOuterRows = 32, kOuterStep = 2 * kOuterRows * 128, kOuterCopies = kOuterStep / 1024, kOuterStores = 8;
struct FewOuterShared {
  uint8_t ring[kFewWaves][2][kOuterStep];
  FewTable<kOuterRows> table;
};

// Odd groups of sixteen lanes give their part of x for the even neighbour's of y: eight columns a lane of one of two tiles instead of four of both.
__device__ __forceinline__ v4i few_pair(v2i x, v2i y) {
  const auto lo = __builtin_amdgcn_permlane16_swap(x[0], y[0], false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(x[1], y[1], false, false);
  return v4i{(int)lo[0], (int)hi[0], (int)lo[1], (int)hi[1]};
}

template <int TYPE>
__global__ void __launch_bounds__(kFewThreads) expert_mm_few_outer_kernel(const ExpertMmArgs g) {
  typedef __attribute__((address_space(3))) char* Lds;
  typedef __attribute__((address_space(3))) v4s* Lds4;
  __shared__ FewOuterShared s;
  const int tid = threadIdx.x, lane = tid & 63, wave = few_uniform(tid >> 6), l16 = lane & 15, gq = lane >> 4;
  s.table.build(g);
  const int pitch = g.n * 2, w_pitch = g.k * 2;
  const uint32_t col_tiles = (g.k + 63) / 64, tiles = (uint32_t)((g.n + 63) / 64) * col_tiles, total = (uint32_t)g.num_experts * tiles;
  const MmPlace at = mm_place((total + kFewWaves - 1) / kFewWaves);
  const uint32_t ring = (uint32_t)few_uniform((int)(uint32_t)(uintptr_t)(Lds)(char*)s.ring[wave][0]);
  const int row8 = lane >> 3, x = lane & 7;
  int chunk[2];
#pragma unroll
  for (int q = 0; q < 2; q++) chunk[q] = ((x >> 1 ^ ((row8 >> 1 & 1) | q << 1)) << 1 | (x & 1)) * 16;

  // The copies' item (of those with rows) and step, ahead of the products'.
  const uint32_t first = at.place * kFewWaves + wave, stride = at.of * kFewWaves;
  uint32_t copy_p = first;
  int copy_step = 0, copy_rows = 0;   // (counted in steps: one behind the last row may pass 31 bits)
  auto find = [&] {   // from copy_p on
    while (copy_p < total && (copy_rows = few_uniform(s.table.rows[copy_p / tiles])) == 0) copy_p += stride;
  };
  auto copy = [&](uint32_t slot) {
    const bool any = copy_p < total;
    const uint32_t expert = any ? copy_p / tiles : 0, i = any ? copy_p - expert * tiles : 0, row = i / col_tiles, col = i - row * col_tiles;
    const int m0 = copy_step * kOuterRows, have = !any ? 0 : copy_rows - m0 < kOuterRows ? copy_rows - m0 : kOuterRows;
    const long from = (long)few_uniform(s.table.off[expert]) + m0;
    const v4i td = few_descriptor((const char*)g.t + from * pitch + row * 128, have * pitch - (int)row * 128),
              wd = few_descriptor((const char*)g.w + from * w_pitch + col * 128, have * w_pitch - (int)col * 128);
#pragma unroll
    for (int q = 0; q < 4; q++) few_copy<false>(few_uniform(ring + slot + q * 1024), td, chunk[q & 1] + (q * 8 + row8) * pitch);
#pragma unroll
    for (int q = 0; q < 4; q++) few_copy<false>(few_uniform(ring + slot + kOuterStep / 2 + q * 1024), wd, chunk[q & 1] + (q * 8 + row8) * w_pitch);
    if (any && ++copy_step == mm_steps(copy_rows, kOuterRows)) {
      copy_step = 0;
      copy_p += stride;
      find();
    }
  };
  find();
  copy(0);
  copy(kOuterStep);
  uint32_t slot = 0;
  int stored = 0;   // an item's stores are younger than the copies that this step waits for
  for (uint32_t p = first; p < total; p += stride) {
    const uint32_t expert = p / tiles, i0 = p - expert * tiles, tile = i0 / col_tiles;
    const int row0 = (int)tile * 64, col0 = (int)(i0 - tile * col_tiles) * 64, rows = few_uniform(s.table.rows[expert]);
    v4f c[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) c[i][j] = v4f{0, 0, 0, 0};
    for (int left = mm_steps(rows, kOuterRows); left > 0; left--) {
      asm volatile("s_cmp_lg_u32 %2, 0\n\ts_cbranch_scc1 .Lesmoe_wait%=\n\ts_waitcnt vmcnt(%0) ; explicit\n.Lesmoe_wait%=:\n\ts_waitcnt vmcnt(%1) ; explicit"
                   ::"n"(kOuterCopies), "n"(kOuterCopies + kOuterStores), "s"(few_uniform(stored)) : "memory", "scc");
      const Lds step = (Lds)(uintptr_t)(ring + slot);
      // four lanes read 16 columns of a row, sixteen lanes of four rows, and the hardware hands lane i column i
      auto read = [&](int part, int i) {
        const int row = gq * 8 + (l16 >> 2), f = (row >> 1 & 1) | (row >> 3 & 1) << 1;
        const Lds from = step + part + row * 128 + (i ^ f) * 32 + (l16 & 3) * 8;   // (row + 4: of the same bits 1 and 3)
        const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)from)),
                  hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)(from + 4 * 128)));
        return v4i{lo[0], lo[1], hi[0], hi[1]};
      };
      v4i tf[4], wf[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        tf[i] = read(0, i);
        wf[i] = read(kOuterStep / 2, i);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) c[i][j] = few_product<TYPE>(wf[j], tf[i], c[i][j]);
      if (left > 1) {
        copy(slot);
        slot ^= kOuterStep;
        stored = 0;
      }
    }
    // A lane has row i * 16 + l % 16, after the exchange eight columns of one of two tiles: stored in front of the copies into the last step's place.
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((char*)g.out + (((long)expert * g.n + row0) * g.k + col0) * 2, 0,
                                                        (g.n - row0 < 64 ? g.n - row0 : 64) * w_pitch - col0 * 2, 0x00020000);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const int col = j * 16 + (gq & 1) * 16 + (gq >> 1) * 8;
        __builtin_amdgcn_raw_buffer_store_b128(few_pair(few_half4(c[i][j], TYPE == kMmFp16), few_half4(c[i][j + 1], TYPE == kMmFp16)), rsrc,
                                               col0 + col < g.k ? (i * 16 + l16) * w_pitch + col * 2 : kFewNowhere, 0, 0);
      }
    __builtin_amdgcn_sched_barrier(0);
    if (rows > 0) {
      copy(slot);
      slot ^= kOuterStep;
      stored = 1;
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (nothing may arrive in LDS that is another workgroup's by then)
}

template <int TYPE, int KIND, int NT, int NC, int DEPTH>
int few_launch(const ExpertMmArgs& g, int cus, bool stream_weights, hipStream_t stream) {
  const long experts = g.num_experts < g.total_rows ? g.num_experts : g.total_rows;
  const int cols = KIND == kFewRowsGrad ? g.k : KIND == kFewForward ? g.n : g.n / 2, wide = KIND == kFewSwiglu || KIND == kFewSwigluSave ? NC * 8 : NC * 16;
  const long items = (g.total_rows / (16 * NT) + experts) * ((cols + wide - 1) / wide);
  const long most = (160 * 1024 / sizeof(FewShared<NT, NC, DEPTH>)) * (long)cus, grid = items < most ? items : most;
  if (grid == 0) return 0;
  if (stream_weights) hipLaunchKernelGGL((expert_mm_few_kernel<TYPE, KIND, NT, NC, DEPTH, true>), dim3((unsigned)grid), dim3(kFewThreads), 0, stream, g);
  else hipLaunchKernelGGL((expert_mm_few_kernel<TYPE, KIND, NT, NC, DEPTH, false>), dim3((unsigned)grid), dim3(kFewThreads), 0, stream, g);
  return (int)hipGetLastError();
}

}  // namespace esmoe

using namespace esmoe;

// kind: 0 forward, 1 forward with SwiGLU, 2 gradient of the rows, 3 of the weights
extern "C" int esmoe_launch_expert_mm_few(const ExpertMmArgs* args, int kind, int cus, hipStream_t stream) {
  const ExpertMmArgs& g = *args;
  if (kind == 3) {
    const long items = ((long)g.num_experts * ((g.n + 63) / 64) * ((g.k + 63) / 64) + kFewWaves - 1) / kFewWaves, grid = items < 2 * cus ? items : 2 * cus;
    if (g.type == kMmBf16) hipLaunchKernelGGL((expert_mm_few_outer_kernel<kMmBf16>), dim3((unsigned)grid), dim3(kFewThreads), 0, stream, g);
    else hipLaunchKernelGGL((expert_mm_few_outer_kernel<kMmFp16>), dim3((unsigned)grid), dim3(kFewThreads), 0, stream, g);
    return (int)hipGetLastError();
  }
  const long cols = kind == 1 ? g.n / 2 : g.n, experts = g.num_experts < g.total_rows ? g.num_experts : g.total_rows;
  // Half as wide an item where rows are few, or to leave no CU without (us, 32 and 64 columns, 4096 x 7168: 2 experts x 16 rows 23 / 30, 8 x 16 rows 72 / 70;
  // 8 x 32 rows 86 / 73, one x 256 rows 61 / 46: the rows come from L2 once for each item).
  const long units = experts > g.total_rows / 32 ? experts : g.total_rows / 32, wide = kind == 1 ? 16 : 32;   // of 32 rows, if they are spread evenly
  const bool narrow = units * ((cols + wide - 1) / wide) <= cus || g.total_rows <= 16 * experts;
  // Rows of whole lines, of more weights than the caches hold, read once but for popular experts: past the caches (us so and through them: 32 experts x 8 rows,
  // 4096 x 7168 267 / 298, 8 x 32 rows 74 / 82; but read twice or more, 4 experts x 128 rows, 108 / 95, and lines in two pieces, k = 7176, 373 / 339).
  const bool once = expert_mm_whole_lines(g) && g.total_rows <= 32 * experts;
  auto launch = [&](auto type, auto k) {
    constexpr int TYPE = decltype(type)::value, KIND = decltype(k)::value;
    if constexpr (KIND == kFewRowsGrad) {
      if (g.total_rows <= 16) return few_launch<TYPE, KIND, 1, 4, 3>(g, cus, once, stream);
    } else {
      if (g.total_rows <= 16) return few_launch<TYPE, KIND, 1, 2, 4>(g, cus, once, stream);
      if (narrow) return few_launch<TYPE, KIND, 2, 2, 3>(g, cus, once, stream);
    }
    return few_launch<TYPE, KIND, 2, 4, 2>(g, cus, once, stream);
  };
  constexpr std::integral_constant<int, kFewForward> forward;
  constexpr std::integral_constant<int, kFewSwiglu> swiglu;
  constexpr std::integral_constant<int, kFewSwigluSave> save;
  constexpr std::integral_constant<int, kFewRowsGrad> grad;
  auto launch16 = [&](auto type) {
    return kind == 2 ? launch(type, grad) : kind == 0 ? launch(type, forward) : g.gate_up ? launch(type, save) : launch(type, swiglu);
  };
  if (g.type == kMmBf16) return launch16(std::integral_constant<int, kMmBf16>());
  if (g.type == kMmFp16) return launch16(std::integral_constant<int, kMmFp16>());
  constexpr std::integral_constant<int, kMmInt8> int8;
  return kind == 0 ? launch(int8, forward) : launch(int8, swiglu);
}
