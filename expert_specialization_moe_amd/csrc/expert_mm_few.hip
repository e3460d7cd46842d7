// Grouped products of experts with few rows each (decode), 16 bits and int8: the sums of expert_mm.hip's forward forms.
//
// Bound by the weights' way from memory, and nothing is reused that would pay for LDS: an item is 16, 32 or 64 columns (SwiGLU: half of them gate
// columns, half their up columns) of up to 16 or 32 rows of an expert, whose sum the four wavefronts of a workgroup split in steps of 128 bytes dealt
// in turn.  Each loads weights and rows in the layout of the matrix instruction, several steps ahead in registers, across items; the four
// sums are added in LDS, in one order.  An expert's items of the same columns are neighbours on one XCD: their weights come from memory once.
// What lies beyond an expert's rows, the columns or the sum's length arrives as zeros without a load.
// One row of each of 8 experts, 4096 x 7168 with SwiGLU, bf16: 79 us (5.9 TB/s of weights), int8 43 us.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "expert_mm.h"
#include "mxfp4_units.h"
#include "swiglu.h"
#include "wave_scan.h"

namespace esmoe {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));

enum { kFewForward = 0, kFewSwiglu = 1, kFewSwigluSave = 2 };

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
__device__ __forceinline__ __amdgpu_buffer_rsrc_t few_buffer(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes > 0 ? bytes : 0, 0x00020000);
}
__device__ __forceinline__ v4i few_load(__amdgpu_buffer_rsrc_t rsrc, int at) {
  return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0));
}
__device__ __forceinline__ v2i few_half4(v4f v, bool fp16) {
  return fp16 ? __builtin_bit_cast(v2i, __builtin_convertvector(v, v4h)) : __builtin_bit_cast(v2i, __builtin_convertvector(v, v4bf));
}

template <int NT, int NC>
struct FewShared {
  v4f sums[kFewWaves][NT * NC][64];   // [row tile * NC + column tile][lane]
  int rows[kMmExperts], off[kMmExperts];
  uint32_t unit_end[kMmExperts];   // running sums of the experts' units of NT * 16 rows
  uint32_t units;
};

struct FewItem {
  __amdgpu_buffer_rsrc_t t, w0, w1;
  int expert, rows, col0;
  long row0;
};

// NT row tiles x NC column tiles of sixteen; SwiGLU: the second half of the latter are the up columns.
template <int TYPE, int KIND, int NT, int NC, int AHEAD>
__global__ void __launch_bounds__(kFewThreads, 2) expert_mm_few_kernel(const ExpertMmArgs g) {
  typedef typename FewAcc<TYPE>::T Acc;
  constexpr bool kSw = KIND != kFewForward;
  constexpr int kTiles = kSw ? NC / 2 : NC, kWide = kTiles * 16, kRows = NT * 16, kSize = TYPE == kMmInt8 ? 1 : 2;
  __shared__ FewShared<NT, NC> s;
  const int tid = threadIdx.x, lane = tid & 63, wave = few_uniform(tid >> 6);
  if (wave == 0) {
    uint32_t units = 0;
    for (int e0 = 0; e0 < g.num_experts; e0 += 64) {
      const int e = e0 + lane, off = e < g.num_experts ? g.expert_offsets[e] : 0;
      const int rows = e < g.num_experts ? fp4_rows(g.problem_sizes[e * 3], off, g.total_rows) : 0;
      const uint32_t end = sum_or_most(units, wave_inclusive_sum_or_most(((uint32_t)rows + kRows - 1) / kRows));
      if (e < g.num_experts) {
        s.rows[e] = rows;
        s.off[e] = off;
        s.unit_end[e] = end;
      }
      units = (uint32_t)__builtin_amdgcn_readlane((int)end, 63);
    }
    if (lane == 0) {   // no more than experts with rows of their own can have
      const uint32_t most = (uint32_t)(g.total_rows / kRows) + (uint32_t)(g.num_experts < g.total_rows ? g.num_experts : g.total_rows);
      s.units = units < most ? units : most;
    }
  }
  __syncthreads();
  const int cols = kSw ? g.n / 2 : g.n, pitch = g.k * kSize;
  const uint32_t col_items = (cols + kWide - 1) / kWide, total = (uint32_t)few_uniform((int)s.units) * col_items;

  auto item = [&](uint32_t p) {
    FewItem t;
    t.expert = g.num_experts - 1;
    t.rows = t.col0 = 0;
    t.row0 = 0;
    if (p < total) {
      // the expert whose units' running sum is the first above this unit
      const uint32_t unit = p / col_items;
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
      const int from = (int)(i - col_item * units) * kRows, left = few_uniform(s.rows[t.expert]) - from;
      t.rows = left < kRows ? left : kRows;
      t.row0 = (long)few_uniform(s.off[t.expert]) + from;
      t.col0 = (int)col_item * kWide;
    }
    const long w_row = (long)t.expert * g.n + t.col0;
    const int wide = cols - t.col0 < kWide ? cols - t.col0 : kWide, w_len = t.rows ? wide * pitch : 0;
    t.t = few_buffer((const char*)g.t + t.row0 * pitch, t.rows * pitch);
    t.w0 = few_buffer((const char*)g.w + w_row * pitch, w_len);
    t.w1 = few_buffer((const char*)g.w + (w_row + (kSw ? cols : 0)) * pitch, w_len);
    return t;
  };

  // A wavefront's steps, AHEAD of them on their way: lane l has 16 bytes along the sum of row (column) l % 16 at 16 * (l / 16), in each half of a
  // step.  An item's last steps are followed by the first ones of the next item.
  const int rounds = (pitch + kFewWaves * 128 - 1) / (kFewWaves * 128), row_at = (lane & 15) * pitch, along = wave * 128 + (lane >> 4) * 16;
  v4i tf[AHEAD][NT][2], wf[AHEAD][NC][2];
  Acc c[NT][NC];
  auto load = [&](const FewItem& t, int step, int d) {
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      const int k = step * (kFewWaves * 128) + along + ks * 64, at = k < pitch ? row_at + k : kFewNowhere;
#pragma unroll
      for (int j = 0; j < NC; j++) wf[d][j][ks] = few_load(kSw && j >= kTiles ? t.w1 : t.w0, at + j % kTiles * 16 * pitch);
#pragma unroll
      for (int i = 0; i < NT; i++) tf[d][i][ks] = few_load(t.t, at + i * 16 * pitch);
    }
    __builtin_amdgcn_sched_barrier(0);   // (steps stay in their order: the compiler would put all loads together and wait for them together)
  };
  auto multiply = [&](int d) {
#pragma unroll
    for (int ks = 0; ks < 2; ks++)
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < NC; j++) c[i][j] = few_product<TYPE>(wf[d][j][ks], tf[d][i][ks], c[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  };

  const MmPlace at = mm_place(total);
  uint32_t p = at.place;
  FewItem next = item(p);
#pragma unroll
  for (int d = 0; d < AHEAD; d++) load(next, d, d);
  for (; p < total; p += at.of) {
    const FewItem t = next;
    next = item(p + at.of);
    // Outputs: a unit is a tile's lane: row l % 16, columns 4 (l / 16) .. + 4.
    constexpr int kUnits = NT * kTiles * 64, kEach = (kUnits + kFewThreads - 1) / kFewThreads;
    // int8: scales, asked for ahead of the sums
    float sa[kEach];
    v4f sb[kEach][kSw ? 2 : 1];
    if constexpr (TYPE == kMmInt8) {
      const auto of_rows = few_buffer(g.sa + t.row0, t.rows * 4), of_cols = few_buffer(g.sb + (long)t.expert * g.n, g.n * 4);
#pragma unroll
      for (int u = 0; u < kEach; u++) {
        const int tile = (tid + u * kFewThreads) >> 6, row = tile / kTiles * 16 + (lane & 15), col = tile % kTiles * 16 + (lane >> 4) * 4;
        sa[u] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(of_rows, row * 4, 0, 0));
#pragma unroll
        for (int h = 0; h < (kSw ? 2 : 1); h++) sb[u][h] = __builtin_bit_cast(v4f, few_load(of_cols, (h * cols + t.col0 + col) * 4));
      }
    }

#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
      for (int j = 0; j < NC; j++) c[i][j] = Acc{0, 0, 0, 0};
    // (an item's steps are a multiple of AHEAD, the last ones of nothing: conditions among them would make the compiler move what is under way)
    for (int r = AHEAD; r < rounds; r += AHEAD) {
#pragma unroll
      for (int d = 0; d < AHEAD; d++) {
        multiply(d);
        load(t, r + d, d);
      }
    }
#pragma unroll
    for (int d = 0; d < AHEAD; d++) {
      multiply(d);
      load(next, d, d);
    }

    __syncthreads();   // (the sums of the item before have been read)
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
      for (int j = 0; j < NC; j++) s.sums[wave][i * NC + j][lane] = __builtin_bit_cast(v4f, c[i][j]);
    __syncthreads();
    const bool fp16 = TYPE == kMmFp16 || (TYPE == kMmInt8 && g.out_fp16);
    auto put = [&](void* out, int width, v2i v, int row, int col) { *(v2i*)((char*)out + ((t.row0 + row) * width + col) * 2) = v; };
#pragma unroll
    for (int u = 0; u < kEach; u++) {
      const int tile = (tid + u * kFewThreads) >> 6;
      if (kUnits % kFewThreads && tile * 64 >= kUnits) break;
      const int row = tile / kTiles * 16 + (lane & 15), col = t.col0 + tile % kTiles * 16 + (lane >> 4) * 4;
      v4f sum[kSw ? 2 : 1];
#pragma unroll
      for (int h = 0; h < (kSw ? 2 : 1); h++) {
        const int at = tile / kTiles * NC + h * kTiles + tile % kTiles;
        Acc all = __builtin_bit_cast(Acc, s.sums[0][at][lane]);
#pragma unroll
        for (int w = 1; w < kFewWaves; w++) all += __builtin_bit_cast(Acc, s.sums[w][at][lane]);
#pragma unroll
        for (int x = 0; x < 4; x++) sum[h][x] = TYPE == kMmInt8 ? (float)all[x] * sa[u] * sb[u][h][x] : (float)all[x];
      }
      if (row >= t.rows || col >= cols) continue;
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
}

}  // namespace esmoe

using namespace esmoe;

extern "C" int esmoe_launch_expert_mm_few(const ExpertMmArgs* args, int kind, int cus, hipStream_t stream) {
  const ExpertMmArgs& g = *args;
  const long cols = kind == 1 ? g.n / 2 : g.n, experts = g.num_experts < g.total_rows ? g.num_experts : g.total_rows;
  const int row_tiles = g.total_rows <= 16 ? 1 : 2;
  auto col_items = [&](int col_tiles) {
    const int wide = col_tiles * 16 / (kind == 1 ? 2 : 1);
    return (cols + wide - 1) / wide;
  };
  // As wide an item as leaves one for every CU: the rows come from L2 once for each (us, wide and narrow, 4096 x 7168: 4 experts x 16 rows 53 / 60, one
  // x 256 rows 77 / 101; with half as many items as CUs, 2 x 16 rows 47 / 32).  16 rows at most are little beside 32 columns.
  const long least = experts > g.total_rows / 32 ? experts : g.total_rows / 32;   // units, if rows are spread evenly
  const int col_tiles = row_tiles == 1 ? (kind == 0 && experts * col_items(2) < cus ? 1 : 2) : least * col_items(4) < cus ? 2 : 4;
  const long items = (g.total_rows / (16 * row_tiles) + experts) * col_items(col_tiles), grid = items < 2 * cus ? items : 2 * cus;
  if (grid == 0) return 0;
  // (as many steps ahead as let two workgroups live on a CU)
#define ESMOE_FEW(T, K, NT, NC, AHEAD) \
  hipLaunchKernelGGL((expert_mm_few_kernel<T, K, NT, NC, AHEAD>), dim3((unsigned)grid), dim3(kFewThreads), 0, stream, g)
#define ESMOE_FEW3(T, K)                                                              \
  {                                                                                   \
    if (row_tiles == 2 && col_tiles == 4) ESMOE_FEW(T, K, 2, 4, 2);                   \
    else if (row_tiles == 2) ESMOE_FEW(T, K, 2, 2, 4);                                \
    else if (K != kFewForward || col_tiles == 2) ESMOE_FEW(T, K, 1, 2, 4);            \
    else ESMOE_FEW(T, K, 1, (K == kFewForward ? 1 : 2), 4);                           \
  }
#define ESMOE_FEW9(T)                                    \
  {                                                      \
    if (kind == 0) ESMOE_FEW3(T, kFewForward)            \
    else if (g.gate_up) ESMOE_FEW3(T, kFewSwigluSave)    \
    else ESMOE_FEW3(T, kFewSwiglu)                       \
  }
  if (g.type == kMmBf16) ESMOE_FEW9(kMmBf16)
  else if (g.type == kMmFp16) ESMOE_FEW9(kMmFp16)
  else if (kind == 0) ESMOE_FEW3(kMmInt8, kFewForward)
  else ESMOE_FEW3(kMmInt8, kFewSwiglu)
#undef ESMOE_FEW9
#undef ESMOE_FEW3
#undef ESMOE_FEW
  return (int)hipGetLastError();
}
