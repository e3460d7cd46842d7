// Grouped products of the experts in 16 bits, with their gradients, and in 8-bit integers.
//
//   forward         out[off_e + m, j] = cast( sum_c a[off_e + m, c] * b[e, j, c] )
//   SwiGLU, n = 2 * inter, gate rows first: out = cast( silu(gate) * up ) of the two fp32 sums; gate_up = cast(sums), where asked for
//   rows' gradient  grad_a[off_e + m, c] = cast( sum_j grad_out[off_e + m, j] * b[e, j, c] )
//   weights'        grad_b[e, j, c] = cast( sum_m grad_out[off_e + m, j] * a[off_e + m, c] ), 0 for an expert without rows
//   int8            sums in int32 (exact), out = cast( sum * sa[off_e + m] * sb[e, j] )
// The reference has 8-bit floating point products alone and no gradients.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "expert_mm.h"
#include "swiglu.h"

namespace esmoe {

template <int TYPE> struct MmType;
template <> struct MmType<kMmBf16> { typedef __bf16 T; typedef float Acc; };
template <> struct MmType<kMmFp16> { typedef _Float16 T; typedef float Acc; };
template <> struct MmType<kMmInt8> { typedef int8_t T; typedef int Acc; };

constexpr int kTile = 64, kDeep = 16;

__device__ __forceinline__ int rows_in_tensor(int m, int off, int total_rows) {
  return off < 0 || off >= total_rows || m < 0 ? 0 : m > total_rows - off ? total_rows - off : m;
}

// One element of the output per thread and quarter; both operands staged through LDS, kDeep of the sum at a time.
template <int TYPE, typename FT, typename FW>
__device__ __forceinline__ void tile_product(int depth, FT&& t_at, FW&& w_at, typename MmType<TYPE>::Acc (&acc)[4][4]) {
  typedef typename MmType<TYPE>::Acc Acc;
  __shared__ Acc s_t[kDeep][kTile + 1], s_w[kDeep][kTile + 1];
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < 4; j++) acc[i][j] = 0;
  for (int c0 = 0; c0 < depth; c0 += kDeep) {
    for (int u = tid; u < kTile * kDeep; u += 256) {
      const int i = u / kDeep, c = u % kDeep;
      s_t[c][i] = c0 + c < depth ? t_at(i, c0 + c) : (Acc)0;
      s_w[c][i] = c0 + c < depth ? w_at(i, c0 + c) : (Acc)0;
    }
    __syncthreads();
    for (int c = 0; c < kDeep; c++)
      for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) acc[i][j] += s_t[c][ty * 4 + i] * s_w[c][tx + 16 * j];
    __syncthreads();
  }
}

// WT: the sum runs along w's columns (the rows' gradient).  SWIGLU: 32 gate columns and the matching 32 up columns a tile.
template <int TYPE, bool WT, bool SWIGLU>
__global__ void __launch_bounds__(256) expert_rows_kernel(ExpertMmArgs g) {
  typedef typename MmType<TYPE>::T T;
  typedef typename MmType<TYPE>::Acc Acc;
  const int depth = WT ? g.n : g.k, cols = WT ? g.k : g.n, wide = SWIGLU ? cols / 2 : cols;
  int unit = blockIdx.y, expert = -1, row0 = 0, rows = 0;
  for (int e = 0; e < g.num_experts; e++) {
    const int off = g.expert_offsets[e], m = rows_in_tensor(g.problem_sizes[e * 3], off, g.total_rows), tiles = (m + kTile - 1) / kTile;
    if (unit < tiles) {
      expert = e;
      row0 = off + unit * kTile;
      rows = m - unit * kTile;
      break;
    }
    unit -= tiles;
  }
  if (expert < 0) return;
  const int col0 = blockIdx.x * (SWIGLU ? kTile / 2 : kTile);
  const T* t = (const T*)g.t + (long)row0 * depth;
  const T* w = (const T*)g.w + (long)expert * g.n * g.k;
  auto col_of = [&](int j) { return SWIGLU ? (j & 31) + col0 + (j >> 5) * wide : j + col0; };
  Acc acc[4][4];
  tile_product<TYPE>(depth, [&](int i, int c) { return i < rows ? (Acc)t[(long)i * depth + c] : (Acc)0; },
                     [&](int j, int c) {
                       if ((SWIGLU ? (j & 31) : j) + col0 >= wide) return (Acc)0;
                       return (Acc)w[WT ? (long)c * cols + col_of(j) : (long)col_of(j) * depth + c];
                     }, acc);
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  for (int i = 0; i < 4; i++) {
    const int m = ty * 4 + i;
    if (m >= rows) continue;
    const long row = row0 + m;
    float v[4];
    for (int j = 0; j < 4; j++) {
      v[j] = (float)acc[i][j];
      if constexpr (TYPE == kMmInt8) {
        const int c = col_of(tx + 16 * j);
        v[j] = v[j] * g.sa[row] * (c < cols ? g.sb[(long)expert * g.n + c] : 0.f);
      }
    }
    auto put = [&](void* p, long at, float x) {
      if (TYPE == kMmFp16 || (TYPE == kMmInt8 && g.out_fp16)) ((_Float16*)p)[at] = (_Float16)x;
      else ((__bf16*)p)[at] = (__bf16)x;
    };
    for (int j = 0; j < (SWIGLU ? 2 : 4); j++) {
      const int c = col0 + tx + 16 * j;
      if (c >= wide) continue;
      if constexpr (SWIGLU) {
        if (g.gate_up) {
          put(g.gate_up, row * cols + c, v[j]);
          put(g.gate_up, row * cols + wide + c, v[j + 2]);
        }
        put(g.out, row * wide + c, swiglu_f32(v[j], v[j + 2]));
      } else put(g.out, row * wide + c, v[j]);
    }
  }
}

template <int TYPE>
__global__ void __launch_bounds__(256) expert_weights_kernel(ExpertMmArgs g) {
  typedef typename MmType<TYPE>::T T;
  const int tiles_k = (g.k + kTile - 1) / kTile, expert = blockIdx.y;
  const int n0 = blockIdx.x / tiles_k * kTile, k0 = blockIdx.x % tiles_k * kTile;
  const int off = g.expert_offsets[expert], rows = rows_in_tensor(g.problem_sizes[expert * 3], off, g.total_rows);
  const T *t = (const T*)g.t + (long)off * g.n, *w = (const T*)g.w + (long)off * g.k;
  float acc[4][4];
  tile_product<TYPE>(rows, [&](int i, int c) { return n0 + i < g.n ? (float)t[(long)c * g.n + n0 + i] : 0.f; },
                     [&](int j, int c) { return k0 + j < g.k ? (float)w[(long)c * g.k + k0 + j] : 0.f; }, acc);
  T* out = (T*)g.out + (long)expert * g.n * g.k;
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < 4; j++) {
      const int r = n0 + threadIdx.x / 16 * 4 + i, c = k0 + threadIdx.x % 16 + 16 * j;
      if (r < g.n && c < g.k) out[(long)r * g.k + c] = (T)acc[i][j];
    }
}

}  // namespace esmoe

using namespace esmoe;

// kind: 0 forward, 1 forward with SwiGLU, 2 gradient of the rows, 3 gradient of the weights
extern "C" int esmoe_launch_expert_mm(const ExpertMmArgs* args, int kind, int cus, hipStream_t stream) {
  const ExpertMmArgs& g = *args;
  const int cols = kind == 2 ? g.k : kind == 1 ? g.n / 2 : g.n, tile = kind == 1 ? kTile / 2 : kTile;
  const dim3 grid((cols + tile - 1) / tile, g.num_experts + g.total_rows / kTile);
#define ESMOE_MM(T)                                                                                             \
  switch (kind) {                                                                                               \
    case 0: hipLaunchKernelGGL((expert_rows_kernel<T, false, false>), grid, dim3(256), 0, stream, g); break;    \
    case 1: hipLaunchKernelGGL((expert_rows_kernel<T, false, true>), grid, dim3(256), 0, stream, g); break;     \
    case 2: hipLaunchKernelGGL((expert_rows_kernel<T, true, false>), grid, dim3(256), 0, stream, g); break;     \
    default: hipLaunchKernelGGL((expert_weights_kernel<T>), dim3(((g.n + 63) / 64) * ((g.k + 63) / 64), g.num_experts), dim3(256), 0, stream, g); \
  }
  if (g.type == kMmBf16) { ESMOE_MM(kMmBf16) }
  else if (g.type == kMmFp16) { ESMOE_MM(kMmFp16) }
  else if (kind == 0) hipLaunchKernelGGL((expert_rows_kernel<kMmInt8, false, false>), grid, dim3(256), 0, stream, g);
  else hipLaunchKernelGGL((expert_rows_kernel<kMmInt8, false, true>), grid, dim3(256), 0, stream, g);
#undef ESMOE_MM
  return (int)hipGetLastError();
}
