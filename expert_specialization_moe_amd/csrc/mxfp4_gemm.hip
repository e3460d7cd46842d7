// Grouped product of few rows per expert with 4-bit weights: bf16/fp16 activations, e2m1 weights, one E8M0 scale per 32 along K.
//
//   out[off_e + m, n] = cast( sum_k a[off_e + m, k] * e2m1(b[e, n, k]) * 2^(sf[e, n, k / 32] - 127) )
//   swiglu form, n = 2 * inter, gate rows first: out[off_e + m, i] = cast( silu(gate) * up ) of the two fp32 sums
//
// Decode: every weight of an expert with rows is read once, 17/32 bytes each, and used for a handful of rows; the bound is HBM.
// The 4-bit codes become bf16/fp16 values exactly (v_cvt_scalef32_pk_*_fp4, scale 1) and go through v_mfma_f32_16x16x32 with up to
// sixteen rows of `a`; a product of 32 columns belongs to one scale, which its fp32 result is multiplied by as it is added up: no range
// of scales is lost in a 16-bit format.
//
// A workgroup of four wavefronts takes 16 weight rows (16 of the gate and 16 of the up projection) for 16 rows of `a`; the wavefronts
// split K, their sums are added in LDS in wavefront order.  No counterpart in the reference (its operators are 8-bit).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "swiglu.h"
#include "wave_scan.h"

namespace esmoe {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

constexpr int kFp4Threads = 256, kFp4Waves = 4, kFp4Rows = 16;

// Eight weights of a dword as values of the activations' type.
template <bool FP16>
__device__ __forceinline__ v4i fp4_values(uint32_t w) {
  v4i r;
  if constexpr (FP16) {
    r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0));
    r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1));
    r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2));
    r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3));
  } else {
    r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0));
    r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1));
    r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2));
    r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3));
  }
  return r;
}

template <bool FP16>
__device__ __forceinline__ v4f mfma32(v4i a, v4i b) {
  const v4f zero = {0.f, 0.f, 0.f, 0.f};
  if constexpr (FP16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), zero, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), zero, 0, 0, 0);
}

// 2^(code - 127); NaN for 255.
__device__ __forceinline__ float e8m0(uint32_t code) {
  return __builtin_bit_cast(float, code == 0 ? 0x00400000u : code == 255 ? 0x7fc00000u : code << 23);
}

// Dword i of lane row r (sixteen lanes) goes to dword r of lane row i.
__device__ __forceinline__ void transpose_rows(uint32_t* d) {
  auto swap32 = [](uint32_t& x, uint32_t& y) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    x = r[0];
    y = r[1];
  };
  auto swap16 = [](uint32_t& x, uint32_t& y) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
    x = r[0];
    y = r[1];
  };
  swap32(d[0], d[2]);
  swap32(d[1], d[3]);
  swap16(d[0], d[1]);
  swap16(d[2], d[3]);
}

struct Fp4Unit {
  int expert, row0, rows;   // rows 0: no such unit
};

// Unit u of the launch: experts in order, each in tiles of kFp4Rows rows.  Rows are clamped to the tensor.
__device__ __forceinline__ Fp4Unit fp4_unit(int u, const int* __restrict__ problem_sizes, const int* __restrict__ expert_offsets,
                                            int num_experts, int total_rows) {
  const int lane = threadIdx.x & 63;
  for (int e0 = 0; e0 < num_experts; e0 += 64) {
    const int e = e0 + lane;
    int m = 0, off = 0;
    if (e < num_experts) {
      m = problem_sizes[e * 3];
      off = expert_offsets[e];
      m = off < 0 || off >= total_rows || m < 0 ? 0 : m > total_rows - off ? total_rows - off : m;
    }
    const int tiles = (m + kFp4Rows - 1) / kFp4Rows;
    const int end = wave_inclusive_sum(tiles);
    const unsigned long long behind = __ballot(end > u);
    if (behind) {
      const int l = __builtin_ctzll(behind);
      const int tile = u - (__builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(tiles, l));
      const int rows = __builtin_amdgcn_readlane(m, l) - tile * kFp4Rows;
      return {e0 + l, __builtin_amdgcn_readlane(off, l) + tile * kFp4Rows, rows < kFp4Rows ? rows : kFp4Rows};
    }
    u -= __builtin_amdgcn_readlane(end, 63);
  }
  return {0, 0, 0};
}

template <bool FP16, bool SWIGLU>
__global__ void __launch_bounds__(kFp4Threads) mxfp4_grouped_mm_kernel(const uint16_t* __restrict__ a, const uint8_t* __restrict__ b,
                                                                       const uint8_t* __restrict__ sf, const int* __restrict__ problem_sizes,
                                                                       const int* __restrict__ expert_offsets, int num_experts,
                                                                       int total_rows, int n, int k, int col_tiles, int unit0,
                                                                       uint16_t* __restrict__ out) {
  constexpr int NT = SWIGLU ? 2 : 1;
  __shared__ float s_sum[kFp4Waves][NT][kFp4Rows][16];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int l16 = lane & 15, lr = lane >> 4;
  const int unit = blockIdx.x / col_tiles, tile = blockIdx.x - unit * col_tiles;
  const Fp4Unit g = fp4_unit(unit0 + unit, problem_sizes, expert_offsets, num_experts, total_rows);
  if (g.rows == 0) return;   // the whole workgroup
  const int wide = n / NT;   // columns of the output
  const long kb = k / 2, ks = k / 32;
  const uint8_t* bp[NT];
  const uint8_t* sp[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const long row = (long)g.expert * n + t * wide + tile * 16 + l16;
    bp[t] = b + row * kb + lr * 16;
    sp[t] = sf + row * ks;
  }
  const bool has_row = l16 < g.rows;
  const uint16_t* ap = a + (long)(g.row0 + (has_row ? l16 : 0)) * k + lr * 8;
  v4f acc[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};
  const int chunks = k / 128, per = (chunks + kFp4Waves - 1) / kFp4Waves;
  const int end = (w + 1) * per < chunks ? (w + 1) * per : chunks;
#pragma unroll 2
  for (int c = w * per; c < end; c++) {
    uint32_t d[NT][4], s[NT];
    v4i x[4];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const v4i raw = __builtin_nontemporal_load((const v4i*)(bp[t] + c * 64));
#pragma unroll
      for (int i = 0; i < 4; i++) d[t][i] = (uint32_t)raw[i];
      s[t] = *(const uint32_t*)(sp[t] + c * 4);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[i] = v4i{0, 0, 0, 0};
      if (has_row) x[i] = *(const v4i*)(ap + c * 128 + i * 32);
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
      transpose_rows(d[t]);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const v4f p = mfma32<FP16>(x[i], fp4_values<FP16>(d[t][i]));
        const float scale = e8m0(s[t] >> (8 * i) & 0xff);
#pragma unroll
        for (int r = 0; r < 4; r++) acc[t][r] = __builtin_fmaf(p[r], scale, acc[t][r]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int r = 0; r < 4; r++) s_sum[w][t][lr * 4 + r][l16] = acc[t][r];
  __syncthreads();
  const int m = tid >> 4, col = tid & 15;
  if (m >= g.rows) return;
  float v[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) v[t] = (s_sum[0][t][m][col] + s_sum[1][t][m][col]) + (s_sum[2][t][m][col] + s_sum[3][t][m][col]);
  float y = v[0];
  if constexpr (SWIGLU) y = swiglu_f32(v[0], v[1]);
  uint16_t bits;
  if constexpr (FP16) bits = __builtin_bit_cast(uint16_t, (_Float16)y);
  else bits = __builtin_bit_cast(uint16_t, (__bf16)y);
  out[(long)(g.row0 + m) * wide + tile * 16 + col] = bits;
}

}  // namespace esmoe

extern "C" int esmoe_launch_mxfp4_grouped_mm(const void* a, int dtype, const void* b, const uint8_t* sf, const int* problem_sizes,
                                             const int* expert_offsets, int num_experts, int total_rows, int n, int k, int swiglu, void* out,
                                             hipStream_t stream) {
  using namespace esmoe;
  const int col_tiles = n / (swiglu ? 32 : 16);
  // units with rows: at most one per expert or row, and one more per full tile
  const long units = (num_experts < total_rows ? num_experts : total_rows) + (long)total_rows / kFp4Rows;
  const long step = (1L << 23) / col_tiles > 1 ? (1L << 23) / col_tiles : 1;   // units of a launch: a grid holds fewer than 2^32 threads
  auto kernel = dtype ? swiglu ? mxfp4_grouped_mm_kernel<true, true> : mxfp4_grouped_mm_kernel<true, false>
                      : swiglu ? mxfp4_grouped_mm_kernel<false, true> : mxfp4_grouped_mm_kernel<false, false>;
  for (long u = 0; u < units; u += step) {
    const long some = units - u < step ? units - u : step;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(some * col_tiles)), dim3(kFp4Threads), 0, stream, (const uint16_t*)a, (const uint8_t*)b, sf,
                       problem_sizes, expert_offsets, num_experts, total_rows, n, k, col_tiles, (int)u, (uint16_t*)out);
  }
  return (int)hipGetLastError();
}
