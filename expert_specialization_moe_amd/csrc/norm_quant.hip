// Residual addition, root-mean-square norm and 1x128 FP8 quantisation in one pass over a row.
//
//   h = in + residual (fp32, rounded to the tensors' type: the new residual), or in
//   y = h * (1 / sqrt(mean(h^2) + eps)) * weight      (fp32)
//   normed = y rounded to the tensors' type (optional: what a router reads)
//   per 128 columns: amax = max(|y|, 1e-4), q = e4m3fn(y * (1 / amax * 448)), scale = amax * fl(1 / 448)
// The quantisation is fp8_quant.hip's, of y as it is: one rounding less than quantising the rounded norm.  A NaN of y is a NaN of its
// block's scale and bytes.  The reference has no norm; its callers quantise with a torch helper (test/test_es_grouped_gemm.py:36-44).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wave_scan.h"

namespace esmoe {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));

template <bool FP16>
__device__ __forceinline__ float half_to_f32(uint32_t bits) {
  if constexpr (FP16) return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  else return __builtin_bit_cast(float, bits << 16);
}
template <bool FP16>
__device__ __forceinline__ uint32_t f32_to_half(float v) {
  if constexpr (FP16) return __builtin_bit_cast(uint16_t, (_Float16)v);
  else return __builtin_bit_cast(uint16_t, (__bf16)v);
}

template <bool STREAM>
__device__ __forceinline__ v4i load8(const uint16_t* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load((const v4i*)p);
  else return *(const v4i*)p;
}

// Maximum over sixteen lanes; on bit patterns of non-negative floats, so that a NaN is the largest.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax16(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
  return v > o ? v : o;
}

// A row's values stay in registers: CHUNKS times eight per thread, THREADS threads per row; with 64 (a wavefront) four rows per workgroup.
// The squares of 512 columns, a wavefront's chunk, are summed for themselves and then one after the other by column: the same order for
// any number of threads, so a row's bytes do not hang on how many rows a call has.
// Nothing is read twice: the stores of 16-bit values and bytes are non-temporal (a scale is 4 bytes: stored plainly), or, where a call's tensors are
// more than the memory-side cache holds (STREAM), the loads and the stores of 16-bit values.  us, no hints / stores / STREAM, over three sets of
// tensors: 16384 x 7168 194 / 189 / 189, 65536 x 512 55.3 / 54.1 / 49.1; below the cache's size 1024 x 4096 8.7 / 7.3 / 8.4, 16384 x 1024
// 30.6 / 24.4 / 27.1.  (16384 x 7168 with the outputs in one place: 170.)
template <bool FP16, int THREADS, int CHUNKS, bool STREAM>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) add_rms_norm_quant_kernel(const uint16_t* in, const uint16_t* residual,
                                                                          const uint16_t* __restrict__ weight, float eps, long rows, int hidden,
                                                                          uint16_t* residual_out, uint16_t* __restrict__ normed,
                                                                          uint8_t* __restrict__ q, float* __restrict__ scales) {
  constexpr int kWaves = THREADS / 64;
  __shared__ float s_sum[kWaves * CHUNKS];   // by column
  const int tid = THREADS < 256 ? threadIdx.x % THREADS : threadIdx.x;
  const long number = THREADS < 256 ? (long)blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS : blockIdx.x;
  if (number >= rows) return;   // (a whole wavefront, and no barrier where there are several rows)
  const long row = number * hidden;
  float h[CHUNKS][8], part[CHUNKS];
#pragma unroll
  for (int u = 0; u < CHUNKS; u++) {
    const int col = (u * THREADS + tid) * 8;
    part[u] = 0;
    if (col < hidden) {
      const v4i a = load8<STREAM>(in + row + col);
      v4i r = {0, 0, 0, 0};
      if (residual) r = load8<STREAM>(residual + row + col);
      v4i o;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float lo = half_to_f32<FP16>((uint32_t)a[i] & 0xffffu), hi = half_to_f32<FP16>((uint32_t)a[i] >> 16);
        if (residual) {
          const uint32_t l = f32_to_half<FP16>(lo + half_to_f32<FP16>((uint32_t)r[i] & 0xffffu));
          const uint32_t g = f32_to_half<FP16>(hi + half_to_f32<FP16>((uint32_t)r[i] >> 16));
          o[i] = (int)(l | g << 16);
          lo = half_to_f32<FP16>(l);
          hi = half_to_f32<FP16>(g);
        }
        h[u][2 * i] = lo;
        h[u][2 * i + 1] = hi;
        part[u] = __builtin_fmaf(lo, lo, part[u]);
        part[u] = __builtin_fmaf(hi, hi, part[u]);
      }
      if (residual) __builtin_nontemporal_store(o, (v4i*)(residual_out + row + col));
    }
  }
#pragma unroll
  for (int u = 0; u < CHUNKS; u++) part[u] = wave_sum_last(part[u]);
  float sum;
  if constexpr (THREADS == 64) {
    sum = 0;
#pragma unroll
    for (int u = 0; u < CHUNKS; u++) sum += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, part[u]), 63));
  } else {
    if ((tid & 63) == 63) {
#pragma unroll
      for (int u = 0; u < CHUNKS; u++) s_sum[u * kWaves + (tid >> 6)] = part[u];
    }
    __syncthreads();
    sum = s_sum[0];
#pragma unroll
    for (int i = 1; i < kWaves * CHUNKS; i++) sum += s_sum[i];   // (0 past the row's end)
  }
  const float rstd = 1.0f / sqrtf(sum / (float)hidden + eps);
#pragma unroll
  for (int u = 0; u < CHUNKS; u++) {
    const int col = (u * THREADS + tid) * 8;   // sixteen lanes hold 128 columns: in or out of the row as one
    if (col < hidden) {
      const v4i g = *(const v4i*)(weight + col);
      uint32_t amax = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        h[u][i] = h[u][i] * rstd * half_to_f32<FP16>(i & 1 ? (uint32_t)g[i / 2] >> 16 : (uint32_t)g[i / 2] & 0xffffu);
        const uint32_t b = __builtin_bit_cast(uint32_t, h[u][i]) & 0x7fffffffu;
        amax = amax > b ? amax : b;
      }
      amax = dpp_umax16<0x140>(dpp_umax16<0x141>(dpp_umax16<0x4E>(dpp_umax16<0xB1>(amax))));
      const uint32_t least = __builtin_bit_cast(uint32_t, 1e-4f);
      const float top = __builtin_bit_cast(float, amax > least ? amax : least);
      const float mult = (1.0f / top) * 448.0f;
      if (normed) {
        v4i o;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = (int)(f32_to_half<FP16>(h[u][2 * i]) | f32_to_half<FP16>(h[u][2 * i + 1]) << 16);
        __builtin_nontemporal_store(o, (v4i*)(normed + row + col));
      }
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; i++) y[i] = h[u][i] * mult;   // (at most 448 and an ulp or two, which rounds to 448)
      int w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w0, true);
      int w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
      w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], w1, true);
      if constexpr (STREAM) *(v2i*)(q + row + col) = v2i{w0, w1};
      else __builtin_nontemporal_store(v2i{w0, w1}, (v2i*)(q + row + col));
      if ((tid & 15) == 0) scales[(row + col) >> 7] = top * (1.0f / 448.0f);
    }
  }
}

template <bool FP16, bool STREAM>
static int launch_norm(const void* in, const void* residual, const void* weight, float eps, long rows, int hidden, void* residual_out,
                       void* normed, void* q, float* scales, hipStream_t stream) {
  // Threads per row: a wavefront where a row is short enough to be its registers' (no barrier, more rows in flight); sixteen wavefronts
  // where there is at most a row per CU (what counts is how long one takes); four else.  us, always four / as chosen: 8 rows x 7168 4.5 /
  // 3.45, 256 x 7168 5.8 / 4.9, 16384 x 256 12.0 / 10.1, 65536 x 512 63.9 / 49.9, 16384 x 1024 24.6 / 23.5.
  const int threads = rows <= 256 && hidden > 1024 ? 1024 : hidden <= 1024 ? 64 : 256;
  const int chunks = (hidden + threads * 8 - 1) / (threads * 8);
  const long step = 1L << 22;
  for (long r = 0; r < rows; r += step) {
    const long n = rows - r < step ? rows - r : step, at = r * hidden;
    const unsigned grid = (unsigned)(threads == 64 ? (n + 3) / 4 : n);
#define ESMOE_NORM(T, C)                                                                                                          \
  hipLaunchKernelGGL((add_rms_norm_quant_kernel<FP16, T, C, STREAM>), dim3(grid), dim3(T < 256 ? 256 : T), 0, stream,                      \
                     (const uint16_t*)in + at, residual ? (const uint16_t*)residual + at : nullptr, (const uint16_t*)weight, eps, n, \
                     hidden, residual ? (uint16_t*)residual_out + at : nullptr, normed ? (uint16_t*)normed + at : nullptr,        \
                     (uint8_t*)q + at, scales + at / 128)
    if (threads == 64) {
      if (chunks <= 1) ESMOE_NORM(64, 1);
      else ESMOE_NORM(64, 2);
    } else if (threads == 1024) {
      if constexpr (!STREAM) {   // (256 rows fit in the cache)
        if (chunks <= 1) ESMOE_NORM(1024, 1);
        else if (chunks <= 2) ESMOE_NORM(1024, 2);
        else ESMOE_NORM(1024, 4);
      }
    } else {
      if (chunks <= 1) ESMOE_NORM(256, 1);
      else if (chunks <= 2) ESMOE_NORM(256, 2);
      else if (chunks <= 4) ESMOE_NORM(256, 4);
      else if (chunks <= 8) ESMOE_NORM(256, 8);
      else ESMOE_NORM(256, 16);
    }
#undef ESMOE_NORM
  }
  return (int)hipGetLastError();
}

}  // namespace esmoe

extern "C" int esmoe_launch_add_rms_norm_quant(const void* in, int in_dtype, const void* residual, const void* weight, float eps, long rows,
                                               int hidden, void* residual_out, void* normed, void* q, float* scales, hipStream_t stream) {
  using namespace esmoe;
  const bool stream_in = (residual ? normed ? 9 : 7 : normed ? 5 : 3) * rows * hidden > (1L << 28);   // (bytes an element)
  auto launch = in_dtype ? (stream_in ? launch_norm<true, true> : launch_norm<true, false>)
                         : (stream_in ? launch_norm<false, true> : launch_norm<false, false>);
  return launch(in, residual, weight, eps, rows, hidden, residual_out, normed, q, scales, stream);
}
