// Rows to 8-bit integers with a scale each, the operands of the int8 grouped product:
//   amax = max |x| of a row,  scale = amax / 127 (fp32),  q = x * 127 / amax rounded to the nearest integer, ties to even
// The rounding is that of the exact quotient.  x * inv, inv = fp32(127 / amax), is off by less than 2^-16, so it rounds the same unless the
// exact quotient is that near to a half; a thread that meets such a value does its eight again with a division: x * 127 is exact in fp32,
// and a quotient of two numbers of at most eleven bits is a half, or further from one than the division's error.
// A row of zeros has scale 0 and zeros; one with an infinity or a NaN has the scale NaN and zeros.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "expert_mm.h"

namespace esmoe {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef uint16_t v2u16 __attribute__((ext_vector_type(2)));

template <bool FP16>
__device__ __forceinline__ float half_value(uint32_t bits) {
  if constexpr (FP16) return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  else return __builtin_bit_cast(float, bits << 16);
}

// Maximum over a wavefront of pairs of 16-bit magnitudes, in its last lane.
__device__ __forceinline__ uint32_t wave_max_last(uint32_t v) {
  auto step = [&](int below) {
    v = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2u16, v), __builtin_bit_cast(v2u16, below)));
  };
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
  return v;
}

// A row stays in registers: CHUNKS times eight per thread, THREADS threads per row; with 64 (a wavefront) four rows per workgroup.
// Magnitudes are compared as 15-bit integers, which have the order of the numbers and NaN above infinity.
template <bool FP16, int THREADS, int CHUNKS>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) int8_quant_kernel(const uint16_t* __restrict__ in, long rows, int k,
                                                                                   int8_t* __restrict__ q, float* __restrict__ scales) {
  constexpr int kWaves = THREADS / 64;
  __shared__ uint32_t s_top[kWaves];
  const int tid = THREADS < 256 ? threadIdx.x % THREADS : threadIdx.x;
  const long row = THREADS < 256 ? (long)blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS : blockIdx.x;
  if (row >= rows) return;   // (a whole wavefront, and no barrier where there are several rows)
  in += row * k;
  q += row * k;
  v4i raw[CHUNKS];
  uint32_t top = 0;
#pragma unroll
  for (int u = 0; u < CHUNKS; u++) {
    const int col = (u * THREADS + tid) * 8;
    raw[u] = v4i{0, 0, 0, 0};
    if (col < k) raw[u] = __builtin_nontemporal_load((const v4i*)(in + col));
  }
#pragma unroll
  for (int u = 0; u < CHUNKS; u++)
#pragma unroll
    for (int i = 0; i < 4; i++)
      top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2u16, top),
                                                                   __builtin_bit_cast(v2u16, (uint32_t)raw[u][i] & 0x7fff7fffu)));
  top = wave_max_last(top);
  if constexpr (THREADS == 64) {
    top = (uint32_t)__builtin_amdgcn_readlane((int)top, 63);
  } else {
    if ((tid & 63) == 63) s_top[tid >> 6] = top;
    __syncthreads();
    top = s_top[0];
#pragma unroll
    for (int i = 1; i < kWaves; i++)
      top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2u16, top), __builtin_bit_cast(v2u16, s_top[i])));
  }
  const uint32_t bits = (top >> 16) > (top & 0xffffu) ? top >> 16 : top & 0xffffu;
  const float amax = half_value<FP16>(bits);
  const bool finite = bits < (FP16 ? 0x7c00u : 0x7f80u);
  if (tid == 0) scales[row] = finite ? amax / 127.0f : __builtin_nanf("");
  // (where 127 / amax is no number, or no longer as exact as it has to be, every thread divides)
  const bool divide = amax < 0x1p-100f && bits != 0;
  const float inv = finite && bits ? 127.0f / amax : 0.0f;
  const float shift = amax < 1.0f ? 0x1p64f : 0x1p-64f, scaled = amax * shift;   // x * 127 has to stay a number
  constexpr float kMagic = 12582912.0f;   // 1.5 * 2^23: a sum with it is rounded to an integer, whose low byte is the sum's
#pragma unroll
  for (int u = 0; u < CHUNKS; u++) {
    const int col = (u * THREADS + tid) * 8;
    if (col >= k) continue;
    float x[8];
    uint32_t t[8];
    float far = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t w = (uint32_t)raw[u][j / 2];
      x[j] = finite ? half_value<FP16>(j & 1 ? w >> 16 : w & 0xffffu) : 0.0f;
      const float sum = __builtin_fmaf(x[j], inv, kMagic);
      t[j] = __builtin_bit_cast(uint32_t, sum);
      far = __builtin_fmaxf(far, __builtin_fabsf(__builtin_fmaf(x[j], inv, kMagic - sum)));
    }
    if (divide || far > 0.5f - 0x1p-15f) {
#pragma unroll
      for (int j = 0; j < 8; j++)
        t[j] = finite && bits ? (uint32_t)(int)__builtin_rintf(x[j] * shift * 127.0f / scaled) : 0u;
    }
    v2i o;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint32_t lo = __builtin_amdgcn_perm(t[4 * h + 1], t[4 * h], 0x0c0c0400u), hi = __builtin_amdgcn_perm(t[4 * h + 3], t[4 * h + 2], 0x0c0c0400u);
      o[h] = (int)(lo | hi << 16);
    }
    __builtin_nontemporal_store(o, (v2i*)(q + col));
  }
}

template <bool FP16>
static int launch_int8_quant(const void* in, long rows, int k, void* q, float* scales, hipStream_t stream) {
  // Threads per row as in the norm that works the same way: a wavefront for a short row; sixteen where there is at most a row per CU, or a
  // row is more than the registers of four; four else.
  const int threads = k <= 1024 ? 64 : rows <= 256 || k > 32768 ? 1024 : 256;
  const int chunks = (k + threads * 8 - 1) / (threads * 8);
  const long step = 1L << 22;
  for (long r = 0; r < rows; r += step) {
    const long n = rows - r < step ? rows - r : step;
    const unsigned grid = (unsigned)(threads == 64 ? (n + 3) / 4 : n);
#define ESMOE_QUANT(T, C)                                                                                                               \
  hipLaunchKernelGGL((int8_quant_kernel<FP16, T, C>), dim3(grid), dim3(T < 256 ? 256 : T), 0, stream, (const uint16_t*)in + r * k, n, k, \
                     (int8_t*)q + r * k, scales + r)
    if (threads == 64) {
      if (chunks <= 1) ESMOE_QUANT(64, 1);
      else ESMOE_QUANT(64, 2);
    } else if (threads == 1024) {
      if (chunks <= 1) ESMOE_QUANT(1024, 1);
      else if (chunks <= 2) ESMOE_QUANT(1024, 2);
      else if (chunks <= 4) ESMOE_QUANT(1024, 4);
      else ESMOE_QUANT(1024, 8);
    } else {
      if (chunks <= 1) ESMOE_QUANT(256, 1);
      else if (chunks <= 2) ESMOE_QUANT(256, 2);
      else if (chunks <= 4) ESMOE_QUANT(256, 4);
      else if (chunks <= 8) ESMOE_QUANT(256, 8);
      else ESMOE_QUANT(256, 16);
    }
#undef ESMOE_QUANT
  }
  return (int)hipGetLastError();
}

}  // namespace esmoe

extern "C" int esmoe_launch_int8_quant(const void* in, int fp16, long rows, int k, void* q, float* scales, hipStream_t stream) {
  using namespace esmoe;
  return (fp16 ? launch_int8_quant<true> : launch_int8_quant<false>)(in, rows, k, q, scales, stream);
}
