// The way back from the experts: every token's packed rows summed with its routing weights, and the gradients of both.
//
//   out[t]           = sum over j < topk with a local row of weights[t, j] * in[dst_row[t * topk + j]]     (fp32, j rising, one rounding)
//   grad_in[dst]     = weights[t, j] * grad_out[t]
//   grad_weights[t,j]= <grad_out[t], in[dst]>, 0 without a local row
// dst_row is what the routing metadata give: a row of the packed tensor, or -1 for a pair of another GPU's expert (any other row outside
// the tensor counts as -1).  Without weights the sum is the gradient of the row packing (out[dst_row[p]] = in[p / topk]).
// The reference has no such step: its benchmark stops behind the grouped GEMM (benchmark/benchmark_es_fp8_blockwise_moe.py:200-260).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wave_scan.h"

namespace esmoe {

typedef int v4i __attribute__((ext_vector_type(4)));

template <bool FP16>
__device__ __forceinline__ void unpack8(v4i raw, float* x) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t w = (uint32_t)raw[i];
    if constexpr (FP16) {
      x[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w & 0xffffu));
      x[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
    } else {
      x[2 * i] = __builtin_bit_cast(float, w << 16);
      x[2 * i + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
    }
  }
}
template <bool FP16>
__device__ __forceinline__ v4i pack8(const float* x) {
  v4i r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t lo, hi;
    if constexpr (FP16) {
      lo = __builtin_bit_cast(uint16_t, (_Float16)x[2 * i]);
      hi = __builtin_bit_cast(uint16_t, (_Float16)x[2 * i + 1]);
    } else {
      lo = __builtin_bit_cast(uint16_t, (__bf16)x[2 * i]);
      hi = __builtin_bit_cast(uint16_t, (__bf16)x[2 * i + 1]);
    }
    r[i] = (int)(lo | hi << 16);
  }
  return r;
}

// One wavefront per 512 columns of a token.
template <bool FP16>
__global__ void __launch_bounds__(256) combine_rows_kernel(const uint16_t* __restrict__ in, const int* __restrict__ dst_row,
                                                           const float* __restrict__ weights, long tokens, int topk, long rows,
                                                           int hidden, uint32_t pieces, uint16_t* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const uint32_t piece = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long t = pieces == 1 ? piece : piece / pieces;
  if (t >= tokens) return;
  const int col = (int)(piece - (uint32_t)t * pieces) * 512 + lane * 8;
  float acc[8] = {};
  for (int j0 = 0; j0 < topk; j0 += 64) {
    const int j = j0 + lane;
    int mine = j < topk ? dst_row[t * topk + j] : -1;
    if ((unsigned long)(long)mine >= (unsigned long)rows) mine = -1;
    const float weight = mine < 0 ? 0.f : weights ? weights[t * topk + j] : 1.f;
    for (unsigned long long todo = __ballot(mine >= 0); todo; todo &= todo - 1) {
      const int k = __builtin_ctzll(todo);
      const long row = __builtin_amdgcn_readlane(mine, k);
      const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), k));
      if (col < hidden) {
        float x[8];
        unpack8<FP16>(*(const v4i*)(in + row * hidden + col), x);
#pragma unroll
        for (int i = 0; i < 8; i++) acc[i] = __builtin_fmaf(w, x[i], acc[i]);
      }
    }
  }
  if (col < hidden) *(v4i*)(out + t * hidden + col) = pack8<FP16>(acc);
}

// One wavefront per pair; the four of a workgroup are mostly a token's, whose gradient row comes from HBM once and then from a cache.
// A workgroup per token that took its pairs one after the other was the same speed for many long rows, but three times as long for few
// tokens (one token x top-8 x 7168: 10.7 us, as it is 4.5; 16384 tokens
// x top-8 x 512 95 / 51).
template <bool FP16>
__global__ void __launch_bounds__(256) combine_rows_backward_kernel(const uint16_t* __restrict__ grad_out, const uint16_t* __restrict__ in,
                                                                    const int* __restrict__ dst_row, const float* __restrict__ weights,
                                                                    uint32_t num_pairs, uint32_t topk, long rows, int hidden,
                                                                    uint16_t* __restrict__ grad_in, float* __restrict__ grad_weights) {
  const int lane = threadIdx.x & 63;
  const uint32_t pair = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (pair >= num_pairs) return;
  const long row = dst_row[pair];
  if ((unsigned long)row >= (unsigned long)rows) {
    if (lane == 0) grad_weights[pair] = 0.f;
    return;
  }
  const float weight = weights[pair];
  const uint16_t* gp = grad_out + (long)(pair / topk) * hidden;
  const uint16_t* xp = in + row * hidden;
  uint16_t* op = grad_in + row * hidden;
  float dot = 0;
  for (int col = lane * 8; col < hidden; col += 2048) {
    v4i g[4], x[4];
#pragma unroll
    for (int u = 0; u < 4; u++)
      if (col + u * 512 < hidden) {
        g[u] = *(const v4i*)(gp + col + u * 512);
        x[u] = __builtin_nontemporal_load((const v4i*)(xp + col + u * 512));
      }
#pragma unroll
    for (int u = 0; u < 4; u++)
      if (col + u * 512 < hidden) {
        float gf[8], xf[8];
        unpack8<FP16>(g[u], gf);
        unpack8<FP16>(x[u], xf);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          dot = __builtin_fmaf(gf[i], xf[i], dot);
          gf[i] *= weight;
        }
        *(v4i*)(op + col + u * 512) = pack8<FP16>(gf);
      }
  }
  dot = wave_sum_last(dot);
  if (lane == 63) grad_weights[pair] = dot;
}

}  // namespace esmoe

extern "C" int esmoe_launch_combine_rows(const void* in, int dtype, const int* dst_row, const float* weights, long tokens, int topk, long rows,
                                         int hidden, void* out, hipStream_t stream) {
  using namespace esmoe;
  const long pieces = (hidden + 511) / 512;
  const long step = (1L << 24) / pieces;   // tokens of a launch: a grid holds fewer than 2^32 threads
  auto kernel = dtype ? combine_rows_kernel<true> : combine_rows_kernel<false>;
  for (long t = 0; t < tokens; t += step) {
    const long n = tokens - t < step ? tokens - t : step;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((n * pieces + 3) / 4)), dim3(256), 0, stream, (const uint16_t*)in, dst_row + t * topk,
                       weights ? weights + t * topk : nullptr, n, topk, rows, hidden, (uint32_t)pieces, (uint16_t*)out + t * hidden);
  }
  return (int)hipGetLastError();
}

extern "C" int esmoe_launch_combine_rows_backward(const void* grad_out, const void* in, int dtype, const int* dst_row, const float* weights,
                                                  long tokens, int topk, long rows, int hidden, void* grad_in, float* grad_weights,
                                                  hipStream_t stream) {
  using namespace esmoe;
  const long step = (1L << 25) / topk > 0 ? (1L << 25) / topk : 1;   // tokens of a launch: a grid holds fewer than 2^32 threads
  auto kernel = dtype ? combine_rows_backward_kernel<true> : combine_rows_backward_kernel<false>;
  for (long t = 0; t < tokens; t += step) {
    const long n = tokens - t < step ? tokens - t : step;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((n * topk + 3) / 4)), dim3(256), 0, stream, (const uint16_t*)grad_out + t * hidden,
                       (const uint16_t*)in, dst_row + t * topk, weights + t * topk, (uint32_t)(n * topk), (uint32_t)topk, rows, hidden,
                       (uint16_t*)grad_in, grad_weights + t * topk);
  }
  return (int)hipGetLastError();
}
