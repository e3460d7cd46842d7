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

// Each row is read once, and what is written is another kernel's to read: the stores are non-temporal, and where a call's tensor of rows is more
// than the memory-side cache holds (STREAM) the loads are too.  us, plain / stores / both: 4096 tokens x top-8 x 7168 105 / 99.3 / 91.3, its
// gradient 201 / 203 / 191.  The rule goes by the tensor, not by the rows that the pairs point to, which stand on the device alone: on a
// share of the experts these may fit in the cache.  Then the hint gains where they come from memory and costs where they are in the cache,
// us, stores / both, from memory and again: 8003 x top-8 x 4096, a quarter of the pairs 37.1 / 34.9 and 29.6 / 32.8, its gradient
// 65.5 / 57.9 and 54.1 / 56.1; an eighth or less costs either way (16384 x top-8 x 4096, a sixteenth 31.4 / 39.5 and 29.2 / 40.3).
constexpr long kCacheBytes = 1L << 28;
template <bool STREAM>
__device__ __forceinline__ v4i load8(const uint16_t* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load((const v4i*)p);
  else return *(const v4i*)p;
}

// One wavefront per 512 columns of a token, eight rows' loads in flight.  Bound by memory: 90 us for 4096 tokens x top-8 x 7168 are 5.9 TB/s.
// One row after the other was 3.7 us for one token, this is 2.6.
template <bool FP16, bool STREAM>
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
    // (a lane beyond the columns loads from the row's start)
    for (unsigned long long todo = __ballot(mine >= 0); todo;) {
      v4i raw[8];
      float w[8];
      int n = 0;
#pragma unroll
      for (int u = 0; u < 8; u++)
        if (todo) {
          const int k = __builtin_ctzll(todo);
          todo &= todo - 1;
          n = u + 1;
          w[u] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), k));
          raw[u] = load8<STREAM>(in + (long)__builtin_amdgcn_readlane(mine, k) * hidden + (col < hidden ? col : 0));
        }
#pragma unroll
      for (int u = 0; u < 8; u++)
        if (u < n) {
          float x[8];
          unpack8<FP16>(raw[u], x);
#pragma unroll
          for (int i = 0; i < 8; i++) acc[i] = __builtin_fmaf(w[u], x[i], acc[i]);
        }
    }
  }
  if (col < hidden) __builtin_nontemporal_store(pack8<FP16>(acc), (v4i*)(out + t * hidden + col));
}

// One wavefront per pair; the four of a workgroup are mostly a token's, whose gradient row comes from HBM once and then from a cache.
// A workgroup per token that took its pairs one after the other was the same speed for many long rows, but three times as long for few
// tokens (one token x top-8 x 7168: 10.7 us, as it is 4.5; 16384 tokens x top-8 x 512 95 / 51).  All of a token's pairs on one XCD: no change.
template <bool FP16, bool STREAM>
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
        x[u] = load8<STREAM>(xp + col + u * 512);
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
        __builtin_nontemporal_store(pack8<FP16>(gf), (v4i*)(op + col + u * 512));
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
  const bool stream_in = 2 * (rows < tokens * topk ? rows : tokens * topk) * hidden > kCacheBytes;
  auto kernel = dtype ? (stream_in ? combine_rows_kernel<true, true> : combine_rows_kernel<true, false>)
                      : (stream_in ? combine_rows_kernel<false, true> : combine_rows_kernel<false, false>);
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
  const bool stream_in = 4 * (rows < tokens * topk ? rows : tokens * topk) * hidden > kCacheBytes;   // (with their gradients)
  auto kernel = dtype ? (stream_in ? combine_rows_backward_kernel<true, true> : combine_rows_backward_kernel<true, false>)
                      : (stream_in ? combine_rows_backward_kernel<false, true> : combine_rows_backward_kernel<false, false>);
  for (long t = 0; t < tokens; t += step) {
    const long n = tokens - t < step ? tokens - t : step;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((n * topk + 3) / 4)), dim3(256), 0, stream, (const uint16_t*)grad_out + t * hidden,
                       (const uint16_t*)in, dst_row + t * topk, weights + t * topk, (uint32_t)(n * topk), (uint32_t)topk, rows, hidden,
                       (uint16_t*)grad_in, grad_weights + t * topk);
  }
  return (int)hipGetLastError();
}
