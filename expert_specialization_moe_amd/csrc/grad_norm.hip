// The norm over many gradients and their clipping to a largest norm.
//
//   norm = sqrt( sum over all elements of x^2 ),   coef = max_norm / (norm + eps);  where coef < 1 (or NaN):  out = x * coef, else out = x
// Squares are formed and added in 64 bits: no gradient is too large or too small for its square, and the order of the sum does not show.
// A workgroup sums a contiguous share of all chunks into one partial sum; whoever needs the norm adds the partial sums in one fixed order,
// so a call's result does not hang on which workgroup ends first and needs neither atomics nor cleared memory.
// Bound by memory: every gradient is read for the norm, and read and written for the clipping.  3.2 GB of bf16 gradients: 478 us (6.7 TB/s)
// and 1297 us (5.0 TB/s).  A chunk's loads are all under way before the first is used (one piece at a time: 762 and 1445 us).  What is
// written is not kept in the caches, which hold 256 MB, and so is what is read of more than twice as much, whose second pass finds little of it
// (us, read past the caches and kept there, both passes: 3.2 GB 1768 / 1830, 400 MB 223 / 220, 200 MB 112 / 95, 100 MB 58 / 52).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "grad_norm.h"

namespace esmoe {

// Sum over the workgroup, in one order, in every thread.
__device__ __forceinline__ double workgroup_sum(double v, double* s) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = v;
  __syncthreads();
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// Aligned as its elements are: a gradient may begin anywhere.
template <typename T> struct Eight { typedef T V __attribute__((ext_vector_type(8), aligned(sizeof(T)))); };

// f(tensor, first element, elements) for every chunk of this workgroup's share; backwards, for what a pass over all gradients read last is
// still in the caches when the next pass begins (3.2 GB: 1290 us against 1305).
template <bool BACKWARDS, typename F>
__device__ __forceinline__ void for_chunks(const GradTable& t, F&& f) {
  const long chunks = t.end[t.count - 1], from = chunks * blockIdx.x / gridDim.x, to = chunks * (blockIdx.x + 1) / gridDim.x;
  if (from == to) return;
  long c = BACKWARDS ? to - 1 : from;
  int i = 0;   // the tensors that end in front of it
#pragma unroll
  for (int j = 0; j < (kGradTensors + 63) / 64; j++) {
    const int at = j * 64 + (threadIdx.x & 63);
    i += __popcll(__ballot(at < t.count && t.end[at < t.count ? at : 0] <= c));
  }
  for (; BACKWARDS ? c >= from : c < to; c += BACKWARDS ? -1 : 1) {
    while (!BACKWARDS && t.end[i] <= c) i++;
    while (BACKWARDS && i && t.end[i - 1] > c) i--;
    const long first = (c - (i ? t.end[i - 1] : 0)) * kGradChunk, left = t.size[i] - first;
    f(i, first, (int)(left < kGradChunk ? left : kGradChunk));
  }
}

// A chunk in registers, 8 elements at a time, and what is left over.
constexpr int kPieces = kGradChunk / 8 / 256;
template <typename T>
struct Chunk {
  typedef typename Eight<T>::V V;
  V v[kPieces];
  T rest;
  template <bool STREAM>
  __device__ __forceinline__ static V piece(const V* p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(p);
    else return *p;
  }
  template <bool STREAM>
  __device__ __forceinline__ void read(const T* x, int n) {
    const int whole = n / 8;
    rest = (T)0.0f;
    if (n == kGradChunk) {   // (all loads under way at once)
#pragma unroll
      for (int i = 0; i < kPieces; i++) v[i] = piece<STREAM>((const V*)x + threadIdx.x + i * 256);
    } else {
#pragma unroll
      for (int i = 0; i < kPieces; i++) {
        v[i] = V{};
        if ((int)threadIdx.x + i * 256 < whole) v[i] = piece<STREAM>((const V*)x + threadIdx.x + i * 256);
      }
      if ((int)threadIdx.x < n - whole * 8) rest = x[whole * 8 + threadIdx.x];
    }
  }
  __device__ __forceinline__ double squares() const {
    double sum[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kPieces; i++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const double e = (double)(float)v[i][j];
        sum[j & 1] = __builtin_fma(e, e, sum[j & 1]);
      }
    const double e = (double)(float)rest;
    return __builtin_fma(e, e, sum[0]) + sum[1];
  }
  __device__ __forceinline__ void scale(float coef) {
#pragma unroll
    for (int i = 0; i < kPieces; i++)
#pragma unroll
      for (int j = 0; j < 8; j++) v[i][j] = (T)((float)v[i][j] * coef);
    rest = (T)((float)rest * coef);
  }
  __device__ __forceinline__ void write(T* y, int n) const {
    const int whole = n / 8;
#pragma unroll
    for (int i = 0; i < kPieces; i++)
      if (n == kGradChunk || (int)threadIdx.x + i * 256 < whole) __builtin_nontemporal_store(v[i], (V*)y + threadIdx.x + i * 256);
    if ((int)threadIdx.x < n - whole * 8) y[whole * 8 + threadIdx.x] = rest;
  }
};

__global__ void __launch_bounds__(256) grad_squares_kernel(GradTable t, double* __restrict__ partial) {
  __shared__ double s[4];
  double sum = 0;
  for_chunks<false>(t, [&](int i, long first, int n) {
    auto add = [&](auto zero) {
      typedef decltype(zero) T;
      Chunk<T> chunk;
      if (t.stream) chunk.template read<true>((const T*)t.in[i] + first, n);
      else chunk.template read<false>((const T*)t.in[i] + first, n);
      sum += chunk.squares();
    };
    if (t.type[i] == kGradFp32) add(0.0f);
    else if (t.type[i] == kGradFp16) add((_Float16)0.0f);
    else add((__bf16)0.0f);
  });
  sum = workgroup_sum(sum, s);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__device__ __forceinline__ double sum_partials(const double* __restrict__ partial, int count, double* s) {
  double sum = 0;
  for (int i = threadIdx.x; i < count; i += 256) sum += partial[i];
  return workgroup_sum(sum, s);
}

__global__ void __launch_bounds__(256) grad_norm_kernel(const double* __restrict__ partial, int count, const float* __restrict__ given,
                                                        float* __restrict__ norm) {
  __shared__ double s[4];
  const double sum = sum_partials(partial, count, s);
  if (threadIdx.x == 0) *norm = given ? *given : (float)sqrt(sum);
}

// given: a norm from elsewhere instead of the partial sums'.  norm_out: of a call's launches one writes it.
__global__ void __launch_bounds__(256) grad_clip_kernel(GradTable t, const double* __restrict__ partial, int count, const float* __restrict__ given,
                                                        double max_norm, double eps, float* __restrict__ norm_out) {
  __shared__ double s[4];
  bool have = false;
  float coef = 1.0f;
  auto find = [&] {   // (behind the first chunk's loads: the whole workgroup comes here together)
    if (have) return;
    have = true;
    const double norm = given ? (double)*given : sqrt(sum_partials(partial, count, s));
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const float ratio = max_norm < __builtin_inf() ? (float)(max_norm / (norm + eps)) : 1.0f;
    coef = ratio >= 1.0f ? 1.0f : ratio;   // (a NaN stays one)
  };
  for_chunks<true>(t, [&](int i, long first, int n) {
    if (have && coef == 1.0f && t.in[i] == t.out[i]) return;
    auto clip = [&](auto zero) {
      typedef decltype(zero) T;
      Chunk<T> chunk;
      chunk.template read<false>((const T*)t.in[i] + first, n);
      find();
      if (coef == 1.0f && t.in[i] == t.out[i]) return;
      chunk.scale(coef);
      chunk.write((T*)t.out[i] + first, n);
    };
    if (t.type[i] == kGradFp32) clip(0.0f);
    else if (t.type[i] == kGradFp16) clip((_Float16)0.0f);
    else clip((__bf16)0.0f);
  });
  find();
}

}  // namespace esmoe

extern "C" int esmoe_launch_grad_squares(const esmoe::GradTable* t, int grid, double* partial, hipStream_t stream) {
  hipLaunchKernelGGL(esmoe::grad_squares_kernel, dim3(grid), dim3(256), 0, stream, *t, partial);
  return (int)hipGetLastError();
}
extern "C" int esmoe_launch_grad_norm(const double* partial, int count, const float* given, float* norm, hipStream_t stream) {
  hipLaunchKernelGGL(esmoe::grad_norm_kernel, dim3(1), dim3(256), 0, stream, partial, count, given, norm);
  return (int)hipGetLastError();
}
extern "C" int esmoe_launch_grad_clip(const esmoe::GradTable* t, int grid, const double* partial, int count, const float* given, double max_norm,
                                      double eps, float* norm_out, hipStream_t stream) {
  hipLaunchKernelGGL(esmoe::grad_clip_kernel, dim3(grid), dim3(256), 0, stream, *t, partial, count, given, max_norm, eps, norm_out);
  return (int)hipGetLastError();
}
