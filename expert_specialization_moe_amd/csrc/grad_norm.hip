// The norm over many gradients and their clipping to a largest norm.
//
//   norm = sqrt( sum over all elements of x^2 ),   coef = max_norm / (norm + eps);  where coef < 1 (or NaN):  out = x * coef, else out = x
// Squares are formed and added in 64 bits: no gradient is too large or too small for its square, and the order of the sum does not show.
// A workgroup sums a contiguous share of all chunks into one partial sum; whoever needs the norm adds the partial sums in one fixed order,
// so a call's result does not hang on which workgroup ends first and needs neither atomics nor cleared memory.  Bound by memory: every
// gradient is read for the norm, and read and written for the clipping.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "grad_norm.h"

namespace esmoe {

// Sum over the workgroup in one order, in every thread.
__device__ __forceinline__ double workgroup_sum(double v, double* s) {
  s[threadIdx.x] = v;
  __syncthreads();
  for (int d = 128; d; d /= 2) {
    if ((int)threadIdx.x < d) s[threadIdx.x] += s[threadIdx.x + d];
    __syncthreads();
  }
  return s[0];
}

template <typename T> struct Eight { T v[8]; };   // aligned as its elements are: a gradient may begin anywhere

// f(tensor, first element, elements) for every chunk of this workgroup's share.
template <typename F>
__device__ __forceinline__ void for_chunks(const GradTable& t, F&& f) {
  const long chunks = t.end[t.count - 1];
  long c = chunks * blockIdx.x / gridDim.x;
  const long last = chunks * (blockIdx.x + 1) / gridDim.x;
  int i = 0;
  while (c < last) {
    while (t.end[i] <= c) i++;
    const long first = (c - (i ? t.end[i - 1] : 0)) * kGradChunk, left = t.size[i] - first;
    f(i, first, left < kGradChunk ? left : kGradChunk);
    c++;
  }
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* x, long n) {
  double sum = 0;
  const long whole = n / 8;
  for (long p = threadIdx.x; p < whole; p += 256) {
    const Eight<T> e = ((const Eight<T>*)x)[p];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const double v = (double)(float)e.v[j];
      sum = __builtin_fma(v, v, sum);
    }
  }
  if (threadIdx.x < n - whole * 8) {
    const double v = (double)(float)x[whole * 8 + threadIdx.x];
    sum = __builtin_fma(v, v, sum);
  }
  return sum;
}

__global__ void __launch_bounds__(256) grad_squares_kernel(GradTable t, double* __restrict__ partial) {
  __shared__ double s[256];
  double sum = 0;
  for_chunks(t, [&](int i, long first, long n) {
    if (t.type[i] == kGradFp32) sum += chunk_squares((const float*)t.in[i] + first, n);
    else if (t.type[i] == kGradFp16) sum += chunk_squares((const _Float16*)t.in[i] + first, n);
    else sum += chunk_squares((const __bf16*)t.in[i] + first, n);
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
  __shared__ double s[256];
  const double sum = sum_partials(partial, count, s);
  if (threadIdx.x == 0) *norm = given ? *given : (float)sqrt(sum);
}

template <typename T>
__device__ __forceinline__ void clip_chunk(const T* x, T* y, long n, float coef) {
  const long whole = n / 8;
  for (long p = threadIdx.x; p < whole; p += 256) {
    Eight<T> e = ((const Eight<T>*)x)[p];
#pragma unroll
    for (int j = 0; j < 8; j++) e.v[j] = (T)((float)e.v[j] * coef);
    ((Eight<T>*)y)[p] = e;
  }
  if (threadIdx.x < n - whole * 8) y[whole * 8 + threadIdx.x] = (T)((float)x[whole * 8 + threadIdx.x] * coef);
}

// given: a norm from elsewhere instead of the partial sums'.  write_norm: of a call's launches one writes it.
__global__ void __launch_bounds__(256) grad_clip_kernel(GradTable t, const double* __restrict__ partial, int count, const float* __restrict__ given,
                                                        double max_norm, double eps, float* __restrict__ norm_out) {
  __shared__ double s[256];
  const double norm = given ? (double)*given : sqrt(sum_partials(partial, count, s));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const float ratio = max_norm < __builtin_inf() ? (float)(max_norm / (norm + eps)) : 1.0f;
  const float coef = ratio >= 1.0f ? 1.0f : ratio;   // (a NaN stays one)
  for_chunks(t, [&](int i, long first, long n) {
    if (coef == 1.0f && t.in[i] == t.out[i]) return;
    if (t.type[i] == kGradFp32) clip_chunk((const float*)t.in[i] + first, (float*)t.out[i] + first, n, coef);
    else if (t.type[i] == kGradFp16) clip_chunk((const _Float16*)t.in[i] + first, (_Float16*)t.out[i] + first, n, coef);
    else clip_chunk((const __bf16*)t.in[i] + first, (__bf16*)t.out[i] + first, n, coef);
  });
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
