// Gradient of silu(gate) * up with respect to both, elementwise:
//   s = sigmoid(g):   grad_gate = d * u * s * (1 + g * (1 - s)),   grad_up = d * g * s
// in fp32.  Two roundings to the tensors' type are choices: the projections as the forward pass stored them (in 32 bits they would be twice the
// memory that a training step keeps, 4 bytes more an element written there and read here), and the gradient itself, whose two products take their
// operands in that type (as two parts of 16 bits it would double them).  They cost a gradient's norm 3.0e-3 instead of 1.7e-3 in bf16, 3.7e-4 instead of
// 2.1e-4 in fp16.  Bound by memory: 10 bytes an element of the output.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "expert_mm.h"

namespace esmoe {

typedef int v4i __attribute__((ext_vector_type(4)));

template <bool FP16>
__device__ __forceinline__ float grad_in(uint32_t bits) {
  if constexpr (FP16) return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  else return __builtin_bit_cast(float, bits << 16);
}
template <bool FP16>
__device__ __forceinline__ uint32_t grad_out(float v) {
  if constexpr (FP16) return __builtin_bit_cast(uint16_t, (_Float16)v);
  else return __builtin_bit_cast(uint16_t, (__bf16)v);
}

// Eight columns a thread; `gate_up` and `grad` may be the same tensor: a thread reads what it writes.
template <bool FP16>
__global__ void __launch_bounds__(256) swiglu_grad_kernel(const uint16_t* __restrict__ grad_h, const uint16_t* gate_up, long pieces,
                                                          int per_row, uint16_t* grad) {
  const long piece = (long)blockIdx.x * 256 + threadIdx.x;
  if (piece >= pieces) return;
  const long row = piece / per_row, col = (piece - row * per_row) * 8, inter = (long)per_row * 8;
  const v4i d4 = *(const v4i*)(grad_h + row * inter + col);
  const v4i g4 = *(const v4i*)(gate_up + row * 2 * inter + col), u4 = *(const v4i*)(gate_up + (row * 2 + 1) * inter + col);
  v4i og, ou;
  // Rare values that a thread does its eight again for, in 64 bits: in bf16 a product d * u that leaves fp32 next to a slope that brings it back; in fp16
  // a projection that was stored as infinite, a finite sum beyond 65504.  It counts as the largest number: what is not zero beside it gets infinite,
  // but zeros stay zeros.
  float far = 0;
  auto each = [&](auto wide) {
    constexpr bool kWide = decltype(wide)::value;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      uint32_t a[2], b[2];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const float d = grad_in<FP16>((uint32_t)d4[i] >> (16 * j) & 0xffffu), g0 = grad_in<FP16>((uint32_t)g4[i] >> (16 * j) & 0xffffu),
                    u0 = grad_in<FP16>((uint32_t)u4[i] >> (16 * j) & 0xffffu);
        auto held = [](float v) { return FP16 && kWide && __builtin_fabsf(v) == __builtin_inff() ? __builtin_copysignf(0x1.fffffep127f, v) : v; };
        const float g = held(g0), u = held(u0);
        // (1 - s as a sigmoid of its own: the difference cancels)
        const float e = __builtin_amdgcn_exp2f(g * -1.44269504088896340736f);   // exp(-g), up to infinity
        const float s = __builtin_amdgcn_rcpf(1.0f + e);
        const float rest = e < __builtin_inff() ? e * s : 1.0f;
        const float slope = s * __builtin_fmaf(g, rest, 1.0f);
        if constexpr (kWide) {
          a[j] = grad_out<FP16>((float)((double)d * (double)u * (double)slope));
        } else {
          const float du = d * u;
          far = __builtin_fmaxf(far, FP16 ? __builtin_fmaxf(__builtin_fabsf(g), __builtin_fabsf(u)) : __builtin_fabsf(du));
          a[j] = grad_out<FP16>(du * slope);
        }
        b[j] = grad_out<FP16>(d * (g * s));
      }
      og[i] = (int)(a[0] | a[1] << 16);
      ou[i] = (int)(b[0] | b[1] << 16);
    }
  };
  each(std::false_type());
  if (far == __builtin_inff()) each(std::true_type());
  *(v4i*)(grad + row * 2 * inter + col) = og;
  *(v4i*)(grad + (row * 2 + 1) * inter + col) = ou;
}

}  // namespace esmoe

extern "C" int esmoe_launch_swiglu_grad(const void* grad_h, const void* gate_up, int fp16, long rows, int inter, void* grad, hipStream_t stream) {
  using namespace esmoe;
  const int per_row = inter / 8;
  const long step = (1L << 30) / per_row;   // rows of a launch: a grid holds fewer than 2^32 threads
  for (long r = 0; r < rows; r += step) {
    const long n = rows - r < step ? rows - r : step, pieces = n * per_row;
    hipLaunchKernelGGL(fp16 ? swiglu_grad_kernel<true> : swiglu_grad_kernel<false>, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, stream,
                       (const uint16_t*)grad_h + r * inter, (const uint16_t*)gate_up + r * 2 * inter, pieces, per_row,
                       (uint16_t*)grad + r * 2 * inter);
  }
  return (int)hipGetLastError();
}
