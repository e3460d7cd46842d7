// What the entry points hand to the 16-bit and int8 grouped products (expert_mm.hip) and to the kernels beside them.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace esmoe {

constexpr int kMmExperts = 1024;   // at most (ESMOE_MAX_EXPERTS)
enum { kMmBf16 = 0, kMmFp16 = 1, kMmInt8 = 2 };

// out[m, j] = sum_c t[m, c] * w_e(j, c) for the rows m of expert e.
//   forward:        t = a [rows, k], w_e = b[e] [n, k] along its rows, out [rows, n]
//   rows' gradient: t = grad_out [rows, n], w_e = b[e] [n, k] along its columns, out = grad_a [rows, k]
// weights' gradient: out[e][i, j] = sum over the rows m of expert e of t[m, i] * w[m, j], t = grad_out [rows, n], w = a [rows, k], out [E, n, k]
struct ExpertMmArgs {
  const void *t, *w;
  void* out;
  void* gate_up;              // SwiGLU: the two projections as well, or null
  const float *sa, *sb;       // int8: scales of rows and of weight rows [E, n]
  const int *problem_sizes, *expert_offsets;
  int num_experts, total_rows, n, k;
  int type;                   // of t and w
  int out_fp16;               // int8: type of out
};

}  // namespace esmoe

// kind: 0 forward, 1 forward with SwiGLU, 2 gradient of the rows, 3 gradient of the weights
extern "C" int esmoe_launch_expert_mm(const esmoe::ExpertMmArgs* args, int kind, int cus, hipStream_t stream);
extern "C" int esmoe_launch_swiglu_grad(const void* grad_h, const void* gate_up, int fp16, long rows, int inter, void* grad, hipStream_t stream);
extern "C" int esmoe_launch_int8_quant(const void* in, int fp16, long rows, int k, void* q, float* scales, hipStream_t stream);
