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

// Whether weight rows are whole lines of 128 bytes and all of them more than the memory-side cache holds: a stream.
inline bool expert_mm_whole_lines(const ExpertMmArgs& g) {
  const long row = (long)g.k * (g.type == kMmInt8 ? 1 : 2);
  return row % 128 == 0 && (uintptr_t)g.w % 128 == 0 && row * g.n * g.num_experts > (256L << 20);
}

// A workgroup's place among those that share `total` items, round by round.  Workgroups go to the eight XCDs in turn: neighbours are on one, and where
// there are fewer items than workgroups (the launch knows an upper bound alone) every XCD has as many.
struct MmPlace {
  uint32_t place, of;   // place >= total: nothing to do
};
__device__ __forceinline__ MmPlace mm_place(uint32_t total) {
  if (gridDim.x % 8) return {blockIdx.x, gridDim.x};
  const uint32_t each = (total < gridDim.x ? total + 7 : gridDim.x) / 8, at = blockIdx.x >> 3;
  return {at < each ? (blockIdx.x & 7) * each + at : total, 8 * each};
}

}  // namespace esmoe

// kind: 0 forward, 1 forward with SwiGLU, 2 gradient of the rows, 3 gradient of the weights
extern "C" int esmoe_launch_expert_mm(const esmoe::ExpertMmArgs* args, int kind, int cus, hipStream_t stream);
extern "C" int esmoe_launch_expert_mm_few(const esmoe::ExpertMmArgs* args, int kind, int cus, hipStream_t stream);
extern "C" int esmoe_launch_swiglu_grad(const void* grad_h, const void* gate_up, int fp16, long rows, int inter, void* grad, hipStream_t stream);
extern "C" int esmoe_launch_int8_quant(const void* in, int fp16, long rows, int k, void* q, float* scales, hipStream_t stream);
