// A launch's share of the gradients that a norm is taken over (grad_norm.hip): passed by value, so that a captured graph holds it.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace esmoe {

enum { kGradBf16 = 0, kGradFp16 = 1, kGradFp32 = 2 };
constexpr int kGradTensors = 96;       // of a launch: the table has to fit in a kernel's arguments (4 KB)
constexpr long kGradChunk = 8192;      // elements
constexpr int kGradWorkgroups = 2048;  // that a call's chunks are dealt to, and one more per launch at most

constexpr long kGradStream = 512L << 20;

struct GradTable {
  const void* in[kGradTensors];
  void* out[kGradTensors];             // clipping alone
  long size[kGradTensors];             // elements
  long end[kGradTensors];              // chunks up to and with the tensor's
  int type[kGradTensors];
  int count;
  int stream;                          // all gradients of the call are more than kGradStream bytes
};
static_assert(sizeof(GradTable) <= 3600, "kernel arguments");

}  // namespace esmoe

extern "C" int esmoe_launch_grad_squares(const esmoe::GradTable* t, int grid, double* partial, hipStream_t stream);
extern "C" int esmoe_launch_grad_norm(const double* partial, int count, const float* given, float* norm, hipStream_t stream);
extern "C" int esmoe_launch_grad_clip(const esmoe::GradTable* t, int grid, const double* partial, int count, const float* given, double max_norm,
                                      double eps, float* norm_out, hipStream_t stream);
