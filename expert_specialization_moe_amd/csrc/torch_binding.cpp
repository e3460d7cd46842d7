// PyTorch-ROCm operator registration for the three expert_specialization ops.
//
// Same library name, schemas and dispatch key as the reference
// (expert_specialization/csrc/expert_specialization.cpp:56-73); the argument
// checks mirror its TORCH_CHECKs (es_fp8_blockwise.cu:47-56,
// es_sm100_mxfp8_blockscaled.cu:15-25, es_sm100_mxfp8_blockscaled_group_quant.cu:13-24,
// es_fp8_blockwise_launcher.cuh:53).  Everything below the checks is the C ABI of
// libesmoe.so (include/esmoe.h): this file only unwraps tensors.
//
// Validation is also registered for CPU tensors so that it can be exercised on a
// machine without a GPU; after the checks pass a CPU call fails loudly, there is
// no CPU implementation of the ops.
#include <Python.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPStream.h>
#include <torch/all.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <vector>

#include "esmoe.h"

extern "C" {
// Empty module so that `import ..._C` loads this library and runs the static
// registrations below (same device as the reference, expert_specialization.cpp:4-21).
PyObject* PyInit__C(void) {
  static struct PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_C", NULL, -1, NULL};
  return PyModule_Create(&module_def);
}
}

namespace {

void* current_stream(const torch::Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

void require_device(const torch::Tensor& t, const char* op) {
  TORCH_CHECK(t.is_cuda(), op, ": tensors must live on a HIP device (MI355X); there is no CPU implementation");
}

void check_rc(int rc, const char* op) { TORCH_CHECK(rc == 0, op, " failed (", rc, "): ", esmoe_last_error()); }

int out_dtype_of(const torch::Tensor& t) { return t.scalar_type() == torch::kBFloat16 ? ESMOE_OUT_BF16 : ESMOE_OUT_FP16; }

// Scratch for the device-built schedule: the operators pass no workspace to the library, which then uses its own
// workspace of the current stream (zeroed once, left clean by every launch) and needs one launch per call instead of
// two.  The `workspace` tensor of the reference's signature is accepted and not used: its contents are the caller's,
// and a schedule built in it would need a kernel of its own in front of the GEMM to clear the counters.
}  // namespace

void es_fp8_blockwise_scaled_grouped_mm(torch::Tensor& output, const torch::Tensor& a, const torch::Tensor& b,
                                        const torch::Tensor& scales_a, const torch::Tensor& scales_b,
                                        const torch::Tensor& stride_a, const torch::Tensor& stride_b,
                                        const torch::Tensor& stride_d, const torch::Tensor& problem_sizes,
                                        const torch::Tensor& expert_offsets, const torch::Tensor& workspace) {
  TORCH_CHECK(problem_sizes.dim() == 2, "problem_sizes must be 2D tensor");
  TORCH_CHECK(problem_sizes.size(1) == 3, "problem_sizes must have shape (num_experts, 3)");
  TORCH_CHECK(problem_sizes.size(0) == expert_offsets.size(0),
              "Number of experts in problem_sizes must match expert_offsets");
  TORCH_CHECK(problem_sizes.dtype() == torch::kInt32, "problem_sizes must be int32");
  TORCH_CHECK(expert_offsets.dtype() == torch::kInt32, "expert_offsets must be int32");
  TORCH_CHECK(a.scalar_type() == torch::kFloat8_e4m3fn, "a must be kFloat8_e4m3fn");
  TORCH_CHECK(b.scalar_type() == torch::kFloat8_e4m3fn, "b must be kFloat8_e4m3fn");
  TORCH_CHECK(output.scalar_type() == torch::kBFloat16 || output.scalar_type() == torch::kHalf,
              "output must be bfloat16 or half");
  const int64_t num_experts = problem_sizes.size(0);
  TORCH_CHECK(num_experts >= 1 && num_experts <= ESMOE_MAX_EXPERTS, "Number of experts cannot exceed 1024");
  // Layout contract (the reference only ever dereferences data_ptr(), so the views below are the
  // ones its callers build: test/test_es_grouped_gemm.py:145-170).
  TORCH_CHECK(a.dim() == 2 && a.stride(1) == 1 && a.stride(0) == a.size(1), "a must be a packed row-major (rows, k) tensor");
  TORCH_CHECK(b.dim() == 3 && b.size(0) == num_experts, "b must be a (num_experts, k, n) tensor");
  TORCH_CHECK(b.stride(1) == 1 && b.stride(2) == b.size(1) && b.stride(0) == b.size(1) * b.size(2),
              "b must be the column-major (num_experts, k, n) view of a packed (num_experts, n, k) tensor");
  const int64_t total_rows = a.size(0), k = a.size(1), n = b.size(2);
  TORCH_CHECK(b.size(1) == k, "a and b disagree on k");
  TORCH_CHECK(k % 128 == 0 && n % 128 == 0, "n and k must be multiples of 128");
  TORCH_CHECK(output.dim() == 2 && output.size(0) == total_rows && output.size(1) == n && output.is_contiguous(),
              "output must be a contiguous (rows, n) tensor");
  TORCH_CHECK(scales_a.scalar_type() == torch::kFloat32 && scales_b.scalar_type() == torch::kFloat32,
              "scales must be float32");
  TORCH_CHECK(scales_a.dim() == 2 && scales_a.size(0) == total_rows && scales_a.size(1) == k / 128 &&
                  scales_a.is_contiguous(),
              "scales_a must be a contiguous (rows, k/128) tensor");
  TORCH_CHECK(scales_b.dim() == 3 && scales_b.size(0) == num_experts && scales_b.size(1) == k / 128 &&
                  scales_b.size(2) == n / 128 && scales_b.stride(1) == 1 &&
                  (scales_b.size(2) == 1 || scales_b.stride(2) == k / 128),
              "scales_b must be the (num_experts, k/128, n/128) view of a packed (num_experts, n/128, k/128) tensor");
  for (const torch::Tensor* s : {&stride_a, &stride_b, &stride_d}) {
    TORCH_CHECK(s->dim() == 1 && s->size(0) == num_experts, "stride tensors must have one entry per expert");
  }
  TORCH_CHECK(total_rows < (int64_t(1) << 31) && n < (int64_t(1) << 31) && k < (int64_t(1) << 31), "tensor too large");

  require_device(a, "es_fp8_blockwise_scaled_grouped_mm");
  for (const torch::Tensor* t :
       {(const torch::Tensor*)&output, &b, &scales_a, &scales_b, &problem_sizes, &expert_offsets}) {
    TORCH_CHECK(t->device() == a.device(), "all tensors must be on the same device");
  }
  TORCH_CHECK(problem_sizes.is_contiguous() && expert_offsets.is_contiguous(), "metadata tensors must be contiguous");
  if (total_rows == 0) return;
  c10::DeviceGuard guard(a.device());
  int rc = esmoe_fp8_blockwise_grouped_mm(
      output.data_ptr(), out_dtype_of(output), a.data_ptr(), b.data_ptr(), scales_a.data_ptr<float>(),
      scales_b.data_ptr<float>(), problem_sizes.data_ptr<int32_t>(), expert_offsets.data_ptr<int32_t>(),
      (int)num_experts, (int)total_rows, (int)n, (int)k, /*force_bm=*/0, /*workspace=*/nullptr, 0, current_stream(a));
  check_rc(rc, "es_fp8_blockwise_scaled_grouped_mm");
}

// The gate_up projection with SwiGLU and 1x128 re-quantisation fused into its epilogue (no counterpart in the
// reference).  Operand layouts as es_fp8_blockwise_scaled_grouped_mm with n = 2 * inter; `mid_dtype_bf16` selects the
// type the projection and the activation are rounded to on the way (true: bfloat16, false: half).
void es_fp8_blockwise_scaled_grouped_mm_swiglu_quant(torch::Tensor& quant_output, torch::Tensor& scales_out,
                                                     const torch::Tensor& a, const torch::Tensor& b,
                                                     const torch::Tensor& scales_a, const torch::Tensor& scales_b,
                                                     const torch::Tensor& problem_sizes,
                                                     const torch::Tensor& expert_offsets, const torch::Tensor& workspace,
                                                     bool mid_dtype_bf16) {
  TORCH_CHECK(problem_sizes.dim() == 2 && problem_sizes.size(1) == 3, "problem_sizes must have shape (num_experts, 3)");
  TORCH_CHECK(expert_offsets.dim() == 1 && problem_sizes.size(0) == expert_offsets.size(0),
              "Number of experts in problem_sizes must match expert_offsets");
  TORCH_CHECK(problem_sizes.dtype() == torch::kInt32 && expert_offsets.dtype() == torch::kInt32,
              "problem_sizes and expert_offsets must be int32");
  TORCH_CHECK(a.scalar_type() == torch::kFloat8_e4m3fn && b.scalar_type() == torch::kFloat8_e4m3fn,
              "a and b must be kFloat8_e4m3fn");
  const int64_t num_experts = problem_sizes.size(0);
  TORCH_CHECK(num_experts >= 1 && num_experts <= ESMOE_MAX_EXPERTS, "Number of experts cannot exceed 1024");
  TORCH_CHECK(a.dim() == 2 && a.stride(1) == 1 && a.stride(0) == a.size(1), "a must be a packed row-major (rows, k) tensor");
  TORCH_CHECK(b.dim() == 3 && b.size(0) == num_experts, "b must be a (num_experts, k, n) tensor");
  TORCH_CHECK(b.stride(1) == 1 && b.stride(2) == b.size(1) && b.stride(0) == b.size(1) * b.size(2),
              "b must be the column-major (num_experts, k, n) view of a packed (num_experts, n, k) tensor");
  const int64_t total_rows = a.size(0), k = a.size(1), n = b.size(2);
  TORCH_CHECK(b.size(1) == k, "a and b disagree on k");
  TORCH_CHECK(k % 128 == 0 && n % 256 == 0, "k must be a multiple of 128 and n = 2 * inter a multiple of 256");
  const int64_t inter = n / 2;
  TORCH_CHECK(quant_output.is_contiguous() && quant_output.element_size() == 1 && quant_output.numel() == total_rows * inter,
              "quant_output must be a contiguous 1-byte tensor of rows * n / 2 elements");
  TORCH_CHECK(scales_out.is_contiguous() && scales_out.scalar_type() == torch::kFloat32 &&
                  scales_out.numel() == total_rows * (inter / 128),
              "scales_out must be a contiguous float32 tensor of rows * n / 256 elements");
  TORCH_CHECK(scales_a.scalar_type() == torch::kFloat32 && scales_b.scalar_type() == torch::kFloat32,
              "scales must be float32");
  TORCH_CHECK(scales_a.dim() == 2 && scales_a.size(0) == total_rows && scales_a.size(1) == k / 128 &&
                  scales_a.is_contiguous(),
              "scales_a must be a contiguous (rows, k/128) tensor");
  TORCH_CHECK(scales_b.dim() == 3 && scales_b.size(0) == num_experts && scales_b.size(1) == k / 128 &&
                  scales_b.size(2) == n / 128 && scales_b.stride(1) == 1 && scales_b.stride(2) == k / 128,
              "scales_b must be the (num_experts, k/128, n/128) view of a packed (num_experts, n/128, k/128) tensor");
  TORCH_CHECK(total_rows < (int64_t(1) << 31) && n < (int64_t(1) << 31) && k < (int64_t(1) << 31), "tensor too large");
  require_device(a, "es_fp8_blockwise_scaled_grouped_mm_swiglu_quant");
  for (const torch::Tensor* t : {(const torch::Tensor*)&quant_output, (const torch::Tensor*)&scales_out, &b, &scales_a,
                                 &scales_b, &problem_sizes, &expert_offsets}) {
    TORCH_CHECK(t->device() == a.device(), "all tensors must be on the same device");
  }
  TORCH_CHECK(problem_sizes.is_contiguous() && expert_offsets.is_contiguous(), "metadata tensors must be contiguous");
  if (total_rows == 0) return;
  c10::DeviceGuard guard(a.device());
  int rc = esmoe_fp8_blockwise_grouped_mm_swiglu_quant(
      quant_output.data_ptr(), scales_out.data_ptr<float>(), mid_dtype_bf16 ? ESMOE_OUT_BF16 : ESMOE_OUT_FP16, a.data_ptr(),
      b.data_ptr(), scales_a.data_ptr<float>(), scales_b.data_ptr<float>(), problem_sizes.data_ptr<int32_t>(),
      expert_offsets.data_ptr<int32_t>(), (int)num_experts, (int)total_rows, (int)n, (int)k, /*force_bm=*/0, /*workspace=*/nullptr, 0, current_stream(a));
  check_rc(rc, "es_fp8_blockwise_scaled_grouped_mm_swiglu_quant");
}

void es_sm100_mxfp8_blockscaled_grouped_mm(const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& sfa,
                                           const torch::Tensor& sfb, torch::Tensor& d,
                                           const torch::Tensor& problem_sizes, const torch::Tensor& expert_offsets,
                                           const torch::Tensor& blockscale_offsets) {
  TORCH_CHECK(problem_sizes.dim() == 2, "problem_sizes must be 2D tensor");
  TORCH_CHECK(problem_sizes.size(1) == 3, "problem_sizes must have shape (num_experts, 3)");
  TORCH_CHECK(problem_sizes.size(0) == expert_offsets.size(0),
              "Number of experts in problem_sizes must match expert_offsets");
  TORCH_CHECK(problem_sizes.dtype() == torch::kInt32, "problem_sizes must be int32");
  TORCH_CHECK(a.dim() == 2, "a must be a 2D tensor of shape (num_tokens, k)");
  TORCH_CHECK(b.dim() == 3, "b must be a 3D tensor of shape (num_experts, k, n)");
  TORCH_CHECK(a.size(1) == b.size(1) && a.size(1) % 128 == 0, "k should align 128");
  TORCH_CHECK(b.size(2) % 128 == 0, "n should align 128");
  TORCH_CHECK(a.strides()[1] == 1, "a must be row major");
  TORCH_CHECK(b.strides()[1] == 1, "b must be column major");
  TORCH_CHECK(d.scalar_type() == torch::kBFloat16 || d.scalar_type() == torch::kHalf,
              "dtype must be kFloat16 or kBFloat16");
  const int64_t num_experts = problem_sizes.size(0);
  TORCH_CHECK(num_experts >= 1 && num_experts <= ESMOE_MAX_EXPERTS,
              "Number of experts cannot exceed 1024, the maximum number of threads per block.");
  // a and b are read through data_ptr() as e4m3 bytes whatever their dtype: the reference's own test
  // passes 2-byte tensors that the quant op filled with bytes
  // (test/test_es_sm100_mxfp8_blockscaled_grouped_quant.py:72-76,95-101).
  TORCH_CHECK(a.stride(0) == a.size(1), "a must be packed");
  TORCH_CHECK(b.size(0) == num_experts && b.stride(2) == b.size(1) && b.stride(0) == b.size(1) * b.size(2),
              "b must be the column-major (num_experts, k, n) view of a packed (num_experts, n, k) tensor");
  const int64_t total_rows = a.size(0), k = a.size(1), n = b.size(2);
  TORCH_CHECK(d.dim() == 2 && d.size(0) == total_rows && d.size(1) == n && d.is_contiguous(),
              "d must be a contiguous (num_tokens, n) tensor");
  TORCH_CHECK(sfa.element_size() == 1 && sfb.element_size() == 1, "scale factors must be 1-byte E8M0");
  TORCH_CHECK(sfb.numel() >= num_experts * n * (k / 32), "sfb is smaller than num_experts * n * k / 32 bytes");
  // every expert's scale rows are padded to 128, so the tensor holds at least the row total rounded up (a bound that
  // needs no look at the device-side metadata)
  TORCH_CHECK(sfa.numel() >= (total_rows + 127) / 128 * 128 * (k / 32),
              "sfa is smaller than the rows rounded up to 128 times k / 32 bytes");
  TORCH_CHECK(expert_offsets.dtype() == torch::kInt32 && blockscale_offsets.dtype() == torch::kInt32,
              "offset tensors must be int32");
  TORCH_CHECK(blockscale_offsets.dim() == 1 && blockscale_offsets.size(0) == num_experts,
              "blockscale_offsets must be 1D and have size equal to the number of experts");
  TORCH_CHECK(total_rows < (int64_t(1) << 31), "tensor too large");

  require_device(a, "es_sm100_mxfp8_blockscaled_grouped_mm");
  for (const torch::Tensor* t :
       {&b, &sfa, &sfb, (const torch::Tensor*)&d, &problem_sizes, &expert_offsets, &blockscale_offsets}) {
    TORCH_CHECK(t->device() == a.device(), "all tensors must be on the same device");
  }
  TORCH_CHECK(problem_sizes.is_contiguous() && expert_offsets.is_contiguous() && blockscale_offsets.is_contiguous(),
              "metadata tensors must be contiguous");
  if (total_rows == 0) return;
  c10::DeviceGuard guard(a.device());
  int rc = esmoe_mxfp8_grouped_mm(d.data_ptr(), out_dtype_of(d), a.data_ptr(), b.data_ptr(),
                                  (const uint8_t*)sfa.data_ptr(), (const uint8_t*)sfb.data_ptr(),
                                  problem_sizes.data_ptr<int32_t>(), expert_offsets.data_ptr<int32_t>(),
                                  blockscale_offsets.data_ptr<int32_t>(), (int)num_experts, (int)total_rows, (int)n,
                                  (int)k, /*force_bm=*/0, /*workspace=*/nullptr, 0, current_stream(a));
  check_rc(rc, "es_sm100_mxfp8_blockscaled_grouped_mm");
}

// The mxfp8 gate_up projection with SwiGLU and the 1x32 E8M0 re-quantisation fused into its epilogue (no counterpart
// in the reference).  Operand layouts as es_sm100_mxfp8_blockscaled_grouped_mm with n = 2 * inter; the outputs are what
// es_sm100_mxfp8_blockscaled_grouped_quant would write for a (rows, inter) input.
void es_mxfp8_blockscaled_grouped_mm_swiglu_quant(torch::Tensor& quant_output, torch::Tensor& scale_factor,
                                                  const torch::Tensor& a, const torch::Tensor& b,
                                                  const torch::Tensor& sfa, const torch::Tensor& sfb,
                                                  const torch::Tensor& problem_sizes, const torch::Tensor& expert_offsets,
                                                  const torch::Tensor& blockscale_offsets, bool mid_dtype_bf16) {
  TORCH_CHECK(problem_sizes.dim() == 2 && problem_sizes.size(1) == 3, "problem_sizes must have shape (num_experts, 3)");
  const int64_t num_experts = problem_sizes.size(0);
  TORCH_CHECK(expert_offsets.dim() == 1 && expert_offsets.size(0) == num_experts && blockscale_offsets.dim() == 1 &&
                  blockscale_offsets.size(0) == num_experts,
              "expert_offsets and blockscale_offsets must be 1D and have size equal to the number of experts");
  TORCH_CHECK(problem_sizes.dtype() == torch::kInt32 && expert_offsets.dtype() == torch::kInt32 &&
                  blockscale_offsets.dtype() == torch::kInt32,
              "problem_sizes, expert_offsets and blockscale_offsets must be int32");
  TORCH_CHECK(num_experts >= 1 && num_experts <= ESMOE_MAX_EXPERTS, "Number of experts cannot exceed 1024");
  TORCH_CHECK(a.dim() == 2 && a.stride(1) == 1 && a.stride(0) == a.size(1), "a must be a packed row-major (rows, k) tensor");
  TORCH_CHECK(b.dim() == 3 && b.size(0) == num_experts, "b must be a (num_experts, k, n) tensor");
  TORCH_CHECK(b.stride(1) == 1 && b.stride(2) == b.size(1) && b.stride(0) == b.size(1) * b.size(2),
              "b must be the column-major (num_experts, k, n) view of a packed (num_experts, n, k) tensor");
  TORCH_CHECK(a.element_size() == 1 && b.element_size() == 1, "a and b must be 1-byte e4m3 tensors");
  const int64_t total_rows = a.size(0), k = a.size(1), n = b.size(2);
  TORCH_CHECK(b.size(1) == k, "a and b disagree on k");
  TORCH_CHECK(k % 128 == 0 && n % 256 == 0, "k must be a multiple of 128 and n = 2 * inter a multiple of 256");
  const int64_t inter = n / 2;
  TORCH_CHECK(quant_output.is_contiguous() && quant_output.element_size() == 1 && quant_output.numel() == total_rows * inter,
              "quant_output must be a contiguous 1-byte tensor of rows * n / 2 elements");
  TORCH_CHECK(scale_factor.is_contiguous() && scale_factor.element_size() == 1,
              "scale_factor must be a contiguous 1-byte tensor");
  const int64_t sf_rows = (scale_factor.numel() / (inter / 32)) / 128 * 128;
  TORCH_CHECK(sf_rows >= (total_rows + 127) / 128 * 128,
              "scale_factor is smaller than the rows rounded up to 128 times n / 64 bytes");
  TORCH_CHECK(sfa.element_size() == 1 && sfb.element_size() == 1, "scale factors must be 1-byte E8M0");
  TORCH_CHECK(sfb.numel() >= num_experts * n * (k / 32), "sfb is smaller than num_experts * n * k / 32 bytes");
  TORCH_CHECK(sfa.numel() >= (total_rows + 127) / 128 * 128 * (k / 32),
              "sfa is smaller than the rows rounded up to 128 times k / 32 bytes");
  TORCH_CHECK(total_rows < (int64_t(1) << 31) && sf_rows < (int64_t(1) << 31) && n < (int64_t(1) << 31) &&
                  k < (int64_t(1) << 31),
              "tensor too large");
  require_device(a, "es_mxfp8_blockscaled_grouped_mm_swiglu_quant");
  for (const torch::Tensor* t : {(const torch::Tensor*)&quant_output, (const torch::Tensor*)&scale_factor, &b, &sfa, &sfb,
                                 &problem_sizes, &expert_offsets, &blockscale_offsets}) {
    TORCH_CHECK(t->device() == a.device(), "all tensors must be on the same device");
  }
  TORCH_CHECK(problem_sizes.is_contiguous() && expert_offsets.is_contiguous() && blockscale_offsets.is_contiguous(),
              "metadata tensors must be contiguous");
  if (total_rows == 0) return;
  c10::DeviceGuard guard(a.device());
  int rc = esmoe_mxfp8_grouped_mm_swiglu_quant(
      quant_output.data_ptr(), (uint8_t*)scale_factor.data_ptr(), mid_dtype_bf16 ? ESMOE_OUT_BF16 : ESMOE_OUT_FP16,
      a.data_ptr(), b.data_ptr(), (const uint8_t*)sfa.data_ptr(), (const uint8_t*)sfb.data_ptr(),
      problem_sizes.data_ptr<int32_t>(), expert_offsets.data_ptr<int32_t>(), blockscale_offsets.data_ptr<int32_t>(),
      (int)num_experts, (int)total_rows, (int)sf_rows, (int)n, (int)k, /*force_bm=*/0, /*workspace=*/nullptr, 0,
      current_stream(a));
  check_rc(rc, "es_mxfp8_blockscaled_grouped_mm_swiglu_quant");
}

void es_sm100_mxfp8_blockscaled_grouped_quant(const torch::Tensor& input, const torch::Tensor& problem_sizes,
                                              const torch::Tensor& expert_offsets,
                                              const torch::Tensor& blockscale_offsets, torch::Tensor& quant_output,
                                              torch::Tensor& scale_factor) {
  TORCH_CHECK(input.dim() == 2, "input must be 2D tensor");
  TORCH_CHECK(input.size(1) % 128 == 0, "k must align to 128");
  TORCH_CHECK(input.strides()[1] == 1, "input must be row major");
  TORCH_CHECK(problem_sizes.dim() == 2, "problem_sizes must be 2D tensor");
  const int64_t groups = problem_sizes.size(0);
  TORCH_CHECK(expert_offsets.dim() == 1 && expert_offsets.size(0) == groups,
              "expert_offsets must be 1D and have size equal to the number of groups");
  TORCH_CHECK(blockscale_offsets.dim() == 1 && blockscale_offsets.size(0) == groups,
              "blockscale_offsets must be 1D and have size equal to the number of groups");
  TORCH_CHECK(input.scalar_type() == torch::kBFloat16 || input.scalar_type() == torch::kHalf,
              "dtype must be kFloat16 or kBFloat16");
  TORCH_CHECK(problem_sizes.size(1) == 3 && problem_sizes.dtype() == torch::kInt32 &&
                  expert_offsets.dtype() == torch::kInt32 && blockscale_offsets.dtype() == torch::kInt32,
              "problem_sizes (groups, 3), expert_offsets and blockscale_offsets must be int32");
  TORCH_CHECK(groups >= 1 && groups <= ESMOE_MAX_EXPERTS, "number of groups must be in [1, 1024]");
  TORCH_CHECK(input.stride(0) == input.size(1), "input must be packed");
  const int64_t total_rows = input.size(0), k = input.size(1);
  // The reference's test hands over zeros_like(input) (2-byte elements) and lets the kernel write
  // bytes into it (test/test_es_sm100_mxfp8_blockscaled_grouped_quant.py:72); any contiguous
  // tensor with room for rows*k bytes is accepted.
  TORCH_CHECK(quant_output.is_contiguous() && (int64_t)quant_output.nbytes() >= total_rows * k,
              "quant_output must be contiguous and hold at least rows * k bytes");
  TORCH_CHECK(scale_factor.is_contiguous() && scale_factor.element_size() == 1,
              "scale_factor must be a contiguous 1-byte tensor");
  const int64_t sf_rows = (scale_factor.numel() / (k / 32)) / 128 * 128;
  TORCH_CHECK(sf_rows >= (total_rows + 127) / 128 * 128,
              "scale_factor is smaller than the rows rounded up to 128 times k / 32 bytes");
  TORCH_CHECK(total_rows < (int64_t(1) << 31) && sf_rows < (int64_t(1) << 31), "tensor too large");

  require_device(input, "es_sm100_mxfp8_blockscaled_grouped_quant");
  for (const torch::Tensor* t : {&problem_sizes, &expert_offsets, &blockscale_offsets, (const torch::Tensor*)&quant_output,
                                 (const torch::Tensor*)&scale_factor}) {
    TORCH_CHECK(t->device() == input.device(), "all tensors must be on the same device");
  }
  TORCH_CHECK(problem_sizes.is_contiguous() && expert_offsets.is_contiguous() && blockscale_offsets.is_contiguous(),
              "metadata tensors must be contiguous");
  if (total_rows == 0) return;
  c10::DeviceGuard guard(input.device());
  int rc = esmoe_mxfp8_grouped_quant(
      input.data_ptr(), input.scalar_type() == torch::kBFloat16 ? ESMOE_IN_BF16 : ESMOE_IN_FP16,
      problem_sizes.data_ptr<int32_t>(), expert_offsets.data_ptr<int32_t>(), blockscale_offsets.data_ptr<int32_t>(),
      quant_output.data_ptr(), (uint8_t*)scale_factor.data_ptr(), (int)groups, (int)total_rows, (int)sf_rows, (int)k,
      current_stream(input));
  check_rc(rc, "es_sm100_mxfp8_blockscaled_grouped_quant");
}

// Extension beyond the reference's three operators: the 1x128 activation quantiser its callers run in
// torch (per_token_cast_to_fp8, test/test_es_grouped_gemm.py:36-44), as a device operator.
void es_fp8_quant_act_1x128(const torch::Tensor& input, torch::Tensor& quant_output, torch::Tensor& scales) {
  TORCH_CHECK(input.dim() == 2, "input must be 2D tensor");
  TORCH_CHECK(input.size(1) % 128 == 0, "k must align to 128");
  TORCH_CHECK(input.scalar_type() == torch::kBFloat16 || input.scalar_type() == torch::kHalf,
              "dtype must be kFloat16 or kBFloat16");
  TORCH_CHECK(input.is_contiguous(), "input must be packed row major");
  const int64_t total_rows = input.size(0), k = input.size(1);
  TORCH_CHECK(quant_output.is_contiguous() && quant_output.element_size() == 1 && quant_output.numel() == total_rows * k,
              "quant_output must be a contiguous 1-byte tensor of rows * k elements");
  TORCH_CHECK(scales.is_contiguous() && scales.scalar_type() == torch::kFloat32 && scales.numel() == total_rows * (k / 128),
              "scales must be a contiguous float32 tensor of rows * k / 128 elements");
  require_device(input, "es_fp8_quant_act_1x128");
  TORCH_CHECK(quant_output.device() == input.device() && scales.device() == input.device(),
              "all tensors must be on the same device");
  if (total_rows == 0) return;
  c10::DeviceGuard guard(input.device());
  int rc = esmoe_fp8_quant_act_1x128(input.data_ptr(), input.scalar_type() == torch::kBFloat16 ? ESMOE_IN_BF16 : ESMOE_IN_FP16,
                                     quant_output.data_ptr(), scales.data_ptr<float>(), (long)total_rows, (int)k,
                                     current_stream(input));
  check_rc(rc, "es_fp8_quant_act_1x128");
}

// Fused SwiGLU + 1x128 quantisation (no counterpart in the reference).
void es_swiglu_quant_1x128(const torch::Tensor& input, torch::Tensor& quant_output, torch::Tensor& scales) {
  TORCH_CHECK(input.dim() == 2 && input.is_contiguous(), "input must be a contiguous 2D tensor");
  TORCH_CHECK(input.size(1) % 256 == 0, "the row length must be 2 * inter with inter aligned to 128");
  TORCH_CHECK(input.scalar_type() == torch::kBFloat16 || input.scalar_type() == torch::kHalf,
              "dtype must be kFloat16 or kBFloat16");
  const int64_t rows = input.size(0), inter = input.size(1) / 2;
  TORCH_CHECK(quant_output.is_contiguous() && quant_output.element_size() == 1 && quant_output.numel() == rows * inter,
              "quant_output must be a contiguous 1-byte tensor of rows * inter elements");
  TORCH_CHECK(scales.is_contiguous() && scales.scalar_type() == torch::kFloat32 && scales.numel() == rows * (inter / 128),
              "scales must be a contiguous float32 tensor of rows * inter / 128 elements");
  require_device(input, "es_swiglu_quant_1x128");
  TORCH_CHECK(quant_output.device() == input.device() && scales.device() == input.device(),
              "all tensors must be on the same device");
  if (rows == 0) return;
  c10::DeviceGuard guard(input.device());
  int rc = esmoe_swiglu_quant_1x128(input.data_ptr(), input.scalar_type() == torch::kBFloat16 ? ESMOE_IN_BF16 : ESMOE_IN_FP16,
                                    quant_output.data_ptr(), scales.data_ptr<float>(), (long)rows, (int)inter,
                                    current_stream(input));
  check_rc(rc, "es_swiglu_quant_1x128");
}

// Routing metadata and row packing on the device (no counterpart among the reference's operators; its
// callers build these tensors on the host, benchmark/benchmark_es_fp8_blockwise_moe.py:44-56,72-88).
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> es_route_metadata(const torch::Tensor& topk_ids,
                                                                                         int64_t first_expert,
                                                                                         int64_t num_experts, int64_t n,
                                                                                         int64_t k) {
  TORCH_CHECK(topk_ids.scalar_type() == torch::kInt32 && topk_ids.is_contiguous(), "topk_ids must be contiguous int32");
  TORCH_CHECK(num_experts >= 1 && num_experts <= ESMOE_MAX_EXPERTS, "num_experts must be in [1, 1024]");
  require_device(topk_ids, "es_route_metadata");
  c10::DeviceGuard guard(topk_ids.device());
  const int64_t pairs = topk_ids.numel();
  auto opts = topk_ids.options();
  torch::Tensor ps = torch::empty({num_experts, 3}, opts), eo = torch::empty({num_experts + 1}, opts),
                bso = torch::empty({num_experts + 1}, opts), dst = torch::empty({pairs}, opts);
  torch::Tensor ws = torch::empty({(int64_t)esmoe_route_workspace_bytes((long)pairs, (int)num_experts)},
                                  opts.dtype(torch::kUInt8));
  int rc = esmoe_route_metadata(pairs ? topk_ids.data_ptr<int32_t>() : nullptr, (long)pairs, (int)first_expert,
                                (int)num_experts, (int)n, (int)k, ps.data_ptr<int32_t>(), eo.data_ptr<int32_t>(),
                                bso.data_ptr<int32_t>(), pairs ? dst.data_ptr<int32_t>() : nullptr, ws.data_ptr(),
                                ws.nbytes(), current_stream(topk_ids));
  check_rc(rc, "es_route_metadata");
  return {ps, eo, bso, dst};
}

void es_permute_rows(const torch::Tensor& input, const torch::Tensor& dst_row, int64_t topk, torch::Tensor& output) {
  TORCH_CHECK(input.dim() == 2 && output.dim() == 2 && input.is_contiguous() && output.is_contiguous(),
              "input and output must be contiguous 2D tensors");
  TORCH_CHECK(input.size(1) == output.size(1) && input.scalar_type() == output.scalar_type(),
              "input and output must have the same row length and dtype");
  TORCH_CHECK(dst_row.scalar_type() == torch::kInt32 && dst_row.is_contiguous(), "dst_row must be contiguous int32");
  TORCH_CHECK(topk >= 1 && dst_row.numel() == input.size(0) * topk, "dst_row must have rows * topk entries");
  const int64_t row_bytes = input.size(1) * input.element_size();
  TORCH_CHECK(row_bytes % 16 == 0, "rows must be a multiple of 16 bytes");
  require_device(input, "es_permute_rows");
  TORCH_CHECK(dst_row.device() == input.device() && output.device() == input.device(),
              "all tensors must be on the same device");
  if (dst_row.numel() == 0) return;
  c10::DeviceGuard guard(input.device());
  int rc = esmoe_permute_rows(input.data_ptr(), dst_row.data_ptr<int32_t>(), (long)dst_row.numel(), (int)topk,
                              (long)row_bytes, output.data_ptr(), current_stream(input));
  check_rc(rc, "es_permute_rows");
}

// Weight-side companion of es_fp8_quant_act_1x128: per_block_cast_to_fp8
// (test/test_es_grouped_gemm.py:47-59) on the physical [..., N, K] weight tensor.
void es_fp8_quant_weight_128x128(const torch::Tensor& input, torch::Tensor& quant_output, torch::Tensor& scales) {
  TORCH_CHECK(input.dim() >= 2, "input must have at least 2 dimensions");
  const int64_t k = input.size(-1), n = input.size(-2);
  TORCH_CHECK(k % 128 == 0 && n % 128 == 0, "n and k must align to 128");
  TORCH_CHECK(input.scalar_type() == torch::kBFloat16 || input.scalar_type() == torch::kHalf,
              "dtype must be kFloat16 or kBFloat16");
  TORCH_CHECK(input.is_contiguous(), "input must be contiguous");
  const int64_t rows = input.numel() / k;
  TORCH_CHECK(quant_output.is_contiguous() && quant_output.element_size() == 1 && quant_output.numel() == rows * k,
              "quant_output must be a contiguous 1-byte tensor with the input's number of elements");
  TORCH_CHECK(scales.is_contiguous() && scales.scalar_type() == torch::kFloat32 &&
                  scales.numel() == (rows / 128) * (k / 128),
              "scales must be a contiguous float32 tensor with one element per 128x128 block");
  require_device(input, "es_fp8_quant_weight_128x128");
  TORCH_CHECK(quant_output.device() == input.device() && scales.device() == input.device(),
              "all tensors must be on the same device");
  if (rows == 0) return;
  c10::DeviceGuard guard(input.device());
  int rc = esmoe_fp8_quant_weight_128x128(input.data_ptr(),
                                          input.scalar_type() == torch::kBFloat16 ? ESMOE_IN_BF16 : ESMOE_IN_FP16,
                                          quant_output.data_ptr(), scales.data_ptr<float>(), (long)rows, (int)k,
                                          current_stream(input));
  check_rc(rc, "es_fp8_quant_weight_128x128");
}

// Fused SwiGLU + MXFP8 grouped quantisation: the gate_up output [rows, 2*inter] -> the down projection's operands
// (no counterpart in the reference; metadata and output layouts as es_sm100_mxfp8_blockscaled_grouped_quant with K = inter).
void es_swiglu_mxfp8_grouped_quant(const torch::Tensor& input, const torch::Tensor& problem_sizes,
                                   const torch::Tensor& expert_offsets, const torch::Tensor& blockscale_offsets,
                                   torch::Tensor& quant_output, torch::Tensor& scale_factor) {
  TORCH_CHECK(input.dim() == 2 && input.is_contiguous(), "input must be a contiguous 2D tensor");
  TORCH_CHECK(input.size(1) % 256 == 0, "the row length must be 2 * inter with inter aligned to 128");
  TORCH_CHECK(input.scalar_type() == torch::kBFloat16 || input.scalar_type() == torch::kHalf,
              "dtype must be kFloat16 or kBFloat16");
  TORCH_CHECK(problem_sizes.dim() == 2 && problem_sizes.size(1) == 3, "problem_sizes must be (groups, 3)");
  const int64_t groups = problem_sizes.size(0);
  TORCH_CHECK(expert_offsets.dim() == 1 && expert_offsets.size(0) == groups && blockscale_offsets.dim() == 1 &&
                  blockscale_offsets.size(0) == groups,
              "expert_offsets and blockscale_offsets must be 1D and have size equal to the number of groups");
  TORCH_CHECK(problem_sizes.dtype() == torch::kInt32 && expert_offsets.dtype() == torch::kInt32 &&
                  blockscale_offsets.dtype() == torch::kInt32,
              "problem_sizes, expert_offsets and blockscale_offsets must be int32");
  TORCH_CHECK(groups >= 1 && groups <= ESMOE_MAX_EXPERTS, "number of groups must be in [1, 1024]");
  const int64_t total_rows = input.size(0), inter = input.size(1) / 2;
  TORCH_CHECK(quant_output.is_contiguous() && (int64_t)quant_output.nbytes() >= total_rows * inter,
              "quant_output must be contiguous and hold at least rows * inter bytes");
  TORCH_CHECK(scale_factor.is_contiguous() && scale_factor.element_size() == 1,
              "scale_factor must be a contiguous 1-byte tensor");
  const int64_t sf_rows = (scale_factor.numel() / (inter / 32)) / 128 * 128;
  TORCH_CHECK(sf_rows >= (total_rows + 127) / 128 * 128,
              "scale_factor is smaller than the rows rounded up to 128 times inter / 32 bytes");
  TORCH_CHECK(total_rows < (int64_t(1) << 31) && sf_rows < (int64_t(1) << 31), "tensor too large");
  require_device(input, "es_swiglu_mxfp8_grouped_quant");
  for (const torch::Tensor* t : {&problem_sizes, &expert_offsets, &blockscale_offsets, (const torch::Tensor*)&quant_output,
                                 (const torch::Tensor*)&scale_factor}) {
    TORCH_CHECK(t->device() == input.device(), "all tensors must be on the same device");
  }
  TORCH_CHECK(problem_sizes.is_contiguous() && expert_offsets.is_contiguous() && blockscale_offsets.is_contiguous(),
              "metadata tensors must be contiguous");
  if (total_rows == 0) return;
  c10::DeviceGuard guard(input.device());
  int rc = esmoe_swiglu_mxfp8_grouped_quant(
      input.data_ptr(), input.scalar_type() == torch::kBFloat16 ? ESMOE_IN_BF16 : ESMOE_IN_FP16,
      problem_sizes.data_ptr<int32_t>(), expert_offsets.data_ptr<int32_t>(), blockscale_offsets.data_ptr<int32_t>(),
      quant_output.data_ptr(), (uint8_t*)scale_factor.data_ptr(), (int)groups, (int)total_rows, (int)sf_rows, (int)inter,
      current_stream(input));
  check_rc(rc, "es_swiglu_mxfp8_grouped_quant");
}

// MXFP8 quantisation of a weight tensor [..., N, K] (no counterpart among the reference's operators: its test
// passes the activation operator a transposed problem list, test/test_es_sm100_mxfp8_blockscaled_grouped_quant.py:87-96).
void es_mxfp8_quant_weight(const torch::Tensor& input, torch::Tensor& quant_output, torch::Tensor& scale_factor) {
  TORCH_CHECK(input.dim() >= 2, "input must have at least 2 dimensions");
  const int64_t k = input.size(-1), n = input.size(-2);
  TORCH_CHECK(k % 128 == 0 && n % 128 == 0, "n and k must align to 128");
  TORCH_CHECK(input.scalar_type() == torch::kBFloat16 || input.scalar_type() == torch::kHalf,
              "dtype must be kFloat16 or kBFloat16");
  TORCH_CHECK(input.is_contiguous(), "input must be contiguous");
  const int64_t rows = input.numel() / k;
  TORCH_CHECK(quant_output.is_contiguous() && quant_output.element_size() == 1 && quant_output.numel() == rows * k,
              "quant_output must be a contiguous 1-byte tensor with the input's number of elements");
  TORCH_CHECK(scale_factor.is_contiguous() && scale_factor.element_size() == 1 && scale_factor.numel() == rows * (k / 32),
              "scale_factor must be a contiguous 1-byte tensor of rows * k / 32 elements");
  require_device(input, "es_mxfp8_quant_weight");
  TORCH_CHECK(quant_output.device() == input.device() && scale_factor.device() == input.device(),
              "all tensors must be on the same device");
  if (rows == 0) return;
  c10::DeviceGuard guard(input.device());
  int rc = esmoe_mxfp8_quant_weight(input.data_ptr(), input.scalar_type() == torch::kBFloat16 ? ESMOE_IN_BF16 : ESMOE_IN_FP16,
                                    quant_output.data_ptr(), (uint8_t*)scale_factor.data_ptr(), (long)rows, (int)k,
                                    current_stream(input));
  check_rc(rc, "es_mxfp8_quant_weight");
}

// ---- the operators around the grouped GEMMs of a mixture-of-experts block (no counterparts in the reference) ----
namespace {

// These operators are not part of autograd: where a gradient exists it is an operator of its own, and a result that silently had
// none would train nothing.  In forward mode, which no_grad leaves on, there is none at all: no result has a tangent, and an output
// would keep one of what it held before.
void check_no_autograd(const char* op, std::initializer_list<const torch::Tensor*> inputs,
                       std::initializer_list<const torch::Tensor*> outputs = {}) {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
    for (const auto& tensors : {inputs, outputs})
      for (const torch::Tensor* t : tensors)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), op, ": not differentiable, a tensor with a tangent is refused");
  if (!at::GradMode::is_enabled()) return;
  for (const torch::Tensor* t : inputs)
    TORCH_CHECK(!t->defined() || !t->requires_grad(), op,
                ": not differentiable by autograd (call it under torch.no_grad(); gradients are operators of their own)");
  for (const torch::Tensor* t : outputs)   // (what a graph has recorded of it would be overwritten)
    TORCH_CHECK(!t->defined() || !t->requires_grad(), op, ": output that requires a gradient (write to it under torch.no_grad())");
}

void check_device(const torch::Tensor& like, std::initializer_list<const torch::Tensor*> tensors) {
  for (const torch::Tensor* t : tensors)
    TORCH_CHECK(!t->defined() || t->device() == like.device(), "all tensors must be on the same device");
}

bool is_half_type(const torch::Tensor& t) { return t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kHalf; }

int logits_dtype_of(const torch::Tensor& t) {
  return t.scalar_type() == torch::kFloat32 ? ESMOE_LOGITS_FP32 : t.scalar_type() == torch::kHalf ? ESMOE_LOGITS_FP16 : ESMOE_LOGITS_BF16;
}

void check_logits(const torch::Tensor& logits, int64_t topk) {
  TORCH_CHECK(logits.dim() == 2, "logits must be 2D tensor");
  TORCH_CHECK(logits.scalar_type() == torch::kFloat32 || is_half_type(logits), "logits must be float32, bfloat16 or half");
  const int64_t experts = logits.size(1);
  TORCH_CHECK(experts >= 1 && experts <= ESMOE_MAX_EXPERTS, "Number of experts must be in [1, 1024]");
  TORCH_CHECK(experts == 1 || logits.stride(1) == 1, "logits must be row major");
  TORCH_CHECK(topk >= 1 && topk <= ESMOE_MAX_TOPK && topk <= experts, "topk must be in [1, 64] and at most the number of experts");
  TORCH_CHECK(logits.size(0) < (int64_t(1) << 31) / topk, "tensor too large");
}

const torch::Tensor& tensor_or_none(const c10::optional<torch::Tensor>& t) {
  static const torch::Tensor none;
  return t.has_value() ? *t : none;
}

}  // namespace

std::tuple<torch::Tensor, torch::Tensor> es_topk_gating(const torch::Tensor& logits, int64_t topk, const c10::optional<torch::Tensor>& bias_,
                                                        bool sigmoid, bool renormalize, double scale, int64_t num_groups,
                                                        int64_t topk_groups) {
  const torch::Tensor& bias = tensor_or_none(bias_);
  check_logits(logits, topk);
  const int64_t tokens = logits.size(0), experts = logits.size(1);
  TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == experts && bias.scalar_type() == torch::kFloat32 && bias.is_contiguous()),
              "bias must be a contiguous float32 tensor with one element per expert");
  TORCH_CHECK(num_groups >= 1 && num_groups <= 64 && experts % num_groups == 0, "num_groups must be in [1, 64] and divide the number of experts");
  TORCH_CHECK(topk_groups >= 1 && topk_groups <= num_groups, "topk_groups must be in [1, num_groups]");
  TORCH_CHECK(topk <= experts / num_groups * topk_groups, "topk is more than the experts of topk_groups groups");
  TORCH_CHECK(std::isfinite((float)scale), "scale must be finite");
  check_no_autograd("es_topk_gating", {&logits, &bias});
  require_device(logits, "es_topk_gating");
  check_device(logits, {&bias});
  c10::DeviceGuard guard(logits.device());
  torch::Tensor ids = torch::empty({tokens, topk}, logits.options().dtype(torch::kInt32)),
                weights = torch::empty({tokens, topk}, logits.options().dtype(torch::kFloat32));
  if (tokens == 0) return {ids, weights};
  int rc = esmoe_topk_gating(logits.data_ptr(), logits_dtype_of(logits), (long)logits.stride(0), bias.defined() ? bias.data_ptr<float>() : nullptr,
                             (long)tokens, (int)experts, (int)topk, sigmoid ? ESMOE_SCORING_SIGMOID : ESMOE_SCORING_SOFTMAX, renormalize,
                             (float)scale, (int)num_groups, (int)topk_groups, ids.data_ptr<int32_t>(), weights.data_ptr<float>(),
                             current_stream(logits));
  check_rc(rc, "es_topk_gating");
  return {ids, weights};
}

torch::Tensor es_topk_gating_backward(const torch::Tensor& grad_weights, const torch::Tensor& logits, const torch::Tensor& topk_ids,
                                      bool sigmoid, bool renormalize, double scale) {
  TORCH_CHECK(topk_ids.dim() == 2 && topk_ids.scalar_type() == torch::kInt32 && topk_ids.is_contiguous(),
              "topk_ids must be a contiguous int32 (tokens, topk) tensor");
  const int64_t topk = topk_ids.size(1);
  check_logits(logits, topk);
  const int64_t tokens = logits.size(0), experts = logits.size(1);
  TORCH_CHECK(topk_ids.size(0) == tokens, "topk_ids must have a row per row of logits");
  TORCH_CHECK(grad_weights.sizes() == topk_ids.sizes() && grad_weights.scalar_type() == torch::kFloat32 && grad_weights.is_contiguous(),
              "grad_weights must be a contiguous float32 tensor of topk_ids' shape");
  TORCH_CHECK(std::isfinite((float)scale), "scale must be finite");
  check_no_autograd("es_topk_gating_backward", {&grad_weights, &logits});
  require_device(logits, "es_topk_gating_backward");
  check_device(logits, {&grad_weights, &topk_ids});
  c10::DeviceGuard guard(logits.device());
  torch::Tensor grad = torch::empty({tokens, experts}, logits.options());
  if (tokens == 0) return grad;
  int rc = esmoe_topk_gating_backward(grad_weights.data_ptr<float>(), logits.data_ptr(), logits_dtype_of(logits), (long)logits.stride(0),
                                      topk_ids.data_ptr<int32_t>(), (long)tokens, (int)experts, (int)topk,
                                      sigmoid ? ESMOE_SCORING_SIGMOID : ESMOE_SCORING_SOFTMAX, renormalize, (float)scale, grad.data_ptr(),
                                      current_stream(logits));
  check_rc(rc, "es_topk_gating_backward");
  return grad;
}

namespace {
// Checks that both directions of the combine share; returns the tokens.
int64_t check_combine(const torch::Tensor& rows, const torch::Tensor& dst_row, int64_t topk, const torch::Tensor& weights) {
  TORCH_CHECK(rows.dim() == 2 && rows.is_contiguous() && is_half_type(rows), "input must be a contiguous 2D bfloat16 or half tensor");
  TORCH_CHECK(rows.size(1) > 0 && rows.size(1) % 8 == 0, "rows must be a multiple of 16 bytes");
  TORCH_CHECK(dst_row.scalar_type() == torch::kInt32 && dst_row.is_contiguous(), "dst_row must be contiguous int32");
  TORCH_CHECK(topk >= 1 && dst_row.numel() % topk == 0, "dst_row must have tokens * topk entries");
  TORCH_CHECK(!weights.defined() || (weights.scalar_type() == torch::kFloat32 && weights.is_contiguous() && weights.numel() == dst_row.numel()),
              "weights must be a contiguous float32 tensor of dst_row's size");
  TORCH_CHECK(rows.size(0) < (int64_t(1) << 31) && rows.size(1) <= (int64_t(1) << 24) && dst_row.numel() < (int64_t(1) << 31), "tensor too large");
  return dst_row.numel() / topk;
}
bool overlap(const torch::Tensor& a, const torch::Tensor& b) {
  const char *pa = (const char*)a.data_ptr(), *pb = (const char*)b.data_ptr();
  return a.numel() && b.numel() && pa < pb + b.nbytes() && pb < pa + a.nbytes();
}
// (undefined tensors overlap nothing)
bool any_overlap(const torch::Tensor& out, std::initializer_list<const torch::Tensor*> others) {
  for (const torch::Tensor* t : others)
    if (out.defined() && t->defined() && overlap(out, *t)) return true;
  return false;
}
}  // namespace

void es_combine_rows(const torch::Tensor& input, const torch::Tensor& dst_row, int64_t topk, const c10::optional<torch::Tensor>& weights_,
                     torch::Tensor& output) {
  const torch::Tensor& weights = tensor_or_none(weights_);
  const int64_t tokens = check_combine(input, dst_row, topk, weights);
  TORCH_CHECK(output.dim() == 2 && output.is_contiguous() && output.scalar_type() == input.scalar_type() && output.size(0) == tokens &&
                  output.size(1) == input.size(1),
              "output must be a contiguous (tokens, row length) tensor of input's dtype");
  check_no_autograd("es_combine_rows", {&input, &weights}, {&output});
  require_device(input, "es_combine_rows");
  check_device(input, {&dst_row, &weights, &output});
  TORCH_CHECK(!any_overlap(output, {&input, &dst_row, &weights}), "output may not overlap input, dst_row or weights");
  if (tokens == 0) return;
  c10::DeviceGuard guard(input.device());
  int rc = esmoe_combine_rows(input.data_ptr(), input.scalar_type() == torch::kBFloat16 ? ESMOE_IN_BF16 : ESMOE_IN_FP16,
                              dst_row.data_ptr<int32_t>(), weights.defined() ? weights.data_ptr<float>() : nullptr, (long)dst_row.numel(),
                              (int)topk, (long)input.size(0), (int)input.size(1), output.data_ptr(), current_stream(input));
  check_rc(rc, "es_combine_rows");
}

// The same into a new tensor (allocated here: a tensor made in Python costs a call twice as much).
torch::Tensor es_combine_rows_new(const torch::Tensor& input, const torch::Tensor& dst_row, int64_t topk,
                                  const c10::optional<torch::Tensor>& weights) {
  const int64_t tokens = check_combine(input, dst_row, topk, tensor_or_none(weights));
  torch::Tensor output = torch::empty({tokens, input.size(1)}, input.options().requires_grad(false));
  es_combine_rows(input, dst_row, topk, weights, output);
  return output;
}

void es_combine_rows_backward(const torch::Tensor& grad_output, const torch::Tensor& input, const torch::Tensor& dst_row, int64_t topk,
                              const torch::Tensor& weights, torch::Tensor& grad_input, torch::Tensor& grad_weights) {
  const int64_t tokens = check_combine(input, dst_row, topk, weights);
  TORCH_CHECK(grad_output.dim() == 2 && grad_output.is_contiguous() && grad_output.scalar_type() == input.scalar_type() &&
                  grad_output.size(0) == tokens && grad_output.size(1) == input.size(1),
              "grad_output must be a contiguous (tokens, row length) tensor of input's dtype");
  TORCH_CHECK(grad_input.sizes() == input.sizes() && grad_input.is_contiguous() && grad_input.scalar_type() == input.scalar_type(),
              "grad_input must be a contiguous tensor of input's shape and dtype");
  TORCH_CHECK(grad_weights.scalar_type() == torch::kFloat32 && grad_weights.is_contiguous() && grad_weights.numel() == dst_row.numel(),
              "grad_weights must be a contiguous float32 tensor of dst_row's size");
  check_no_autograd("es_combine_rows_backward", {&grad_output, &input, &weights}, {&grad_input, &grad_weights});
  require_device(input, "es_combine_rows_backward");
  check_device(input, {&grad_output, &dst_row, &weights, &grad_input, &grad_weights});
  TORCH_CHECK(!any_overlap(grad_input, {&input, &grad_output, &dst_row, &weights, &grad_weights}) &&
                  !any_overlap(grad_weights, {&input, &grad_output, &dst_row, &weights}),
              "grad_input and grad_weights may not overlap each other or the inputs");
  if (tokens == 0) return;
  c10::DeviceGuard guard(input.device());
  int rc = esmoe_combine_rows_backward(grad_output.data_ptr(), input.data_ptr(),
                                       input.scalar_type() == torch::kBFloat16 ? ESMOE_IN_BF16 : ESMOE_IN_FP16, dst_row.data_ptr<int32_t>(),
                                       weights.data_ptr<float>(), (long)dst_row.numel(), (int)topk, (long)input.size(0), (int)input.size(1),
                                       grad_input.data_ptr(), grad_weights.data_ptr<float>(), current_stream(input));
  check_rc(rc, "es_combine_rows_backward");
}

void es_add_rms_norm_quant_1x128(const torch::Tensor& input, const torch::Tensor& weight, double eps,
                                 const c10::optional<torch::Tensor>& residual_, const c10::optional<torch::Tensor>& residual_out_,
                                 const c10::optional<torch::Tensor>& normed_, torch::Tensor& quant_output, torch::Tensor& scales) {
  const torch::Tensor &residual = tensor_or_none(residual_), &residual_out = tensor_or_none(residual_out_), &normed = tensor_or_none(normed_);
  TORCH_CHECK(input.dim() == 2 && input.is_contiguous(), "input must be a contiguous 2D tensor");
  TORCH_CHECK(is_half_type(input), "dtype must be kFloat16 or kBFloat16");
  const int64_t rows = input.size(0), k = input.size(1);
  TORCH_CHECK(k > 0 && k % 128 == 0 && k <= 32768, "k must align to 128 and be at most 32768");
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == k && weight.is_contiguous() && weight.scalar_type() == input.scalar_type(),
              "weight must be a contiguous tensor of k elements of input's dtype");
  TORCH_CHECK(eps >= 0 && std::isfinite((float)eps), "eps must be finite and not negative");
  TORCH_CHECK(residual.defined() == residual_out.defined(), "residual and residual_out go together");
  for (const torch::Tensor* t : {&residual, &residual_out, &normed})
    TORCH_CHECK(!t->defined() || (t->sizes() == input.sizes() && t->is_contiguous() && t->scalar_type() == input.scalar_type()),
                "residual, residual_out and normed must be contiguous tensors of input's shape and dtype");
  TORCH_CHECK(quant_output.is_contiguous() && quant_output.element_size() == 1 && quant_output.numel() == rows * k,
              "quant_output must be a contiguous 1-byte tensor of rows * k elements");
  TORCH_CHECK(scales.is_contiguous() && scales.scalar_type() == torch::kFloat32 && scales.numel() == rows * (k / 128),
              "scales must be a contiguous float32 tensor of rows * k / 128 elements");
  check_no_autograd("es_add_rms_norm_quant_1x128", {&input, &weight, &residual},
                    {&residual_out, &normed, &quant_output, &scales});
  require_device(input, "es_add_rms_norm_quant_1x128");
  check_device(input, {&weight, &residual, &residual_out, &normed, &quant_output, &scales});
  if (rows == 0) return;
  TORCH_CHECK(!any_overlap(quant_output, {&input, &residual, &weight, &scales, &normed, &residual_out}) &&
                  !any_overlap(scales, {&input, &residual, &weight, &normed, &residual_out}) &&
                  !any_overlap(normed, {&input, &residual, &weight, &residual_out}) && !any_overlap(residual_out, {&weight}),
              "outputs may not overlap inputs or each other");
  // a row is read before its new residual is written
  for (const torch::Tensor* in : {&input, &residual})
    TORCH_CHECK(!any_overlap(residual_out, {in}) || in->data_ptr() == residual_out.data_ptr(), "residual_out may be input or residual, not a part of them");
  c10::DeviceGuard guard(input.device());
  int rc = esmoe_add_rms_norm_quant_1x128(
      input.data_ptr(), input.scalar_type() == torch::kBFloat16 ? ESMOE_IN_BF16 : ESMOE_IN_FP16, residual.defined() ? residual.data_ptr() : nullptr,
      weight.data_ptr(), (float)eps, (long)rows, (int)k, residual.defined() ? residual_out.data_ptr() : nullptr,
      normed.defined() ? normed.data_ptr() : nullptr, quant_output.data_ptr(), scales.data_ptr<float>(), current_stream(input));
  check_rc(rc, "es_add_rms_norm_quant_1x128");
}

// The same into new tensors; those that are not asked for stay undefined (None in Python).
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> es_add_rms_norm_quant_1x128_new(
    const torch::Tensor& input, const torch::Tensor& weight, double eps, const c10::optional<torch::Tensor>& residual, bool return_normed) {
  TORCH_CHECK(input.dim() == 2, "input must be a contiguous 2D tensor");
  const auto opts = input.options().requires_grad(false);
  torch::Tensor q = torch::empty({input.size(0), input.size(1)}, opts.dtype(torch::kFloat8_e4m3fn)),
                scales = torch::empty({input.size(0), input.size(1) / 128}, opts.dtype(torch::kFloat32)), residual_out, normed;
  if (residual.has_value() && residual->defined()) residual_out = torch::empty(input.sizes(), opts);
  if (return_normed) normed = torch::empty(input.sizes(), opts);
  const auto given = [](const torch::Tensor& t) { return t.defined() ? c10::optional<torch::Tensor>(t) : c10::nullopt; };
  es_add_rms_norm_quant_1x128(input, weight, eps, residual, given(residual_out), given(normed), q, scales);
  return {q, scales, residual_out, normed};
}

namespace {
void mxfp4_grouped_mm(const char* op, bool swiglu, torch::Tensor& output, const torch::Tensor& a, const torch::Tensor& b,
                      const torch::Tensor& sfb, const torch::Tensor& problem_sizes, const torch::Tensor& expert_offsets) {
  TORCH_CHECK(problem_sizes.dim() == 2 && problem_sizes.size(1) == 3, "problem_sizes must have shape (num_experts, 3)");
  const int64_t num_experts = problem_sizes.size(0);
  TORCH_CHECK(expert_offsets.dim() == 1 && expert_offsets.size(0) == num_experts, "Number of experts in problem_sizes must match expert_offsets");
  TORCH_CHECK(problem_sizes.dtype() == torch::kInt32 && expert_offsets.dtype() == torch::kInt32, "problem_sizes and expert_offsets must be int32");
  TORCH_CHECK(num_experts >= 1 && num_experts <= ESMOE_MAX_EXPERTS, "Number of experts cannot exceed 1024");
  TORCH_CHECK(is_half_type(a), "a must be bfloat16 or half");
  TORCH_CHECK(a.dim() == 2 && a.is_contiguous(), "a must be a packed row-major (rows, k) tensor");
  const int64_t total_rows = a.size(0), k = a.size(1);
  TORCH_CHECK(k > 0 && k % 128 == 0 && k <= 32768, "k must be a multiple of 128 up to 32768");
  TORCH_CHECK(b.dim() == 3 && b.size(0) == num_experts && b.element_size() == 1 && b.size(1) == k / 2,
              "b must be a 1-byte (num_experts, k/2, n) tensor of two 4-bit codes each");
  const int64_t n = b.size(2);
  TORCH_CHECK(n > 0 && n % (swiglu ? 32 : 16) == 0 && n <= (int64_t(1) << 20), "n must be a multiple of 16 (of 32 with SwiGLU) up to 2^20");
  TORCH_CHECK(b.stride(1) == 1 && b.stride(2) == k / 2 && (num_experts == 1 || b.stride(0) == n * (k / 2)),
              "b must be the column-major (num_experts, k/2, n) view of a packed (num_experts, n, k/2) tensor");
  TORCH_CHECK(sfb.dim() == 3 && sfb.element_size() == 1 && sfb.size(0) == num_experts && sfb.size(1) == k / 32 && sfb.size(2) == n &&
                  sfb.stride(1) == 1 && sfb.stride(2) == k / 32 && (num_experts == 1 || sfb.stride(0) == n * (k / 32)),
              "sfb must be the 1-byte column-major (num_experts, k/32, n) view of a packed (num_experts, n, k/32) tensor");
  TORCH_CHECK(output.dim() == 2 && output.is_contiguous() && output.scalar_type() == a.scalar_type() && output.size(0) == total_rows &&
                  output.size(1) == (swiglu ? n / 2 : n),
              "output must be a contiguous (rows, n) tensor, (rows, n / 2) with SwiGLU, of a's dtype");
  TORCH_CHECK(total_rows < (int64_t(1) << 31), "tensor too large");
  check_no_autograd(op, {&a}, {&output});
  require_device(a, op);
  check_device(a, {&output, &b, &sfb, &problem_sizes, &expert_offsets});
  TORCH_CHECK(problem_sizes.is_contiguous() && expert_offsets.is_contiguous(), "metadata tensors must be contiguous");
  TORCH_CHECK(!any_overlap(output, {&a, &b, &sfb, &problem_sizes, &expert_offsets}), "output may not overlap an input");
  if (total_rows == 0) return;
  c10::DeviceGuard guard(a.device());
  int rc = esmoe_mxfp4_grouped_mm(output.data_ptr(), out_dtype_of(output), a.data_ptr(), b.data_ptr(), (const uint8_t*)sfb.data_ptr(),
                                  problem_sizes.data_ptr<int32_t>(), expert_offsets.data_ptr<int32_t>(), (int)num_experts, (int)total_rows,
                                  (int)n, (int)k, swiglu, current_stream(a));
  check_rc(rc, op);
}
}  // namespace

void es_mxfp4_grouped_mm(torch::Tensor& output, const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& sfb,
                         const torch::Tensor& problem_sizes, const torch::Tensor& expert_offsets) {
  mxfp4_grouped_mm("es_mxfp4_grouped_mm", false, output, a, b, sfb, problem_sizes, expert_offsets);
}

void es_mxfp4_grouped_mm_swiglu(torch::Tensor& output, const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& sfb,
                                const torch::Tensor& problem_sizes, const torch::Tensor& expert_offsets) {
  mxfp4_grouped_mm("es_mxfp4_grouped_mm_swiglu", true, output, a, b, sfb, problem_sizes, expert_offsets);
}

// ---- the experts' products in 16 bits with their gradients, and in 8-bit integers ----
namespace {
// A (num_experts, k, n) view of packed rows of k, and the metadata that go with it.
void check_experts(const char* op, const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& problem_sizes,
                   const torch::Tensor& expert_offsets, int64_t k_step, int64_t most_k, bool swiglu) {
  TORCH_CHECK(problem_sizes.dim() == 2 && problem_sizes.size(1) == 3, "problem_sizes must have shape (num_experts, 3)");
  const int64_t num_experts = problem_sizes.size(0);
  TORCH_CHECK(expert_offsets.dim() == 1 && expert_offsets.size(0) == num_experts, "Number of experts in problem_sizes must match expert_offsets");
  TORCH_CHECK(problem_sizes.dtype() == torch::kInt32 && expert_offsets.dtype() == torch::kInt32, "problem_sizes and expert_offsets must be int32");
  TORCH_CHECK(num_experts >= 1 && num_experts <= ESMOE_MAX_EXPERTS, "Number of experts cannot exceed 1024");
  TORCH_CHECK(a.dim() == 2 && a.is_contiguous(), "a must be a packed row-major (rows, k) tensor");
  const int64_t k = a.size(1);
  TORCH_CHECK(k > 0 && k % k_step == 0 && k <= most_k, "k must be a multiple of ", k_step, " up to ", most_k);
  TORCH_CHECK(b.dim() == 3 && b.size(0) == num_experts && b.size(1) == k && b.scalar_type() == a.scalar_type(),
              "b must be a (num_experts, k, n) tensor of a's dtype");
  const int64_t n = b.size(2);
  TORCH_CHECK(n > 0 && n % (swiglu ? 16 : 8) == 0 && n <= (int64_t(1) << 20), "n must be a multiple of 8 (of 16 with SwiGLU) up to 2^20");
  TORCH_CHECK(b.stride(1) == 1 && b.stride(2) == k && (num_experts == 1 || b.stride(0) == n * k),
              "b must be the column-major (num_experts, k, n) view of a packed (num_experts, n, k) tensor");
  TORCH_CHECK(a.size(0) < (int64_t(1) << 31), "tensor too large");
  TORCH_CHECK(problem_sizes.is_contiguous() && expert_offsets.is_contiguous(), "metadata tensors must be contiguous");
}

void check_rows(const torch::Tensor& t, const char* name, int64_t rows, int64_t cols, const torch::Tensor& like) {
  TORCH_CHECK(t.dim() == 2 && t.is_contiguous() && t.size(0) == rows && t.size(1) == cols && t.scalar_type() == like.scalar_type(), name,
              " must be a contiguous (", rows, ", ", cols, ") tensor of a's dtype");
}

// The binding's workspaces are the allocator's, on the current stream: no call waits for the device.
void grouped_mm(const char* op, bool swiglu, torch::Tensor& output, const torch::Tensor& a, const torch::Tensor& b,
                const torch::Tensor& problem_sizes, const torch::Tensor& expert_offsets, const torch::Tensor& gate_up) {
  TORCH_CHECK(is_half_type(a), "a must be bfloat16 or half");
  check_experts(op, a, b, problem_sizes, expert_offsets, 8, int64_t(1) << 20, swiglu);
  const int64_t rows = a.size(0), k = a.size(1), n = b.size(2);
  check_rows(output, "output", rows, swiglu ? n / 2 : n, a);
  if (gate_up.defined()) check_rows(gate_up, "gate_up", rows, n, a);
  check_no_autograd(op, {&a, &b}, {&output, &gate_up});
  require_device(a, op);
  check_device(a, {&output, &b, &gate_up, &problem_sizes, &expert_offsets});
  TORCH_CHECK(!any_overlap(output, {&a, &b, &gate_up, &problem_sizes, &expert_offsets}) &&
                  !any_overlap(gate_up, {&a, &b, &problem_sizes, &expert_offsets}),
              "output and gate_up may not overlap each other or an input");
  if (rows == 0) return;
  c10::DeviceGuard guard(a.device());
  int rc = esmoe_grouped_mm(output.data_ptr(), out_dtype_of(a), a.data_ptr(), b.data_ptr(), problem_sizes.data_ptr<int32_t>(),
                            expert_offsets.data_ptr<int32_t>(), (int)problem_sizes.size(0), (int)rows, (int)n, (int)k, swiglu,
                            gate_up.defined() ? gate_up.data_ptr() : nullptr, current_stream(a));
  check_rc(rc, op);
}

void grouped_mm_backward(const char* op, const torch::Tensor* gate_up, const torch::Tensor& grad_output, const torch::Tensor& a,
                         const torch::Tensor& b, const torch::Tensor& problem_sizes, const torch::Tensor& expert_offsets,
                         const torch::Tensor& grad_a, const torch::Tensor& grad_b) {
  TORCH_CHECK(is_half_type(a), "a must be bfloat16 or half");
  check_experts(op, a, b, problem_sizes, expert_offsets, 8, int64_t(1) << 20, gate_up != nullptr);
  const int64_t rows = a.size(0), k = a.size(1), n = b.size(2), experts = b.size(0);
  static const torch::Tensor none;
  const torch::Tensor& saved = gate_up ? *gate_up : none;
  check_rows(grad_output, "grad_output", rows, gate_up ? n / 2 : n, a);
  if (gate_up) check_rows(saved, "gate_up", rows, n, a);
  if (grad_a.defined()) check_rows(grad_a, "grad_a", rows, k, a);
  TORCH_CHECK(!grad_b.defined() || (grad_b.sizes() == b.sizes() && grad_b.scalar_type() == b.scalar_type() && grad_b.stride(1) == 1 &&
                                    grad_b.stride(2) == k && (experts == 1 || grad_b.stride(0) == n * k)),
              "grad_b must be the column-major (num_experts, k, n) view of a packed (num_experts, n, k) tensor of b's dtype");
  check_no_autograd(op, {&grad_output, &a, &b, &saved}, {&grad_a, &grad_b});
  require_device(a, op);
  check_device(a, {&grad_output, &b, &saved, &problem_sizes, &expert_offsets, &grad_a, &grad_b});
  TORCH_CHECK(!any_overlap(grad_a, {&grad_output, &a, &b, &saved, &problem_sizes, &expert_offsets, &grad_b}) &&
                  !any_overlap(grad_b, {&grad_output, &a, &b, &saved, &problem_sizes, &expert_offsets}),
              "grad_a and grad_b may not overlap each other or the inputs");
  c10::DeviceGuard guard(a.device());
  const int dtype = out_dtype_of(a);
  torch::Tensor grad = grad_output;
  if (gate_up && rows && (grad_a.defined() || grad_b.defined())) {
    grad = torch::empty({rows, n}, a.options().requires_grad(false));
    check_rc(esmoe_swiglu_backward(grad_output.data_ptr(), saved.data_ptr(), dtype, (long)rows, (int)(n / 2), grad.data_ptr(), current_stream(a)), op);
  }
  int rc = esmoe_grouped_mm_backward(rows ? grad.data_ptr() : nullptr, dtype, rows ? a.data_ptr() : nullptr, b.data_ptr(),
                                     problem_sizes.data_ptr<int32_t>(), expert_offsets.data_ptr<int32_t>(), (int)experts, (int)rows, (int)n,
                                     (int)k, grad_a.defined() && rows ? grad_a.data_ptr() : nullptr, grad_b.defined() ? grad_b.data_ptr() : nullptr,
                                     current_stream(a));
  check_rc(rc, op);
}
}  // namespace

void es_grouped_mm(torch::Tensor& output, const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& problem_sizes,
                   const torch::Tensor& expert_offsets) {
  grouped_mm("es_grouped_mm", false, output, a, b, problem_sizes, expert_offsets, torch::Tensor());
}

void es_grouped_mm_swiglu(torch::Tensor& output, const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& problem_sizes,
                          const torch::Tensor& expert_offsets, const c10::optional<torch::Tensor>& gate_up) {
  grouped_mm("es_grouped_mm_swiglu", true, output, a, b, problem_sizes, expert_offsets, tensor_or_none(gate_up));
}

void es_grouped_mm_backward(const torch::Tensor& grad_output, const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& problem_sizes,
                            const torch::Tensor& expert_offsets, const c10::optional<torch::Tensor>& grad_a,
                            const c10::optional<torch::Tensor>& grad_b) {
  grouped_mm_backward("es_grouped_mm_backward", nullptr, grad_output, a, b, problem_sizes, expert_offsets, tensor_or_none(grad_a),
                      tensor_or_none(grad_b));
}

void es_grouped_mm_swiglu_backward(const torch::Tensor& grad_output, const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& gate_up,
                                   const torch::Tensor& problem_sizes, const torch::Tensor& expert_offsets,
                                   const c10::optional<torch::Tensor>& grad_a, const c10::optional<torch::Tensor>& grad_b) {
  grouped_mm_backward("es_grouped_mm_swiglu_backward", &gate_up, grad_output, a, b, problem_sizes, expert_offsets, tensor_or_none(grad_a),
                      tensor_or_none(grad_b));
}

void es_int8_quant(const torch::Tensor& input, torch::Tensor& quant_output, torch::Tensor& scales) {
  TORCH_CHECK(input.dim() >= 1 && input.is_contiguous(), "input must be contiguous with at least 1 dimension");
  TORCH_CHECK(is_half_type(input), "dtype must be kFloat16 or kBFloat16");
  const int64_t k = input.size(-1);
  TORCH_CHECK(k > 0 && k % 16 == 0 && k <= 65536, "k must be a multiple of 16 up to 65536");
  const int64_t rows = input.numel() / k;
  TORCH_CHECK(quant_output.is_contiguous() && quant_output.scalar_type() == torch::kInt8 && quant_output.numel() == rows * k,
              "quant_output must be a contiguous int8 tensor of input's number of elements");
  TORCH_CHECK(scales.is_contiguous() && scales.scalar_type() == torch::kFloat32 && scales.numel() == rows,
              "scales must be a contiguous float32 tensor with one element per row");
  check_no_autograd("es_int8_quant", {&input}, {&scales});
  require_device(input, "es_int8_quant");
  check_device(input, {&quant_output, &scales});
  TORCH_CHECK(!any_overlap(quant_output, {&input, &scales}) && !any_overlap(scales, {&input}), "outputs may not overlap input or each other");
  if (rows == 0) return;
  c10::DeviceGuard guard(input.device());
  int rc = esmoe_int8_quant(input.data_ptr(), input.scalar_type() == torch::kBFloat16 ? ESMOE_IN_BF16 : ESMOE_IN_FP16, quant_output.data_ptr(),
                            scales.data_ptr<float>(), (long)rows, (int)k, current_stream(input));
  check_rc(rc, "es_int8_quant");
}

// The same into new tensors.
std::tuple<torch::Tensor, torch::Tensor> es_int8_quant_new(const torch::Tensor& input) {
  TORCH_CHECK(input.dim() >= 1, "input must be contiguous with at least 1 dimension");
  const auto opts = input.options().requires_grad(false);
  torch::Tensor q = torch::empty(input.sizes(), opts.dtype(torch::kInt8)),
                scales = torch::empty(input.sizes().slice(0, input.dim() - 1), opts.dtype(torch::kFloat32));
  es_int8_quant(input, q, scales);
  return {q, scales};
}

namespace {
void int8_scaled_grouped_mm(const char* op, bool swiglu, torch::Tensor& output, const torch::Tensor& a, const torch::Tensor& b,
                            const torch::Tensor& scales_a, const torch::Tensor& scales_b, const torch::Tensor& problem_sizes,
                            const torch::Tensor& expert_offsets) {
  TORCH_CHECK(a.scalar_type() == torch::kInt8, "a must be int8");
  check_experts(op, a, b, problem_sizes, expert_offsets, 16, 65536, swiglu);
  const int64_t rows = a.size(0), k = a.size(1), n = b.size(2), experts = b.size(0);
  TORCH_CHECK(is_half_type(output) && output.dim() == 2 && output.is_contiguous() && output.size(0) == rows && output.size(1) == (swiglu ? n / 2 : n),
              "output must be a contiguous bfloat16 or half (rows, n) tensor, (rows, n / 2) with SwiGLU");
  TORCH_CHECK(scales_a.scalar_type() == torch::kFloat32 && scales_a.is_contiguous() && scales_a.numel() == rows,
              "scales_a must be a contiguous float32 tensor with one element per row");
  TORCH_CHECK(scales_b.scalar_type() == torch::kFloat32 && scales_b.is_contiguous() && scales_b.dim() == 2 && scales_b.size(0) == experts &&
                  scales_b.size(1) == n,
              "scales_b must be a contiguous float32 (num_experts, n) tensor");
  check_no_autograd(op, {&scales_a, &scales_b}, {&output});
  require_device(a, op);
  check_device(a, {&output, &b, &scales_a, &scales_b, &problem_sizes, &expert_offsets});
  TORCH_CHECK(!any_overlap(output, {&a, &b, &scales_a, &scales_b, &problem_sizes, &expert_offsets}), "output may not overlap an input");
  if (rows == 0) return;
  c10::DeviceGuard guard(a.device());
  int rc = esmoe_int8_grouped_mm(output.data_ptr(), out_dtype_of(output), a.data_ptr(), b.data_ptr(), scales_a.data_ptr<float>(),
                                 scales_b.data_ptr<float>(), problem_sizes.data_ptr<int32_t>(), expert_offsets.data_ptr<int32_t>(), (int)experts,
                                 (int)rows, (int)n, (int)k, swiglu, current_stream(a));
  check_rc(rc, op);
}
}  // namespace

void es_int8_scaled_grouped_mm(torch::Tensor& output, const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& scales_a,
                               const torch::Tensor& scales_b, const torch::Tensor& problem_sizes, const torch::Tensor& expert_offsets) {
  int8_scaled_grouped_mm("es_int8_scaled_grouped_mm", false, output, a, b, scales_a, scales_b, problem_sizes, expert_offsets);
}

void es_int8_scaled_grouped_mm_swiglu(torch::Tensor& output, const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& scales_a,
                                      const torch::Tensor& scales_b, const torch::Tensor& problem_sizes, const torch::Tensor& expert_offsets) {
  int8_scaled_grouped_mm("es_int8_scaled_grouped_mm_swiglu", true, output, a, b, scales_a, scales_b, problem_sizes, expert_offsets);
}

// ---- the norm of gradients and their clipping ----
namespace {
struct GradList {
  std::vector<const void*> in;
  std::vector<void*> out;
  std::vector<int> dtypes;
  std::vector<long> sizes;
  torch::Tensor workspace;
};

GradList grad_list(const char* op, at::TensorList grads) {
  TORCH_CHECK(!grads.empty(), op, ": no gradients given");
  GradList l;
  l.in.reserve(grads.size());
  l.dtypes.reserve(grads.size());
  l.sizes.reserve(grads.size());
  const c10::Device device = grads[0].defined() ? grads[0].device() : c10::Device(c10::kCPU);
  for (const torch::Tensor& g : grads) {
    TORCH_CHECK(g.defined() && g.layout() == torch::kStrided, op, ": gradients must be dense tensors");
    const torch::ScalarType type = g.scalar_type();
    TORCH_CHECK(type == torch::kBFloat16 || type == torch::kHalf || type == torch::kFloat32, op, ": gradients must be float32, bfloat16 or half");
    TORCH_CHECK(g.is_non_overlapping_and_dense(), op, ": gradients must be dense in memory (their elements in any order, without gaps)");
    TORCH_CHECK(g.device() == device, "all tensors must be on the same device");
    check_no_autograd(op, {&g});
    l.dtypes.push_back(type == torch::kFloat32 ? ESMOE_GRAD_FP32 : type == torch::kHalf ? ESMOE_GRAD_FP16 : ESMOE_GRAD_BF16);
    l.sizes.push_back((long)g.numel());
  }
  return l;
}

// Whether a range that is written overlaps any other.
bool written_overlaps(at::TensorList grads, at::TensorList outputs, const torch::Tensor& norm) {
  struct Range { const char *from, *to; bool written; };
  std::vector<Range> ranges;
  ranges.reserve(2 * grads.size() + 1);
  const auto add = [&](const torch::Tensor& t, bool written) {
    if (t.defined() && t.numel()) ranges.push_back({(const char*)t.data_ptr(), (const char*)t.data_ptr() + t.nbytes(), written});
  };
  for (size_t i = 0; i < grads.size(); i++) {
    add(outputs[i], true);
    if (outputs[i].data_ptr() != grads[i].data_ptr()) add(grads[i], false);
  }
  add(norm, false);
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
  const char *any = nullptr, *written = nullptr;   // ends of those before
  for (const Range& r : ranges) {
    if (r.from < written || (r.written && r.from < any)) return true;
    any = std::max(any, r.to);
    if (r.written) written = std::max(written, r.to);
  }
  return false;
}

void grad_pointers(GradList& l, at::TensorList grads) {
  for (const torch::Tensor& g : grads) l.in.push_back(g.data_ptr());
  l.workspace = torch::empty({(int64_t)esmoe_grad_norm_workspace_bytes((int)grads.size())}, grads[0].options().dtype(torch::kUInt8).requires_grad(false));
}
}  // namespace

torch::Tensor es_grad_norm(at::TensorList grads) {
  GradList l = grad_list("es_grad_norm", grads);
  require_device(grads[0], "es_grad_norm");
  c10::DeviceGuard guard(grads[0].device());
  grad_pointers(l, grads);
  torch::Tensor norm = torch::empty({}, grads[0].options().dtype(torch::kFloat32).requires_grad(false));
  int rc = esmoe_grad_norm(l.in.data(), l.dtypes.data(), l.sizes.data(), (int)l.in.size(), norm.data_ptr<float>(), l.workspace.data_ptr(),
                           l.workspace.nbytes(), current_stream(grads[0]));
  check_rc(rc, "es_grad_norm");
  return norm;
}

torch::Tensor es_clip_grad_norm(at::TensorList grads, double max_norm, double eps, const c10::optional<torch::Tensor>& norm_, at::TensorList outputs) {
  const char* op = "es_clip_grad_norm";
  const torch::Tensor& given = tensor_or_none(norm_);
  GradList l = grad_list(op, grads);
  TORCH_CHECK(max_norm >= 0, "max_norm must not be negative or NaN");
  TORCH_CHECK(eps >= 0 && std::isfinite(eps), "eps must be finite and not negative");
  TORCH_CHECK(!given.defined() || (given.scalar_type() == torch::kFloat32 && given.numel() == 1), "norm must be a float32 scalar");
  TORCH_CHECK(outputs.size() == grads.size(), "outputs must have a tensor per gradient");
  for (size_t i = 0; i < grads.size(); i++) {
    TORCH_CHECK(outputs[i].defined() && outputs[i].sizes() == grads[i].sizes() && outputs[i].strides() == grads[i].strides() &&
                    outputs[i].scalar_type() == grads[i].scalar_type(),
                "outputs must have their gradients' shapes, strides and dtypes");
    check_no_autograd(op, {&given}, {&outputs[i]});
  }
  require_device(grads[0], op);
  check_device(grads[0], {&given});
  for (const torch::Tensor& o : outputs) check_device(grads[0], {&o});
  TORCH_CHECK(!written_overlaps(grads, outputs, given), "outputs may not overlap other gradients, each other or norm");
  c10::DeviceGuard guard(grads[0].device());
  grad_pointers(l, grads);
  for (const torch::Tensor& o : outputs) l.out.push_back(o.data_ptr());
  torch::Tensor norm = torch::empty({}, grads[0].options().dtype(torch::kFloat32).requires_grad(false));
  int rc = esmoe_clip_grad_norm(l.in.data(), l.out.data(), l.dtypes.data(), l.sizes.data(), (int)l.in.size(), max_norm, eps,
                                given.defined() ? given.data_ptr<float>() : nullptr, norm.data_ptr<float>(), l.workspace.data_ptr(),
                                l.workspace.nbytes(), current_stream(grads[0]));
  check_rc(rc, op);
  return norm;
}

TORCH_LIBRARY(expert_specialization, m) {
  m.def(
      "es_fp8_blockwise_scaled_grouped_mm(Tensor output, Tensor a, Tensor b, Tensor scales_a, Tensor scales_b, Tensor "
      "stride_a, Tensor stride_b, Tensor stride_d, Tensor problem_sizes, Tensor expert_offsets, Tensor workspace) -> "
      "()");
  m.def(
      "es_sm100_mxfp8_blockscaled_grouped_mm(Tensor a, Tensor b, Tensor sfa, Tensor sfb, Tensor d, Tensor "
      "problem_sizes, Tensor expert_offsets, Tensor blockscale_offsets) -> ()");
  m.def(
      "es_sm100_mxfp8_blockscaled_grouped_quant(Tensor input, Tensor problem_sizes, Tensor expert_offsets, Tensor "
      "blockscale_offsets, Tensor quant_output, Tensor scale_factor) -> () ");
  m.def(
      "es_fp8_blockwise_scaled_grouped_mm_swiglu_quant(Tensor quant_output, Tensor scales_out, Tensor a, Tensor b, Tensor "
      "scales_a, Tensor scales_b, Tensor problem_sizes, Tensor expert_offsets, Tensor workspace, bool mid_dtype_bf16) -> ()");
  m.def("es_fp8_quant_act_1x128(Tensor input, Tensor quant_output, Tensor scales) -> ()");
  m.def("es_fp8_quant_weight_128x128(Tensor input, Tensor quant_output, Tensor scales) -> ()");
  m.def("es_swiglu_quant_1x128(Tensor input, Tensor quant_output, Tensor scales) -> ()");
  m.def(
      "es_mxfp8_blockscaled_grouped_mm_swiglu_quant(Tensor quant_output, Tensor scale_factor, Tensor a, Tensor b, Tensor "
      "sfa, Tensor sfb, Tensor problem_sizes, Tensor expert_offsets, Tensor blockscale_offsets, bool mid_dtype_bf16) -> ()");
  m.def(
      "es_swiglu_mxfp8_grouped_quant(Tensor input, Tensor problem_sizes, Tensor expert_offsets, Tensor "
      "blockscale_offsets, Tensor quant_output, Tensor scale_factor) -> ()");
  m.def("es_mxfp8_quant_weight(Tensor input, Tensor quant_output, Tensor scale_factor) -> ()");
  m.def("es_route_metadata(Tensor topk_ids, int first_expert, int num_experts, int n, int k) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("es_permute_rows(Tensor input, Tensor dst_row, int topk, Tensor output) -> ()");
  m.def(
      "es_topk_gating(Tensor logits, int topk, Tensor? bias, bool sigmoid, bool renormalize, float scale, int num_groups, int "
      "topk_groups) -> (Tensor, Tensor)");
  m.def(
      "es_topk_gating_backward(Tensor grad_weights, Tensor logits, Tensor topk_ids, bool sigmoid, bool renormalize, float scale) -> "
      "Tensor");
  m.def("es_combine_rows(Tensor input, Tensor dst_row, int topk, Tensor? weights, Tensor output) -> ()");
  m.def("es_combine_rows.new(Tensor input, Tensor dst_row, int topk, Tensor? weights) -> Tensor");
  m.def(
      "es_combine_rows_backward(Tensor grad_output, Tensor input, Tensor dst_row, int topk, Tensor weights, Tensor grad_input, Tensor "
      "grad_weights) -> ()");
  m.def(
      "es_add_rms_norm_quant_1x128(Tensor input, Tensor weight, float eps, Tensor? residual, Tensor? residual_out, Tensor? normed, "
      "Tensor quant_output, Tensor scales) -> ()");
  m.def(
      "es_add_rms_norm_quant_1x128.new(Tensor input, Tensor weight, float eps, Tensor? residual, bool return_normed) -> (Tensor, Tensor, "
      "Tensor, Tensor)");
  m.def("es_mxfp4_grouped_mm(Tensor output, Tensor a, Tensor b, Tensor sfb, Tensor problem_sizes, Tensor expert_offsets) -> ()");
  m.def("es_mxfp4_grouped_mm_swiglu(Tensor output, Tensor a, Tensor b, Tensor sfb, Tensor problem_sizes, Tensor expert_offsets) -> ()");
  m.def("es_grouped_mm(Tensor output, Tensor a, Tensor b, Tensor problem_sizes, Tensor expert_offsets) -> ()");
  m.def("es_grouped_mm_swiglu(Tensor output, Tensor a, Tensor b, Tensor problem_sizes, Tensor expert_offsets, Tensor? gate_up) -> ()");
  m.def(
      "es_grouped_mm_backward(Tensor grad_output, Tensor a, Tensor b, Tensor problem_sizes, Tensor expert_offsets, Tensor? grad_a, Tensor? "
      "grad_b) -> ()");
  m.def(
      "es_grouped_mm_swiglu_backward(Tensor grad_output, Tensor a, Tensor b, Tensor gate_up, Tensor problem_sizes, Tensor expert_offsets, "
      "Tensor? grad_a, Tensor? grad_b) -> ()");
  m.def("es_int8_quant(Tensor input, Tensor quant_output, Tensor scales) -> ()");
  m.def("es_int8_quant.new(Tensor input) -> (Tensor, Tensor)");
  m.def(
      "es_int8_scaled_grouped_mm(Tensor output, Tensor a, Tensor b, Tensor scales_a, Tensor scales_b, Tensor problem_sizes, Tensor "
      "expert_offsets) -> ()");
  m.def(
      "es_int8_scaled_grouped_mm_swiglu(Tensor output, Tensor a, Tensor b, Tensor scales_a, Tensor scales_b, Tensor problem_sizes, Tensor "
      "expert_offsets) -> ()");
  m.def("es_grad_norm(Tensor[] grads) -> Tensor");
  m.def("es_clip_grad_norm(Tensor[] grads, float max_norm, float eps, Tensor? norm, Tensor[] outputs) -> Tensor");
}

TORCH_LIBRARY_IMPL(expert_specialization, CUDA, m) {
  m.impl("es_fp8_blockwise_scaled_grouped_mm", &es_fp8_blockwise_scaled_grouped_mm);
  m.impl("es_sm100_mxfp8_blockscaled_grouped_mm", &es_sm100_mxfp8_blockscaled_grouped_mm);
  m.impl("es_sm100_mxfp8_blockscaled_grouped_quant", &es_sm100_mxfp8_blockscaled_grouped_quant);
  m.impl("es_fp8_blockwise_scaled_grouped_mm_swiglu_quant", &es_fp8_blockwise_scaled_grouped_mm_swiglu_quant);
  m.impl("es_fp8_quant_act_1x128", &es_fp8_quant_act_1x128);
  m.impl("es_fp8_quant_weight_128x128", &es_fp8_quant_weight_128x128);
  m.impl("es_swiglu_quant_1x128", &es_swiglu_quant_1x128);
  m.impl("es_mxfp8_blockscaled_grouped_mm_swiglu_quant", &es_mxfp8_blockscaled_grouped_mm_swiglu_quant);
  m.impl("es_swiglu_mxfp8_grouped_quant", &es_swiglu_mxfp8_grouped_quant);
  m.impl("es_mxfp8_quant_weight", &es_mxfp8_quant_weight);
  m.impl("es_route_metadata", &es_route_metadata);
  m.impl("es_permute_rows", &es_permute_rows);
  m.impl("es_topk_gating", &es_topk_gating);
  m.impl("es_topk_gating_backward", &es_topk_gating_backward);
  m.impl("es_combine_rows", &es_combine_rows);
  m.impl("es_combine_rows.new", &es_combine_rows_new);
  m.impl("es_combine_rows_backward", &es_combine_rows_backward);
  m.impl("es_add_rms_norm_quant_1x128", &es_add_rms_norm_quant_1x128);
  m.impl("es_add_rms_norm_quant_1x128.new", &es_add_rms_norm_quant_1x128_new);
  m.impl("es_mxfp4_grouped_mm", &es_mxfp4_grouped_mm);
  m.impl("es_mxfp4_grouped_mm_swiglu", &es_mxfp4_grouped_mm_swiglu);
  m.impl("es_grouped_mm", &es_grouped_mm);
  m.impl("es_grouped_mm_swiglu", &es_grouped_mm_swiglu);
  m.impl("es_grouped_mm_backward", &es_grouped_mm_backward);
  m.impl("es_grouped_mm_swiglu_backward", &es_grouped_mm_swiglu_backward);
  m.impl("es_int8_quant", &es_int8_quant);
  m.impl("es_int8_quant.new", &es_int8_quant_new);
  m.impl("es_int8_scaled_grouped_mm", &es_int8_scaled_grouped_mm);
  m.impl("es_int8_scaled_grouped_mm_swiglu", &es_int8_scaled_grouped_mm_swiglu);
  m.impl("es_grad_norm", &es_grad_norm);
  m.impl("es_clip_grad_norm", &es_clip_grad_norm);
}

// Same functions on the CPU key: the checks run, then require_device() raises.
TORCH_LIBRARY_IMPL(expert_specialization, CPU, m) {
  m.impl("es_fp8_blockwise_scaled_grouped_mm", &es_fp8_blockwise_scaled_grouped_mm);
  m.impl("es_sm100_mxfp8_blockscaled_grouped_mm", &es_sm100_mxfp8_blockscaled_grouped_mm);
  m.impl("es_sm100_mxfp8_blockscaled_grouped_quant", &es_sm100_mxfp8_blockscaled_grouped_quant);
  m.impl("es_fp8_blockwise_scaled_grouped_mm_swiglu_quant", &es_fp8_blockwise_scaled_grouped_mm_swiglu_quant);
  m.impl("es_fp8_quant_act_1x128", &es_fp8_quant_act_1x128);
  m.impl("es_fp8_quant_weight_128x128", &es_fp8_quant_weight_128x128);
  m.impl("es_swiglu_quant_1x128", &es_swiglu_quant_1x128);
  m.impl("es_mxfp8_blockscaled_grouped_mm_swiglu_quant", &es_mxfp8_blockscaled_grouped_mm_swiglu_quant);
  m.impl("es_swiglu_mxfp8_grouped_quant", &es_swiglu_mxfp8_grouped_quant);
  m.impl("es_mxfp8_quant_weight", &es_mxfp8_quant_weight);
  m.impl("es_route_metadata", &es_route_metadata);
  m.impl("es_permute_rows", &es_permute_rows);
  m.impl("es_topk_gating", &es_topk_gating);
  m.impl("es_topk_gating_backward", &es_topk_gating_backward);
  m.impl("es_combine_rows", &es_combine_rows);
  m.impl("es_combine_rows.new", &es_combine_rows_new);
  m.impl("es_combine_rows_backward", &es_combine_rows_backward);
  m.impl("es_add_rms_norm_quant_1x128", &es_add_rms_norm_quant_1x128);
  m.impl("es_add_rms_norm_quant_1x128.new", &es_add_rms_norm_quant_1x128_new);
  m.impl("es_mxfp4_grouped_mm", &es_mxfp4_grouped_mm);
  m.impl("es_mxfp4_grouped_mm_swiglu", &es_mxfp4_grouped_mm_swiglu);
  m.impl("es_grouped_mm", &es_grouped_mm);
  m.impl("es_grouped_mm_swiglu", &es_grouped_mm_swiglu);
  m.impl("es_grouped_mm_backward", &es_grouped_mm_backward);
  m.impl("es_grouped_mm_swiglu_backward", &es_grouped_mm_swiglu_backward);
  m.impl("es_int8_quant", &es_int8_quant);
  m.impl("es_int8_quant.new", &es_int8_quant_new);
  m.impl("es_int8_scaled_grouped_mm", &es_int8_scaled_grouped_mm);
  m.impl("es_int8_scaled_grouped_mm_swiglu", &es_int8_scaled_grouped_mm_swiglu);
  m.impl("es_grad_norm", &es_grad_norm);
  m.impl("es_clip_grad_norm", &es_clip_grad_norm);
}
