// Prefix sum over a wavefront, on the vector ALU alone.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace esmoe {

// Sum of `v` over this lane and the lanes below it (DPP row shifts and row broadcasts; a ds_bpermute shuffle costs a trip to
// LDS per step).
__device__ __forceinline__ int wave_inclusive_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr:1, :2, :4, :8 (rows of 16 lanes)
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31 into rows 2 and 3
  return v;
}

// The same where a sum of more than 32 bits stays at the largest number.
__device__ __forceinline__ uint32_t wave_inclusive_sum_or_most(uint32_t v) {
  auto step = [&](int below) { v = __builtin_elementwise_add_sat(v, (uint32_t)below); };
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
  return v;
}

// Sum of `v` over the whole wavefront, in its last lane (the same steps).
__device__ __forceinline__ float wave_sum_last(float v) {
  auto step = [&](int shifted) { v += __builtin_bit_cast(float, shifted); };
  step(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x111, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x112, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x114, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x118, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x142, 0xa, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x143, 0xc, 0xf, false));
  return v;
}

}  // namespace esmoe
