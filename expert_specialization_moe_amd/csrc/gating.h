// What the C API hands to the router gating kernels (gating.hip).
#pragma once

namespace esmoe {

constexpr int kGateMaxExperts = 1024;   // sixteen per lane
constexpr int kGateMaxGroups = 64;      // a lane per group
constexpr int kGateF32 = 0, kGateF16 = 1, kGateBf16 = 2;

struct GateArgs {
  long tokens;
  int experts, topk, groups, topk_groups;
  int sigmoid, renormalize;
  int exact;   // the order goes by fp32(score + bias) from 64 bits, not by the logits
  float scale;
};

}  // namespace esmoe
