// Router gating: logits -> the top-k experts of every token and their weights, and the gradient of the weights.
//
//   s_e = softmax(x)_e or 1 / (1 + exp(-x_e))
//   choice_e = x_e, or fp32(s_e + bias_e) formed in 64 bits where a bias or groups take part (the order of experts then hangs on
//              the last bit of a sum, and the ids are whole numbers that have to be the same everywhere)
//   groups: of the G groups of E / G consecutive experts the topk_groups with the largest fp32 sum of their two largest choices stay
//   ids = the topk largest choices left, in falling order, ties to the lower index; NaN above every number; an expert whose logit or
//         choice is -inf is never taken: a place that no expert is left for gets id -1 and weight 0
//   w_j = scale * s_{id_j}, or scale * s_{id_j} / sum_i s_{id_i}
// Gradient, ids held fixed (r: renormalised, w' = w / scale, G_e = sum of scale * g_j over id_j = e):
//   softmax r: dx = w'_j (scale g_j - sum_i w'_i scale g_i) at id_j;   softmax: dx_e = s_e (G_e - sum_i G_i s_i) everywhere
//   sigmoid r: dx = w'_j (1 - s_j) (scale g_j - sum_i w'_i scale g_i); sigmoid: dx = s_j (1 - s_j) scale g_j
//
// The reference has no router: its callers draw the ids at random (benchmark/benchmark_es_fp8_blockwise_moe.py:44-56).
//
// One wavefront per token, every expert's order key (a float mapped to an unsigned integer of the same order) in a register: lane l
// holds experts l * PER .. l * PER + PER - 1, so that the lowest lane of a ballot holds the lowest index.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "gating.h"

namespace esmoe {

constexpr int kGateWaves = 4;

// Orders a wavefront's writes to its own part of LDS before its reads.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <typename T>
__device__ __forceinline__ float gate_load(const T* p) {
  if constexpr (sizeof(T) == 4) return *p;
  else if constexpr (std::is_same<T, _Float16>::value) return (float)*p;
  else return __builtin_bit_cast(float, (uint32_t)*(const uint16_t*)p << 16);
}

// Unsigned integers of the same order as the floats: 0 for -inf (taken by nobody), all ones for NaN; -0 and 0 are one value.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __builtin_bit_cast(uint32_t, f + 0.0f);
  const uint32_t k = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  if (f != f) return 0xffffffffu;
  return b == 0xff800000u ? 0u : k;
}

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
  return v > o ? v : o;
}
// Maximum over the wavefront, in every lane.
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  v = dpp_umax<0x111, 0xf>(v);
  v = dpp_umax<0x112, 0xf>(v);
  v = dpp_umax<0x114, 0xf>(v);
  v = dpp_umax<0x118, 0xf>(v);
  v = dpp_umax<0x142, 0xa>(v);
  v = dpp_umax<0x143, 0xc>(v);
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
template <typename F>
__device__ __forceinline__ F wave_sum_all(F v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}
// NaN where any lane holds one (the maximum of a softmax).
__device__ __forceinline__ float wave_max_nan(float v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const float o = __shfl_xor(v, d);
    v = o != o ? o : (v != v ? v : (v > o ? v : o));
  }
  return v;
}

template <typename T, int PER>
__global__ void __launch_bounds__(64 * kGateWaves) topk_gating_kernel(const T* __restrict__ logits, long ld, const float* __restrict__ bias,
                                                                      GateArgs a, int* __restrict__ ids, float* __restrict__ weights) {
  __shared__ uint32_t s_key[kGateWaves][64 * PER];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const long t = (long)blockIdx.x * kGateWaves + w;
  if (t >= a.tokens) return;   // (no barrier below: a wavefront's LDS is its own)
  const T* row = logits + t * ld;
  float x[PER];
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int e = lane * PER + i;
    x[i] = e < a.experts ? gate_load(row + e) : -__builtin_inff();
    key[i] = order_key(x[i]);
  }
  float top = 0, sum = 0;   // of the softmax over all experts
  if (!a.sigmoid) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < PER; i++) m = x[i] != x[i] ? x[i] : (m != m ? m : (m > x[i] ? m : x[i]));
    top = wave_max_nan(m);
  }
  if (!a.sigmoid && !a.renormalize) {
    float s = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) s += lane * PER + i < a.experts ? expf(x[i] - top) : 0.f;
    sum = wave_sum_all(s);
  }
  if (a.exact) {
    double s[PER], all = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      s[i] = a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[i])) : lane * PER + i < a.experts ? exp((double)x[i] - (double)top) : 0.0;
      all += s[i];
    }
    if (!a.sigmoid) all = wave_sum_all(all);
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int e = lane * PER + i;
      double c = a.sigmoid ? s[i] : s[i] / all;
      if (bias && e < a.experts) c += (double)bias[e];
      key[i] = key[i] == 0 ? 0 : order_key((float)c);
    }
  }
  if (a.groups > 1) {
#pragma unroll
    for (int i = 0; i < PER; i++) s_key[w][lane * PER + i] = key[i];
    wave_lds_fence();
    const int width = a.experts / a.groups;
    uint32_t first = 0, second = 0;
    if (lane < a.groups)
      for (int i = 0; i < width; i++) {
        const uint32_t k = s_key[w][lane * width + i];
        if (k > first) { second = first; first = k; }
        else if (k > second) second = k;
      }
    auto value = [](uint32_t k) {   // the float behind a key; nothing for an expert that is out
      return k == 0 ? 0.f : __builtin_bit_cast(float, k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
    };
    uint32_t score = first == 0 ? 0u : order_key(value(first) + value(second));
    if (first != 0 && score == 0) score = 1;   // two finite choices whose sum is -inf
    unsigned long long keep = 0;
    for (int j = 0; j < a.topk_groups; j++) {
      const uint32_t best = wave_umax(score);
      if (best == 0) break;
      const int g = __builtin_ctzll(__ballot(score == best));
      keep |= 1ull << g;
      if (lane == g) score = 0;
    }
#pragma unroll
    for (int i = 0; i < PER; i++)
      if (!((keep >> ((lane * PER + i) / width & 63)) & 1)) key[i] = 0;
  }
  int mine = -1;   // lane j: the j-th expert
  for (int j = 0; j < a.topk; j++) {
    uint32_t best = key[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < PER; i++)
      if (key[i] > best) { best = key[i]; at = i; }
    const uint32_t max = wave_umax(best);
    if (max == 0) break;
    const int winner = __builtin_ctzll(__ballot(best == max));
    const int e = winner * PER + __builtin_amdgcn_readlane(at, winner);
    if (lane == j) mine = e;
#pragma unroll
    for (int i = 0; i < PER; i++)
      if (lane == winner && at == i) key[i] = 0;
  }
  // the weights, a lane per place
  const bool real = mine >= 0;
  const float xs = real ? gate_load(row + mine) : -__builtin_inff();
  float v;
  if (!a.renormalize) {
    v = a.sigmoid ? 1.0f / (1.0f + expf(-xs)) : expf(xs - top) / sum;
  } else {
    // scaled by the largest of them, so that the sum is never 0 / 0
    const float m = wave_max_nan(xs);
    if (!a.sigmoid) v = expf(xs - m);
    else if (xs >= 0) v = 1.0f / (1.0f + expf(-xs));
    else v = expf(xs - (m < 0 ? m : 0.f)) / (1.0f + expf(xs));
    v = real ? v : 0.f;
    v /= wave_sum_all(v);
  }
  if (lane < a.topk) {
    ids[t * a.topk + lane] = mine;
    weights[t * a.topk + lane] = real ? v * a.scale : 0.f;
  }
}

// One wavefront per token; ids that stand twice in a row add up, ids outside [0, experts) are places without an expert.
template <typename T>
__global__ void __launch_bounds__(64 * kGateWaves) topk_gating_backward_kernel(const float* __restrict__ grad, const T* __restrict__ logits,
                                                                               long ld, const int* __restrict__ ids, GateArgs a,
                                                                               T* __restrict__ out) {
  __shared__ float s_grad[kGateWaves][kGateMaxExperts];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const long t = (long)blockIdx.x * kGateWaves + w;
  if (t >= a.tokens) return;
  const T* row = logits + t * ld;
  int id = lane < a.topk ? ids[t * a.topk + lane] : -1;
  if ((unsigned)id >= (unsigned)a.experts) id = -1;
  const bool real = id >= 0;
  const float g = real ? grad[t * a.topk + lane] * a.scale : 0.f;
  const float xs = real ? gate_load(row + id) : -__builtin_inff();
  const bool dense = !a.sigmoid && !a.renormalize;
  float d = 0, top = 0, sum = 0, mean = 0;
  if (dense) {
    float m = -__builtin_inff();
    for (int e = lane; e < a.experts; e += 64) {
      const float x = gate_load(row + e);
      m = x != x ? x : (m != m ? m : (m > x ? m : x));
    }
    top = wave_max_nan(m);
    if (top == -__builtin_inff()) top = 0;   // every expert masked: all terms 0
    float s = 0;
    for (int e = lane; e < a.experts; e += 64) s += expf(gate_load(row + e) - top);
    sum = wave_sum_all(s);
    sum = sum == 0 ? 1.f : sum;
    mean = wave_sum_all(real ? g * (expf(xs - top) / sum) : 0.f);
    d = g;
  } else if (a.renormalize) {
    const float m = wave_max_nan(xs);
    float v = 0;
    if (real) {
      if (!a.sigmoid) v = expf(xs - m);
      else if (xs >= 0) v = 1.0f / (1.0f + expf(-xs));
      else v = expf(xs - (m < 0 ? m : 0.f)) / (1.0f + expf(xs));
    }
    const float all = wave_sum_all(v);
    v = real ? v / all : 0.f;
    const float mid = wave_sum_all(g * v);
    d = real ? v * (g - mid) * (a.sigmoid ? 1.0f / (1.0f + expf(xs)) : 1.0f) : 0.f;
  } else {
    d = real ? g / (1.0f + expf(-xs)) / (1.0f + expf(xs)) : 0.f;
  }
  float total = 0;   // of all places with this lane's id
  for (int j = 0; j < a.topk; j++) {
    const int other = __builtin_amdgcn_readlane(id, j);
    const float od = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, d), j));
    total += other == id ? od : 0.f;
  }
  for (int e = lane; e < a.experts; e += 64) s_grad[w][e] = 0.f;
  wave_lds_fence();
  if (real) s_grad[w][id] = total;
  wave_lds_fence();
  for (int e = lane; e < a.experts; e += 64) {
    float v = s_grad[w][e];
    if (dense) v = expf(gate_load(row + e) - top) / sum * (v - mean);
    T* o = out + t * a.experts + e;
    if constexpr (sizeof(T) == 4) *o = v;
    else if constexpr (std::is_same<T, _Float16>::value) *o = (_Float16)v;
    else *o = (__bf16)v;
  }
}

template <typename T>
static int launch_gating(const void* logits, long ld, const float* bias, const GateArgs& a, int* ids, float* weights, hipStream_t stream) {
  const unsigned grid = (unsigned)((a.tokens + kGateWaves - 1) / kGateWaves);
  const int per = (a.experts + 63) / 64;
#define ESMOE_GATE(P)                                                                                                              \
  hipLaunchKernelGGL((topk_gating_kernel<T, P>), dim3(grid), dim3(64 * kGateWaves), 0, stream, (const T*)logits, ld, bias, a, ids, weights)
  if (per <= 1) ESMOE_GATE(1);
  else if (per <= 2) ESMOE_GATE(2);
  else if (per <= 4) ESMOE_GATE(4);
  else if (per <= 8) ESMOE_GATE(8);
  else ESMOE_GATE(16);
#undef ESMOE_GATE
  return (int)hipGetLastError();
}

template <typename T>
static int launch_gating_backward(const float* grad, const void* logits, long ld, const int* ids, const GateArgs& a, void* out,
                                  hipStream_t stream) {
  const unsigned grid = (unsigned)((a.tokens + kGateWaves - 1) / kGateWaves);
  hipLaunchKernelGGL((topk_gating_backward_kernel<T>), dim3(grid), dim3(64 * kGateWaves), 0, stream, grad, (const T*)logits, ld, ids, a,
                     (T*)out);
  return (int)hipGetLastError();
}

}  // namespace esmoe

extern "C" int esmoe_launch_topk_gating(const void* logits, int dtype, long ld, const float* bias, const esmoe::GateArgs* a, int* ids,
                                        float* weights, hipStream_t stream) {
  using namespace esmoe;
  if (dtype == kGateF32) return launch_gating<float>(logits, ld, bias, *a, ids, weights, stream);
  if (dtype == kGateF16) return launch_gating<_Float16>(logits, ld, bias, *a, ids, weights, stream);
  return launch_gating<__bf16>(logits, ld, bias, *a, ids, weights, stream);
}

extern "C" int esmoe_launch_topk_gating_backward(const float* grad, const void* logits, int dtype, long ld, const int* ids,
                                                 const esmoe::GateArgs* a, void* out, hipStream_t stream) {
  using namespace esmoe;
  if (dtype == kGateF32) return launch_gating_backward<float>(grad, logits, ld, ids, *a, out, stream);
  if (dtype == kGateF16) return launch_gating_backward<_Float16>(grad, logits, ld, ids, *a, out, stream);
  return launch_gating_backward<__bf16>(grad, logits, ld, ids, *a, out, stream);
}
