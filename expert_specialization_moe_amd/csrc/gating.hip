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
// Two kernels.  Sixteen lanes per token, four tokens per wavefront, for up to 256 experts and 16 places: what a router has.  One
// wavefront per token for everything else.  Both order experts by unsigned keys that have the floats' order.
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

__device__ __forceinline__ float key_value(uint32_t k) {   // the float behind a key other than 0
  return __builtin_bit_cast(float, k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// A wavefront's reductions run on the vector ALU: row shifts, then row broadcasts; the last lane's value is everybody's.
template <int CTRL, int ROWS, typename F, typename Op>
__device__ __forceinline__ F dpp_step(F v, F neutral, Op op) {
  const int o = __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, neutral), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false);
  return op(v, __builtin_bit_cast(F, o));
}
template <typename F, typename Op>
__device__ __forceinline__ F wave_reduce(F v, F neutral, Op op) {
  v = dpp_step<0x111, 0xf>(v, neutral, op);
  v = dpp_step<0x112, 0xf>(v, neutral, op);
  v = dpp_step<0x114, 0xf>(v, neutral, op);
  v = dpp_step<0x118, 0xf>(v, neutral, op);
  v = dpp_step<0x142, 0xa>(v, neutral, op);
  v = dpp_step<0x143, 0xc>(v, neutral, op);
  return __builtin_bit_cast(F, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  return wave_reduce(v, 0u, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ float wave_sum_all(float v) {
  return wave_reduce(v, 0.f, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ double wave_sum_all(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}
// NaN where any lane holds one (the maximum of a softmax).
__device__ __forceinline__ float wave_max_nan(float v) {
  const float m = wave_reduce(v, -__builtin_inff(), [](float a, float b) { return __builtin_fmaxf(a, b); });
  return __ballot(v != v) ? __builtin_nanf("") : m;
}

// A renormalised weight before the division by the places' sum: the score, scaled by the largest of them (of logit m), so that the sum
// is never 0 / 0.
__device__ __forceinline__ float gate_term(float x, float m, int sigmoid) {
  if (!sigmoid) return expf(x - m);
  if (x >= 0) return 1.0f / (1.0f + expf(-x));
  return expf(x - (m < 0 ? m : 0.f)) / (1.0f + expf(x));
}

// One token by a whole wavefront: the order from 64 bits wherever it hangs on them.  Lane l holds experts l * PER .. l * PER + PER - 1, so
// that the lowest lane of a ballot holds the lowest index.
template <typename T, int PER>
__device__ __forceinline__ void gate_token(const T* __restrict__ row, const float* __restrict__ bias, const GateArgs& a, uint32_t* s_key,
                                           int* __restrict__ ids, float* __restrict__ weights) {
  const int lane = threadIdx.x & 63;
  float x[PER];
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int e = lane * PER + i;
    x[i] = e < a.experts ? gate_load(row + e) : -__builtin_inff();
    key[i] = order_key(x[i]);
  }
  float top = 0, sum = 0;   // of the softmax over all experts
  if (!a.sigmoid && (a.exact || !a.renormalize)) {
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
    for (int i = 0; i < PER; i++) s_key[lane * PER + i] = key[i];
    wave_lds_fence();
    const int width = a.experts / a.groups;
    const int log = 31 - __builtin_clz(64 / a.groups), lanes = 1 << log, own = lane >> log;   // lanes of a group, the lane's group
    uint32_t first = 0, second = 0;
    auto join = [&](uint32_t f, uint32_t s) {
      const uint32_t low = first < f ? first : f, high = second > s ? second : s;
      first = first > f ? first : f;
      second = high > low ? high : low;
    };
    if (own < a.groups)
      for (int i = lane & (lanes - 1); i < width; i += lanes) join(s_key[own * width + i], 0);
    for (int d = 1; d < lanes; d <<= 1) join(__shfl_xor(first, d), __shfl_xor(second, d));
    // (1: finite choices whose sum is -inf; 0: no expert left)
    uint32_t score = first == 0 ? 0u : order_key(key_value(first) + (second ? key_value(second) : 0.f));
    if (first != 0 && score == 0) score = 1;
    unsigned long long keep = 0;
    for (int j = 0; j < a.topk_groups; j++) {
      const uint32_t best = wave_umax(score);
      if (best == 0) break;
      const int g = __builtin_ctzll(__ballot(score == best)) >> log;
      keep |= 1ull << g;
      if (own == g) score = 0;
    }
#pragma unroll
    for (int i = 0; i < PER; i++)
      if (!((keep >> ((lane * PER + i) / width & 63)) & 1)) key[i] = 0;
    wave_lds_fence();   // (another token's keys may come next)
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
    v = gate_term(xs, wave_max_nan(xs), a.sigmoid);
    v = real ? v : 0.f;
    v /= wave_sum_all(v);
  }
  if (lane < a.topk) {
    ids[lane] = mine;
    weights[lane] = real ? v * a.scale : 0.f;
  }
}

template <typename T, int PER>
__global__ void __launch_bounds__(64 * kGateWaves) topk_gating_kernel(const T* __restrict__ logits, long ld, const float* __restrict__ bias,
                                                                      GateArgs a, int* __restrict__ ids, float* __restrict__ weights) {
  __shared__ uint32_t s_key[kGateWaves][64 * PER];
  const int w = threadIdx.x >> 6;
  const long t = (long)blockIdx.x * kGateWaves + w;
  if (t < a.tokens) gate_token<T, PER>(logits + t * ld, bias, a, s_key[w], ids + t * a.topk, weights + t * a.topk);
}

// A lane's PER values from `first` on, `none` past the last; VEC: in whole, aligned pieces of sixteen bytes (or all PER).
template <bool VEC, typename T, int PER>
__device__ __forceinline__ void load_lane(const T* row, int first, int count, float none, float (&v)[PER]) {
  if constexpr (VEC) {
    constexpr int kPiece = PER * sizeof(T) < 16 ? PER : 16 / sizeof(T);
    struct alignas(sizeof(T) * kPiece) Piece { T v[kPiece]; };
    Piece c[PER / kPiece];
#pragma unroll
    for (int u = 0; u < PER / kPiece; u++) {
      c[u] = Piece{};
      if (first + u * kPiece < count) c[u] = *(const Piece*)(row + first + u * kPiece);
    }
#pragma unroll
    for (int i = 0; i < PER; i++) v[i] = first + i / kPiece * kPiece < count ? gate_load(&c[i / kPiece].v[i % kPiece]) : none;
  } else {
#pragma unroll
    for (int i = 0; i < PER; i++) v[i] = first + i < count ? gate_load(row + first + i) : none;
  }
}

template <typename T>
__device__ __forceinline__ T gate_round(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, _Float16>::value) return (_Float16)v;
  else return (__bf16)v;
}
template <bool VEC, typename T, int PER>
__device__ __forceinline__ void store_lane(T* row, int first, int count, const float (&v)[PER]) {
  if constexpr (VEC) {
    constexpr int kPiece = PER * sizeof(T) < 16 ? PER : 16 / sizeof(T);
    struct alignas(sizeof(T) * kPiece) Piece { T v[kPiece]; };
#pragma unroll
    for (int u = 0; u < PER / kPiece; u++) {
      Piece c;
#pragma unroll
      for (int i = 0; i < kPiece; i++) c.v[i] = gate_round<T>(v[u * kPiece + i]);
      if (first + u * kPiece < count) *(Piece*)(row + first + u * kPiece) = c;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; i++)
      if (first + i < count) row[first + i] = gate_round<T>(v[i]);
  }
}

// Sixteen lanes' reductions, to all of them.
template <int CTRL, typename F, typename Op>
__device__ __forceinline__ F row_step(F v, Op op) {   // (every lane has a partner: the move becomes part of the operation)
  return op(v, __builtin_bit_cast(F, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true)));
}
template <typename F, typename Op>
__device__ __forceinline__ F row_reduce(F v, Op op) {
  v = row_step<0xB1>(v, op);    // lane ^ 1, ^ 2, then the mirrors of eight and of sixteen lanes
  v = row_step<0x4E>(v, op);
  v = row_step<0x141>(v, op);
  return row_step<0x140>(v, op);
}
__device__ __forceinline__ float row_sum(float v) {
  return row_reduce(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float row_max(float v) {
  return row_reduce(v, [](float a, float b) { return __builtin_fmaxf(a, b); });
}

__device__ __forceinline__ float row_max_nan(float v) {
  return row_reduce(v, [](float a, float b) { return a != a || b != b ? __builtin_nanf("") : __builtin_fmaxf(a, b); });
}

// Sum of d over the token's later places of the same id, in their order; `first` goes where an earlier place has it.
template <int R>
__device__ __forceinline__ float later_terms(int id, float d, int l, bool& first) {
  if constexpr (R < 16) {
    // lane l - R of the sixteen (row_ror takes from the lanes below, around the end): a later place where R lanes around is above
    const int other = __builtin_amdgcn_update_dpp(0, id, 0x120 + R, 0xf, 0xf, false);
    const float od = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, d), 0x120 + R, 0xf, 0xf, false));
    if (l >= R && other == id) first = false;
    const float mine = l < R && other == id ? od : 0.f;
    return mine + later_terms<R + 1>(id, d, l, first);
  }
  return 0.f;
}

// Counts the groups whose score is ahead of the lane's by more than `near`, and those that are not as far behind; R lanes on, and so forth.
// (A group without an expert left has -inf: behind all others, and what is said of it does not matter.)
template <int R>
__device__ __forceinline__ void compare_rotated(float score, float near, int lanes, int& sure, int& maybe) {
  if constexpr (R < 16) {
    if (R % lanes == 0) {
      const float d = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, score), 0x120 + R, 0xf, 0xf, false)) - score;
      sure += d > near;
      maybe += d >= -near;
    }
    compare_rotated<R + 1>(score, near, lanes, sure, maybe);
  }
}

// How many of the sixteen lanes' keys are ahead of the lane's: larger, or as large and of a lower id.
template <int R>
__device__ __forceinline__ int order_rotated(uint32_t key, int id) {
  if constexpr (R < 16) {
    const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)key, 0x120 + R, 0xf, 0xf, false);
    const int oid = __builtin_amdgcn_update_dpp(0, id, 0x120 + R, 0xf, 0xf, false);
    return (other > key || (other == key && oid < id) ? 1 : 0) + order_rotated<R + 1>(key, id);
  }
  return 0;
}

// Four tokens per wavefront, a lane l of sixteen holds a token's experts l * PER .. l * PER + PER - 1.
//
// Bound by the instructions that find the largest of E keys topk times.  So a key is one register: the upper 24 bits of the choice's order
// and below them 255 - expert, and a largest one stands for itself and its place.  The largest key below the one before is
//   before + max over keys of (key - before mod 2^32),
// a subtraction per key and no removal: what is not below `before` wraps to the small side.
// 24 bits hold the order key of a bf16 or fp16 logit whole.  Anything else becomes a fixed-point number from the token's smallest choice
// (or 64 below the largest) on, and has a bound on its error: the choices that groups and a bias decide about are formed in fp32, off from
// the 64-bit ones by less than `slack`.  Where two neighbours of the order are too close to tell, the candidates alone are put in order by
// their exact choices, unless they are the same logit and bias; where the last of them and the next, or two groups' scores are, the wavefront
// does the token again by gate_token.  Equal logits are the rule in 16 bits: bf16 softmax, 256 experts, 4 of 8 groups, every near pair to
// gate_token / this: 16384 tokens 32.5 / 14.9 us, 2048 23.3 / 10.3, 256 19.0 / 5.7.
// us for 256 experts, top-8, sigmoid and bias, 4 of 8 groups, a wavefront per token / this: 16384 tokens 29.9 / 13.3 (11.6 where none is done
// again), one 6.3 / 4.6; softmax over 128 experts, bf16, 16384 tokens 11.2 / 4.8.  The code of what is rare stands behind the rest: .5 of
// these us.
template <typename T, int PER, bool VEC>
__global__ void __launch_bounds__(64 * kGateWaves) topk_gating_rows_kernel(const T* __restrict__ logits, long ld,
                                                                           const float* __restrict__ bias, GateArgs a, int* __restrict__ ids,
                                                                           float* __restrict__ weights) {
  constexpr int kTokenPer = PER / 4;   // experts of a lane where a wavefront takes a token
  __shared__ uint32_t s_key[kGateWaves][64 * kTokenPer];
  const int lane = threadIdx.x & 63, l = lane & 15, w = threadIdx.x >> 6;
  const long t0 = ((long)blockIdx.x * kGateWaves + w) * 4;
  if (t0 >= a.tokens) return;   // (no barrier below)
  const long t = t0 + (lane >> 4);
  const bool in = t < a.tokens;
  const T* row = logits + (in ? t : t0) * ld;
  const float ninf = -__builtin_inff();
  float x[PER], b[PER];
  load_lane<VEC>(row, l * PER, a.experts, ninf, x);
  if (bias) {
    load_lane<VEC>(bias, l * PER, a.experts, 0.f, b);
  } else {
#pragma unroll
    for (int i = 0; i < PER; i++) b[i] = 0.f;
  }
  bool unsure = false;
  float top = 0, sum = 1;   // of the softmax over all experts
  if (!a.sigmoid && (a.exact || !a.renormalize)) {
    top = x[0];
    bool nan = x[0] != x[0];
#pragma unroll
    for (int i = 1; i < PER; i++) {
      top = __builtin_fmaxf(top, x[i]);
      nan |= x[i] != x[i];
    }
    top = row_max(top);
    unsure = nan;
    // e^x by 2^(x log2 e): off by |x - top| 2^-24 of itself, which is below .4 * 2^-24 of 1, and by a unit of the last place
    sum = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) sum += __builtin_amdgcn_exp2f((x[i] - top) * 1.44269504088896340736f);
    sum = row_sum(sum);
  }
  uint32_t key[PER];
  const bool whole = sizeof(T) == 2 && !a.exact;   // the keys hold all of a choice
  uint32_t near = 0;                               // keys' upper 24 bits no further apart than this may be in either order
  if (whole) {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const uint32_t k = order_key(x[i]);
      key[i] = (k & 0xffffff00u) | (uint32_t)(255 - (l * PER + i));   // (below 256: out)
    }
  } else {
    float choice[PER], slack = 0.f, lo = __builtin_inff(), any = 0.f;   // (any: NaN where a choice is)
    if (!a.exact) {
      float hi = x[0];
#pragma unroll
      for (int i = 1; i < PER; i++) hi = __builtin_fmaxf(hi, x[i]);
      lo = row_max(hi) - 64.f;   // (as below)
#pragma unroll
      for (int i = 0; i < PER; i++) {
        any += x[i] == ninf ? 0.f : x[i];
        choice[i] = x[i] == ninf ? ninf : __builtin_fmaxf(x[i], lo);
      }
    } else {
      const float scale = a.sigmoid ? 1.f : 1.0f / sum;
#pragma unroll
      for (int i = 0; i < PER; i++) {
        const float e = __builtin_amdgcn_exp2f((a.sigmoid ? -x[i] : x[i] - top) * 1.44269504088896340736f);
        const float c = (a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + e) : e * scale) + b[i];
        any += c;
        lo = __builtin_fminf(lo, c);
        choice[i] = x[i] == ninf ? ninf : c;
      }
      float largest = choice[0];
#pragma unroll
      for (int i = 1; i < PER; i++) largest = __builtin_fmaxf(largest, choice[i]);
      largest = row_max(largest);
      lo = -row_max(-lo);
      const bool far = lo < largest - 64.f;   // a bias that is -inf or very low
      if (__builtin_expect(far, 0)) {
        lo = __builtin_inff();
#pragma unroll
        for (int i = 0; i < PER; i++) lo = __builtin_fminf(lo, choice[i] == ninf ? __builtin_inff() : choice[i]);
        lo = -row_max(-lo);
      }
      // in units of 2^-24: a sigmoid's error is below 3.8 (|x| s (1 - s) < .23 from the argument's rounding, .5 from 2^x, 1 and 2 from the
      // sum and its reciprocal), a softmax's below 33 of the largest score (its sum's 20 additions and the mean |x - top| of its terms
      // among them); and half a unit of the last place for the fp32 sum on either side
      const float err = a.sigmoid ? 2.5e-7f : 2e-6f * scale;
      if (a.groups > 1) {
        float first = choice[0], second = ninf;
#pragma unroll
        for (int i = 1; i < PER; i++) {
          const float low = __builtin_fminf(first, choice[i]);
          first = __builtin_fmaxf(first, choice[i]);
          second = __builtin_fmaxf(second, low);
        }
        const int lanes = a.experts / a.groups / PER;   // of a group: a power of two
        auto join = [&](float f, float s) {
          const float low = __builtin_fminf(first, f), high = __builtin_fmaxf(second, s);
          first = __builtin_fmaxf(first, f);
          second = __builtin_fmaxf(low, high);
        };
        auto other = [](float v, auto ctrl) {
          return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, true));
        };
        if (lanes > 1) join(other(first, std::integral_constant<int, 0xB1>()), other(second, std::integral_constant<int, 0xB1>()));
        if (lanes > 2) join(other(first, std::integral_constant<int, 0x4E>()), other(second, std::integral_constant<int, 0x4E>()));
        if (lanes > 4) join(other(first, std::integral_constant<int, 0x141>()), other(second, std::integral_constant<int, 0x141>()));
        const float score = first == ninf ? ninf : first + (second == ninf ? 0.f : second);
        int sure = 0, maybe = 0;
        // (two scores of two choices each; a sum, of up to twice the largest, is rounded on either side too: half of the 2.5e-7)
        compare_rotated<1>(score, 4.f * (err + 2.5e-7f * __builtin_fmaxf(largest, -lo)), lanes, sure, maybe);
        // (a sum that overflowed says nothing)
        unsure |= (sure < a.topk_groups ? maybe >= a.topk_groups : false) || (score == ninf && first != ninf);
        if (sure >= a.topk_groups) {
#pragma unroll
          for (int i = 0; i < PER; i++) choice[i] = ninf;
        }
      }
      if (__builtin_expect(far, 0)) {   // (what lies far below the largest is hardly taken: it gets one key, and is close to its like)
        lo = __builtin_fmaxf(lo, largest - 64.f);
#pragma unroll
        for (int i = 0; i < PER; i++) choice[i] = choice[i] == ninf ? ninf : __builtin_fmaxf(choice[i], lo);
      }
      slack = err + 1.25e-7f * __builtin_fmaxf(largest, -lo);
    }
    float hi = choice[0];
#pragma unroll
    for (int i = 1; i < PER; i++) hi = __builtin_fmaxf(hi, choice[i]);
    hi = row_max(hi);
    // fixed point from 1 on; an expert that is out gets 0
    const float units = 16777200.f / (hi > lo ? hi - lo : 1.f);   // (its own rounding and the products' stay below 2^24)
    // (three units of rounding on either side; where the units are not finite numbers nothing is sure)
    const float apart = 2.f * slack * units + 6.f;
    unsure |= any != any || hi == __builtin_inff() || (!(apart < 16777216.f) && hi != ninf);
    near = (uint32_t)apart;
    const uint32_t place = 255 - l * PER;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const uint32_t q = (uint32_t)__builtin_fmaxf(__builtin_fmaf(choice[i] - lo, units, 1.f), 0.f);   // (the conversion's own clamp)
      key[i] = (q << 8) + (place - i);
    }
  }
  uint32_t place_key = 0;   // lane j of a token: the key of its place j
  uint32_t before = 0;   // (as if 2^32: every key is below)
  bool left = true, close = false;
  auto next = [&]() {   // the largest key below the last one, if there is one; whether it is near that
    uint32_t d = key[0] - before;
#pragma unroll
    for (int i = 1; i < PER; i++) {
      const uint32_t o = key[i] - before;
      d = d > o ? d : o;
    }
    d = row_reduce(d, [](uint32_t u, uint32_t v) { return u > v ? u : v; });
    const uint32_t max = left ? before + d : 0;
    left = max >= 256u;
    const bool by = left && (before >> 8) - (max >> 8) <= near;
    before = left ? max : 0;
    return by;
  };
  for (int j = 0; j < a.topk + (whole ? 0 : 1); j++) {   // (one more than are taken: how close it came)
    const bool by = next();
    if (l == j) place_key = before;
    close |= !whole && j > 0 && by;
  }
  int mine = place_key ? 255 - (int)(place_key & 255u) : -1;   // lane j: the j-th expert
  if (__builtin_expect(__ballot(close) != 0, 0)) {
    // Experts of one logit and one bias have one choice and go by their index, as their keys do; other neighbours that are near are in doubt.
    struct Expert { float x, b; };
    auto same = [](Expert u, Expert v) { return u.x == v.x && u.b == v.b; };
    auto expert = [&](bool is, int e) { return is ? Expert{gate_load(row + e), bias ? bias[e] : 0.f} : Expert{ninf, 0.f}; };
    auto lane_behind = [](auto v) {   // row_shl:1
      return __builtin_bit_cast(decltype(v), __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x101, 0xf, 0xf, true));
    };
    const Expert own = expert(mine >= 0, mine), spare = expert(left, 255 - (int)(before & 255u));   // (spare: the first that is not taken)
    Expert behind = {lane_behind(own.x), lane_behind(own.b)};
    uint32_t key_behind = lane_behind(place_key);
    if (l == a.topk - 1) {
      behind = spare;
      key_behind = before;
    }
    const bool near_next = l < a.topk && key_behind != 0 && (place_key >> 8) - (key_behind >> 8) <= near;
    const uint32_t doubts = (uint32_t)(__ballot(near_next && !same(own, behind)) >> (lane & 48)) & 0xffffu;
    const bool cut = (__ballot(near_next) >> (lane & 48)) >> (a.topk - 1) & 1;   // the spare one is near the last place
    if (__ballot(cut)) {
      // What is near the spare one has to be the same, and nothing else may be in doubt; of one more nothing is known.
      const bool second = next();
      const Expert e = expert(second, 255 - (int)(before & 255u));
      const bool third = next();
      unsure |= cut && second && (third || doubts || !same(e, spare));
      unsure |= cut && doubts && a.topk > 15;   // (no lane for the spare one)
    }
    if (__ballot(doubts != 0)) {
      // The taken ones and the spare one by their exact choices, a lane each (softmax scores hang on all experts: they are left to gate_token).
      unsure |= doubts && a.exact && !a.sigmoid;
      uint32_t exact = 0;
      int id = 256 + l;
      if (mine >= 0) {
        id = mine;
        exact = order_key(a.exact ? (float)(1.0 / (1.0 + exp(-(double)own.x)) + (double)own.b) : own.x);
      }
      const int to = order_rotated<1>(exact, id);
      const int sorted = __builtin_amdgcn_ds_permute(((lane & 48) + to) * 4, mine);
      if (doubts) mine = sorted;
    }
  }
  if (l >= a.topk) mine = -1;
  // the weights, a lane per place
  const bool real = mine >= 0;
  const float xs = real ? gate_load(row + mine) : ninf;
  float v;
  if (!a.renormalize) {
    v = a.sigmoid ? 1.0f / (1.0f + expf(-xs)) : expf(xs - top) / sum;
  } else {
    unsure |= xs != xs;
    v = gate_term(xs, row_max(xs), a.sigmoid);
    v = real ? v : 0.f;
    v /= row_sum(v);
  }
  const unsigned long long again = __ballot(unsure);
  const bool mine_again = (again >> (lane & 48)) & 0xffff;
  if (in && l < a.topk && !mine_again) {
    ids[t * a.topk + l] = mine;
    weights[t * a.topk + l] = real ? v * a.scale : 0.f;
  }
  if (__builtin_expect(again == 0, 1)) return;
  for (int r = 0; r < 4; r++)
    if (t0 + r < a.tokens && (again >> (16 * r) & 0xffff))
      gate_token<T, kTokenPer>(logits + (t0 + r) * ld, bias, a, s_key[w], ids + (t0 + r) * a.topk, weights + (t0 + r) * a.topk);
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
    float v = real ? gate_term(xs, m, a.sigmoid) : 0.f;
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
    out[t * a.experts + e] = gate_round<T>(v);
  }
}

// The same by sixteen lanes per token, under the conditions of topk_gating_rows_kernel: a token's logits are read once, in whole pieces,
// and its gradient is written so; the places' terms meet their experts in LDS.  A place whose id an earlier one has leaves its term to
// that one.  us, a wavefront per token / this: 16384 tokens, softmax over all, 256 experts fp32
// 16.2 / 11.5, 128 experts bf16 11.5 / 5.0.
template <typename T, int PER, bool VEC>
__global__ void __launch_bounds__(64 * kGateWaves) topk_gating_backward_rows_kernel(const float* __restrict__ grad,
                                                                                    const T* __restrict__ logits, long ld,
                                                                                    const int* __restrict__ ids, GateArgs a,
                                                                                    T* __restrict__ out) {
  __shared__ float __attribute__((aligned(16))) s_grad[kGateWaves][4][16 * PER];
  const int lane = threadIdx.x & 63, l = lane & 15, w = threadIdx.x >> 6;
  const long t0 = ((long)blockIdx.x * kGateWaves + w) * 4;
  if (t0 >= a.tokens) return;   // (no barrier below)
  const long t = t0 + (lane >> 4);
  const bool in = t < a.tokens;
  const T* row = logits + (in ? t : t0) * ld;
  const bool dense = !a.sigmoid && !a.renormalize;
  float x[PER];
  if (dense) load_lane<VEC>(row, l * PER, a.experts, -__builtin_inff(), x);
  int id = in && l < a.topk ? ids[t * a.topk + l] : -1;
  if ((unsigned)id >= (unsigned)a.experts) id = -1;
  const bool real = id >= 0;
  const float g = real ? grad[t * a.topk + l] * a.scale : 0.f;
  const float xs = real ? gate_load(row + id) : -__builtin_inff();
  float* mine = s_grad[w][lane >> 4];
#pragma unroll
  for (int i = 0; i < PER; i++) mine[l * PER + i] = 0.f;
  float d, mean = 0;
  if (dense) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < PER; i++) top = __builtin_fmaxf(top, x[i]);
    top = row_max(top);
    if (top == -__builtin_inff()) top = 0;   // every expert masked: all terms 0
    float sum = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      x[i] = expf(x[i] - top);
      sum += x[i];
    }
    sum = row_sum(sum);
    const float scale = 1.0f / (sum == 0 ? 1.f : sum);
#pragma unroll
    for (int i = 0; i < PER; i++) x[i] *= scale;   // the scores
    const float part = real ? g * (expf(xs - top) * scale) : 0.f;
    mean = row_sum(part);
    d = g;
  } else if (a.renormalize) {
    const float m = row_max_nan(xs);   // (with every lane)
    float v = real ? gate_term(xs, m, a.sigmoid) : 0.f;
    const float all = row_sum(v);
    v = real ? v / all : 0.f;
    const float mid = row_sum(g * v);
    d = real ? v * (g - mid) * (a.sigmoid ? 1.0f / (1.0f + expf(xs)) : 1.0f) : 0.f;
  } else {
    d = real ? g / (1.0f + expf(-xs)) / (1.0f + expf(xs)) : 0.f;
  }
  bool first = real;
  const float total = d + later_terms<1>(id, d, l, first);
  wave_lds_fence();
  if (first) mine[id] = total;
  wave_lds_fence();
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const float v = mine[l * PER + i];
    x[i] = dense ? x[i] * (v - mean) : v;
  }
  if (in) store_lane<VEC>(out + t * a.experts, l * PER, a.experts, x);
}

template <typename T>
static int launch_gating(const void* logits, long ld, const float* bias, const GateArgs& a, int* ids, float* weights, hipStream_t stream) {
  const int rows_per = a.experts <= 64 ? 4 : a.experts <= 128 ? 8 : 16;
  // Whether a group is a power of two of a sixteenth's lanes (1, 2, 4 or 8), or there are none.
  const int width = a.experts / a.groups, lanes = width / rows_per;
  const bool groups_fit = a.groups == 1 || (width == lanes * rows_per && lanes >= 1 && lanes <= 8 && (lanes & (lanes - 1)) == 0);
  if (a.experts <= 256 && a.topk <= 16 && groups_fit) {
    const unsigned grid = (unsigned)((a.tokens + 4 * kGateWaves - 1) / (4 * kGateWaves));
#define ESMOE_GATE(P)                                                                                                                \
  do {                                                                                                                               \
    constexpr int kPiece = P * sizeof(T) < 16 ? P : 16 / sizeof(T);                                                                  \
    const bool vec = a.experts % kPiece == 0 && ld % kPiece == 0 && (uintptr_t)logits % (kPiece * sizeof(T)) == 0 &&                  \
                     a.experts % 4 == 0 && (uintptr_t)bias % 16 == 0;                                                                \
    hipLaunchKernelGGL((vec ? topk_gating_rows_kernel<T, P, true> : topk_gating_rows_kernel<T, P, false>), dim3(grid),               \
                       dim3(64 * kGateWaves), 0, stream, (const T*)logits, ld, bias, a, ids, weights);                               \
  } while (0)
    if (rows_per == 4) ESMOE_GATE(4);
    else if (rows_per == 8) ESMOE_GATE(8);
    else ESMOE_GATE(16);
#undef ESMOE_GATE
    return (int)hipGetLastError();
  }
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
  if (a.experts <= 256 && a.topk <= 16) {
    const unsigned grid = (unsigned)((a.tokens + 4 * kGateWaves - 1) / (4 * kGateWaves));
#define ESMOE_GATE(P)                                                                                                                \
  do {                                                                                                                               \
    constexpr int kPiece = P * sizeof(T) < 16 ? P : 16 / sizeof(T);                                                                  \
    const bool vec = a.experts % kPiece == 0 && ld % kPiece == 0 && (uintptr_t)logits % (kPiece * sizeof(T)) == 0 &&                  \
                     (uintptr_t)out % (kPiece * sizeof(T)) == 0;                                                                     \
    hipLaunchKernelGGL((vec ? topk_gating_backward_rows_kernel<T, P, true> : topk_gating_backward_rows_kernel<T, P, false>),         \
                       dim3(grid), dim3(64 * kGateWaves), 0, stream, grad, (const T*)logits, ld, ids, a, (T*)out);                   \
  } while (0)
    if (a.experts <= 64) ESMOE_GATE(4);
    else if (a.experts <= 128) ESMOE_GATE(8);
    else ESMOE_GATE(16);
#undef ESMOE_GATE
    return (int)hipGetLastError();
  }
  const unsigned grid = (unsigned)((a.tokens + kGateWaves - 1) / kGateWaves);
  hipLaunchKernelGGL((topk_gating_backward_kernel<T>), dim3(grid), dim3(64 * kGateWaves), 0, stream, grad, (const T*)logits, ld, ids, a,
                     (T*)out);
  return (int)hipGetLastError();
}

}  // namespace esmoe

namespace {
// A launch of some of the tokens, from t on: a grid holds fewer than 2^32 threads.
constexpr long kGateStep = 1L << 24;
template <typename Launch>
int gate_steps(int dtype, const esmoe::GateArgs& a, Launch launch) {
  int rc = 0;
  for (long t = 0; t < a.tokens && rc == 0; t += kGateStep) {
    esmoe::GateArgs some = a;
    some.tokens = a.tokens - t < kGateStep ? a.tokens - t : kGateStep;
    rc = dtype == esmoe::kGateF32 ? launch(float(), t, some) : dtype == esmoe::kGateF16 ? launch(_Float16(), t, some) : launch(__bf16(), t, some);
  }
  return rc;
}
}  // namespace

extern "C" int esmoe_launch_topk_gating(const void* logits, int dtype, long ld, const float* bias, const esmoe::GateArgs* a, int* ids,
                                        float* weights, hipStream_t stream) {
  return gate_steps(dtype, *a, [=](auto type, long t, const esmoe::GateArgs& some) {
    using T = decltype(type);
    return esmoe::launch_gating<T>((const T*)logits + t * ld, ld, bias, some, ids + t * a->topk, weights + t * a->topk, stream);
  });
}

extern "C" int esmoe_launch_topk_gating_backward(const float* grad, const void* logits, int dtype, long ld, const int* ids,
                                                 const esmoe::GateArgs* a, void* out, hipStream_t stream) {
  return gate_steps(dtype, *a, [=](auto type, long t, const esmoe::GateArgs& some) {
    using T = decltype(type);
    return esmoe::launch_gating_backward<T>(grad + t * a->topk, (const T*)logits + t * ld, ld, ids + t * a->topk, some,
                                            (T*)out + t * a->experts, stream);
  });
}
