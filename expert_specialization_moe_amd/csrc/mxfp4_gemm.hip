// Grouped product of few rows per expert with 4-bit weights: bf16/fp16 activations, e2m1 weights, one E8M0 scale per 32 along K.
//
//   out[off_e + m, n] = cast( sum_k a[off_e + m, k] * e2m1(b[e, n, k]) * 2^(sf[e, n, k / 32] - 127) )
//   swiglu form, n = 2 * inter, gate rows first: out[off_e + m, i] = cast( silu(gate) * up ) of the two fp32 sums
//
// Decode: every weight of an expert with rows is read once, 17/32 bytes each, and used for a handful of rows; the bound is HBM.
// The 4-bit codes become bf16/fp16 values exactly (v_cvt_scalef32_pk_*_fp4) and go through v_mfma_f32_16x16x32 with up to sixteen rows of
// `a`.  A product of 32 columns belongs to one scale: where the scaled value is exact in the 16-bit type the conversion takes it in,
// otherwise the product's fp32 result is multiplied by it as it is added up, so that no range of scales is lost.
//
// The wavefronts of a workgroup split K; their sums are added in LDS in wavefront order.  No counterpart in the reference (its operators are
// 8-bit).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "mxfp4_units.h"
#include "swiglu.h"
#include "wave_scan.h"

namespace esmoe {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kLongWaves = 8;

// Eight weights of a dword as values of the activations' type.
template <bool FP16>
__device__ __forceinline__ v4i fp4_values(uint32_t w, float scale) {
  v4i r;
  if constexpr (FP16) {
    r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0));
    r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1));
    r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2));
    r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3));
  } else {
    r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
    r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
  }
  return r;
}

template <bool FP16>
__device__ __forceinline__ v4f mfma32(v4i a, v4i b, v4f c) {
  if constexpr (FP16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

// 2^(code - 127); NaN for 255.
__device__ __forceinline__ float e8m0(uint32_t code) {
  return __builtin_bit_cast(float, code == 0 ? 0x00400000u : code == 255 ? 0x7fc00000u : code << 23);
}

// Dword i of lane row r (sixteen lanes) goes to dword r of lane row i.
__device__ __forceinline__ void transpose_rows(uint32_t* d) {
  auto swap32 = [](uint32_t& x, uint32_t& y) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    x = r[0];
    y = r[1];
  };
  auto swap16 = [](uint32_t& x, uint32_t& y) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
    x = r[0];
    y = r[1];
  };
  swap32(d[0], d[2]);
  swap32(d[1], d[3]);
  swap16(d[0], d[1]);
  swap16(d[2], d[3]);
}

template <bool FP16>
__device__ __forceinline__ uint16_t to_half(float v) {
  if constexpr (FP16) return __builtin_bit_cast(uint16_t, (_Float16)v);
  else return __builtin_bit_cast(uint16_t, (__bf16)v);
}

// A barrier that orders LDS alone: loads from memory stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The units of a launch: experts in order, each in tiles of sixteen rows; a lane per expert, 64 at a time.
struct Fp4Units {
  int m, off;
  uint32_t end;   // units up to and with the lane's expert, from the 64's first on
  __device__ __forceinline__ void read(int e0, const int* __restrict__ problem_sizes, const int* __restrict__ expert_offsets, int num_experts,
                                       int total_rows) {
    const int e = e0 + (threadIdx.x & 63);
    m = off = 0;
    if (e < num_experts) {
      m = problem_sizes[e * 3];
      off = expert_offsets[e];
    }
    m = fp4_rows(m, off, total_rows);
    end = wave_inclusive_sum_or_most(fp4_tiles(m));
  }
  __device__ __forceinline__ uint32_t count() const { return (uint32_t)__builtin_amdgcn_readlane((int)end, 63); }
  __device__ __forceinline__ Fp4Unit unit(int e0, uint32_t u) const {   // u < count()
    const int l = __builtin_ctzll(__ballot(end > u));
    const uint32_t start = l ? (uint32_t)__builtin_amdgcn_readlane((int)end, l - 1) : 0u;
    return fp4_unit(e0 + l, __builtin_amdgcn_readlane(off, l), __builtin_amdgcn_readlane(m, l), u, start);
  }
};

// For a K whose sixteen rows of `a` are more than a workgroup's registers: a workgroup takes two tiles of sixteen weight rows (one of the
// gate's and one of the up projection's) for sixteen rows of `a`, which come from a cache as they are needed; its wavefronts split K.
// Bound by the loads it has in flight, a chunk's per wavefront (64 registers, eight wavefronts a SIMD): 16 experts x 2048 x K 12288, a row
// each 67.6 us (3.1 TB/s), 16 rows 99; with four tiles 71 and 84, but two experts of K 14336 44 instead of 23; non-temporal loads of the
// weights, half a line each, 72.7.
template <bool FP16, bool SWIGLU>
__global__ void __launch_bounds__(64 * kLongWaves) mxfp4_long_kernel(const uint16_t* __restrict__ a, const uint8_t* __restrict__ b,
                                                                     const uint8_t* __restrict__ sf, const int* __restrict__ problem_sizes,
                                                                     const int* __restrict__ expert_offsets, int num_experts, int total_rows,
                                                                     int n, int k, int col_tiles, int unit0, uint16_t* __restrict__ out) {
  constexpr int kCols = SWIGLU ? 16 : 32;   // of the output
  __shared__ float s_sum[kLongWaves][2][kFp4Rows][16];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int l16 = lane & 15, lr = lane >> 4;
  const int unit = blockIdx.x / col_tiles, col0 = (blockIdx.x - unit * col_tiles) * kCols;
  Fp4Unit g = {0, 0, 0};
  uint32_t u = unit0 + unit;
  for (int e0 = 0; e0 < num_experts; e0 += 64) {
    Fp4Units some;
    some.read(e0, problem_sizes, expert_offsets, num_experts, total_rows);
    if (u < some.count()) {
      g = some.unit(e0, u);
      break;
    }
    u -= some.count();
  }
  if (g.rows == 0) return;   // the whole workgroup
  const int wide = SWIGLU ? n / 2 : n;   // columns of the output
  const long kb = k / 2, ks = k / 32;
  const uint8_t* bp[2];
  const uint8_t* sp[2];
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const int col = SWIGLU ? t * wide + col0 : col0 + t * 16;   // (a tile beyond the last column is the last one again, and not stored)
    const long row = (long)g.expert * n + (col < n ? col : n - 16) + l16;
    bp[t] = b + row * kb + lr * 16;
    sp[t] = sf + row * ks;
  }
  const bool has_row = l16 < g.rows;   // (loads of a row that is not there: 69 us instead of 67.6)
  const uint16_t* ap = a + (long)(g.row0 + (has_row ? l16 : 0)) * k + lr * 8;
  v4f acc[2];
#pragma unroll
  for (int t = 0; t < 2; t++) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};
  const int chunks = k / 128, end = (int)((long)chunks * (w + 1) / kLongWaves);
  for (int c = (int)((long)chunks * w / kLongWaves); c < end; c++) {
    uint32_t d[2][4], s[2];
    v4i x[4];
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const v4i raw = *(const v4i*)(bp[t] + c * 64);   // (half a line: the other half is the next chunk's)
#pragma unroll
      for (int i = 0; i < 4; i++) d[t][i] = (uint32_t)raw[i];
      s[t] = *(const uint32_t*)(sp[t] + c * 4);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[i] = v4i{0, 0, 0, 0};
      if (has_row) x[i] = *(const v4i*)(ap + c * 128 + i * 32);
    }
#pragma unroll
    for (int t = 0; t < 2; t++) {
      transpose_rows(d[t]);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const v4f p = mfma32<FP16>(x[i], fp4_values<FP16>(d[t][i], 1.0f), v4f{0.f, 0.f, 0.f, 0.f});
        const float scale = e8m0(s[t] >> (8 * i) & 0xff);
#pragma unroll
        for (int r = 0; r < 4; r++) acc[t][r] = __builtin_fmaf(p[r], scale, acc[t][r]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int r = 0; r < 4; r++) s_sum[w][t][lr * 4 + r][l16] = acc[t][r];
  __syncthreads();
  for (int i = tid; i < g.rows * kCols; i += 64 * kLongWaves) {
    const int m = i / kCols, col = i % kCols;
    if (col0 + col >= wide) continue;
    float y = 0, up = 0;
    for (int u = 0; u < kLongWaves; u++) {
      y += s_sum[u][col >> 4][m][col & 15];
      if constexpr (SWIGLU) up += s_sum[u][1][m][col];
    }
    if constexpr (SWIGLU) y = swiglu_f32(y, up);
    out[(long)(g.row0 + m) * wide + col0 + col] = to_half<FP16>(y);
  }
}

// Sixteen rows of `a` stay in registers: wavefront w of a workgroup holds their K range of up to four pairs of chunks (a chunk is 128
// columns, a pair 128 bytes of weights), and the workgroup streams tiles of sixteen weight rows past them, two tiles a step (SwiGLU: the
// gate's and the up projection's; otherwise neighbours).  A step's partial sums meet in LDS; a tile's registers are loaded again as soon
// as it is used up, and the barrier waits for LDS alone.  The tiles' scales come in whole, two dwords per thread, a step ahead.  The steps
// of all units are one line that is cut evenly over the workgroups, as many as are resident at once.
//
// A load takes 128 bytes of eight rows (whole cache lines); lanes eight apart then trade halves, so that a lane has one row's chunk.
// A lane's sixteen bytes are the 32 columns of one scale, which goes into the conversion: the value is exact in bf16 up to a scale of
// 2^125, in fp16 from 2^-23 to 2^13.  A step that meets other scales is done again by fp4_any_scale.
constexpr int kFp4MaxWaves = 8, kFp4MaxPairs = 4;
// Wavefronts of a CU, by the pairs of chunks that each holds registers for (110, 160, 210 and 256 of them; with four pairs none spill, but
// 18 to 60 scalar ones do, into lanes).
constexpr int fp4_waves(int pairs) { return pairs == 1 ? 16 : pairs == 2 ? 12 : 8; }

struct Fp4Args {
  const uint16_t* a;
  const uint8_t *b, *sf;
  const int *problem_sizes, *expert_offsets;
  int num_experts, total_rows, n, k;
  uint32_t most_units;
  uint16_t* out;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_bytes(const uint8_t* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00027000);
}

// Lanes with bit 3 clear keep x and get y's place of the lane eight above in y; lanes with it set the other way round.
__device__ __forceinline__ void trade_halves(v4i& x, v4i& y) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int a = x[i], b = y[i];
    x[i] = __builtin_amdgcn_update_dpp(a, b, 0x128, 0xf, 0xc, false);   // row_ror:8 into lanes 8 .. 15
    y[i] = __builtin_amdgcn_update_dpp(b, a, 0x128, 0xf, 0x3, false);   // into lanes 0 .. 7
  }
}

// Sums of `count` chunks of sixteen weight rows times sixteen rows of `a`, whatever the scales: a product of 32 columns is multiplied by
// its scale when it is added up.  src, ssrc, ap: the lane's row (l16) and, of the bytes and columns, its lane row's first.
template <bool FP16>
__device__ __forceinline__ v4f fp4_any_scale(const uint8_t* src, const uint8_t* ssrc, const uint16_t* ap, bool has_row, int count) {
  v4f acc = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < count; c++) {
    const v4i raw = *(const v4i*)(src + c * 64);
    const uint32_t s = *(const uint32_t*)(ssrc + c * 4);
    v4i x[4];
    uint32_t d[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[i] = v4i{0, 0, 0, 0};
      if (has_row) x[i] = *(const v4i*)(ap + c * 128 + i * 32);
      d[i] = (uint32_t)raw[i];
    }
    transpose_rows(d);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const v4f r = mfma32<FP16>(x[i], fp4_values<FP16>(d[i], 1.0f), v4f{0.f, 0.f, 0.f, 0.f});
      const float scale = e8m0(s >> (8 * i) & 0xff);
#pragma unroll
      for (int q = 0; q < 4; q++) acc[q] = __builtin_fmaf(r[q], scale, acc[q]);
    }
  }
  return acc;
}

template <bool FP16, bool SWIGLU, int PAIRS>
__global__ void __launch_bounds__(64 * kFp4MaxWaves) __attribute__((amdgpu_waves_per_eu(fp4_waves(PAIRS) / 4)))
mxfp4_stream_kernel(Fp4Args p) {
  constexpr int kChunks = 2 * PAIRS;
  constexpr uint32_t kLeast = FP16 ? 104 : 0, kSpan = FP16 ? 36 : 252;   // scale codes of exact values
  extern __shared__ uint32_t s_mem[];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
  const int l16 = lane & 15, lr = lane >> 4;
  const int chunks = p.k / 128, pairs = (chunks + 1) / 2;
  float* s_part = (float*)s_mem;                    // [2 steps][2 tiles][wavefronts][256]
  uint32_t* s_scale = s_mem + 1024 * waves;         // [2 steps][2 tiles][chunks][16 rows]
  uint32_t* s_far = s_scale + 64 * chunks;          // [2 steps]: whether a wavefront met a scale that needs fp4_any_scale
  const int inter = p.n / 2;
  const int steps = SWIGLU ? p.n / 32 : (p.n / 16 + 1) / 2;   // of a unit
  const long kb = p.k / 2, ks = p.k / 32;
  const int p0 = pairs * w / waves, c0 = 2 * p0;
  const int count = 2 * (pairs * (w + 1) / waves) < chunks ? 2 * (pairs * (w + 1) / waves) - c0 : chunks - c0;   // (1 .. kChunks)
  Fp4Units some;
  some.read(0, p.problem_sizes, p.expert_offsets, p.num_experts, p.total_rows);
  uint32_t units = some.count();
  for (int e0 = 64; e0 < p.num_experts; e0 += 64) {
    Fp4Units more;
    more.read(e0, p.problem_sizes, p.expert_offsets, p.num_experts, p.total_rows);
    units = sum_or_most(units, more.count());
  }
  // (more where experts claim the same rows; the launch sees to it that the steps of these are fewer than 2^31)
  units = units < p.most_units ? units : p.most_units;
  const uint32_t total = units * steps, share = total / gridDim.x, rest = total % gridDim.x;
  uint32_t at = blockIdx.x * share + (blockIdx.x < rest ? blockIdx.x : rest);
  const uint32_t end = at + share + (blockIdx.x < rest ? 1 : 0);
  // The lane's place in the wavefront's bytes of eight weight rows: row l16 % 8, half l16 / 8 of a pair's line (a pair that ends a row of
  // an odd number of chunks has one half: taken twice, times zeros of `a`; so is the last pair of a wavefront that has only one).
  uint32_t wlane[PAIRS];
#pragma unroll
  for (int q = 0; q < PAIRS; q++) {
    const int pair = 2 * q < count ? q : 0;
    wlane[q] = (uint32_t)((l16 & 7) * (int)kb + pair * 128 + (l16 >= 8 && 2 * pair + 1 < count ? 64 : 0) + lr * 16);
  }
  // the thread's two dwords of a tile's scales, [16 rows][chunks] in memory, [chunks][16 rows] in LDS
  int splace[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int at = tid + i * (int)blockDim.x, row = at / chunks;
    splace[i] = row < 16 ? (at - row * chunks) * 16 + row : -1;
  }
  if (tid < 2) s_far[tid] = 0;   // (before the first step's barrier)
  int e0 = 0;
  uint32_t before = 0;   // `some` holds the experts from e0 on, whose units are those from `before` on
  int buf = 0;
  while (at < end) {
    const uint32_t unit = at / steps;
    int step = (int)(at - unit * steps);
    const int last = end - unit * steps < (uint32_t)steps ? (int)(end - unit * steps) : steps;
    while (unit >= sum_or_most(before, some.count())) {   // (ends: unit is less than all counts together)
      before += some.count();
      e0 += 64;
      some.read(e0, p.problem_sizes, p.expert_offsets, p.num_experts, p.total_rows);
    }
    const Fp4Unit g = some.unit(e0, unit - before);
    const uint8_t* bw = p.b + (long)g.expert * p.n * kb + p0 * 128;
    const uint8_t* sw = p.sf + (long)g.expert * p.n * ks;
    v4i wt[2][kChunks];
    uint32_t sc[2][2];
    auto first_row = [&](int h, int st) {   // of half h of step st; the second half of a last step that has none: the one before
      const int row = SWIGLU ? h * inter + st * 16 : st * 32 + h * 16;
      return (long)(!SWIGLU && row >= p.n ? p.n - 16 : row);
    };
    // (descriptors of a tile's bytes: a lane's place in them is all that the loads take from vector registers, and a dword past the
    // tile's scales reads as 0)
    auto load = [&](int q, int h, int st, bool some) {   // pair q of the wavefront's range; none: zeros, without a read
      const auto src = tile_bytes(bw + first_row(h, st) * kb, some ? (int)(16 * kb) - p0 * 128 : 0);
#pragma unroll
      for (int r = 0; r < 2; r++) wt[h][2 * q + r] = __builtin_amdgcn_raw_buffer_load_b128(src, wlane[q], r * 8 * (int)kb, 0);
    };
    auto load_scales = [&](int st) {
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int i = 0; i < 2; i++)
          sc[h][i] = __builtin_amdgcn_raw_buffer_load_b32(tile_bytes(sw + first_row(h, st) * ks, 16 * (int)ks), (tid + i * (int)blockDim.x) * 4, 0, 0);
    };
    auto store_scales = [&](int b) {
#pragma unroll
      for (int i = 0; i < 2; i++)
        if (splace[i] >= 0) {
          s_scale[(b * 2 + 0) * 16 * chunks + splace[i]] = sc[0][i];
          s_scale[(b * 2 + 1) * 16 * chunks + splace[i]] = sc[1][i];
        }
    };
    load_scales(step);
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int q = 0; q < PAIRS; q++) load(q, h, step, true);
    __builtin_amdgcn_sched_barrier(0);   // (ahead of the rows of `a`, which come from a cache)
    v4i x[kChunks][4];
    {
      const bool has_row = l16 < g.rows;
      const uint16_t* ap = p.a + (long)(g.row0 + (has_row ? l16 : 0)) * p.k + c0 * 128 + lr * 32;
#pragma unroll
      for (int j = 0; j < kChunks; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const v4i v = *(const v4i*)(ap + (j < count ? j : 0) * 128 + i * 8);
          x[j][i] = has_row && j < count ? v : v4i{0, 0, 0, 0};
        }
    }
    // The outputs of a step from its partial sums, in the wavefronts' order.
    auto finish = [&](int b, int st) {
      int t = tid, parts = waves;
      // (what follows from these is worked out here, not kept in registers over the steps; scalar ones are short with SwiGLU alone)
      if constexpr (SWIGLU) asm volatile("" : "+v"(t), "+s"(parts));
      else asm volatile("" : "+v"(t));
      for (; t < (SWIGLU ? 16 : 32) * g.rows; t += blockDim.x) {
        const int col = t & 15, h = SWIGLU ? 0 : t >> 4 & 1, m = SWIGLU ? t >> 4 : t >> 5;
        const float* part = s_part + b * 2 * parts * 256 + (m >> 2) * 64 + col * 4 + (m & 3);
        float f[SWIGLU ? 2 : 1][kFp4MaxWaves];
#pragma unroll
        for (int u = 0; u < (SWIGLU ? 2 : 1); u++)
#pragma unroll
          for (int i = 0; i < kFp4MaxWaves; i++) f[u][i] = part[((SWIGLU ? u : h) * parts + (i < parts ? i : 0)) * 256];
#pragma unroll
        for (int u = 0; u < (SWIGLU ? 2 : 1); u++)
#pragma unroll
          for (int i = 1; i < kFp4MaxWaves; i++) f[u][0] += i < parts ? f[u][i] : 0.f;
        const int c = SWIGLU ? st * 16 + col : st * 32 + h * 16 + col;
        float y = f[0][0];
        if constexpr (SWIGLU) y = swiglu_f32(y, f[1][0]);
        if (SWIGLU || c < p.n) p.out[(long)(g.row0 + m) * (SWIGLU ? inter : p.n) + c] = to_half<FP16>(y);
      }
    };
    store_scales(buf);
    lds_barrier();
    for (; step < last; step++) {
      // (the last step's loads are empty: 3 % where a workgroup has four steps, 8 experts x 4096 x 7168 31.2 / 30.2 us)
      const int next = step + 1 < last ? step + 1 : step;
      load_scales(next);
#pragma unroll
      for (int h = 0; h < 2; h++) {
        int code[kChunks];
        uint32_t far = 0;
#pragma unroll
        for (int j = 0; j < kChunks; j++) {
          const uint32_t four = s_scale[((buf * 2 + h) * chunks + c0 + (j < count ? j : 0)) * 16 + l16];
          code[j] = (int)__builtin_amdgcn_ubfe(four, lr * 8, 8);
          const uint32_t d = (uint32_t)code[j] - kLeast;
          far = far > d ? far : d;
        }
        v4f sum[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};   // (of even and odd chunks: two chains of matrix instructions)
        if (far > kSpan) s_far[buf] = 1;
#pragma unroll
        for (int q = 0; q < PAIRS; q++) {
          trade_halves(wt[h][2 * q], wt[h][2 * q + 1]);
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 2 * q; j < 2 * q + 2; j++)
              sum[j & 1] = mfma32<FP16>(x[j][i], fp4_values<FP16>((uint32_t)wt[h][j][i], __builtin_bit_cast(float, code[j] << 23)), sum[j & 1]);
          __builtin_amdgcn_sched_barrier(0);   // (a pair's registers are loaded again as soon as it is used up)
          load(q, h, next, step + 1 < last);
        }
        const v4f acc = sum[0] + sum[1];
        *(v4f*)&s_part[((buf * 2 + h) * waves + w) * 256 + lane * 4] = acc;
      }
      store_scales(buf ^ 1);
      lds_barrier();
      if (__builtin_amdgcn_readfirstlane(s_far[buf]) != 0) {
        lds_barrier();   // (everyone has seen it)
        if (tid == 0) s_far[buf] = 0;
#pragma unroll 1
        for (int h = 0; h < 2; h++) {
          int place = lane;
          asm volatile("" : "+v"(place));   // (as in finish)
          const int row = place & 15, part = place >> 4;
          const bool has_row = row < g.rows;
          *(v4f*)&s_part[((buf * 2 + h) * waves + w) * 256 + place * 4] = fp4_any_scale<FP16>(
              bw + (first_row(h, step) + row) * kb + part * 16, sw + (first_row(h, step) + row) * ks + c0 * 4,
              p.a + (long)(g.row0 + (has_row ? row : 0)) * p.k + c0 * 128 + part * 8, has_row, count);
        }
        lds_barrier();
      }
      finish(buf, step);
      buf ^= 1;
    }
    at = unit * steps + last;
  }
}

}  // namespace esmoe

extern "C" int esmoe_launch_mxfp4_grouped_mm(const void* a, int dtype, const void* b, const uint8_t* sf, const int* problem_sizes,
                                             const int* expert_offsets, int num_experts, int total_rows, int n, int k, int swiglu, void* out,
                                             int cus, hipStream_t stream) {
  using namespace esmoe;
  const int steps = swiglu ? n / 32 : (n / 16 + 1) / 2, chunks = k / 128, pairs = (chunks + 1) / 2;
  const long units = fp4_most_units(num_experts, total_rows), most = units * steps;
  if (pairs <= kFp4MaxPairs * kFp4MaxWaves && most < 1L << 31) {
    // As many wavefronts as a workgroup has, each with as little of K as that takes.  us, as few wavefronts as K takes / this:
    // 32 experts x 7168 x K 2048, a row each 49.2 / 46.3, eight rows 55.8 / 52.0; 8 experts, 64 rows each 44 / 37; 64 experts x 1536 x
    // K 4096, eight rows 46.6 / 45.8; (sixteen wavefronts of one workgroup instead of eight: 57.0).
    const int each = (pairs + kFp4MaxWaves - 1) / kFp4MaxWaves;
    const int waves = (pairs + each - 1) / each, per_cu = fp4_waves(each) / waves;
    const unsigned grid = (unsigned)(most < (long)cus * per_cu ? most : (long)cus * per_cu);
    const Fp4Args args{(const uint16_t*)a, (const uint8_t*)b, sf, problem_sizes, expert_offsets, num_experts, total_rows, n, k,
                       (uint32_t)units, (uint16_t*)out};
#define ESMOE_FP4(P)                                                                                                               \
  do {                                                                                                                             \
    auto kernel = dtype ? swiglu ? mxfp4_stream_kernel<true, true, P> : mxfp4_stream_kernel<true, false, P>                        \
                        : swiglu ? mxfp4_stream_kernel<false, true, P> : mxfp4_stream_kernel<false, false, P>;                     \
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * waves), 4096 * waves + 256 * chunks + 8, stream, args);                       \
  } while (0)
    if (each == 1) ESMOE_FP4(1);
    else if (each == 2) ESMOE_FP4(2);
    else if (each == 3) ESMOE_FP4(3);
    else ESMOE_FP4(4);
#undef ESMOE_FP4
    return (int)hipGetLastError();
  }
  const int cols = swiglu ? 16 : 32, col_tiles = ((swiglu ? n / 2 : n) + cols - 1) / cols;
  const long step = (1L << 22) / col_tiles > 1 ? (1L << 22) / col_tiles : 1;   // units of a launch: a grid holds fewer than 2^32 threads
  auto kernel = dtype ? swiglu ? mxfp4_long_kernel<true, true> : mxfp4_long_kernel<true, false>
                      : swiglu ? mxfp4_long_kernel<false, true> : mxfp4_long_kernel<false, false>;
  for (long u = 0; u < units; u += step) {
    const long some = units - u < step ? units - u : step;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(some * col_tiles)), dim3(64 * kLongWaves), 0, stream, (const uint16_t*)a, (const uint8_t*)b, sf,
                       problem_sizes, expert_offsets, num_experts, total_rows, n, k, col_tiles, (int)u, (uint16_t*)out);
  }
  return (int)hipGetLastError();
}
