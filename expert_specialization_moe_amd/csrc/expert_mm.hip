// Grouped products of the experts in 16 bits, with their gradients, and in 8-bit integers.
//
//   forward         out[off_e + m, j] = cast( sum_c a[off_e + m, c] * b[e, j, c] )
//   SwiGLU, n = 2 * inter, gate rows first: out = cast( silu(gate) * up ) of the two fp32 sums; gate_up = cast(sums), where asked for
//   rows' gradient  grad_a[off_e + m, c] = cast( sum_j grad_out[off_e + m, j] * b[e, j, c] )
//   weights'        grad_b[e, j, c] = cast( sum_m grad_out[off_e + m, j] * a[off_e + m, c] ), 0 for an expert without rows
//   int8            sums in int32 (exact), out = cast( sum * sa[off_e + m] * sb[e, j] )
// The reference has 8-bit floating point products alone and no gradients.
//
// One persistent workgroup of eight wavefronts per CU; a tile is 256 output rows ("T" operand) x 256 output columns ("W" operand; with
// SwiGLU 128 gate columns and the matching 128 up columns), the sum goes in steps of 128 bytes (64 16-bit elements).  A step's operands are
// copied from memory straight into LDS, in four parts of 16 KB (W0, T0, W1, T1: the halves of each operand), two steps deep.
//
// The step is four phases, a quarter of the tile each: (T0, W0), (T0, W1), (T1, W0), (T1, W1).  A phase is a memory half (fragments LDS ->
// registers, the copy of a part of a coming step), a barrier, a matrix half (16 MFMAs a wavefront), and a barrier.  The wavefronts form
// two groups of four, one wavefront of each per SIMD, and one group runs a barrier behind the other: while one feeds the matrix cores the
// other moves data.  No memory half waits for fragments that it reads itself: a trip to LDS is longer than it.
//     phase                      0                     1                  2                3
//     memory half reads          T0's 2nd half                            T1's 2nd half    W0 of the next step
//     memory half copies         T1 of +1              W0 of +2           T0 of +2         W1 of +2
//     memory half waits (copies) T1                                       W0, T0 of +1     W1 of +1
//     matrix half reads          W1                    T1's 1st half                       T0's 1st half of the next step
// A second half of T is waited for behind the first products of its matrix half; its registers are those of the half before, which the products
// are done with.  In half phases since the step's first, of the group that runs behind: W0 and T0's 1st half are read and waited for at 2
// (the end of phase 0's memory half), T0's 2nd half at 3, W1 at 5, T1 at 7.  The group that runs ahead copies into their places at 2 (W0),
// 4 (T0), 6 (W1) and 8 (T1).  And a part is read, by the group ahead, a barrier or more behind the memory half in which the group behind
// waits for its own shares of it: then four younger copies, of two instructions, may be on their way.
//
// The copies run on across tiles: their state is ahead of the one that multiplies, so that a tile begins with its first steps in LDS.
// They go through buffer descriptors: what lies beyond an expert's rows, the columns or the sum's length arrives as zeros without a load.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "expert_mm.h"
#include "expert_mm_rule.h"
#include "expert_mm_units.h"
#include "mxfp4_units.h"
#include "swiglu.h"
#include "wave_scan.h"

namespace esmoe {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));

enum { kForward = 0, kSwiglu = 1, kSwigluSave = 2, kRowsGrad = 3, kWeightsGrad = 4 };

constexpr int kMmThreads = 512;
constexpr int kPart = 16384, kMmStage = 4 * kPart;   // a half of an operand's step in LDS; a step
constexpr int kW0 = 0, kT0 = kPart, kW1 = 2 * kPart, kT1 = 3 * kPart;
constexpr uint32_t kNowhere = 0x80000000u;           // an offset beyond every descriptor
constexpr int kBias = 1024;                          // of descriptors: a copy's second half is 1024 bytes on in LDS and, by the same field, in memory

template <int TYPE> struct MmAcc { typedef v4f T; };
template <> struct MmAcc<kMmInt8> { typedef v4i T; };

// What a copy of two times 64 x 16 bytes into LDS needs: lds and 1024 bytes behind it, a descriptor, the lanes' offsets.
struct MmCopy {
  uint32_t lds;
  v4i rsrc;
  uint32_t v0, v1;
};
// STREAM: no cache is to keep it.
template <bool STREAM = false>
__device__ __forceinline__ void mm_copy(const MmCopy& p) {
  // (a scalar register that a vector instruction wrote is there for a memory instruction five slots on)
#define ESMOE_COPY(hint)                                                                                                            \
  asm volatile("s_mov_b32 m0, %[lds]\n\ts_nop 4\n\tbuffer_load_dwordx4 %[v0], %[rsrc], 0 offen" hint " lds\n\t"                     \
               "buffer_load_dwordx4 %[v1], %[rsrc], 0 offen offset:1024" hint " lds"                                                 \
               ::[lds] "s"(p.lds), [v0] "v"(p.v0), [v1] "v"(p.v1), [rsrc] "s"(p.rsrc) : "memory")   // (the compiler keeps nothing in m0)
  if constexpr (STREAM) ESMOE_COPY(" nt");
  else ESMOE_COPY("");
#undef ESMOE_COPY
}

// Products of a step: c[i][j] += rows of t[i] x columns of w[j], i = I, I + 1, j < 2; not where `rows` is at most LIMIT.  One statement with its branches
// inside: around the compiler's own matrix instructions a condition makes it copy the accumulators.  Between two products of one
// accumulator stand three others; whoever reads it next has to wait (mm_results).
// A matrix half is kBegin for the first two i (both halves of the step; raises the wave's priority), then kNext and kEnd for the others (a half of the
// step each).  kEnd has the barrier that ends the matrix half in front of its last four products, at a priority above the other group's first
// ones, which queue up behind them: without, the matrix cores idle from one group's last product until the other's first.
enum { kBegin, kNext, kEnd };
#define ESMOE_MMA(op, i, j, ks) op " %[c" #i #j "], %[w" #j #ks "], %[t" #i #ks "], %[c" #i #j "]\n\t"
#define ESMOE_MMA4(op, ks) ESMOE_MMA(op, 0, 0, ks) ESMOE_MMA(op, 0, 1, ks) ESMOE_MMA(op, 1, 0, ks) ESMOE_MMA(op, 1, 1, ks)
#define ESMOE_MMA_C [c00] "+v"(c[I][0]), [c01] "+v"(c[I][1]), [c10] "+v"(c[I + 1][0]), [c11] "+v"(c[I + 1][1])
#define ESMOE_MMA_IN(ks) [w0##ks] "v"(w[0][ks]), [w1##ks] "v"(w[1][ks]), [t0##ks] "v"(t[I][ks]), [t1##ks] "v"(t[I + 1][ks])
#define ESMOE_MMA_IF [rows] "s"(rows), [limit] "n"(LIMIT) : "scc", "memory"
#define ESMOE_SKIP "s_cmp_le_i32 %[rows], %[limit]\n\ts_cbranch_scc1 .Lesmoe_end%=\n\t"
#define ESMOE_PRODUCTS(op)                                                                                                            \
  if constexpr (PART == kBegin)                                                                                                       \
    asm volatile("s_setprio 1\n\t" ESMOE_SKIP ESMOE_MMA4(op, 0) ESMOE_MMA4(op, 1) ".Lesmoe_end%=:"                                    \
                 : ESMOE_MMA_C : ESMOE_MMA_IN(0), ESMOE_MMA_IN(1), ESMOE_MMA_IF);                                                     \
  else if constexpr (PART == kNext)                                                                                                   \
    asm volatile(ESMOE_SKIP ESMOE_MMA4(op, 0) ".Lesmoe_end%=:" : ESMOE_MMA_C : ESMOE_MMA_IN(0), ESMOE_MMA_IF);                        \
  else                                                                                                                                \
    asm volatile("s_setprio 2\n\ts_cmp_le_i32 %[rows], %[limit]\n\ts_barrier\n\ts_cbranch_scc1 .Lesmoe_end%=\n\t" ESMOE_MMA4(op, 1) ".Lesmoe_end%=:\n\ts_setprio 0" : ESMOE_MMA_C : ESMOE_MMA_IN(1), ESMOE_MMA_IF)
template <int TYPE, int PART, int I, int LIMIT>
__device__ __forceinline__ void products(typename MmAcc<TYPE>::T (&c)[4][2], const v4i (&w)[2][2], const v4i (&t)[4][2], int rows) {
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (TYPE == kMmInt8) { ESMOE_PRODUCTS("v_mfma_i32_16x16x64_i8"); }
  else if constexpr (TYPE == kMmFp16) { ESMOE_PRODUCTS("v_mfma_f32_16x16x32_f16"); }
  else { ESMOE_PRODUCTS("v_mfma_f32_16x16x32_bf16"); }
  __builtin_amdgcn_sched_barrier(0);
}
// In front of the first vector instruction that reads or writes an accumulator: the last product's result is there 7 issue slots on.
__device__ __forceinline__ void mm_results() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

struct MmShared {
  uint8_t ring[2 * kMmStage];
  int rows[kMmExperts], off[kMmExperts], order[kMmExperts];
  uint32_t unit_end[kMmExperts], units;   // running sums, in order
};
static_assert(sizeof(MmShared) <= 160 * 1024, "LDS");

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Until at most N of the wavefront's copies are on their way; MORE of its stores are younger than these where `stored` is set.
template <int N, int MORE>
__device__ __forceinline__ void mm_wait_copies(int stored) {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_cmp_lg_u32 %2, 0\n\ts_cbranch_scc1 .Lesmoe_wait%=\n\ts_waitcnt vmcnt(%0) ; explicit\n.Lesmoe_wait%=:\n\ts_waitcnt vmcnt(%1) ; explicit"
               ::"n"(N), "n"(N + MORE), "s"(uniform(stored)) : "memory", "scc");
}
template <int N>
__device__ __forceinline__ void mm_wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0) ; explicit" ::"n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void mm_wait_fragments() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(N < 15 ? N : 15) : "memory");
}
__device__ __forceinline__ void mm_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

struct MmTile {
  int expert;
  int row0, rows;   // of the tensor of rows (weights' gradient: of an expert's weights)
  int col0, width;  // of the output
  int steps;
};

// Which tiles a workgroup multiplies, one a round: experts by falling rows of a unit (the weights' gradient: rows), odd rounds dealt backwards, so that
// what a round is uneven in evens out.
template <int TYPE, int KIND>
struct MmTiles {
  const MmShared& s;
  const ExpertMmArgs& g;
  int cols, col_tiles, row_tiles;
  uint32_t total, rounds, last, split, place, per_round;

  static constexpr bool kSw = KIND == kSwiglu || KIND == kSwigluSave;
  static constexpr int kWide = kSw ? 128 : 256;

  __device__ __forceinline__ MmTiles(const MmShared& s_, const ExpertMmArgs& g_) : s(s_), g(g_) {
    cols = kSw ? g.n / 2 : KIND >= kRowsGrad ? g.k : g.n;
    col_tiles = (cols + kWide - 1) / kWide;
    row_tiles = (g.n + 255) / 256;
    total = (KIND == kWeightsGrad ? (uint32_t)g.num_experts * row_tiles : (uint32_t)uniform((int)s.units)) * col_tiles;
    // The last round's tiles in halves or quarters where there are workgroups for them (us whole and so: one expert x 1024 rows, 4096 x 7168, 142 / 126, with
    // SwiGLU 138 / 113; 9 x 300 rows, 4096 x 4096, 161 / 146, either way): by columns; with SwiGLU, whose gate and up columns no half of the products can leave out, by rows if more than 64.
    const uint32_t grid = gridDim.x, over = total % grid;
    split = over == 0 || over > grid / 2 ? 1 : over > grid / 4 ? 2 : 4;
    const uint32_t all = total < grid ? total * split : total;
    const MmPlace at = mm_place(all);
    place = at.place;
    per_round = at.of;
    rounds = place < all ? (total < grid ? 1 : (total + grid - 1) / grid) : 0;
    last = split > 1 ? (total < grid ? 0 : total / grid) : ~0u;   // the round of parts
  }

  // This workgroup's tile of a round; false where it has none.
  __device__ __forceinline__ bool tile(uint32_t round, MmTile& t) const {
    const uint32_t turn = round & 1 ? per_round - 1 - place : place, parts = round == last ? split : 1, q = turn / parts, part = turn - q * parts,
                   p = round * per_round + q;
    if (p >= total) return false;
    uint32_t first, units;   // of the expert's tiles; its rows' tiles
    int high = 256, m = 0;
    if constexpr (KIND == kWeightsGrad) {
      units = (uint32_t)row_tiles;
      const uint32_t rank = p / (units * col_tiles);
      first = rank * units * col_tiles;
      t.expert = uniform(s.order[rank]);
      t.steps = mm_steps(uniform(s.rows[t.expert]), 64);
    } else {
      // the expert whose units' running sum is the first above this unit
      const uint32_t unit = p / col_tiles;
      const int lane = threadIdx.x & 63;
      int rank = g.num_experts - 1;
      uint32_t before = 0;
      for (int e0 = 0; e0 < g.num_experts; e0 += 64) {
        const uint32_t end = e0 + lane < g.num_experts ? s.unit_end[e0 + lane] : 0xffffffffu;
        const unsigned long long past = __ballot(end > unit);
        if (past) {
          const int l = __builtin_ctzll(past);
          if (e0 + l < g.num_experts) rank = e0 + l;
          if (l) before = (uint32_t)__builtin_amdgcn_readlane((int)end, l - 1);
          break;
        }
        before = (uint32_t)__builtin_amdgcn_readlane((int)end, 63);
      }
      t.expert = uniform(s.order[rank]);
      m = uniform(s.rows[t.expert]);
      high = mm_unit_rows(m);
      units = mm_units(m);
      first = before * col_tiles;
      t.steps = KIND == kRowsGrad ? (g.n + 63) >> 6 : TYPE == kMmInt8 ? (g.k + 127) >> 7 : (g.k + 63) >> 6;
    }
    // four of the rows' tiles a group, a column's together: the 32 CUs of an XCD have four by eight tiles, which is the least to read (one expert
    // 16384 x 4096 x 4096, us with 2 x 16 tiles and 4 x 8: forward 417 / 407, the weights' gradient 425 / 418)
    const uint32_t i = p - first, group = i / (4 * col_tiles), j = i - group * 4 * col_tiles, have = units - 4 * group, wide = have < 4 ? have : 4,
                   col = j / wide, row = 4 * group + j - col * wide;
    const int from = (int)row * high;
    if constexpr (KIND == kWeightsGrad) {
      t.row0 = from;
      t.rows = g.n - from < 256 ? g.n - from : 256;
    } else {   // (the last unit may be short of rows, or without any)
      t.row0 = uniform(s.off[t.expert]) + from;
      t.rows = m - from < high ? m - from : high;
      if (t.rows <= 0) return false;
    }
    t.col0 = (int)col * kWide;
    t.width = kWide;
    if (parts > 1) {
      if (kSw && t.rows > 64) {
        const int piece = ((t.rows + (int)parts - 1) / (int)parts + 15) & ~15, at = (int)part * piece;
        t.row0 += at;
        t.rows = t.rows - at < piece ? t.rows - at : piece;
        if (t.rows <= 0) return false;
      } else {
        t.width = kWide / (int)parts;
        t.col0 += (int)part * t.width;
        if (t.col0 >= cols) return false;
      }
    }
    return true;
  }
};

// Reads the experts' rows and offsets, cut at the tensor's, and puts the experts in order.
template <int KIND>
__device__ __forceinline__ void mm_schedule(MmShared& s, const ExpertMmArgs& g) {
  const int tid = threadIdx.x;
  auto height = [&](int e) { return KIND == kWeightsGrad ? s.rows[e] : mm_unit_rows(s.rows[e]); };
  for (int e = tid; e < g.num_experts; e += kMmThreads) {
    const int off = g.expert_offsets[e];
    s.rows[e] = fp4_rows(g.problem_sizes[e * 3], off, g.total_rows);
    s.off[e] = off;
    s.unit_end[e] = (uint32_t)height(e);
  }
  __syncthreads();
  for (int e = tid; e < g.num_experts; e += kMmThreads) {
    const uint32_t h = s.unit_end[e];
    int rank = 0;
    for (int j = 0; j < g.num_experts; j++) rank += s.unit_end[j] > h || (s.unit_end[j] == h && j < e);
    s.order[rank] = e;
  }
  __syncthreads();
  if (KIND != kWeightsGrad && tid < 64) {
    uint32_t units = 0;
    for (int p0 = 0; p0 < g.num_experts; p0 += 64) {
      const int p = p0 + tid;
      const uint32_t end = sum_or_most(units, wave_inclusive_sum_or_most(p < g.num_experts ? mm_units(s.rows[s.order[p]]) : 0));
      if (p < g.num_experts) s.unit_end[p] = end;
      units = (uint32_t)__builtin_amdgcn_readlane((int)end, 63);
    }
    if (tid == 0) {   // no more than experts with rows of their own can have
      const uint32_t most = (uint32_t)(g.total_rows / 256) + (uint32_t)(g.num_experts < g.total_rows ? g.num_experts : g.total_rows);
      s.units = units < most ? units : most;
    }
  }
  __syncthreads();
}

// The copies' state: the tile and the step that they are at, as buffer descriptors and lane offsets.
template <int TYPE, int KIND>
struct MmCopies {
  static constexpr bool kSw = KIND == kSwiglu || KIND == kSwigluSave;
  static constexpr bool kTT = KIND == kWeightsGrad, kWT = KIND >= kRowsGrad;   // the operand's rows run along the sum
  static constexpr int kSize = TYPE == kMmInt8 ? 1 : 2;
  const MmTiles<TYPE, KIND>& tiles;
  uint32_t round, lds;
  int left, end_rows, along;   // steps; rows of a transposed operand in the last one; bytes of a step along rows
  int steps, wrap;             // of the tile; those in front of its first one, which come last
  uint64_t t_base, w_base;
  uint64_t w1_base;            // SwiGLU: the up rows
  int t_len, w_len, w1_len, t_pitch, w_pitch, t_col, w_col;
  uint32_t vt[2][2], vw[2][2];   // lane offsets of [half][copy]
  // kNowhere where a lane's columns lie beyond the sum (in its last step) or, by half, beyond a transposed operand's columns
  uint32_t tail[2], now[2], edge_t0, edge_t1, edge_w0, edge_w1;

  __device__ __forceinline__ MmCopies(const MmTiles<TYPE, KIND>& tiles_, uint32_t ring) : tiles(tiles_) {
    const ExpertMmArgs& g = tiles.g;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    lds = ring + wave * 2048;
    t_pitch = (KIND >= kRowsGrad ? g.n : g.k) * kSize;
    w_pitch = g.k * kSize;
    const int depth_bytes = (KIND == kRowsGrad ? g.n : g.k) * kSize;   // of rows along which the sum runs
#pragma unroll
    for (int c = 0; c < 2; c++) {
      // 128-byte rows, eight a copy: lane l fetches what belongs in slot l % 8 of row l / 8 (the slot of chunk x of row r is x ^ (r / 2 % 8):
      // sixteen rows' reads of one chunk fall on different banks)
      const int row = wave * 16 + c * 8 + (lane >> 3), chunk = (lane & 7) ^ ((row >> 1) & 7);
      // 256-byte rows, four a copy: pairs of 16-byte chunks change places by the row's bits 0, 1 and 3
      const int trow = wave * 8 + c * 4 + (lane >> 4), tchunk = (lane & 15) ^ (((trow & 3) | (trow >> 1 & 4)) << 1);
      tail[c] = (depth_bytes & 127) && chunk * 16 >= (depth_bytes & 127) ? kNowhere : 0;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        vt[h][c] = (kTT ? trow * t_pitch + h * 256 + tchunk * 16 : (h * 128 + row) * t_pitch + chunk * 16) + (c ? 0 : kBias);
        vw[h][c] = (kWT ? trow * w_pitch + h * 256 + tchunk * 16 : (h * 128 * !kSw + row) * w_pitch + chunk * 16) + (c ? 0 : kBias);
      }
    }
    round = 0;
    left = wrap = 0;
    along = 128;
    next_tile();
  }

  __device__ __forceinline__ void next_tile() {
    const ExpertMmArgs& g = tiles.g;
    MmTile t;
    do {   // (there are tiles without rows or steps)
      if (round == tiles.rounds) {
        left = 1 << 30;   // no more tiles: descriptors of nothing from here on
        t_len = w_len = w1_len = along = 0;
        return;
      }
      if (!tiles.tile(round++, t)) t.steps = 0;
    } while (t.steps == 0);
    left = steps = t.steps;
    const long w_expert = (long)t.expert * g.n * g.k * kSize;
    if constexpr (KIND == kWeightsGrad) {
      end_rows = uniform(tiles.s.rows[t.expert]) - (t.steps - 1) * 64;
      const long first = uniform(tiles.s.off[t.expert]);
      t_col = t.row0 * 2;
      w_col = t.col0 * 2;
      t_base = (uint64_t)g.t + first * t_pitch + t_col - kBias;
      w_base = (uint64_t)g.w + first * w_pitch + w_col - kBias;
    } else {
      t_base = (uint64_t)g.t + (long)t.row0 * t_pitch - kBias;
      t_len = uniform(t.rows * t_pitch + kBias);
      if constexpr (KIND == kRowsGrad) {
        end_rows = g.n - (t.steps - 1) * 64;
        w_col = t.col0 * 2;
        w_base = (uint64_t)g.w + w_expert + w_col - kBias;
      } else {
        const int left_rows = tiles.cols - t.col0, n = left_rows < t.width ? left_rows : t.width;
        w_base = (uint64_t)g.w + w_expert + (long)t.col0 * w_pitch - kBias;
        w_len = uniform(n * w_pitch + kBias);
        if constexpr (kSw) {
          w1_base = w_base + (long)tiles.cols * w_pitch;
          w1_len = w_len;
        }
      }
    }
    if constexpr (kTT || kWT) {
      const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
      const int trow = wave * 8 + (lane >> 4), tchunk = (lane & 15) ^ (((trow & 3) | (trow >> 1 & 4)) << 1);
      const int at = tchunk * 8;   // the lane's first column in a half
      if constexpr (kTT) {
        edge_t0 = t.row0 + at >= g.n ? kNowhere : 0;
        edge_t1 = t.row0 + at + 128 >= g.n ? kNowhere : 0;
      }
      edge_w0 = at >= t.width || t.col0 + at >= g.k ? kNowhere : 0;
      edge_w1 = at + 128 >= t.width || t.col0 + at + 128 >= g.k ? kNowhere : 0;
      lengths(64);
    }
    now[0] = now[1] = 0;
    if constexpr (KIND < kRowsGrad) {
      wrap = w_pitch % 4096 ? 0 : first_step(t);
      left -= wrap;
      forward(wrap);
    }
    if (left == 1) last();
  }

  // Workgroups that begin together stay together, and where rows are whole 4096 bytes long what they read of a step is behind a few of the
  // memory's channels.  There, tiles begin their sums at different steps (32 experts x 64 rows, 8192 x 2048: 191 us, all at the first 247; x 512
  // rows, 4096 x 2048: 238, 240; rows of 14336 bytes, with many rows an expert, lose 1 to 3% by it).  Not so the tiles that read the same rows, of eight columns of an expert;
  // and by nothing but expert and column: the other rows of a call do not change a row's sum.
  __device__ __forceinline__ int first_step(const MmTile& t) const {
    const uint32_t group = (uint32_t)t.expert * ((tiles.col_tiles + 7) / 8) + (uint32_t)t.col0 / (8 * MmTiles<TYPE, KIND>::kWide);
    return uniform((int)__umulhi(group * 2654435769u, (uint32_t)t.steps));   // (by the golden ratio: any number of them is spread evenly)
  }
  // Steps on along rows, or back.
  __device__ __forceinline__ void forward(int n) {
    t_base += n * 128;
    w_base += n * 128;
    t_len -= n * 128;
    w_len -= n * 128;
    if constexpr (kSw) {
      w1_base += n * 128;
      w1_len -= n * 128;
    }
  }

  // Descriptors' lengths of transposed operands, of which a step has `rows` rows.
  __device__ __forceinline__ void lengths(int rows) {
    if constexpr (kTT) t_len = uniform(rows * t_pitch - t_col + kBias);
    if constexpr (kWT) w_len = uniform(rows * w_pitch - w_col + kBias);
  }

  // In front of a tile's last step, in which the sum may end.
  __device__ __forceinline__ void last() {
    if constexpr (kTT || kWT) lengths(end_rows);
    now[0] = tail[0];
    now[1] = tail[1];
  }

  // The step after this one of the same tile.
  __device__ __forceinline__ void advance() {
    t_base += kTT ? 64 * (long)t_pitch : 128;
    w_base += kWT ? 64 * (long)w_pitch : 128;
    if constexpr (!kTT) t_len -= along;
    if constexpr (!kWT) w_len -= along;
    if constexpr (kSw) {
      w1_base += 128;
      w1_len -= along;
    }
  }
  // What there is to do when one step or none is left.
  __device__ __forceinline__ void passed() {
    if (KIND < kRowsGrad && left == 0 && wrap) {   // (rows of whole 4096 bytes: no step is short)
      left = wrap;
      wrap = 0;
      forward(-steps);
    } else if (left == 0) next_tile();
    else if (left == 1) last();
  }

  __device__ __forceinline__ static v4i descriptor(uint64_t base, int len) {
    return v4i{uniform((int)base), uniform((int)(base >> 32)), uniform(len), 0x00020000};
  }
  template <int H>
  __device__ __forceinline__ MmCopy t_part(uint32_t stage) const {
    return {(uint32_t)uniform(lds + stage + (H ? kT1 : kT0)), descriptor(t_base, t_len), vt[H][0] | (kTT ? (H ? edge_t1 : edge_t0) : now[0]),
            vt[H][1] | (kTT ? (H ? edge_t1 : edge_t0) : now[1])};
  }
  template <int H>
  __device__ __forceinline__ MmCopy w_part(uint32_t stage) const {
    return {(uint32_t)uniform(lds + stage + (H ? kW1 : kW0)), kSw && H ? descriptor(w1_base, w1_len) : descriptor(w_base, w_len),
            vw[H][0] | (kWT ? (H ? edge_w1 : edge_w0) : now[0]), vw[H][1] | (kWT ? (H ? edge_w1 : edge_w0) : now[1])};
  }
};

// Lane addresses of fragments in a part: sixteen rows (or columns) each, a lane has 16 bytes along the sum for each half of the step.
template <bool TRANSPOSED, int COUNT, int EVERY>
struct MmFragments {
  uint32_t at[TRANSPOSED ? COUNT : 1];
  // first: the wavefront's first sixteen; the next ones are EVERY sixteens on
  __device__ __forceinline__ MmFragments(uint32_t ring, int first) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    if constexpr (TRANSPOSED) {
      // rows of 256 bytes along the sum; four lanes read 16 columns of a row, sixteen lanes of four rows, and the hardware hands lane i column i
      const int f = (l16 >> 2) | (g & 1) << 2;
#pragma unroll
      for (int i = 0; i < COUNT; i++) at[i] = ring + (8 * g + (l16 >> 2)) * 256 + (((first + i * EVERY) ^ f) * 32) + (l16 & 3) * 8;
    } else {
      at[0] = ring + first * 2048 + l16 * 128 + ((g ^ (l16 >> 1)) * 16);
    }
  }
  // PART: which of a step's parts; the sixteens FROM .. TO
  template <int PART, int FROM = 0, int TO = COUNT>
  __device__ __forceinline__ void read(uint32_t stage, v4i (&f)[COUNT][2]) const {
#pragma unroll
    for (int i = FROM; i < TO; i++)
#pragma unroll
      for (int ks = 0; ks < 2; ks++) {
        if constexpr (TRANSPOSED) {
          typedef __attribute__((address_space(3))) char* Lds;
          typedef v4s __attribute__((address_space(3))) * Lds4;
          const Lds p = (Lds)(uintptr_t)(at[i] + stage) + PART + ks * 8192;
          const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)p)),
                    hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)(p + 1024)));
          f[i][ks] = v4i{lo[0], lo[1], hi[0], hi[1]};
        } else {
          typedef const __attribute__((address_space(3))) char* Lds;
          typedef const v4i __attribute__((address_space(3))) * Lds16;
          f[i][ks] = *(Lds16)((Lds)(uintptr_t)((ks ? at[0] ^ 64 : at[0]) + stage) + PART + i * EVERY * 2048);
        }
      }
  }
};

__device__ __forceinline__ v2i mm_half4(v4f v, bool fp16) {
  return fp16 ? __builtin_bit_cast(v2i, __builtin_convertvector(v, v4h)) : __builtin_bit_cast(v2i, __builtin_convertvector(v, v4bf));
}
// A lane of group gq = lane / 16 holds columns 4 gq .. + 4 of one row in each of two tiles of 16 columns.  Odd groups give their part of x for
// the even neighbour's of y: groups 0 and 2 end with columns 0 .. 8 and 8 .. 16 of the first tile, groups 1 and 3 with those of the second.
__device__ __forceinline__ v4i mm_pair(v2i x, v2i y) {
  const auto lo = __builtin_amdgcn_permlane16_swap(x[0], y[0], false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(x[1], y[1], false, false);
  return v4i{(int)lo[0], (int)hi[0], (int)lo[1], (int)hi[1]};
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t mm_buffer(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00020000);
}

// Stores of 16 bytes of a tile's outputs, always all of them: a lane whose row or columns lie beyond goes nowhere.
struct MmOut {
  __amdgpu_buffer_rsrc_t rsrc;
  int pitch;
  __device__ __forceinline__ MmOut(void* out, long row0, int rows, int col0, int cols) {
    pitch = cols * 2;
    rsrc = mm_buffer((char*)out + row0 * pitch + (long)col0 * 2, rows * pitch - col0 * 2);
  }
  // col: of the tile; room: columns that the output has from the tile's first on
  __device__ __forceinline__ void put(v4i v, int row, int col, int room) const {
    __builtin_amdgcn_raw_buffer_store_b128(v, rsrc, col < room ? row * pitch + col * 2 : (int)kNowhere, 0, 0);
  }
};

template <int TYPE, int KIND, bool STREAM>
__global__ void __launch_bounds__(kMmThreads, 2) expert_mm_kernel(const ExpertMmArgs g) {
  typedef typename MmAcc<TYPE>::T Acc;
  constexpr bool kSw = KIND == kSwiglu || KIND == kSwigluSave;
  constexpr int kStores = KIND == kSwiglu ? 8 : KIND == kSwigluSave ? 24 : 16;      // of a tile's epilogue, per wavefront
  constexpr int kTReads = KIND == kWeightsGrad ? 8 : 4;   // LDS instructions of half a T
  __shared__ MmShared s;
  mm_schedule<KIND>(s, g);
  const MmTiles<TYPE, KIND> tiles(s, g);
  if (tiles.rounds == 0) return;   // (the whole workgroup)
  const int wave = uniform(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
  const int lane = threadIdx.x & 63, l16 = lane & 15, gq = lane >> 4;
  const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)s.ring;
  MmCopies<TYPE, KIND> copies(tiles, ring);
  const MmFragments<KIND == kWeightsGrad, 4, 2> t_at(ring, wm);         // sixteens 0, 2, 4, 6 of a half's 128 rows, or 1, 3, 5, 7
  const MmFragments<(KIND >= kRowsGrad), 2, 1> w_at(ring, wn * 2);
  v4i tf[4][2], wf0[2][2], wf1[2][2];
  Acc acc[2][2][4][2];

  mm_copy<STREAM>(copies.template w_part<0>(0));
  mm_copy(copies.template t_part<0>(0));
  mm_copy<STREAM>(copies.template w_part<1>(0));
  mm_copy(copies.template t_part<1>(0));
  copies.advance();
  copies.left--;
  copies.passed();
  mm_copy<STREAM>(copies.template w_part<0>(kMmStage));
  mm_copy(copies.template t_part<0>(kMmStage));
  mm_copy<STREAM>(copies.template w_part<1>(kMmStage));
  mm_wait_copies<8>();
  mm_barrier();
  w_at.template read<kW0>(0, wf0);
  t_at.template read<kT0, 0, 2>(0, tf);
  if (wm) mm_barrier();   // this group runs a barrier behind from here on

  uint32_t stage = 0;
  int stored = 0;   // a tile's stores are younger than the copies that this step waits for
  for (uint32_t round = 0; round < tiles.rounds; round++) {
    MmTile t;
    if (!tiles.tile(round, t)) continue;
#pragma unroll
    for (int a = 0; a < 2; a++)
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < 2; j++) acc[a][b][i][j] = Acc{0, 0, 0, 0};
    auto arrived = [&] { mm_wait_copies<8, kStores>(stored); };
    // A phase's matrix half, of the tile's upper or lower half of rows; behind its first products the first half of the next fragments of T, into
    // the registers that these leave.  A group whose sixteens have no rows has nothing to multiply.
    const int rows0 = t.rows - wm * 16, rows1 = kSw || t.width > 128 ? rows0 : 0;   // for the first and second half of the columns
    auto multiply = [&](auto lower, int rows, Acc (&c)[4][2], const v4i (&w)[2][2], auto&& early0, auto&& early1) {
      constexpr int kFirst = decltype(lower)::value * 128;
      products<TYPE, kBegin, 0, kFirst>(c, w, tf, rows);
      early0();
      products<TYPE, kNext, 2, kFirst + 64>(c, w, tf, rows);
      early1();
      products<TYPE, kEnd, 2, kFirst + 64>(c, w, tf, rows);
    };
    constexpr std::integral_constant<int, 0> upper;
    constexpr std::integral_constant<int, 1> lower;
    const auto none = [] {};
    for (int left = t.steps; left > 0; left--) {
      t_at.template read<kT0, 2, 4>(stage, tf);
      mm_copy(copies.template t_part<1>(stage ^ kMmStage));
      copies.advance();
      arrived();
      mm_wait_fragments<kTReads>();   // (all but those just read)
      mm_barrier();
      multiply(upper, rows0, acc[0][0], wf0, [&] { w_at.template read<kW1, 0, 1>(stage, wf1); }, [&] { w_at.template read<kW1, 1, 2>(stage, wf1); });

      if (__builtin_expect(--copies.left <= 1, 0)) copies.passed();
      mm_copy<STREAM>(copies.template w_part<0>(stage));
      mm_barrier();
      multiply(upper, rows1, acc[0][1], wf1, [&] { t_at.template read<kT1, 0, 1>(stage, tf); }, [&] { t_at.template read<kT1, 1, 2>(stage, tf); });

      t_at.template read<kT1, 2, 4>(stage, tf);
      mm_copy(copies.template t_part<0>(stage));
      arrived();
      mm_barrier();
      multiply(lower, rows0, acc[1][0], wf0, none, none);

      w_at.template read<kW0>(stage ^ kMmStage, wf0);
      mm_copy<STREAM>(copies.template w_part<1>(stage));
      arrived();
      mm_barrier();
      stage ^= kMmStage;
      multiply(lower, rows1, acc[1][1], wf1, [&] { t_at.template read<kT0, 0, 1>(stage, tf); }, [&] { t_at.template read<kT0, 1, 2>(stage, tf); });
      stored = 0;
    }

    mm_results();
    // a lane holds, of rows a * 128 + (2 i + wm) * 16 + l16, columns b * 128 + wn * 32 + j * 16 + 4 gq .. + 4
    const int room = tiles.cols - t.col0 < t.width ? tiles.cols - t.col0 : t.width, col = wn * 32 + (gq & 1) * 16 + (gq >> 1) * 8;
    const long out_row0 = KIND == kWeightsGrad ? (long)t.expert * g.n + t.row0 : (long)t.row0;
    const MmOut out(g.out, out_row0, t.rows, t.col0, tiles.cols);
    const bool fp16 = TYPE == kMmFp16 || (TYPE == kMmInt8 && g.out_fp16);
    v4f sb[2][2];
    if constexpr (TYPE == kMmInt8) {
#pragma unroll
      for (int b = 0; b < 2; b++) {
        const int first = kSw ? b * tiles.cols + t.col0 : t.col0 + b * 128;
        const auto rsrc = mm_buffer(g.sb + (long)t.expert * g.n, g.n * 4);
#pragma unroll
        for (int j = 0; j < 2; j++)
          sb[b][j] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (first + wn * 32 + j * 16 + gq * 4) * 4, 0, 0));
      }
    }
    // (a row's scale is asked for a row ahead: the loads come behind all copies under way, together once instead of each)
    auto row_scale = [&](int row) {
      if constexpr (TYPE == kMmInt8)
        return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(mm_buffer(g.sa + t.row0, t.rows * 4), row * 4, 0, 0));
      else return 1.0f;
    };
    float next_sa = row_scale(wm * 16 + l16);
#pragma unroll
    for (int a = 0; a < 2; a++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        __builtin_amdgcn_sched_barrier(0);   // (a row's values at a time: all at once are more than the registers)
        const int row = a * 128 + (2 * i + wm) * 16 + l16;
        const float sa = next_sa;
        if (a * 4 + i < 7) next_sa = row_scale(((i + 1) / 4 + a) * 128 + (2 * ((i + 1) & 3) + wm) * 16 + l16);
        auto value = [&](int b, int j) {
          const Acc sum = acc[a][b][i][j];
          if constexpr (TYPE == kMmInt8) {
            v4f v;
#pragma unroll
            for (int x = 0; x < 4; x++) v[x] = (float)sum[x] * sa * sb[b][j][x];
            return v;
          } else return sum;
        };
        if constexpr (kSw) {
          v2i h[2];
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const v4f gate = value(0, j), up = value(1, j);
            v4f y;
#pragma unroll
            for (int x = 0; x < 4; x++) y[x] = swiglu_f32(gate[x], up[x]);
            h[j] = mm_half4(y, fp16);
          }
          out.put(mm_pair(h[0], h[1]), row, col, room);
          if constexpr (KIND == kSwigluSave) {
#pragma unroll
            for (int b = 0; b < 2; b++) {
              const MmOut both(g.gate_up, t.row0, t.rows, b * tiles.cols + t.col0, g.n);
              both.put(mm_pair(mm_half4(value(b, 0), fp16), mm_half4(value(b, 1), fp16)), row, col, room);
            }
          }
        } else {
#pragma unroll
          for (int b = 0; b < 2; b++) out.put(mm_pair(mm_half4(value(b, 0), fp16), mm_half4(value(b, 1), fp16)), row, b * 128 + col, room);
        }
      }
    __builtin_amdgcn_sched_barrier(0);
    stored = 1;
  }
  if (!wm) mm_barrier();
  mm_wait_copies<0>();   // (nothing may arrive in LDS that is another workgroup's by then)
}

}  // namespace esmoe

using namespace esmoe;

extern "C" int esmoe_launch_expert_mm(const ExpertMmArgs* args, int kind, int cus, hipStream_t stream) {
  const ExpertMmArgs& g = *args;
  if (expert_mm_takes_few(kind, g.num_experts, g.total_rows, g.n, g.k, cus)) return esmoe_launch_expert_mm_few(args, kind, cus, stream);
  const MmTileCount count = expert_mm_tiles(kind, g.num_experts, g.total_rows, g.n, g.k);
  const long tiles = count.units * count.col_tiles, grid = 4 * tiles < cus ? 4 * tiles : cus;   // (a tile may be four workgroups' work)
  if (grid == 0) return 0;
  // (rows' tiles that are few enough read their weights past the caches, us so and through them: 32 experts x 64 rows, 4096 x 7168: 301 / 325; x 256 rows
  // 440 / 436, 8192 rows by Zipf 533 / 518, one expert x 16384 rows, 4096 x 4096: 430 / 411; 4096 x 2048, 32 experts x 16 / 64 / 128 rows: forward 86 / 97,
  // 98 / 105, 108 / 116, rows' gradient 86 / 99, 89 / 102, 98 / 105)
  const long experts = g.num_experts < g.total_rows ? g.num_experts : g.total_rows;
  const bool once = kind <= 2 && expert_mm_whole_lines(g) && g.total_rows <= 128 * experts;
#define ESMOE_MM(T, K) hipLaunchKernelGGL((expert_mm_kernel<T, K, false>), dim3((unsigned)grid), dim3(kMmThreads), 0, stream, g)
#define ESMOE_MM_ONCE(T, K)                                                                                                         \
  {                                                                                                                                 \
    if (once) hipLaunchKernelGGL((expert_mm_kernel<T, K, true>), dim3((unsigned)grid), dim3(kMmThreads), 0, stream, g);               \
    else ESMOE_MM(T, K);                                                                                                            \
  }
#define ESMOE_MM16(T)                                  \
  switch (kind) {                                      \
    case 0: ESMOE_MM_ONCE(T, kForward) break;          \
    case 1:                                            \
      if (g.gate_up) ESMOE_MM_ONCE(T, kSwigluSave)     \
      else ESMOE_MM_ONCE(T, kSwiglu)                   \
      break;                                           \
    case 2: ESMOE_MM_ONCE(T, kRowsGrad) break;         \
    default: ESMOE_MM(T, kWeightsGrad);                \
  }
  if (g.type == kMmBf16) { ESMOE_MM16(kMmBf16) }
  else if (g.type == kMmFp16) { ESMOE_MM16(kMmFp16) }
  else if (kind == 0) ESMOE_MM_ONCE(kMmInt8, kForward)
  else ESMOE_MM_ONCE(kMmInt8, kSwiglu)
#undef ESMOE_MM16
#undef ESMOE_MM_ONCE
#undef ESMOE_MM
  return (int)hipGetLastError();
}
