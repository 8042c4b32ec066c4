// lsamp_skinny.h — the product of a few rows with a large matrix (decode
// batches, verify windows): out[m][n] = sum_k x[m][k] W[n][k] for m <= 64.
//
// Bound by reading W once (float32 past 16 rows by its matrix instruction).  Nothing
// is staged: a wave reads chunks of 16 bytes
// of 16 rows of W (and of x, which stays in L2) straight into the fragments of
// the matrix instruction, a 128-byte slab of the reduction at a time, the next
// slab's loads in flight while one is multiplied.  The WK waves of a work-group
// take slabs in turn and join their sums in LDS, so that even one token over a
// 2048 x 2048 matrix keeps 1,024 waves loading.  No alignment is needed: the
// loads take any element address, and the last slab is read by elements where
// it ends (unaligned rows of W halve its rate).  Measured, bf16: 1 x 2048 x 2048
// 5.0 us (a launch alone 3.9), over 151,936 columns 104-112 us for one row (5.6 to
// 6.0 TB/s), 118 for the loss of 20 rows, 140 for the logits of 64.  Float32 over
// 151,936 columns: one row 236 us (5.3 TB/s), 20 rows 277, 64 rows 405 (98 TFLOP/s).
#ifndef LSAMP_SKINNY_H
#define LSAMP_SKINNY_H

#include "lsamp_gemm.h"

namespace lsamp {
namespace gemm {

// NF x 16 columns and MF x 16 rows a work-group of WK waves.
//
// One wave's 16 rows of x come straight from L2.  With more (MF > 1) those reads
// would cross the vector memory path as often as W's, in half lines: a wave then
// brings its slab of x to its own LDS, in whole lines (the loss of 64 rows x 2048 x
// 151936: 147 -> 125 us); x's rows are 16-byte chunks there (MatrixRef).
//
// Epilogues without a step over the work-group (ROWWISE) get four columns at a
// time with 16 lanes along a row, so that a row's 64 columns are stored as one
// line; others get WK x 16 columns of all rows, WK waves along n.
template <int DT, int MF, int NF, int WK, bool ROWWISE, class Epi>
__global__ __launch_bounds__(WK* kWave, 2) void k_skinny(GemmPlan g, Epi epi) {
  constexpr int kEb = El<DT>::kBytes, kSlab = kSlabOf<DT>, kChunk = kChunkOf<DT>;
  constexpr int kFrags = NF * MF;
  constexpr bool kStaged = MF > 1;
  using X = Side<DT, false, MF * 16, 1>;
  constexpr int kStageBytes = kStaged ? WK * 2 * X::kBytes : 0;
  constexpr int kSumBytes = WK * kFrags * kWave * 16;
  // (an epilogue's pair of floats a row and wave, or its 16 rows of 16 columns a wave)
  constexpr int kRedBytes = ROWWISE ? 0 : WK * (MF * 128 > 1024 ? MF * 128 : 1024);
  constexpr int kLds = kStageBytes > kSumBytes + kRedBytes ? kStageBytes : kSumBytes + kRedBytes;
  __shared__ __attribute__((aligned(1024))) char lds[kLds];
  static_assert(ROWWISE || NF == WK, "a wave for every 16 columns");

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n0 = (int)blockIdx.x * (NF * 16);
  const int row = lane & 15, at = (lane >> 4) * kChunk;
  const int k_all = g.b.cols, whole = k_all / kSlab;

  const char* w[NF];
#pragma unroll
  for (int i = 0; i < NF; ++i)
    w[i] = (const char*)g.b.p + (int64_t)min(n0 + i * 16 + row, g.b.rows - 1) * g.b.ld * kEb;
  const char* x0 = (const char*)g.a.p + (int64_t)min(row, g.a.rows - 1) * g.a.ld * kEb;
  X x;
  if constexpr (kStaged) x.init(g.a, 0, 0, 0, lane);
  const char* const x_base = x.base;
  char* const mine = lds + wave * 2 * X::kBytes;

  v4f acc[NF][MF];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < MF; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

  struct Step {
    v4i w[NF][2], x[2];
  };
  constexpr int kLoads = 2 * NF + (kStaged ? X::kUnits : 2);
  // (x first: waiting for W's chunks then waits for x's too)
  const auto load = [&](Step& s, int slab, int buffer) {
    if constexpr (kStaged) {
      x.base = x_base + (int64_t)slab * kSlabBytes;
      x.template load_counted<false>(mine + buffer * X::kBytes, 0, 0, lane);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int64_t k = ((int64_t)slab * kSlab + kk * (kSlab / 2) + at) * kEb;
      if constexpr (!kStaged) s.x[kk] = load_chunk<DT>(x0 + k);
#pragma unroll
      for (int i = 0; i < NF; ++i) s.w[i][kk] = load_chunk<DT>(w[i] + k);
    }
  };
  const auto multiply = [&](const Step& s, int buffer) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      v4i f[MF];
#pragma unroll
      for (int j = 0; j < MF; ++j)
        f[j] = kStaged ? X::frag(mine + buffer * X::kBytes, j * 16, kk, lane) : s.x[kk];
#pragma unroll
      for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < MF; ++j) mma<DT>(acc[i][j], s.w[i][kk], f[j]);
    }
  };

  // This wave's whole slabs: wave, wave + WK, ...; each work-group starts at
  // another one, since rows a power of two apart lie in the same few L2 channels.
  const int steps = whole > wave ? (whole - wave + WK - 1) / WK : 0;
  int at_step = steps ? (int)(blockIdx.x % (unsigned)steps) : 0;
  const auto next = [&] {
    const int slab = wave + WK * at_step;
    at_step = at_step + 1 == steps ? 0 : at_step + 1;
    return slab;
  };
  // A step: the next one's loads, then its own products once only those are under
  // way.  The LDS reads of the step before are done by then (wait_loads), so its
  // buffer may be filled.  MORE is known when it is compiled: where the loads are
  // in doubt the compiler waits for all of them.
  const auto step = [&](Step& now, Step& then, int buffer, auto more) {
    constexpr bool MORE = decltype(more)::value;
    if constexpr (kStaged) {
      __builtin_amdgcn_sched_barrier(0);
      wait_loads<kLoads>();
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (MORE) load(then, next(), buffer ^ 1);
    if constexpr (kStaged) {
      __builtin_amdgcn_sched_barrier(0);
      wait_loads<MORE ? kLoads : 0>();
      __builtin_amdgcn_sched_barrier(0);
    }
    multiply(now, buffer);
  };
  Step s0, s1;
  if (steps > 0) {
    load(s0, next(), 0);
    int u = 0;
    for (; u + 2 < steps; u += 2) {
      step(s0, s1, 0, std::true_type{});
      step(s1, s0, 1, std::true_type{});
    }
    if (u + 1 < steps) {
      step(s0, s1, 0, std::true_type{});
      step(s1, s0, 1, std::false_type{});
    } else {
      step(s0, s1, 0, std::false_type{});
    }
  }
  if (whole * kSlab < k_all && wave == whole % WK) {  // the last slab, where it ends
    if constexpr (kStaged) {
      __builtin_amdgcn_sched_barrier(0);
      wait_loads<0>();
      __builtin_amdgcn_sched_barrier(0);
      x.base = x_base + (int64_t)whole * kSlabBytes;
      x.template load_counted<true>(mine, g.a.cols - whole * kSlab, 0, lane);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int k = whole * kSlab + kk * (kSlab / 2) + at;
      if constexpr (!kStaged) s0.x[kk] = load_chunk_end<DT>(x0, k, k_all);
#pragma unroll
      for (int i = 0; i < NF; ++i) s0.w[i][kk] = load_chunk_end<DT>(w[i], k, k_all);
    }
    if constexpr (kStaged) {
      __builtin_amdgcn_sched_barrier(0);
      wait_loads<0>();
      __builtin_amdgcn_sched_barrier(0);
    }
    multiply(s0, 0);
  }

  if constexpr (kStaged) __syncthreads();  // (the sums take the slabs' place)
  v4f* sums = (v4f*)lds;                   // [wave][fragment][lane]
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < MF; ++j) sums[(wave * kFrags + i * MF + j) * kWave + lane] = acc[i][j];
  __syncthreads();
  const auto total = [&](int frag, int l) {
    v4f v = sums[frag * kWave + l];
#pragma unroll
    for (int k = 1; k < WK; ++k) v += sums[(k * kFrags + frag) * kWave + l];
    return v;
  };
  if constexpr (ROWWISE) {
    for (int q = threadIdx.x; q < MF * 16 * NF * 4; q += WK * kWave) {
      const int r = q / (NF * 4), c = q % (NF * 4) * 4;
      if (r < epi.m && n0 + c < epi.n)
        epi.put(r, n0 + c, total(c / 16 * MF + r / 16, (r & 15) + (c % 16) * 4), 0);
    }
  } else {
    v4f part[1][MF];
#pragma unroll
    for (int j = 0; j < MF; ++j) part[0][j] = total(wave * MF + j, lane);
    epi.template run<MF, 1, MF * 16, NF * 16, 1, NF>(part, 0, n0, TileAt{0, (int)blockIdx.x, 0}, 0,
                                                     wave, lane, lds + kSumBytes);
  }
}

}  // namespace gemm
}  // namespace lsamp

#endif
