// lsamp_gemm.h — the tiled matrix product of the hidden-state operators.
//
//   C[m][n] = sum_k A(m, k) B(n, k)
//
// Each operand is a matrix in HBM that the product reads in one of two roles:
// rows along its output index with the reduction along the row ("row-major":
// x and W of the forward product), or rows along the reduction ("k-major": W in
// dX = G W, both operands in dW = G^T X).  No operand is transposed in memory.
//
// A work-group computes a BM x BN tile.  It steps over the reduction in slabs of
// 128 bytes (64 16-bit or 32 float elements): slab t + 1 goes from HBM to LDS
// (16 bytes a lane, straight to LDS, no registers) while slab t is multiplied.
// Row-major slabs lie in LDS as [tile row][8 chunks of 16 bytes], k-major ones
// as [block of 128 bytes of output columns][slab row][8 chunks]; chunk c of row
// r is kept at a permuted place, so that the reads of a matrix instruction's 16
// rows fall on different LDS banks.  A 16-bit k-major fragment is read with the
// transposing LDS read (4 reduction steps of one column a lane), a row-major one
// with 16-byte reads; both give a lane 8 consecutive reduction steps, so the two
// roles mix freely.
//
// The matrix instructions get W's side as the first operand: a lane's 4 results
// are then 4 consecutive output columns of one row, which epilogues read and
// store as vectors.  All sums are float32.
#ifndef LSAMP_GEMM_H
#define LSAMP_GEMM_H

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "lsamp_head.h"

namespace lsamp {
namespace gemm {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

#define LSAMP_GLOBAL(p) ((const __attribute__((address_space(1))) void*)(p))
#define LSAMP_LDS(p) ((__attribute__((address_space(3))) void*)(p))

// What loads past the end of the reduction read.
__device__ __attribute__((aligned(16))) const uint32_t kZeros[4] = {0, 0, 0, 0};

constexpr int kSlabBytes = 128;
constexpr int kWave = 64;

template <int DT>
struct El;
template <>
struct El<LSAMP_DTYPE_F32> {
  using S = float;
  static constexpr int kBytes = 4;
};
template <>
struct El<LSAMP_DTYPE_BF16> {
  using S = __bf16;
  static constexpr int kBytes = 2;
};
template <>
struct El<LSAMP_DTYPE_F16> {
  using S = _Float16;
  static constexpr int kBytes = 2;
};
template <int DT>
constexpr int kChunkOf = 16 / El<DT>::kBytes;  // elements of a 16-byte chunk
template <int DT>
constexpr int kSlabOf = kSlabBytes / El<DT>::kBytes;  // reduction steps of a slab

// acc += 16 x 16 outer products over the reduction steps of one chunk per lane
// (32 steps of 16-bit elements, 16 of float32).  Lane l holds row l & 15 and the
// chunk of steps l >> 4.  The float32 instruction takes one step of a lane at a
// time: step j of every lane's chunk, which is a different set of reduction steps
// on both sides alike.
template <int DT>
__device__ __forceinline__ void mma(v4f& acc, const v4i& b, const v4i& a) {
  if constexpr (DT == LSAMP_DTYPE_BF16) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, b),
                                                  __builtin_bit_cast(v8bf, a), acc, 0, 0, 0);
  } else if constexpr (DT == LSAMP_DTYPE_F16) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, b),
                                                 __builtin_bit_cast(v8h, a), acc, 0, 0, 0);
  } else {
    const v4f bf = __builtin_bit_cast(v4f, b), af = __builtin_bit_cast(v4f, a);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(bf[j], af[j], acc, 0, 0, 0);
  }
}

// Where chunk `c` of slab row `r` of a k-major slab is kept.  16-bit: a fragment
// is a 32-byte pair of chunks of the rows 8 g + j (g, j = 0..3), and the pair
// moves with bits of j and g; float32: a 64-byte half of the rows 4 g + j.
template <int DT>
__device__ __forceinline__ int kmajor_place(int r, int c) {
  if constexpr (El<DT>::kBytes == 2)
    return c ^ ((((r >> 1) & 1) | (((r >> 3) & 1) << 1)) << 1);
  else
    return c ^ (((r >> 2) & 1) << 2);
}

// One operand's side of a work-group's tile: ROWS output rows (or columns), read
// by WAVES waves, each wave 1 KB units of 8 LDS rows.
template <int DT, bool KMAJ, int ROWS, int WAVES>
struct Side {
  static constexpr int kEb = El<DT>::kBytes;
  static constexpr int kSlab = kSlabOf<DT>;
  static constexpr int kChunk = kChunkOf<DT>;
  static constexpr int kUnits = ROWS / 8 / WAVES;
  static constexpr int kBytes = ROWS * kSlabBytes;
  static_assert(ROWS % (8 * WAVES) == 0, "whole units a wave");

  const char* p[kUnits];
  int64_t step;
  int koff;  // row-major: the lane's chunk's first step of the slab

  // slab row of this lane in unit i (k-major)
  static __device__ __forceinline__ int slab_row(int wave, int lane, int i) {
    return ((wave * kUnits + i) % (kSlab / 8)) * 8 + (lane >> 3);
  }

  __device__ __forceinline__ void init(const MatrixRef& o, int first, int slab0, int wave, int lane) {
    if constexpr (!KMAJ) {
      koff = ((lane & 7) ^ (lane >> 3)) * kChunk;
      step = kSlabBytes;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        int r = first + (wave * kUnits + i) * 8 + (lane >> 3);
        r = r < o.rows ? r : o.rows - 1;  // (rows past the end repeat the last: never stored)
        p[i] = (const char*)o.p + (int64_t)r * o.ld * kEb +
               ((int64_t)slab0 * kSlab + koff) * kEb;
      }
    } else {
      koff = 0;
      step = (int64_t)kSlab * o.ld * kEb;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int u = wave * kUnits + i;
        const int r = slab_row(wave, lane, i);
        int c = first + (u / (kSlab / 8)) * kSlab + kmajor_place<DT>(r, lane & 7) * kChunk;
        c = c < o.cols ? c : o.cols - kChunk;
        p[i] = (const char*)o.p + ((int64_t)(slab0 * (int64_t)kSlab + r) * o.ld + c) * kEb;
      }
    }
  }

  // One slab to LDS.  `left`: reduction steps from this slab on; the chunks (rows)
  // past them come from a zeroed buffer.
  __device__ __forceinline__ void load(char* lds, int left, const char* zero, int wave, int lane) {
    if (left >= kSlab) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i)
        __builtin_amdgcn_global_load_lds(LSAMP_GLOBAL(p[i]),
                                         LSAMP_LDS(lds + (wave * kUnits + i) * 1024), 16, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int k = KMAJ ? slab_row(wave, lane, i) : koff;
        __builtin_amdgcn_global_load_lds(LSAMP_GLOBAL(k < left ? p[i] : zero),
                                         LSAMP_LDS(lds + (wave * kUnits + i) * 1024), 16, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) p[i] += step;
  }

  // The fragment of 16 output rows from `row0` (a multiple of 16), half `kk` of the slab.
  static __device__ __forceinline__ v4i frag(const char* lds, int row0, int kk, int lane) {
    if constexpr (!KMAJ) {
      const int r = row0 + (lane & 15);
      const int c = (kk * 4 + (lane >> 4)) ^ (lane & 7);
      return *reinterpret_cast<const v4i*>(lds + r * kSlabBytes + c * 16);
    } else if constexpr (kEb == 2) {
      const char* blk = lds + (row0 / kSlab) * (kSlab * kSlabBytes);
      const int c = ((row0 % kSlab) / 16) * 2 + ((lane & 3) >> 1);
      v4s h[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = kk * 32 + (lane >> 4) * 8 + i * 4 + ((lane & 15) >> 2);
        const char* a = blk + r * kSlabBytes + kmajor_place<DT>(r, c) * 16 + (lane & 1) * 8;
        h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) v4s*)LSAMP_LDS(a));
      }
      v4i out;
      __builtin_memcpy(&out, h, 16);
      return out;
    } else {
      const char* blk = lds + (row0 / kSlab) * (kSlab * kSlabBytes);
      const int col = row0 % kSlab + (lane & 15);
      v4f out;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = kk * 16 + (lane >> 4) * 4 + j;
        out[j] = *reinterpret_cast<const float*>(blk + r * kSlabBytes +
                                                 kmajor_place<DT>(r, col / 4) * 16 + (col % 4) * 4);
      }
      return __builtin_bit_cast(v4i, out);
    }
  }
};

// Work-group -> (tile row, tile column, part of the reduction).  Consecutive
// work-groups go to the 8 XCDs in turn, so each XCD is given a contiguous range
// of the order; in the order, 8 tile rows by tile columns run together, so that
// the tiles in flight on one XCD share their operands' slabs in its L2.
struct TileAt {
  int m, n, part;
};
__device__ __forceinline__ TileAt tile_at(int bid, int tm, int tn, int parts) {
  const int total = tm * tn * parts;
  const int xcd = bid & 7, q = total >> 3, rem = total & 7;
  int i = xcd * q + (xcd < rem ? xcd : rem) + (bid >> 3);
  TileAt t;
  t.part = i / (tm * tn);
  i -= t.part * (tm * tn);
  const int group = i / (8 * tn), in = i - group * 8 * tn;
  const int height = tm - group * 8 < 8 ? tm - group * 8 : 8;
  t.m = group * 8 + in % height;
  t.n = in / height;
  return t;
}

// One tile.  Epi: what happens to the sums; called once per work-group with
//   run(acc, m0, n0, part, lane, wave-in-M, wave-in-N, lds)
// where acc[fn][fm][i] is row m0 + fm * 16 + (lane & 15), column
// n0 + fn * 16 + (lane >> 4) * 4 + i.
template <int DT, bool AK, bool BK, int BM, int BN, int WM, int WN, class Epi>
__global__ __launch_bounds__(WM* WN* kWave) void k_gemm(GemmPlan g, Epi epi) {
  constexpr int kWaves = WM * WN;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  using A = Side<DT, AK, BM, kWaves>;
  using B = Side<DT, BK, BN, kWaves>;
  constexpr int kStage = A::kBytes + B::kBytes;
  __shared__ __attribute__((aligned(1024))) char lds[2 * kStage];

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const TileAt at = tile_at((int)blockIdx.x, g.tiles_m, g.tiles_n, g.parts);
  const int m0 = at.m * BM, n0 = at.n * BN;
  const int slab0 = at.part * g.slabs_per_part;
  const int slabs = min(g.slabs_per_part, g.slabs - slab0);
  const int wm = wave % WM, wn = wave / WM;
  const char* zero = (const char*)kZeros;

  A a;
  B b;
  a.init(g.a, m0, slab0, wave, lane);
  b.init(g.b, n0, slab0, wave, lane);
  int left_a = (AK ? g.a.rows : g.a.cols) - slab0 * kSlabOf<DT>;
  int left_b = (BK ? g.b.rows : g.b.cols) - slab0 * kSlabOf<DT>;

  v4f acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

  a.load(lds, left_a, zero, wave, lane);
  b.load(lds + A::kBytes, left_b, zero, wave, lane);
  __syncthreads();
  for (int t = 0; t < slabs; ++t) {
    const char* cur = lds + (t & 1) * kStage;
    if (t + 1 < slabs) {
      char* next = lds + ((t + 1) & 1) * kStage;
      left_a -= kSlabOf<DT>;
      left_b -= kSlabOf<DT>;
      a.load(next, left_a, zero, wave, lane);
      b.load(next + A::kBytes, left_b, zero, wave, lane);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      v4i fa[FM], fb[FN];
#pragma unroll
      for (int i = 0; i < FN; ++i)
        fb[i] = B::frag(cur + A::kBytes, wn * (FN * 16) + i * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[i] = A::frag(cur, wm * (FM * 16) + i * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) mma<DT>(acc[i][j], fb[i], fa[j]);
    }
    __syncthreads();
  }
  epi.template run<FM, FN, BM, BN, WM, WN>(acc, m0, n0, at, wm, wn, lane, lds);
}

}  // namespace gemm
}  // namespace lsamp

#endif
