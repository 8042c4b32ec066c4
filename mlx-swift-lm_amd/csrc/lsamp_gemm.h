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

#include <type_traits>

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

// Waits until at most `N` of this wave's vector memory operations (in the order
// of their issue) and none of its LDS operations are under way.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "six bits");
  // vmcnt in bits 3:0 and 15:14, expcnt 6:4 (unused: 7), lgkmcnt 11:8
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x70);
}

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
// Whole numbers of 8 bits: an operand type of row-major products only, summed in 32 bits.
constexpr int kInt8 = 3;
template <>
struct El<kInt8> {
  using S = int8_t;
  static constexpr int kBytes = 1;
};
template <int DT>
using Sum = std::conditional_t<DT == kInt8, v4i, v4f>;  // four sums of a lane
template <int DT>
constexpr int kChunkOf = 16 / El<DT>::kBytes;  // elements of a 16-byte chunk
template <int DT>
constexpr int kSlabOf = kSlabBytes / El<DT>::kBytes;  // reduction steps of a slab

// Waits until none of this wave's LDS operations are under way.
__device__ __forceinline__ void wait_lds() {
  __builtin_amdgcn_s_waitcnt(0xc07f);  // (lgkmcnt 0; the others at their most)
}

// Every wave's barrier, with no memory access moved across it by the compiler
// (and no wait: what has to be done by then is waited for by wait_loads).
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// acc += 16 x 16 products over the reduction steps of one chunk per lane
// (64 steps of 8-bit elements, 32 of 16-bit ones, 16 of float32).  Lane l holds row l & 15 and the
// chunk of steps l >> 4.  The float32 instruction takes one step of a lane at a
// time: step j of every lane's chunk, which is a different set of reduction steps
// on both sides alike.
template <int DT>
__device__ __forceinline__ void mma(Sum<DT>& acc, const v4i& b, const v4i& a) {
  if constexpr (DT == kInt8) {
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, a, acc, 0, 0, 0);
  } else if constexpr (DT == LSAMP_DTYPE_BF16) {
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

// Float32 products on the bfloat16 matrix instructions.  A value is split into
// three bfloat16 parts, a = h + m + l, h its first 8 bits (cut off, so that it is
// finite), m and l the rest rounded; a b = hh + hm + mh + mm + hl + lh, and what
// is left out is below 2^-22 |a b|, 2^-26 in the mean, so the sums are those of
// float32.  Six instructions of 16 cycles take 32 steps of a 16 x 16 tile, the
// float32 instruction takes 256 cycles.  The parts end at bfloat16's last step,
// 2^-133: a value is kept to 24 bits or to 2^-134, whichever is larger, so below
// 2^-110 it has fewer bits than float32.
//
// An infinity or a NaN has no remainder: it turns its row or column of the tile
// into NaN.  A tile that ends with one is computed again with such values left
// out of the products of remainders (`hx`).  The products of finite values are
// the same ones in the same order, so no other row of the result changes.
struct Split {
  v8bf h, m, l;
};
struct SplitAny {
  v8bf h, hx, m, l;
};
__device__ __forceinline__ Split split8(const v4i& a, const v4i& b) {
  Split s;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int bits = i < 4 ? a[i] : b[i - 4];
    const float h = __builtin_bit_cast(float, bits & (int)0xffff0000);
    const float r = __builtin_bit_cast(float, bits) - h;
    const __bf16 m = (__bf16)r;
    s.h[i] = __builtin_bit_cast(__bf16, (short)(bits >> 16));
    s.m[i] = m;
    s.l[i] = (__bf16)(r - (float)m);
  }
  return s;
}
__device__ __forceinline__ SplitAny split8_any(const v4i& a, const v4i& b) {
  SplitAny s;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int bits = i < 4 ? a[i] : b[i - 4];
    const float v = __builtin_bit_cast(float, bits);
    const bool finite = (bits & 0x7f800000) != 0x7f800000;
    const float h = __builtin_bit_cast(float, bits & (int)0xffff0000);
    const float r = finite ? v - h : 0.f;
    const __bf16 m = (__bf16)r;
    s.h[i] = (__bf16)(finite ? h : v);
    s.hx[i] = (__bf16)(finite ? h : 0.f);
    s.m[i] = m;
    s.l[i] = (__bf16)(r - (float)m);
  }
  return s;
}
__device__ __forceinline__ void mma_split(v4f& acc, const v8bf& bh, const v8bf& bx, const v8bf& bm,
                                          const v8bf& bl, const v8bf& ah, const v8bf& ax,
                                          const v8bf& am, const v8bf& al) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bl, ax, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bx, al, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bm, am, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bm, ax, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bx, am, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bh, ah, acc, 0, 0, 0);
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

// 16 bytes a lane from memory to LDS, lane after lane from LDS address `lds` (the
// same for the wave).  Written out because the compiler makes every later LDS
// read wait for such loads, also a read of the other buffer; here the wave waits
// where it must (wait_loads) and nowhere else.  No vector register is written.  M0
// is named as overwritten: the compiler allocates it to nothing and sets it ahead
// of what reads it, but it joins settings of equal values, which an unnamed one
// between them would break.  (It warns that it does not preserve the register for
// us: nothing here expects that.)
__device__ __forceinline__ uint32_t lds_address(char* lds) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(uint32_t lds, const char* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds(uint32_t lds, const char* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds), "v"(p)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// Two bases that load_to_lds may read at once.  A vector instruction that writes a scalar
// register has to be five wait states ahead of a memory instruction that reads it; the
// compiler sees to that for its own loads, but does not look into the text above.  Nothing
// but scalar arithmetic is meant to make these; should the compiler take some of it through
// vector registers, it reads them back ahead of the wait.
__device__ __forceinline__ void settled(const char*& a, const char*& b) {
  asm volatile("s_nop 4" : "+s"(a), "+s"(b));
}

// 16 bytes from an address aligned to elements only.
template <int DT>
__device__ __forceinline__ v4i load_chunk(const char* p) {
  struct __attribute__((packed, aligned(El<DT>::kBytes))) Any {
    v4i v;
  };
  return ((const Any*)p)->v;
}
// The chunk at element k of a row of `cols` elements, zero past its end.
__device__ __forceinline__ v4i moved_down(v4i v, int bytes) {  // 0 .. 15
  unsigned __int128 w;
  __builtin_memcpy(&w, &v, 16);
  w >>= 8 * bytes;
  __builtin_memcpy(&v, &w, 16);
  return v;
}
template <int DT>
__device__ __forceinline__ v4i load_chunk_end(const char* row, int k, int cols) {
  using S = typename El<DT>::S;
  constexpr int N = kChunkOf<DT>;
  if constexpr (DT == kInt8) {
    // (bytes: the row's last 16, moved down, in place of sixteen loads in turn)
    if (cols >= N) {
      const int over = k + N - cols;
      const v4i v = load_chunk<DT>(row + min(k, cols - N));
      return over >= N ? v4i{0, 0, 0, 0} : over > 0 ? moved_down(v, over) : v;
    }
  }
  if (k + N <= cols) return load_chunk<DT>(row + (int64_t)k * El<DT>::kBytes);
  S e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = k + i < cols ? ((const S*)row)[k + i] : (S)0.f;
  v4i v;
  __builtin_memcpy(&v, e, 16);
  return v;
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
  static_assert(!KMAJ || ROWS % kSlab == 0, "whole blocks of 128 bytes of columns");

  const char* base;         // the slab's first element (the same for every lane)
  int64_t step;             // bytes from slab to slab
  uint32_t off[kUnits];     // the lane's chunk of each unit, from base
  int koff;                 // row-major: the lane's chunk's first step of the slab

  // slab row of this lane in unit i (k-major)
  static __device__ __forceinline__ int slab_row(int wave, int lane, int i) {
    return ((wave * kUnits + i) % (kSlab / 8)) * 8 + (lane >> 3);
  }

  // `first`: the tile's first output row (column); it exists.
  __device__ __forceinline__ void init(const MatrixRef& o, int first, int slab0, int wave, int lane) {
    if constexpr (!KMAJ) {
      koff = ((lane & 7) ^ (lane >> 3)) * kChunk;
      step = kSlabBytes;
      base = (const char*)o.p + ((int64_t)first * o.ld + (int64_t)slab0 * kSlab) * kEb;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        // (rows past the end repeat the last: what they give is never stored)
        const int r = min((wave * kUnits + i) * 8 + (lane >> 3), o.rows - 1 - first);
        off[i] = ((uint32_t)r * (uint32_t)o.ld + (uint32_t)koff) * kEb;
      }
    } else {
      koff = 0;
      step = (int64_t)kSlab * o.ld * kEb;
      base = (const char*)o.p + ((int64_t)slab0 * kSlab * o.ld + first) * kEb;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int u = wave * kUnits + i;
        const int r = slab_row(wave, lane, i);
        const int c = min((u / (kSlab / 8)) * kSlab + kmajor_place<DT>(r, lane & 7) * kChunk,
                          o.cols - kChunk - first);
        off[i] = ((uint32_t)r * (uint32_t)o.ld + (uint32_t)c) * kEb;
      }
    }
  }

  // One slab to LDS.  TAIL: only `left` reduction steps remain; the chunks (rows)
  // past them come from a zeroed buffer.
  template <bool TAIL>
  __device__ __forceinline__ void load(uint32_t lds, int left, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const uint32_t dst = lds + (wave * kUnits + i) * 1024;
      if constexpr (TAIL) {
        const int k = KMAJ ? slab_row(wave, lane, i) : koff;
        load_to_lds(dst, k < left ? base + off[i] : (const char*)kZeros);
      } else {
        load_to_lds(dst, base, off[i]);
      }
    }
    base += step;
  }
  __device__ __forceinline__ void load_unit(int i, uint32_t lds, int wave) {
    load_to_lds(lds + (wave * kUnits + i) * 1024, base, off[i]);
  }
  // The same, known to the compiler: among loads whose results it waits for.
  template <bool TAIL>
  __device__ __forceinline__ void load_counted(char* lds, int left, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const char* p = base + off[i];
      if constexpr (TAIL) {
        const int k = KMAJ ? slab_row(wave, lane, i) : koff;
        p = k < left ? p : (const char*)kZeros;
      }
      __builtin_amdgcn_global_load_lds(LSAMP_GLOBAL(p),
                                       LSAMP_LDS(lds + (wave * kUnits + i) * 1024), 16, 0, 0);
    }
    base += step;
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

// The same for a matrix whose rows lie anywhere and end anywhere (`cols` exact):
// chunks go through registers, taken by elements where a row or the reduction
// ends, and are written to the same places of LDS.
template <int DT, bool KMAJ, int ROWS, int WAVES>
struct LooseSide : Side<DT, KMAJ, ROWS, WAVES> {
  using Base = Side<DT, KMAJ, ROWS, WAVES>;
  static constexpr int kEb = Base::kEb, kSlab = Base::kSlab, kChunk = Base::kChunk;
  static constexpr int kUnits = Base::kUnits;
  const char* row[kUnits];  // row-major: the row; k-major: the slab's first row
  int col[kUnits];          // k-major: the chunk's first column
  int64_t ld;
  int cols;
  v4i held[kUnits];

  __device__ __forceinline__ void init(const MatrixRef& o, int first, int slab0, int wave, int lane) {
    ld = o.ld * kEb;
    cols = o.cols;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int u = wave * kUnits + i;
      if constexpr (!KMAJ) {
        const int r = min(first + u * 8 + (lane >> 3), o.rows - 1);
        row[i] = (const char*)o.p + (int64_t)r * ld;
      } else {
        row[i] = (const char*)o.p;
        col[i] = first + (u / (kSlab / 8)) * kSlab +
                 kmajor_place<DT>(Base::slab_row(wave, lane, i), lane & 7) * kChunk;
      }
    }
  }
  // Slab `slab` to registers; `rows`: k-major rows in all.
  __device__ __forceinline__ void hold(int slab, int rows, int wave, int lane) {
    hold(held, slab, rows, wave, lane);
  }
  __device__ __forceinline__ void hold(v4i (&held)[kUnits], int slab, int rows, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      if constexpr (!KMAJ) {
        const int k = slab * kSlab + ((lane & 7) ^ (lane >> 3)) * kChunk;
        held[i] = load_chunk_end<DT>(row[i], k, cols);
      } else {
        const int r = slab * kSlab + Base::slab_row(wave, lane, i);
        held[i] = r < rows ? load_chunk_end<DT>(row[i] + (int64_t)r * ld, col[i], cols)
                           : v4i{0, 0, 0, 0};
      }
    }
  }
  __device__ __forceinline__ void place(char* lds, int wave, int lane) { place(held, lds, wave, lane); }
  __device__ __forceinline__ void place(const v4i (&held)[kUnits], char* lds, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
      *(v4i*)(lds + (wave * kUnits + i) * 1024 + lane * 16) = held[i];
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

// The same for a batch of equal products: `part` is the product.  Of a symmetric one
// (C = C^T) only the tiles at or right of the diagonal are computed, column after
// column.
__device__ __forceinline__ TileAt tile_at(int bid, const BatchPlan& g) {
  const int each = g.symmetric ? g.tiles_n * (g.tiles_n + 1) / 2 : g.tiles_m * g.tiles_n;
  TileAt t;
  if (!g.symmetric) {
    t = tile_at(bid, g.tiles_m, g.tiles_n, g.parts);
  } else {
    const int total = each * g.parts;
    const int xcd = bid & 7, q = total >> 3, rem = total & 7;
    int i = xcd * q + (xcd < rem ? xcd : rem) + (bid >> 3);
    t.part = i / each;
    i -= t.part * each;
    int n = (int)((__builtin_sqrtf(8.f * (float)i + 1.f) - 1.f) * 0.5f);
    n += (n + 1) * (n + 2) / 2 <= i ? 1 : 0;  // (the root is off by less than one)
    n -= n * (n + 1) / 2 > i ? 1 : 0;
    t.n = n;
    t.m = i - n * (n + 1) / 2;
  }
  // (vector units took the quotients and the root: back to scalars, for all that follows)
  t.m = __builtin_amdgcn_readfirstlane(t.m);
  t.n = __builtin_amdgcn_readfirstlane(t.n);
  t.part = __builtin_amdgcn_readfirstlane(t.part);
  return t;
}

// One tile.  Epi: what happens to the sums, with kBarriers barriers; called by the
// waves that hold them with
//   run(acc, m0, n0, at, wave-in-M, wave-in-N, lane, lds)
// where acc[fn][fm][i] is row m0 + fm * 16 + (lane & 15), column
// n0 + fn * 16 + (lane >> 4) * 4 + i of the wave's part.
//
// STAGES 2: two slabs in LDS, one on its way while the other is multiplied; a
// barrier a slab.  Work-groups that share a CU hide each other's waits.  (More
// stages change nothing: a slab's time is its barrier, its LDS reads and its
// products one after the other, 0.4 us on a 64 x 64 tile, not the loads.)
// GROUPS: so many slabs are multiplied at a time, each by its own WM x WN waves,
// and the groups' sums joined through LDS at the end: for products with fewer
// tiles than the device has CUs, whose time is the length of the reduction.
// STAGES 3: two slabs of a group on their way, for short reductions, whose time is the
// latency of their loads one after the other (8-bit 301 x 1537 x 2053 18.4 -> 16.7 us).
// LOOSE: operands that are no 16-byte chunks, through registers (301 x 1537 x 2053
// f16: 16 us; 304 x 1536 x 2048 of whole chunks 10).
// Measured, bf16: the 256 x 256 tile without an epilogue 1.47 PFLOP/s on random
// values (1.75 on zeros: the clock falls with the load), with plain stores 8192 x
// 4096 x 4096 213-220 us (1.25-1.29 PFLOP/s; a library product 209-216), d_weight's
// roles 196 us; 64 x 64 and four slabs at a time 304 x 1536 x 2048 10 us.  Float32
// 515 x 896 x 1152 16-17 us a product of either direction.
// STAGES 0 (the 256 x 256 tile, one work-group a CU): two slabs in two halves.
// While the products of one half run, the fragments of the next are read from
// LDS.  In the middle of slab t every wave has its last fragments of the slab in
// registers: after that barrier slab t + 2 may overwrite it, and slab t + 1
// (loaded a whole slab ago) is complete.
template <int DT, bool AK, bool BK, int BM, int BN, int WM, int WN, int STAGES, int GROUPS, bool LOOSE,
          class Epi, class Plan = GemmPlan>
__global__ __launch_bounds__(WM* WN* GROUPS* kWave, 2) void k_gemm(Plan g, Epi epi) {
  constexpr bool kBatch = std::is_same_v<Plan, BatchPlan>;
  constexpr int kWaves = WM * WN;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  using A = std::conditional_t<LOOSE, LooseSide<DT, AK, BM, kWaves>, Side<DT, AK, BM, kWaves>>;
  using B = std::conditional_t<LOOSE, LooseSide<DT, BK, BN, kWaves>, Side<DT, BK, BN, kWaves>>;
  static_assert(!LOOSE || STAGES >= 2, "two buffers");
  constexpr int kStage = A::kBytes + B::kBytes;
  __shared__ __attribute__((aligned(1024))) char lds[2 * GROUPS * kStage];

  const int lane = threadIdx.x & (kWave - 1);
  const int wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wave = wave_all % kWaves, group = wave_all / kWaves;
  TileAt at;
  int slab0, slabs;
  if constexpr (kBatch) {
    at = tile_at((int)blockIdx.x, g);
    g.a.p = (const char*)g.a.p + at.part * g.step_a;
    g.b.p = (const char*)g.b.p + at.part * g.step_b;
    slab0 = 0;
    slabs = g.rest_a ? 3 * g.slabs : g.slabs;
  } else {
    at = tile_at((int)blockIdx.x, g.tiles_m, g.tiles_n, g.parts);
    slab0 = at.part * g.slabs_per_part;
    slabs = min(g.slabs_per_part, g.slabs - slab0);
  }
  const int m0 = at.m * BM, n0 = at.n * BN;
  const int wm = wave % WM, wn = wave / WM;

  A a;
  B b;
  const auto start = [&] {
    a.init(g.a, m0, slab0 + group, wave, lane);
    b.init(g.b, n0, slab0 + group, wave, lane);
    if constexpr (!LOOSE) {
      a.step *= GROUPS;
      b.step *= GROUPS;
    }
  };
  if constexpr (!kBatch) start();
  // reduction steps of this part's last slab
  const int last_a = (AK ? g.a.rows : g.a.cols) - (slab0 + slabs - 1) * kSlabOf<DT>;
  const int last_b = (BK ? g.b.rows : g.b.cols) - (slab0 + slabs - 1) * kSlabOf<DT>;

  using V = Sum<DT>;
  V acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = V{0, 0, 0, 0};

  const uint32_t lds0 = lds_address(lds);
  // Batches: slab t of the reduction, which goes over the operands' parts in turn.
  const char *base_a = nullptr, *base_b = nullptr;
  if constexpr (kBatch) {
    a.init(g.a, m0, 0, wave, lane);
    b.init(g.b, n0, 0, wave, lane);
    base_a = a.base;
    base_b = b.base;
  }
  const auto seek = [&](int t) {
    if constexpr (kBatch) {
      const bool second = t >= g.slabs, third = t >= 2 * g.slabs;
      // (a slab is at most 64 rows of 2^22 elements: a step has 32 bits)
      const uint64_t at_slab = (uint32_t)(t - (third ? 2 * g.slabs : second ? g.slabs : 0));
      a.base = base_a + at_slab * (uint32_t)a.step + (third ? g.rest_a : 0);
      b.base = base_b + at_slab * (uint32_t)b.step + (third ? 0 : second ? g.rest_b : 0);
      settled(a.base, b.base);
    }
  };
  const auto fetch_full = [&](int buffer) {
    if constexpr (!LOOSE) {
      const uint32_t dst = lds0 + buffer * kStage;
      a.template load<false>(dst, 0, wave, lane);
      b.template load<false>(dst + A::kBytes, 0, wave, lane);
    }
  };
  // (inlined: called, it would keep both sides and what they hold in scratch memory, and
  // wait there for a slab's loads before its products)
  const auto fetch = [&](int slab, int buffer) __attribute__((always_inline)) {
    if constexpr (LOOSE) {
      a.hold(slab0 + slab, g.a.rows, wave, lane);
      b.hold(slab0 + slab, g.b.rows, wave, lane);
    } else if constexpr (kBatch) {
      seek(slab);
      fetch_full(buffer);
    } else if (slab + 1 < slabs) {
      fetch_full(buffer);
    } else {
      const uint32_t dst = lds0 + buffer * kStage;
      a.template load<true>(dst, last_a, wave, lane);
      b.template load<true>(dst + A::kBytes, last_b, wave, lane);
    }
  };
  const auto land = [&](int buffer) {  // LOOSE: what fetch() holds
    if constexpr (LOOSE) {
      a.place(lds + buffer * kStage, wave, lane);
      b.place(lds + buffer * kStage + A::kBytes, wave, lane);
    }
  };
  const auto read = [&](v4i (&fa)[FM], v4i (&fb)[FN], int buffer, int kk) {
    const char* cur = lds + buffer * kStage;
#pragma unroll
    for (int i = 0; i < FN; ++i)
      fb[i] = B::frag(cur + A::kBytes, wn * (FN * 16) + i * 16, kk, lane);
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[i] = A::frag(cur, wm * (FM * 16) + i * 16, kk, lane);
  };
  const auto multiply = [&](const v4i (&fa)[FM], const v4i (&fb)[FN]) {
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int i = 0; i < FN; ++i) mma<DT>(acc[i][j], fb[i], fa[j]);
  };

  // The groups' sums to the first one's waves, and the epilogue.
  const auto join_groups = [&] {
    if constexpr (GROUPS > 1) {
      // [group - 1][fragment][lane] of every wave; the first group adds them up in order
      constexpr int kFrags = FM * FN;
      __syncthreads();
      V* sums = (V*)lds;
      static_assert((GROUPS - 1) * kWaves * kFrags * kWave * 16 + WN * BM * 8 <= (int)sizeof(lds),
                    "the sums and an epilogue's pair of floats for every row and wave");
      static_assert((GROUPS - 1) * kWaves * kFrags * kWave * 16 + kWaves * FN * 1024 <= (int)sizeof(lds),
                    "the sums and an epilogue's 16 rows for every wave");
      if (group > 0) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
          for (int j = 0; j < FM; ++j)
            sums[(((group - 1) * kWaves + wave) * kFrags + i * FM + j) * kWave + lane] = acc[i][j];
      }
      __syncthreads();
      if (group > 0) {
        for (int k = 0; k < Epi::kBarriers; ++k) __syncthreads();  // (those of the epilogue)
        return;
      }
      for (int k = 0; k < GROUPS - 1; ++k)
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
          for (int j = 0; j < FM; ++j)
            acc[i][j] += sums[((k * kWaves + wave) * kFrags + i * FM + j) * kWave + lane];
      epi.template run<FM, FN, BM, BN, WM, WN>(
          acc, m0, n0, at, wm, wn, lane,
          lds + (GROUPS - 1) * kWaves * kFrags * kWave * 16);
    }
  };

  if constexpr (STAGES == 0) {
    const auto settle = [] {
      __builtin_amdgcn_sched_barrier(0);
      wait_loads<0>();
      barrier();
    };
    v4i fa[2][FM], fb[2][FN];
    fetch(0, 0);
    settle();
    if (slabs > 1) fetch(1, 1);
    read(fa[0], fb[0], 0, 0);
    int t = 0;
    // Half a slab's products, a row of fragments at a time, the next half's fragments
    // and (LOADS) a slab's loads on their way between them: left alone the compiler
    // reads all fragments after the products, into the same registers, and the
    // loads go out in one burst that the products stand behind (8192 x 4096 x 4096:
    // 213 us, and 203 in this order; k-major 209 and 197).
    const auto half = [&](v4i (&na)[FM], v4i (&nb)[FN], int buffer, int kk, const v4i (&ca)[FM],
                          const v4i (&cb)[FN], auto loads, int filled) {
      const char* cur = lds + buffer * kStage;
      const uint32_t dst = lds0 + filled * kStage;
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        if (j < FN) nb[j] = B::frag(cur + A::kBytes, wn * (FN * 16) + j * 16, kk, lane);
        na[j] = A::frag(cur, wm * (FM * 16) + j * 16, kk, lane);
        if constexpr (decltype(loads)::value) {
          if (j < A::kUnits)
            a.load_unit(j, dst, wave);
          else
            b.load_unit(j - A::kUnits, dst + A::kBytes, wave);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < FN; ++i) mma<DT>(acc[i][j], cb[i], ca[j]);
      }
    };
    static_assert(FN <= FM && A::kUnits + B::kUnits == FM, "a load a row of fragments");
    for (; t + 3 < slabs; ++t) {
      half(fa[1], fb[1], t & 1, 1, fa[0], fb[0], std::false_type{}, 0);
      settle();
      seek(t + 2);
      half(fa[0], fb[0], (t + 1) & 1, 0, fa[1], fb[1], std::true_type{}, t & 1);
      if constexpr (!kBatch) {
        a.base += a.step;
        b.base += b.step;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    for (; t < slabs; ++t) {
      read(fa[1], fb[1], t & 1, 1);
      multiply(fa[0], fb[0]);
      settle();
      if (t + 2 < slabs) fetch(t + 2, t & 1);
      if (t + 1 < slabs) read(fa[0], fb[0], (t + 1) & 1, 0);
      multiply(fa[1], fb[1]);
    }
  } else if constexpr (STAGES == 3) {
    static_assert(DT != LSAMP_DTYPE_F32 && GROUPS > 1, "the products of a slab at once");
    const auto step = [&](int buffer) {
      v4i fa[2][FM], fb[2][FN];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) read(fa[kk], fb[kk], buffer, kk);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) multiply(fa[kk], fb[kk]);
    };
    // (every wave makes as many turns as the first group: their barriers)
    if constexpr (LOOSE) {
      v4i ha[2][A::kUnits], hb[2][B::kUnits];
      const auto hold = [&](int t, int set) {
        a.hold(ha[set], slab0 + t, g.a.rows, wave, lane);
        b.hold(hb[set], slab0 + t, g.b.rows, wave, lane);
      };
      const auto put = [&](int buffer, int set) {
        a.place(ha[set], lds + buffer * kStage, wave, lane);
        b.place(hb[set], lds + buffer * kStage + A::kBytes, wave, lane);
      };
      // slab t is in LDS, t + GROUPS in set `set`, t + 2 GROUPS in the other
      const auto turn = [&](int t, int buffer, int set) {
        __builtin_amdgcn_sched_barrier(0);
        wait_lds();
        barrier();
        if (t < slabs) step(buffer);
        const int other = buffer < GROUPS ? buffer + GROUPS : buffer - GROUPS;
        if (t + GROUPS < slabs) put(other, set);
        if (t + 3 * GROUPS < slabs) hold(t + 3 * GROUPS, set);
      };
      if (group < slabs) hold(group, 0);
      if (group + GROUPS < slabs) hold(group + GROUPS, 1);
      if (group < slabs) put(group, 0);
      if (group + 2 * GROUPS < slabs) hold(group + 2 * GROUPS, 0);
      for (int t = group; t - group < slabs; t += 2 * GROUPS) {
        turn(t, group, 1);
        if (t + GROUPS - group < slabs) turn(t + GROUPS, group + GROUPS, 0);
      }
    } else {
      constexpr int kFetch = A::kUnits + B::kUnits;
      if (group < slabs) fetch(group, group);
      if (group + GROUPS < slabs) fetch(group + GROUPS, group + GROUPS);
      int buffer = group;
      for (int t = group; t - group < slabs; t += GROUPS) {
        __builtin_amdgcn_sched_barrier(0);
        if (t + GROUPS < slabs)
          wait_loads<kFetch>();
        else
          wait_loads<0>();
        barrier();
        if (t < slabs) step(buffer);
        if (t + 2 * GROUPS - group < slabs) {  // (the same for all: the buffer is read by then)
          __builtin_amdgcn_sched_barrier(0);
          wait_lds();
          barrier();
          if (t + 2 * GROUPS < slabs) fetch(t + 2 * GROUPS, buffer);
        }
        buffer = buffer < GROUPS ? buffer + GROUPS : buffer - GROUPS;
      }
    }
    join_groups();
    return;
  } else {
    // ANY: float32 values that may not be finite.
    const auto reduce = [&](auto any) {
      // buffer: (parity of the step) * GROUPS + group
      if (group < slabs) {
        fetch(group, group);
        land(group);
      }
      int buffer = group;
      for (int t = group; t - group < slabs; t += GROUPS) {
        __builtin_amdgcn_sched_barrier(0);
        wait_loads<0>();
        barrier();
        const int other = buffer < GROUPS ? buffer + GROUPS : buffer - GROUPS;
        // (the slab that the other buffer held was multiplied before the barrier)
        if (t + GROUPS < slabs) fetch(t + GROUPS, other);
        if (GROUPS == 1 || t < slabs) {
          v4i fa[2][FM], fb[2][FN];
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) read(fa[kk], fb[kk], buffer, kk);
          if constexpr (DT != LSAMP_DTYPE_F32) {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) multiply(fa[kk], fb[kk]);
          } else if constexpr (!decltype(any)::value) {
            Split sb[FN];
#pragma unroll
            for (int i = 0; i < FN; ++i) sb[i] = split8(fb[0][i], fb[1][i]);
#pragma unroll
            for (int j = 0; j < FM; ++j) {
              __builtin_amdgcn_sched_barrier(0);  // (one split fragment of A at a time)
              const Split sa = split8(fa[0][j], fa[1][j]);
#pragma unroll
              for (int i = 0; i < FN; ++i)
                mma_split(acc[i][j], sb[i].h, sb[i].h, sb[i].m, sb[i].l, sa.h, sa.h, sa.m, sa.l);
            }
          } else {
#pragma unroll
            for (int j = 0; j < FM; ++j)
#pragma unroll
              for (int i = 0; i < FN; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                const SplitAny sb = split8_any(fb[0][i], fb[1][i]), sa = split8_any(fa[0][j], fa[1][j]);
                mma_split(acc[i][j], sb.h, sb.hx, sb.m, sb.l, sa.h, sa.hx, sa.m, sa.l);
              }
          }
        }
        if (t + GROUPS < slabs) land(other);
        buffer = other;
      }
    };
    reduce(std::false_type{});
    if constexpr (DT == LSAMP_DTYPE_F32) {
      bool nan = false;
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) nan |= acc[i][j][k] != acc[i][j][k];
      if (__syncthreads_or(nan)) {
        start();
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
          for (int j = 0; j < FM; ++j) acc[i][j] = V{0, 0, 0, 0};
        reduce(std::true_type{});
      }
    }
    if constexpr (GROUPS > 1) {
      join_groups();
      return;
    }
  }
  __syncthreads();
  epi.template run<FM, FN, BM, BN, WM, WN>(acc, m0, n0, at, wm, wn, lane, lds);
}

}  // namespace gemm
}  // namespace lsamp

#endif
