// lsamp_int8.hip — products of 8-bit integers whose rows have scales:
//
//   out[m][n] = act(xs[m] ws[n] sum_k x[m][k] w[n][k] + bias[n]) + residual[m][n]
//
// Compiled once per element type of bias, residual and out (LSAMP_DT).  The sums
// are whole numbers of 32 bits (127^2 k, exact for the lengths that the entry
// point takes); one becomes float32 with a rounding of 2^-24, and its two scales
// are multiplied first, another, where that gives a normal number.  The tiles are
// lsamp_gemm.h's and lsamp_skinny.h's: a slab of 128 bytes is 128 steps, an instruction
// takes 64 steps of a 16 x 16 tile in the time that it takes 32 of 16-bit elements, so a
// product moves half the bytes and takes half the time of a 16-bit one on either side of
// the roofline: 8192 x 4096 x 4096 130 to 133 us without a residual (2.1 POP/s; a library
// product 127), 64 x 2048 x 151936 65, one row of it 55 (5.7 TB/s).  Rows of W that are
// no 16-byte chunks cost more (301 x 1537 x 2053 12 us, 304 x 1536 x 2048 7).
#include <hip/hip_runtime.h>

#include "lsamp_epilogue.h"
#include "lsamp_gemm.h"
#include "lsamp_head.h"
#include "lsamp_quant.h"
#include "lsamp_skinny.h"

namespace lsamp {
namespace gemm {
namespace {

struct LinearInt8 : Linear {
  const float* x_scale;
  const float* w_scale;
  __device__ __forceinline__ v4f w_at(int c) const { return load4f(w_scale + c, n - c); }
  // The smallest and largest magnitude of four scales (past the last column they are 0).
  struct Range {
    float low, high;
  };
  static __device__ __forceinline__ Range range(v4f ws) {
    return Range{fminf(fminf(fabsf(ws[0]), fabsf(ws[1])), fminf(fabsf(ws[2]), fabsf(ws[3]))),
                 fmaxf(fmaxf(fabsf(ws[0]), fabsf(ws[1])), fmaxf(fabsf(ws[2]), fabsf(ws[3])))};
  }
  // The sums of N rows by their scales, four columns each.  Two scales of tiny or huge rows
  // may have a product that is no normal number: the sum then takes the smaller one first,
  // which leaves it one, for a scale is 2^-126 or more.
  template <int N>
  static __device__ __forceinline__ void scale(v4f (&r)[N], const v4i (&v)[N], const float (&xs)[N],
                                               v4f ws, Range w) {
    Range x{fabsf(xs[0]), fabsf(xs[0])};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x.low = fminf(x.low, fabsf(xs[i]));
      x.high = fmaxf(x.high, fabsf(xs[i]));
      r[i] = __builtin_convertvector(v[i], v4f) * (ws * xs[i]);
    }
    if (!(x.low * w.low >= 1.17549435e-38f && x.high * w.high <= 3.4028234e38f)) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool less = fabsf(ws[k]) < fabsf(xs[i]);
          r[i][k] = (float)v[i][k] * (less ? ws[k] : xs[i]) * (less ? xs[i] : ws[k]);
        }
    }
  }
  static __device__ __forceinline__ v4f scaled(v4i v, float xs, v4f ws) {
    v4f r[1];
    scale<1>(r, {v}, {xs}, ws, range(ws));
    return r[0];
  }
  __device__ __forceinline__ v4f result(v4f v, v4f b, v4f res) const {
    v = activate(activation, softcap, v + b);
    return residual ? v + res : v;
  }
  __device__ __forceinline__ void put(int r, int c, v4i v, int) const {
    finish(r, c, scaled(v, x_scale[r], w_at(c)), bias_at(c), residual_at(r, c));
  }
  // A row's residual as it lies in memory.
  typedef uint32_t Raw __attribute__((ext_vector_type(sizeof(S))));
  __device__ __forceinline__ Raw raw_residual(int r, int c) const {
    Raw o = 0;
    if (!residual || r >= m || c >= n) return o;
    const S* const p = (const S*)residual + (int64_t)r * ld_residual + c;
    if (n - c >= 4) {
      o = ((const Any<Raw, S>*)p)->v;
    } else {
      S e[4] = {};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < n - c) e[k] = p[k];
      __builtin_memcpy(&o, e, sizeof o);
    }
    return o;
  }
  // Linear::run, but with four rows' residuals on their way (float32: two): with one, their
  // loads add 29 us to the 133 of 8192 x 4096 x 4096, so 12.
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4i (&acc)[FN][FM], int m0, int n0, TileAt, int wm, int wn,
                                      int lane, char* lds) const {
    const Along<FN> at(lane);
    char* const mine = lds + (wn * WM + wm) * (FN * 1024);
    const int r0 = m0 + wm * (FM * 16) + at.row, c = n0 + wn * (FN * 16) + at.col;
    const v4f b = bias_at(c), ws = c < n ? w_at(c) : v4f{0.f, 0.f, 0.f, 0.f};
    const Range w = range(ws);
    constexpr int kAhead = 8 / sizeof(S) < FM ? 8 / sizeof(S) : FM;
    Raw res[kAhead][FN];
    float xs[FN];
    const auto scale_of = [&](int j) {
#pragma unroll
      for (int i = 0; i < FN; ++i) xs[i] = x_scale[min(r0 + j * 16 + i * at.kRows, m - 1)];
    };
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
#pragma unroll
      for (int i = 0; i < FN; ++i) res[j][i] = raw_residual(r0 + j * 16 + i * at.kRows, c);
    scale_of(0);
#pragma unroll 1
    for (int j = 0; j < FM; ++j) {
      const int r = r0 + j * 16;
      v4i v[FN];
      Raw add[FN];
      float s[FN];
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        v[i] = acc[i][0];
#pragma unroll
        for (int k = 0; k + 1 < FM; ++k) acc[i][k] = acc[i][k + 1];
        add[i] = res[0][i];
#pragma unroll
        for (int k = 0; k + 1 < kAhead; ++k) res[k][i] = res[k + 1][i];
        res[kAhead - 1][i] = raw_residual(j + kAhead < FM ? r + kAhead * 16 + i * at.kRows : m, c);
        s[i] = xs[i];
      }
      scale_of(j + 1);
      exchange<FN>(v, mine, lane);
      v4f y[FN];
      scale<FN>(y, v, s, ws, w);
#pragma unroll
      for (int i = 0; i < FN; ++i)
        if (r + i * at.kRows < m && c < n)
          finish(r + i * at.kRows, c, y[i], b,
                 __builtin_convertvector(__builtin_bit_cast(v4e, add[i]), v4f));
    }
  }
};

#if LSAMP_DT == 0
struct PartialInt8 : EpiPartial {
  static constexpr int kBarriers = 0;
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4i (&acc)[FN][FM], int m0, int n0, TileAt tile, int wm, int wn,
                                      int lane, char* lds) const {
    const int r0 = m0 + wm * (FM * 16) + (lane & 15);
    const int c0 = n0 + wn * (FN * 16) + (lane >> 4) * 4;
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int i = 0; i < FN; ++i)
        if (r0 + j * 16 < m && c0 + i * 16 < n)
          *(v4i*)(out + tile.part * part_stride + (int64_t)(r0 + j * 16) * ld + c0 + i * 16) =
              acc[i][j];
  }
};
#endif

#define LSAMP_TILE(THREADS, ...)                                                                  \
  hipLaunchKernelGGL((k_gemm<kInt8, false, false, __VA_ARGS__, E>), grid, dim3(THREADS), 0, st, g, e)

template <class E>
int launch(GemmTile tile, const GemmPlan& g, const E& e, void* stream) {
  const dim3 grid((unsigned)(g.tiles_m * g.tiles_n * g.parts));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (tile) {
    case kTile256: LSAMP_TILE(512, 256, 256, 2, 4, 0, 1, false); break;
    case kTile128: LSAMP_TILE(256, 128, 128, 2, 2, 2, 1, false); break;
    case kTile64: LSAMP_TILE(256, 64, 64, 2, 2, 2, 1, false); break;
    case kTile128x2: LSAMP_TILE(512, 128, 128, 2, 2, 2, 2, false); break;
    case kTile64x4: LSAMP_TILE(1024, 64, 64, 2, 2, 3, 4, false); break;
    case kLoose128: LSAMP_TILE(256, 128, 128, 2, 2, 2, 1, true); break;
    case kLoose64: LSAMP_TILE(256, 64, 64, 2, 2, 2, 1, true); break;
    case kLoose64x4: LSAMP_TILE(1024, 64, 64, 2, 2, 3, 4, true); break;
    default: return (int)hipErrorInvalidValue;
  }
  return (int)hipGetLastError();
}

template <int NF, int WK>
int launch_skinny(const GemmPlan& g, const LinearInt8& e, void* stream) {
  const dim3 grid((unsigned)g.tiles_n), threads(WK * kWave);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (g.a.rows <= 16)
    hipLaunchKernelGGL((k_skinny<kInt8, 1, NF, WK, true, LinearInt8>), grid, threads, 0, st, g, e);
  else if (g.a.rows <= 32)
    hipLaunchKernelGGL((k_skinny<kInt8, 2, NF, WK, true, LinearInt8>), grid, threads, 0, st, g, e);
  else
    hipLaunchKernelGGL((k_skinny<kInt8, 4, NF, WK, true, LinearInt8>), grid, threads, 0, st, g, e);
  return (int)hipGetLastError();
}

// ------------------------------------------------------------ x kept in LDS
// Up to 64 rows whose 8-bit values fit in LDS (128 KB: 64 x 2048, 16 x 8192): a work-group
// brings x there once, and its eight waves read nothing but W, chunks of 16 bytes of
// 16 of its rows straight into fragments, kDepth slabs ahead and from one block of 16
// columns to the next (k_skinny reads a slab of x beside every slab of W).  WK 1: a wave
// has blocks of its own, for outputs that are many of them for all waves; 8: the waves
// share a block, its slabs in turn, and join their sums.  ONCE: every work-group has one
// block, and a wave at most kDepth slabs.
//
// LINES: the eight waves' blocks lie side by side, and rows of 128 columns are stored
// together, from LDS, and past the L2: left there, 19 MB of them are written back when the
// kernel ends, after the last of W has been read (64 x 2048 x 151936: 74 us so, stored
// past it 66; 56 without any stores).
//
// A row of W ends anywhere: the last slab's chunks are read from the row's last 16 bytes
// where they would pass its end, and moved down; what lies behind meets zeros of x.
//
// FUSED: x is of the block's own type, and every work-group quantises it as it brings
// it (a launch less, for one row or two: 1 x 2048 x 2048 7.3 -> 4.7 us).
constexpr int kResidentWaves = 8;

template <int MF, int WK, int KB, bool FUSED, bool ONCE, bool LINES>
__global__ __launch_bounds__(kResidentWaves* kWave, 2) void k_resident(ResidentPlan g, LinearInt8 e) {
  constexpr int kThreads = kResidentWaves * kWave;
  constexpr int kDepth = WK == 1 || ONCE ? 8 : 4;
  constexpr int kLine = kResidentWaves * 16 + 8;  // elements of a row of results in LDS
  static_assert(!LINES || (WK == 1 && DT != LSAMP_DTYPE_F32), "blocks of 16-bit elements side by side");
  __shared__ __attribute__((aligned(16))) S lines[LINES ? MF * 16 : 1][LINES ? kLine : 1];
  __shared__ __attribute__((aligned(1024))) char xs[KB * 1024];
  __shared__ float scales[MF * 16];
  __shared__ v4i sums[WK > 1 ? WK - 1 : 1][WK > 1 ? MF : 1][kWave];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int slabs = (g.k + 127) / 128, pitch = (g.k + 255) / 256 * 256;
  // (16 rows' chunks of one number fall on all banks)
  const auto turned = [](int r, int chunk) { return (chunk & ~15) | ((chunk ^ r) & 15); };
  const auto place = [&](int r, int chunk) { return r * pitch + turned(r, chunk) * 16; };

  // This wave's blocks of 16 columns, and its slabs of one: first, first + WK, ...
  const int blocks = (e.n + 15) / 16;
  const int block0 = WK == 1 ? (int)blockIdx.x * kResidentWaves + wave : (int)blockIdx.x;
  const int block_step = WK == 1 ? (int)gridDim.x * kResidentWaves : (int)gridDim.x;
  const int first = WK == 1 ? 0 : wave;
  const int steps = slabs > first ? (slabs - first + WK - 1) / WK : 0;
  const int turns = (steps + kDepth - 1) / kDepth;
  const int row = lane & 15, at = (lane >> 4) * 16;

  v4i ring[kDepth][2];
  // (always loads, so that the compiler counts what is under way: past the last step the
  // last one's bytes again)
  const auto load = [&](v4i (&to)[2], int block, int step) {
    const int slab = first + WK * min(step, max(steps - 1, 0));
    const int64_t r = min(min(block, blocks - 1) * 16 + row, e.n - 1);
    const char* const p = (const char*)g.w + r * g.ld_w;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
      to[kk] = load_chunk<kInt8>(p + min(slab * 128 + kk * 64 + at, g.k - 16));
  };
  const auto fill = [&] {
#pragma unroll
    for (int u = 0; u < kDepth; ++u)
      if (!ONCE || u < steps) load(ring[u], block0, u);
  };
  if constexpr (FUSED) {
    __shared__ uint32_t tops[2][kResidentWaves];
    constexpr int kChunks = 2;  // of eight values a thread: 8,192 in all
    constexpr int kPer = 8 / kChunkOf<DT>;
    v4i raw[kChunks][kPer];
    const auto fetch = [&](int r) {
      const char* const x = (const char*)g.x + (int64_t)r * g.ld_x * El<DT>::kBytes;
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
#pragma unroll
        for (int h = 0; h < kPer; ++h) {
          const int c = (i * kThreads + (int)threadIdx.x) * 8 + h * kChunkOf<DT>;
          raw[i][h] = load_chunk<DT>(x + (int64_t)min(c, g.k - kChunkOf<DT>) * El<DT>::kBytes);
        }
      if (g.k % kChunkOf<DT>) {  // (where the row ends)
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
#pragma unroll
          for (int h = 0; h < kPer; ++h) {
            const int c = (i * kThreads + (int)threadIdx.x) * 8 + h * kChunkOf<DT>;
            if (c < g.k && c + kChunkOf<DT> > g.k) raw[i][h] = load_chunk_end<DT>(x, c, g.k);
          }
      }
    };
    const auto value = [&](int i, int k, S v) {  // (0 past the row's end)
      return (i * kThreads + (int)threadIdx.x) * 8 + k < g.k ? (float)v : 0.f;
    };
    // (x first: loads are waited for in their order, and W's come from far)
    fetch(0);
    fill();
    for (int r = 0; r < g.m; ++r) {
      float v[kChunks][8];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        S el[8];
        __builtin_memcpy(el, raw[i], 16 * kPer);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          v[i][k] = value(i, k, el[k]);
          top = max(top, magnitude(v[i][k]));
        }
      }
#pragma unroll
      for (int d = 32; d > 0; d /= 2) top = max(top, (uint32_t)__shfl_xor(top, d));
      if (lane == 0) tops[r & 1][wave] = top;
      __syncthreads();  // (a row's tops are read before the next but one's are written)
#pragma unroll
      for (int i = 0; i < kResidentWaves; ++i) top = max(top, tops[r & 1][i]);
      const float scale = row_scale(top), inverse = 1.f / scale;
      if (threadIdx.x == 0) scales[r] = scale;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int c = (i * kThreads + (int)threadIdx.x) * 8;
        if (i * kThreads * 8 < pitch) {
          const uint64_t q = quantize8(v[i], scale, inverse);
          if (c < pitch) *(uint64_t*)(xs + place(r, c / 16) + c % 16) = q;
        }
      }
      if (r + 1 < g.m) fetch(r + 1);
    }
  } else {
    fill();
    // (rows of 256 bytes, straight to LDS: 64 chunks in order an instruction, so the
    // chunks that the order asks for are read)
    const int chunks = pitch / 16, last = g.m * chunks - 1;
    for (int u = wave; u * kWave <= last; u += kResidentWaves) {
      const int i = min(u * kWave + lane, last), r = i / chunks, c = i - r * chunks;
      __builtin_amdgcn_global_load_lds(
          LSAMP_GLOBAL((const char*)g.x + (int64_t)r * g.ld_x + turned(r, c) * 16),
          LSAMP_LDS(xs + u * 1024), 16, 0, 0);
    }
    if ((int)threadIdx.x < g.m) scales[threadIdx.x] = e.x_scale[threadIdx.x];
    __builtin_amdgcn_sched_barrier(0);
    wait_loads<0>();
  }
  __syncthreads();

  v4i acc[MF];
#pragma unroll
  for (int j = 0; j < MF; ++j) acc[j] = v4i{0, 0, 0, 0};
  // (rows past the last repeat it)
  int x_row[MF];
#pragma unroll
  for (int j = 0; j < MF; ++j) x_row[j] = min(j * 16 + row, g.m - 1);
  // What fragment j's end needs: on its way from the block's start.
  struct Ends {
    v4f ws, b, res[WK == 1 ? MF : 1];
  };
  const auto ends = [&](int block, int j0) {
    Ends o;
    const int c = block * 16 + (lane >> 4) * 4;
    o.ws = c < e.n ? e.w_at(c) : v4f{0.f, 0.f, 0.f, 0.f};
    o.b = c < e.n ? e.bias_at(c) : v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < (WK == 1 ? MF : 1); ++j)
      o.res[j] = c < e.n ? e.residual_at((j0 + j) * 16 + row, c) : v4f{0.f, 0.f, 0.f, 0.f};
    return o;
  };
  const auto put = [&](int j, int block, v4i v, const Ends& o, v4f res) {
    const int r = j * 16 + row, c = block * 16 + (lane >> 4) * 4;
    if (r < g.m && c < e.n) e.finish(r, c, e.scaled(v, scales[r], o.ws), o.b, res);
  };
  // (LINES: every wave stays until the last of them has stored)
  for (int block = block0; (LINES ? block - wave : block) < blocks; block += block_step) {
    Ends o;
    if (WK == 1 || wave < MF) o = ends(block, WK == 1 ? 0 : wave);
    for (int turn = 0; turn < turns; ++turn) {
      const bool next = turn + 1 < turns;
      const int to_block = next ? block : block + block_step, to_turn = next ? turn + 1 : 0;
#pragma unroll
      for (int u = 0; u < kDepth; ++u) {
        const int step = turn * kDepth + u;
        if (step < steps) {  // (the same for the wave)
          const int slab = first + WK * step;
          v4i w[2] = {ring[u][0], ring[u][1]};
          if ((slab + 1) * 128 > g.k) {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
              const int over = slab * 128 + kk * 64 + at + 16 - g.k;
              w[kk] = moved_down(w[kk], min(max(over, 0), 15));
            }
          }
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) {
            v4i x[MF];
#pragma unroll
            for (int j = 0; j < MF; ++j)
              x[j] = *(const v4i*)(xs + place(x_row[j], slab * 8 + kk * 4 + (lane >> 4)));
#pragma unroll
            for (int j = 0; j < MF; ++j) mma<kInt8>(acc[j], w[kk], x[j]);
          }
        }
        if constexpr (!ONCE) load(ring[u], to_block, to_turn * kDepth + u);
      }
    }
    if constexpr (LINES) {
#pragma unroll
      for (int j = 0; j < MF; ++j) {
        const v4f v = e.result(e.scaled(acc[j], scales[x_row[j]], o.ws), o.b, o.res[j]);
        *(v4e*)&lines[j * 16 + row][wave * 16 + (lane >> 4) * 4] = __builtin_convertvector(v, v4e);
      }
      __syncthreads();
      const int c0 = (block - wave) * 16;
#pragma unroll
      for (int i = 0; i < MF * 16 * 16 / kThreads + (MF == 1); ++i) {
        const int q = i * kThreads + (int)threadIdx.x, r = q / 16, c = q % 16 * 8;
        if (r >= g.m || c0 + c >= e.n) continue;
        S* const to = (S*)e.out + (int64_t)r * e.ld_out + c0 + c;
        if (c0 + c + 8 <= e.n) {
          const v4i v = *(const v4i*)&lines[r][c];
          // (two wait states before its data may be overwritten, which the compiler does not
          // know to be a store's)
          asm volatile("global_store_dwordx4 %0, %1, off sc0 sc1 nt\n\ts_nop 1"
                       :
                       : "v"(to), "v"(v)
                       : "memory");
        } else {
          for (int k = 0; c0 + c + k < e.n; ++k) to[k] = lines[r][c + k];
        }
      }
      __syncthreads();
    } else if constexpr (WK == 1) {
#pragma unroll
      for (int j = 0; j < MF; ++j) put(j, block, acc[j], o, o.res[j]);
    } else {
      // (wave j adds up the rows of fragment j, its own sums among them)
#pragma unroll
      for (int j = 0; j < MF; ++j)
        if (wave != j) sums[wave - (wave > j)][j][lane] = acc[j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < MF; ++j)
        if (wave == j) {
          v4i v = acc[j];
#pragma unroll
          for (int k = 0; k < WK - 1; ++k) v += sums[k][j][lane];
          put(j, block, v, o, o.res[0]);
        }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < MF; ++j) acc[j] = v4i{0, 0, 0, 0};
  }
}

template <int MF, int KB, bool FUSED>
int launch_resident(const ResidentPlan& g, const LinearInt8& e, hipStream_t st) {
  const dim3 grid((unsigned)g.groups), threads(kResidentWaves * kWave);
  const bool once = g.groups >= (e.n + 15) / 16 && g.k <= 8 * 8 * 128;
  if (g.shared) {
    if (once)
      hipLaunchKernelGGL((k_resident<MF, 8, KB, FUSED, true, false>), grid, threads, 0, st, g, e);
    else
      hipLaunchKernelGGL((k_resident<MF, 8, KB, FUSED, false, false>), grid, threads, 0, st, g, e);
    return (int)hipGetLastError();
  }
  if constexpr (DT != LSAMP_DTYPE_F32 && KB == 128) {
    if (!e.wide) {
      hipLaunchKernelGGL((k_resident<MF, 1, KB, FUSED, false, true>), grid, threads, 0, st, g, e);
      return (int)hipGetLastError();
    }
  }
  hipLaunchKernelGGL((k_resident<MF, 1, KB, FUSED, false, false>), grid, threads, 0, st, g, e);
  return (int)hipGetLastError();
}

// The parts of a split reduction added up, and the epilogue: a quad of columns a thread.
__global__ __launch_bounds__(256) void k_join_int8(EpiPartial from, int parts, LinearInt8 e) {
  const int quads = (e.n + 3) / 4;
  const int64_t total = (int64_t)e.m * quads;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int r = (int)(i / quads), c = (int)(i % quads) * 4;
    const float* p = from.out + (int64_t)r * from.ld + c;
    v4i v = {0, 0, 0, 0};
#pragma unroll 8
    for (int k = 0; k < parts; ++k) v += *(const v4i*)(p + k * from.part_stride);
    e.put(r, c, v, 0);
  }
}

LinearInt8 epilogue(const EpiLinearInt8& p) {
  LinearInt8 e;
  static_cast<EpiLinear&>(e) = p;
  e.x_scale = p.x_scale;
  e.w_scale = p.w_scale;
  return e;
}

}  // namespace
}  // namespace gemm

using namespace gemm;

template <>
int Int8Ops<DT>::gemm_linear(GemmTile t, const GemmPlan& g, const EpiLinearInt8& p, void* st) {
  const LinearInt8 e = epilogue(p);
  if (t == kSkinny64) return launch_skinny<4, 4>(g, e, st);
  if (t == kSkinny16) return launch_skinny<1, 8>(g, e, st);
  return launch(t, g, e, st);
}
template <>
int Int8Ops<DT>::resident_linear(const ResidentPlan& g, const EpiLinearInt8& p, void* stream) {
  const LinearInt8 e = epilogue(p);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool small = (int64_t)g.m * ((g.k + 255) / 256 * 256) <= 16 << 10;
  if (g.m > 32) return launch_resident<4, 128, false>(g, e, st);
  if (g.m > 16) return launch_resident<2, 128, false>(g, e, st);
  if (!small) return launch_resident<1, 128, false>(g, e, st);
  return g.fused ? launch_resident<1, 16, true>(g, e, st) : launch_resident<1, 16, false>(g, e, st);
}
template <>
int Int8Ops<DT>::join_linear(const EpiPartial& from, int parts, const EpiLinearInt8& p, void* st) {
  const int64_t quads = (int64_t)p.m * ((p.n + 3) / 4);
  const int64_t blocks = (quads + 255) / 256;
  hipLaunchKernelGGL(k_join_int8, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0,
                     reinterpret_cast<hipStream_t>(st), from, parts, epilogue(p));
  return (int)hipGetLastError();
}

#if LSAMP_DT == 0
// (one for all element types: the sums are whole numbers)
int launch_partial_int8(GemmTile t, const GemmPlan& g, const EpiPartial& p, void* st) {
  PartialInt8 e;
  static_cast<EpiPartial&>(e) = p;
  return launch(t, g, e, st);
}
#endif

}  // namespace lsamp
