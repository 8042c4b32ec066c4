// lsamp_orth.hip — the orthogonal factor of a matrix, nearly: Newton-Schulz steps
//
//   X <- G / (|G|_F + eps);  a step:  A = X X^T,  B = b A + c A A,  X <- a X + B X
//
// for a wide or square matrix (rows <= columns), X X^T the smaller Gram matrix; for
// a tall one A = X^T X and X <- a X + X B.  An odd polynomial of the singular
// values, a step at a time, without taking the matrix apart.  Compiled once per
// type that the products are taken in (LSAMP_DT):
//
// float32: X, A and B are float32, the products those of lsamp_gemm.h (24 bits).
//
// float16 (for bfloat16 results): the products are float16's, at the full rate.  What
// a rounding of X does grows with the polynomial's slope at 0 in every step (485
// times in five of Muon's), and near-singular momenta are the rule: X alone in
// float16 leaves 1e-2 of such a result's norm, in bfloat16 1e-1.  So X has two
// float16 parts, x = hi + lo: the products take hi, the linear term a X both.  Then B's
// rounding is the largest; its diagonal (about -2.7 once the singular values are
// near 1, against an off-diagonal part of 0.3) is kept apart in float32 and joins the
// linear term.  What is left is 4e-4 to 1.1e-3 of the result's norm in five steps,
// below bfloat16's own 1.7e-3.  X is held times 2^10, A and B times 2^8, so that
// small elements stay normal numbers and the largest (singular values up to 8,
// |B| up to 128: the entry point checks the polynomials) stay finite.
//
// Of A and A A, which are symmetric, only the tiles at and right of the diagonal
// are computed, and stored on both sides.
#include <hip/hip_runtime.h>

#include "lsamp_epilogue.h"
#include "lsamp_gemm.h"
#include "lsamp_orth.h"

namespace lsamp {
namespace gemm {
namespace {

constexpr bool kHalf = DT == LSAMP_DTYPE_F16;
constexpr float kOfX = kHalf ? 1024.f : 1.f;  // what X, and what A and B are held times
constexpr float kOfA = kHalf ? 256.f : 1.f;
constexpr int kThreads = 256;

// ----------------------------------------------------------------- the start
template <int IN>
__device__ __forceinline__ float element(const void* p, int64_t i) {
  return (float)((const typename El<IN>::S*)p)[i];
}

// Sums of squares in 64 bits, which neither overflow nor underflow: a work-group's
// share of a matrix, added in a fixed order.
template <int IN>
__global__ __launch_bounds__(kThreads) void k_norm2(OrthStart p) {
  __shared__ double red[kThreads / kWave];
  const int matrix = (int)blockIdx.y;
  const char* const x = (const char*)p.x + (int64_t)matrix * p.step_x;
  double s = 0.0;
  for (int r = (int)blockIdx.x; r < p.rows; r += (int)gridDim.x)
    for (int c = (int)threadIdx.x; c < p.cols; c += kThreads) {
      const double v = (double)element<IN>(x, (int64_t)r * p.ld_x + c);
      s += v * v;
    }
  for (int d = 32; d > 0; d /= 2) s += __shfl_xor(s, d);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / kWave; ++w) s += red[w];
    p.part[(int64_t)matrix * p.parts + blockIdx.x] = s;
  }
}

// X0 = G 2^-e with 2^e <= |G|_F + eps < 2^(e + 1): no rounding of 16-bit values, and
// what is left of the norm goes into the first step's factors.
template <int IN>
__global__ __launch_bounds__(kThreads) void k_start(OrthStart p) {
  __shared__ double red[kThreads / kWave];
  const int matrix = (int)blockIdx.y;
  double s = 0.0;
  for (int i = (int)threadIdx.x; i < p.parts; i += kThreads)
    s += p.part[(int64_t)matrix * p.parts + i];
  for (int d = 32; d > 0; d /= 2) s += __shfl_xor(s, d);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = s;
  __syncthreads();
  s = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / kWave; ++w) s += red[w];
  const double norm = sqrt(s) + (double)p.eps;
  const bool finite = norm < INFINITY;
  const int e = finite ? ilogb(norm) : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) p.left[matrix] = finite ? (float)(ldexp(1.0, e) / norm) : NAN;
  const char* const x = (const char*)p.x + (int64_t)matrix * p.step_x;
  const double scale = ldexp((double)kOfX, -e);
  S* const hi = (S*)p.hi + (int64_t)matrix * p.step;
  S* const lo = kHalf ? (S*)p.lo + (int64_t)matrix * p.step : nullptr;
  const int wide = (p.cols + 7) / 8 * 8;
  for (int r = (int)blockIdx.x; r < p.rows; r += (int)gridDim.x)
    for (int c = (int)threadIdx.x; c < wide; c += kThreads) {
      // (a product of doubles: the scale of a tiny matrix is beyond float32)
      const float v =
          c < p.cols ? (float)((double)element<IN>(x, (int64_t)r * p.ld_x + c) * scale) : 0.f;
      const S h = (S)v;
      hi[(int64_t)r * p.ld + c] = h;
      if constexpr (kHalf) lo[(int64_t)r * p.ld + c] = (S)(v - (float)h);
    }
}

// ----------------------------------------------------------------- epilogues
// Sums and the same tile's mirror image: what is stored at (r, c) is stored at
// (c, r) too, unless the tile lies on the diagonal.  `value(r, c, sums)` gives four
// columns' results, zero past the last.
struct Symmetric : EpiSymmetric {
  static constexpr int kBarriers = 0;
  template <int FM, int FN, int BM, int BN, int WM, int WN, class F>
  __device__ __forceinline__ void store(v4f (&acc)[FN][FM], S* to, int m0, int n0, TileAt at, int wm,
                                        int wn, int lane, F value) const {
    const int r0 = m0 + wm * (FM * 16) + (lane & 15);
    const int c0 = n0 + wn * (FN * 16) + (lane >> 4) * 4;
    const int wide = (n + 7) / 8 * 8;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int r = r0 + j * 16;
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        const int c = c0 + i * 16;
        if (r >= n || c >= wide) continue;
        const v4f v = value(r, c, acc[i][j]);
        v4e e;
#pragma unroll
        for (int k = 0; k < 4; ++k) e[k] = c + k < n ? (S)v[k] : (S)0.f;
        *(v4e*)(to + (int64_t)r * ld + c) = e;
        if (at.m != at.n) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (c + k < n) to[(int64_t)(c + k) * ld + r] = e[k];
        }
      }
    }
  }
};

struct Gram : Symmetric {
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4f (&acc)[FN][FM], int m0, int n0, TileAt at, int wm, int wn,
                                      int lane, char*) const {
    const float s = left ? left[at.part] : 1.f;
    const float f = s * s * (kOfA / (kOfX * kOfX));
    store<FM, FN, BM, BN, WM, WN>(acc, (S*)out + at.part * step, m0, n0, at, wm, wn, lane,
                                  [&](int, int, v4f v) { return v * f; });
  }
};

struct Poly : Symmetric {
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4f (&acc)[FN][FM], int m0, int n0, TileAt at, int wm, int wn,
                                      int lane, char*) const {
    const S* const g = (const S*)in + at.part * step;
    float* const d = kHalf ? diagonal + at.part * step_d : nullptr;
    const float fc = c3 / kOfA;
    store<FM, FN, BM, BN, WM, WN>(
        acc, (S*)out + at.part * step, m0, n0, at, wm, wn, lane, [&](int r, int c, v4f v) {
          const v4e a = *(const v4e*)(g + (int64_t)r * ld + c);  // (whole quads of a row)
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = b3 * (float)a[k] + fc * v[k];
          if constexpr (kHalf) {
            const int k = r - c;
            if ((unsigned)k < 4u) {
              d[r] = (k == 0 ? v[0] : k == 1 ? v[1] : k == 2 ? v[2] : v[3]) * (1.f / kOfA);
#pragma unroll
              for (int q = 0; q < 4; ++q) v[q] = q == k ? 0.f : v[q];
            }
          }
          return v;
        });
  }
};

// X' = (a + diagonal) X + sums, as the next X or, at the last step, the result.
struct Update : EpiOrthUpdate {
  static constexpr int kBarriers = 0;
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4f (&acc)[FN][FM], int m0, int n0, TileAt at, int wm, int wn,
                                      int lane, char* lds) const {
    const Along<FN> along(lane);
    char* const mine = lds + (wn * WM + wm) * (FN * 1024);
    const int r0 = m0 + wm * (FM * 16) + along.row, c = n0 + wn * (FN * 16) + along.col;
    const int wide = (n + 7) / 8 * 8, valid = n - c;
    const float s = left ? left[at.part] : 1.f;
    const S* const hi = (const S*)x_hi + at.part * step;
    const S* const lo = kHalf ? (const S*)x_lo + at.part * step : nullptr;
    const float* const d = kHalf ? diagonal + at.part * step_d : nullptr;
    v4f by_col = {a1, a1, a1, a1};
    if (kHalf && tall && c < n) by_col += load4f(d + c, valid);
#pragma unroll 1
    for (int j = 0; j < FM; ++j) {
      v4f v[FN];
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        v[i] = acc[i][0];
#pragma unroll
        for (int k = 0; k + 1 < FM; ++k) acc[i][k] = acc[i][k + 1];
      }
      exchange<FN>(v, mine, lane);
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        const int r = r0 + j * 16 + i * along.kRows;
        if (r >= m || c >= wide) continue;
        const v4e h = *(const v4e*)(hi + (int64_t)r * ld + c);
        v4f x = __builtin_convertvector(h, v4f);
        v4f f = by_col;
        if constexpr (kHalf) {
          x += __builtin_convertvector(*(const v4e*)(lo + (int64_t)r * ld + c), v4f);
          if (!tall) f += d[r];
        }
        v4f y = (x * f + v[i] * (1.f / kOfA)) * s;
        if (!out) {
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = k < valid ? y[k] : 0.f;
          const v4e top = __builtin_convertvector(y, v4e);
          *(v4e*)((S*)to_hi + at.part * step + (int64_t)r * ld + c) = top;
          if constexpr (kHalf) {
            const v4f rest = y - __builtin_convertvector(top, v4f);
            *(v4e*)((S*)to_lo + at.part * step + (int64_t)r * ld + c) =
                __builtin_convertvector(rest, v4e);
          }
        } else if (valid > 0) {
          finish(at.part, r, c, y * (scale / kOfX), valid);
        }
      }
    }
  }
  template <typename O>
  __device__ __forceinline__ void finish_as(int64_t matrix, int r, int c, v4f v, int valid) const {
    O* const o = (O*)((char*)out + matrix * step_out) + (int64_t)r * ld_out + c;
    const O* const b = base ? (const O*)((const char*)base + matrix * step_base) +
                                  (int64_t)r * ld_base + c
                            : nullptr;
    typedef O v4o __attribute__((ext_vector_type(4)));
    typedef O v4u __attribute__((ext_vector_type(4), aligned(sizeof(O))));
    if (valid >= 4) {
      if (b) v += keep * __builtin_convertvector((v4o) * (const v4u*)b, v4f);
      *(v4u*)o = __builtin_convertvector(v, v4o);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < valid) o[k] = (O)(b ? v[k] + keep * (float)b[k] : v[k]);
    }
  }
  __device__ __forceinline__ void finish(int64_t matrix, int r, int c, v4f v, int valid) const {
    if constexpr (kHalf)
      finish_as<__bf16>(matrix, r, c, v, valid);
    else if (out_dtype == LSAMP_DTYPE_F32)
      finish_as<float>(matrix, r, c, v, valid);
    else
      finish_as<_Float16>(matrix, r, c, v, valid);
  }
};

template <class E, class P>
E with(const P& plan) {
  E e;
  static_cast<P&>(e) = plan;
  return e;
}

#define LSAMP_TILE(THREADS, ...)                                                                    \
  hipLaunchKernelGGL((k_gemm<DT, AK, BK, __VA_ARGS__, E, BatchPlan>), grid, dim3(THREADS), 0, st, g, \
                     e)

template <bool AK, bool BK, class E>
int launch(GemmTile tile, const BatchPlan& g, const E& e, void* stream) {
  const int64_t tiles = g.symmetric ? (int64_t)g.tiles_n * (g.tiles_n + 1) / 2
                                    : (int64_t)g.tiles_m * g.tiles_n;
  const dim3 grid((unsigned)(tiles * g.parts));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (tile) {
    case kTile256:
      if constexpr (kHalf) {
        LSAMP_TILE(512, 256, 256, 2, 4, 0, 1, false);
        break;
      }
      return (int)hipErrorInvalidValue;
    case kTile128: LSAMP_TILE(256, 128, 128, 2, 2, 2, 1, false); break;
    case kTile64: LSAMP_TILE(256, 64, 64, 2, 2, 2, 1, false); break;
    case kTile128x2: LSAMP_TILE(512, 128, 128, 2, 2, 2, 2, false); break;
    case kTile64x4: LSAMP_TILE(1024, 64, 64, 2, 2, 2, 4, false); break;
    default: return (int)hipErrorInvalidValue;
  }
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace gemm

using namespace gemm;

template <>
int OrthOps<DT>::start(const OrthStart& p, int batch, int in_dtype, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)p.parts, (unsigned)batch);
#define LSAMP_START(IN)                                                     \
  hipLaunchKernelGGL((k_norm2<IN>), grid, dim3(kThreads), 0, st, p);        \
  hipLaunchKernelGGL((k_start<IN>), grid, dim3(kThreads), 0, st, p)
  switch (in_dtype) {
    case LSAMP_DTYPE_F32: LSAMP_START(LSAMP_DTYPE_F32); break;
    case LSAMP_DTYPE_BF16: LSAMP_START(LSAMP_DTYPE_BF16); break;
    default: LSAMP_START(LSAMP_DTYPE_F16); break;
  }
  return (int)hipGetLastError();
}
template <>
int OrthOps<DT>::gram(bool tall, GemmTile t, const BatchPlan& g, const EpiSymmetric& p, void* st) {
  const Gram e = with<Gram>(p);
  return tall ? launch<true, true>(t, g, e, st) : launch<false, false>(t, g, e, st);
}
template <>
int OrthOps<DT>::poly(GemmTile t, const BatchPlan& g, const EpiSymmetric& p, void* st) {
  return launch<false, false>(t, g, with<Poly>(p), st);
}
template <>
int OrthOps<DT>::update(bool tall, GemmTile t, const BatchPlan& g, const EpiOrthUpdate& p, void* st) {
  const Update e = with<Update>(p);
  return tall ? launch<false, false>(t, g, e, st) : launch<false, true>(t, g, e, st);
}

}  // namespace lsamp
