// lsamp_orth.hip — the orthogonal factor of a matrix, nearly: Newton-Schulz steps
//
//   X <- G / (|G|_F + eps);  a step:  A = X X^T,  B = b A + c A A,  X <- a X + B X
//
// for a wide or square matrix (rows <= columns), X X^T the smaller Gram matrix; for
// a tall one A = X^T X and X <- a X + X B.  An odd polynomial of the singular
// values, a step at a time, without taking the matrix apart.
//
// The products are float16's, at the full rate of the matrix instructions.  What a
// rounding of X does grows with the polynomial's slope at 0 in every step (485 times in
// five of Muon's), and near-singular momenta are the rule: X in float16 alone leaves
// 1e-2 of such a result's norm, in bfloat16 1e-1.  So X, A and B have two float16 parts, x
// = hi + lo, 22 bits, and a product is three, hi hi + hi lo + lo hi, one after the other
// into the same float32 sums (WIDE): 3e-7 to 2e-6 of the result's norm in five steps of
// falling spectra and 1.3e-5 of a matrix of rank 8, float32's own steps 2e-7 to 1.3e-6 and
// 2.5e-5.
//
// Not WIDE, where the caller of a bfloat16 result asks for it: X has two parts, of which
// products take hi and the linear term a X both; A and B have one.  Then B's rounding is
// the largest; its diagonal (about -2.7 once the singular values are near 1, against
// an off-diagonal part of 0.3) is kept apart in float32 and joins the linear term.
// What is left is 4e-4 to 1.1e-3 of the result's norm in five steps, below
// bfloat16's own 1.7e-3; in ten, 1e-2 to 5e-2 of a spectrum down to 1e-6.
//
// X is held times 2^10, A and B times 2^8, so that small elements stay normal numbers
// and the largest (singular values up to 8, |B| up to 128: the entry point checks the
// polynomials) stay finite.  All matrices are held with zeros up to multiples of 64
// rows and columns, which the products keep.  Of A and A A, which are symmetric, only
// the tiles at and right of the diagonal are computed, and stored on both sides.
#include <hip/hip_runtime.h>

#include "lsamp_epilogue.h"
#include "lsamp_gemm.h"
#include "lsamp_orth.h"

namespace lsamp {
namespace gemm {
namespace {

static_assert(DT == LSAMP_DTYPE_F16, "the products' type");
constexpr float kOfX = 1024.f, kOfA = 256.f;
constexpr int kThreads = 256;
typedef _Float16 v8e __attribute__((ext_vector_type(8)));

// ----------------------------------------------------------------- the start
// Eight elements of a row, `valid` of them in it.
template <int IN>
__device__ __forceinline__ void load8(float (&v)[8], const char* row, int c, int valid) {
  using T = typename El<IN>::S;
  constexpr int N = kChunkOf<IN>;
  if (valid >= 8) {
#pragma unroll
    for (int i = 0; i < 8 / N; ++i) {
      const v4i q = load_chunk<IN>(row + (int64_t)(c + i * N) * El<IN>::kBytes);
      T e[N];
      __builtin_memcpy(e, &q, 16);
#pragma unroll
      for (int k = 0; k < N; ++k) v[i * N + k] = (float)e[k];
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < valid ? (float)((const T*)row)[c + k] : 0.f;
  }
}
__device__ __forceinline__ double block_sum(double s, double* red) {
  for (int d = 32; d > 0; d /= 2) s += __shfl_xor(s, d);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = s;
  __syncthreads();
  s = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / kWave; ++w) s += red[w];
  return s;
}

// Sums of squares in 64 bits, which neither overflow nor underflow: a work-group's
// share of a matrix, added in a fixed order.  Bound by memory: 4096 x 4096 bf16 9 us.
template <int IN>
__global__ __launch_bounds__(kThreads) void k_norm2(OrthStart p) {
  __shared__ double red[kThreads / kWave];
  const int matrix = (int)blockIdx.y;
  const char* const x = (const char*)p.x + (int64_t)matrix * p.step_x;
  const int lane = (int)threadIdx.x & ((1 << p.log_x) - 1), per = kThreads >> p.log_x;
  double s = 0.0;
  for (int r = (int)blockIdx.x * per + ((int)threadIdx.x >> p.log_x); r < p.rows;
       r += (int)gridDim.x * per)
    for (int c = lane * 8; c < p.cols; c += 8 << p.log_x) {
      float v[8];
      load8<IN>(v, x + (int64_t)r * p.ld_x * El<IN>::kBytes, c, p.cols - c);
#pragma unroll
      for (int k = 0; k < 8; ++k) s = fma((double)v[k], (double)v[k], s);
    }
  s = block_sum(s, red);
  if (threadIdx.x == 0) p.part[(int64_t)matrix * p.parts + blockIdx.x] = s;
}

// X0 = G 2^-e with 2^e <= |G|_F + eps < 2^(e + 1): no rounding of 16-bit values, and
// what is left of the norm goes into the first step's factors.  Memory: 4096 x 4096 bf16 to
// two parts 18 us (100 MB, 5.6 TB/s).
template <int IN>
__global__ __launch_bounds__(kThreads) void k_start(OrthStart p) {
  __shared__ double red[kThreads / kWave];
  const int matrix = (int)blockIdx.y;
  double s = 0.0;
  for (int i = (int)threadIdx.x; i < p.parts; i += kThreads)
    s += p.part[(int64_t)matrix * p.parts + i];
  const double norm = sqrt(block_sum(s, red)) + (double)p.eps;
  const bool finite = norm < INFINITY;
  const int e = finite ? ilogb(norm) : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0)
    p.left[matrix] = finite ? (float)(ldexp(1.0, e) / norm) : NAN;
  const char* const x = (const char*)p.x + (int64_t)matrix * p.step_x;
  // (in two factors: the scale of a tiny matrix is beyond float32)
  const float scale = ldexpf(kOfX, -e / 2), scale2 = ldexpf(1.f, -(e - e / 2));
  S* const hi = (S*)p.hi + (int64_t)matrix * p.step;
  S* const lo = (S*)p.lo + (int64_t)matrix * p.step;
  const int lane = (int)threadIdx.x & ((1 << p.log_x) - 1), per = kThreads >> p.log_x;
  for (int r = (int)blockIdx.x * per + ((int)threadIdx.x >> p.log_x); r < p.all_rows;
       r += (int)gridDim.x * per)
    for (int c = lane * 8; c < p.ld; c += 8 << p.log_x) {
      float v[8];
      load8<IN>(v, x + (int64_t)r * p.ld_x * El<IN>::kBytes, c, r < p.rows ? p.cols - c : 0);
      v8e h, l;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float f = v[k] * scale * scale2;
        h[k] = (S)f;
        l[k] = (S)(f - (float)h[k]);
      }
      *(v8e*)(hi + (int64_t)r * p.ld + c) = h;
      *(v8e*)(lo + (int64_t)r * p.ld + c) = l;
    }
}

// ----------------------------------------------------------------- epilogues
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
// Four columns of a row a lane -> four rows of a column, among four lanes whose rows
// follow one another: two exchanges of a 32-bit word.
__device__ __forceinline__ v4e turned(v4e in, int lane) {
  const v2u w = __builtin_bit_cast(v2u, in);
  const bool high = lane & 2, odd = lane & 1;
  // the columns 0, 1 (high: 2, 3) of the rows l & 1 and (l & 1) + 2
  const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)(high ? w[0] : w[1]), 0x4E, 0xf, 0xf, false);
  const uint32_t r0 = high ? got : w[0], r2 = high ? w[1] : got;
  const uint32_t lower = (r0 & 0xffffu) | (r2 << 16), upper = (r0 >> 16) | (r2 & 0xffff0000u);
  const uint32_t rest = (uint32_t)__builtin_amdgcn_mov_dpp((int)(odd ? lower : upper), 0xB1, 0xf, 0xf, false);
  const uint32_t mine = odd ? upper : lower;
  // rows 0 .. 3: an even lane has 0 and 2, an odd one 1 and 3
  const uint32_t a = odd ? rest : mine, b = odd ? mine : rest;
  v2u o;
  o[0] = (a & 0xffffu) | (b << 16);
  o[1] = (a >> 16) | (b & 0xffff0000u);
  return __builtin_bit_cast(v4e, o);
}

// A tile and its mirror image (A of 4096 x 4096, one part 75 us, two 213; B 80 and 223; A
// and B of 2048 x 2048 in two parts 60 each): what is stored at (r, c) is stored at (c, r)
// too, unless the tile lies on the diagonal.  `value(r, c, sums)` gives four columns' results.
template <bool WIDE>
struct Symmetric : EpiSymmetric {
  static constexpr int kBarriers = 0;
  template <int FM, int FN, int BM, int BN, int WM, int WN, class F>
  __device__ __forceinline__ void store(v4f (&acc)[FN][FM], int m0, int n0, TileAt at, int wm, int wn,
                                        int lane, F value) const {
    S* const to = (S*)out + at.part * step;
    S* const rest = WIDE ? (S*)out_lo + at.part * step : nullptr;
    const int r0 = m0 + wm * (FM * 16), c0 = n0 + wn * (FN * 16);
    const int row = lane & 15, quad = (lane >> 4) * 4;
    // (all values before the first store, which the compiler moves no load past)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int i = 0; i < FN; ++i)
        if (r0 + j * 16 < n && c0 + i * 16 < n)  // (the same for the wave; n is a multiple of 64)
          acc[i][j] = value(r0 + j * 16 + row, c0 + i * 16 + quad, acc[i][j]);
#pragma unroll
    for (int j = 0; j < FM; ++j) {
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        const int rb = r0 + j * 16, cb = c0 + i * 16;
        if (rb >= n || cb >= n) continue;
        const v4f v = acc[i][j];
        const v4e e = __builtin_convertvector(v, v4e);
        const int64_t here = (int64_t)(rb + row) * n + cb + quad;
        const int64_t there = (int64_t)(cb + quad + (lane & 3)) * n + rb + (row & 12);
        *(v4e*)(to + here) = e;
        if (at.m != at.n) *(v4e*)(to + there) = turned(e, lane);
        if constexpr (WIDE) {
          const v4e l = __builtin_convertvector(v - __builtin_convertvector(e, v4f), v4e);
          *(v4e*)(rest + here) = l;
          if (at.m != at.n) *(v4e*)(rest + there) = turned(l, lane);
        }
      }
    }
  }
};

template <bool WIDE>
struct Gram : Symmetric<WIDE> {
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4f (&acc)[FN][FM], int m0, int n0, TileAt at, int wm, int wn,
                                      int lane, char*) const {
    const float s = this->left ? this->left[at.part] : 1.f;
    const float f = s * s * (kOfA / (kOfX * kOfX));
    this->template store<FM, FN, BM, BN, WM, WN>(acc, m0, n0, at, wm, wn, lane,
                                                 [&](int, int, v4f v) { return v * f; });
  }
};

template <bool WIDE>
struct Poly : Symmetric<WIDE> {
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4f (&acc)[FN][FM], int m0, int n0, TileAt at, int wm, int wn,
                                      int lane, char*) const {
    const int n = this->n;
    const S* const g = (const S*)this->in + at.part * this->step;
    const S* const gl = WIDE ? (const S*)this->in_lo + at.part * this->step : nullptr;
    float* const d = this->diagonal + (int64_t)at.part * n;
    const float b = this->b3, c3 = this->c3 * (1.f / kOfA);
    this->template store<FM, FN, BM, BN, WM, WN>(
        acc, m0, n0, at, wm, wn, lane, [&](int r, int c, v4f v) {
          v4f a = __builtin_convertvector(*(const v4e*)(g + (int64_t)r * n + c), v4f);
          if constexpr (WIDE) a += __builtin_convertvector(*(const v4e*)(gl + (int64_t)r * n + c), v4f);
          v = b * a + c3 * v;
          const int k = r - c;
          if ((unsigned)k < 4u) {
            d[r] = (k == 0 ? v[0] : k == 1 ? v[1] : k == 2 ? v[2] : v[3]) * (1.f / kOfA);
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = q == k ? 0.f : v[q];
          }
          return v;
        });
  }
};

// X' = (a + diagonal) X + sums, as the next X or, at the last step, the result.  4096 x 4096
// of one part 125 us, 96 of them products, then 134 MB that nothing hides (one tile a CU);
// of two 304.
template <bool WIDE>
struct Update : EpiOrthUpdate {
  static constexpr int kBarriers = 0;
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4f (&acc)[FN][FM], int m0, int n0, TileAt at, int wm, int wn,
                                      int lane, char* lds) const {
    const Along<FN> along(lane);
    char* const mine = lds + (wn * WM + wm) * (FN * 1024);
    const int r0 = m0 + wm * (FM * 16) + along.row, c = n0 + wn * (FN * 16) + along.col;
    if (c >= ld) return;  // (ld: a multiple of 64, as every wave's columns)
    const float s = left ? left[at.part] : 1.f;
    const S* const hi = (const S*)x_hi + at.part * step;
    const S* const lo = (const S*)x_lo + at.part * step;
    const float* const d = diagonal + at.part * step_d;
    v4f by_col = {a1, a1, a1, a1};
    if (tall) by_col += *(const v4f*)(d + c);
    // (the next rows' X on its way while these are stored: the compiler does not move
    // loads past stores that may be to their memory)
    v4e nh[FN], nl[FN];
    float nd[FN];
    const auto fetch = [&](int j) {
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        const int r = min(r0 + j * 16 + i * along.kRows, all_m - 1);
        nh[i] = *(const v4e*)(hi + (int64_t)r * ld + c);
        nl[i] = *(const v4e*)(lo + (int64_t)r * ld + c);
        nd[i] = tall ? 0.f : d[r];
      }
    };
    fetch(0);
#pragma unroll 1
    for (int j = 0; j < FM; ++j) {
      v4f v[FN];
      v4e h[FN], l[FN];
      float dr[FN];
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        v[i] = acc[i][0];
#pragma unroll
        for (int k = 0; k + 1 < FM; ++k) acc[i][k] = acc[i][k + 1];
        h[i] = nh[i];
        l[i] = nl[i];
        dr[i] = nd[i];
      }
      if (j + 1 < FM) fetch(j + 1);
      exchange<FN>(v, mine, lane);
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        const int r = r0 + j * 16 + i * along.kRows;
        if (r >= all_m) continue;
        const int64_t here = (int64_t)r * ld + c;
        const v4f x = __builtin_convertvector(h[i], v4f) + __builtin_convertvector(l[i], v4f);
        const v4f f = by_col + dr[i];
        const v4f y = (x * f + v[i] * (1.f / kOfA)) * s;
        if (!out) {
          const v4e top = __builtin_convertvector(y, v4e);
          *(v4e*)((S*)to_hi + at.part * step + here) = top;
          *(v4e*)((S*)to_lo + at.part * step + here) =
              __builtin_convertvector(y - __builtin_convertvector(top, v4f), v4e);
        } else if (r < m && c < n) {
          finish(at.part, r, c, y * (scale / kOfX), n - c);
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
    if (!WIDE || out_dtype == LSAMP_DTYPE_BF16)
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
    case kTile256: LSAMP_TILE(512, 256, 256, 2, 4, 0, 1, false); break;
    case kTile128: LSAMP_TILE(256, 128, 128, 2, 2, 2, 1, false); break;
    case kTile64: LSAMP_TILE(256, 64, 64, 2, 2, 2, 1, false); break;
    case kTile128x2: LSAMP_TILE(512, 128, 128, 2, 2, 2, 2, false); break;
    case kTile64x4: LSAMP_TILE(1024, 64, 64, 2, 2, 3, 4, false); break;
    case kTile32x8:
      if constexpr (!AK && !BK) {
        LSAMP_TILE(512, 32, 32, 1, 1, 3, 8, false);
        break;
      }
      return (int)hipErrorInvalidValue;
    case kTile192:
      if constexpr (std::is_base_of_v<EpiSymmetric, E>) {
        LSAMP_TILE(512, 192, 192, 2, 4, 0, 1, false);
        break;
      }
      return (int)hipErrorInvalidValue;
    default: return (int)hipErrorInvalidValue;
  }
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace gemm

using namespace gemm;

int launch_orth_start(const OrthStart& p, int batch, int in_dtype, void* stream) {
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
template <bool WIDE>
int OrthOps<WIDE>::gram(bool tall, GemmTile t, const BatchPlan& g, const EpiSymmetric& p, void* st) {
  const Gram<WIDE> e = with<Gram<WIDE>>(p);
  return tall ? launch<true, true>(t, g, e, st) : launch<false, false>(t, g, e, st);
}
template <bool WIDE>
int OrthOps<WIDE>::poly(GemmTile t, const BatchPlan& g, const EpiSymmetric& p, void* st) {
  return launch<false, false>(t, g, with<Poly<WIDE>>(p), st);
}
template <bool WIDE>
int OrthOps<WIDE>::update(bool tall, GemmTile t, const BatchPlan& g, const EpiOrthUpdate& p,
                          void* st) {
  const Update<WIDE> e = with<Update<WIDE>>(p);
  return tall ? launch<false, false>(t, g, e, st) : launch<false, true>(t, g, e, st);
}
template struct OrthOps<false>;
template struct OrthOps<true>;

}  // namespace lsamp
