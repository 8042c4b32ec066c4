// lsamp_int8.hip — products of 8-bit integers whose rows have scales:
//
//   out[m][n] = act(xs[m] ws[n] sum_k x[m][k] w[n][k] + bias[n]) + residual[m][n]
//
// Compiled once per element type of bias, residual and out (LSAMP_DT).  The sums
// are whole numbers of 32 bits (127^2 k, exact for the lengths that the entry
// point takes); one becomes float32 with a rounding of 2^-24, and its two scales
// are multiplied first, another.  The tiles are lsamp_gemm.h's and lsamp_skinny.h's:
// a slab of 128 bytes is 128 steps, an instruction takes 64 steps of a 16 x 16 tile in
// the time that it takes 32 of 16-bit elements, so a product moves half the bytes
// and takes half the time of a 16-bit one on either side of the roofline.
#include <hip/hip_runtime.h>

#include "lsamp_epilogue.h"
#include "lsamp_gemm.h"
#include "lsamp_head.h"
#include "lsamp_skinny.h"

namespace lsamp {
namespace gemm {
namespace {

struct LinearInt8 : Linear {
  const float* x_scale;
  const float* w_scale;
  __device__ __forceinline__ v4f w_at(int c) const { return load4f(w_scale + c, n - c); }
  __device__ __forceinline__ v4f scaled(v4i v, float xs, v4f ws) const {
    return __builtin_convertvector(v, v4f) * (ws * xs);
  }
  __device__ __forceinline__ void put(int r, int c, v4i v, int) const {
    finish(r, c, scaled(v, x_scale[r], w_at(c)), bias_at(c), residual_at(r, c));
  }
  // (Linear::run, with a row's scale on its way beside its residual)
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4i (&acc)[FN][FM], int m0, int n0, TileAt, int wm, int wn,
                                      int lane, char* lds) const {
    const Along<FN> at(lane);
    char* const mine = lds + (wn * WM + wm) * (FN * 1024);
    const int r0 = m0 + wm * (FM * 16) + at.row, c = n0 + wn * (FN * 16) + at.col;
    const v4f b = bias_at(c), ws = c < n ? w_at(c) : v4f{0.f, 0.f, 0.f, 0.f};
    const auto x_at = [&](int r) { return r < m ? x_scale[r] : 0.f; };
    v4f res[FN], next[FN];
    float xs[FN], next_xs[FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      next[i] = residual_at(r0 + i * at.kRows, c);
      next_xs[i] = x_at(r0 + i * at.kRows);
    }
#pragma unroll 1
    for (int j = 0; j < FM; ++j) {
      const int r = r0 + j * 16;
      v4i v[FN];
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        v[i] = acc[i][0];
#pragma unroll
        for (int k = 0; k + 1 < FM; ++k) acc[i][k] = acc[i][k + 1];
        res[i] = next[i];
        xs[i] = next_xs[i];
        next[i] = residual_at(j + 1 < FM ? r + 16 + i * at.kRows : m, c);
        next_xs[i] = x_at(j + 1 < FM ? r + 16 + i * at.kRows : m);
      }
      exchange<FN>(v, mine, lane);
#pragma unroll
      for (int i = 0; i < FN; ++i)
        if (r + i * at.kRows < m && c < n)
          finish(r + i * at.kRows, c, scaled(v[i], xs[i], ws), b, res[i]);
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
    case kTile64x4: LSAMP_TILE(1024, 64, 64, 2, 2, 2, 4, false); break;
    case kLoose128: LSAMP_TILE(256, 128, 128, 2, 2, 2, 1, true); break;
    case kLoose64: LSAMP_TILE(256, 64, 64, 2, 2, 2, 1, true); break;
    case kLoose64x4: LSAMP_TILE(1024, 64, 64, 2, 2, 2, 4, true); break;
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
