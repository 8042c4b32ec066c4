// lsamp_head.hip — the hidden-state operators: linear blocks, the vocabulary
// head's cross entropy, and their gradients.  Compiled once per element type
// (LSAMP_DT).  The matrix products are lsamp_gemm.h; this file holds what
// happens to their sums, and the passes between them.
#include <hip/hip_runtime.h>

#include "lsamp_epilogue.h"
#include "lsamp_gemm.h"
#include "lsamp_head.h"
#include "lsamp_skinny.h"

namespace lsamp {
namespace gemm {
namespace {

struct Store : EpiStore {
  static constexpr int kBarriers = 0;
  __device__ __forceinline__ void put(int r, int c, v4f v, int) const {
    if (scale) v *= *scale;
    store4(out, (int64_t)r * ld_out + c, v, n - c);
  }
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4f (&acc)[FN][FM], int m0, int n0, TileAt, int wm, int wn,
                                      int lane, char* lds) const {
    // (once: the stores may be to its memory for all the compiler knows)
    const float s = scale ? *scale : 1.f;
    const Along<FN> at(lane);
    char* const mine = lds + (wn * WM + wm) * (FN * 1024);
    const int r0 = m0 + wm * (FM * 16) + at.row, c = n0 + wn * (FN * 16) + at.col;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      v4e v[FN];
#pragma unroll
      for (int i = 0; i < FN; ++i) v[i] = __builtin_convertvector(acc[i][j] * s, v4e);
      exchange<FN>(v, mine, lane);
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        const int r = r0 + j * 16 + i * at.kRows;
        if (r < m && c < n) {
          if (stream)
            store4e<true>(out, (int64_t)r * ld_out + c, v[i], n - c);
          else
            store4e(out, (int64_t)r * ld_out + c, v[i], n - c);
        }
      }
    }
  }
};

struct Partial : EpiPartial {
  static constexpr int kBarriers = 0;
  __device__ __forceinline__ v4f* at(int r, int c, int part) const {
    return (v4f*)(out + part * part_stride + (int64_t)r * ld + c);
  }
  __device__ __forceinline__ void put(int r, int c, v4f v, int part) const {
    v4f* p = at(r, c, part);
    if (accumulate) v += *p;
    *p = v;
  }
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4f (&acc)[FN][FM], int m0, int n0, TileAt tile, int wm, int wn,
                                      int lane, char* lds) const {
    const int r0 = m0 + wm * (FM * 16) + (lane & 15);
    const int c0 = n0 + wn * (FN * 16) + (lane >> 4) * 4;
    if (accumulate) {  // all reads before the first store
#pragma unroll
      for (int j = 0; j < FM; ++j)
#pragma unroll
        for (int i = 0; i < FN; ++i)
          if (r0 + j * 16 < m && c0 + i * 16 < n) acc[i][j] += *at(r0 + j * 16, c0 + i * 16, tile.part);
    }
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int i = 0; i < FN; ++i)
        if (r0 + j * 16 < m && c0 + i * 16 < n) *at(r0 + j * 16, c0 + i * 16, tile.part) = acc[i][j];
  }
};

// z = softcap(sum + bias) of four columns, and the slope of the cap.
__device__ __forceinline__ v4f logits4(v4f v, v4f b, float softcap, float inverse, v4f* slope) {
  v += b;
  if (softcap > 0.f) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float s;
      v[k] = soft_cap(v[k], softcap, inverse, &s);
      if (slope) (*slope)[k] = s;
    }
  }
  return v;
}
__device__ __forceinline__ v4f head_bias(const void* bias, int col, int valid) {
  return bias ? load4(bias, col, valid) : v4f{0.f, 0.f, 0.f, 0.f};
}

// The forward pass keeps, of a tile's logits, each row's maximum and the sum of
// exp(z - maximum): 4 columns x FN fragments in a lane, the four lanes of a row,
// then the waves of the row through LDS.  A row whose logits here are all -inf
// has maximum -inf and sum 0.  8 bytes leave a tile's row in place of its logits;
// ten instructions an element remain: 4096 x 4096 x 16384 389 us, its product
// without an epilogue 370.
struct Stats : EpiStats {
  static constexpr int kBarriers = 1;
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4f (&acc)[FN][FM], int m0, int n0, TileAt at, int wm, int wn,
                                      int lane, char* lds) const {
    float* red = (float*)lds;  // [WN][BM][2]
    const float inverse = softcap > 0.f ? inverse_cap(softcap) : 0.f;
    v4f b[FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      const int c = n0 + wn * (FN * 16) + i * 16 + (lane >> 4) * 4;
      b[i] = head_bias(bias, first_col + c, n - c);
    }
    const bool inside = n0 + BN <= n;  // (every column of the tile exists)
    int t[FM];
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int r = m0 + wm * (FM * 16) + j * 16 + (lane & 15);
      t[j] = r < m ? targets[r] - first_col : -1;
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int rl = wm * (FM * 16) + j * 16 + (lane & 15);
      const int r = m0 + rl;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        const int c = n0 + wn * (FN * 16) + i * 16 + (lane >> 4) * 4;
        v4f v = logits4(acc[i][j], b[i], softcap, inverse, nullptr);
        if (!inside) {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = c + k < n ? v[k] : -INFINITY;
        }
        if ((unsigned)(t[j] - c) < 4u && t[j] < n) {
          const int k = t[j] - c;
          target[r] = k == 0 ? v[0] : k == 1 ? v[1] : k == 2 ? v[2] : v[3];
        }
        top = fmaxf(fmaxf(fmaxf(top, v[0]), fmaxf(v[1], v[2])), v[3]);
        acc[i][j] = v;
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      float sum = 0.f;
      // (NaN logits are no maximum; they make the sum NaN)
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) sum += expe(acc[i][j][k] - base);
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (lane < 16) {
        red[(wn * BM + rl) * 2] = top;
        red[(wn * BM + rl) * 2 + 1] = sum;
      }
    }
    __syncthreads();
    for (int rl = threadIdx.x; rl < BM; rl += WM * WN * kWave) {
      if (m0 + rl >= m) break;
      float top = -INFINITY, sum = 0.f;
      for (int w = 0; w < WN; ++w) top = fmaxf(top, red[(w * BM + rl) * 2]);
      const float base = top == -INFINITY ? 0.f : top;
      for (int w = 0; w < WN; ++w) {
        const float t = red[(w * BM + rl) * 2], s = red[(w * BM + rl) * 2 + 1];
        sum += t == -INFINITY ? s : s * expe(t - base);  // (a NaN sum stays)
      }
      float* o = part + ((int64_t)(m0 + rl) * blocks + first_block + at.n) * 2;
      o[0] = top;
      o[1] = sum;
    }
  }
};

// The gradient at the logits, d_loss[r] (softmax(z) - onehot(target)), from the
// recomputed logits and the forward pass's log-sum-exp.  Rounded to the
// operands' type because the two products that read it are matrix instructions
// of that type, and scaled first (k_grad_scale).  A row without
// a loss (target ignored or out of range, every logit -inf) is zero.  The columns'
// sums for d_bias are taken here, in float32 and before the rounding: a wave's rows
// in registers, joined later in a fixed order.  4096 x 4096 x 151936 in ten pieces:
// 4.16 ms (1.22 PFLOP/s), the plain product 3.84.
struct Grad : EpiGrad {
  static constexpr int kBarriers = 0;
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4f (&acc)[FN][FM], int m0, int n0, TileAt, int wm, int wn,
                                      int lane, char* lds) const {
    const Along<FN> along(lane);
    char* const mine = lds + (wn * WM + wm) * (FN * 1024);
    const int out_col = n0 + wn * (FN * 16) + along.col;
    const float s = scale[0];
    const float inverse = softcap > 0.f ? inverse_cap(softcap) : 0.f;
    const int r0 = m0 + wm * (FM * 16) + (lane & 15);
    const int c0 = n0 + wn * (FN * 16) + (lane >> 4) * 4;
    v4f b[FN];
    int target[FM];
    float l[FM], w[FM];
#pragma unroll
    for (int i = 0; i < FN; ++i) b[i] = head_bias(bias, first_col + c0 + i * 16, n - c0 - i * 16);
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int r = min(r0 + j * 16, m - 1);
      target[j] = targets[r];
      l[j] = lse[r];
      w[j] = d_loss[r] * s;
    }
    v4f sum[FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) sum[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const bool none = target[j] < 0 || target[j] >= vocab || l[j] == -INFINITY || r0 + j * 16 >= m;
      v4e q[FN];
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        const int c = c0 + i * 16;
        v4f slope = {1.f, 1.f, 1.f, 1.f}, g;
        const int valid = n - c;
        const v4f z = logits4(acc[i][j], b[i], softcap, inverse, &slope);
#pragma unroll
        for (int k = 0; k < 4; ++k) g[k] = expe(z[k] - l[j]);
        const int at = target[j] - first_col - c;
        if ((unsigned)at < 4u) {
#pragma unroll
          for (int k = 0; k < 4; ++k) g[k] -= k == at ? 1.f : 0.f;
        }
        g *= w[j];
        if (softcap > 0.f) g *= slope;
        if (none || valid < 4) {
#pragma unroll
          for (int k = 0; k < 4; ++k) g[k] = none || k >= valid ? 0.f : g[k];
        }
        sum[i] += g;
        q[i] = __builtin_convertvector(g, v4e);
      }
      exchange<FN>(q, mine, lane);
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        const int r = m0 + wm * (FM * 16) + j * 16 + i * along.kRows + along.row;
        if (r < m && out_col < n_pad) store4e(out, (int64_t)r * ld_out + out_col, q[i], 4);
      }
    }
    if (sums) {
      float* const to = sums + (int64_t)(m0 / BM * WM + wm) * ld_sums;
#pragma unroll
      for (int i = 0; i < FN; ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int d = 1; d < 16; d *= 2) sum[i][k] += __shfl_xor(sum[i][k], d);
        // (columns n .. are zero, and lie within the row)
        if ((lane & 15) == 0 && c0 + i * 16 < n) *(v4f*)(to + c0 + i * 16) = sum[i];
      }
    }
  }
};

template <class E, class P>
E with(const P& plan) {
  E e;
  static_cast<P&>(e) = plan;
  return e;
}

#define LSAMP_TILE(THREADS, ...)                                                               \
  hipLaunchKernelGGL((k_gemm<DT, AK, BK, __VA_ARGS__, E>), grid, dim3(THREADS), 0, st, g, e)

// LOOSE: the 64 x 64 shapes that take any rows too.  Float32 tiles go up to 128 x
// 128: a wave's split fragments need the registers.
template <bool AK, bool BK, bool LOOSE, class E>
int launch(GemmTile tile, const GemmPlan& g, const E& e, void* stream) {
  const dim3 grid((unsigned)(g.tiles_m * g.tiles_n * g.parts));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (tile) {
    case kTile256:
      if constexpr (DT != LSAMP_DTYPE_F32) {
        LSAMP_TILE(512, 256, 256, 2, 4, 0, 1, false);
        break;
      }
      return (int)hipErrorInvalidValue;
    case kTile128:
      LSAMP_TILE(256, 128, 128, 2, 2, 2, 1, false);
      break;
    case kTile64:
      LSAMP_TILE(256, 64, 64, 2, 2, 2, 1, false);
      break;
    case kTile128x2:
      LSAMP_TILE(512, 128, 128, 2, 2, 2, 2, false);
      break;
    case kLoose64:
      if constexpr (LOOSE) {
        LSAMP_TILE(256, 64, 64, 2, 2, 2, 1, true);
        break;
      }
      return (int)hipErrorInvalidValue;
    case kLoose128:
      LSAMP_TILE(256, 128, 128, 2, 2, 2, 1, true);
      break;
    case kLoose64x4:
      if constexpr (LOOSE) {
        LSAMP_TILE(1024, 64, 64, 2, 2, 2, 4, true);
        break;
      }
      return (int)hipErrorInvalidValue;
    case kTile64x4:
      LSAMP_TILE(1024, 64, 64, 2, 2, 2, 4, false);
      break;
    default:
      return (int)hipErrorInvalidValue;
  }
  return (int)hipGetLastError();
}

template <int NF, int WK, bool ROWWISE, class E>
int launch_skinny(const GemmPlan& g, const E& e, void* stream) {
  const dim3 grid((unsigned)g.tiles_n), threads(WK * kWave);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (g.a.rows <= 16)
    hipLaunchKernelGGL((k_skinny<DT, 1, NF, WK, ROWWISE, E>), grid, threads, 0, st, g, e);
  else if (g.a.rows <= 32)
    hipLaunchKernelGGL((k_skinny<DT, 2, NF, WK, ROWWISE, E>), grid, threads, 0, st, g, e);
  else
    hipLaunchKernelGGL((k_skinny<DT, 4, NF, WK, ROWWISE, E>), grid, threads, 0, st, g, e);
  return (int)hipGetLastError();
}

// ------------------------------------------------------------- passes between
constexpr int kThreads = 256;

// The parts of a split reduction, summed, and the epilogue: 64 quads of columns a
// work-group, each wave a quarter of the parts, always in the same order.  Bound by
// memory: 4096 x 4096 float32 sums to bfloat16 41 us (2.5 TB/s), small ones 4 us.
template <class E>
__global__ __launch_bounds__(kThreads) void k_join(EpiPartial from, int parts, E e) {
  __shared__ v4f red[3][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int quads = (e.n + 3) / 4;
  const int64_t total = (int64_t)e.m * quads;
  for (int64_t first = (int64_t)blockIdx.x * 64; first < total; first += (int64_t)gridDim.x * 64) {
    const int64_t i = first + lane;
    const int r = (int)(i / quads), c = (int)(i % quads) * 4;
    v4f v = {0.f, 0.f, 0.f, 0.f};
    if (i < total) {
      const float* p = from.out + (int64_t)r * from.ld + c;
#pragma unroll 8
      for (int k = wave; k < parts; k += 4) v += *(const v4f*)(p + k * from.part_stride);
    }
    if (wave > 0) red[wave - 1][lane] = v;
    __syncthreads();
    if (wave == 0 && i < total) {
      for (int k = 0; k < 3; ++k) v += red[k][lane];
      e.put(r, c, v, 0);
    }
    __syncthreads();
  }
}
template <class E, class P>
int launch_join(const EpiPartial& from, int parts, const P& plan, void* stream) {
  const E e = with<E>(plan);
  const int64_t quads = (int64_t)e.m * ((e.n + 3) / 4);
  int64_t blocks = (quads + 63) / 64;
  blocks = blocks < 8192 ? blocks : 8192;
  hipLaunchKernelGGL((k_join<E>), dim3((unsigned)blocks), dim3(kThreads), 0,
                     reinterpret_cast<hipStream_t>(stream), from, parts, e);
  return (int)hipGetLastError();
}

// Column sums of a chunk of rows: 64 lanes x 4 columns, 4 waves taking rows in
// turn and joined in LDS.  With `pre`: of in * activation'(pre), which is also
// written out for the products that follow, so that both read it once rounded and
// the activation is evaluated once.  Bound by memory: 8192 x 4096 bf16 with silu
// and float32 pre 51 us (268 MB, 5.2 TB/s).
__global__ __launch_bounds__(kThreads) void k_col_sum(ColSumPlan p) {
  __shared__ v4f red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = ((int)blockIdx.x * 64 + lane) * 4;
  const int valid = p.cols - c;
  const int r0 = (int)blockIdx.y * p.rows_per_chunk;
  const int r1 = min(p.rows, r0 + p.rows_per_chunk);
  v4f sum = {0.f, 0.f, 0.f, 0.f};
  if (c < p.cols || (p.out && c < p.out_cols)) {
    for (int r = r0 + wave; r < r1; r += 4) {
      v4f v = load4(p.in, (int64_t)r * p.ld_in + c, valid);
      if (p.pre) {
        const v4f z = load4f(p.pre + (int64_t)r * p.ld_pre + c, valid);
        const v4f slope = activate_slope(p.activation, p.softcap, z);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = k < valid ? v[k] * slope[k] : 0.f;
        store4(p.out, (int64_t)r * p.ld_out + c, v, p.out_cols - c);
      }
      sum += v;
    }
  }
  if (!p.part && !p.sums) return;
  red[wave][lane] = sum;
  __syncthreads();
  if (wave != 0) return;
  for (int w = 1; w < 4; ++w) sum += red[w][lane];
  if (p.sums) {  // (the only chunk)
    if (c < p.cols) store4(p.sums, c, sum, valid);
  } else if (c < p.ld_part) {
    *(v4f*)(p.part + (int64_t)blockIdx.y * p.ld_part + c) = sum;
  }
}
// 64 columns a work-group, its waves taking chunks in turn: four, or sixteen for the
// sums of many rows of tiles over few columns (the bias of 262,144 rows x 256 x 4000,
// trained: 1.47 of 7.1 ms with four, 0.55 of 6.0 with sixteen; up to 256 rows of sums
// either takes a launch).
template <int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void k_col_sum_join(ColSumPlan p, S* out,
                                                               const float* scale) {
  __shared__ float red[WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (int)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < p.cols) {
#pragma unroll 8
    for (int i = wave; i < p.chunks; i += WAVES) s += p.part[(int64_t)i * p.ld_part + c];
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= p.cols) return;
  s = red[0][lane];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) s += red[w][lane];
  out[c] = (S)(scale ? s * *scale : s);
}

}  // namespace
}  // namespace gemm

using namespace gemm;

template <>
int HeadOps<DT>::gemm_linear(GemmTile t, const GemmPlan& g, const EpiLinear& p, void* st) {
  const Linear e = with<Linear>(p);
  if (t == kSkinny64) return launch_skinny<4, 4, true>(g, e, st);
  if (t == kSkinny16) return launch_skinny<1, 8, true>(g, e, st);
  return launch<false, false, true>(t, g, e, st);
}
template <>
int HeadOps<DT>::gemm_stats(GemmTile t, const GemmPlan& g, const EpiStats& p, void* st) {
  const Stats e = with<Stats>(p);
  if (t == kSkinny64) return launch_skinny<4, 4, false>(g, e, st);
  return launch<false, false, false>(t, g, e, st);
}
template <>
int HeadOps<DT>::gemm_grad(GemmTile t, const GemmPlan& g, const EpiGrad& p, void* st) {
  const Grad e = with<Grad>(p);
  if (t == kSkinny64) return launch_skinny<4, 4, false>(g, e, st);
  return launch<false, false, false>(t, g, e, st);
}
template <>
int HeadOps<DT>::gemm_store(GemmRoles roles, GemmTile t, const GemmPlan& g, const EpiStore& p,
                            void* st) {
  const Store e = with<Store>(p);
  return roles == kRolesNN ? launch<false, true, true>(t, g, e, st)
                           : launch<true, true, true>(t, g, e, st);
}
template <>
int HeadOps<DT>::gemm_partial(GemmRoles roles, GemmTile t, const GemmPlan& g, const EpiPartial& p,
                              void* st) {
  const Partial e = with<Partial>(p);
  switch (roles) {
    case kRolesNT: return launch<false, false, true>(t, g, e, st);
    case kRolesNN: return launch<false, true, true>(t, g, e, st);
    default: return launch<true, true, true>(t, g, e, st);
  }
}
template <>
int HeadOps<DT>::join_linear(const EpiPartial& from, int parts, const EpiLinear& e, void* st) {
  return launch_join<Linear>(from, parts, e, st);
}
template <>
int HeadOps<DT>::join_store(const EpiPartial& from, int parts, const EpiStore& e, void* st) {
  return launch_join<Store>(from, parts, e, st);
}
template <>
int HeadOps<DT>::col_sum(const ColSumPlan& p, void* stream) {
  const int cols = p.out && p.out_cols > p.cols ? p.out_cols : p.cols;
  const dim3 grid((unsigned)((cols + 255) / 256), (unsigned)p.chunks);
  hipLaunchKernelGGL(k_col_sum, grid, dim3(kThreads), 0, reinterpret_cast<hipStream_t>(stream), p);
  return (int)hipGetLastError();
}
template <>
int HeadOps<DT>::col_sum_join(const ColSumPlan& p, void* out, const float* scale, void* stream) {
  const dim3 grid((unsigned)((p.cols + 63) / 64));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (p.join_wide)
    hipLaunchKernelGGL(k_col_sum_join<16>, grid, dim3(16 * kWave), 0, st, p, (S*)out, scale);
  else
    hipLaunchKernelGGL(k_col_sum_join<4>, grid, dim3(4 * kWave), 0, st, p, (S*)out, scale);
  return (int)hipGetLastError();
}

}  // namespace lsamp
