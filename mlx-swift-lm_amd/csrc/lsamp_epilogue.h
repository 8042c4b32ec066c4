// lsamp_epilogue.h — what the products' epilogues share, for elements of type
// LSAMP_DT: accesses of four columns, the activations and their slopes, the change
// of lanes before a store, and the epilogue of a linear block.
#ifndef LSAMP_EPILOGUE_H
#define LSAMP_EPILOGUE_H

#include <hip/hip_runtime.h>

#include "lsamp_gemm.h"
#include "lsamp_head.h"

namespace lsamp {
namespace gemm {
namespace {

constexpr int DT = LSAMP_DT;
using S = El<DT>::S;
typedef S v4e __attribute__((ext_vector_type(4)));

// Four columns of a row, `valid` of them in it: one access of any alignment, or
// by elements at a row's end.
template <typename V, typename E>
struct __attribute__((packed, aligned(sizeof(E)))) Any {
  V v;
};
__device__ __forceinline__ v4f load4(const void* base, int64_t i, int valid) {
  const S* p = (const S*)base + i;
  v4f v = {0.f, 0.f, 0.f, 0.f};
  if (valid >= 4) {
    const v4e e = ((const Any<v4e, S>*)p)->v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = (float)e[k];
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < valid) v[k] = (float)p[k];
  }
  return v;
}
// STREAM: past the caches (an output that is larger than they are).
template <bool STREAM = false>
__device__ __forceinline__ void store4e(void* base, int64_t i, v4e v, int valid) {
  typedef S v4u __attribute__((ext_vector_type(4), aligned(sizeof(S))));
  S* p = (S*)base + i;
  if (valid >= 4) {
    if constexpr (STREAM)
      __builtin_nontemporal_store(v, (v4u*)p);
    else
      *(v4u*)p = v;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < valid) p[k] = v[k];
  }
}
__device__ __forceinline__ void store4(void* base, int64_t i, v4f v, int valid) {
  store4e(base, i, __builtin_convertvector(v, v4e), valid);
}
__device__ __forceinline__ v4f load4f(const float* p, int valid) {
  if (valid >= 4) return ((const Any<v4f, float>*)p)->v;
  v4f v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < valid) v[k] = p[k];
  return v;
}
template <bool STREAM = false>
__device__ __forceinline__ void store4f(float* p, v4f v, int valid) {
  typedef float v4u __attribute__((ext_vector_type(4), aligned(4)));
  if (valid >= 4) {
    if constexpr (STREAM)
      __builtin_nontemporal_store(v, (v4u*)p);
    else
      *(v4u*)p = v;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < valid) p[k] = v[k];
  }
}

// exp(x).  For 16-bit elements exp2(x log2 e), relatively off by |x| 2^-24 from
// the product's rounding; for float32 that rounding is put back.
__device__ __forceinline__ float expe(float x) {
  if constexpr (DT == LSAMP_DTYPE_F32) {
    constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
    x = x < -150.f ? -150.f : x;  // (0 either way; -inf has no remainder)
    const float t = x * kLog2e;
    const float e = __builtin_amdgcn_exp2f(t);
    return x > 88.f ? __expf(x) : fmaf(e, fmaf(x, kLog2e, -t) * kLn2, e);
  } else {
    return __expf(x);
  }
}

// 1 / (1 + exp(-z)) and tanh.  For 16-bit elements with the hardware's
// reciprocal (1 ulp) in place of a division of some ten instructions, and tanh
// as (1 - e) / (1 + e) with e = exp(-2 |x|), a polynomial below 0.3 where that
// cancels: off by less than 8 2^-24, far below the result's own rounding.
__device__ __forceinline__ float reciprocal(float v) {
  if constexpr (DT == LSAMP_DTYPE_F32)
    return 1.f / v;
  else
    return __builtin_amdgcn_rcpf(v);
}
__device__ __forceinline__ float sigmoid(float z) { return reciprocal(1.f + expe(-z)); }
// tanh(x) from e = exp(-2 |x|) and r = 1 / (1 + e).
__device__ __forceinline__ float tanh_of(float x, float e, float r) {
  if constexpr (DT == LSAMP_DTYPE_F32) {
    return tanhf(x);
  } else {
    const float a = fabsf(x), q = x * x;
    const float p = fmaf(q, fmaf(q, fmaf(q, 62.f / 2835, -17.f / 315), 2.f / 15), -1.f / 3);
    return copysignf(a < 0.3f ? fmaf(a * q, p, a) : (1.f - e) * r, x);
  }
}
// cap tanh(z / cap), given 1 / cap (see inverse_cap), and its slope 4 e / (1 + e)^2,
// of which nothing cancels on either side.  Both are relatively right: a cap far
// above the logits takes nothing from them.
__device__ __forceinline__ float soft_cap(float z, float cap, float inverse, float* slope) {
  const float t = z * inverse;
  const float e = expe(-2.f * fabsf(t)), r = reciprocal(1.f + e);
  if (slope) *slope = 4.f * e * r * r;
  return cap * tanh_of(t, e, r);
}
// (finite, so that a logit of 0 stays 0 under the smallest caps)
__device__ __forceinline__ float inverse_cap(float cap) { return fminf(1.f / cap, 3.4e38f); }

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kGeluA = 0.79788456080286536f;  // sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

#define LSAMP_EACH(expr)                                 \
  do {                                                   \
    _Pragma("unroll") for (int k = 0; k < 4; ++k) {      \
      const float z = v[k];                              \
      v[k] = (expr);                                     \
    }                                                    \
    return v;                                            \
  } while (0)

// (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)): nothing cancels, and no tanh.  Past 1e4
// it is 0 or 1 all the same, and the cube finite.
__device__ __forceinline__ float clamped(float z) { return fminf(fmaxf(z, -1e4f), 1e4f); }
__device__ __forceinline__ float gelu_gate(float z) {
  const float c = clamped(z);
  return sigmoid(2.f * kGeluA * (c + kGeluB * c * c * c));
}
__device__ __forceinline__ float gelu_tanh(float z) {
  return z * gelu_gate(z);
}
// act(z) and act'(z) of four columns (one branch for them: it costs as much as
// the arithmetic of one).
__device__ __forceinline__ v4f activate(int act, float cap, v4f v) {
  switch (act) {
    case LSAMP_ACT_RELU: LSAMP_EACH(z < 0.f ? 0.f : z);  // (a NaN stays)
    case LSAMP_ACT_SILU: LSAMP_EACH(z * sigmoid(z));
    case LSAMP_ACT_GELU: LSAMP_EACH(0.5f * z * (1.f + erff(z * kSqrtHalf)));
    case LSAMP_ACT_GELU_TANH: LSAMP_EACH(gelu_tanh(z));
    case LSAMP_ACT_SOFTCAP: {
      const float inverse = inverse_cap(cap);
      LSAMP_EACH(soft_cap(z, cap, inverse, nullptr));
    }
    default: return v;
  }
}
__device__ __forceinline__ float silu_slope(float z) {
  const float s = sigmoid(z);
  return s * (1.f + z * (1.f - s));
}
__device__ __forceinline__ float gelu_tanh_slope(float z) {
  const float s = gelu_gate(z), c = clamped(z);
  return s + 2.f * kGeluA * z * (s * (1.f - s)) * (1.f + 3.f * kGeluB * c * c);
}
__device__ __forceinline__ float cap_slope(float z, float cap, float inverse) {
  float slope;
  soft_cap(z, cap, inverse, &slope);
  return slope;
}
__device__ __forceinline__ v4f activate_slope(int act, float cap, v4f v) {
  switch (act) {
    case LSAMP_ACT_RELU: LSAMP_EACH(z > 0.f ? 1.f : 0.f);
    case LSAMP_ACT_SILU: LSAMP_EACH(silu_slope(z));
    case LSAMP_ACT_GELU:
      LSAMP_EACH(0.5f * (1.f + erff(z * kSqrtHalf)) + z * kInvSqrt2Pi * expe(-0.5f * z * z));
    case LSAMP_ACT_GELU_TANH: LSAMP_EACH(gelu_tanh_slope(z));
    case LSAMP_ACT_SOFTCAP: {
      const float inverse = inverse_cap(cap);
      LSAMP_EACH(cap_slope(z, cap, inverse));
    }
    default: return v4f{1.f, 1.f, 1.f, 1.f};
  }
}

// ------------------------------------------------------------------ epilogues
// A wave's sums lie with 16 lanes down a column of rows; stored like that, an
// instruction writes 16 rows of 32 bytes, and rows a power of two apart meet in
// the same few channels (4096 x 4096 x 16384: 490 us, 371 without its stores).
// So the quads of columns of 16 rows change lanes through LDS, a KB a quad of
// columns and wave: 4 FN lanes then lie along a row, 16 / FN rows a quad.  (Float32
// parts, whose quads are 64 bytes of a row, gain nothing by it.)
template <int FN>
struct Along {
  static constexpr int kLanes = 4 * FN, kRows = 16 / FN;
  int row, col;  // of the 16 rows, of the wave's columns
  __device__ __forceinline__ explicit Along(int lane) : row(lane / kLanes), col(lane % kLanes * 4) {}
};
template <int FN, class V>
__device__ __forceinline__ void exchange(V (&v)[FN], char* lds, int lane) {
  constexpr int kLanes = 4 * FN;
  V* const rows = (V*)lds;
  // (permuted within the row: 16 rows' writes fall on different banks)
  const auto place = [](int r, int q) { return r * kLanes + (q ^ (r / (4 / FN))); };
#pragma unroll
  for (int i = 0; i < FN; ++i) rows[place(lane & 15, i * 4 + (lane >> 4))] = v[i];
  __builtin_amdgcn_wave_barrier();  // (other lanes' quads: a wave's LDS accesses stay in order)
#pragma unroll
  for (int i = 0; i < FN; ++i) v[i] = rows[place(i * (16 / FN) + lane / kLanes, lane % kLanes)];
  __builtin_amdgcn_wave_barrier();
}

struct Linear : EpiLinear {
  static constexpr int kBarriers = 0;
  __device__ __forceinline__ v4f bias_at(int c) const {
    return bias ? load4(bias, c, n - c) : v4f{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ v4f residual_at(int r, int c) const {
    return residual && r < m ? load4(residual, (int64_t)r * ld_residual + c, n - c)
                             : v4f{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void finish(int r, int c, v4f v, v4f b, v4f res) const {
    const int valid = n - c;
    v += b;
    if (pre) {
      float* p = pre + (int64_t)r * ld_pre + c;
      if (stream)
        store4f<true>(p, v, valid);
      else
        store4f(p, v, valid);
    }
    v = activate(activation, softcap, v);
    if (residual) v += res;
    if (wide) {
      store4f((float*)out + (int64_t)r * ld_out + c, v, valid);
    } else {
      const v4e e = __builtin_convertvector(v, v4e);
      if (stream)
        store4e<true>(out, (int64_t)r * ld_out + c, e, valid);
      else
        store4e(out, (int64_t)r * ld_out + c, e, valid);
    }
  }
  __device__ __forceinline__ void put(int r, int c, v4f v, int) const {
    finish(r, c, v, bias_at(c), residual_at(r, c));
  }
  // The next rows' residual is on its way while these are stored (which may be
  // the residual's own memory, so the compiler keeps the order as written).  One
  // copy of the code for all rows, the sums moved down to it: unrolled, the
  // activations are 150 KB of instructions that no cache holds (silu over 8192 x
  // 4096 x 4096 took 40 us).
  template <int FM, int FN, int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void run(v4f (&acc)[FN][FM], int m0, int n0, TileAt, int wm, int wn,
                                      int lane, char* lds) const {
    const Along<FN> at(lane);
    char* const mine = lds + (wn * WM + wm) * (FN * 1024);
    const int r0 = m0 + wm * (FM * 16) + at.row, c = n0 + wn * (FN * 16) + at.col;
    const v4f b = bias_at(c);
    v4f res[FN], next[FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) next[i] = residual_at(r0 + i * at.kRows, c);
#pragma unroll 1
    for (int j = 0; j < FM; ++j) {
      const int r = r0 + j * 16;
      v4f v[FN];
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        v[i] = acc[i][0];
#pragma unroll
        for (int k = 0; k + 1 < FM; ++k) acc[i][k] = acc[i][k + 1];
        res[i] = next[i];
        next[i] = residual_at(j + 1 < FM ? r + 16 + i * at.kRows : m, c);
      }
      exchange<FN>(v, mine, lane);
#pragma unroll
      for (int i = 0; i < FN; ++i)
        if (r + i * at.kRows < m && c < n) finish(r + i * at.kRows, c, v[i], b, res[i]);
    }
  }
};

}  // namespace
}  // namespace gemm
}  // namespace lsamp

#endif
