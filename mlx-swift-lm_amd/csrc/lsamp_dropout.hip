// lsamp_dropout.hip — dropout from a counter-based generator.
//
//   out[r][c] = residual[r][c] + (keep(r, c) ? x[r][c] / (1 - p') : 0)
//
// keep is a function of (key, offset, r, c) alone, so no mask is stored: the
// backward pass makes the same call on the gradient.  Eight elements of a row
// share one Philox4x32-10 draw of 128 bits, 16 bits each (counter: column / 8,
// row, offset; key: key); an element is kept where its bits are at least
// cut = round(p 2^16), and p' = cut / 2^16, so the expectation is exact.  With
// 32 bits an element the ten rounds of 32-bit products would take longer than
// the memory traffic.  Bound by memory: 16384 x 8192 bf16 with a residual and back
// 242 us for both (1.34 GB, 5.5 TB/s); 64 x 2048 a launch each (4 us).
#include <hip/hip_runtime.h>

#include "lsamp_head.h"

namespace lsamp {
namespace {

constexpr int kThreads = 256;

struct Words {
  uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3,
                                        uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0;
    const uint64_t p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

template <typename E>
struct Vec8 {
  E v[8];
};
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename E>
struct __attribute__((packed, aligned(sizeof(E)))) Any16 {  // 16 bytes of any alignment
  u32x4 v;
};

template <typename E>
__device__ __forceinline__ Vec8<E> load8(const E* p, int valid) {
  Vec8<E> o;
  if (valid >= 8) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) {
      const u32x4 q = ((const Any16<E>*)p)[i].v;
      __builtin_memcpy((char*)o.v + 16 * i, &q, 16);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) o.v[k] = k < valid ? p[k] : (E)0.f;
  }
  return o;
}

// A thread takes one group of eight columns of a row; 2^log_x threads a row.
template <typename E>
__global__ __launch_bounds__(kThreads) void k_dropout(DropoutPlan p, int log_x) {
  const int groups = (p.cols + 7) / 8;
  const int per_block = kThreads >> log_x;
  const int g = (int)(blockIdx.x << log_x) + ((int)threadIdx.x & ((1 << log_x) - 1));
  if (g >= groups) return;
  const uint64_t offset = p.offset + (p.step ? *p.step : 0);
  const int valid = p.cols - g * 8;
  for (int64_t r = (int64_t)blockIdx.y * per_block + (threadIdx.x >> log_x); r < p.rows;
       r += (int64_t)gridDim.y * per_block) {
    const Vec8<E> x = load8((const E*)p.x + r * p.ld_x + g * 8, valid);
    Vec8<E> y;
    if (p.residual) y = load8((const E*)p.residual + r * p.ld_residual + g * 8, valid);
    const Words w = philox((uint32_t)g, (uint32_t)r, (uint32_t)offset, (uint32_t)(offset >> 32),
                           (uint32_t)p.key, (uint32_t)(p.key >> 32));
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t bits = (w.w[k / 2] >> (16 * (k & 1))) & 0xFFFFu;
      float v = bits >= p.cut ? (float)x.v[k] * p.scale : 0.f;
      if (p.residual) v += (float)y.v[k];
      y.v[k] = (E)v;
    }
    E* out = (E*)p.out + r * p.ld_out + g * 8;
    if (valid >= 8) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(E) / 2; ++i) {
        u32x4 q;
        __builtin_memcpy(&q, (const char*)y.v + 16 * i, 16);
        ((Any16<E>*)out)[i].v = q;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < valid) out[k] = y.v[k];
    }
  }
}

template <typename E>
int launch(const DropoutPlan& p, void* stream) {
  const int groups = (p.cols + 7) / 8;
  int log_x = 0;
  while (log_x < 8 && (1 << log_x) < groups) ++log_x;
  const int64_t gx = (groups + (1 << log_x) - 1) >> log_x;
  const int64_t rows = ((int64_t)p.rows + (kThreads >> log_x) - 1) / (kThreads >> log_x);
  const int64_t most = gx < 16384 ? 16384 / gx : 1;
  hipLaunchKernelGGL((k_dropout<E>), dim3((unsigned)gx, (unsigned)(rows < most ? rows : most)),
                     dim3(kThreads), 0, reinterpret_cast<hipStream_t>(stream), p, log_x);
  return (int)hipGetLastError();
}

}  // namespace

int launch_dropout(const DropoutPlan& p, int dtype, void* stream) {
  switch (dtype) {
    case LSAMP_DTYPE_F32: return launch<float>(p, stream);
    case LSAMP_DTYPE_BF16: return launch<__bf16>(p, stream);
    default: return launch<_Float16>(p, stream);
  }
}

}  // namespace lsamp
