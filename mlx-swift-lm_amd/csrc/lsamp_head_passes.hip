// lsamp_head_passes.hip — the small passes of the hidden-state operators that
// do not depend on the matrix instructions' element type: laying operands out
// for 16-byte loads, joining the tiles' softmax statistics, and the scale of a
// float16 gradient.
#include <hip/hip_runtime.h>

#include "lsamp_head.h"

namespace lsamp {
namespace {

constexpr int kThreads = 256;

// Rows whose start, distance or length keeps them from being read as 16-byte
// chunks are copied once to rows that can, zero-filled to whole chunks.  A
// thread writes one chunk, read by one access of any alignment; bound by memory,
// one read and one write (8192 x 4097 bf16 24 us, 5.6 TB/s).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename U>
struct __attribute__((packed, aligned(sizeof(U)))) Any16 {
  u32x4 v;
};
template <typename U>
__global__ __launch_bounds__(kThreads) void k_pack(PackPlan p) {
  constexpr int N = 16 / (int)sizeof(U);
  const int chunks = p.dst_cols / N;
  for (int r = (int)blockIdx.y; r < p.rows; r += (int)gridDim.y) {
    const U* src = (const U*)p.src + (int64_t)r * p.src_ld;
    U* dst = (U*)p.dst + (int64_t)r * p.dst_ld;
    for (int c = (int)(blockIdx.x * kThreads + threadIdx.x); c < chunks;
         c += (int)gridDim.x * kThreads) {
      u32x4 o;
      if (c * N + N <= p.cols) {
        o = ((const Any16<U>*)(src + c * N))->v;
      } else {
        U v[N];
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = c * N + k < p.cols ? src[c * N + k] : (U)0;
        __builtin_memcpy(&o, v, 16);
      }
      *(u32x4*)(dst + c * N) = o;
    }
  }
}

// One work-group per row: the tiles' (maximum, sum) pairs to the row's
// log-sum-exp, and the loss.  Latency at few rows (20 rows of 2,374 pairs: 6.6 us),
// memory at many (4,096 rows of 594 pairs: 14 us, 19 MB).
__global__ __launch_bounds__(kThreads) void k_join_stats(JoinStatsPlan p) {
  __shared__ float red[2][4];
  const int r = (int)blockIdx.x;
  const float2* part = (const float2*)p.part + (int64_t)r * p.blocks;
  float top = -INFINITY, sum = 0.f;
  for (int i = (int)threadIdx.x; i < p.blocks; i += kThreads) {
    const float2 v = part[i];
    const float t = fmaxf(top, v.x);
    // (-inf - -inf: an empty tile adds its sum, 0 or NaN, unscaled)
    sum = (top == -INFINITY ? sum : sum * expf(top - t)) + (v.x == -INFINITY ? v.y : v.y * expf(v.x - t));
    top = t;
  }
  for (int d = 1; d < 64; d *= 2) {
    const float ot = __shfl_xor(top, d), os = __shfl_xor(sum, d);
    const float t = fmaxf(top, ot);
    sum = (top == -INFINITY ? sum : sum * expf(top - t)) + (ot == -INFINITY ? os : os * expf(ot - t));
    top = t;
  }
  if ((threadIdx.x & 63) == 0) {
    red[0][threadIdx.x >> 6] = top;
    red[1][threadIdx.x >> 6] = sum;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 4; ++w) {
    const float ot = red[0][w], os = red[1][w];
    const float t = fmaxf(top, ot);
    sum = (top == -INFINITY ? sum : sum * expf(top - t)) + (ot == -INFINITY ? os : os * expf(ot - t));
    top = t;
  }
  const float lse = top + logf(sum);
  const int target = p.targets[r];
  const bool empty = lse == -INFINITY, outside = target >= p.vocab;
  p.lse[r] = lse;
  p.loss[r] = target < 0 ? 0.f : empty || outside ? NAN : lse - p.target[r];
  if (p.row_flags) {
    uint32_t f = 0;
    if (lse != lse || lse == INFINITY) f |= LSAMP_ROW_NONFINITE;
    if (empty) f |= LSAMP_ROW_EMPTY;
    if (outside) f |= LSAMP_ROW_TOKEN_RANGE;
    p.row_flags[r] = f;
  }
}

// A row's gradient is led by its target's entry, d_loss (p - 1), nearly d_loss
// itself where the target is unlikely.  The scale brings the largest |d_loss|
// to 32640 = 255 x 2^7: exact in bfloat16 and float16 and just below a power of
// two, where a rounding is relatively smallest; small probabilities stay
// normal numbers of float16 down to 2^-29.  Only rows that have a gradient count
// (the epilogue that writes it leaves the same ones out), and only finite values:
// what a caller keeps at ignored rows must not shrink the others'.
//
// Float32 gradients are multiplied by a power of two, which changes no bit of the
// result, to a largest |d_loss| of 2^14 to 2^15: the products split them into
// bfloat16 parts, whose last step is 2^-133, so that values below 2^-110 would
// keep fewer than 24 bits (a loss times 2^-106: its gradients were off by 2^-17 in the norm).
constexpr float kGradTop = 32640.f;

__global__ __launch_bounds__(1024) void k_grad_scale(GradScalePlan p) {
  __shared__ float red[16];
  float top = 0.f;
  // (eight rows of a thread on their way together: 2^20 rows 0.75 ms less than one by one)
#pragma unroll 8
  for (int r = (int)threadIdx.x; r < p.rows; r += 1024) {
    const int target = p.targets[r];
    const float d = fabsf(p.d_loss[r]), lse = p.lse[r];
    const bool counts = (target >= 0) & (target < p.vocab) & (lse != -INFINITY) & (d < INFINITY);
    top = fmaxf(top, counts ? d : 0.f);
  }
  for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 16; ++w) top = fmaxf(top, red[w]);
  float s = 1.f;
  if (p.exact) {
    if (top > 0.f) s = ldexpf(1.f, max(-100, min(100, 14 - ilogbf(top))));
  } else {
    if (top > 0.f) s = kGradTop / top;
    if (!(s < 1e30f)) s = 1e30f;
    if (s < 1e-30f) s = 1e-30f;
  }
  p.scale[0] = s;
  p.scale[1] = 1.f / s;
}

}  // namespace

int launch_pack(const PackPlan& p, int element_bytes, void* stream) {
  const int chunks = p.dst_cols / (16 / element_bytes);
  const dim3 grid((unsigned)((chunks + kThreads - 1) / kThreads),
                  (unsigned)(p.rows < 32768 ? p.rows : 32768));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (element_bytes == 1)
    hipLaunchKernelGGL((k_pack<uint8_t>), grid, dim3(kThreads), 0, st, p);
  else if (element_bytes == 2)
    hipLaunchKernelGGL((k_pack<uint16_t>), grid, dim3(kThreads), 0, st, p);
  else
    hipLaunchKernelGGL((k_pack<uint32_t>), grid, dim3(kThreads), 0, st, p);
  return (int)hipGetLastError();
}

int launch_join_stats(const JoinStatsPlan& p, void* stream) {
  hipLaunchKernelGGL(k_join_stats, dim3((unsigned)p.rows), dim3(kThreads), 0,
                     reinterpret_cast<hipStream_t>(stream), p);
  return (int)hipGetLastError();
}

int launch_grad_scale(const GradScalePlan& p, void* stream) {
  hipLaunchKernelGGL(k_grad_scale, dim3(1), dim3(1024), 0, reinterpret_cast<hipStream_t>(stream), p);
  return (int)hipGetLastError();
}

}  // namespace lsamp
