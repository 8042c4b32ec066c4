// lsamp_norm.hip — layer norm over the rows of a matrix, its gradients, and rows
// quantised to 8-bit integers.
//
//   y = (x - mean) rstd w + b,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   d_x = rstd (g - mean(g) - xh mean(g xh)) + residual,  g = d w,  xh = (x - mean) rstd
//   d_w = sum over rows of d xh,  d_b = sum over rows of d
//   q = rint(x / s),  s = max |x| / 127 (as a product with 1 / 127)
//
// All are bound by memory: a row of up to 16,384 elements is read once, into
// registers, eight elements of a thread in each of V groups; the variance is that
// of the centred values (their squares do not cancel).  Longer rows are read
// again for every sum.  All sums are float32.
#include <hip/hip_runtime.h>

#include "lsamp_head.h"
#include "lsamp_quant.h"

namespace lsamp {
namespace {

constexpr int kWave = 64;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename E>
struct __attribute__((packed, aligned(sizeof(E)))) Any16 {  // 16 bytes of any alignment
  u32x4 v;
};
struct Eight {
  float v[8];
};
// Eight elements of a row as they lie in memory, `valid` of them in the row, the others
// zero.
template <typename E>
struct Raw {
  E e[8];
  __device__ __forceinline__ void load(const E* p, int valid) {
    if (valid >= 8) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(E) / 2; ++i) {
        const u32x4 q = ((const Any16<E>*)p)[i].v;
        __builtin_memcpy((char*)e + 16 * i, &q, 16);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] = k < valid ? p[k] : (E)0.f;
    }
  }
  __device__ __forceinline__ float at(int k) const { return (float)e[k]; }
  __device__ __forceinline__ void fill(float v) {
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = (E)v;
  }
};
// `stream`: past the caches.
template <typename E>
__device__ __forceinline__ void store8(E* p, const Eight& x, int valid, bool stream = false) {
  E e[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) e[k] = (E)x.v[k];
  if (valid >= 8) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) {
      u32x4 q;
      __builtin_memcpy(&q, (const char*)e + 16 * i, 16);
      if (stream)  // (as a builtin it would be joined with the other store, and lost)
        // (two wait states before its data may be overwritten, which the compiler does not
        // know to be a store's)
        asm volatile("global_store_dwordx4 %0, %1, off nt\n\ts_nop 1"
                     :
                     : "v"((char*)p + 16 * i), "v"(q)
                     : "memory");
      else
        ((Any16<E>*)p)[i].v = q;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < valid) p[k] = e[k];
  }
}

// Sums of N values (maxima of whole numbers) over the THREADS threads of a row: a wave,
// or a work-group.  Every thread gets them.  `red` has 2 N of them a wave: a row's
// exchange may begin while the one before is still read.
__device__ __forceinline__ float joined(float a, float b) { return a + b; }
__device__ __forceinline__ uint32_t joined(uint32_t a, uint32_t b) { return max(a, b); }
template <int THREADS, int N, typename T>
__device__ __forceinline__ void join(T (&s)[N], T* red, int& turn) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2)
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = joined(s[i], (T)__shfl_xor(s[i], d));
  if constexpr (THREADS > kWave) {
    constexpr int kWaves = THREADS / kWave;
    const int wave = (int)threadIdx.x / kWave;
    T* const at = red + turn * (kWaves * N);
    turn ^= 1;
    if ((threadIdx.x & (kWave - 1)) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) at[wave * N + i] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      T t = at[i];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) t = joined(t, at[w * N + i]);
      s[i] = t;
    }
  }
}

constexpr int kStay = 2048, kFew = 768;
constexpr int kBlock = 256;  // threads of a work-group whose rows are a wave's

// A row's threads and the rows of a work-group.
template <int THREADS>
struct Rows {
  static constexpr int kPer = THREADS < kBlock ? kBlock / THREADS : 1;
  static constexpr int kGroup = THREADS < kBlock ? kBlock : THREADS;
  int first, step, t;  // the thread's first row, the distance to the next, its place in the row
  __device__ __forceinline__ Rows(int group, int groups)
      : first(group * kPer + (int)threadIdx.x / THREADS), step(groups * kPer),
        t((int)threadIdx.x % THREADS) {}
};

// A thread's groups of a row: group i of span s (one span unless LONG).
template <int THREADS, int V>
__device__ __forceinline__ int col_of(int t, int s, int i) {
  return ((s * V + i) * THREADS + t) * 8;
}
template <int THREADS, int V, typename E>
__device__ __forceinline__ void fetch(Raw<E> (&a)[V], const void* p, int64_t row, int cols, int t, int s) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = col_of<THREADS, V>(t, s, i);
    a[i].load((const E*)p + row + c, cols - c);
  }
}

// The next row is on its way while one is summed; weight and bias stay in registers.
// 16384 x 4096 bf16 46 us (5.8 TB/s; a row a work-group, without the next one, 67); one row of
// 2048 a launch.  LONG: rows of any length, read three times (300 x 40000 18 us).
template <typename E, int THREADS, int V, bool LONG>
__global__ __launch_bounds__(Rows<THREADS>::kGroup) void k_norm(NormPlan p) {
  __shared__ float red[2 * THREADS / kWave];
  const Rows<THREADS> rows((int)blockIdx.x, (int)gridDim.x);
  int turn = 0;
  const float per = 1.f / (float)p.cols;
  const int span = LONG ? (p.cols + V * THREADS * 8 - 1) / (V * THREADS * 8) : 1;
  const auto col = [&](int s, int i) { return col_of<THREADS, V>(rows.t, s, i); };
  Raw<E> a[V], next[LONG ? 1 : V], w[V], b[V];
  const auto vectors = [&](int s) {
    if (p.weight) fetch<THREADS, V>(w, p.weight, 0, p.cols, rows.t, s);
    if (p.bias) fetch<THREADS, V>(b, p.bias, 0, p.cols, rows.t, s);
  };
  if constexpr (!LONG) {
    if (rows.first < p.rows) fetch<THREADS, V>(next, p.x, rows.first * p.ld_x, p.cols, rows.t, 0);
    vectors(0);
  }
  for (int64_t r = rows.first; r < p.rows; r += rows.step) {
    if constexpr (!LONG) {
#pragma unroll
      for (int i = 0; i < V; ++i) a[i] = next[i];
      if (r + rows.step < p.rows)
        fetch<THREADS, V>(next, p.x, (r + rows.step) * p.ld_x, p.cols, rows.t, 0);
    }
    float sum[1] = {0.f};
    for (int s = 0; s < span; ++s) {
      if (LONG) fetch<THREADS, V>(a, p.x, r * p.ld_x, p.cols, rows.t, s);
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[0] += a[i].at(k);
    }
    join<THREADS>(sum, red, turn);
    const float mean = sum[0] * per;
    float sq[1] = {0.f};
    for (int s = 0; s < span; ++s) {
      if (LONG) fetch<THREADS, V>(a, p.x, r * p.ld_x, p.cols, rows.t, s);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int valid = p.cols - col(s, i);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float d = a[i].at(k) - mean;
          sq[0] += k < valid ? d * d : 0.f;
        }
      }
    }
    join<THREADS>(sq, red, turn);
    const float rstd = 1.f / sqrtf(sq[0] * per + p.eps);
    if (rows.t == 0) {
      if (p.mean) p.mean[r] = mean;
      if (p.rstd) p.rstd[r] = rstd;
    }
    for (int s = 0; s < span; ++s) {
      if (LONG) {
        fetch<THREADS, V>(a, p.x, r * p.ld_x, p.cols, rows.t, s);
        vectors(s);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = col(s, i), valid = p.cols - c;
        if (valid <= 0) continue;
        Eight y;
#pragma unroll
        for (int k = 0; k < 8; ++k) y.v[k] = (a[i].at(k) - mean) * rstd;
        if (p.weight) {
#pragma unroll
          for (int k = 0; k < 8; ++k) y.v[k] *= w[i].at(k);
        }
        if (p.bias) {
#pragma unroll
          for (int k = 0; k < 8; ++k) y.v[k] += b[i].at(k);
        }
        store8((E*)p.out + r * p.ld_out + c, y, valid, p.stream);
      }
    }
  }
}

// A row's gradient, and (SUMS) the work-group's share of the columns' sums, which
// stay in registers over its rows; the next row is on its way meanwhile (16384 x 4096 bf16
// with a residual 108 us, 4.9 TB/s; 171 without the next row).  1024 threads
// have 128 registers each: their sums lie in LDS, a thread's own 16 bytes beside its
// neighbours', and rows of more than 8,192 elements are not fetched ahead (4096 x 16384
// bf16: 433 us with the sums in registers, spilled; 111 so).  LONG: d_x only, each row
// read twice.
template <typename E, int THREADS, int V, bool SUMS, bool LONG>
__device__ __forceinline__ void backward_rows(const NormBackwardPlan& p, const Rows<THREADS>& rows) {
  static_assert(!(SUMS && LONG), "a long row's sums are another kernel's");
  constexpr int kPer = Rows<THREADS>::kPer;
  __shared__ float red[4 * THREADS / kWave];
  int turn = 0;
  const float per = 1.f / (float)p.cols;
  const int span = LONG ? (p.cols + V * THREADS * 8 - 1) / (V * THREADS * 8) : 1;
  const auto col = [&](int s, int i) { return col_of<THREADS, V>(rows.t, s, i); };
  constexpr bool kInLds = SUMS && THREADS == 1024;
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  __shared__ f32x4 kept[kInLds ? V * 4 : 1][kInLds ? THREADS : 1];
  Eight sum_w[SUMS ? V : 1], sum_b[SUMS ? V : 1];
  if constexpr (SUMS) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) sum_w[i].v[k] = sum_b[i].v[k] = 0.f;
  }
  if constexpr (kInLds) {
#pragma unroll
    for (int i = 0; i < V * 4; ++i) kept[i][rows.t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // four terms of group i's sums (which: of d xh, of d), its half h
  const auto add = [&](int i, int which, int h, const f32x4& v) {
    if constexpr (kInLds) kept[(i * 2 + which) * 2 + h][rows.t] += v;
  };
  struct Row {
    Raw<E> x[V], d[V], res[V];
    float mean, rstd;
  };
  const auto load = [&](Row& o, int64_t r, int s, bool residual) {
    fetch<THREADS, V>(o.x, p.x, r * p.ld_x, p.cols, rows.t, s);
    fetch<THREADS, V>(o.d, p.d_out, r * p.ld_d, p.cols, rows.t, s);
    if (residual) fetch<THREADS, V>(o.res, p.residual, r * p.ld_residual, p.cols, rows.t, s);
    o.mean = p.mean[r];
    o.rstd = p.rstd[r];
  };
  Raw<E> w[V];
  const auto weights = [&](int s) {
    if (p.weight) {
      fetch<THREADS, V>(w, p.weight, 0, p.cols, rows.t, s);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i].fill(1.f);
    }
  };
  const bool has_residual = p.residual != nullptr;
  constexpr bool kAhead = !LONG && (THREADS < 1024 || V == 1);
  Row row, next;
  if constexpr (kAhead) {
    if (rows.first < p.rows) load(next, rows.first, 0, has_residual);
  }
  if (!LONG) weights(0);
  for (int64_t r = rows.first; r < p.rows; r += rows.step) {
    if constexpr (kAhead) {
      row = next;
      if (r + rows.step < p.rows) load(next, r + rows.step, 0, has_residual);
    } else if constexpr (!LONG) {
      load(row, r, 0, has_residual);
    }
    float c12[2] = {0.f, 0.f};
    for (int s = 0; s < span; ++s) {
      if (LONG) {
        weights(s);
        load(row, r, s, false);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int valid = p.cols - col(s, i);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f32x4 tw, tb;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            // (past the row's end d is 0, and so is every term)
            const int k = h * 4 + q;
            const float d = row.d[i].at(k), xh = (row.x[i].at(k) - row.mean) * row.rstd;
            const float dx = k < valid ? d * xh : 0.f;
            if constexpr (SUMS && !kInLds) {
              sum_w[i].v[k] += dx;
              sum_b[i].v[k] += d;
            }
            tw[q] = dx;
            tb[q] = d;
            c12[0] += d * w[i].at(k);
            c12[1] += dx * w[i].at(k);
          }
          add(i, 0, h, tw);
          add(i, 1, h, tb);
        }
      }
    }
    if (!p.d_x) continue;  // (the same for every thread)
    join<THREADS>(c12, red, turn);
    const float c1 = c12[0] * per, c2 = c12[1] * per;
    for (int s = 0; s < span; ++s) {
      if (LONG) {
        weights(s);
        load(row, r, s, has_residual);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = col(s, i), valid = p.cols - c;
        if (valid <= 0) continue;
        Eight y;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float g = row.d[i].at(k) * w[i].at(k);
          const float xh = (row.x[i].at(k) - row.mean) * row.rstd;
          y.v[k] = row.rstd * (g - c1 - xh * c2);
        }
        if (has_residual) {
#pragma unroll
          for (int k = 0; k < 8; ++k) y.v[k] += row.res[i].at(k);
        }
        store8((E*)p.d_x + r * p.ld_dx + c, y, valid, p.stream);
      }
    }
  }
  if constexpr (kInLds) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        sum_w[i].v[k] = kept[i * 4 + k / 4][rows.t][k % 4];
        sum_b[i].v[k] = kept[i * 4 + 2 + k / 4][rows.t][k % 4];
      }
  }
  if constexpr (SUMS) {
    // [work-group][2][ld_part]; rows of a wave each are joined first
    if constexpr (kPer > 1) {
      __shared__ float both[kPer - 1][V][8][2][kWave];
      const int wave = (int)threadIdx.x / kWave;
      if (wave > 0)
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            both[wave - 1][i][k][0][rows.t] = sum_w[i].v[k];
            both[wave - 1][i][k][1][rows.t] = sum_b[i].v[k];
          }
      __syncthreads();
      if (wave > 0) return;
      for (int o = 0; o < kPer - 1; ++o)
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            sum_w[i].v[k] += both[o][i][k][0][rows.t];
            sum_b[i].v[k] += both[o][i][k][1][rows.t];
          }
    }
    float* const part = p.part + (int64_t)blockIdx.x * 2 * p.ld_part;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = col(0, i);
      if (c >= p.cols) continue;  // (rows of sums are whole groups of eight)
      store8(part + c, sum_w[i], 8);
      store8(part + p.ld_part + c, sum_b[i], 8);
    }
  }
}

template <typename E, int THREADS, int V, bool SUMS, bool LONG>
__global__ __launch_bounds__(Rows<THREADS>::kGroup) void k_norm_backward(NormBackwardPlan p) {
  backward_rows<E, THREADS, V, SUMS, LONG>(p, Rows<THREADS>((int)blockIdx.x, (int)gridDim.x));
}

// Column sums of long rows: a column a thread, a chunk of rows a work-group.
template <typename E>
__global__ __launch_bounds__(kBlock) void k_norm_sums(NormBackwardPlan p) {
  const int c = (int)blockIdx.x * kBlock + (int)threadIdx.x;
  if (c >= p.cols) return;
  const int per = (p.rows + p.chunks - 1) / p.chunks;
  const int r0 = (int)blockIdx.y * per, r1 = min(p.rows, r0 + per);
  float w = 0.f, b = 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    const float d = (float)((const E*)p.d_out)[r * p.ld_d + c];
    const float xh = ((float)((const E*)p.x)[r * p.ld_x + c] - p.mean[r]) * p.rstd[r];
    w += d * xh;
    b += d;
  }
  float* const part = p.part + (int64_t)blockIdx.y * 2 * p.ld_part;
  part[c] = w;
  part[p.ld_part + c] = b;
}

// Few rows (301 x 1537 f16 4.2 us, shares and their join 10.4): one launch, whose first
// `row_groups` work-groups take rows and the others 16 columns each, which they read from
// the L2 once more: 16 threads a column take rows in turn.
template <typename E>
__device__ __forceinline__ void columns(const NormBackwardPlan& p, int group) {
  __shared__ float red[2][16][17];
  const int lane = (int)threadIdx.x & 15, part = (int)threadIdx.x >> 4;
  const int c = group * 16 + lane;
  float w = 0.f, b = 0.f;
  if (c < p.cols) {
#pragma unroll 8
    for (int r = part; r < p.rows; r += 16) {
      const float d = (float)((const E*)p.d_out)[(int64_t)r * p.ld_d + c];
      const float xh = ((float)((const E*)p.x)[(int64_t)r * p.ld_x + c] - p.mean[r]) * p.rstd[r];
      w += d * xh;
      b += d;
    }
  }
  red[0][part][lane] = w;
  red[1][part][lane] = b;
  __syncthreads();
  if (part > 1 || c >= p.cols) return;
  float s = red[part][0][lane];
#pragma unroll
  for (int i = 1; i < 16; ++i) s += red[part][i][lane];
  E* const out = (E*)(part ? p.d_bias : p.d_weight);
  if (out) out[c] = (E)s;
}

template <typename E, int THREADS, int V>
__global__ __launch_bounds__(kBlock) void k_norm_backward_few(NormBackwardPlan p, int row_groups) {
  const int group = (int)blockIdx.x;
  if (group < row_groups)
    backward_rows<E, THREADS, V, false, false>(p, Rows<THREADS>(group, row_groups));
  else
    columns<E>(p, group - row_groups);
}

// The work-groups' shares, joined in their order: 64 columns a work-group of
// sixteen waves, the waves taking shares in turn (512 of 4096 columns 5 us).
constexpr int kJoinWaves = 16;
template <typename E>
__global__ __launch_bounds__(kJoinWaves* kWave) void k_norm_join(NormBackwardPlan p) {
  __shared__ float red[kJoinWaves][kWave];
  const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
  const int c = (int)blockIdx.x * kWave + lane, which = (int)blockIdx.y;
  E* const out = (E*)(which ? p.d_bias : p.d_weight);
  if (!out) return;
  float s = 0.f;
  if (c < p.cols) {
#pragma unroll 8
    for (int i = wave; i < p.chunks; i += kJoinWaves) s += p.part[((int64_t)i * 2 + which) * p.ld_part + c];
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= p.cols) return;
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w) s += red[w][lane];
  out[c] = (E)s;
}

// A row's largest magnitude, then its bytes (lsamp_quant.h): 151936 x 2048 bf16 178 us, at the
// memory rate (0.93 GB, 5.2 TB/s); 64 x 4096 a launch.
template <typename E, int THREADS, int V, bool LONG>
__global__ __launch_bounds__(Rows<THREADS>::kGroup) void k_quantize(QuantizePlan p) {
  __shared__ uint32_t red[2 * THREADS / kWave];
  const Rows<THREADS> rows((int)blockIdx.x, (int)gridDim.x);
  int turn = 0;
  const int span = LONG ? (p.cols + V * THREADS * 8 - 1) / (V * THREADS * 8) : 1;
  Raw<E> a[V], next[LONG ? 1 : V];
  if constexpr (!LONG) {
    if (rows.first < p.rows) fetch<THREADS, V>(next, p.x, rows.first * p.ld_x, p.cols, rows.t, 0);
  }
  for (int64_t r = rows.first; r < p.rows; r += rows.step) {
    if constexpr (!LONG) {
#pragma unroll
      for (int i = 0; i < V; ++i) a[i] = next[i];
      if (r + rows.step < p.rows)
        fetch<THREADS, V>(next, p.x, (r + rows.step) * p.ld_x, p.cols, rows.t, 0);
    }
    uint32_t top[1] = {0};
    for (int s = 0; s < span; ++s) {
      if (LONG) fetch<THREADS, V>(a, p.x, r * p.ld_x, p.cols, rows.t, s);
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) top[0] = max(top[0], magnitude(a[i].at(k)));
    }
    join<THREADS>(top, red, turn);
    const float scale = row_scale(top[0]), inverse = 1.f / scale;
    if (rows.t == 0) p.scale[r] = scale;
    for (int s = 0; s < span; ++s) {
      if (LONG) fetch<THREADS, V>(a, p.x, r * p.ld_x, p.cols, rows.t, s);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = col_of<THREADS, V>(rows.t, s, i), valid = p.out_cols - c;
        float v[8];  // (past the row's end 0)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = a[i].at(k);
        const uint64_t word = quantize8(v, scale, inverse);
        if (valid <= 0) continue;
        int8_t* const to = p.q + r * p.ld_q + c;
        if (valid >= 8) {
          struct __attribute__((packed)) Any8 {
            uint64_t v;
          };
          ((Any8*)to)->v = word;
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < valid) to[k] = (int8_t)(word >> (8 * k));
        }
      }
    }
  }
}

// The shape of a row of `cols` elements: a wave, 256 or 1024 threads, one, two or
// four groups of eight of a thread.  Few rows take more threads a row (1023 x 2048:
// 4.6 us, 1024 rows with a wave each 5.5; gradients 14.8 and 13.0).
enum Shape { kWave1, kWave2, kWave4, kBlock1, kBlock2, kWide1, kWide2, kLong };
Shape shape_of(int rows, int cols) {
  if (cols <= 2048 && rows >= 1024) return cols <= 512 ? kWave1 : cols <= 1024 ? kWave2 : kWave4;
  if (cols <= 512) return kWave1;
  if (cols <= 2048) return kBlock1;
  if (cols <= 4096) return kBlock2;
  return cols <= 8192 ? kWide1 : cols <= 16384 ? kWide2 : kLong;
}
// Whether the columns' sums are taken beside the rows, in the same launch (forward and
// gradients of 700 x 4096 16.0 us, with shares and their join 19.6; 768 x 1024 10.9 and 15.6;
// 1000 x 4096 24 and 21): not where the rows' gradients are written over the d_out or the x
// that the columns read.
bool few(int rows, int cols, bool in_place) { return rows <= kFew && cols <= 4096 && !in_place; }
int rows_per_group(Shape s) { return s <= kWave4 ? kBlock / kWave : 1; }
int threads_of(Shape s) { return s >= kWide1 ? 1024 : kBlock; }

// Work-groups that stay, each for several rows of a long matrix.
unsigned launched(int64_t groups, Shape s) {
  const int64_t most = s >= kWide1 ? kStay / 4 : kStay;
  return (unsigned)(groups < most ? groups : most);
}

#define LSAMP_SHAPES(s, K, ARGS)        \
  switch (s) {                          \
    case kWave1: K(64, 1, false); break;  \
    case kWave2: K(64, 2, false); break;  \
    case kWave4: K(64, 4, false); break;  \
    case kBlock1: K(256, 1, false); break; \
    case kBlock2: K(256, 2, false); break; \
    case kWide1: K(1024, 1, false); break; \
    case kWide2: K(1024, 2, false); break; \
    default: K(1024, 1, true); break;     \
  }

template <typename E>
int norm(const NormPlan& p, hipStream_t st) {
  const Shape s = shape_of(p.rows, p.cols);
  const int64_t groups = ((int64_t)p.rows + rows_per_group(s) - 1) / rows_per_group(s);
  const dim3 grid(launched(groups, s)), block((unsigned)threads_of(s));
#define K(T, V, L) hipLaunchKernelGGL((k_norm<E, T, V, L>), grid, block, 0, st, p)
  LSAMP_SHAPES(s, K, )
#undef K
  return (int)hipGetLastError();
}

template <typename E>
int norm_backward(const NormBackwardPlan& p, hipStream_t st) {
  const Shape s = shape_of(p.rows, p.cols);
  const bool sums = p.d_weight || p.d_bias;
  const int64_t groups = ((int64_t)p.rows + rows_per_group(s) - 1) / rows_per_group(s);
  if (sums && !p.chunks) {
    const int row_groups = p.d_x ? (int)groups : 0;
    const dim3 all((unsigned)(row_groups + (p.cols + 15) / 16));
#define K(T, V) hipLaunchKernelGGL((k_norm_backward_few<E, T, V>), all, dim3(kBlock), 0, st, p, row_groups)
    switch (s) {
      case kWave1: K(64, 1); break;
      case kBlock1: K(256, 1); break;
      default: K(256, 2); break;
    }
#undef K
    return (int)hipGetLastError();
  }
  const dim3 grid(sums && s != kLong ? (unsigned)p.chunks : launched(groups, s));
  const dim3 block((unsigned)threads_of(s));
  if (s == kLong) {
    // (the sums first: d_x may be d_out or x itself)
    if (sums)
      hipLaunchKernelGGL((k_norm_sums<E>),
                         dim3((unsigned)((p.cols + kBlock - 1) / kBlock), (unsigned)p.chunks),
                         dim3(kBlock), 0, st, p);
    if (p.d_x) hipLaunchKernelGGL((k_norm_backward<E, 1024, 1, false, true>), grid, block, 0, st, p);
  } else if (sums) {
#define K(T, V, L) hipLaunchKernelGGL((k_norm_backward<E, T, V, !(L), L>), grid, block, 0, st, p)
    LSAMP_SHAPES(s, K, )
#undef K
  } else {
#define K(T, V, L) hipLaunchKernelGGL((k_norm_backward<E, T, V, false, L>), grid, block, 0, st, p)
    LSAMP_SHAPES(s, K, )
#undef K
  }
  if (sums)
    hipLaunchKernelGGL((k_norm_join<E>), dim3((unsigned)((p.cols + kWave - 1) / kWave), 2),
                       dim3(kJoinWaves * kWave), 0, st, p);
  return (int)hipGetLastError();
}

template <typename E>
int quantize(const QuantizePlan& p, hipStream_t st) {
  const Shape s = shape_of(p.rows, p.cols);
  const int64_t groups = ((int64_t)p.rows + rows_per_group(s) - 1) / rows_per_group(s);
  const dim3 grid(launched(groups, s)), block((unsigned)threads_of(s));
#define K(T, V, L) hipLaunchKernelGGL((k_quantize<E, T, V, L>), grid, block, 0, st, p)
  LSAMP_SHAPES(s, K, )
#undef K
  return (int)hipGetLastError();
}

#define LSAMP_EACH_TYPE(call)                                 \
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);     \
  switch (dtype) {                                            \
    case LSAMP_DTYPE_F32: return call<float>(p, st);          \
    case LSAMP_DTYPE_BF16: return call<__bf16>(p, st);        \
    default: return call<_Float16>(p, st);                    \
  }

}  // namespace

// Shares of the columns' sums: a work-group's.
int norm_chunks(int rows, int cols, bool in_place) {
  if (few(rows, cols, in_place)) return 0;
  const Shape s = shape_of(rows, cols);
  if (s == kLong) return rows < 64 ? 1 : rows / 32 < 256 ? rows / 32 : 256;
  const int groups = (rows + rows_per_group(s) - 1) / rows_per_group(s);
  const int most = s == kWide2 ? 256 : 512;
  return groups < most ? groups : most;
}

int launch_norm(const NormPlan& p, int dtype, void* stream) { LSAMP_EACH_TYPE(norm) }
int launch_norm_backward(const NormBackwardPlan& p, int dtype, void* stream) {
  LSAMP_EACH_TYPE(norm_backward)
}
int launch_quantize(const QuantizePlan& p, int dtype, void* stream) { LSAMP_EACH_TYPE(quantize) }

}  // namespace lsamp
