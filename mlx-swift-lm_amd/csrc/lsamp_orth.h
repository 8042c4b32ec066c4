// lsamp_orth.h — plans of the orthogonalised update, shared by its entry point and
// its kernels.
#ifndef LSAMP_ORTH_H
#define LSAMP_ORTH_H

#include "lsamp_head.h"

namespace lsamp {

// Matrices of the workspace are float16, in one part or two (lo: the rest); their rows
// and columns are multiples of 64.  Steps are in elements there, else in bytes.
struct OrthStart {
  int32_t rows, cols, all_rows;
  int32_t parts;  // work-groups of a matrix
  int32_t log_x;  // 2^log_x threads a row
  float eps;
  const void* x;
  int64_t ld_x, step_x;
  double* part;  // [batch][parts]
  float* left;   // [batch]: 2^e / (norm + eps)
  void* hi;
  void* lo;
  int64_t ld, step;
};
struct EpiSymmetric {  // A, or B
  int32_t n;           // rows, columns and their distance
  float b3, c3;
  const float* left;  // of the first step's A, else NULL
  const void* in;     // B: A
  const void* in_lo;
  void* out;
  void* out_lo;
  int64_t step;
  float* diagonal;  // [batch][n] B's
};
struct EpiOrthUpdate {
  int32_t m, n, all_m;
  int32_t tall;
  int32_t out_dtype;
  float a1;
  const float* left;
  const void* x_hi;
  const void* x_lo;
  const float* diagonal;
  int64_t step_d;
  void* to_hi;
  void* to_lo;
  int64_t ld, step;
  void* out;  // the last step's: scale X' + keep base; else NULL
  int64_t ld_out, step_out;
  const void* base;
  int64_t ld_base, step_base;
  float scale, keep;
};

int launch_orth_start(const OrthStart& p, int batch, int in_dtype, void* stream);

// WIDE: A and B in two parts.  Tiles: 256, 128 and 64, the latter grouped too; 32x8 where
// both operands have rows along the output (not a tall gram, not a wide update); 192 for
// gram and poly.
template <bool WIDE>
struct OrthOps {
  static int gram(bool tall, GemmTile tile, const BatchPlan& g, const EpiSymmetric& e, void* stream);
  static int poly(GemmTile tile, const BatchPlan& g, const EpiSymmetric& e, void* stream);
  static int update(bool tall, GemmTile tile, const BatchPlan& g, const EpiOrthUpdate& e,
                    void* stream);
};

}  // namespace lsamp

#endif
