// lsamp_orth.h — plans of the orthogonalised update, shared by its entry point and
// its kernels.
#ifndef LSAMP_ORTH_H
#define LSAMP_ORTH_H

#include "lsamp_head.h"

namespace lsamp {

// Steps are in elements where they are of the workspace's matrices, else in bytes.
struct OrthStart {
  int32_t rows, cols, parts;  // work-groups of a matrix
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
  int32_t n;
  const float* left;  // of the first step's A, else NULL
  const void* in;     // B: A
  void* out;
  int64_t ld, step;
  float b3, c3;
  float* diagonal;  // [batch][step_d] B's, where it is kept apart
  int64_t step_d;
};
struct EpiOrthUpdate {
  int32_t m, n;
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

// LSAMP_DTYPE_F32 or LSAMP_DTYPE_F16: what the products are taken in.  Tiles: 128 and
// 64, alone or grouped; 256 for float16.
template <int DT>
struct OrthOps {
  static int start(const OrthStart& p, int batch, int in_dtype, void* stream);
  static int gram(bool tall, GemmTile tile, const BatchPlan& g, const EpiSymmetric& e, void* stream);
  static int poly(GemmTile tile, const BatchPlan& g, const EpiSymmetric& e, void* stream);
  static int update(bool tall, GemmTile tile, const BatchPlan& g, const EpiOrthUpdate& e,
                    void* stream);
};

}  // namespace lsamp

#endif
