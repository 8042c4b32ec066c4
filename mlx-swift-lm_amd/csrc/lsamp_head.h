// lsamp_head.h — plans of the hidden-state operators (linear blocks, the
// vocabulary head's loss, dropout) shared by the C entry points, which build
// them, and the kernels, which run them.
#ifndef LSAMP_HEAD_H
#define LSAMP_HEAD_H

#include <stdint.h>

#include "../../include/lsamp.h"

namespace lsamp {

// A matrix in HBM: `rows` rows of `cols` readable elements, `ld` elements
// apart.  The tiled products read 16-byte chunks: p and ld in bytes are multiples
// of 16, cols of a chunk's elements.  Loose shapes take rows of any address,
// distance and length, as the kernels of few rows do of W (and of x up to 16 rows).
struct MatrixRef {
  const void* p;
  int64_t ld;
  int32_t rows, cols;
};

struct GemmPlan {
  MatrixRef a, b;
  int32_t tiles_m, tiles_n, parts;
  int32_t slabs, slabs_per_part;  // 128-byte slabs of the reduction
};

// `parts` equal products, one after another in memory, of operands in whole slabs.
struct BatchPlan : GemmPlan {
  int64_t step_a, step_b;  // bytes
  int32_t symmetric;       // the result is: tiles left of the diagonal are left out
  // Operands in two parts, `rest_*` bytes from a's and b's first to its second: the
  // sums are those of first first + first second + second first.  Else 0.
  int64_t rest_a, rest_b;
};

// Which operand is read along the reduction's rows (lsamp_gemm.h).
enum GemmRoles { kRolesNT = 0, kRolesNN = 1, kRolesTN = 2 };
// Tile shapes.  256 x 256, 128 x 128 and 64 x 64; 128 and 64 with two and four
// slabs of the reduction at a time, for launches of at most a tile a CU; loose ones
// for operands whose rows are no 16-byte chunks; the products of at most 16, 32 or 64
// rows (lsamp_skinny.h), 64 or 16 columns a work-group; 192 x 192 for symmetric products,
// and 32 x 32 with eight slabs at a time for batches of at most one such tile a CU.
enum GemmTile {
  kTile256,
  kTile128,
  kTile64,
  kTile128x2,
  kTile64x4,
  kLoose128,
  kLoose64,
  kLoose64x4,
  kSkinny64,
  kSkinny16,
  kTile192,
  kTile32x8,
};
constexpr int kTileSide[] = {256, 128, 64, 128, 64, 128, 64, 64, 64, 16, 192, 32};
constexpr int kTileWavesM[] = {2, 2, 2, 2, 2, 2, 2, 2, 1, 1, 2, 1};  // waves that share a tile's rows
constexpr int kSkinnyRows = 64;

// Epilogues.  `m`, `n`: rows and columns that exist.
struct EpiLinear {
  int32_t m, n;
  int32_t activation, wide;  // wide: out is float32
  int32_t stream;            // pre, and out unless it is float32, are stored past the caches
  float softcap;
  const void* bias;
  const void* residual;
  int64_t ld_residual;
  void* out;
  int64_t ld_out;
  float* pre;
  int64_t ld_pre;
};
struct EpiStore {  // out = sums * *scale, in the operands' type
  int32_t m, n;
  void* out;
  int64_t ld_out;
  const float* scale;  // device, or NULL for 1
  int32_t stream;      // stored past the caches
};
struct EpiPartial {  // float32 sums of one part, added to what is there
  int32_t m, n;
  int32_t accumulate;
  float* out;
  int64_t ld;           // a multiple of 4
  int64_t part_stride;
};
struct EpiStats {  // a tile's maximum and sum of exponentials of every row
  int32_t m, n;
  int32_t first_col, blocks, first_block;
  float softcap;
  const void* bias;
  const int32_t* targets;
  float* part;    // [m][blocks][2]
  float* target;  // [m] the target's logit
};
struct EpiGrad {  // the loss's gradient at a piece of the logits
  int32_t m, n;
  int32_t first_col, n_pad;  // columns n .. n_pad - 1 are written as zero
  float softcap;
  const void* bias;
  const int32_t* targets;
  int32_t vocab;
  const float* lse;
  const float* d_loss;
  const float* scale;  // [2] device: what the stored values are multiplied by, and its inverse
  void* out;
  int64_t ld_out;
  float* sums;  // [rows of tiles x their waves][ld_sums] column sums before rounding, or NULL
  int64_t ld_sums;
};

struct PackPlan {  // rows copied to 16-byte aligned rows, zeros up to dst_cols
  const void* src;
  int64_t src_ld;
  void* dst;
  int64_t dst_ld;
  int32_t rows, cols, dst_cols;
};

struct JoinStatsPlan {
  int32_t rows, blocks, vocab;
  const float* part;
  const float* target;
  const int32_t* targets;
  float* loss;
  float* lse;
  uint32_t* row_flags;
};

// scale[0]: what the gradient at the logits is multiplied by (1 where no d_loss of
// a row with a gradient is finite and not 0), scale[1] = 1 / scale[0].
struct GradScalePlan {
  int32_t rows, vocab;
  int32_t exact;  // a power of two (float32)
  const float* d_loss;
  const float* lse;
  const int32_t* targets;
  float* scale;
};

struct ColSumPlan {  // column sums of a matrix, rows_per_chunk rows a partial sum
  int32_t rows, cols;
  int32_t chunks, rows_per_chunk;
  int32_t activation;  // with `pre`: in * activation'(pre) is summed, and written to out
  float softcap;
  const void* in;
  int64_t ld_in;
  const float* pre;
  int64_t ld_pre;
  void* out;
  int64_t ld_out;
  int32_t out_cols;  // columns cols .. out_cols - 1 of out are written as zero
  float* part;       // [chunks][ld_part], or NULL
  int64_t ld_part;
  void* sums;        // one chunk: the sums themselves
  int32_t join_wide;  // the chunks are joined by sixteen waves, not four
};

struct DropoutPlan {
  int32_t rows, cols;
  uint32_t cut;  // an element is kept where its 16 bits are at least this
  float scale;
  uint64_t key, offset;
  const uint64_t* step;
  const void* x;
  int64_t ld_x;
  const void* residual;
  int64_t ld_residual;
  void* out;
  int64_t ld_out;
};

struct EpiLinearInt8 : EpiLinear {
  const float* x_scale;  // [m]
  const float* w_scale;  // [n]
};

// A product of few rows that are kept in LDS: up to 64, of 128 KB in rows of 256 bytes.
struct ResidentPlan {
  int32_t m, k;
  int32_t groups;  // work-groups
  int32_t shared;  // the waves of one share a block of columns
  int32_t fused;   // x is of the block's type (at most 8,192 values), else 8-bit integers in
                   // aligned rows of multiples of 256 bytes, zero behind their ends
  const void* x;
  int64_t ld_x;
  const void* w;
  int64_t ld_w;
};

struct NormPlan {
  int32_t rows, cols;
  int32_t stream;  // out is stored past the caches
  float eps;
  const void* x;
  int64_t ld_x;
  const void* weight;  // or NULL, as bias
  const void* bias;
  void* out;
  int64_t ld_out;
  float* mean;  // or NULL, as rstd
  float* rstd;
};
struct NormBackwardPlan {
  int32_t rows, cols;
  int32_t chunks;  // shares of the columns' sums (norm_chunks), 0 where there are none
  int32_t stream;  // d_x is stored past the caches
  const void* x;
  int64_t ld_x;
  const void* weight;
  const float* mean;
  const float* rstd;
  const void* d_out;
  int64_t ld_d;
  const void* residual;  // or NULL: added to d_x
  int64_t ld_residual;
  void* d_x;  // or NULL
  int64_t ld_dx;
  void* d_weight;  // or NULL
  void* d_bias;
  float* part;  // [chunks][2][ld_part]
  int64_t ld_part;  // a multiple of 8
};
struct QuantizePlan {
  int32_t rows, cols;
  int32_t out_cols;  // columns cols .. out_cols - 1 of q are written as zero
  const void* x;
  int64_t ld_x;
  int8_t* q;
  int64_t ld_q;
  float* scale;
};

// One set of these for each element type; 0 or a hipError_t.
template <int DT>
struct HeadOps {
  // kSkinny16: gemm_linear only; kSkinny64: not gemm_store and gemm_partial;
  // kLoose64 and kLoose64x4: not gemm_stats and gemm_grad; kTile256: not float32.
  static int gemm_linear(GemmTile tile, const GemmPlan& g, const EpiLinear& e, void* stream);
  static int gemm_stats(GemmTile tile, const GemmPlan& g, const EpiStats& e, void* stream);
  static int gemm_grad(GemmTile tile, const GemmPlan& g, const EpiGrad& e, void* stream);
  static int gemm_store(GemmRoles roles, GemmTile tile, const GemmPlan& g, const EpiStore& e,
                        void* stream);
  static int gemm_partial(GemmRoles roles, GemmTile tile, const GemmPlan& g, const EpiPartial& e,
                          void* stream);
  static int join_linear(const EpiPartial& from, int parts, const EpiLinear& e, void* stream);
  static int join_store(const EpiPartial& from, int parts, const EpiStore& e, void* stream);
  static int col_sum(const ColSumPlan& p, void* stream);
  static int col_sum_join(const ColSumPlan& p, void* out, const float* scale, void* stream);
};
// One set for each element type of bias, residual and out.  Tiles: not kTile* for rows
// that are no chunks.
template <int DT>
struct Int8Ops {
  static int gemm_linear(GemmTile tile, const GemmPlan& g, const EpiLinearInt8& e, void* stream);
  static int resident_linear(const ResidentPlan& g, const EpiLinearInt8& e, void* stream);
  static int join_linear(const EpiPartial& from, int parts, const EpiLinearInt8& e, void* stream);
};
// Sums of parts as whole numbers of 32 bits.
int launch_partial_int8(GemmTile tile, const GemmPlan& g, const EpiPartial& e, void* stream);
int norm_chunks(int rows, int cols, bool in_place);  // in_place: d_x is d_out or x
int launch_norm(const NormPlan& p, int dtype, void* stream);
int launch_norm_backward(const NormBackwardPlan& p, int dtype, void* stream);
int launch_quantize(const QuantizePlan& p, int dtype, void* stream);
int launch_dropout(const DropoutPlan& p, int dtype, void* stream);
// Element size 1, 2 or 4.
int launch_pack(const PackPlan& p, int element_bytes, void* stream);
int launch_join_stats(const JoinStatsPlan& p, void* stream);
int launch_grad_scale(const GradScalePlan& p, void* stream);

}  // namespace lsamp

#endif
