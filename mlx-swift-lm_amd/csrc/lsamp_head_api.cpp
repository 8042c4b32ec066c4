// lsamp_head_api.cpp — the C entry points of the hidden-state operators:
// argument checks, the choice of tiles, pieces and parts, and the launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "lsamp_head.h"
#include "lsamp_internal.h"

using namespace lsamp;

namespace {

constexpr int32_t kMaxDim = 1 << 27;
// Columns of a matrix: a tile's rows lie within 32 bits of its first (256 rows of
// 16-bit elements, 128 of float32).
constexpr int32_t kMaxFeatures = 1 << 22;
constexpr int32_t kMaxLossRows = 1 << 23;  // (a work-group a row)
constexpr int64_t kAlign = 256;
// Work-groups of a launch: 512 threads each, below 2^32 threads in all.
constexpr int64_t kMaxBlocks = (int64_t)1 << 22;

struct OnDevice {
  int prev = -1;
  bool changed = false;
  explicit OnDevice(int dev) {
    if (hipGetDevice(&prev) == hipSuccess && prev != dev) changed = hipSetDevice(dev) == hipSuccess;
  }
  ~OnDevice() {
    if (changed) (void)hipSetDevice(prev);
  }
};

int element_bytes(int dtype) { return dtype == LSAMP_DTYPE_F32 ? 4 : 2; }
int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
int64_t ceil_div(int64_t v, int64_t a) { return (v + a - 1) / a; }

#define HEAD_OP(dtype, call)                                              \
  ((dtype) == LSAMP_DTYPE_F32    ? HeadOps<LSAMP_DTYPE_F32>::call         \
   : (dtype) == LSAMP_DTYPE_BF16 ? HeadOps<LSAMP_DTYPE_BF16>::call        \
                                 : HeadOps<LSAMP_DTYPE_F16>::call)

// Parts of the caller's workspace, in the order they are taken; with base NULL
// only their sizes are added up.
struct Arena {
  char* base;
  int64_t used = 0;
  explicit Arena(void* p) : base((char*)p) {}
  template <typename T = void>
  T* take(int64_t bytes) {
    T* p = (T*)(base ? base + used : nullptr);
    used += round_up(bytes, kAlign);
    return p;
  }
};

// Whether the tiled products read a matrix as it is: rows of whole aligned
// chunks, and a tile's rows within 32 bits of its first.
bool chunked(const void* p, int64_t ld, int32_t cols, int eb) {
  return (uintptr_t)p % 16 == 0 && ld * eb % 16 == 0 && (int64_t)cols * eb % 16 == 0 &&
         ld * eb <= ((int64_t)1 << 32) / 512;
}

// A matrix of the arguments, and what the products read: itself, or a copy in
// the workspace that is made before the first of them.
struct Operand {
  MatrixRef ref;
  bool chunked, packed;
  PackPlan pack;
};
Operand operand(const void* p, int64_t ld, int32_t rows, int32_t cols, int eb) {
  Operand o{};
  o.ref = MatrixRef{p, ld, rows, cols};
  o.chunked = chunked(p, ld, cols, eb);
  return o;
}
// Rows in the workspace: whole chunks, and 128-byte lines apart, since a slab of a
// row that lies across two lines reads both (2000 x 4097 x 4097 with its copies: 164
// us with rows 8,208 bytes apart, 128 with rows 8,320 apart).
int64_t row_chunks(int64_t cols, int eb) { return round_up(cols, 16 / eb); }
int64_t row_pitch(int64_t cols, int eb) { return round_up(cols, 128 / eb); }
// Lays the operand out, if it has to be.
MatrixRef packed(Arena& ws, Operand& o, int eb) {
  if (!o.chunked && !o.packed) {
    const int64_t pitch = row_pitch(o.ref.cols, eb);
    void* dst = ws.take((int64_t)o.ref.rows * pitch * eb);
    o.packed = true;
    o.pack = PackPlan{o.ref.p,    o.ref.ld,   dst, pitch, o.ref.rows,
                      o.ref.cols, (int32_t)row_chunks(o.ref.cols, eb)};
  }
  return o.packed ? MatrixRef{o.pack.dst, o.pack.dst_ld, o.pack.rows, o.pack.dst_cols} : o.ref;
}
int lay_out(const Operand& o, int eb, void* stream) {
  return o.packed ? launch_pack(o.pack, eb, stream) : 0;
}

// Tile shape and number of parts of the reduction for an m x n product over
// `slabs` 128-byte slabs, by the time that they take.  A CU holds 1, 2 or 4
// work-groups of the three shapes; a slab takes at least its barrier, its LDS
// reads and its products in turn, and at least the time of the products of all
// groups on the CU.  Measured in microseconds (16-bit elements): alone on a CU
// 1.5, 0.63 and 0.2 (304 x 2048 x 1536, 1024 x 4096 x 2048), in company 1.6, 0.46
// and 0.18 (8192 x 4096 x 4096); two or four slabs at a time alone 0.57 and 0.15.
// A tile ends with its epilogue's `bytes` an element at the CU's share of the
// memory rate, hidden behind other work-groups' products where a CU has some
// (151936 x 4096 gradients of few rows: 513 us on 256 x 256 tiles, 230 on 128 x
// 128).  A split reduction is another launch, and its sums' traffic.
struct Choice {
  GemmTile tile;
  int32_t parts;
  double us;
};
enum Rows { kChunked, kLooseSmall, kLooseAny };  // kLooseAny: under every epilogue
Choice choose(int64_t m, int64_t n, int64_t slabs, int dtype, double bytes, bool may_split,
              Rows rows = kChunked) {
  struct Shape {
    GemmTile tile, grouped, loose, loose_grouped;
    int resident;
    double exposed, fixed;
    struct {
      double alone, alone_grouped, busy;
    } us[2];  // 16-bit elements, float32
  };
  static const Shape kShapes[] = {
      {kTile256, kTile256, kTile256, kTile256, 1, 1.0, 2.0, {{1.5, 1.5, 1.6}, {1e30, 1e30, 1e30}}},
      {kTile128, kTile128x2, kLoose128, kLoose128, 2, 0.6, 1.0, {{0.63, 0.57, 0.46}, {0.95, 0.8, 0.8}}},
      {kTile64, kTile64x4, kLoose64, kLoose64x4, 4, 0.5, 0.5, {{0.2, 0.15, 0.18}, {0.5, 0.38, 0.38}}}};
  constexpr int kCus = 256;
  constexpr double kBytesPerUs = 5e6;  // of the device
  Choice best{rows == kChunked ? kTile64 : kLoose128, 1, 1e300};
  for (const Shape& s : kShapes) {
    if (rows != kChunked && s.tile == kTile256) continue;
    if (rows == kLooseAny && s.tile == kTile64) continue;
    const int64_t side = kTileSide[s.tile], tiles = ceil_div(m, side) * ceil_div(n, side);
    const auto& us_of = s.us[dtype == LSAMP_DTYPE_F32];
    for (int parts = 1; parts <= (may_split ? 64 : 1) && parts <= slabs; parts *= 2) {
      const int64_t each = ceil_div(tiles * parts, kCus), rounds = ceil_div(each, s.resident);
      const bool grouped = each == 1;
      const double per_slab = std::max((double)each * us_of.busy,
                                       (double)rounds * (grouped ? us_of.alone_grouped : us_of.alone));
      const double out = parts > 1 ? 4.0 : bytes;
      double us = per_slab * (double)ceil_div(slabs, parts) + (double)rounds * s.fixed +
                  (double)each * (double)(side * side) * out * s.exposed * kCus / kBytesPerUs;
      us = std::max(us, (double)parts * (double)m * (double)n * out / kBytesPerUs);
      if (parts > 1) us += 4.0 + (double)m * (double)n * ((double)parts * 4.0 + bytes) / kBytesPerUs;
      if (us < best.us)
        best = Choice{rows == kChunked ? (grouped ? s.grouped : s.tile)
                                       : (grouped ? s.loose_grouped : s.loose),
                      parts, us};
    }
  }
  return best;
}
// What laying a matrix out for the tiled products takes: a launch, and its bytes
// read and written.
double pack_us(int64_t rows, int64_t cols, int eb) {
  return 4.0 + (double)rows * (double)cols * eb * 2.0 / 4e6;
}
double pack_all(const Operand& a, const Operand& b, int eb) {
  double us = 0.0;
  for (const Operand* o : {&a, &b})
    if (!o->chunked && !o->packed) us += pack_us(o->ref.rows, o->ref.cols, eb);
  return us;
}
bool is_loose(const Choice& c) {
  return c.tile == kLoose128 || c.tile == kLoose64 || c.tile == kLoose64x4;
}
// For operands of which some are no chunks: loose tiles (about 1.4 times an
// aligned one's time), or any tile after `pack` microseconds of copies.
Choice choose_rows(int64_t m, int64_t n, int64_t slabs, int dtype, double bytes, double pack) {
  const Choice best = choose(m, n, slabs, dtype, bytes, true);
  if (pack == 0.0) return best;
  const Choice any = choose(m, n, slabs, dtype, bytes, true, kLooseSmall);
  return any.us * 1.4 < best.us + pack ? any : best;
}
// At most 64 rows are bound by reading the other operand, which the kernels of
// lsamp_skinny.h do without a detour: 64 columns a work-group where that leaves
// none of the device idle, else 16 (64 x 16384 x 4096: 31 us and 54; 64 x 4096 x
// 4096: 26 and 14; 8 x 4096 x 4096: 13 and 9).  They take any rows of the other
// operand, and of x up to kLooseRows.
constexpr int kLooseRows = 16;
Choice choose_skinny(int64_t m, int64_t n, bool whole_rows) {
  return Choice{whole_rows || n >= (m > kLooseRows ? 8192 : 16384) ? kSkinny64 : kSkinny16, 1, 0.0};
}

// `k`: elements of the reduction.  `slabs_per_part`: of an earlier plan whose parts
// these are added to.  (Parts of equal shares of a shorter reduction can be more:
// 680 slabs in 32 shares are 31 parts of 22, 668 are 32 of 21.)
GemmPlan plan_gemm(const Choice& c, const MatrixRef& a, const MatrixRef& b, int64_t m, int64_t n,
                   int64_t k, int eb, int32_t slabs_per_part = 0) {
  GemmPlan g{};
  g.a = a;
  g.b = b;
  const bool skinny = c.tile == kSkinny64 || c.tile == kSkinny16;
  g.tiles_m = skinny ? 1 : (int32_t)ceil_div(m, kTileSide[c.tile]);
  g.tiles_n = (int32_t)ceil_div(n, kTileSide[c.tile]);
  g.slabs = (int32_t)ceil_div(k, 128 / eb);
  g.slabs_per_part = slabs_per_part ? slabs_per_part : (int32_t)ceil_div(g.slabs, c.parts);
  g.parts = (int32_t)ceil_div(g.slabs, g.slabs_per_part);
  return g;
}
bool too_many(const GemmPlan& g) {
  return (int64_t)g.tiles_m * g.tiles_n * g.parts > kMaxBlocks;
}

// Outputs of more than half the last-level cache (256 MB) only push the operands
// out of it and are stored past it (a float32 `out` is not: 4096 x 2048 x 32000 504
// us, 481 in 16 bits): 8192 x 4096 x 4096 with kept pre-activations
// (201 MB) 287 us and 246, 4096 x 2048 x 32000 (262 MB) 490 and 458.  Smaller ones
// are found there by what reads them next: the head's gradients of 333 x 1000 x
// 40003 (80 MB) take 138 us, stored past it 152.
bool streams(int64_t bytes) { return bytes > (int64_t)128 << 20; }

int64_t slabs_of(int64_t k, int eb) { return ceil_div(k, 128 / eb); }

// A product into `out`: straight, or in parts through float32 sums.
EpiPartial take_partial(Arena& ws, int64_t m, int64_t n, int parts) {
  EpiPartial p{};
  p.m = (int32_t)m;
  p.n = (int32_t)n;
  p.ld = round_up(n, 4);
  p.part_stride = m * p.ld;
  p.out = ws.take<float>((int64_t)parts * p.part_stride * 4);
  return p;
}

lsamp_status device_error(int err) {
  return set_error(LSAMP_ERR_DEVICE, "kernel launch failed: %s", hipGetErrorString((hipError_t)err));
}

#define LSAMP_TRY(expr)                    \
  do {                                     \
    const int try_err = (expr);            \
    if (try_err) return device_error(try_err); \
  } while (0)

// --------------------------------------------------------------------- checks
lsamp_status check_dims(const char* what, int32_t v, int32_t most = kMaxFeatures) {
  if (v <= 0 || v > most)
    return set_error(LSAMP_ERR_SHAPE, "%s %d out of range [1, %d]", what, v, most);
  return LSAMP_OK;
}
lsamp_status check_dtype(int32_t dtype) {
  if (dtype < LSAMP_DTYPE_F32 || dtype > LSAMP_DTYPE_F16)
    return set_error(LSAMP_ERR_DTYPE, "dtype %d is not float32, bfloat16 or float16", dtype);
  return LSAMP_OK;
}
// A matrix of the arguments: present, its elements aligned, its rows apart.
lsamp_status check_matrix(const char* what, const void* p, int64_t ld, int32_t rows, int32_t cols,
                          int eb) {
  if (!p) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "%s is required", what);
  if ((uintptr_t)p % eb)
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "%s is not aligned to its elements", what);
  if (rows > 1 && ld < cols)
    return set_error(LSAMP_ERR_SHAPE, "%s stride %lld is below its %d columns", what, (long long)ld,
                     cols);
  if (ld < 0 || ld > ((int64_t)1 << 40))
    return set_error(LSAMP_ERR_SHAPE, "%s stride %lld out of range", what, (long long)ld);
  return LSAMP_OK;
}
// A vector (or a float output): present if required, aligned.
lsamp_status check_vector(const char* what, const void* p, int eb, bool required) {
  if (!p && required) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "%s is required", what);
  if ((uintptr_t)p % eb)
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "%s is not aligned to its elements", what);
  return LSAMP_OK;
}
lsamp_status check_activation(int32_t act, float softcap) {
  if (act < LSAMP_ACT_NONE || act > LSAMP_ACT_SOFTCAP)
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "activation %d is unknown", act);
  if (act == LSAMP_ACT_SOFTCAP && !(softcap > 0.f && std::isfinite(softcap)))
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "softcap %g must be positive and finite", softcap);
  return LSAMP_OK;
}
lsamp_status check_workspace(const void* p, int64_t have, int64_t need) {
  if (need == 0) return LSAMP_OK;
  if (!p || have < need)
    return set_error(LSAMP_ERR_CAPACITY, "the workspace holds %lld bytes, %lld are needed",
                     p ? (long long)have : 0LL, (long long)need);
  if ((uintptr_t)p % kAlign)
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "the workspace is not aligned to %lld bytes",
                     (long long)kAlign);
  return LSAMP_OK;
}
// (a one-row matrix may carry any stride: its rows are taken as dense)
int64_t stride_of(int64_t ld, int32_t rows, int32_t cols) { return rows > 1 ? ld : cols; }

#define LSAMP_CHECK(expr)                     \
  do {                                        \
    const lsamp_status check_st = (expr);     \
    if (check_st != LSAMP_OK) return check_st; \
  } while (0)

// ---------------------------------------------------------------------- linear
struct LinearPlan {
  Operand x, w;
  Choice choice;
  GemmPlan gemm;
  EpiPartial partial;
  EpiLinear epi;
  int64_t bytes;
};

lsamp_status plan_linear(const lsamp_linear_args* a, void* base, LinearPlan* out) {
  if (!a) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "args is NULL");
  LSAMP_CHECK(check_dims("rows", a->rows, kMaxDim));
  LSAMP_CHECK(check_dims("in_features", a->in_features));
  LSAMP_CHECK(check_dims("out_features", a->out_features));
  LSAMP_CHECK(check_dtype(a->dtype));
  if (a->out_dtype != a->dtype && a->out_dtype != LSAMP_DTYPE_F32)
    return set_error(LSAMP_ERR_DTYPE, "out_dtype %d must be the dtype %d or float32", a->out_dtype,
                     a->dtype);
  LSAMP_CHECK(check_activation(a->activation, a->softcap));
  const int eb = element_bytes(a->dtype), ob = element_bytes(a->out_dtype);
  const int32_t m = a->rows, n = a->out_features, k = a->in_features;
  LSAMP_CHECK(check_matrix("x", a->x, a->x_stride, m, k, eb));
  LSAMP_CHECK(check_matrix("weight", a->weight, a->weight_stride, n, k, eb));
  LSAMP_CHECK(check_matrix("out", a->out, a->out_stride, m, n, ob));
  LSAMP_CHECK(check_vector("bias", a->bias, eb, false));
  if (a->residual)
    LSAMP_CHECK(check_matrix("residual", a->residual, a->residual_stride, m, n, eb));
  if (a->pre) LSAMP_CHECK(check_matrix("pre", a->pre, a->pre_stride, m, n, 4));

  LinearPlan P{};
  Arena ws(base);
  P.x = operand(a->x, stride_of(a->x_stride, m, k), m, k, eb);
  P.w = operand(a->weight, stride_of(a->weight_stride, n, k), n, k, eb);
  MatrixRef x = P.x.ref, w = P.w.ref;
  if (m <= kSkinnyRows) {
    P.choice = choose_skinny(m, n, false);
    if (m > kLooseRows) x = packed(ws, P.x, eb);
  } else {
    P.choice = choose_rows(m, n, slabs_of(k, eb), a->dtype,
                           ob + (a->residual ? eb : 0) + (a->pre ? 4 : 0), pack_all(P.x, P.w, eb));
    if (!is_loose(P.choice)) {
      x = packed(ws, P.x, eb);
      w = packed(ws, P.w, eb);
    }
  }
  P.gemm = plan_gemm(P.choice, x, w, m, n, k, eb);
  if (too_many(P.gemm))
    return set_error(LSAMP_ERR_SHAPE, "%d rows of %d outputs are too many for one call", m, n);
  if (P.gemm.parts > 1) P.partial = take_partial(ws, m, n, P.gemm.parts);
  EpiLinear& e = P.epi;
  e.m = m;
  e.n = n;
  e.activation = a->activation;
  e.softcap = a->softcap;
  e.wide = a->out_dtype == LSAMP_DTYPE_F32;
  e.stream = streams((int64_t)m * n * (ob + (a->pre ? 4 : 0)));
  e.bias = a->bias;
  e.residual = a->residual;
  e.ld_residual = stride_of(a->residual_stride, m, n);
  e.out = a->out;
  e.ld_out = stride_of(a->out_stride, m, n);
  e.pre = a->pre;
  e.ld_pre = stride_of(a->pre_stride, m, n);
  P.bytes = ws.used;
  *out = P;
  return LSAMP_OK;
}

// ------------------------------------------------------------ linear, backward
// Column sums in chunks of rows, enough of them to fill the device.
void plan_col_sum(ColSumPlan& s, int32_t rows, int32_t cols) {
  s.rows = rows;
  s.cols = cols;
  const int64_t across = ceil_div(cols, 256);
  // (up to 128 rows one chunk: its sums need no second pass)
  int64_t chunks = rows <= 128 ? 1 : std::min(ceil_div(2048, across), ceil_div(rows, 16));
  s.rows_per_chunk = (int32_t)ceil_div(rows, chunks);
  s.chunks = (int32_t)ceil_div(rows, s.rows_per_chunk);
}

struct Product {  // one product of a backward pass
  GemmRoles roles;
  Choice choice;
  GemmPlan gemm;
  EpiPartial partial;
  EpiStore store;
};
// out = A B in `roles`; `k` reduction elements.
Product plan_product(Arena& ws, GemmRoles roles, Operand& a, Operand& b, int64_t m, int64_t n,
                     int64_t k, int dtype, void* out, int64_t ld) {
  const int eb = element_bytes(dtype);
  Product p{};
  p.roles = roles;
  p.choice = choose_rows(m, n, slabs_of(k, eb), dtype, eb, pack_all(a, b, eb));
  const bool loose = is_loose(p.choice);
  p.gemm = plan_gemm(p.choice, loose ? a.ref : packed(ws, a, eb), loose ? b.ref : packed(ws, b, eb),
                     m, n, k, eb);
  if (p.gemm.parts > 1) p.partial = take_partial(ws, m, n, p.gemm.parts);
  p.store.m = (int32_t)m;
  p.store.n = (int32_t)n;
  p.store.out = out;
  p.store.ld_out = ld;
  p.store.stream = streams(m * n * eb);
  return p;
}
int run_product(const Product& p, int dtype, void* stream) {
  if (p.gemm.parts == 1)
    return HEAD_OP(dtype, gemm_store(p.roles, p.choice.tile, p.gemm, p.store, stream));
  const int err =
      HEAD_OP(dtype, gemm_partial(p.roles, p.choice.tile, p.gemm, p.partial, stream));
  return err ? err : HEAD_OP(dtype, join_store(p.partial, p.gemm.parts, p.store, stream));
}

struct LinearBackwardPlan {
  Operand x, w, d;
  bool sum;  // the pass over d_out: d_bias, or dz (then `d`) for an activation
  ColSumPlan col;
  bool want_x, want_w;
  Product dx, dw;
  int64_t bytes;
};

lsamp_status plan_linear_backward(const lsamp_linear_backward_args* a, void* base,
                                  LinearBackwardPlan* out) {
  if (!a) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "args is NULL");
  LSAMP_CHECK(check_dims("rows", a->rows, kMaxDim));
  LSAMP_CHECK(check_dims("in_features", a->in_features));
  LSAMP_CHECK(check_dims("out_features", a->out_features));
  LSAMP_CHECK(check_dtype(a->dtype));
  LSAMP_CHECK(check_activation(a->activation, a->softcap));
  const int eb = element_bytes(a->dtype);
  const int32_t m = a->rows, n = a->out_features, k = a->in_features;
  const bool act = a->activation != LSAMP_ACT_NONE;
  if (!a->d_x && !a->d_weight && !a->d_bias)
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "no gradient is asked for");
  LSAMP_CHECK(check_matrix("d_out", a->d_out, a->d_out_stride, m, n, eb));
  if (act) LSAMP_CHECK(check_matrix("pre", a->pre, a->pre_stride, m, n, 4));
  if (a->d_x) {
    LSAMP_CHECK(check_matrix("weight", a->weight, a->weight_stride, n, k, eb));
    LSAMP_CHECK(check_matrix("d_x", a->d_x, a->d_x_stride, m, k, eb));
  }
  if (a->d_weight) {
    LSAMP_CHECK(check_matrix("x", a->x, a->x_stride, m, k, eb));
    LSAMP_CHECK(check_matrix("d_weight", a->d_weight, a->d_weight_stride, n, k, eb));
  }
  LSAMP_CHECK(check_vector("d_bias", a->d_bias, eb, false));

  LinearBackwardPlan P{};
  Arena ws(base);
  P.want_x = a->d_x != nullptr;
  P.want_w = a->d_weight != nullptr;
  const int64_t ld_d = stride_of(a->d_out_stride, m, n);
  if (act) {
    const int64_t pitch = row_pitch(n, eb);
    P.d = operand(ws.take((int64_t)m * pitch * eb), pitch, m, (int32_t)row_chunks(n, eb), eb);
    // (written by the pass below, after any copy: read as it lies, as copies themselves
    // are.  float32 rows of up to 16 MiB: a tile of them has at most 128, 2^31 bytes)
    P.d.chunked = true;
  } else {
    P.d = operand(a->d_out, ld_d, m, n, eb);
  }
  P.sum = act || a->d_bias;
  if (P.sum) {
    ColSumPlan& s = P.col;
    plan_col_sum(s, m, n);
    s.in = a->d_out;
    s.ld_in = ld_d;
    s.activation = a->activation;
    s.softcap = a->softcap;
    if (act) {
      s.pre = a->pre;
      s.ld_pre = stride_of(a->pre_stride, m, n);
      s.out = const_cast<void*>(P.d.ref.p);
      s.ld_out = P.d.ref.ld;
      s.out_cols = P.d.ref.cols;
    }
    if (a->d_bias) {
      s.ld_part = round_up(n, 4);
      if (s.chunks > 1)
        s.part = ws.take<float>((int64_t)s.chunks * s.ld_part * 4);
      else
        s.sums = a->d_bias;
    }
  }
  if (P.want_x) {
    P.w = operand(a->weight, stride_of(a->weight_stride, n, k), n, k, eb);
    P.dx = plan_product(ws, kRolesNN, P.d, P.w, m, k, n, a->dtype, a->d_x,
                        stride_of(a->d_x_stride, m, k));
  }
  if (P.want_w) {
    P.x = operand(a->x, stride_of(a->x_stride, m, k), m, k, eb);
    P.dw = plan_product(ws, kRolesTN, P.d, P.x, n, k, m, a->dtype, a->d_weight,
                        stride_of(a->d_weight_stride, n, k));
  }
  if ((P.want_x && too_many(P.dx.gemm)) || (P.want_w && too_many(P.dw.gemm)))
    return set_error(LSAMP_ERR_SHAPE, "%d x %d x %d is too large for one call", m, n, k);
  P.bytes = ws.used;
  *out = P;
  return LSAMP_OK;
}

// ------------------------------------------------------------------- head loss
// The checks that both directions share.
template <typename A>
lsamp_status check_head(const A* a) {
  if (!a) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "args is NULL");
  LSAMP_CHECK(check_dims("rows", a->rows, kMaxLossRows));
  LSAMP_CHECK(check_dims("hidden", a->hidden));
  LSAMP_CHECK(check_dims("vocab", a->vocab));
  LSAMP_CHECK(check_dtype(a->dtype));
  if (!(a->softcap >= 0.f && std::isfinite(a->softcap)))
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "softcap %g must be finite and not negative",
                     a->softcap);
  const int eb = element_bytes(a->dtype);
  LSAMP_CHECK(check_matrix("x", a->x, a->x_stride, a->rows, a->hidden, eb));
  LSAMP_CHECK(check_matrix("weight", a->weight, a->weight_stride, a->vocab, a->hidden, eb));
  LSAMP_CHECK(check_vector("bias", a->bias, eb, false));
  LSAMP_CHECK(check_vector("targets", a->targets, 4, true));
  LSAMP_CHECK(check_vector("lse", a->lse, 4, true));
  return LSAMP_OK;
}

// A piece of the vocabulary is a multiple of the largest tile's columns, so that
// the tiles of all pieces are those of the whole.
constexpr int64_t kPieceStep = 256;
int64_t piece_cols(int64_t vocab, int64_t most) {
  most = std::max(kPieceStep, most / kPieceStep * kPieceStep);
  const int64_t pieces = ceil_div(vocab, most);
  return std::min(round_up(ceil_div(vocab, pieces), kPieceStep), round_up(vocab, kPieceStep));
}
// The weight rows of a piece: themselves, or their copy at `packed`.
Operand weight_piece(const void* w, int64_t ld, int32_t first, int32_t rows, int32_t hidden, int eb,
                     void* packed) {
  const char* p = (const char*)w + (int64_t)first * ld * eb;
  Operand o{};
  if (!packed) {
    o.ref = MatrixRef{p, ld, rows, hidden};
    return o;
  }
  const int32_t wide = (int32_t)row_chunks(hidden, eb);
  const int64_t pitch = row_pitch(hidden, eb);
  o.packed = true;
  o.pack = PackPlan{p, ld, packed, pitch, rows, hidden, wide};
  o.ref = MatrixRef{packed, pitch, rows, wide};
  return o;
}

// Weight rows that are no chunks are read as they are up to so many rows of x,
// where that costs less than copying them (a copy moves 4 bytes an element, a
// loose product takes some 40% longer); backward, with three products, half.
constexpr int kLooseLossRows = 1024;
// The loss's epilogues as bytes an element: some ten instructions, and what the
// gradient's stores.
constexpr double kStatsBytes = 2.0, kGradBytes = 3.0;

struct LossPlan {
  Operand x;
  MatrixRef x_ref;
  Choice choice;
  int64_t piece;  // vocabulary columns at a time
  void* packed;
  EpiStats epi;
  JoinStatsPlan join;
  int64_t bytes;
};

lsamp_status plan_loss(const lsamp_head_loss_args* a, void* base, LossPlan* out) {
  LSAMP_CHECK(check_head(a));
  LSAMP_CHECK(check_vector("loss", a->loss, 4, true));
  LSAMP_CHECK(check_vector("row_flags", a->row_flags, 4, false));
  const int eb = element_bytes(a->dtype);
  const int32_t m = a->rows, v = a->vocab, k = a->hidden;
  LossPlan P{};
  Arena ws(base);
  const bool skinny = m <= kSkinnyRows;
  const int64_t ld_w = stride_of(a->weight_stride, v, k);
  const bool loose = !chunked(a->weight, ld_w, k, eb) && m <= kLooseLossRows;
  P.x = operand(a->x, stride_of(a->x_stride, m, k), m, k, eb);
  P.x_ref = m <= kLooseRows || (loose && !skinny) ? P.x.ref : packed(ws, P.x, eb);
  P.piece = round_up(v, kPieceStep);
  if (!loose && !chunked(a->weight, ld_w, k, eb)) {
    const int64_t row = row_pitch(k, eb) * eb;
    P.piece = piece_cols(v, ((int64_t)128 << 20) / row);
    P.packed = ws.take(std::min(P.piece, (int64_t)v) * row);
    if (!base) P.packed = (void*)1;  // (sizes only)
  }
  P.choice = skinny ? choose_skinny(m, v, true)
                    : choose(m, std::min(P.piece, (int64_t)v), slabs_of(k, eb), a->dtype, kStatsBytes,
                             false, loose ? kLooseAny : kChunked);
  const int64_t side = kTileSide[P.choice.tile];
  if (ceil_div(m, side) * ceil_div(P.piece, side) > kMaxBlocks)
    return set_error(LSAMP_ERR_SHAPE, "%d rows of %d logits are too many for one call", m, v);
  EpiStats& e = P.epi;
  e.m = m;
  e.blocks = (int32_t)ceil_div(v, side);
  e.softcap = a->softcap;
  e.bias = a->bias;
  e.targets = a->targets;
  e.part = ws.take<float>((int64_t)m * e.blocks * 8);
  e.target = ws.take<float>((int64_t)m * 4);
  P.join = JoinStatsPlan{m, e.blocks, v, e.part, e.target, a->targets, a->loss, a->lse, a->row_flags};
  P.bytes = ws.used;
  *out = P;
  return LSAMP_OK;
}

struct LossBackwardPlan {
  Operand x;
  MatrixRef x_ref;
  bool loose;  // weight rows and x are read as they are
  int64_t piece;
  void* packed;
  void* g;      // [rows, ld_g]: the gradient at a piece of the logits
  int64_t ld_g;
  float* scale;  // {scale, 1 / scale} of g
  Choice grad, dx, dw;
  EpiPartial dx_sum, dw_sum;  // float32 sums of d_x (all pieces), of a piece's d_weight
  int32_t dx_parts, dx_slabs_per_part;  // of the first piece, the longest
  bool dx_straight, dw_split;
  ColSumPlan col;  // d_bias: the join of the tiles' column sums
  int64_t bytes;
};

lsamp_status plan_loss_backward(const lsamp_head_loss_backward_args* a, void* base,
                                LossBackwardPlan* out) {
  LSAMP_CHECK(check_head(a));
  LSAMP_CHECK(check_vector("d_loss", a->d_loss, 4, true));
  const int eb = element_bytes(a->dtype);
  const int32_t m = a->rows, v = a->vocab, k = a->hidden;
  if (!a->d_x && !a->d_weight && !a->d_bias)
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "no gradient is asked for");
  if (a->d_x) LSAMP_CHECK(check_matrix("d_x", a->d_x, a->d_x_stride, m, k, eb));
  if (a->d_weight)
    LSAMP_CHECK(check_matrix("d_weight", a->d_weight, a->d_weight_stride, v, k, eb));
  LSAMP_CHECK(check_vector("d_bias", a->d_bias, eb, false));

  LossBackwardPlan P{};
  Arena ws(base);
  P.x = operand(a->x, stride_of(a->x_stride, m, k), m, k, eb);
  const int64_t ld_w = stride_of(a->weight_stride, v, k);
  P.loose = !chunked(a->weight, ld_w, k, eb) && m <= kLooseLossRows / 2;
  const Rows rows = P.loose ? kLooseAny : kChunked, rows2 = P.loose ? kLooseSmall : kChunked;
  P.x_ref = P.loose && m > kSkinnyRows ? P.x.ref : packed(ws, P.x, eb);
  // A piece's gradient stays in the 256 MB last-level cache between the pass
  // that writes it and the products that read it.
  P.piece = piece_cols(v, ((int64_t)128 << 20) / ((int64_t)m * eb));
  if (!P.loose && !chunked(a->weight, ld_w, k, eb)) {
    const int64_t row = row_pitch(k, eb) * eb;
    P.piece = std::min(P.piece, piece_cols(v, ((int64_t)128 << 20) / row));
    P.packed = ws.take(std::min(P.piece, (int64_t)v) * row);
    if (!base) P.packed = (void*)1;  // (sizes only)
  }
  const int64_t cols = std::min(P.piece, (int64_t)v);
  P.ld_g = round_up(cols, 64);
  P.g = ws.take((int64_t)m * P.ld_g * eb);
  P.scale = ws.take<float>(8);
  P.grad = m <= kSkinnyRows ? choose_skinny(m, cols, true)
                            : choose(m, cols, slabs_of(k, eb), a->dtype, kGradBytes, false, rows);
  const int64_t side = kTileSide[P.grad.tile];
  if (ceil_div(m, side) * ceil_div(cols, side) > kMaxBlocks)
    return set_error(LSAMP_ERR_SHAPE, "%d rows of %d logits are too many for one call", m, v);
  if (a->d_x) {
    // (the sums of all pieces are added in float32, unless there is one)
    P.dx = choose(m, k, slabs_of(cols, eb), a->dtype, cols == v ? eb : 8, true, rows2);
    const GemmPlan g = plan_gemm(P.dx, MatrixRef{}, MatrixRef{}, m, k, cols, eb);
    if (too_many(g)) return set_error(LSAMP_ERR_SHAPE, "%d x %d is too large for one call", m, k);
    P.dx_parts = g.parts;
    P.dx_slabs_per_part = g.slabs_per_part;
    P.dx_straight = g.parts == 1 && cols == v;
    if (!P.dx_straight) P.dx_sum = take_partial(ws, m, k, g.parts);
  }
  if (a->d_weight) {
    P.dw = choose(cols, k, slabs_of(m, eb), a->dtype, eb, true, rows2);
    const GemmPlan g = plan_gemm(P.dw, MatrixRef{}, MatrixRef{}, cols, k, m, eb);
    if (too_many(g)) return set_error(LSAMP_ERR_SHAPE, "%d x %d is too large for one call", v, k);
    P.dw_split = g.parts > 1;
    if (P.dw_split) P.dw_sum = take_partial(ws, cols, k, g.parts);
  }
  if (a->d_bias) {
    P.col.chunks = (int32_t)ceil_div(m, side) * kTileWavesM[P.grad.tile];
    P.col.ld_part = round_up(cols, 4);
    P.col.join_wide = P.col.chunks > 256;
    P.col.part = ws.take<float>((int64_t)P.col.chunks * P.col.ld_part * 4);
  }
  P.bytes = ws.used;
  *out = P;
  return LSAMP_OK;
}

int64_t needed(lsamp_status st, int64_t bytes) {
  if (st != LSAMP_OK) return st;
  clear_error();
  return bytes;
}

}  // namespace

int64_t lsamp_linear_workspace(const lsamp_linear_args* a) {
  LinearPlan P;
  const lsamp_status st = plan_linear(a, nullptr, &P);
  return needed(st, st == LSAMP_OK ? P.bytes : 0);
}

lsamp_status lsamp_linear(lsamp_context* ctx, const lsamp_linear_args* a, void* stream) {
  if (!ctx) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "context is NULL");
  LinearPlan P;
  LSAMP_CHECK(plan_linear(a, a ? a->workspace : nullptr, &P));
  LSAMP_CHECK(check_workspace(a->workspace, a->workspace_bytes, P.bytes));
  OnDevice guard(context_device(ctx));
  const int eb = element_bytes(a->dtype);
  LSAMP_TRY(lay_out(P.x, eb, stream));
  LSAMP_TRY(lay_out(P.w, eb, stream));
  if (P.gemm.parts == 1) {
    LSAMP_TRY(HEAD_OP(a->dtype, gemm_linear(P.choice.tile, P.gemm, P.epi, stream)));
  } else {
    LSAMP_TRY(HEAD_OP(a->dtype, gemm_partial(kRolesNT, P.choice.tile, P.gemm, P.partial, stream)));
    LSAMP_TRY(HEAD_OP(a->dtype, join_linear(P.partial, P.gemm.parts, P.epi, stream)));
  }
  return clear_error();
}

int64_t lsamp_linear_backward_workspace(const lsamp_linear_backward_args* a) {
  LinearBackwardPlan P;
  const lsamp_status st = plan_linear_backward(a, nullptr, &P);
  return needed(st, st == LSAMP_OK ? P.bytes : 0);
}

lsamp_status lsamp_linear_backward(lsamp_context* ctx, const lsamp_linear_backward_args* a,
                                   void* stream) {
  if (!ctx) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "context is NULL");
  LinearBackwardPlan P;
  LSAMP_CHECK(plan_linear_backward(a, a ? a->workspace : nullptr, &P));
  LSAMP_CHECK(check_workspace(a->workspace, a->workspace_bytes, P.bytes));
  OnDevice guard(context_device(ctx));
  const int eb = element_bytes(a->dtype);
  LSAMP_TRY(lay_out(P.d, eb, stream));
  if (P.sum) LSAMP_TRY(HEAD_OP(a->dtype, col_sum(P.col, stream)));
  if (P.col.part) LSAMP_TRY(HEAD_OP(a->dtype, col_sum_join(P.col, a->d_bias, nullptr, stream)));
  if (P.want_x) {
    LSAMP_TRY(lay_out(P.w, eb, stream));
    LSAMP_TRY(run_product(P.dx, a->dtype, stream));
  }
  if (P.want_w) {
    LSAMP_TRY(lay_out(P.x, eb, stream));
    LSAMP_TRY(run_product(P.dw, a->dtype, stream));
  }
  return clear_error();
}

int64_t lsamp_head_loss_workspace(const lsamp_head_loss_args* a) {
  LossPlan P;
  const lsamp_status st = plan_loss(a, nullptr, &P);
  return needed(st, st == LSAMP_OK ? P.bytes : 0);
}

lsamp_status lsamp_head_loss(lsamp_context* ctx, const lsamp_head_loss_args* a, void* stream) {
  if (!ctx) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "context is NULL");
  LossPlan P;
  LSAMP_CHECK(plan_loss(a, a ? a->workspace : nullptr, &P));
  LSAMP_CHECK(check_workspace(a->workspace, a->workspace_bytes, P.bytes));
  OnDevice guard(context_device(ctx));
  const int eb = element_bytes(a->dtype);
  const int32_t v = a->vocab, k = a->hidden;
  LSAMP_TRY(lay_out(P.x, eb, stream));
  for (int64_t first = 0; first < v; first += P.piece) {
    const int32_t n = (int32_t)std::min(P.piece, v - first);
    const Operand w = weight_piece(a->weight, stride_of(a->weight_stride, v, k), (int32_t)first, n,
                                   k, eb, P.packed);
    LSAMP_TRY(lay_out(w, eb, stream));
    EpiStats e = P.epi;
    e.n = n;
    e.first_col = (int32_t)first;
    e.first_block = (int32_t)(first / kTileSide[P.choice.tile]);
    const GemmPlan g = plan_gemm(P.choice, P.x_ref, w.ref, a->rows, n, k, eb);
    LSAMP_TRY(HEAD_OP(a->dtype, gemm_stats(P.choice.tile, g, e, stream)));
  }
  LSAMP_TRY(launch_join_stats(P.join, stream));
  return clear_error();
}

int64_t lsamp_head_loss_backward_workspace(const lsamp_head_loss_backward_args* a) {
  LossBackwardPlan P;
  const lsamp_status st = plan_loss_backward(a, nullptr, &P);
  return needed(st, st == LSAMP_OK ? P.bytes : 0);
}

lsamp_status lsamp_head_loss_backward(lsamp_context* ctx, const lsamp_head_loss_backward_args* a,
                                      void* stream) {
  if (!ctx) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "context is NULL");
  LossBackwardPlan P;
  LSAMP_CHECK(plan_loss_backward(a, a ? a->workspace : nullptr, &P));
  LSAMP_CHECK(check_workspace(a->workspace, a->workspace_bytes, P.bytes));
  OnDevice guard(context_device(ctx));
  const int eb = element_bytes(a->dtype);
  const int32_t m = a->rows, v = a->vocab, k = a->hidden;
  const float* inverse = P.scale + 1;
  LSAMP_TRY(lay_out(P.x, eb, stream));
  LSAMP_TRY(launch_grad_scale(
      GradScalePlan{m, v, a->dtype == LSAMP_DTYPE_F32, a->d_loss, a->lse, a->targets, P.scale},
      stream));
  EpiStore dx{};
  dx.m = m;
  dx.n = k;
  dx.out = a->d_x;
  dx.ld_out = stride_of(a->d_x_stride, m, k);
  dx.scale = inverse;
  dx.stream = streams((int64_t)m * k * eb);
  for (int64_t first = 0; first < v; first += P.piece) {
    const int32_t n = (int32_t)std::min(P.piece, v - first);
    const Operand w = weight_piece(a->weight, stride_of(a->weight_stride, v, k), (int32_t)first, n,
                                   k, eb, P.packed);
    LSAMP_TRY(lay_out(w, eb, stream));
    EpiGrad e{};
    e.m = m;
    e.n = n;
    e.n_pad = (int32_t)round_up(n, 16 / eb);
    e.first_col = (int32_t)first;
    e.softcap = a->softcap;
    e.bias = a->bias;
    e.targets = a->targets;
    e.vocab = v;
    e.lse = a->lse;
    e.d_loss = a->d_loss;
    e.scale = P.scale;
    e.out = P.g;
    e.ld_out = P.ld_g;
    e.sums = P.col.part;
    e.ld_sums = P.col.ld_part;
    LSAMP_TRY(HEAD_OP(a->dtype, gemm_grad(P.grad.tile,
                                          plan_gemm(P.grad, P.x_ref, w.ref, m, n, k, eb), e, stream)));
    const MatrixRef g{P.g, P.ld_g, m, e.n_pad};
    if (a->d_x) {
      const GemmPlan plan = plan_gemm(P.dx, g, w.ref, m, k, n, eb, P.dx_slabs_per_part);
      if (P.dx_straight) {
        LSAMP_TRY(HEAD_OP(a->dtype, gemm_store(kRolesNN, P.dx.tile, plan, dx, stream)));
      } else {
        EpiPartial sum = P.dx_sum;
        sum.accumulate = first > 0;
        LSAMP_TRY(HEAD_OP(a->dtype, gemm_partial(kRolesNN, P.dx.tile, plan, sum, stream)));
      }
    }
    if (a->d_weight) {
      EpiStore dw{};
      dw.m = n;
      dw.n = k;
      dw.ld_out = stride_of(a->d_weight_stride, v, k);
      dw.out = (char*)a->d_weight + first * dw.ld_out * eb;
      dw.scale = inverse;
      dw.stream = streams((int64_t)v * k * eb);
      const GemmPlan plan = plan_gemm(P.dw, g, P.x_ref, n, k, m, eb);
      if (!P.dw_split) {
        LSAMP_TRY(HEAD_OP(a->dtype, gemm_store(kRolesTN, P.dw.tile, plan, dw, stream)));
      } else {
        EpiPartial sum = P.dw_sum;
        sum.m = n;
        LSAMP_TRY(HEAD_OP(a->dtype, gemm_partial(kRolesTN, P.dw.tile, plan, sum, stream)));
        LSAMP_TRY(HEAD_OP(a->dtype, join_store(sum, plan.parts, dw, stream)));
      }
    }
    if (a->d_bias) {
      ColSumPlan s = P.col;
      s.cols = n;
      LSAMP_TRY(HEAD_OP(a->dtype, col_sum_join(s, (char*)a->d_bias + first * eb, inverse, stream)));
    }
  }
  if (a->d_x && !P.dx_straight)
    LSAMP_TRY(HEAD_OP(a->dtype, join_store(P.dx_sum, P.dx_parts, dx, stream)));
  return clear_error();
}

lsamp_status lsamp_dropout(lsamp_context* ctx, const lsamp_dropout_args* a, void* stream) {
  if (!ctx) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "context is NULL");
  if (!a) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "args is NULL");
  LSAMP_CHECK(check_dims("rows", a->rows, kMaxDim));
  LSAMP_CHECK(check_dims("cols", a->cols, kMaxDim));
  LSAMP_CHECK(check_dtype(a->dtype));
  if (!(a->p >= 0.f && a->p <= 1.f))
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "p %g out of range [0, 1]", a->p);
  const int eb = element_bytes(a->dtype);
  LSAMP_CHECK(check_matrix("x", a->x, a->x_stride, a->rows, a->cols, eb));
  LSAMP_CHECK(check_matrix("out", a->out, a->out_stride, a->rows, a->cols, eb));
  if (a->residual)
    LSAMP_CHECK(check_matrix("residual", a->residual, a->residual_stride, a->rows, a->cols, eb));
  LSAMP_CHECK(check_vector("step", a->step, 8, false));
  DropoutPlan P{};
  P.rows = a->rows;
  P.cols = a->cols;
  P.cut = (uint32_t)std::lrint((double)a->p * 65536.0);
  P.scale = P.cut == 65536u ? 0.f : (float)(65536.0 / (65536.0 - (double)P.cut));
  P.key = a->key;
  P.offset = a->offset;
  P.step = a->step;
  P.x = a->x;
  P.ld_x = stride_of(a->x_stride, a->rows, a->cols);
  P.residual = a->residual;
  P.ld_residual = stride_of(a->residual_stride, a->rows, a->cols);
  P.out = a->out;
  P.ld_out = stride_of(a->out_stride, a->rows, a->cols);
  OnDevice guard(context_device(ctx));
  LSAMP_TRY(launch_dropout(P, a->dtype, stream));
  return clear_error();
}
