// lsamp_head_plan.h — what the C entry points of the hidden-state operators share:
// argument checks, the parts of a workspace, and the choice of tiles, pieces and
// parts of a product.  Host code, included by each file of entry points.
#ifndef LSAMP_HEAD_PLAN_H
#define LSAMP_HEAD_PLAN_H

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "lsamp_head.h"
#include "lsamp_internal.h"

namespace lsamp {
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
// Lays the operand out, if it has to be; `rows_of`: in rows of so many bytes, zeros
// behind their ends, also where its own are chunks.
MatrixRef packed(Arena& ws, Operand& o, int eb, int64_t rows_of = 0) {
  if ((!o.chunked || rows_of) && !o.packed) {
    const int64_t pitch = rows_of ? round_up(o.ref.cols, rows_of / eb) : row_pitch(o.ref.cols, eb);
    void* dst = ws.take((int64_t)o.ref.rows * pitch * eb);
    o.packed = true;
    o.pack = PackPlan{o.ref.p,    o.ref.ld,   dst, pitch, o.ref.rows,
                      o.ref.cols, (int32_t)(rows_of ? pitch : row_chunks(o.ref.cols, eb))};
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
// `batch`: so many products in one launch; `symmetric`: the tiles right of the diagonal.
Choice choose(int64_t m, int64_t n, int64_t slabs, int dtype, double bytes, bool may_split,
              Rows rows = kChunked, int64_t batch = 1, bool symmetric = false) {
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
    const int64_t side = kTileSide[s.tile], across = ceil_div(n, side);
    const int64_t tiles = batch * (symmetric ? across * (across + 1) / 2 : ceil_div(m, side) * across);
    const auto& us_of = s.us[dtype == LSAMP_DTYPE_F32];
    for (int parts = 1; parts <= (may_split ? 64 : 1) && parts <= slabs; parts *= 2) {
      const int64_t each = ceil_div(tiles * parts, kCus), rounds = ceil_div(each, s.resident);
      const bool grouped = each == 1;
      const double per_slab = std::max((double)each * us_of.busy,
                                       (double)rounds * (grouped ? us_of.alone_grouped : us_of.alone));
      const double out = parts > 1 ? 4.0 : bytes;
      double us = per_slab * (double)ceil_div(slabs, parts) + (double)rounds * s.fixed +
                  (double)each * (double)(side * side) * out * s.exposed * kCus / kBytesPerUs;
      us = std::max(us, (double)(parts * batch) * (double)m * (double)n * out / kBytesPerUs);
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
// aligned one's time; `loose128`: the large one's), or any tile after `pack` microseconds
// of copies.
Choice choose_rows(int64_t m, int64_t n, int64_t slabs, int dtype, double bytes, double pack,
                   double loose128 = 1.4) {
  const Choice best = choose(m, n, slabs, dtype, bytes, true);
  if (pack == 0.0) return best;
  const Choice any = choose(m, n, slabs, dtype, bytes, true, kLooseSmall);
  return any.us * (any.tile == kLoose128 ? loose128 : 1.4) < best.us + pack ? any : best;
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

int64_t needed(lsamp_status st, int64_t bytes) {
  if (st != LSAMP_OK) return st;
  clear_error();
  return bytes;
}

}  // namespace
}  // namespace lsamp

#endif
