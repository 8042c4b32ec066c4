// lsamp_head_api.cpp — the C entry points of the hidden-state operators:
// their plans and launches.
#include "lsamp_head_plan.h"

using namespace lsamp;

namespace {

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
