// lsamp_blocks_api.cpp — the C entry points of a block's other operators: layer
// norm and its gradients, rows of 8-bit integers and their products, and the
// orthogonalised update.
#include "lsamp_head_plan.h"
#include "lsamp_orth.h"

using namespace lsamp;

namespace {

constexpr int32_t kMaxInt8Features = (1 << 17) - 1;  // (2^14 k below 2^31)
constexpr int64_t kKeptBytes = 128 << 10, kKeptRow = 256;  // x in LDS (ResidentPlan)

lsamp_status check_positive(const char* what, float v) {
  if (!(v > 0.f && std::isfinite(v)))
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "%s %g must be positive and finite", what, v);
  return LSAMP_OK;
}

// ------------------------------------------------------------------ layer norm
// Whether a result is stored past the last-level cache (256 MB), which cannot hold it:
// 32768 x 4096 bf16 (268 MB) forward 110 us through it, 89 past it, and with a linear
// block and all gradients 1020 and 1005; 16384 x 4096 is 45 and 44 alone, but 565 and 577
// with what reads it next.
bool past_cache(int64_t bytes) { return bytes >= (int64_t)256 << 20; }

lsamp_status plan_norm(const lsamp_layer_norm_args* a, NormPlan* out) {
  if (!a) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "args is NULL");
  LSAMP_CHECK(check_dims("rows", a->rows, kMaxDim));
  LSAMP_CHECK(check_dims("cols", a->cols));
  LSAMP_CHECK(check_dtype(a->dtype));
  LSAMP_CHECK(check_positive("eps", a->eps));
  const int eb = element_bytes(a->dtype);
  LSAMP_CHECK(check_matrix("x", a->x, a->x_stride, a->rows, a->cols, eb));
  LSAMP_CHECK(check_matrix("out", a->out, a->out_stride, a->rows, a->cols, eb));
  LSAMP_CHECK(check_vector("weight", a->weight, eb, false));
  LSAMP_CHECK(check_vector("bias", a->bias, eb, false));
  LSAMP_CHECK(check_vector("mean", a->mean, 4, false));
  LSAMP_CHECK(check_vector("rstd", a->rstd, 4, false));
  *out = NormPlan{a->rows,   a->cols, past_cache((int64_t)a->rows * a->cols * eb), a->eps,
                  a->x,      stride_of(a->x_stride, a->rows, a->cols),
                  a->weight, a->bias,
                  a->out,    stride_of(a->out_stride, a->rows, a->cols),
                  a->mean,   a->rstd};
  return LSAMP_OK;
}

lsamp_status plan_norm_backward(const lsamp_layer_norm_backward_args* a, void* base,
                                NormBackwardPlan* out, int64_t* bytes) {
  if (!a) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "args is NULL");
  LSAMP_CHECK(check_dims("rows", a->rows, kMaxDim));
  LSAMP_CHECK(check_dims("cols", a->cols));
  LSAMP_CHECK(check_dtype(a->dtype));
  const int eb = element_bytes(a->dtype);
  const int32_t m = a->rows, n = a->cols;
  if (!a->d_x && !a->d_weight && !a->d_bias)
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "no gradient is asked for");
  LSAMP_CHECK(check_matrix("x", a->x, a->x_stride, m, n, eb));
  LSAMP_CHECK(check_matrix("d_out", a->d_out, a->d_out_stride, m, n, eb));
  LSAMP_CHECK(check_vector("weight", a->weight, eb, false));
  LSAMP_CHECK(check_vector("mean", a->mean, 4, true));
  LSAMP_CHECK(check_vector("rstd", a->rstd, 4, true));
  if (a->residual && !a->d_x)
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "a residual without d_x to add it to");
  if (a->residual)
    LSAMP_CHECK(check_matrix("residual", a->residual, a->residual_stride, m, n, eb));
  if (a->d_x) LSAMP_CHECK(check_matrix("d_x", a->d_x, a->d_x_stride, m, n, eb));
  LSAMP_CHECK(check_vector("d_weight", a->d_weight, eb, false));
  LSAMP_CHECK(check_vector("d_bias", a->d_bias, eb, false));
  NormBackwardPlan P{};
  Arena ws(base);
  P.rows = m;
  P.cols = n;
  P.x = a->x;
  P.ld_x = stride_of(a->x_stride, m, n);
  P.weight = a->weight;
  P.mean = a->mean;
  P.rstd = a->rstd;
  P.d_out = a->d_out;
  P.ld_d = stride_of(a->d_out_stride, m, n);
  P.residual = a->residual;
  P.ld_residual = stride_of(a->residual_stride, m, n);
  P.stream = past_cache((int64_t)m * n * eb);
  P.d_x = a->d_x;
  P.ld_dx = stride_of(a->d_x_stride, m, n);
  P.d_weight = a->d_weight;
  P.d_bias = a->d_bias;
  if (a->d_weight || a->d_bias) {
    P.chunks = norm_chunks(m, n, a->d_x && (a->d_x == a->d_out || a->d_x == a->x));
    P.ld_part = round_up(n, 8);
    if (P.chunks) P.part = ws.take<float>((int64_t)P.chunks * 2 * P.ld_part * 4);
  }
  *out = P;
  *bytes = ws.used;
  return LSAMP_OK;
}

// ------------------------------------------------------------- 8-bit integers
lsamp_status check_quantized(const char* what, const void* p, int64_t ld, int32_t rows, int32_t cols) {
  return check_matrix(what, p, ld, rows, cols, 1);
}

struct LinearInt8Plan {
  bool quantize, kept;
  ResidentPlan resident;  // (kept)
  QuantizePlan quant;
  Operand x, w;
  Choice choice;
  GemmPlan gemm;
  EpiPartial partial;
  EpiLinearInt8 epi;
  int64_t bytes;
};

lsamp_status plan_linear_int8(const lsamp_linear_int8_args* a, void* base, LinearInt8Plan* out) {
  if (!a) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "args is NULL");
  LSAMP_CHECK(check_dims("rows", a->rows, kMaxDim));
  LSAMP_CHECK(check_dims("in_features", a->in_features, kMaxInt8Features));
  LSAMP_CHECK(check_dims("out_features", a->out_features));
  LSAMP_CHECK(check_dtype(a->dtype));
  if (a->out_dtype != a->dtype && a->out_dtype != LSAMP_DTYPE_F32)
    return set_error(LSAMP_ERR_DTYPE, "out_dtype %d must be the dtype %d or float32", a->out_dtype,
                     a->dtype);
  LSAMP_CHECK(check_activation(a->activation, a->softcap));
  const int eb = element_bytes(a->dtype), ob = element_bytes(a->out_dtype);
  const int32_t m = a->rows, n = a->out_features, k = a->in_features;
  const bool given = a->x_scale != nullptr;
  LSAMP_CHECK(check_matrix("x", a->x, a->x_stride, m, k, given ? 1 : eb));
  LSAMP_CHECK(check_vector("x_scale", a->x_scale, 4, false));
  LSAMP_CHECK(check_quantized("weight", a->weight, a->weight_stride, n, k));
  LSAMP_CHECK(check_vector("weight_scale", a->weight_scale, 4, true));
  LSAMP_CHECK(check_matrix("out", a->out, a->out_stride, m, n, ob));
  LSAMP_CHECK(check_vector("bias", a->bias, eb, false));
  if (a->residual)
    LSAMP_CHECK(check_matrix("residual", a->residual, a->residual_stride, m, n, eb));

  LinearInt8Plan P{};
  Arena ws(base);
  const int64_t ld_x = stride_of(a->x_stride, m, k);
  const float* x_scale = a->x_scale;
  const int64_t kept_bytes = m * round_up(k, kKeptRow);
  P.kept = m <= kSkinnyRows && k >= 16 && kept_bytes <= kKeptBytes;
  // (two rows of 2048, to 2048: quantised by every work-group 5.3 us, by a launch of its own
  // 6.1; three 6.2, four 7.1)
  const bool fused = P.kept && !given && m <= 2 && m * (int64_t)k <= 8192;
  if (given || fused) {
    P.x = operand(a->x, ld_x, m, k, given ? 1 : eb);
  } else {
    // (rows of whole chunks, or as they are kept, zeros behind their ends)
    const int64_t pitch = P.kept ? round_up(k, kKeptRow) : row_pitch(k, 1);
    const int32_t wide = P.kept ? (int32_t)pitch : (int32_t)row_chunks(k, 1);
    int8_t* const q = ws.take<int8_t>((int64_t)m * pitch);
    float* const s = ws.take<float>((int64_t)m * 4);
    P.quantize = true;
    P.quant = QuantizePlan{m, k, wide, a->x, ld_x, q, pitch, s};
    P.x.ref = MatrixRef{q, pitch, m, wide};
    P.x.chunked = true;
    x_scale = s;
  }
  P.w = operand(a->weight, stride_of(a->weight_stride, n, k), n, k, 1);
  MatrixRef x = P.x.ref, w = P.w.ref;
  if (P.kept) {
    if (given && !(P.x.chunked && k % kKeptRow == 0)) x = packed(ws, P.x, 1, kKeptRow);
    ResidentPlan& g = P.resident;
    g = ResidentPlan{m, k, 0, 0, fused, x.p, x.ld, w.p, w.ld};
    // (a work-group a CU, of little LDS two; waves share blocks that are fewer than they: one
    // row over 16,384 columns of 4096 16 us, 1,024 work-groups of a block each 22)
    const int64_t most = kept_bytes <= 16 << 10 ? 512 : 256, blocks = ceil_div(n, 16);
    g.shared = blocks < 8 * most;
    g.groups = (int32_t)std::min(most, g.shared ? blocks : ceil_div(blocks, 8));
  } else if (m <= kSkinnyRows) {
    P.choice = choose_skinny(m, n, false);
    if (m > kLooseRows) x = packed(ws, P.x, 1);
  } else {
    // (an instruction's slab of bytes takes what one of 16-bit elements does.  A loose 128 x
    // 128 tile, every chunk of which may end its row, takes over twice an aligned one's, and
    // copies are cheaper than pack_us has them: 3.2 keeps it where W is large beside the
    // products.  So and copied: 301 x 1537 x 32003 92 us and 56, 700 x 1537 x 8195 47 and
    // 35, 73 x 24997 x 3643 90 and 58; 100 x 300 x 60001 21 and 39, 108 x 933 x 27106 32 and 35)
    P.choice = choose_rows(m, n, slabs_of(k, 1), LSAMP_DTYPE_BF16, ob + (a->residual ? eb : 0),
                           pack_all(P.x, P.w, 1), 3.2);
    if (!is_loose(P.choice)) {
      x = packed(ws, P.x, 1);
      w = packed(ws, P.w, 1);
    }
  }
  if (!P.kept) {
    P.gemm = plan_gemm(P.choice, x, w, m, n, k, 1);
    if (too_many(P.gemm))
      return set_error(LSAMP_ERR_SHAPE, "%d rows of %d outputs are too many for one call", m, n);
    if (P.gemm.parts > 1) P.partial = take_partial(ws, m, n, P.gemm.parts);
  }
  EpiLinearInt8& e = P.epi;
  e.m = m;
  e.n = n;
  e.activation = a->activation;
  e.softcap = a->softcap;
  e.wide = a->out_dtype == LSAMP_DTYPE_F32;
  e.stream = streams((int64_t)m * n * ob);
  e.bias = a->bias;
  e.residual = a->residual;
  e.ld_residual = stride_of(a->residual_stride, m, n);
  e.out = a->out;
  e.ld_out = stride_of(a->out_stride, m, n);
  e.x_scale = x_scale;
  e.w_scale = a->weight_scale;
  P.bytes = ws.used;
  *out = P;
  return LSAMP_OK;
}

#define INT8_OP(dtype, call)                                              \
  ((dtype) == LSAMP_DTYPE_F32    ? Int8Ops<LSAMP_DTYPE_F32>::call         \
   : (dtype) == LSAMP_DTYPE_BF16 ? Int8Ops<LSAMP_DTYPE_BF16>::call        \
                                 : Int8Ops<LSAMP_DTYPE_F16>::call)

// --------------------------------------------------------- orthogonalised update
// What the steps' matrices hold at most: singular values start at most at 1, and a
// step takes s to |a s + b s^3 + c s^5|.  The largest |B| is that of b t + c t^2 over
// the squares t.
constexpr double kMostValue = 8.0, kMostPoly = 128.0;
constexpr int kMaxSteps = 64;
lsamp_status check_steps(const float* coefficients, int32_t steps) {
  if (steps < 1 || steps > kMaxSteps)
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "steps %d out of range [1, %d]", steps, kMaxSteps);
  if (!coefficients) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "coefficients is required");
  double top = 1.0;
  for (int i = 0; i < steps; ++i) {
    const double a = coefficients[3 * i], b = coefficients[3 * i + 1], c = coefficients[3 * i + 2];
    const auto p = [&](double t) { return std::sqrt(t) * std::fabs(a + b * t + c * t * t); };
    const auto q = [&](double t) { return std::fabs(b * t + c * t * t); };
    const double end = top * top;
    double most = p(end), poly = q(end);
    const auto at = [&](double t) {  // a place where a slope may be 0, if it is one
      if (!(t > 0.0 && t < end)) return;
      most = std::max(most, p(t));
      poly = std::max(poly, q(t));
    };
    // (the roots of a + 3 b t + 5 c t^2 without a difference of near values, which a small c
    // would lose one to; 0 or none of them where c is 0)
    const double d = 9.0 * b * b - 20.0 * a * c;
    if (d >= 0.0) {
      const double sum = -0.5 * (3.0 * b + std::copysign(std::sqrt(d), b));
      at(sum / (5.0 * c));
      at(a / sum);
    }
    at(-b / (2.0 * c));
    if (!(most <= kMostValue && poly <= kMostPoly))
      return set_error(LSAMP_ERR_INVALID_ARGUMENT,
                       "coefficients of step %d take singular values of up to %g to %g", i, top, most);
    top = most;
  }
  return LSAMP_OK;
}

struct OrthPlan {
  bool wide, tall;
  OrthStart start;
  Choice gram, poly, update;
  BatchPlan g_gram, g_poly, g_update;  // (of the first step: X is in the first buffer)
  void* x[2][2];                       // [buffer][part]
  EpiSymmetric e_gram, e_poly;
  EpiOrthUpdate e_update;
  int64_t bytes;
};

// The tile shape for `batch` products of m x n over `slabs` slabs, one round of the
// device after the other (see choose).  192 x 192 tiles, 0.95 us a slab, are for symmetric
// products that they spread over the device (4096: 253 tiles).
// A launch of few tiles is bound by what a CU loads, some 70 GB/s: 32 x 32 tiles, where
// there is a CU for each, have half the bytes of 64 x 64 ones (`rows_out`: both operands
// have rows along the output; the A of four 256 x 256 float32
// ones 7.8 us and 5.4).
Choice choose_batch(int64_t m, int64_t n, int64_t slabs, double bytes, int64_t batch, bool symmetric,
                    bool rows_out) {
  const int64_t fine = ceil_div(n, kTileSide[kTile32x8]);
  if (rows_out && batch * (symmetric ? fine * (fine + 1) / 2 : ceil_div(m, kTileSide[kTile32x8]) * fine) <= 256)
    return Choice{kTile32x8, 1, 0.0};
  Choice best = choose(m, n, slabs, LSAMP_DTYPE_F16, bytes, false, kChunked, batch, symmetric);
  if (symmetric) {
    const int64_t across = ceil_div(n, kTileSide[kTile192]);
    const double rounds = (double)ceil_div(batch * (across * (across + 1) / 2), 256);
    const double us = rounds * (0.95 * (double)slabs + 2.0 + 192.0 * 192.0 * bytes * 256.0 / 5e6);
    if (us < best.us) best = Choice{kTile192, 1, us};
  }
  return best;
}

lsamp_status plan_orth(const lsamp_orthogonalize_args* a, void* base, OrthPlan* out) {
  if (!a) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "args is NULL");
  LSAMP_CHECK(check_dims("batch", a->batch, 65535));
  LSAMP_CHECK(check_dims("rows", a->rows));
  LSAMP_CHECK(check_dims("cols", a->cols));
  LSAMP_CHECK(check_dtype(a->in_dtype));
  LSAMP_CHECK(check_dtype(a->out_dtype));
  LSAMP_CHECK(check_positive("eps", a->eps));
  if (!std::isfinite(a->scale) || !std::isfinite(a->keep))
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "scale %g and keep %g must be finite", a->scale,
                     a->keep);
  if (a->fast != 0 && a->fast != 1)
    return set_error(LSAMP_ERR_INVALID_ARGUMENT, "fast %d must be 0 or 1", a->fast);
  if (a->fast && a->out_dtype != LSAMP_DTYPE_BF16)
    return set_error(LSAMP_ERR_DTYPE, "fast products are for a bfloat16 out, not dtype %d",
                     a->out_dtype);
  LSAMP_CHECK(check_steps(a->coefficients, a->steps));
  const int ib = element_bytes(a->in_dtype), ob = element_bytes(a->out_dtype);
  const int32_t batch = a->batch, m = a->rows, n = a->cols;
  LSAMP_CHECK(check_matrix("x", a->x, a->x_stride, m, n, ib));
  LSAMP_CHECK(check_matrix("out", a->out, a->out_stride, m, n, ob));
  if (a->base) LSAMP_CHECK(check_matrix("base", a->base, a->base_stride, m, n, ob));
  const int64_t ld_out = stride_of(a->out_stride, m, n);
  const int64_t most = (int64_t)1 << 40;
  if (batch > 1) {
    if (a->out_batch_stride < (int64_t)(m - 1) * ld_out + n || a->out_batch_stride > most)
      return set_error(LSAMP_ERR_SHAPE, "out batch stride %lld is below a matrix or out of range",
                       (long long)a->out_batch_stride);
    if (a->x_batch_stride < 0 || a->x_batch_stride > most ||
        (a->base && (a->base_batch_stride < 0 || a->base_batch_stride > most)))
      return set_error(LSAMP_ERR_SHAPE, "a batch stride is out of range");
  }

  OrthPlan P{};
  Arena ws(base);
  P.wide = !a->fast;
  P.tall = m > n;
  const int eb = 2;
  const int32_t M = (int32_t)round_up(m, 64), N = (int32_t)round_up(n, 64);
  const int32_t p = std::min(M, N), q = std::max(M, N);
  const int64_t step_x = (int64_t)M * N, step_a = (int64_t)p * p;

  OrthStart& s = P.start;
  s.rows = m;
  s.cols = n;
  s.all_rows = M;
  while (s.log_x < 8 && (8 << s.log_x) < N) ++s.log_x;
  s.parts = (int32_t)std::min<int64_t>(ceil_div(M, 256 >> s.log_x), std::max(1, 2048 / batch));
  s.eps = a->eps;
  s.x = a->x;
  s.ld_x = stride_of(a->x_stride, m, n);
  s.step_x = batch > 1 ? a->x_batch_stride * ib : 0;
  s.part = ws.take<double>((int64_t)batch * s.parts * 8);
  s.left = ws.take<float>((int64_t)batch * 4);
  for (auto& buffer : P.x)
    for (auto& part : buffer) part = ws.take(batch * step_x * eb);
  s.hi = P.x[0][0];
  s.lo = P.x[0][1];
  s.ld = N;
  s.step = step_x;
  void *gram[2] = {}, *poly[2] = {};
  for (int i = 0; i < (P.wide ? 2 : 1); ++i) {
    gram[i] = ws.take(batch * step_a * eb);
    poly[i] = ws.take(batch * step_a * eb);
  }
  float* const diagonal = ws.take<float>((int64_t)batch * p * 4);

  const int64_t turns = P.wide ? 3 : 1;  // (products of parts)
  const double parts = P.wide ? 2.0 : 1.0;
  P.gram = choose_batch(p, p, turns * slabs_of(q, eb), 2 * eb * parts, batch, true, !P.tall);
  P.poly = choose_batch(p, p, turns * slabs_of(p, eb), 3 * eb * parts, batch, true, true);
  P.update = choose_batch(M, N, turns * slabs_of(p, eb), 4 * eb, batch, false, P.tall);
  const MatrixRef x{P.x[0][0], N, M, N}, A{gram[0], p, p, p}, B{poly[0], p, p, p};
  const int64_t rest_x = (char*)P.x[0][1] - (char*)P.x[0][0];
  const auto rest = [&](void* const* two) { return (char*)two[1] - (char*)two[0]; };
  const auto batched = [&](const Choice& c, const MatrixRef& l, const MatrixRef& r, int64_t rows,
                           int64_t cols, int64_t k, int64_t step_l, int64_t step_r, int64_t rest_l,
                           int64_t rest_r, bool symmetric) {
    BatchPlan g{};
    static_cast<GemmPlan&>(g) = plan_gemm(c, l, r, rows, cols, k, eb);
    g.parts = batch;
    g.step_a = step_l * eb;
    g.step_b = step_r * eb;
    g.symmetric = symmetric;
    if (P.wide) {
      g.rest_a = rest_l;
      g.rest_b = rest_r;
    }
    return g;
  };
  P.g_gram = batched(P.gram, x, x, p, p, q, step_x, step_x, rest_x, rest_x, true);
  P.g_poly = batched(P.poly, A, A, p, p, p, step_a, step_a, rest(gram), rest(gram), true);
  P.g_update = P.tall ? batched(P.update, x, B, M, N, p, step_x, step_a, rest_x, rest(poly), false)
                      : batched(P.update, B, x, M, N, p, step_a, step_x, rest(poly), rest_x, false);
  if (too_many(P.g_gram) || too_many(P.g_poly) || too_many(P.g_update))
    return set_error(LSAMP_ERR_SHAPE, "%d matrices %d x %d are too large for one call", batch, m, n);

  P.e_gram.n = P.e_poly.n = p;
  P.e_gram.out = gram[0];
  P.e_gram.out_lo = gram[1];
  P.e_poly.in = gram[0];
  P.e_poly.in_lo = gram[1];
  P.e_poly.out = poly[0];
  P.e_poly.out_lo = poly[1];
  P.e_gram.step = P.e_poly.step = step_a;
  P.e_poly.diagonal = diagonal;
  EpiOrthUpdate& e = P.e_update;
  e.m = m;
  e.n = n;
  e.all_m = M;
  e.tall = P.tall;
  e.out_dtype = a->out_dtype;
  e.diagonal = diagonal;
  e.step_d = p;
  e.ld = N;
  e.step = step_x;
  P.bytes = ws.used;
  *out = P;
  return LSAMP_OK;
}

#define ORTH_OP(wide, call) ((wide) ? OrthOps<true>::call : OrthOps<false>::call)

}  // namespace

lsamp_status lsamp_layer_norm(lsamp_context* ctx, const lsamp_layer_norm_args* a, void* stream) {
  if (!ctx) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "context is NULL");
  NormPlan P;
  LSAMP_CHECK(plan_norm(a, &P));
  OnDevice guard(context_device(ctx));
  LSAMP_TRY(launch_norm(P, a->dtype, stream));
  return clear_error();
}

int64_t lsamp_layer_norm_backward_workspace(const lsamp_layer_norm_backward_args* a) {
  NormBackwardPlan P;
  int64_t bytes = 0;
  const lsamp_status st = plan_norm_backward(a, nullptr, &P, &bytes);
  return needed(st, bytes);
}

lsamp_status lsamp_layer_norm_backward(lsamp_context* ctx, const lsamp_layer_norm_backward_args* a,
                                       void* stream) {
  if (!ctx) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "context is NULL");
  NormBackwardPlan P;
  int64_t bytes = 0;
  LSAMP_CHECK(plan_norm_backward(a, a ? a->workspace : nullptr, &P, &bytes));
  LSAMP_CHECK(check_workspace(a->workspace, a->workspace_bytes, bytes));
  OnDevice guard(context_device(ctx));
  LSAMP_TRY(launch_norm_backward(P, a->dtype, stream));
  return clear_error();
}

lsamp_status lsamp_quantize_rows(lsamp_context* ctx, const lsamp_quantize_rows_args* a,
                                 void* stream) {
  if (!ctx) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "context is NULL");
  if (!a) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "args is NULL");
  LSAMP_CHECK(check_dims("rows", a->rows, kMaxDim));
  LSAMP_CHECK(check_dims("cols", a->cols));
  LSAMP_CHECK(check_dtype(a->dtype));
  LSAMP_CHECK(check_matrix("x", a->x, a->x_stride, a->rows, a->cols, element_bytes(a->dtype)));
  LSAMP_CHECK(check_quantized("q", a->q, a->q_stride, a->rows, a->cols));
  LSAMP_CHECK(check_vector("scale", a->scale, 4, true));
  const QuantizePlan P{a->rows, a->cols, a->cols,
                       a->x,    stride_of(a->x_stride, a->rows, a->cols),
                       a->q,    stride_of(a->q_stride, a->rows, a->cols),
                       a->scale};
  OnDevice guard(context_device(ctx));
  LSAMP_TRY(launch_quantize(P, a->dtype, stream));
  return clear_error();
}

int64_t lsamp_linear_int8_workspace(const lsamp_linear_int8_args* a) {
  LinearInt8Plan P;
  const lsamp_status st = plan_linear_int8(a, nullptr, &P);
  return needed(st, st == LSAMP_OK ? P.bytes : 0);
}

lsamp_status lsamp_linear_int8(lsamp_context* ctx, const lsamp_linear_int8_args* a, void* stream) {
  if (!ctx) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "context is NULL");
  LinearInt8Plan P;
  LSAMP_CHECK(plan_linear_int8(a, a ? a->workspace : nullptr, &P));
  LSAMP_CHECK(check_workspace(a->workspace, a->workspace_bytes, P.bytes));
  OnDevice guard(context_device(ctx));
  if (P.quantize) LSAMP_TRY(launch_quantize(P.quant, a->dtype, stream));
  LSAMP_TRY(lay_out(P.x, 1, stream));
  LSAMP_TRY(lay_out(P.w, 1, stream));
  if (P.kept) {
    LSAMP_TRY(INT8_OP(a->dtype, resident_linear(P.resident, P.epi, stream)));
  } else if (P.gemm.parts == 1) {
    LSAMP_TRY(INT8_OP(a->dtype, gemm_linear(P.choice.tile, P.gemm, P.epi, stream)));
  } else {
    LSAMP_TRY(launch_partial_int8(P.choice.tile, P.gemm, P.partial, stream));
    LSAMP_TRY(INT8_OP(a->dtype, join_linear(P.partial, P.gemm.parts, P.epi, stream)));
  }
  return clear_error();
}

int64_t lsamp_orthogonalize_workspace(const lsamp_orthogonalize_args* a) {
  OrthPlan P;
  const lsamp_status st = plan_orth(a, nullptr, &P);
  return needed(st, st == LSAMP_OK ? P.bytes : 0);
}

lsamp_status lsamp_orthogonalize(lsamp_context* ctx, const lsamp_orthogonalize_args* a,
                                 void* stream) {
  if (!ctx) return set_error(LSAMP_ERR_INVALID_ARGUMENT, "context is NULL");
  OrthPlan P;
  LSAMP_CHECK(plan_orth(a, a ? a->workspace : nullptr, &P));
  LSAMP_CHECK(check_workspace(a->workspace, a->workspace_bytes, P.bytes));
  OnDevice guard(context_device(ctx));
  LSAMP_TRY(launch_orth_start(P.start, a->batch, a->in_dtype, stream));
  const int ob = element_bytes(a->out_dtype);
  for (int i = 0; i < a->steps; ++i) {
    const float* const c = a->coefficients + 3 * i;
    void* const* const now = P.x[i & 1];
    void* const* const next = P.x[~i & 1];
    P.g_gram.a.p = P.g_gram.b.p = now[0];
    (P.tall ? P.g_update.a : P.g_update.b).p = now[0];
    P.e_gram.left = P.e_update.left = i == 0 ? P.start.left : nullptr;
    P.e_poly.b3 = c[1];
    P.e_poly.c3 = c[2];
    EpiOrthUpdate& e = P.e_update;
    e.a1 = c[0];
    e.x_hi = now[0];
    e.x_lo = now[1];
    e.to_hi = next[0];
    e.to_lo = next[1];
    if (i + 1 == a->steps) {
      e.out = a->out;
      e.ld_out = stride_of(a->out_stride, a->rows, a->cols);
      e.step_out = a->batch > 1 ? a->out_batch_stride * ob : 0;
      e.base = a->base;
      e.ld_base = stride_of(a->base_stride, a->rows, a->cols);
      e.step_base = a->batch > 1 ? a->base_batch_stride * ob : 0;
      e.scale = a->scale;
      e.keep = a->keep;
    }
    LSAMP_TRY(ORTH_OP(P.wide, gram(P.tall, P.gram.tile, P.g_gram, P.e_gram, stream)));
    LSAMP_TRY(ORTH_OP(P.wide, poly(P.poly.tile, P.g_poly, P.e_poly, stream)));
    LSAMP_TRY(ORTH_OP(P.wide, update(P.tall, P.update.tile, P.g_update, e, stream)));
  }
  return clear_error();
}
