// The entry points of lsamp_blocks_api.cpp over launches that are written down in
// place of being run, for CPU tests: what each launch reads and writes, as ranges of
// bytes.  Compiled together with lsamp_blocks_api.cpp, without a device or the HIP runtime.
#include <hip/hip_runtime.h>

#include <vector>

#include "lsamp_head.h"
#include "lsamp_internal.h"
#include "lsamp_orth.h"

extern "C" {
// A launch reads or writes a range: [at, at + bytes).
struct Access {
  int32_t launch, kind, write, tile;
  int64_t at, bytes;
};
}

namespace {
std::vector<Access> g_all;
int32_t g_launch = 0;
int32_t g_kind = 0, g_tile = 0;

void touch(bool write, const void* p, int64_t bytes) {
  if (p && bytes > 0) g_all.push_back(Access{g_launch, g_kind, write, g_tile, (int64_t)(intptr_t)p, bytes});
}
int64_t span(int64_t rows, int64_t ld, int64_t cols, int64_t eb) { return ((rows - 1) * ld + cols) * eb; }
void matrix(bool write, const void* p, int64_t rows, int64_t ld, int64_t cols, int64_t eb) {
  touch(write, p, span(rows, ld, cols, eb));
}
void begin(int32_t kind, int32_t tile = -1) {
  ++g_launch;
  g_kind = kind;
  g_tile = tile;
}
int bytes_of(int dtype) { return dtype == LSAMP_DTYPE_F32 ? 4 : 2; }
void operands(const lsamp::GemmPlan& g, int eb) {
  matrix(false, g.a.p, g.a.rows, g.a.ld, g.a.cols, eb);
  matrix(false, g.b.p, g.b.rows, g.b.ld, g.b.cols, eb);
}
void epilogue(const lsamp::EpiLinearInt8& e, int eb) {
  touch(false, e.x_scale, e.m * 4ll);
  touch(false, e.w_scale, e.n * 4ll);
  touch(false, e.bias, (int64_t)e.n * eb);
  if (e.residual) matrix(false, e.residual, e.m, e.ld_residual, e.n, eb);
  matrix(true, e.out, e.m, e.ld_out, e.n, e.wide ? 4 : eb);
}
// A batch's operands: both parts where there are two.
void batched(const lsamp::BatchPlan& g) {
  for (int part = 0; part < g.parts; part += g.parts > 1 ? g.parts - 1 : 1)
    for (int64_t rest : {(int64_t)0, g.rest_a}) {
      if (rest == 0 || g.rest_a)
        matrix(false, (const char*)g.a.p + part * g.step_a + rest, g.a.rows, g.a.ld, g.a.cols, 2);
      const int64_t rest_b = rest ? g.rest_b : 0;
      matrix(false, (const char*)g.b.p + part * g.step_b + rest_b, g.b.rows, g.b.ld, g.b.cols, 2);
    }
}
}  // namespace

hipError_t hipGetDevice(int* d) {
  *d = 0;
  return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return ""; }

namespace lsamp {

lsamp_status set_error(lsamp_status st, const char*, ...) { return st; }
lsamp_status clear_error() { return LSAMP_OK; }
int32_t context_device(const lsamp_context*) { return 0; }
int norm_chunks(int rows, int cols, bool in_place) { return rows <= 768 && cols <= 4096 && !in_place ? 0 : 5; }

int launch_norm(const NormPlan& p, int dtype, void*) {
  const int eb = bytes_of(dtype);
  begin(0);
  matrix(false, p.x, p.rows, p.ld_x, p.cols, eb);
  touch(false, p.weight, (int64_t)p.cols * eb);
  touch(false, p.bias, (int64_t)p.cols * eb);
  matrix(true, p.out, p.rows, p.ld_out, p.cols, eb);
  touch(true, p.mean, p.rows * 4ll);
  touch(true, p.rstd, p.rows * 4ll);
  return 0;
}
int launch_norm_backward(const NormBackwardPlan& p, int dtype, void*) {
  const int eb = bytes_of(dtype);
  begin(1);
  matrix(false, p.x, p.rows, p.ld_x, p.cols, eb);
  matrix(false, p.d_out, p.rows, p.ld_d, p.cols, eb);
  if (p.residual) matrix(false, p.residual, p.rows, p.ld_residual, p.cols, eb);
  if (p.part) touch(true, p.part, (int64_t)p.chunks * 2 * p.ld_part * 4);
  if (p.d_x) matrix(true, p.d_x, p.rows, p.ld_dx, p.cols, eb);
  touch(true, p.d_weight, (int64_t)p.cols * eb);
  touch(true, p.d_bias, (int64_t)p.cols * eb);
  return (p.d_weight || p.d_bias) && p.chunks && !p.part;
}
int launch_quantize(const QuantizePlan& p, int dtype, void*) {
  begin(2);
  matrix(false, p.x, p.rows, p.ld_x, p.cols, bytes_of(dtype));
  matrix(true, p.q, p.rows, p.ld_q, p.out_cols, 1);
  touch(true, p.scale, p.rows * 4ll);
  return 0;
}
int launch_pack(const PackPlan& p, int eb, void*) {
  begin(3);
  matrix(false, p.src, p.rows, p.src_ld, p.cols, eb);
  matrix(true, p.dst, p.rows, p.dst_ld, p.dst_cols, eb);
  return 0;
}
int launch_partial_int8(GemmTile t, const GemmPlan& g, const EpiPartial& e, void*) {
  begin(4, t);
  operands(g, 1);
  touch(true, e.out, ((g.parts - 1) * e.part_stride + span(e.m, e.ld, e.ld, 1)) * 4);
  return 0;
}
#define EACH_TYPE(DT, EB)                                                                       \
  template <>                                                                                   \
  int Int8Ops<DT>::gemm_linear(GemmTile t, const GemmPlan& g, const EpiLinearInt8& e, void*) {  \
    begin(5, t);                                                                                \
    operands(g, 1);                                                                             \
    epilogue(e, EB);                                                                            \
    return 0;                                                                                   \
  }                                                                                             \
  template <>                                                                                   \
  int Int8Ops<DT>::resident_linear(const ResidentPlan& g, const EpiLinearInt8& e, void*) {      \
    begin(6);                                                                                   \
    if (g.fused)                                                                                \
      matrix(false, g.x, g.m, g.ld_x, g.k, EB);                                                 \
    else /* rows of multiples of 256 bytes */                                                   \
      matrix(false, g.x, g.m, g.ld_x, (g.k + 255) / 256 * 256, 1);                              \
    matrix(false, g.w, e.n, g.ld_w, g.k, 1);                                                    \
    EpiLinearInt8 p = e;                                                                        \
    if (g.fused) p.x_scale = nullptr;                                                           \
    epilogue(p, EB);                                                                            \
    return g.m > 64 || g.m * (int64_t)((g.k + 255) / 256 * 256) > 128 << 10 || g.k < 16 ||      \
           (g.fused && g.m * (int64_t)g.k > 8192);                                              \
  }                                                                                             \
  template <>                                                                                   \
  int Int8Ops<DT>::join_linear(const EpiPartial& f, int parts, const EpiLinearInt8& e, void*) { \
    begin(7);                                                                                   \
    touch(false, f.out, ((parts - 1) * f.part_stride + span(f.m, f.ld, f.ld, 1)) * 4);          \
    epilogue(e, EB);                                                                            \
    return 0;                                                                                   \
  }
EACH_TYPE(LSAMP_DTYPE_F32, 4)
EACH_TYPE(LSAMP_DTYPE_BF16, 2)
EACH_TYPE(LSAMP_DTYPE_F16, 2)

int launch_orth_start(const OrthStart& p, int batch, int in_dtype, void*) {
  begin(8);
  for (int b = 0; b < batch; b += batch > 1 ? batch - 1 : 1)
    matrix(false, (const char*)p.x + b * p.step_x, p.rows, p.ld_x, p.cols, bytes_of(in_dtype));
  touch(true, p.part, (int64_t)batch * p.parts * 8);
  touch(true, p.left, batch * 4ll);
  touch(true, p.hi, batch * p.step * 2);
  touch(true, p.lo, batch * p.step * 2);
  return p.all_rows % 64 || p.ld % 64 || p.step != p.all_rows * p.ld;
}
template <bool WIDE>
int OrthOps<WIDE>::gram(bool, GemmTile t, const BatchPlan& g, const EpiSymmetric& e, void*) {
  begin(9, t);
  batched(g);
  touch(false, e.left, e.left ? g.parts * 4ll : 0);
  touch(true, e.out, g.parts * e.step * 2);
  if (WIDE) touch(true, e.out_lo, g.parts * e.step * 2);
  return e.n % 64 || e.step != (int64_t)e.n * e.n;
}
template <bool WIDE>
int OrthOps<WIDE>::poly(GemmTile t, const BatchPlan& g, const EpiSymmetric& e, void*) {
  begin(10, t);
  batched(g);
  touch(false, e.in, g.parts * e.step * 2);
  if (WIDE) touch(false, e.in_lo, g.parts * e.step * 2);
  touch(true, e.out, g.parts * e.step * 2);
  if (WIDE) touch(true, e.out_lo, g.parts * e.step * 2);
  touch(true, e.diagonal, (int64_t)g.parts * e.n * 4);
  return 0;
}
template <bool WIDE>
int OrthOps<WIDE>::update(bool, GemmTile t, const BatchPlan& g, const EpiOrthUpdate& e, void*) {
  begin(11, t);
  batched(g);
  touch(false, e.left, e.left ? g.parts * 4ll : 0);
  touch(false, e.x_hi, g.parts * e.step * 2);
  touch(false, e.x_lo, g.parts * e.step * 2);
  touch(false, e.diagonal, (int64_t)g.parts * e.step_d * 4);
  if (!e.out) {
    touch(true, e.to_hi, g.parts * e.step * 2);
    touch(true, e.to_lo, g.parts * e.step * 2);
    return 0;
  }
  const int ob = bytes_of(e.out_dtype);
  for (int b = 0; b < g.parts; b += g.parts > 1 ? g.parts - 1 : 1) {
    if (e.base) matrix(false, (const char*)e.base + b * e.step_base, e.m, e.ld_base, e.n, ob);
    matrix(true, (const char*)e.out + b * e.step_out, e.m, e.ld_out, e.n, ob);
  }
  return 0;
}
template struct OrthOps<false>;
template struct OrthOps<true>;

}  // namespace lsamp

extern "C" {
int64_t blocks_access_size() { return (int64_t)sizeof(Access); }
// The accesses since the last call of this.
int64_t blocks_accesses(Access* out, int64_t most) {
  const int64_t n = (int64_t)g_all.size();
  for (int64_t i = 0; i < n && i < most; ++i) out[i] = g_all[i];
  g_all.clear();
  g_launch = 0;
  return n;
}
}
