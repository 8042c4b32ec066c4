// The hidden-state operators' C entry points over launches that are written
// down in place of being run, for CPU tests of the planner: compiled together
// with lsamp_head_api.cpp, without a device or the HIP runtime.
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <vector>

#include "lsamp_head.h"
#include "lsamp_internal.h"

extern "C" {
enum LaunchKind : int32_t {
  kLinear, kStats, kGrad, kStore, kPartial, kJoinLinear, kJoinStore, kColSum, kColSumJoin, kPack,
  kJoinStats, kGradScale, kDropout
};
// One launch.  A field that a kind has no use for is 0.
struct Launch {
  int32_t kind, tile, roles, parts;
  int32_t m, n, slabs, slabs_per_part;
  int32_t accumulate, first_col, chunks, stream;
  int32_t element, unused;         // bytes of the operands' elements
  int64_t a, a_ld, b, b_ld;      // operands (a: what a pass reads)
  int32_t a_rows, a_cols, b_rows, b_cols;
  int64_t out, ld_out, out_bytes;  // what it writes: a range from `out`
  int64_t part_stride;             // floats between parts
  int64_t out2, out2_bytes;
};
}

namespace {
std::vector<Launch> g_launches;

int64_t at(const void* p) { return (int64_t)(intptr_t)p; }
Launch product(int32_t kind, lsamp::GemmTile tile, const lsamp::GemmPlan& g, int32_t element) {
  Launch l{};
  l.kind = kind;
  l.element = element;
  l.tile = tile;
  l.parts = g.parts;
  l.slabs = g.slabs;
  l.slabs_per_part = g.slabs_per_part;
  l.a = at(g.a.p), l.a_ld = g.a.ld, l.a_rows = g.a.rows, l.a_cols = g.a.cols;
  l.b = at(g.b.p), l.b_ld = g.b.ld, l.b_rows = g.b.rows, l.b_cols = g.b.cols;
  return l;
}
void writes(Launch* l, const void* out, int64_t ld, int64_t rows, int64_t cols, int64_t bytes) {
  l->out = at(out);
  l->ld_out = ld;
  l->out_bytes = out ? ((rows - 1) * ld + cols) * bytes : 0;
}
int put(const Launch& l) {
  g_launches.push_back(l);
  return 0;
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

#define EACH_TYPE(DT, EB)                                                                          \
  template <>                                                                                      \
  int HeadOps<DT>::gemm_linear(GemmTile t, const GemmPlan& g, const EpiLinear& e, void*) {         \
    Launch l = product(kLinear, t, g, EB);                                                         \
    l.m = e.m, l.n = e.n, l.stream = e.stream;                                                     \
    writes(&l, e.out, e.ld_out, e.m, e.n, e.wide ? 4 : EB);                                        \
    l.out2 = at(e.pre);                                                                            \
    return put(l);                                                                                 \
  }                                                                                                \
  template <>                                                                                      \
  int HeadOps<DT>::gemm_stats(GemmTile t, const GemmPlan& g, const EpiStats& e, void*) {           \
    Launch l = product(kStats, t, g, EB);                                                          \
    l.m = e.m, l.n = e.n, l.first_col = e.first_col;                                               \
    writes(&l, e.part, (int64_t)e.blocks * 2, e.m, (int64_t)e.blocks * 2, 4);                      \
    l.out2 = at(e.target), l.out2_bytes = (int64_t)e.m * 4;                                        \
    return put(l);                                                                                 \
  }                                                                                                \
  template <>                                                                                      \
  int HeadOps<DT>::gemm_grad(GemmTile t, const GemmPlan& g, const EpiGrad& e, void*) {             \
    Launch l = product(kGrad, t, g, EB);                                                           \
    l.m = e.m, l.n = e.n, l.first_col = e.first_col;                                               \
    writes(&l, e.out, e.ld_out, e.m, e.n_pad, EB);                                                 \
    l.out2 = at(e.sums);                                                                           \
    l.chunks = e.sums ? g.tiles_m * kTileWavesM[t] : 0;                                            \
    if (e.sums) l.out2_bytes = ((l.chunks - 1) * e.ld_sums + (e.n + 3) / 4 * 4) * 4;               \
    return put(l);                                                                                 \
  }                                                                                                \
  template <>                                                                                      \
  int HeadOps<DT>::gemm_store(GemmRoles r, GemmTile t, const GemmPlan& g, const EpiStore& e,       \
                              void*) {                                                             \
    Launch l = product(kStore, t, g, EB);                                                          \
    l.roles = r, l.m = e.m, l.n = e.n, l.stream = e.stream;                                        \
    writes(&l, e.out, e.ld_out, e.m, e.n, EB);                                                     \
    return put(l);                                                                                 \
  }                                                                                                \
  template <>                                                                                      \
  int HeadOps<DT>::gemm_partial(GemmRoles r, GemmTile t, const GemmPlan& g, const EpiPartial& e,   \
                                void*) {                                                           \
    Launch l = product(kPartial, t, g, EB);                                                        \
    l.roles = r, l.m = e.m, l.n = e.n, l.accumulate = e.accumulate, l.part_stride = e.part_stride; \
    writes(&l, e.out, e.ld, e.m, e.ld, 4);                                                         \
    l.out_bytes += (g.parts - 1) * e.part_stride * 4;                                              \
    return put(l);                                                                                 \
  }                                                                                                \
  template <>                                                                                      \
  int HeadOps<DT>::join_linear(const EpiPartial& f, int parts, const EpiLinear& e, void*) {        \
    Launch l{};                                                                                    \
    l.kind = kJoinLinear, l.parts = parts, l.m = e.m, l.n = e.n, l.a = at(f.out);                  \
    writes(&l, e.out, e.ld_out, e.m, e.n, e.wide ? 4 : EB);                                        \
    return put(l);                                                                                 \
  }                                                                                                \
  template <>                                                                                      \
  int HeadOps<DT>::join_store(const EpiPartial& f, int parts, const EpiStore& e, void*) {          \
    Launch l{};                                                                                    \
    l.kind = kJoinStore, l.parts = parts, l.m = e.m, l.n = e.n, l.a = at(f.out);                   \
    writes(&l, e.out, e.ld_out, e.m, e.n, EB);                                                     \
    return put(l);                                                                                 \
  }                                                                                                \
  template <>                                                                                      \
  int HeadOps<DT>::col_sum(const ColSumPlan& p, void*) {                                           \
    Launch l{};                                                                                    \
    l.kind = kColSum, l.m = p.rows, l.n = p.cols, l.chunks = p.chunks, l.a = at(p.in);             \
    writes(&l, p.out, p.ld_out, p.rows, p.out_cols, EB);                                           \
    l.out2 = at(p.part), l.out2_bytes = p.part ? p.chunks * p.ld_part * 4 : 0;                     \
    return put(l);                                                                                 \
  }                                                                                                \
  template <>                                                                                      \
  int HeadOps<DT>::col_sum_join(const ColSumPlan& p, void* out, const float*, void*) {             \
    Launch l{};                                                                                    \
    l.kind = kColSumJoin, l.n = p.cols, l.chunks = p.chunks, l.a = at(p.part);                     \
    writes(&l, out, p.cols, 1, p.cols, EB);                                                        \
    return put(l);                                                                                 \
  }
EACH_TYPE(LSAMP_DTYPE_F32, 4)
EACH_TYPE(LSAMP_DTYPE_BF16, 2)
EACH_TYPE(LSAMP_DTYPE_F16, 2)

int launch_dropout(const DropoutPlan& p, int, void*) {
  Launch l{};
  l.kind = kDropout, l.m = p.rows, l.n = p.cols, l.a = at(p.x), l.out = at(p.out);
  return put(l);
}
int launch_pack(const PackPlan& p, int bytes, void*) {
  Launch l{};
  l.kind = kPack, l.m = p.rows, l.n = p.cols, l.a = at(p.src), l.a_ld = p.src_ld;
  writes(&l, p.dst, p.dst_ld, p.rows, p.dst_cols, bytes);
  return put(l);
}
int launch_join_stats(const JoinStatsPlan& p, void*) {
  Launch l{};
  l.kind = kJoinStats, l.m = p.rows, l.n = p.vocab, l.a = at(p.part);
  writes(&l, p.loss, 1, p.rows, 1, 4);
  return put(l);
}
int launch_grad_scale(const GradScalePlan& p, void*) {
  Launch l{};
  l.kind = kGradScale, l.m = p.rows, l.n = p.vocab, l.a = at(p.d_loss);
  writes(&l, p.scale, 1, 2, 1, 4);
  return put(l);
}

}  // namespace lsamp

extern "C" {
int64_t head_launch_size() { return (int64_t)sizeof(Launch); }
// The launches since the last call of this.
int64_t head_launches(Launch* out, int64_t most) {
  const int64_t n = (int64_t)g_launches.size();
  for (int64_t i = 0; i < n && i < most; ++i) out[i] = g_launches[i];
  g_launches.clear();
  return n;
}
}
