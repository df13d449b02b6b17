// Products of microscaled operands: plans, launches and C entry points (the kernel: ml_mx_grouped.h).
#include <algorithm>
#include <cmath>

#include "ml_mx_grouped.h"

namespace ml {
namespace {

constexpr int64_t kMaxGroups = 4000;   // their edges and tile counts fit the LDS beside the tiles
constexpr int64_t kMaxRows = ((int64_t)1 << 31) - 4096;  // positions a step or a tile on stay 32-bit
constexpr int64_t kMaxLength = 1 << 22;  // rows of a tile stay within 2^32 bytes of its first
constexpr int64_t kUnits = 256;

// Tiles: few rows to a group (64 where the rows are e2m1 and the matrix e4m3: a chunk for every thread), or many.
constexpr int few_rows(int fa, int fb) { return fa == ML_MX_E2M1 && fb == ML_MX_E4M3 ? 64 : 32; }
constexpr int kColumns = 128, kManyRows = 128;

struct MxPlan {
  bool few, merged;
  int bm, splits;
  int64_t bound, plane;
  size_t bytes;
};

int mx_plan(const ml_grouped_shape* s, int fa, int fb, int out, bool equal, MxPlan& p) {
  p = MxPlan{};
  if (!s || s->rows < 0 || s->K < 0 || s->N < 0 || s->groups < 1 || s->matrices < 1 || s->groups % s->matrices)
    return fail(ML_EINVAL, "grouped_matmul_mx: invalid shape (groups must be a positive multiple of the matrices)");
  if (s->K % kMxBlock) return fail(ML_EINVAL, "grouped_matmul_mx: K must be a multiple of 32");
  if (!mx_format(fa) || !mx_format(fb)) return fail(ML_EINVAL, "grouped_matmul_mx: unknown format");
  if (out != ML_F32 && out != ML_BF16 && out != ML_F16) return fail(ML_EINVAL, "grouped_matmul_mx: unsupported dtype");
  if (s->groups > kMaxGroups)
    return fail(ML_EUNSUPPORTED, "grouped_matmul_mx: at most " + std::to_string(kMaxGroups) + " groups are supported");
  if (s->rows > kMaxRows || s->K > kMaxLength || s->N > kMaxLength)
    return fail(ML_EUNSUPPORTED, "grouped_matmul_mx: at most 2^31 - 4096 rows and K, N of at most 4194304 are supported");
  const int64_t groups = s->matrices == 1 ? 1 : s->groups, layers = groups / s->matrices;  // (group_edges)
  // groups that share a matrix make tiles together, as far as their rows' offsets go (and while
  // walking the groups for a row costs little)
  p.merged = layers > 1 && layers <= 32 && s->rows * s->K < ((int64_t)1 << 32);
  const int64_t segments = p.merged ? s->matrices : groups;
  const int64_t used = std::min(segments, std::max<int64_t>(s->rows, 1));  // those that can hold rows
  const double each = (double)s->rows / used;
  p.few = each <= 32.0;
  p.bm = p.few ? few_rows(fa, fb) : kManyRows;
  const int64_t columns = ceil_div(s->N, kColumns), steps = std::max<int64_t>(1, ceil_div(s->K, mx_step(fa, fb)));
  const double x = each / p.bm, rows = used * (equal || segments == 1 ? std::ceil(x) : std::max(1.05, x + 0.5));
  // parts of each tile's reduction where the tiles leave slots without work
  const int most = (int)std::max<int64_t>(1, std::min<int64_t>(steps / 4, 64));
  const int slots = (int)kUnits * (p.few ? 4 : 2);
  p.splits = std::max(1, std::min((int)(slots / std::max(1.0, rows * columns)), most));
  const int64_t tiles = (s->rows / p.bm + std::min(segments + 2, s->rows)) * columns;
  p.bound = tiles * p.splits;
  p.plane = ceil_div(s->rows * s->N, 4) * 4;
  p.bytes = p.splits > 1 ? align256((size_t)p.splits * p.plane * sizeof(float)) : 256;
  // a workgroup to an item, and a launch has fewer than 2^32 threads
  if (p.bound > (int64_t)UINT32_MAX / 256 - 8) return fail(ML_EUNSUPPORTED, "grouped_matmul_mx: too many tiles");
  return ML_OK;
}

template <int FA, int FB, int OUT>
int mx_launch(const ml_grouped_shape* s, const MxPlan& p, MxArgs& x, hipStream_t st) {
  ProfScope ps("grouped_matmul_mx", st);
  const size_t lds = (2 * (size_t)x.g.groups + 3) * sizeof(int);  // edges, tiles of the segments
  const dim3 grid((unsigned)(ceil_div(p.bound, kXcds) * kXcds)), blk(256);
  if (p.few)
    hipLaunchKernelGGL((mx_kernel<FA, FB, OUT, few_rows(FA, FB), kColumns, 1, 4>), grid, blk, lds, st, x);
  else
    hipLaunchKernelGGL((mx_kernel<FA, FB, OUT, kManyRows, kColumns, 2, 2>), grid, blk, lds, st, x);
  const int rc = check_launch("grouped_matmul_mx");
  if (rc || p.splits == 1) return rc;
  const int64_t n = s->rows * s->N;
  hipLaunchKernelGGL(grouped_join_kernel<OUT>, dim3((unsigned)ceil_div(n, kJoinQuads * 4)), dim3(kJoinQuads * kJoinSlices), 0,
                     st, x.g.parts, p.splits, p.plane, n, x.g.c);
  return check_launch("grouped_matmul_mx");
}

template <int FA, int FB>
int mx_out(const ml_grouped_shape* s, const MxPlan& p, MxArgs& x, int out, hipStream_t st) {
  switch (out) {
    case ML_F32: return mx_launch<FA, FB, ML_F32>(s, p, x, st);
    case ML_BF16: return mx_launch<FA, FB, ML_BF16>(s, p, x, st);
    default: return mx_launch<FA, FB, ML_F16>(s, p, x, st);
  }
}

}  // namespace
}  // namespace ml

using namespace ml;

extern "C" size_t ml_grouped_matmul_mx_workspace_size(const ml_grouped_shape* s, int x_format, int weight_format, int dtype) {
  size_t most = 256;  // with and without offsets (a size of 0 stands for a refused shape)
  for (int i = 0; i < 2; ++i) {
    MxPlan p;
    if (mx_plan(s, x_format, weight_format, dtype, i != 0, p)) return 0;
    most = std::max(most, p.bytes);
  }
  return most;
}

extern "C" int ml_grouped_matmul_mx(const ml_grouped_shape* s, int x_format, const void* x, const uint8_t* x_scales,
                                    int weight_format, const void* weight, const uint8_t* weight_scales,
                                    const int64_t* offsets, int dtype, void* y, void* workspace, size_t workspace_bytes,
                                    ml_stream_t stream) {
  MxPlan p;
  const int rc = mx_plan(s, x_format, weight_format, dtype, !offsets, p);
  if (rc) return rc;
  if (s->rows == 0 || s->N == 0) return ML_OK;
  if (!offsets && s->rows % s->groups)
    return fail(ML_EINVAL, "grouped_matmul_mx: without offsets the rows must divide into equal groups");
  if (!y || (s->K > 0 && (!x || !x_scales || !weight || !weight_scales)))
    return fail(ML_EINVAL, "grouped_matmul_mx: null pointer");
  if (!aligned16(x) || !aligned16(weight)) return fail(ML_EINVAL, "grouped_matmul_mx: codes must be 16-byte aligned");
  if (p.splits > 1 && (!workspace || workspace_bytes < p.bytes))
    return fail(ML_EWORKSPACE, "grouped_matmul_mx: workspace too small");
  MxArgs m{};
  GroupedArgs& a = m.g;
  a.a = x;
  a.b = weight;
  a.K = (int)s->K;
  a.lda = mx_bytes(x_format, a.K) / 2;
  a.ldb = mx_bytes(weight_format, a.K) / 2;
  a.N = (int)s->N;
  a.ldc = s->N;
  a.bstride = s->N * a.ldb;
  a.offsets = offsets;
  a.equal = (int)(s->rows / s->groups);
  a.rows = (int)s->rows;
  a.given = (int)s->groups;
  a.groups = s->matrices == 1 ? 1 : a.given;
  a.matrices = (int)s->matrices;
  a.segments = p.merged ? a.matrices : a.groups;
  a.merged = p.merged;
  a.splits = p.splits;
  a.plane = p.plane;
  a.c = y;
  a.parts = (float*)workspace;
  a.cols = fast_div(ceil_div(s->N, kColumns));
  a.layers = fast_div(a.groups / a.matrices);
  a.mtiles = fast_div(1);
  m.sa = x_scales;
  m.sb = weight_scales;
  m.sld = s->K / kMxBlock;
  hipStream_t st = (hipStream_t)stream;
  if (x_format == ML_MX_E4M3)
    return weight_format == ML_MX_E4M3 ? mx_out<ML_MX_E4M3, ML_MX_E4M3>(s, p, m, dtype, st)
                                       : mx_out<ML_MX_E4M3, ML_MX_E2M1>(s, p, m, dtype, st);
  return weight_format == ML_MX_E4M3 ? mx_out<ML_MX_E2M1, ML_MX_E4M3>(s, p, m, dtype, st)
                                     : mx_out<ML_MX_E2M1, ML_MX_E2M1>(s, p, m, dtype, st);
}
