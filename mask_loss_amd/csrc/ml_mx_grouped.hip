// Products of microscaled operands: plans, launches and C entry points (the kernel: ml_mx_grouped.h).
#include <algorithm>
#include <cmath>

#include "ml_mx_grouped.h"

namespace ml {
namespace {

constexpr int64_t kMaxGroups = 4000;   // their edges and tile counts fit the LDS beside the tiles
constexpr int64_t kMaxRows = ((int64_t)1 << 31) - 4096;  // positions a step or a tile on stay 32-bit
constexpr int64_t kMaxLength = 1 << 22;  // rows of a tile stay within 2^32 bytes of its first

// Few rows to a group take mx_few_kernel's tiles, many 128 x 128: the ring where K and the scales' alignment let it, mx_kernel
// otherwise (us, the ring / mx_kernel; e2m1 by e2m1 in bfloat16 unless named): 16,384 rows in 16 groups, K = 1,024, N = 4,096
// 62 / 102, e4m3 by e2m1 83 / 128, in float32 174 / 228, e4m3 by e4m3 108 / 159, in float32 184 / 251; 4,096 rows in 8 groups, K = 1,024,
// N = 2,736, e4m3 by e2m1 24 / 31, in float32 43 / 58; one matrix 8,192 x 8,192 x 8,192 359 / 446.  Larger tiles of the ring move fewer
// bytes through LDS, but a tile's stores wait for less beside them: 128 x 256 and 256 x 256 on 8 waves take 68 and 80 for the
// first of these (and 325 and 283 for the last, alone).
constexpr int kColumns = 128, kManyRows = 128, kRingSlots = 512;
constexpr size_t kRingParts = (size_t)kRingSlots * kManyRows * kColumns * sizeof(float);

struct MxPlan {
  bool few, merged;
  int ring;  // 0, or the bytes of a scale load: 4, 16
  int bm, bn, splits;
  int64_t bound, plane;
  size_t bytes;
};

// aligned: bytes that x_scales' and weight_scales' addresses are multiples of (16 at most); equal: without offsets
int mx_plan(const ml_grouped_shape* s, int fa, int fb, int out, int aligned, bool equal, MxPlan& p) {
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
  const bool exact = mx_exact(fa, fb, out);
  p.few = each <= 32.0;
  p.bm = !p.few ? kManyRows : each <= 16.0 ? 16 : 32;
  p.bn = p.few ? kFewColumns : kColumns;
  p.ring = p.few ? 0 : s->K % 512 == 0 && aligned >= 16 ? 16 : s->K % 128 == 0 && aligned >= 4 ? 4 : 0;
  const int64_t columns = ceil_div(s->N, p.bn);
  // values of a part of a reduction, at least one turn of the kernel's loop
  const int64_t step = p.ring == 16 ? 512 : mx_step(fa, fb), steps = std::max<int64_t>(1, ceil_div(s->K, step));
  const double x = each / p.bm, rows = used * (equal || segments == 1 ? std::ceil(x) : std::max(1.05, x + 0.5));
  // Parts of each tile's reduction where the tiles leave slots without work.  The ring takes 2 us for 512 values of a tile, 4 in bfloat16,
  // and a join 4 us and what its parts' 64 KiB take to memory and back: as many parts as cost the least, if they cost less
  // than none (512 x 8,192 x 1,024 25 us in parts, 43 whole; 512 x 4,096 x 4,096 29 in as many as fit, 25 whole).
  const double all = std::max(1.0, rows * columns);
  const int64_t fit = (int64_t)(kRingSlots / all);
  if (p.ring) {
    const double whole = (exact ? 4.0 : 2.0) * s->K / 512, move = 0.026 * all;
    const int64_t parts = std::min({fit, (int64_t)std::lround(std::sqrt(whole / move)), steps, (int64_t)64});
    p.splits = parts > 1 && s->N % 4 == 0 && whole / parts + 4.0 + move * parts < whole ? (int)parts : 1;  // (joined by whole fours)
  } else if (p.few) {
    // a turn of a workgroup's four waves takes 1.5 us, 3.6 in bfloat16, a join 4
    const int64_t turns = ceil_div(s->K, kFewTurn), parts = std::min({fit, turns, (int64_t)64});
    p.splits = parts > 1 && (double)(turns - ceil_div(turns, parts)) * (exact ? 3.6 : 1.5) > 4.0 ? (int)parts : 1;
  } else {
    p.splits = (int)std::max<int64_t>(1, std::min({fit, steps / 4, (int64_t)64}));
  }
  const int64_t tiles = (s->rows / p.bm + std::min(segments + 2, s->rows)) * columns;
  if (p.ring) {
    p.bound = tiles;
    p.bytes = p.splits > 1 ? kRingParts : 256;  // (the counts on the GPU decide which tiles)
  } else {
    p.bound = tiles * p.splits;
    p.plane = ceil_div(s->rows * s->N, 4) * 4;
    p.bytes = p.splits > 1 ? align256((size_t)p.splits * p.plane * sizeof(float)) : 256;
  }
  // ids are 32-bit; mx_kernel has a workgroup to an item, and a launch fewer than 2^32 threads
  if (p.bound > (p.ring ? (int64_t)INT32_MAX : (int64_t)UINT32_MAX / 256) - 8)
    return fail(ML_EUNSUPPORTED, "grouped_matmul_mx: too many tiles");
  return ML_OK;
}

template <int FA, int FB, int OUT>
int mx_launch(const ml_grouped_shape* s, const MxPlan& p, MxArgs& x, hipStream_t st) {
  ProfScope ps("grouped_matmul_mx", st);
  const size_t lds = (2 * (size_t)x.g.groups + 3) * sizeof(int);  // edges, tiles of the segments
  const dim3 blk(256);
  if (p.ring) {
    // persistent workgroups, all that fit where tiles may be split
    const int64_t items = ceil_div(p.bound, kXcds) * kXcds;
    const dim3 grid((unsigned)(p.splits > 1 ? kRingSlots : std::min<int64_t>(items, kRingSlots)));
    constexpr int BK = mx_step(FA, FB);
    if (p.ring == 16)
      hipLaunchKernelGGL((mx_ring_kernel<FA, FB, OUT, kManyRows, kColumns, 2, 2, BK, 2, 16>), grid, blk, lds, st, x);
    else
      hipLaunchKernelGGL((mx_ring_kernel<FA, FB, OUT, kManyRows, kColumns, 2, 2, BK, 2, 4>), grid, blk, lds, st, x);
    const int rc = check_launch("grouped_matmul_mx");
    if (rc || p.splits == 1) return rc;
    hipLaunchKernelGGL((grouped_tail_kernel<OUT, kMxBand>), grid, blk, lds, st, x.g, 0, kManyRows, kColumns, 2, (int)grid.x / kXcds);
    return check_launch("grouped_matmul_mx");
  }
  const dim3 grid((unsigned)(ceil_div(p.bound, kXcds) * kXcds));
  if (p.few) {
    if (p.bm == 16) hipLaunchKernelGGL((mx_few_kernel<FA, FB, OUT, 1>), grid, blk, lds, st, x);
    else hipLaunchKernelGGL((mx_few_kernel<FA, FB, OUT, 2>), grid, blk, lds, st, x);
  } else {
    hipLaunchKernelGGL((mx_kernel<FA, FB, OUT, kManyRows, kColumns, 2, 2>), grid, blk, lds, st, x);
  }
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
  size_t most = 256;  // with and without offsets, for any alignment (a size of 0 stands for a refused shape)
  for (int i = 0; i < 6; ++i) {
    MxPlan p;
    if (mx_plan(s, x_format, weight_format, dtype, i / 2 == 0 ? 1 : i / 2 == 1 ? 4 : 16, i % 2 != 0, p)) return 0;
    most = std::max(most, p.bytes);
  }
  return most;
}

extern "C" int ml_grouped_matmul_mx(const ml_grouped_shape* s, int x_format, const void* x, const uint8_t* x_scales,
                                    int weight_format, const void* weight, const uint8_t* weight_scales,
                                    const int64_t* offsets, int dtype, void* y, void* workspace, size_t workspace_bytes,
                                    ml_stream_t stream) {
  MxPlan p;
  const uintptr_t at = (uintptr_t)x_scales | (uintptr_t)weight_scales;
  const int rc = mx_plan(s, x_format, weight_format, dtype, at % 16 == 0 ? 16 : at % 4 == 0 ? 4 : 1, !offsets, p);
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
  a.fewest = 2;
  a.plane = p.plane;
  a.c = y;
  a.parts = (float*)workspace;
  a.cols = fast_div(ceil_div(s->N, p.bn));
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
