// Grouped products: plans, launches and C entry points (the kernels: ml_grouped.h).
//
// Tiles, and what the listed products of perf/operators.py take with each (us; KC: the operand's
// reduced index is contiguous):
//
//                                      KC x KC          KC x rows        rows x rows
//                                      experts  masks   experts  masks   experts  masks
//                                      forward  d in    d in     forward d weight d weight
//   128 x 128, 2 stages of 128 bytes   160      195      191      289     266      287
//   128 x 256, 3 stages of 64 bytes    182      248     172      278     211      238
//   256 x 256, 4 stages of 64 bytes    196      227     166      241     187      220
//   256 x 256, 2 stages of 128 bytes   187      203     157      247     189      227
//   grouped_kernel, 128 x 128          229      229     258      402     315      380
//
// (experts: 16,384 rows in 16 groups, K = 1,024, N = 4,096; masks: 16 groups of 200 rows, K = 256,
// N = 65,536; bf16.  The experts' groups are uneven, which their d weight waits for: consecutive tiles are a
// matrix's, an XCD takes two of the 16 matrices whole, and the busiest has 1.4 to 2.0 times the mean number
// of steps; 16 equal groups take 165 us where uneven ones take 167 to 221.)
// Where both operands' reduced index is contiguous, 128-byte stages read whole
// HBM lines and win; operands by rows are whole lines anyway, and the larger tiles read LDS less
// often, in stages of 128 bytes (128 matrix instructions of a SIMD to a barrier, not 64) unless both
// operands are by rows.  (64-byte stages, 4 waves of 128 x 128 instead of 8 of 128 x 64: masks forward 252, d weight 216,
// experts d weight 199.)  The masks' d input varies from machine to machine, 194 to 237 with the same
// code: rows 128 KiB apart.  The choice also weighs how the tiles fill the compute units (grouped_plan).
#include <algorithm>
#include <cmath>

#include "ml_grouped.h"

namespace ml {
namespace {

enum { kForward = 0, kInput = 1, kWeight = 2 };  // the three products

// Tiles: a workgroup's part of the output, and workgroups to a compute unit.
enum Tile { kFew, kPlain, kDeep128, kWide128, kDeep128x256, kDeep256 };
struct TileShape {
  int bm, bn, occ;
};
constexpr TileShape kTiles[] = {{32, 128, 4}, {128, 128, 2}, {128, 128, 2}, {128, 128, 2}, {128, 256, 2}, {256, 256, 1}};

// bytes of the reduced index in an LDS stage of the ring's tiles
constexpr int stage_bytes(Tile t, bool wg) { return t == kWide128 || (t == kDeep256 && !wg) ? 128 : 64; }

struct GroupedPlan {
  Tile tile;
  int splits, fewest;
  bool merged;
  int64_t m, n, k;          // output rows and columns, reduced length (weight gradient: mean rows per matrix)
  int64_t bound;            // work items at most
  int64_t plane;            // elements of a plane
  size_t bytes;             // workspace
};

constexpr int64_t kMaxGroups = 4000;   // their edges and tile counts fit the LDS beside the tiles
constexpr int64_t kMaxRows = ((int64_t)1 << 31) - 4096;  // positions a step or a tile on stay 32-bit
constexpr int64_t kMaxLength = 1 << 22;  // rows of a tile stay within 2^32 bytes of its first
constexpr int64_t kUnits = 256;

// aligned: every row of the operands starts on a 16-byte boundary, rows of all three tensors are whole
// 16-byte chunks (the result may start anywhere); transposed: as the call's;
// equal: without offsets
int grouped_plan(const ml_grouped_shape* s, int dtype, int which, bool transposed, bool aligned, bool equal,
                 GroupedPlan& p) {
  p = GroupedPlan{};
  if (!s || s->rows < 0 || s->K < 0 || s->N < 0 || s->groups < 1 || s->matrices < 1 || s->groups % s->matrices)
    return fail(ML_EINVAL, "grouped_matmul: invalid shape (groups must be a positive multiple of the matrices)");
  if (dtype != ML_F32 && dtype != ML_BF16 && dtype != ML_F16)
    return fail(ML_EINVAL, "grouped_matmul: unsupported dtype");
  if (s->groups > kMaxGroups)
    return fail(ML_EUNSUPPORTED, "grouped_matmul: at most " + std::to_string(kMaxGroups) + " groups are supported");
  if (s->rows > kMaxRows || s->K > kMaxLength || s->N > kMaxLength)
    return fail(ML_EUNSUPPORTED, "grouped_matmul: at most 2^31 - 4096 rows and K, N of at most 4194304 are supported");
  const int64_t es = dtype == ML_F32 ? 4 : 2, bk = 128 / es;
  const int64_t groups = s->matrices == 1 ? 1 : s->groups, layers = groups / s->matrices;  // (group_edges)
  const bool wg = which == kWeight;
  p.m = wg ? (transposed ? s->N : s->K) : s->rows;
  p.n = wg ? (transposed ? s->K : s->N) : which == kInput ? s->K : s->N;
  p.k = which == kForward ? s->K : which == kInput ? s->N : ceil_div(s->rows, s->matrices);
  // groups that share a matrix make tiles together, as far as their rows' offsets go (and while
  // walking the groups for a row costs little)
  p.merged = !wg && layers > 1 && layers <= 32 && s->rows * p.k * es < ((int64_t)1 << 32);
  const int64_t segments = p.merged ? s->matrices : groups;
  const int64_t used = std::min(segments, std::max<int64_t>(s->rows, 1));  // those that can hold rows
  const double each = (double)s->rows / used;
  const int64_t out = (wg ? s->matrices : 1) * p.m * p.n;

  const int64_t steps = std::max<int64_t>(1, ceil_div(p.k, bk));
  const int most = (int)std::max<int64_t>(1, std::min<int64_t>(steps / 4, 64));  // parts of at least four steps
  auto tiles_of = [&](Tile t) {
    const double x = each / kTiles[t].bm;
    const double mt = wg ? (double)s->matrices * ceil_div(p.m, kTiles[t].bm)
                         : used * (equal || segments == 1 ? std::ceil(x) : std::max(1.05, x + 0.5));
    return std::max(1.0, mt * ceil_div(p.n, kTiles[t].bn));
  };
  // Rough time in us of a round of the persistent workgroups, and of all rounds, the last one in parts
  // (ring_share), whose join takes kJoin.
  constexpr double kJoin = 10.0;
  const double unit = dtype == ML_F32 ? 1.75 : 0.5;  // a step of 128 x 128 outputs on one compute unit
  auto round = [&](Tile t) { return kTiles[t].bm * kTiles[t].bn * kTiles[t].occ / 16384.0 * (steps + 3.0) * unit; };
  // a last round that leaves half of the workgroups without work, alone on their compute units then
  auto last = [&](Tile t) { return kTiles[t].occ > 1 ? 0.55 : 1.0; };
  auto fewest_parts = [&](Tile t) {  // it less 1 / parts of a round saved, for more than a join
    const double h = last(t) - kJoin / round(t);
    return h > 0.02 ? std::max(2, (int)std::ceil(1.0 / h)) : 1 << 30;
  };
  // parts of the last round's tiles that are to be expected, 1 for none; `more` rounds than the mean number
  auto expected_parts = [&](Tile t, double& whole, double more) {
    const double rounds = tiles_of(t) / (kUnits * kTiles[t].occ);
    whole = std::floor(rounds + 0.02);
    const double rest = rounds - whole + (whole > 0.0 ? more : 0.0);
    if (whole > 0.0 && rest < 0.02) return 0;
    const int parts = (int)std::min<double>(whole > 0.0 ? std::min(most, kTailParts) : most, 1.0 / rest + 0.02);
    return parts < (whole > 0.0 ? fewest_parts(t) : 2) ? 1 : parts;
  };
  // Their products, or the time that the tensors take at the rate of a copy, and the parts' way through
  // memory.  Ragged groups may make more tiles than the mean, and one too many costs a part of the last round's;
  // the longest one's weight gradient is waited for.
  const double bytes = ((double)s->rows * (s->K + s->N) + (double)s->matrices * s->K * s->N) * es;
  auto cost = [&](Tile t, double products, double copies) {
    double whole;
    const bool ragged = !equal && segments > 1;
    const int parts = expected_parts(t, whole, ragged && !wg ? 0.05 : 0.0);
    const double rest = tiles_of(t) / (kUnits * kTiles[t].occ) - whole;
    const double tail = parts == 0 ? 0.0 : parts > 1 ? 1.0 / parts : rest <= 0.5 ? last(t) : 1.0;
    const double wait = ragged && wg ? 0.4 : 0.0;
    const double planes = parts * rest * kUnits * kTiles[t].occ * kTiles[t].bm * kTiles[t].bn * 4.0;
    return std::max((whole + tail + wait) * round(t) * products, bytes / 5.2e6 * copies) +
           (parts > 1 ? 4.0 + planes / 2.5e6 : 0.0);
  };
  if (!wg && each <= 32.0) {
    p.tile = kFew;
  } else if (!aligned) {
    p.tile = kPlain;
  } else if (dtype == ML_F32) {
    p.tile = wg ? kDeep128 : kWide128;
  } else {
    const int rowops = wg ? 2 : (which == kForward) == transposed ? 0 : 1;  // operands by rows of the reduced index
    // by the tables above: bound by products (per tile area), by HBM.  Over 156 ragged and whole products
    // of 1,000 to 32,768 rows, half of them in float16, the calls take 1.006 times what the best of the three
    // tiles takes on average, and 1.26 at most (55 groups of 12,542 rows, K = 832, N = 400, d weight).
    constexpr double f[3][3] = {{1.0, 1.05, 0.9}, {1.1, 1.02, 0.9}, {1.3, 1.0, 0.92}};
    constexpr double h[3][3] = {{1.05, 1.33, 1.1}, {1.55, 1.47, 1.33}, {1.56, 1.29, 1.2}};
    const Tile ts[3] = {kWide128, kDeep128x256, kDeep256};
    double best = 0.0;
    for (int i = 0; i < 3; ++i) {
      const double c = cost(ts[i], f[rowops][i], h[rowops][i]);
      if (i && c >= best) continue;
      best = c;
      p.tile = ts[i];
    }
  }
  const TileShape& T = kTiles[p.tile];
  const int64_t mt = wg ? s->matrices * ceil_div(p.m, T.bm) : s->rows / T.bm + std::min(segments + 2, s->rows);
  const int64_t tiles = mt * ceil_div(p.n, T.bn);
  if (p.tile >= kDeep128) {
    double whole;
    p.splits = expected_parts(p.tile, whole, 0.0) > 1 ? most : 1;  // (the counts on the GPU decide)
    p.fewest = fewest_parts(p.tile);
    p.bound = tiles;
    p.bytes = p.splits > 1 ? (size_t)kUnits * T.occ * T.bm * T.bn * sizeof(float) : 256;
  } else {
    // parts of each tile's reduction where the tiles leave slots without work
    p.splits = std::max(1, std::min((int)(kUnits * T.occ / tiles_of(p.tile)), most));
    p.bound = tiles * p.splits;
    p.plane = ceil_div(out, 4) * 4;
    p.bytes = p.splits > 1 ? align256((size_t)p.splits * p.plane * sizeof(float)) : 256;
  }
  // ids are 32-bit; grouped_kernel has a workgroup to an item, and a launch fewer than 2^32 threads
  if (p.bound > (p.tile >= kDeep128 ? (int64_t)INT32_MAX : (int64_t)UINT32_MAX / 256) - 8)
    return fail(ML_EUNSUPPORTED, "grouped_matmul: too many tiles");
  return ML_OK;
}

// one workgroup to an item (rounded up for xcd_item), or persistent ones: all that fit where tiles may be split
int64_t grouped_blocks(const GroupedPlan& p) {
  const int64_t items = ceil_div(p.bound, kXcds) * kXcds, slots = kUnits * kTiles[p.tile].occ;
  return p.tile < kDeep128 ? items : p.splits > 1 ? slots : std::min(items, slots);
}

template <int DT, bool WG, bool BKC>
int grouped_launch(const GroupedPlan& p, GroupedArgs& a, hipStream_t st) {
  const TileShape& T = kTiles[p.tile];
  a.cols = fast_div(ceil_div(a.N, T.bn));
  a.layers = fast_div(a.groups / a.matrices);
  a.mtiles = fast_div(WG ? ceil_div(a.M, T.bm) : 1);
  const size_t lds = (2 * (size_t)a.groups + 3) * sizeof(int);  // edges, tiles of the segments
  const bool ring = p.tile >= kDeep128;
  const dim3 grid((unsigned)grouped_blocks(p)), blk(256);
  switch (p.tile) {
    case kFew:
      if constexpr (!WG) hipLaunchKernelGGL((grouped_kernel<DT, false, BKC, 32, 128, 1, 4>), grid, blk, lds, st, a);
      break;
    case kPlain: hipLaunchKernelGGL((grouped_kernel<DT, WG, BKC, 128, 128, 2, 2>), grid, blk, lds, st, a); break;
    case kDeep128:
      if constexpr (DT == ML_F32 && WG)
        hipLaunchKernelGGL((grouped_ring_kernel<DT, WG, BKC, 128, 128, 2, 2, stage_bytes(kDeep128, WG), 4, 2>), grid, blk, lds, st, a);
      break;
    case kWide128:
      if constexpr (DT != ML_F32 || !WG)
        hipLaunchKernelGGL((grouped_ring_kernel<DT, WG, BKC, 128, 128, 2, 2, stage_bytes(kWide128, WG), 2, 2>), grid, blk, lds, st, a);
      break;
    case kDeep128x256:
      if constexpr (DT != ML_F32)
        hipLaunchKernelGGL((grouped_ring_kernel<DT, WG, BKC, 128, 256, 2, 2, stage_bytes(kDeep128x256, WG), 3, 2>), grid, blk, lds, st, a);
      break;
    case kDeep256:
      if constexpr (DT != ML_F32)
        hipLaunchKernelGGL((grouped_ring_kernel<DT, WG, BKC, 256, 256, 2, 4, stage_bytes(kDeep256, WG), WG ? 4 : 2, 1>), grid,
                           dim3(512), lds, st, a);
      break;
  }
  int rc = check_launch("grouped_matmul");
  if (rc || !ring || a.splits == 1) return rc;
  hipLaunchKernelGGL(grouped_tail_kernel<DT>, grid, blk, lds, st, a, WG ? 1 : 0, T.bm, T.bn, p.tile == kDeep256 ? 4 : 2,
                     (int)grid.x / kXcds);
  return check_launch("grouped_matmul");
}

template <int DT>
int grouped_run(const ml_grouped_shape* s, const GroupedPlan& p, int which, const void* rows, const void* other,
                int transposed, const int64_t* offsets, void* out, void* ws, hipStream_t st) {
  ProfScope ps("grouped_matmul", st);
  GroupedArgs a{};
  a.offsets = offsets;
  a.equal = (int)(s->rows / s->groups);
  a.rows = (int)s->rows;
  a.given = (int)s->groups;
  a.groups = s->matrices == 1 ? 1 : a.given;
  a.matrices = (int)s->matrices;
  a.segments = p.merged ? a.matrices : a.groups;
  a.merged = p.merged;
  a.splits = p.splits;
  a.fewest = p.fewest;
  a.plane = p.plane;
  a.c = out;
  a.parts = (float*)ws;
  int rc;
  if (which == kWeight) {
    // stored (K, N): columns of x by columns of grad_out; stored (N, K): the other way round
    a.a = transposed ? other : rows;
    a.b = transposed ? rows : other;
    a.lda = transposed ? s->N : s->K;
    a.ldb = transposed ? s->K : s->N;
    a.M = (int)a.lda;
    a.N = (int)a.ldb;
    a.ldc = a.ldb;
    a.cstride = s->K * s->N;
    rc = grouped_launch<DT, true, false>(p, a, st);
  } else {
    a.a = rows;
    a.b = other;
    a.lda = a.K = (int)p.k;
    a.N = (int)p.n;
    a.ldb = transposed ? s->K : s->N;
    a.bstride = s->K * s->N;
    a.ldc = p.n;
    // the reduced index lies along a row of the matrix for the forward of (N, K) and for
    // the input gradient of (K, N)
    const bool kc = (which == kForward) == (transposed != 0);
    rc = kc ? grouped_launch<DT, false, true>(p, a, st) : grouped_launch<DT, false, false>(p, a, st);
  }
  if (rc || p.splits == 1 || p.tile >= kDeep128) return rc;  // ring kernels join their own parts
  const int64_t n = (which == kWeight ? s->matrices : 1) * p.m * p.n;
  hipLaunchKernelGGL(grouped_join_kernel<DT>, dim3((unsigned)ceil_div(n, kJoinQuads * 4)),
                     dim3(kJoinQuads * kJoinSlices), 0, st, (const float*)ws,
                     p.splits, p.plane, n, out);
  return check_launch("grouped_matmul");
}

// rows of whole 16-byte chunks
bool grouped_whole(const ml_grouped_shape* s, int dtype) {
  const int64_t ch = dtype == ML_F32 ? 4 : 8;
  return s && s->K % ch == 0 && s->N % ch == 0;
}

int grouped_call(const ml_grouped_shape* s, int dtype, int which, const void* rows, const void* other, int transposed,
                 const int64_t* offsets, void* out, void* ws, size_t ws_bytes, ml_stream_t stream) {
  GroupedPlan p;
  const bool aligned = grouped_whole(s, dtype) && ((uintptr_t)rows & 15) == 0 && ((uintptr_t)other & 15) == 0;
  const int rc = grouped_plan(s, dtype, which, transposed != 0, aligned, !offsets, p);
  if (rc) return rc;
  if (p.m == 0 || p.n == 0) return ML_OK;
  const bool reads = s->rows > 0 && p.k > 0;
  if (!offsets && s->rows % s->groups)
    return fail(ML_EINVAL, "grouped_matmul: without offsets the rows must divide into equal groups");
  if (!out || (reads && (!rows || !other))) return fail(ML_EINVAL, "grouped_matmul: null pointer");
  if (p.splits > 1 && (!ws || ws_bytes < p.bytes)) return fail(ML_EWORKSPACE, "grouped_matmul: workspace too small");
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case ML_F32: return grouped_run<ML_F32>(s, p, which, rows, other, transposed, offsets, out, ws, st);
    case ML_BF16: return grouped_run<ML_BF16>(s, p, which, rows, other, transposed, offsets, out, ws, st);
    default: return grouped_run<ML_F16>(s, p, which, rows, other, transposed, offsets, out, ws, st);
  }
}

}  // namespace
}  // namespace ml

using namespace ml;

extern "C" size_t ml_grouped_matmul_workspace_size(const ml_grouped_shape* s, int dtype, int product) {
  if (product < ML_GROUPED_FORWARD || product > ML_GROUPED_BACKWARD_WEIGHT) return 0;
  // over both storage orders, tensors that start on 16-byte boundaries or not, with and without offsets
  size_t most = 256;  // (a size of 0 stands for a refused shape)
  for (int i = 0; i < 8; ++i) {
    GroupedPlan p;
    if (grouped_plan(s, dtype, product, (i & 1) != 0, (i & 2) && grouped_whole(s, dtype), (i & 4) != 0, p)) return 0;
    most = std::max(most, p.bytes);
  }
  return most;
}

extern "C" int ml_grouped_matmul_plan(const ml_grouped_shape* s, int dtype, int product, int transposed, int aligned,
                                      int equal, ml_grouped_plan* plan) {
  if (product < ML_GROUPED_FORWARD || product > ML_GROUPED_BACKWARD_WEIGHT || !plan)
    return fail(ML_EINVAL, "grouped_matmul: unknown product, or no plan to write");
  if (aligned && !grouped_whole(s, dtype))
    return fail(ML_EINVAL, "grouped_matmul: rows of K or N elements are not on 16-byte boundaries");
  GroupedPlan p;
  const int rc = grouped_plan(s, dtype, product, transposed != 0, aligned != 0, equal != 0, p);
  if (rc) return rc;
  const TileShape& T = kTiles[p.tile];
  const bool ring = p.tile >= kDeep128;
  *plan = ml_grouped_plan{T.bm, T.bn, ring, ring ? stage_bytes(p.tile, product == kWeight) : 128, (int32_t)grouped_blocks(p),
                          p.splits, p.fewest, p.merged};
  return ML_OK;
}

extern "C" int ml_grouped_matmul_forward(const ml_grouped_shape* s, int dtype, const void* x, const void* weight,
                                         int transposed, const int64_t* offsets, void* y, void* workspace,
                                         size_t workspace_bytes, ml_stream_t stream) {
  return grouped_call(s, dtype, kForward, x, weight, transposed, offsets, y, workspace, workspace_bytes, stream);
}

extern "C" int ml_grouped_matmul_backward_input(const ml_grouped_shape* s, int dtype, const void* grad_out,
                                                const void* weight, int transposed, const int64_t* offsets,
                                                void* grad_input, void* workspace, size_t workspace_bytes,
                                                ml_stream_t stream) {
  return grouped_call(s, dtype, kInput, grad_out, weight, transposed, offsets, grad_input, workspace, workspace_bytes,
                      stream);
}

extern "C" int ml_grouped_matmul_backward_weight(const ml_grouped_shape* s, int dtype, const void* x,
                                                 const void* grad_out, int transposed, const int64_t* offsets,
                                                 void* grad_weight, void* workspace, size_t workspace_bytes,
                                                 ml_stream_t stream) {
  return grouped_call(s, dtype, kWeight, x, grad_out, transposed, offsets, grad_weight, workspace, workspace_bytes,
                      stream);
}
