// Grouped products: plans, launches and C entry points (the kernel: ml_grouped.h).
//
// Three tile shapes... see grouped_plan.
#include <algorithm>

#include "ml_grouped.h"

namespace ml {
namespace {

enum { kForward = 0, kInput = 1, kWeight = 2 };  // the three products

// Sums of the planes of a split reduction, in plane order, four elements a thread.
template <int DT>
__global__ __launch_bounds__(256) void grouped_join_kernel(const float* planes, int splits, int64_t plane, int64_t n,
                                                          void* c) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  f32x4_t v = *(const f32x4_t*)(planes + i);
  for (int s = 1; s < splits; ++s) v += *(const f32x4_t*)(planes + s * plane + i);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (i + q >= n) break;
    if constexpr (DT == ML_F32) ((float*)c)[i + q] = v[q];
    else ((uint16_t*)c)[i + q] = (uint16_t)GMma<DT>::pack(v[q], 0.f);
  }
}

struct GroupedPlan {
  int tile;                 // 0: 32 x 128, 1: 128 x 128
  int splits;
  int64_t m, n, k;          // output rows and columns, reduced length (weight gradient: mean rows per matrix)
  int64_t bound;            // workgroups
  int64_t plane;            // elements of a plane
  size_t bytes;             // workspace
};

constexpr int64_t kMaxGroups = 4000;   // their edges and tile counts fit the LDS beside the tiles
constexpr int64_t kMaxLength = 1 << 22;  // rows of a tile stay within 2^32 bytes of its first

int grouped_plan(const ml_grouped_shape* s, int dtype, int which, GroupedPlan& p) {
  if (!s || s->rows < 0 || s->K < 0 || s->N < 0 || s->groups < 1 || s->matrices < 1 || s->groups % s->matrices)
    return fail(ML_EINVAL, "grouped_matmul: invalid shape (groups must be a positive multiple of the matrices)");
  if (dtype != ML_F32 && dtype != ML_BF16 && dtype != ML_F16)
    return fail(ML_EINVAL, "grouped_matmul: unsupported dtype");
  if (s->groups > kMaxGroups)
    return fail(ML_EUNSUPPORTED, "grouped_matmul: at most " + std::to_string(kMaxGroups) + " groups are supported");
  if (s->rows > INT32_MAX || s->K > kMaxLength || s->N > kMaxLength)
    return fail(ML_EUNSUPPORTED, "grouped_matmul: at most 2^31 - 1 rows and K, N of at most 4194304 are supported");
  const int64_t bk = kStepBytes / (dtype == ML_F32 ? 4 : 2);
  p.m = which == kWeight ? s->K : s->rows;
  p.n = which == kInput ? s->K : s->N;
  p.k = which == kForward ? s->K : which == kInput ? s->N : ceil_div(s->rows, s->matrices);
  const int64_t used = std::min(s->groups, std::max<int64_t>(s->rows, 1));  // groups that can hold rows
  const int64_t each = ceil_div(s->rows, used);
  p.tile = which == kWeight || each > 32;
  const int64_t bm = p.tile ? 128 : 32, bn = 128, nt = ceil_div(p.n, bn);
  const int64_t likely = (which == kWeight ? s->matrices * ceil_div(p.m, bm) : used * ceil_div(each, bm)) * nt;
  // split the reduction where the tiles leave compute units without work: towards
  // two workgroups each, at least four steps to a part
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({512 / std::max<int64_t>(likely, 1), p.k / (4 * bk), 64}));
  const int64_t mt = which == kWeight ? s->matrices * ceil_div(p.m, bm)
                                      : s->rows / bm + std::min(s->groups + 2, s->rows);
  p.bound = ceil_div(mt * nt * p.splits, kXcds) * kXcds;
  if (p.bound > INT32_MAX) return fail(ML_EUNSUPPORTED, "grouped_matmul: too many tiles");
  const int64_t out = (which == kWeight ? s->matrices : 1) * p.m * p.n;
  p.plane = ceil_div(out, 4) * 4;
  p.bytes = p.splits > 1 ? align256((size_t)p.splits * p.plane * sizeof(float)) : 256;
  return ML_OK;
}

template <int DT, bool WG, bool BKC>
int grouped_launch(const GroupedPlan& p, const GroupedArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)p.bound);
  const size_t lds = (2 * (size_t)a.groups + 3) * sizeof(int);
  if constexpr (!WG) {
    if (p.tile == 0) {
      hipLaunchKernelGGL((grouped_kernel<DT, false, BKC, 32, 128, 1, 4>), grid, dim3(256), lds, st, a);
      return check_launch("grouped_matmul");
    }
  }
  hipLaunchKernelGGL((grouped_kernel<DT, WG, BKC, 128, 128, 2, 2>), grid, dim3(256), lds, st, a);
  return check_launch("grouped_matmul");
}

template <int DT>
int grouped_run(const ml_grouped_shape* s, const GroupedPlan& p, int which, const void* rows, const void* other,
                int transposed, const int64_t* offsets, void* out, void* ws, hipStream_t st) {
  ProfScope ps("grouped_matmul", st);
  GroupedArgs a{};
  a.offsets = offsets;
  a.rows = (int)s->rows;
  a.groups = (int)s->groups;
  a.matrices = (int)s->matrices;
  a.splits = p.splits;
  a.plane = p.plane;
  a.c = p.splits > 1 ? ws : out;
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
  if (rc || p.splits == 1) return rc;
  const int64_t n = (which == kWeight ? s->matrices : 1) * p.m * p.n;
  hipLaunchKernelGGL(grouped_join_kernel<DT>, dim3((unsigned)ceil_div(n, 1024)), dim3(256), 0, st, (const float*)ws,
                     p.splits, p.plane, n, out);
  return check_launch("grouped_matmul");
}

int grouped_call(const ml_grouped_shape* s, int dtype, int which, const void* rows, const void* other, int transposed,
                 const int64_t* offsets, void* out, void* ws, size_t ws_bytes, ml_stream_t stream) {
  GroupedPlan p;
  const int rc = grouped_plan(s, dtype, which, p);
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
  GroupedPlan p;
  if (product < ML_GROUPED_FORWARD || product > ML_GROUPED_BACKWARD_WEIGHT || grouped_plan(s, dtype, product, p))
    return 0;
  return p.bytes;
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
