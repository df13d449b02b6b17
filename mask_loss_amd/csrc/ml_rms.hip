// Root-mean-square norm over the last dimension of (rows, width), with the residual's addition in front of it,
// forward and backward, and with a result in microscaled values (ml_mx.h).
//
//   s = x + residual, rounded to the input's type (s = x without one),  r = 1 / sqrt(mean s^2 + eps),  h = s r,  y = h w
//   g = dy w:  ds = dsum + r (g - h mean(g h)),  dw = sum_rows dy h;  ds is x's and the residual's gradient
//
// The norm reads the rounded s, which is what the next residual addition and the backward see.  Bound by HBM: the
// forward reads x (and the residual) and writes y (and s) once, the backward reads s, dy (and dsum) and writes ds (16,384 x 1,024
// bf16 with a residual, 134 MB each way: 27 us, 5.0 TB/s, and 28 + 4; 8,192 x 4,096 to e4m3 46 us, 5.1 TB/s; a copy of 1 GiB
// runs at 5.2).
// As the layer norm does (ml_norm.hip), a row stays in registers, T threads to a row; there is one
// reduction a row.  Statistics and sums are float32, each result is rounded once; dw as one row of
// partial sums per workgroup, added in a fixed order.  Rows that are not whole 16-byte vectors go element by element: 16-byte
// accesses at any alignment, which the rows by expert gain from, cost here (4,097 x 1,153 f16 forward / backward 8.9 / 12.8 us,
// with them 10.9 / 17.1); so does a wave to a row where four are taken (16,384 x 2,048 bf16 45 / 50 us, with one 57 / 63).
#include <algorithm>

#include "ml_mx.h"

namespace ml {
namespace {

// T threads hold a row, NV vectors of 16 bytes (V elements) each; vector k of thread t starts at column (k T + t) V.
// Rows are whole vectors, or V is 1.
// RES: with a residual; MX: y as codes and scales.
template <int DT, int V, int NV, int T, bool RES, bool MX>
__global__ __launch_bounds__(wg_threads(T)) void rms_fwd_kernel(const void* xv, const void* rv, const void* w, int pf32,
                                                                int64_t rows, int64_t D, float eps, int format, void* sv,
                                                                void* yv, uint8_t* scales, float* rstd) {
  using R = typename Elem<DT>::raw;
  using VT = RowChunk<DT, V>;
  constexpr int G = wg_threads(T) / T;  // rows at once
  __shared__ float red[2][16];
  const R *x = (const R*)xv, *res = (const R*)rv;
  const int t = threadIdx.x % T;
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / T;
  const float inv = 1.f / (float)D;

  float wr[NV * V];
  bool ok[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int64_t c = (int64_t)(k * T + t) * V;
    ok[k] = c < D;
#pragma unroll
    for (int j = 0; j < V; ++j) wr[k * V + j] = ok[k] && w ? param_at<DT>(w, pf32, c + j) : 1.f;
  }
  VT cur[NV], nxt[NV], cr[RES ? NV : 1], nr[RES ? NV : 1];
  auto load = [&](VT(&v)[NV], VT(&u)[RES ? NV : 1], int64_t r) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int n = ok[k] && r < rows ? V : 0;
      const int64_t at = r * D + (int64_t)(k * T + t) * V;
      v[k].template load<true>(x + at, n);
      if constexpr (RES) u[k].template load<true>(res + at, n);
    }
  };
  load(cur, cr, row);
  int flip = 0;
  // every thread of the workgroup makes the same number of rounds (barriers)
  for (int64_t base = (int64_t)blockIdx.x * G; base < rows; base += step, row += step, flip ^= 1) {
    load(nxt, nr, row + step);
    float f[NV * V], s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if constexpr (RES) {
#pragma unroll
        for (int j = 0; j < V; ++j) cur[k].e[j] = from_f32<DT>(to_f32<DT>(cur[k].e[j]) + to_f32<DT>(cr[k].e[j]));
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        f[k * V + j] = to_f32<DT>(cur[k].e[j]);
        s[0] = fmaf(f[k * V + j], f[k * V + j], s[0]);
      }
    }
    row_sum<T>(s, red[flip]);
    const float r = 1.f / sqrtf(fmaf(s[0], inv, eps));
    const bool in = row < rows;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t at = row * D + (int64_t)(k * T + t) * V;
      if constexpr (RES) {
        if (in && ok[k]) cur[k].template store<true>((R*)sv + at, V);
      }
      if constexpr (MX) {
        float y[V];
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] = f[k * V + j] * r * wr[k * V + j];
        const uint32_t code = mx_scale(mx_lane_max<kMxBlock / V>(mx_max(y)), format);  // (outside the branch: all lanes)
        if (ok[k] && in) {
          mx_store(y, code, format, at, (uint8_t*)yv);
          if (at % kMxBlock == 0) scales[at / kMxBlock] = (uint8_t)code;
        }
      } else if (in && ok[k]) {
        VT o;
#pragma unroll
        for (int j = 0; j < V; ++j) o.e[j] = from_f32<DT>(f[k * V + j] * r * wr[k * V + j]);
        o.template store<true>((R*)yv + at, V);
      }
    }
    if (in && t == 0 && rstd) rstd[row] = r;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      cur[k] = nxt[k];
      if constexpr (RES) cr[k] = nr[k];
    }
  }
}

// ds, and one row of partial sums of dw per workgroup, part[blockIdx][D] (part null: ds alone; dx null: the
// sums alone).  SUM: the sum's own gradient comes in, too.
template <int DT, int V, int NV, int T, bool SUM>
__global__ __launch_bounds__(wg_threads(T)) void rms_bwd_kernel(const void* gv, const void* uv, const void* xv,
                                                                const void* w, int pf32, const float* rstd, int64_t rows,
                                                                int64_t D, void* dxv, float* part) {
  using R = typename Elem<DT>::raw;
  using VT = RowChunk<DT, V>;
  constexpr int G = wg_threads(T) / T, E = NV * V;
  __shared__ float red[2][16];
  const R *x = (const R*)xv, *dy = (const R*)gv, *du = (const R*)uv;
  R* dx = (R*)dxv;
  const int t = threadIdx.x % T;
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / T;
  const float inv = 1.f / (float)D;

  float wr[E], dw[E];
  bool ok[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int64_t c = (int64_t)(k * T + t) * V;
    ok[k] = c < D;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      wr[k * V + j] = ok[k] && w ? param_at<DT>(w, pf32, c + j) : 1.f;
      dw[k * V + j] = 0.f;
    }
  }
  VT cx[NV], cg[NV], nx[NV], ng[NV], cu[SUM ? NV : 1], nu[SUM ? NV : 1];
  float cr, nr;
  auto load = [&](VT(&vx)[NV], VT(&vg)[NV], VT(&vu)[SUM ? NV : 1], float& r, int64_t i) {
    const bool in = i < rows;
    r = in ? rstd[i] : 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t o = i * D + (int64_t)(k * T + t) * V;
      const int n = ok[k] && in ? V : 0;
      vx[k].template load<true>(x + o, n);
      vg[k].template load<true>(dy + o, n);
      if constexpr (SUM) vu[k].template load<true>(du + o, n);
    }
  };
  load(cx, cg, cu, cr, row);
  int flip = 0;
  for (int64_t base = (int64_t)blockIdx.x * G; base < rows; base += step, row += step, flip ^= 1) {
    load(nx, ng, nu, nr, row + step);
    float h[E], g[E], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < E; ++i) {
      // columns past the row and rows past the last are zero and count for nothing
      const float d = to_f32<DT>(cg[i / V].e[i % V]);
      h[i] = to_f32<DT>(cx[i / V].e[i % V]) * cr;
      g[i] = d * wr[i];
      dw[i] = fmaf(d, h[i], dw[i]);
      s[0] = fmaf(g[i], h[i], s[0]);
    }
    if (dx) {
      row_sum<T>(s, red[flip]);
      if (row < rows) {
        const float c = s[0] * inv;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          if (!ok[k]) continue;
          VT o;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int i = k * V + j;
            float v = cr * (g[i] - h[i] * c);
            if constexpr (SUM) v += to_f32<DT>(cu[k].e[j]);
            o.e[j] = from_f32<DT>(v);
          }
          o.template store<true>(dx + row * D + (int64_t)(k * T + t) * V, V);
        }
      }
    }
    cr = nr;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      cx[k] = nx[k];
      cg[k] = ng[k];
      if constexpr (SUM) cu[k] = nu[k];
    }
  }
  if (!part) return;
  // add the workgroup's G row groups, then write its row of partial sums
  float* pw = part + (int64_t)blockIdx.x * D;
  if constexpr (G == 1) {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (ok[i / V]) pw[(int64_t)((i / V) * T + t) * V + i % V] = dw[i];
  } else {
    __shared__ float acc[kNormThreads];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      __syncthreads();
      acc[threadIdx.x] = dw[i];
      __syncthreads();
      if (threadIdx.x < T && ok[i / V]) {
        float a = 0.f;
#pragma unroll
        for (int q = 0; q < G; ++q) a += acc[q * T + t];
        pw[(int64_t)((i / V) * T + t) * V + i % V] = a;
      }
    }
  }
}

// ---- rows of any width: a workgroup per row, read twice ---------------------------
template <int DT, bool RES, bool MX>
__global__ __launch_bounds__(kWideThreads) void rms_fwd_wide_kernel(const void* xv, const void* rv, const void* w, int pf32,
                                                                    int64_t rows, int64_t D, float eps, int format,
                                                                    void* sv, void* yv, uint8_t* scales, float* rstd) {
  using R = typename Elem<DT>::raw;
  using VT = RowChunk<DT>;
  constexpr int V = VT::V;
  __shared__ float red[2][16];
  const float inv = 1.f / (float)D;
  int flip = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, flip ^= 1) {
    const R* x = (const R*)xv + row * D;
    const R* res = (const R*)rv + (RES ? row * D : 0);
    R* sum = (R*)sv + (RES ? row * D : 0);
    float s[1] = {0.f};
    for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += kWideThreads * V) {
      VT v;
      v.load(x + c, D - c);
      if constexpr (RES) {
        VT u;
        u.load(res + c, D - c);
#pragma unroll
        for (int j = 0; j < V; ++j) v.e[j] = from_f32<DT>(to_f32<DT>(v.e[j]) + to_f32<DT>(u.e[j]));
        v.store(sum + c, D - c);  // (read again by this thread alone)
      }
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] = fmaf(to_f32<DT>(v.e[j]), to_f32<DT>(v.e[j]), s[0]);
    }
    row_sum<kWideThreads>(s, red[flip]);
    const float r = 1.f / sqrtf(fmaf(s[0], inv, eps));
    const R* from = RES ? sum : x;
    for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += kWideThreads * V) {
      VT v;
      v.load(from + c, D - c);
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = to_f32<DT>(v.e[j]) * r * (w && c + j < D ? param_at<DT>(w, pf32, c + j) : 1.f);
      const int64_t at = row * D + c;
      if constexpr (MX) {
        // (a block's lanes leave the loop together: D is whole blocks)
        const uint32_t code = mx_scale(mx_lane_max<kMxBlock / V>(mx_max(y)), format);
        mx_store(y, code, format, at, (uint8_t*)yv);
        if (at % kMxBlock == 0) scales[at / kMxBlock] = (uint8_t)code;
      } else {
        VT o;
#pragma unroll
        for (int j = 0; j < V; ++j) o.e[j] = from_f32<DT>(y[j]);
        o.store((R*)yv + at, D - c);
      }
    }
    if (threadIdx.x == 0 && rstd) rstd[row] = r;
  }
}

template <int DT, bool SUM>
__global__ __launch_bounds__(kWideThreads) void rms_bwd_wide_kernel(const void* gv, const void* uv, const void* xv,
                                                                    const void* w, int pf32, const float* rstd,
                                                                    int64_t rows, int64_t D, void* dxv) {
  using R = typename Elem<DT>::raw;
  using VT = RowChunk<DT>;
  constexpr int V = VT::V;
  __shared__ float red[2][16];
  const float inv = 1.f / (float)D;
  int flip = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, flip ^= 1) {
    const R *x = (const R*)xv + row * D, *dy = (const R*)gv + row * D;
    const R* du = (const R*)uv + (SUM ? row * D : 0);
    R* dx = (R*)dxv + row * D;
    const float r = rstd[row];
    float s[1] = {0.f};
    for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += kWideThreads * V) {
      VT vx, vg;
      vx.load(x + c, D - c);
      vg.load(dy + c, D - c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float g = to_f32<DT>(vg.e[j]) * (w && c + j < D ? param_at<DT>(w, pf32, c + j) : 1.f);
        s[0] = fmaf(g, to_f32<DT>(vx.e[j]) * r, s[0]);
      }
    }
    row_sum<kWideThreads>(s, red[flip]);
    const float k = s[0] * inv;
    for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += kWideThreads * V) {
      VT vx, vg, vu, o;
      vx.load(x + c, D - c);
      vg.load(dy + c, D - c);
      if constexpr (SUM) vu.load(du + c, D - c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float g = to_f32<DT>(vg.e[j]) * (w && c + j < D ? param_at<DT>(w, pf32, c + j) : 1.f);
        float v = r * (g - to_f32<DT>(vx.e[j]) * r * k);
        if constexpr (SUM) v += to_f32<DT>(vu.e[j]);
        o.e[j] = from_f32<DT>(v);
      }
      o.store(dx + c, D - c);
    }
  }
}

// partial sums of 256 columns over the rows blockIdx.y, blockIdx.y + gridDim.y, ...
template <int DT>
__global__ __launch_bounds__(kNormThreads) void rms_param_wide_kernel(const void* gv, const void* xv, const float* rstd,
                                                                      int64_t rows, int64_t D, float* part) {
  using R = typename Elem<DT>::raw;
  const int64_t c = (int64_t)blockIdx.x * kNormThreads + threadIdx.x;
  if (c >= D) return;
  float dw = 0.f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y)
    dw = fmaf(to_f32<DT>(((const R*)gv)[row * D + c]), to_f32<DT>(((const R*)xv)[row * D + c]) * rstd[row], dw);
  part[(int64_t)blockIdx.y * D + c] = dw;
}

// Workgroups: as the layer norm's.
int64_t rms_fwd_blocks(int T, int E) { return T > kNormThreads || (T == kNormThreads && E > 8) ? 512 : 1024; }
int64_t rms_bwd_blocks(int64_t rows, int64_t D) {
  if (D > kNormHeld) return std::min<int64_t>(rows, 64);
  const int T = kNormCfgs[norm_cfg(D)].T;
  const int64_t rounds = ceil_div(rows, wg_threads(T) / T);
  return std::min<int64_t>(rounds, T > kNormThreads ? 256 : T < kNormThreads ? 768 : 512);
}

struct RmsForward {
  const void *x, *res, *w;
  int pf32;
  int64_t rows, D;
  float eps;
  int format;
  void *sum, *y;
  uint8_t* scales;
  float* rstd;
};

template <int DT, int V, bool RES, bool MX>
int rms_forward_launch(const RmsForward& a, hipStream_t st) {
  if (a.D > kNormHeld) {
    hipLaunchKernelGGL((rms_fwd_wide_kernel<DT, RES, MX>), dim3((unsigned)std::min<int64_t>(a.rows, 65536)),
                       dim3(kWideThreads), 0, st, a.x, a.res, a.w, a.pf32, a.rows, a.D, a.eps, a.format, a.sum, a.y, a.scales,
                       a.rstd);
    return check_launch("rms_norm");
  }
  return norm_dispatch(norm_cfg(a.D), [&](auto tc, auto ec) {
    constexpr int T = decltype(tc)::value, E = decltype(ec)::value;
    const int64_t rounds = ceil_div(a.rows, wg_threads(T) / T);
    hipLaunchKernelGGL((rms_fwd_kernel<DT, V, E / V, T, RES, MX>),
                       dim3((unsigned)std::min<int64_t>(rounds, rms_fwd_blocks(T, E))), dim3(wg_threads(T)), 0, st, a.x, a.res,
                       a.w, a.pf32, a.rows, a.D, a.eps, a.format, a.sum, a.y, a.scales, a.rstd);
    return check_launch("rms_norm");
  });
}

template <int DT, bool MX>
int rms_forward(const RmsForward& a, hipStream_t st) {
  ProfScope ps("rms_norm", st);
  constexpr int V16 = RowChunk<DT>::V;
  if (a.D % V16 == 0)
    return a.res ? rms_forward_launch<DT, V16, true, MX>(a, st) : rms_forward_launch<DT, V16, false, MX>(a, st);
  if constexpr (!MX) return a.res ? rms_forward_launch<DT, 1, true, MX>(a, st) : rms_forward_launch<DT, 1, false, MX>(a, st);
  return ML_OK;  // (MX: rows are whole blocks)
}

struct RmsBackward {
  const void *dy, *du, *x, *w;
  int pf32;
  const float* rstd;
  int64_t rows, D;
  void *dx, *dw;
  float* part;
};

template <int DT, int V, bool SUM>
int rms_backward_launch(const RmsBackward& a, hipStream_t st) {
  const int64_t nblk = rms_bwd_blocks(a.rows, a.D);
  if (a.D > kNormHeld) {
    int rc = ML_OK;
    if (a.dx) {
      hipLaunchKernelGGL((rms_bwd_wide_kernel<DT, SUM>), dim3((unsigned)std::min<int64_t>(a.rows, 65536)),
                         dim3(kWideThreads), 0, st, a.dy, a.du, a.x, a.w, a.pf32, a.rstd, a.rows, a.D, a.dx);
      rc = check_launch("rms_norm_backward");
    }
    if (rc || !a.dw) return rc;
    hipLaunchKernelGGL(rms_param_wide_kernel<DT>, dim3((unsigned)ceil_div(a.D, kNormThreads), (unsigned)nblk),
                       dim3(kNormThreads), 0, st, a.dy, a.x, a.rstd, a.rows, a.D, a.part);
    return check_launch("rms_norm_backward");
  }
  return norm_dispatch(norm_cfg(a.D), [&](auto tc, auto ec) {
    constexpr int T = decltype(tc)::value, E = decltype(ec)::value;
    hipLaunchKernelGGL((rms_bwd_kernel<DT, V, E / V, T, SUM>), dim3((unsigned)nblk), dim3(wg_threads(T)), 0, st, a.dy, a.du,
                       a.x, a.w, a.pf32, a.rstd, a.rows, a.D, a.dx, a.dw ? a.part : nullptr);
    return check_launch("rms_norm_backward");
  });
}

template <int DT>
int rms_backward(const RmsBackward& a, hipStream_t st) {
  ProfScope ps("rms_norm_backward", st);
  int rc = ML_OK;
  if (a.rows > 0) {
    constexpr int V16 = RowChunk<DT>::V;
    if (a.D % V16 == 0) rc = a.du ? rms_backward_launch<DT, V16, true>(a, st) : rms_backward_launch<DT, V16, false>(a, st);
    else rc = a.du ? rms_backward_launch<DT, 1, true>(a, st) : rms_backward_launch<DT, 1, false>(a, st);
  }
  if (rc || !a.dw) return rc;
  hipLaunchKernelGGL(norm_param_kernel<DT>, dim3((unsigned)ceil_div(a.D, kParamCols), 1), dim3(kParamCols * kParamSlices), 0,
                     st, a.part, rms_bwd_blocks(a.rows, a.D), a.D, a.pf32, a.dw, nullptr);
  return check_launch("rms_norm_backward");
}

int rms_check(const char* who, int dtype, int pdtype, int64_t rows, int64_t width) {
  const std::string name(who);
  if (dtype != ML_F32 && dtype != ML_BF16 && dtype != ML_F16) return fail(ML_EINVAL, name + ": unsupported dtype");
  if (pdtype != dtype && pdtype != ML_F32)
    return fail(ML_EINVAL, name + ": the weight must have the input's dtype or be float32");
  if (rows < 0 || width <= 0) return fail(ML_EINVAL, name + ": rows must not be negative, width must be positive");
  // norm_param_kernel takes 32 threads a column, a launch fewer than 2^32
  if (width > ((int64_t)1 << 26) || (rows > 0 && width > INT64_MAX / 8 / rows))
    return fail(ML_EUNSUPPORTED, name + ": too many elements");
  return ML_OK;
}

}  // namespace
}  // namespace ml

using namespace ml;

extern "C" int ml_rms_norm_forward(int dtype, int param_dtype, const void* x, const void* residual, const void* weight,
                                   int64_t rows, int64_t width, float eps, void* sum, void* y, float* rstd,
                                   ml_stream_t stream) {
  int rc = rms_check("rms_norm", dtype, param_dtype, rows, width);
  if (rc) return rc;
  if (!(eps >= 0.f)) return fail(ML_EINVAL, "rms_norm: eps must not be negative");
  if (rows == 0) return ML_OK;
  if (!x || !y || !residual != !sum) return fail(ML_EINVAL, "rms_norm: null pointer (residual and sum go together)");
  const RmsForward a{x, residual, weight, param_dtype == ML_F32, rows, width, eps, 0, sum, y, nullptr, rstd};
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case ML_F32: return rms_forward<ML_F32, false>(a, st);
    case ML_BF16: return rms_forward<ML_BF16, false>(a, st);
    default: return rms_forward<ML_F16, false>(a, st);
  }
}

extern "C" int ml_rms_norm_mx_forward(int dtype, int param_dtype, const void* x, const void* residual, const void* weight,
                                      int64_t rows, int64_t width, float eps, int format, void* sum, void* codes,
                                      uint8_t* scales, ml_stream_t stream) {
  int rc = rms_check("rms_norm_mx", dtype, param_dtype, rows, width);
  if (rc) return rc;
  if (!(eps >= 0.f)) return fail(ML_EINVAL, "rms_norm_mx: eps must not be negative");
  if (!mx_format(format)) return fail(ML_EINVAL, "rms_norm_mx: unknown format");
  if (width % kMxBlock) return fail(ML_EINVAL, "rms_norm_mx: width must be a multiple of 32");
  if (rows == 0) return ML_OK;
  if (!x || !codes || !scales || !residual != !sum)
    return fail(ML_EINVAL, "rms_norm_mx: null pointer (residual and sum go together)");
  if (!aligned16(x) || !aligned16(residual) || !aligned16(sum) || !aligned16(codes))
    return fail(ML_EINVAL, "rms_norm_mx: x, residual, sum and codes must be 16-byte aligned");
  const RmsForward a{x, residual, weight, param_dtype == ML_F32, rows, width, eps, format, sum, codes, scales, nullptr};
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case ML_F32: return rms_forward<ML_F32, true>(a, st);
    case ML_BF16: return rms_forward<ML_BF16, true>(a, st);
    default: return rms_forward<ML_F16, true>(a, st);
  }
}

extern "C" size_t ml_rms_norm_backward_workspace_size(int64_t rows, int64_t width) {
  if (rms_check("rms_norm", ML_F32, ML_F32, rows, width)) return 0;
  return std::max<size_t>(256, align256((size_t)rms_bwd_blocks(rows, width) * (size_t)width * sizeof(float)));
}

extern "C" int ml_rms_norm_backward(int dtype, int param_dtype, const void* grad_out, const void* grad_sum, const void* sum,
                                    const void* weight, const float* rstd, int64_t rows, int64_t width, void* grad_input,
                                    void* grad_weight, void* workspace, size_t workspace_bytes, ml_stream_t stream) {
  int rc = rms_check("rms_norm", dtype, param_dtype, rows, width);
  if (rc) return rc;
  if (!grad_input && !grad_weight) return ML_OK;
  if (rows > 0 && (!grad_out || !sum || !rstd)) return fail(ML_EINVAL, "rms_norm: null pointer");
  if (grad_weight && (!workspace || workspace_bytes < ml_rms_norm_backward_workspace_size(rows, width)))
    return fail(ML_EWORKSPACE, "rms_norm: workspace too small");
  const RmsBackward a{grad_out, grad_sum, sum, weight, param_dtype == ML_F32, rstd, rows, width, grad_input, grad_weight,
                      (float*)workspace};
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case ML_F32: return rms_backward<ML_F32>(a, st);
    case ML_BF16: return rms_backward<ML_BF16>(a, st);
    default: return rms_backward<ML_F16>(a, st);
  }
}
