// Layer norm over the last dimension of (rows, width), forward and backward.
//
//   m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), h = (x - m) r,  y = h w + b
//   g = dy w:  dx = r (g - mean g - h mean(g h)),  dw = sum_rows dy h,  db = sum_rows dy
//
// Both directions are bound by HBM: the forward reads x and writes y once, the
// backward reads x and dy and writes dx once (172,032 x 256 f16: forward 32 us, 5.5
// TB/s; backward 46 + 5 us, 5.2 TB/s; a copy of 1 GiB runs at 5.2).  A row is therefore held in
// registers between its reductions, T threads to a row and 8 or 16 elements
// to a thread (kNormCfgs), so that the variance is summed about the mean (no cancellation)
// without a second read.  Statistics, sums and the weights' gradients are
// float32 whatever the input's type; each result is rounded once.
//
// dw and db are sums over all rows: each thread keeps the sums of its own
// columns in registers over every row that its workgroup takes, the workgroup
// adds its row groups in LDS and writes one row of partial sums, and
// norm_param_kernel adds those rows in a fixed order (no atomics, so a result
// does not change between runs).
//
// Rows wider than 1024 threads hold (8 elements each: 16 in the backward go past
// 128 registers per lane) go through norm_fwd_wide_kernel and
// norm_bwd_wide_kernel, which read a row once per reduction, and
// norm_param_wide_kernel, which sums columns over a slice of the rows.
#include <algorithm>

#include "ml_internal.h"

namespace ml {
namespace {

template <int DT>
struct Elem {
  using raw = uint16_t;
};
template <>
struct Elem<ML_F32> {
  using raw = float;
};

template <int DT>
__device__ __forceinline__ float to_f32(typename Elem<DT>::raw v) {
  if constexpr (DT == ML_F32) return v;
  else if constexpr (DT == ML_BF16) return bf16_lo((uint32_t)v);
  else return (float)__builtin_bit_cast(_Float16, v);
}
template <int DT>
__device__ __forceinline__ typename Elem<DT>::raw from_f32(float v) {
  if constexpr (DT == ML_F32) return v;
  else if constexpr (DT == ML_BF16) return (uint16_t)(pack_bf16x2(v, 0.f) & 0xFFFFu);
  else return __builtin_bit_cast(uint16_t, (_Float16)v);
}

// A weight or bias element: the input's type or float32.
template <int DT>
__device__ __forceinline__ float param_at(const void* p, int f32, int64_t i) {
  return f32 ? ((const float*)p)[i] : to_f32<DT>(((const typename Elem<DT>::raw*)p)[i]);
}
template <int DT>
__device__ __forceinline__ void param_set(void* p, int f32, int64_t i, float v) {
  if (f32) ((float*)p)[i] = v;
  else ((typename Elem<DT>::raw*)p)[i] = from_f32<DT>(v);
}

// V consecutive elements as they lie in memory: 16 bytes, or one element.
template <int DT, int V>
struct alignas(V == 1 ? sizeof(typename Elem<DT>::raw) : 16) Vec {
  typename Elem<DT>::raw e[V];
};

// v plus the value of another lane, in the vector ALU: quad neighbours (xor 1, xor 2), the mirrored
// lane of 8 and of 16 (whose fours and eights hold one value by then), the other 16 and the
// other 32.  About 10 cycles a step where a shuffle through LDS takes 60.
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int T>
__device__ __forceinline__ float lane_sum(float v) {
  static_assert(T == 16 || T == 32 || T == 64, "lanes");
  v = add_dpp<0xB1>(v);   // quad_perm 1 0 3 2
  v = add_dpp<0x4E>(v);   // quad_perm 2 3 0 1
  v = add_dpp<0x141>(v);  // row_half_mirror
  v = add_dpp<0x140>(v);  // row_mirror
  if constexpr (T >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (T >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// Sums of N values over the T threads of a row, the same in all of them; `s` is
// one of two alternating LDS buffers, so one barrier a sum is enough.
template <int T, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* s) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane_sum<(T < 64 ? T : 64)>(v[i]);
  if constexpr (T > 64) {
    constexpr int W = T / 64;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s[i * W + wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int j = 0; j < W; ++j) v[i] += s[i * W + j];
    }
  }
}

constexpr int kNormThreads = 256;
constexpr int wg_threads(int T) { return T > kNormThreads ? T : kNormThreads; }

// T threads hold a row, NV vectors of V elements each; vector k of thread t
// starts at column (k T + t) V.
template <int DT, int V, int NV, int T>
__global__ __launch_bounds__(wg_threads(T)) void norm_fwd_kernel(const void* xv, const void* w, const void* b,
                                                                 int pf32, int64_t rows, int64_t D, float eps,
                                                                 void* yv, float* mean, float* rstd) {
  using R = typename Elem<DT>::raw;
  using VT = Vec<DT, V>;
  constexpr int G = wg_threads(T) / T;  // rows at once
  __shared__ float red[2][16];
  const R* x = (const R*)xv;
  R* y = (R*)yv;
  const int t = threadIdx.x % T;
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / T;
  const float inv = 1.f / (float)D;

  float wr[NV * V], br[NV * V];
  bool ok[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int64_t c = (int64_t)(k * T + t) * V;
    ok[k] = c < D;  // a vector lies inside the row as a whole
#pragma unroll
    for (int j = 0; j < V; ++j) {
      wr[k * V + j] = ok[k] && w ? param_at<DT>(w, pf32, c + j) : 1.f;
      br[k * V + j] = ok[k] && b ? param_at<DT>(b, pf32, c + j) : 0.f;
    }
  }
  VT cur[NV], nxt[NV];
  auto load = [&](VT(&v)[NV], int64_t r) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (ok[k] && r < rows) v[k] = *(const VT*)(x + r * D + (int64_t)(k * T + t) * V);
      else v[k] = VT{};
  };
  load(cur, row);
  // every thread of the workgroup makes the same number of rounds (barriers)
  for (int64_t base = (int64_t)blockIdx.x * G; base < rows; base += step, row += step) {
    load(nxt, row + step);
    float f[NV * V], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV * V; ++i) {
      f[i] = to_f32<DT>(cur[i / V].e[i % V]);
      s[0] += f[i];
    }
    row_sum<T>(s, red[0]);
    const float m = s[0] * inv;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NV * V; ++i) {
      f[i] = ok[i / V] ? f[i] - m : 0.f;
      s[0] = fmaf(f[i], f[i], s[0]);
    }
    row_sum<T>(s, red[1]);
    const float r = 1.f / sqrtf(fmaf(s[0], inv, eps));
    if (row < rows) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (!ok[k]) continue;
        VT o;
#pragma unroll
        for (int j = 0; j < V; ++j)
          o.e[j] = from_f32<DT>(fmaf(f[k * V + j] * r, wr[k * V + j], br[k * V + j]));
        *(VT*)(y + row * D + (int64_t)(k * T + t) * V) = o;
      }
      if (t == 0 && mean) {
        mean[row] = m;
        rstd[row] = r;
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) cur[k] = nxt[k];
  }
}

// dx, and one row of partial sums of dw and db per workgroup:
// part[0][blockIdx][D] and part[1][blockIdx][D] (part null: dx alone; dx null:
// the sums alone).
template <int DT, int V, int NV, int T>
__global__ __launch_bounds__(wg_threads(T)) void norm_bwd_kernel(const void* gv, const void* xv, const void* w,
                                                                 int pf32, const float* mean, const float* rstd,
                                                                 int64_t rows, int64_t D, void* dxv, float* part) {
  using R = typename Elem<DT>::raw;
  using VT = Vec<DT, V>;
  constexpr int G = wg_threads(T) / T, E = NV * V;
  __shared__ float red[2][2 * 16];
  const R *x = (const R*)xv, *dy = (const R*)gv;
  R* dx = (R*)dxv;
  const int t = threadIdx.x % T;
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / T;
  const float inv = 1.f / (float)D;

  float wr[E], dw[E], db[E];
  bool ok[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int64_t c = (int64_t)(k * T + t) * V;
    ok[k] = c < D;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      wr[k * V + j] = ok[k] && w ? param_at<DT>(w, pf32, c + j) : 1.f;
      dw[k * V + j] = db[k * V + j] = 0.f;
    }
  }
  VT cx[NV], cg[NV], nx[NV], ng[NV];
  float cm, cr, nm, nr;
  auto load = [&](VT(&vx)[NV], VT(&vg)[NV], float& m, float& r, int64_t i) {
    const bool in = i < rows;
    m = in ? mean[i] : 0.f;
    r = in ? rstd[i] : 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t o = i * D + (int64_t)(k * T + t) * V;
      if (ok[k] && in) {
        vx[k] = *(const VT*)(x + o);
        vg[k] = *(const VT*)(dy + o);
      } else {
        vx[k] = vg[k] = VT{};
      }
    }
  };
  load(cx, cg, cm, cr, row);
  int flip = 0;
  for (int64_t base = (int64_t)blockIdx.x * G; base < rows; base += step, row += step, flip ^= 1) {
    load(nx, ng, nm, nr, row + step);
    float h[E], g[E], s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float d = to_f32<DT>(cg[i / V].e[i % V]);
      // columns past the row and rows past the last have d = 0 and count for nothing
      h[i] = ok[i / V] ? (to_f32<DT>(cx[i / V].e[i % V]) - cm) * cr : 0.f;
      g[i] = d * wr[i];
      dw[i] = fmaf(d, h[i], dw[i]);
      db[i] += d;
      s[0] += g[i];
      s[1] = fmaf(g[i], h[i], s[1]);
    }
    if (dx) {
      row_sum<T>(s, red[flip]);
      if (row < rows) {
        const float a = s[0] * inv, c = s[1] * inv;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          if (!ok[k]) continue;
          VT o;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int i = k * V + j;
            o.e[j] = from_f32<DT>(cr * (g[i] - a - h[i] * c));
          }
          *(VT*)(dx + row * D + (int64_t)(k * T + t) * V) = o;
        }
      }
    }
    cm = nm;
    cr = nr;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      cx[k] = nx[k];
      cg[k] = ng[k];
    }
  }
  if (!part) return;
  // add the workgroup's G row groups, then write its row of partial sums
  const int64_t plane = (int64_t)gridDim.x * D;
  float* pw = part + (int64_t)blockIdx.x * D;
  if constexpr (G == 1) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int64_t c = (int64_t)((i / V) * T + t) * V + i % V;
      if (!ok[i / V]) continue;
      pw[c] = dw[i];
      pw[plane + c] = db[i];
    }
  } else {
    __shared__ float acc[2][kNormThreads];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      __syncthreads();
      acc[0][threadIdx.x] = dw[i];
      acc[1][threadIdx.x] = db[i];
      __syncthreads();
      if (threadIdx.x < T && ok[i / V]) {
        float a = 0.f, c = 0.f;
#pragma unroll
        for (int q = 0; q < G; ++q) {
          a += acc[0][q * T + t];
          c += acc[1][q * T + t];
        }
        const int64_t col = (int64_t)((i / V) * T + t) * V + i % V;
        pw[col] = a;
        pw[plane + col] = c;
      }
    }
  }
}

// dw[c], db[c]: sums of n partial rows, 32 columns and 32 slices of the rows to a
// workgroup (grid y: dw, db), in an order that the shape alone fixes.
constexpr int kParamCols = 32, kParamSlices = 32;
template <int DT>
__global__ __launch_bounds__(kParamCols* kParamSlices) void norm_param_kernel(const float* part, int64_t n,
                                                                             int64_t D, int pf32, void* dw,
                                                                             void* db) {
  __shared__ float s[kParamSlices][kParamCols + 1];
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int cl = threadIdx.x % kParamCols, sl = threadIdx.x / kParamCols;
  const int64_t c = (int64_t)blockIdx.x * kParamCols + cl;
  const float* p = part + (int64_t)blockIdx.y * n * D;
  float a = 0.f;
  if (c < D) {
    // eight loads in flight: a slice is bound by their latency
    constexpr int kFlight = 8;
    for (int64_t i = sl; i < n; i += kParamSlices * kFlight) {
      float v[kFlight];
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        const int64_t r = i + j * kParamSlices;
        v[j] = r < n ? p[r * D + c] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < kFlight; ++j) a += v[j];
    }
  }
  s[sl][cl] = a;
  __syncthreads();
  if (sl == 0 && c < D) {
#pragma unroll
    for (int i = 1; i < kParamSlices; ++i) a += s[i][cl];
    param_set<DT>(out, pf32, c, a);
  }
}

// ---- rows of any width: a workgroup per row, one read per reduction -------------
constexpr int kWideThreads = 1024;

template <int DT, int V>
__global__ __launch_bounds__(kWideThreads) void norm_fwd_wide_kernel(const void* xv, const void* w, const void* b,
                                                                     int pf32, int64_t rows, int64_t D, float eps,
                                                                     void* yv, float* mean, float* rstd) {
  using R = typename Elem<DT>::raw;
  using VT = Vec<DT, V>;
  __shared__ float red[2][16];
  const float inv = 1.f / (float)D;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const R* x = (const R*)xv + row * D;
    R* y = (R*)yv + row * D;
    float s[1] = {0.f};
    for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += kWideThreads * V) {
      const VT v = *(const VT*)(x + c);
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += to_f32<DT>(v.e[j]);
    }
    row_sum<kWideThreads>(s, red[0]);
    const float m = s[0] * inv;
    s[0] = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += kWideThreads * V) {
      const VT v = *(const VT*)(x + c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = to_f32<DT>(v.e[j]) - m;
        s[0] = fmaf(d, d, s[0]);
      }
    }
    row_sum<kWideThreads>(s, red[1]);
    const float r = 1.f / sqrtf(fmaf(s[0], inv, eps));
    for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += kWideThreads * V) {
      const VT v = *(const VT*)(x + c);
      VT o;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float wc = w ? param_at<DT>(w, pf32, c + j) : 1.f, bc = b ? param_at<DT>(b, pf32, c + j) : 0.f;
        o.e[j] = from_f32<DT>(fmaf((to_f32<DT>(v.e[j]) - m) * r, wc, bc));
      }
      *(VT*)(y + c) = o;
    }
    if (threadIdx.x == 0 && mean) {
      mean[row] = m;
      rstd[row] = r;
    }
  }
}

template <int DT, int V>
__global__ __launch_bounds__(kWideThreads) void norm_bwd_wide_kernel(const void* gv, const void* xv, const void* w,
                                                                     int pf32, const float* mean, const float* rstd,
                                                                     int64_t rows, int64_t D, void* dxv) {
  using R = typename Elem<DT>::raw;
  using VT = Vec<DT, V>;
  __shared__ float red[2][2 * 16];
  const float inv = 1.f / (float)D;
  int flip = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, flip ^= 1) {
    const R *x = (const R*)xv + row * D, *dy = (const R*)gv + row * D;
    R* dx = (R*)dxv + row * D;
    const float m = mean[row], r = rstd[row];
    float s[2] = {0.f, 0.f};
    for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += kWideThreads * V) {
      const VT vx = *(const VT*)(x + c), vg = *(const VT*)(dy + c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float g = to_f32<DT>(vg.e[j]) * (w ? param_at<DT>(w, pf32, c + j) : 1.f);
        s[0] += g;
        s[1] = fmaf(g, (to_f32<DT>(vx.e[j]) - m) * r, s[1]);
      }
    }
    row_sum<kWideThreads>(s, red[flip]);
    const float a = s[0] * inv, k = s[1] * inv;
    for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += kWideThreads * V) {
      const VT vx = *(const VT*)(x + c), vg = *(const VT*)(dy + c);
      VT o;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float g = to_f32<DT>(vg.e[j]) * (w ? param_at<DT>(w, pf32, c + j) : 1.f);
        o.e[j] = from_f32<DT>(r * (g - a - (to_f32<DT>(vx.e[j]) - m) * r * k));
      }
      *(VT*)(dx + c) = o;
    }
  }
}

// partial sums of 256 columns over the rows blockIdx.y, blockIdx.y + gridDim.y, ...
template <int DT>
__global__ __launch_bounds__(kNormThreads) void norm_param_wide_kernel(const void* gv, const void* xv,
                                                                       const float* mean, const float* rstd,
                                                                       int64_t rows, int64_t D, float* part) {
  using R = typename Elem<DT>::raw;
  const int64_t c = (int64_t)blockIdx.x * kNormThreads + threadIdx.x;
  if (c >= D) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float d = to_f32<DT>(((const R*)gv)[row * D + c]);
    dw = fmaf(d, (to_f32<DT>(((const R*)xv)[row * D + c]) - mean[row]) * rstd[row], dw);
    db += d;
  }
  part[(int64_t)blockIdx.y * D + c] = dw;
  part[((int64_t)gridDim.y + blockIdx.y) * D + c] = db;
}

// Threads per row, and elements per thread: the fewest threads that hold the
// row, 8 elements each before 16, so narrow rows share a wave (width 256 in
// bf16: 32 lanes with one 16-byte vector each) and the widest take a workgroup.
struct NormCfg {
  int T, E;
};
constexpr NormCfg kNormCfgs[] = {{16, 8}, {32, 8}, {64, 8}, {64, 16}, {256, 8}, {256, 16}, {1024, 8}};
constexpr int64_t kNormHeld = 1024 * 8;  // widest row that registers hold

int norm_cfg(int64_t D) {
  int i = 0;
  while ((int64_t)kNormCfgs[i].T * kNormCfgs[i].E < D) ++i;
  return i;
}

// Workgroups: a few to a compute unit that walk the rows, so that the weights are loaded once and
// the next row's loads run beside this one's sums.  Forward, 512 / 1,024 / 2,048 / 4,096 workgroups:
// 32,000 x 256 bf16 10.4 / 11.2 / 14.3 / 19.6 us, 172,032 x 256 f16 33.4 / 32.3 / 35.5 / 38.4,
// 2,048 x 1,153 f32 8.0 / 6.9 / 7.0 / 7.1, 16,384 x 4,096 bf16 52.8 / 55.8 / 55.6 / 75.1.
int64_t norm_fwd_blocks(int T, int E) { return T > kNormThreads || (T == kNormThreads && E > 8) ? 512 : 1024; }
// Backward, where each workgroup also writes a row of partial sums that norm_param_kernel reads
// again, 512 / 768 / 1,024: the same cases 14.3 / 13.7 / 14.0 us, 52.7 / 46.4 / 47.0, 9.9 / 10.5 /
// 10.5, 85 / 93 / 100 (and the sums 3.9 / 3.8 / 3.9, 4.6 / 4.6 / 4.6, 3.9 / 4.6 / 5.2, 4.9 / 5.7 / 6.9).
int64_t norm_bwd_blocks(int64_t rows, int64_t D) {
  if (D > kNormHeld) return std::min<int64_t>(rows, 64);
  const int T = kNormCfgs[norm_cfg(D)].T;
  const int64_t rounds = ceil_div(rows, wg_threads(T) / T);
  return std::min<int64_t>(rounds, T > kNormThreads ? 256 : T < kNormThreads ? 768 : 512);
}

template <class F>
int norm_dispatch(int cfg, F&& f) {
  switch (cfg) {
    case 0: return f(std::integral_constant<int, 16>(), std::integral_constant<int, 8>());
    case 1: return f(std::integral_constant<int, 32>(), std::integral_constant<int, 8>());
    case 2: return f(std::integral_constant<int, 64>(), std::integral_constant<int, 8>());
    case 3: return f(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
    case 4: return f(std::integral_constant<int, 256>(), std::integral_constant<int, 8>());
    case 5: return f(std::integral_constant<int, 256>(), std::integral_constant<int, 16>());
    default: return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 8>());
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int DT>
int norm_forward(const void* x, const void* w, const void* b, int pf32, int64_t rows, int64_t D, float eps, void* y,
                 float* mean, float* rstd, hipStream_t st) {
  ProfScope ps("layer_norm", st);
  constexpr int V16 = DT == ML_F32 ? 4 : 8;
  // 16-byte vectors where every row starts on a 16-byte boundary
  const bool vec = D % V16 == 0 && aligned16(x) && aligned16(y);
  if (D > kNormHeld) {
    const dim3 grid((unsigned)std::min<int64_t>(rows, 65536)), blk(kWideThreads);
    if (vec)
      hipLaunchKernelGGL((norm_fwd_wide_kernel<DT, V16>), grid, blk, 0, st, x, w, b, pf32, rows, D, eps, y, mean,
                         rstd);
    else
      hipLaunchKernelGGL((norm_fwd_wide_kernel<DT, 1>), grid, blk, 0, st, x, w, b, pf32, rows, D, eps, y, mean,
                         rstd);
    return check_launch("layer_norm");
  }
  return norm_dispatch(norm_cfg(D), [&](auto tc, auto ec) {
    constexpr int T = decltype(tc)::value, E = decltype(ec)::value;
    const int64_t rounds = ceil_div(rows, wg_threads(T) / T);
    const dim3 grid((unsigned)std::min<int64_t>(rounds, norm_fwd_blocks(T, E))), blk(wg_threads(T));
    if (vec)
      hipLaunchKernelGGL((norm_fwd_kernel<DT, V16, E / V16, T>), grid, blk, 0, st, x, w, b, pf32, rows, D, eps, y,
                         mean, rstd);
    else
      hipLaunchKernelGGL((norm_fwd_kernel<DT, 1, E, T>), grid, blk, 0, st, x, w, b, pf32, rows, D, eps, y, mean,
                         rstd);
    return check_launch("layer_norm");
  });
}

template <int DT>
int norm_backward(const void* g, const void* x, const void* w, int pf32, const float* mean, const float* rstd,
                  int64_t rows, int64_t D, void* dx, void* dw, void* db, float* part, hipStream_t st) {
  ProfScope ps("layer_norm_backward", st);
  const bool params = dw || db;
  const int64_t nblk = norm_bwd_blocks(rows, D);
  constexpr int V16 = DT == ML_F32 ? 4 : 8;
  const bool vec = D % V16 == 0 && aligned16(x) && aligned16(g) && aligned16(dx);
  int rc = ML_OK;
  if (rows > 0 && D > kNormHeld) {
    if (dx) {
      const dim3 grid((unsigned)std::min<int64_t>(rows, 65536)), blk(kWideThreads);
      if (vec)
        hipLaunchKernelGGL((norm_bwd_wide_kernel<DT, V16>), grid, blk, 0, st, g, x, w, pf32, mean, rstd, rows, D,
                           dx);
      else
        hipLaunchKernelGGL((norm_bwd_wide_kernel<DT, 1>), grid, blk, 0, st, g, x, w, pf32, mean, rstd, rows, D, dx);
      rc = check_launch("layer_norm_backward");
    }
    if (!rc && params) {
      hipLaunchKernelGGL(norm_param_wide_kernel<DT>, dim3((unsigned)ceil_div(D, kNormThreads), (unsigned)nblk),
                         dim3(kNormThreads), 0, st, g, x, mean, rstd, rows, D, part);
      rc = check_launch("layer_norm_backward");
    }
  } else if (rows > 0) {
    rc = norm_dispatch(norm_cfg(D), [&](auto tc, auto ec) {
      constexpr int T = decltype(tc)::value, E = decltype(ec)::value;
      const dim3 grid((unsigned)nblk), blk(wg_threads(T));
      float* p = params ? part : nullptr;
      if (vec)
        hipLaunchKernelGGL((norm_bwd_kernel<DT, V16, E / V16, T>), grid, blk, 0, st, g, x, w, pf32, mean, rstd,
                           rows, D, dx, p);
      else
        hipLaunchKernelGGL((norm_bwd_kernel<DT, 1, E, T>), grid, blk, 0, st, g, x, w, pf32, mean, rstd, rows, D, dx,
                           p);
      return check_launch("layer_norm_backward");
    });
  }
  if (rc || !params) return rc;
  hipLaunchKernelGGL(norm_param_kernel<DT>, dim3((unsigned)ceil_div(D, kParamCols), 2),
                     dim3(kParamCols * kParamSlices), 0, st, part, nblk, D, pf32, dw, db);
  return check_launch("layer_norm_backward");
}

constexpr int64_t kNormWidth = (int64_t)1 << 26;

int norm_check(int dtype, int pdtype, int64_t rows, int64_t width) {
  if (dtype != ML_F32 && dtype != ML_BF16 && dtype != ML_F16) return fail(ML_EINVAL, "layer_norm: unsupported dtype");
  if (pdtype != dtype && pdtype != ML_F32)
    return fail(ML_EINVAL, "layer_norm: weight and bias must have the input's dtype or be float32");
  if (rows < 0 || width <= 0) return fail(ML_EINVAL, "layer_norm: rows must not be negative, width must be positive");
  // norm_param_kernel takes 32 threads a column, a launch fewer than 2^32
  if (width > kNormWidth || (rows > 0 && width > INT64_MAX / 8 / rows))
    return fail(ML_EUNSUPPORTED, "layer_norm: too many elements");
  return ML_OK;
}

}  // namespace
}  // namespace ml

using namespace ml;

extern "C" int ml_layer_norm_forward(int dtype, int param_dtype, const void* x, const void* weight, const void* bias,
                                     int64_t rows, int64_t width, float eps, void* y, float* mean, float* rstd,
                                     ml_stream_t stream) {
  int rc = norm_check(dtype, param_dtype, rows, width);
  if (rc) return rc;
  if (!(eps >= 0.f)) return fail(ML_EINVAL, "layer_norm: eps must not be negative");
  if (rows == 0) return ML_OK;
  if (!x || !y || !mean != !rstd) return fail(ML_EINVAL, "layer_norm: null pointer (mean and rstd go together)");
  const int pf32 = param_dtype == ML_F32;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case ML_F32: return norm_forward<ML_F32>(x, weight, bias, pf32, rows, width, eps, y, mean, rstd, st);
    case ML_BF16: return norm_forward<ML_BF16>(x, weight, bias, pf32, rows, width, eps, y, mean, rstd, st);
    default: return norm_forward<ML_F16>(x, weight, bias, pf32, rows, width, eps, y, mean, rstd, st);
  }
}

extern "C" size_t ml_layer_norm_backward_workspace_size(int64_t rows, int64_t width) {
  if (norm_check(ML_F32, ML_F32, rows, width)) return 0;
  return std::max<size_t>(256, align256((size_t)norm_bwd_blocks(rows, width) * (size_t)width * 2 * sizeof(float)));
}

extern "C" int ml_layer_norm_backward(int dtype, int param_dtype, const void* grad_out, const void* x,
                                      const void* weight, const float* mean, const float* rstd, int64_t rows,
                                      int64_t width, void* grad_input, void* grad_weight, void* grad_bias,
                                      void* workspace, size_t workspace_bytes, ml_stream_t stream) {
  int rc = norm_check(dtype, param_dtype, rows, width);
  if (rc) return rc;
  if (!grad_input && !grad_weight && !grad_bias) return ML_OK;
  if (rows > 0 && (!grad_out || !x || !mean || !rstd)) return fail(ML_EINVAL, "layer_norm: null pointer");
  if ((grad_weight || grad_bias) &&
      (!workspace || workspace_bytes < ml_layer_norm_backward_workspace_size(rows, width)))
    return fail(ML_EWORKSPACE, "layer_norm: workspace too small");
  const int pf32 = param_dtype == ML_F32;
  hipStream_t st = (hipStream_t)stream;
  float* part = (float*)workspace;
  switch (dtype) {
    case ML_F32: return norm_backward<ML_F32>(grad_out, x, weight, pf32, mean, rstd, rows, width, grad_input, grad_weight, grad_bias, part, st);
    case ML_BF16: return norm_backward<ML_BF16>(grad_out, x, weight, pf32, mean, rstd, rows, width, grad_input, grad_weight, grad_bias, part, st);
    default: return norm_backward<ML_F16>(grad_out, x, weight, pf32, mean, rstd, rows, width, grad_input, grad_weight, grad_bias, part, st);
  }
}
