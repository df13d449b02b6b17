// What the kernels over rows share: elements of the three types, sums over the threads that hold a
// row, and how many threads hold one.
#pragma once

#include <type_traits>

#include "ml_internal.h"

namespace ml {

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

// 16 bytes of a row from element c on, at the element's alignment (one load or store of 16 bytes still: rows of odd
// length start anywhere); a row's last elements one by one.
typedef u32x4_t u32x4_near_t __attribute__((aligned(2)));
template <int DT, int N = DT == ML_F32 ? 4 : 8>  // (or single elements: N = 1)
struct RowChunk {
  static constexpr int V = N;
  typename Elem<DT>::raw e[V];

  // zeros where n, the elements left, runs out; WHOLE: all or none of the chunk is left; ONCE: past the caches, which keep what is
  // read again and what waits to be written
  template <bool WHOLE = false, bool ONCE = false>
  __device__ __forceinline__ void load(const typename Elem<DT>::raw* p, int64_t n) {
    if constexpr (V == 1) {
      e[0] = n > 0 ? *p : typename Elem<DT>::raw(0);
    } else if (n >= V) {
      const u32x4_t v = ONCE ? __builtin_nontemporal_load((const u32x4_near_t*)p) : *(const u32x4_near_t*)p;
      __builtin_memcpy(e, &v, 16);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) e[j] = !WHOLE && j < n ? p[j] : typename Elem<DT>::raw(0);
    }
  }
  template <bool WHOLE = false, bool ONCE = false>
  __device__ __forceinline__ void store(typename Elem<DT>::raw* p, int64_t n) const {
    if constexpr (V == 1) {
      if (n > 0) *p = e[0];
    } else if (n >= V) {
      u32x4_t v;
      __builtin_memcpy(&v, e, 16);
      if constexpr (ONCE) __builtin_nontemporal_store(v, (u32x4_near_t*)p);
      else *(u32x4_near_t*)p = v;
    } else if constexpr (!WHOLE) {
#pragma unroll
      for (int j = 0; j < V - 1; ++j)
        if (j < n) p[j] = e[j];
    }
  }
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

constexpr int kWideThreads = 1024;  // to a row that registers do not hold

// Threads per row, and elements per thread: the fewest threads that hold the
// row, 8 elements each before 16, so narrow rows share a wave (width 256 in
// bf16: 32 lanes with one 16-byte vector each) and the widest take a workgroup.
struct NormCfg {
  int T, E;
};
constexpr NormCfg kNormCfgs[] = {{16, 8}, {32, 8}, {64, 8}, {64, 16}, {256, 8}, {256, 16}, {1024, 8}};
constexpr int64_t kNormHeld = 1024 * 8;  // widest row that registers hold

inline int norm_cfg(int64_t D) {
  int i = 0;
  while ((int64_t)kNormCfgs[i].T * kNormCfgs[i].E < D) ++i;
  return i;
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

// dw[c], db[c] (grid y 1: dw alone): sums of n partial rows, 32 columns and 32 slices of the rows to a
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

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace ml
