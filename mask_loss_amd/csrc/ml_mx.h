// Microscaled values (the OCP microscaling formats): 32 consecutive values share a scale, a power of two in 8 bits
// (its exponent and 127, 255 for NaN); a value is kept in e2m1 (4 bits, two to a byte, the first in the low ones)
// or e4m3 (8 bits).  Of a block of floats v:
//
//   scale = 2^(floor(log2 max|v|) - emax), emax = 2 (e2m1, largest value 6) or 8 (e4m3, 448), held to 2^-127 .. 2^127
//   value = v / scale, rounded to nearest, ties to even, and held to the format's largest
//
// A block with a NaN or an infinity has the scale NaN (and zeros for values): all of it reads as NaN.  A block of
// zeros has the smallest scale.
#pragma once

#include "ml_rows.h"

namespace ml {

constexpr int kMxBlock = 32;

// The code of the scale, from the block's largest magnitude as bits (so that a NaN counts as the largest).
__device__ __forceinline__ uint32_t mx_scale(uint32_t bits, int format) {
  const int e = (int)(bits >> 23);  // 0 below the normal range, whose scale is the smallest anyway
  return e == 255 ? 255u : (uint32_t)max(e - (format == ML_MX_E4M3 ? 8 : 2), 0);
}
// 1 / scale: a normal number, so that the product with it is exact wherever the format can tell.
__device__ __forceinline__ float mx_inverse(uint32_t code) { return __uint_as_float((254u - code) << 23); }

// Largest magnitude, as bits, of the lanes that hold a block: 4 lanes (8 values to each) or 8 (4 to each).
template <int LANES>
__device__ __forceinline__ uint32_t mx_lane_max(uint32_t v) {
  static_assert(LANES == 4 || LANES == 8, "lanes");
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));  // quad_perm 1 0 3 2
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));  // quad_perm 2 3 0 1
  if constexpr (LANES == 8) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));  // row_half_mirror
  return v;
}

// Four values, already divided by the scale, in e4m3.  The conversion rounds to nearest even but lets values past the
// largest overflow, so they are held to it first.
__device__ __forceinline__ uint32_t mx_e4m3x4(float a, float b, float c, float d) {
  constexpr float m = 448.f;
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_fmed3f(a, -m, m), __builtin_amdgcn_fmed3f(b, -m, m), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_fmed3f(c, -m, m), __builtin_amdgcn_fmed3f(d, -m, m), lo, true);
}
// The same in e2m1, 16 bits; the conversion holds values to the largest itself.
template <int AT>
__device__ __forceinline__ uint32_t mx_e2m1x4(uint32_t old, float a, float b, float c, float d) {
  old = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, a, b, 1.f, 2 * AT);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, c, d, 1.f, 2 * AT + 1);
}

// V values of a lane whose block has the scale `code`: stored as values at, at + 1, .. of `codes`.
template <int V>
__device__ __forceinline__ void mx_store(const float (&y)[V], uint32_t code, int format, int64_t at, uint8_t* codes) {
  static_assert(V == 4 || V == 8, "values of a lane");
  const bool bad = code == 255u;  // NaN or infinity in the block
  const float inv = mx_inverse(bad ? 127u : code);
  float q[V];
#pragma unroll
  for (int j = 0; j < V; ++j) q[j] = bad ? 0.f : y[j] * inv;
  if (format == ML_MX_E4M3) {
    if constexpr (V == 8)
      *(u32x2_t*)(codes + at) = u32x2_t{mx_e4m3x4(q[0], q[1], q[2], q[3]), mx_e4m3x4(q[4], q[5], q[6], q[7])};
    else
      *(uint32_t*)(codes + at) = mx_e4m3x4(q[0], q[1], q[2], q[3]);
  } else {
    const uint32_t lo = mx_e2m1x4<0>(0u, q[0], q[1], q[2], q[3]);
    if constexpr (V == 8) *(uint32_t*)(codes + at / 2) = mx_e2m1x4<1>(lo, q[4], q[5], q[6], q[7]);
    else *(uint16_t*)(codes + at / 2) = (uint16_t)lo;
  }
}

// The magnitudes' maximum, as bits.
template <int V>
__device__ __forceinline__ uint32_t mx_max(const float (&y)[V]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) m = max(m, __float_as_uint(y[j]) & 0x7FFFFFFFu);
  return m;
}

inline bool mx_format(int format) { return format == ML_MX_E2M1 || format == ML_MX_E4M3; }

}  // namespace ml
