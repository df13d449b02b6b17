// Products of ragged groups of microscaled rows with one microscaled matrix per group (gfx950): the kernel.
// See ml_mx_grouped.hip for the entry points and the choice of tiles, ml_grouped.h for groups, tiles and operands,
// ml_mx.h for the formats.
//
//   y_r = sum over blocks b of 32:  2^(a_rb + w_nb) sum_k x_rk w_nk      for all rows n of the group's matrix
//
// Both operands lie with the reduced index contiguous, rows of whole 16-byte chunks (K is whole blocks).  The
// matrix instruction takes 128 of the reduced index with a scale per row and block of 32: lane l has row l % 16 and
//
//   e2m1   the 16 bytes 16 (l / 16) .. of the row's 64
//   e4m3   the 16 bytes 16 (l / 16) .. of the first 64 of the row's 128, and of the last 64
//   scale  of the block l / 16
//
// so either operand's fragment is Operand::frag, and a scale is a byte of the four that a row has here.
//
// What the instruction adds: products of e2m1 exactly (they span 8 bits); of products with an e4m3 operand it takes
// eight neighbours of the reduced index at a time, lined up on the largest of them with 13 bits below its leading one, and
// drops what lies below, then adds in float32 (measured: terms 2^-13 of the largest are kept, 2^-14 are not, at any magnitude).
// Over normal operands that is 1.5e-5 of a result's size, 4e-5 where channels differ by e: far below what a result
// in 16 bits is rounded by (2^-9, 2^-12).  A float32 result shall not lose it: there an e4m3 operand's blocks are converted to
// bfloat16 with their scales (exact: 4 significant bits, and the exponent's 8), and the bfloat16 instruction adds 32 of the
// reduced index with sums in float32, at half the rate.
#pragma once

#include "ml_grouped.h"
#include "ml_mx.h"

namespace ml {

struct MxArgs {
  GroupedArgs g;       // a and b: codes; K in values; lda, ldb, bstride in pairs of bytes
  const uint8_t *sa, *sb;  // scales, rows of sld bytes
  int64_t sld;
};

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32_byte_t __attribute__((aligned(1)));

constexpr bool mx_exact(int fa, int fb, int out) { return out == ML_F32 && (fa == ML_MX_E4M3 || fb == ML_MX_E4M3); }
// values of a step of the reduced index: 128 bytes of the wider operand
constexpr int mx_step(int fa, int fb) { return fa == ML_MX_E4M3 || fb == ML_MX_E4M3 ? 128 : 256; }
constexpr int mx_bytes(int format, int n) { return format == ML_MX_E4M3 ? n : n / 2; }

// 128 of the reduced index of a row, as the instruction takes them
template <int F>
struct MxFrag {
  u32x4_t v[F == ML_MX_E4M3 ? 2 : 1];
  uint32_t scale;
  __device__ __forceinline__ i32x8_t wide() const {
    if constexpr (F == ML_MX_E4M3)
      return i32x8_t{(int)v[0][0], (int)v[0][1], (int)v[0][2], (int)v[0][3], (int)v[1][0], (int)v[1][1], (int)v[1][2], (int)v[1][3]};
    else
      return i32x8_t{(int)v[0][0], (int)v[0][1], (int)v[0][2], (int)v[0][3], 0, 0, 0, 0};
  }
};
template <int FA, int FB>
__device__ __forceinline__ f32x4_t mx_mma(const MxFrag<FA>& a, const MxFrag<FB>& b, const f32x4_t& c) {
  constexpr int ca = FA == ML_MX_E4M3 ? 0 : 4, cb = FB == ML_MX_E4M3 ? 0 : 4;  // the instruction's names of the formats
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.wide(), b.wide(), c, ca, cb, 0, (int)a.scale, 0, (int)b.scale);
}

// One operand of a tile: R rows by a step of BK values, and their scales.
template <int F, int R, int NT, int BK>
struct MxOperand : Operand<ML_BF16, true, R, NT, mx_bytes(F, BK)> {
  using O = Operand<ML_BF16, true, R, NT, mx_bytes(F, BK)>;
  static constexpr int SCALES = R * BK / kMxBlock;  // bytes, [128 of the reduced index][row][4]
  static constexpr int LDS = O::BYTES + SCALES;

  // 128 values from 128 s on, of rows row0 ..
  static __device__ __forceinline__ MxFrag<F> frag(const unsigned char* lds, int row0, int s) {
    const int lane = threadIdx.x & 63;
    MxFrag<F> f;
    f.v[0] = O::frag(lds, row0, F == ML_MX_E4M3 ? 0 : s);
    if constexpr (F == ML_MX_E4M3) f.v[1] = O::frag(lds, row0, 1);
    f.scale = lds[O::BYTES + (s * R + row0 + (lane & 15)) * 4 + (lane >> 4)];
    return f;
  }

  // Block b (32 values) of rows row0 .., in bfloat16 with its scale: lane l holds values 8 (l / 16) .. of row l % 16.
  static __device__ __forceinline__ bf16x8_t block(const unsigned char* lds, int row0, int b) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const uint32_t code = lds[O::BYTES + (row0 + r) * 4 + b];
    const float scale = __uint_as_float(max(code << 23, 0x00400000u));  // 2^-127 is below the normal range
    bf16x2_t v[4];
    if constexpr (F == ML_MX_E4M3) {
      const u32x2_t p = *(const u32x2_t*)(lds + (row0 + r) * O::ROWB + (O::swizzled(r, 2 * b + (g >> 1)) << 4) + 8 * (g & 1));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(p[i], scale, false);
        v[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(p[i], scale, true);
      }
    } else {
      const uint32_t p = *(const uint32_t*)(lds + (row0 + r) * O::ROWB + (O::swizzled(r, b) << 4) + 4 * g);
      v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(p, scale, 0);
      v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(p, scale, 1);
      v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(p, scale, 2);
      v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(p, scale, 3);
    }
    bf16x8_t o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (code == 255u) v[i] = __builtin_bit_cast(bf16x2_t, 0x7FC07FC0u);  // NaN
      o[2 * i] = v[i][0];
      o[2 * i + 1] = v[i][1];
    }
    return o;
  }
};

// The scales of a row for a step of BK values, through registers: their rows start on any byte.
template <int BK>
struct MxScales {
  static constexpr int N = BK / 128;
  uint32_t v[N];
  // p: the row's scale at the step's start; left: blocks from there on
  __device__ __forceinline__ void load(const uint8_t* p, int left) {
    if (left >= 4 * N) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = *(const u32_byte_t*)(p + 4 * i);
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0x7F7F7F7Fu;  // 1, for the zeros past the end
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (4 * i + j < left) v[i] = (v[i] & ~(0xFFu << (8 * j))) | (uint32_t)p[4 * i + j] << (8 * j);
    }
  }
};

// WM x WN waves make BM x BN outputs in OUT.  Work items and dynamic LDS as grouped_kernel's.
template <int FA, int FB, int OUT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void mx_kernel(MxArgs x) {
  constexpr int NT = 64 * WM * WN, BK = mx_step(FA, FB), TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr bool EXACT = mx_exact(FA, FB, OUT);
  using OA = MxOperand<FA, BM, NT, BK>;
  using OB = MxOperand<FB, BN, NT, BK>;
  static_assert(BM + BN <= NT, "a thread for the scales of every row");
  constexpr int STAGE = OA::LDS + OB::LDS;
  __shared__ __align__(1024) unsigned char lds[2 * STAGE];
  extern __shared__ int e[];  // groups + 1 group edges, then groups + 2 tile counts
  const GroupedArgs& a = x.g;

  group_edges(a, e);
  int* t = e + a.groups + 1;
  const int tiles = segment_tiles(a, e, t, BM), count = tiles * a.cols.d, id = xcd_item(count * a.splits);
  if (id < 0) return;
  const int split = id / count;
  const Work it = rows_work(a, e, t, tiles, id - split * count, split, a.splits, BM, BN, BK);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m0 = uniform(it.m0), n0 = uniform(it.n0), mlim = uniform(it.mlim), w = uniform(it.w);
  const int steps = uniform(it.steps), kend = uniform(it.kend), nlim = a.N - n0;
  int k = uniform(it.k);
  const bool mapped = uniform(it.mapped) != 0;
  auto row_at = [&](int r) { return mapped ? merged_row(a, e, w, m0 + r) : r; };

  const uint16_t* pa = (const uint16_t*)a.a + (mapped ? (int64_t)0 : (int64_t)m0 * a.lda);
  const uint16_t* pb = (const uint16_t*)a.b + ((int64_t)w * a.bstride + (int64_t)n0 * a.ldb);
  OA oa;
  OB ob;
  oa.aim(a.lda, mlim, row_at);
  ob.aim(a.ldb, nlim, [](int r) { return r; });
  // threads 0 .. BM - 1 take the rows' scales, the next BN the matrix's
  const bool srow = (int)threadIdx.x < BM;
  const int si = srow ? threadIdx.x : threadIdx.x - BM;
  const uint8_t* ps = srow ? x.sa + ((mapped ? 0 : m0) + row_at(min(si, mlim - 1))) * x.sld
                           : x.sb + ((int64_t)w * a.N + n0 + min(si, nlim - 1)) * x.sld;
  unsigned char* const sat = lds + (srow ? OA::O::BYTES : OA::LDS + OB::O::BYTES) + 4 * si;
  const int sstep = srow ? 4 * BM : 4 * BN;
  MxScales<BK> sc;
  auto fetch = [&]() {  // the step at k
    oa.load(pa + mx_bytes(FA, k) / 2, mlim, mx_bytes(FA, kend - k) / 2);
    ob.load(pb + mx_bytes(FB, k) / 2, nlim, mx_bytes(FB, kend - k) / 2);
    if (threadIdx.x < BM + BN) sc.load(ps + k / kMxBlock, (kend - k) / kMxBlock);
  };
  auto put = [&](int stage) {
    oa.store(lds + stage * STAGE);
    ob.store(lds + stage * STAGE + OA::LDS);
    if (threadIdx.x < BM + BN)
#pragma unroll
      for (int i = 0; i < MxScales<BK>::N; ++i) *(uint32_t*)(sat + stage * STAGE + i * sstep) = sc.v[i];
  };

  f32x4_t acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);

  if (steps > 0) {
    fetch();
    put(0);
    if (steps > 1) {
      k += BK;
      fetch();
    }
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
      const unsigned char* cur = lds + (s & 1) * STAGE;
      if (s + 1 < steps) {
        put((s & 1) ^ 1);
        if (s + 2 < steps) {
          k += BK;
          fetch();
        }
      }
      if constexpr (EXACT) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          bf16x8_t fa[TM], fb[TN];
#pragma unroll
          for (int i = 0; i < TM; ++i) fa[i] = OA::block(cur, wm + 16 * i, b);
#pragma unroll
          for (int i = 0; i < TN; ++i) fb[i] = OB::block(cur + OA::LDS, wn + 16 * i, b);
#pragma unroll
          for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[i], fa[j], acc[i][j], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int h = 0; h < BK / 128; ++h) {
          MxFrag<FA> fa[TM];
          MxFrag<FB> fb[TN];
#pragma unroll
          for (int i = 0; i < TM; ++i) fa[i] = OA::frag(cur, wm + 16 * i, h);
#pragma unroll
          for (int i = 0; i < TN; ++i) fb[i] = OB::frag(cur + OA::LDS, wn + 16 * i, h);
#pragma unroll
          for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) acc[i][j] = mx_mma(fb[i], fa[j], acc[i][j]);
        }
      }
      __syncthreads();
    }
  }

  // lane l holds columns 4 (l / 16) .. + 3 of row l % 16 of each 16 x 16 tile
  const bool planes = a.splits > 1;
  float* cf = planes ? a.parts + (int64_t)split * a.plane : (float*)a.c;
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int m = wm + 16 * j + (lane & 15);
    if (m >= mlim) continue;
    const int64_t row = (int64_t)(mapped ? row_at(m) : m0 + m) * a.ldc;
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      const int n = wn + 16 * i + 4 * (lane >> 4);
      if (n >= nlim) continue;
      const f32x4_t v = acc[i][j];
      const int64_t at = row + n0 + n;
      if (planes || OUT == ML_F32) {
        if (n + 4 <= nlim) {
          *(f32x4_loose*)(cf + at) = v;
        } else {
#pragma unroll
          for (int q = 0; q < 3; ++q)
            if (n + q < nlim) cf[at + q] = v[q];
        }
      } else if constexpr (OUT != ML_F32) {
        const u32x2_t p = {GMma<OUT>::pack(v[0], v[1]), GMma<OUT>::pack(v[2], v[3])};
        uint16_t* c = (uint16_t*)a.c + at;
        if (n + 4 <= nlim) {
          *(u32x2_loose*)c = p;
        } else {
#pragma unroll
          for (int q = 0; q < 3; ++q)
            if (n + q < nlim) c[q] = (uint16_t)(p[q / 2] >> (16 * (q & 1)));
        }
      }
    }
  }
}

}  // namespace ml
