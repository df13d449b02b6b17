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
// Over normal operands that is 1.5e-5 of a result's size, 4e-5 where channels differ by e, 7e-5 by e^2, with no sign of its own: far
// below the half step that a result in 16 bits is rounded by (2^-8, 2^-11).  A float32 result shall not lose it: there an e4m3
// operand's blocks are converted to bfloat16 with their scales, and the bfloat16 instruction adds 32 of the reduced index
// with sums in float32, at half the rate.  The conversion is exact (4 significant bits) for scaled values from 2^-126 up to below
// 2^128, bfloat16's range; smaller ones, down to 2^-136, may count as zero, larger ones are infinite, also where the other
// operand's scale would bring the product back.
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

// Eight values in bfloat16 with their scale (of e2m1: the low word).  The conversion takes the exponent field alone of
// its scale, with 0 for 2^-127 and 255 for NaN whatever the value (all 256 codes of both formats checked).
template <int F>
__device__ __forceinline__ bf16x8_t mx_bf16(uint32_t p0, uint32_t p1, uint32_t code) {
  const float scale = __uint_as_float(code << 23);
  bf16x2_t v[4];
  if constexpr (F == ML_MX_E4M3) {
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(p0, scale, false);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(p0, scale, true);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(p1, scale, false);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(p1, scale, true);
  } else {
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(p0, scale, 0);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(p0, scale, 1);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(p0, scale, 2);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(p0, scale, 3);
  }
  bf16x8_t o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[2 * i] = v[i][0];
    o[2 * i + 1] = v[i][1];
  }
  return o;
}

// Block b (32 values) of rows row0 .. of an operand's LDS image: lane l holds values 8 (l / 16) .. of row l % 16, whose
// scale is `code`.
template <int F, class O>
__device__ __forceinline__ bf16x8_t mx_block(const unsigned char* lds, int row0, int b, uint32_t code) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  if constexpr (F == ML_MX_E4M3) {
    const u32x2_t p = *(const u32x2_t*)(lds + (row0 + r) * O::ROWB + (O::swizzled(r, 2 * b + (g >> 1)) << 4) + 8 * (g & 1));
    return mx_bf16<F>(p[0], p[1], code);
  } else {
    return mx_bf16<F>(*(const uint32_t*)(lds + (row0 + r) * O::ROWB + (O::swizzled(r, b) << 4) + 4 * g), 0u, code);
  }
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
    return mx_block<F, O>(lds, row0, b, lds[O::BYTES + (row0 + (threadIdx.x & 15)) * 4 + b]);
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

// Any K, scales on any byte.  WM x WN waves make BM x BN outputs in OUT.  Work items and dynamic LDS as grouped_kernel's.
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

// The scales of 64 rows: from lane l's dword of row l (its blocks 0 .. 3) to lane l's four bytes of block l / 16 in rows
// l % 16 + 16 j, of which the instruction is told byte j.  A transpose among the lanes l % 16 + 16 g: neighbours g, g ^ 1
// exchange their dwords, each keeps the bytes of blocks g and g ^ 2 of the two, and hands the latter to g ^ 2.
struct MxTurn {
  uint32_t mine, theirs;  // selectors of v_perm_b32
  __device__ __forceinline__ MxTurn() {
    const uint32_t g = (threadIdx.x >> 4) & 3, o = g ^ 2;
    mine = g | (4 + g) << 8 | o << 16 | (4 + o) << 24;
    // of the pairs 0, 1 and 2, 3: what they kept, or what they handed over
    theirs = g < 2 ? 0x07060100u : 0x05040302u;
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t d) const {
    const auto n = __builtin_amdgcn_permlane16_swap(d, d, false, false);  // the even and the odd neighbour's
    const uint32_t u = __builtin_amdgcn_perm(n[1], n[0], mine);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_amdgcn_perm(p[1], p[0], theirs);
  }
};
// (byte: an immediate of the instruction, a constant where the loops are unrolled)
template <int FA, int FB, int BA, int BB>
__device__ __forceinline__ f32x4_t mx_mma_at(const MxFrag<FA>& a, const MxFrag<FB>& b, uint32_t sa, uint32_t sb, const f32x4_t& c) {
  constexpr int ca = FA == ML_MX_E4M3 ? 0 : 4, cb = FB == ML_MX_E4M3 ? 0 : 4;
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.wide(), b.wide(), c, ca, cb, BA, (int)sa, BB, (int)sb);
}
template <int FA, int FB>
__device__ __forceinline__ f32x4_t mx_mma_at(int ba, int bb, const MxFrag<FA>& a, const MxFrag<FB>& b, uint32_t sa, uint32_t sb,
                                             const f32x4_t& c) {
  switch (ba * 4 + bb) {
#define ML_MX_CASE(i) case i: return mx_mma_at<FA, FB, i / 4, i % 4>(a, b, sa, sb, c);
    ML_MX_CASE(0) ML_MX_CASE(1) ML_MX_CASE(2) ML_MX_CASE(3) ML_MX_CASE(4) ML_MX_CASE(5) ML_MX_CASE(6) ML_MX_CASE(7)
    ML_MX_CASE(8) ML_MX_CASE(9) ML_MX_CASE(10) ML_MX_CASE(11) ML_MX_CASE(12) ML_MX_CASE(13) ML_MX_CASE(14)
#undef ML_MX_CASE
    default: return mx_mma_at<FA, FB, 3, 3>(a, b, sa, sb, c);
  }
}

// ---- few rows to a group ------------------------------------------------------------
// The matrices are read once and nothing is reused but a few rows, so the operands go from memory into the registers
// that the matrix instruction takes: a workgroup has 16 MT rows by 32 columns, its four waves take turns over the reduced
// index, 512 of it at a time (so all of a lane's loads are in flight together), and add up through LDS.  32 rows in 32
// groups, K = 2,048, N = 1,024, e4m3 by e2m1: 9.0 us; with tiles through LDS and a join of their parts 9.3 + 2.6.
// Where there are few tiles, their reductions go to several workgroups in whole turns and are joined (calls, 8 rows by e2m1: K =
// 65,536, N = 256 59 -> 11 us, K = 16,384, N = 4,096 20 -> 15).
constexpr int kFewColumns = 32, kFewStep = 512, kFewTurn = 4 * kFewStep;

// 512 values of a row from `codes` and `scales` on, for the lanes l of the row l % 16; left: values of the row from there on.
template <int F>
struct MxRows {
  static constexpr int N = F == ML_MX_E4M3 ? 2 : 1;  // 16-byte chunks of 128 values that a lane has
  u32x4_t v[4][N];
  uint32_t scale;
  __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* scales, int left) {
    const int g = (threadIdx.x >> 4) & 3;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        // e4m3: values 16 g .. of the first 64 and of the last; e2m1: 32 g ..
        const int at = 128 * s + (F == ML_MX_E4M3 ? 64 * i + 16 * g : 32 * g);
        v[s][i] = u32x4_t{0u, 0u, 0u, 0u};
        if (at < left) v[s][i] = *(const u32x4_t*)(codes + mx_bytes(F, at));
      }
    // lane group g: the four scales of 128 values from 128 g on
    scale = 0x7F7F7F7Fu;  // 1, for the zeros past the end
    const int n = left / kMxBlock - 4 * g;
    if (n >= 4) {
      scale = *(const u32_byte_t*)(scales + 4 * g);
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (j < n) scale = (scale & ~(0xFFu << (8 * j))) | (uint32_t)scales[4 * g + j] << (8 * j);
    }
  }
  __device__ __forceinline__ MxFrag<F> frag(int s) const {
    MxFrag<F> f;
#pragma unroll
    for (int i = 0; i < N; ++i) f.v[i] = v[s][i];
    f.scale = 0;
    return f;
  }
};

// The same for products in bfloat16: lane group g has, of each 128 values, those 16 g .. of the first 64 and of the last, in
// either format, and their row's 16 scales.
template <int F>
struct MxExactRows {
  using P = std::conditional_t<F == ML_MX_E4M3, u32x4_t, u32x2_t>;
  P v[4][2];
  uint32_t scale[4];
  __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* scales, int left) {
    const int g = (threadIdx.x >> 4) & 3;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = 128 * s + 64 * i + 16 * g;
        v[s][i] = P{};
        if (at < left) v[s][i] = *(const P*)(codes + mx_bytes(F, at));
      }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      MxScales<128> c;
      c.load(scales + 4 * s, left / kMxBlock - 4 * s);
      scale[s] = c.v[0];
    }
  }
  // eight of them, h: the first or the last of the 16
  __device__ __forceinline__ bf16x8_t eight(int s, int i, int h) const {
    const uint32_t code = scale[s] >> (16 * i + 8 * (threadIdx.x >> 5 & 1)) & 255u;
    if constexpr (F == ML_MX_E4M3) return mx_bf16<F>(v[s][i][2 * h], v[s][i][2 * h + 1], code);
    else return mx_bf16<F>(v[s][i][h], 0u, code);
  }
};

template <int FA, int FB, int OUT, int MT>
__global__ __launch_bounds__(256) void mx_few_kernel(MxArgs x) {
  constexpr bool EXACT = mx_exact(FA, FB, OUT);
  constexpr int BM = 16 * MT, NT = kFewColumns / 16;
  __shared__ f32x4_t part[3][MT * NT][64];
  extern __shared__ int e[];
  const GroupedArgs& a = x.g;
  group_edges(a, e);
  int* t = e + a.groups + 1;
  const int tiles = segment_tiles(a, e, t, BM), count = tiles * a.cols.d, id = xcd_item(count * a.splits);
  if (id < 0) return;
  const int split = id / count;
  const Work it = rows_work(a, e, t, tiles, id - split * count, split, a.splits, BM, kFewColumns, kFewTurn);
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int m0 = uniform(it.m0), n0 = uniform(it.n0), mlim = uniform(it.mlim), w = uniform(it.w);
  const int nlim = a.N - n0, k0 = uniform(it.k), K = uniform(min(it.kend, it.k + it.steps * kFewTurn));  // the part's
  const bool mapped = uniform(it.mapped) != 0;

  const uint8_t *pa[MT], *sa[MT], *pb[NT], *sb[NT];
  int64_t row[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {  // rows past the last read the last one (their outputs are not stored)
    const int r = min(16 * i + (lane & 15), mlim - 1);
    row[i] = mapped ? merged_row(a, e, w, m0 + r) : m0 + r;
    pa[i] = (const uint8_t*)a.a + row[i] * (a.lda * 2);
    sa[i] = x.sa + row[i] * x.sld;
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int64_t r = (int64_t)w * a.N + n0 + min(16 * i + (lane & 15), nlim - 1);
    pb[i] = (const uint8_t*)a.b + r * (a.ldb * 2);
    sb[i] = x.sb + r * x.sld;
  }
  f32x4_t acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const MxTurn turn;
  for (int k = k0 + wave * kFewStep; k < K; k += kFewTurn) {
    std::conditional_t<EXACT, MxExactRows<FA>, MxRows<FA>> ra[MT];
    std::conditional_t<EXACT, MxExactRows<FB>, MxRows<FB>> rb[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) rb[i].load(pb[i] + mx_bytes(FB, k), sb[i] + k / kMxBlock, K - k);
#pragma unroll
    for (int j = 0; j < MT; ++j) ra[j].load(pa[j] + mx_bytes(FA, k), sa[j] + k / kMxBlock, K - k);
    if constexpr (EXACT) {
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        bf16x8_t xa[MT], xb[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) xb[i] = rb[i].eight(q >> 2, q >> 1 & 1, q & 1);
#pragma unroll
        for (int j = 0; j < MT; ++j) xa[j] = ra[j].eight(q >> 2, q >> 1 & 1, q & 1);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j < MT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xb[i], xa[j], acc[i][j], 0, 0, 0);
      }
    } else {
      uint32_t ta[MT], tb[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) tb[i] = turn(rb[i].scale);  // byte s: of the 128 values from 128 s on
#pragma unroll
      for (int j = 0; j < MT; ++j) ta[j] = turn(ra[j].scale);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j < MT; ++j) acc[i][j] = mx_mma_at(s, s, rb[i].frag(s), ra[j].frag(s), tb[i], ta[j], acc[i][j]);
    }
  }
  if (wave)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) part[wave - 1][i * MT + j][lane] = acc[i][j];
  __syncthreads();
  if (wave) return;
  const bool planes = a.splits > 1;
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    if (16 * j + (lane & 15) >= mlim) continue;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      f32x4_t v = acc[i][j];
#pragma unroll
      for (int q = 0; q < 3; ++q) v += part[q][i * MT + j][lane];
      const int n = 16 * i + 4 * (lane >> 4), room = nlim - n;
      if (room <= 0) continue;
      const int64_t at = row[j] * a.ldc + n0 + n;
      if (planes || OUT == ML_F32) {
        float* c = (planes ? a.parts + (int64_t)split * a.plane : (float*)a.c) + at;
        if (room >= 4) *(f32x4_loose*)c = v;
        else
#pragma unroll
          for (int q = 0; q < 3; ++q)
            if (q < room) c[q] = v[q];
      } else if constexpr (OUT != ML_F32) {
        const u32x2_t p = {GMma<OUT>::pack(v[0], v[1]), GMma<OUT>::pack(v[2], v[3])};
        uint16_t* c = (uint16_t*)a.c + at;
        if (room >= 4) *(u32x2_loose*)c = p;
        else
#pragma unroll
          for (int q = 0; q < 3; ++q)
            if (q < room) c[q] = (uint16_t)(p[q / 2] >> (16 * (q & 1)));
      }
    }
  }
}

// ---- scales in whole fours: stages filled by direct loads into LDS ---------------------
// Where K is a multiple of 128 (and the scales start on 4-byte boundaries), a row's four scales of a fragment are one
// dword, and everything of a stage comes by direct loads: grouped_ring_kernel's ring (there: stages, persistent workgroups, turns,
// waits), with the dwords of the stage's scales behind its codes, [128 of the reduced index][rows of both operands].

// Four bytes from base + off, or from p, of each lane to LDS at `lds` + 4 lane; base as ring_loads'.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void ring_dwords(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dword %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void ring_dwords(const char* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               :
               : "s"(lds), "v"(p)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// One operand of a stage, filled by NW waves.
template <int F, int R, int NW, int BK>
struct MxRing : RingOperand<ML_BF16, true, R, NW, mx_bytes(F, BK)> {
  using O = typename RingOperand<ML_BF16, true, R, NW, mx_bytes(F, BK)>::O;
  // 128 values from 128 s on, of rows row0 .. (the scale is elsewhere)
  static __device__ __forceinline__ MxFrag<F> frag(const unsigned char* lds, int row0, int s) {
    MxFrag<F> f;
    f.v[0] = O::frag(lds, row0, F == ML_MX_E4M3 ? 0 : s);
    if constexpr (F == ML_MX_E4M3) f.v[1] = O::frag(lds, row0, 1);
    f.scale = 0;
    return f;
  }
};

// Order of a sub-step's LDS reads (the scales' first, RB and RA for a fragment of either operand) and products (N for each
// of M fragments).
template <int RS, int RB, int RA, int N, int M>
__device__ __forceinline__ void mx_interleave() {
  constexpr int kMfma = 0x8, kRead = 0x100;
  __builtin_amdgcn_sched_group_barrier(kRead, RS, 0);
  interleave<RB, RA, N, M, 1>();
}

// What a workgroup is to do next, as rows_work tells it, for 32 of its work items at a time, one to a lane: a search
// through the segments and divisions are a microsecond's wait, which the others of a tile would be waiting for.
struct alignas(16) MxItem {
  int m0, n0, mlim, w;
  int block;       // of a split tile's parts, or -1
  int steps, k;    // k: where the reduced index starts
  int kind;        // 1: rows of several groups (merged_row); 2: rows in no group, zeros
};
constexpr int kMxItems = 32;
// (1, 2, 3, 4 row tiles to a band: 16,384 rows in 16 groups, K = 1,024, N = 4,096, e2m1 69, 71, 70, 77 us with operands from memory,
// e4m3 by e4m3 102, 105, 103, 111; one matrix 8,192 x 8,192 x 8,192, e2m1 399, 363, 350, 352, e4m3 by e2m1 563, 492, 489, 486.)
constexpr int kMxBand = 3;

__device__ __forceinline__ MxItem mx_item(const GroupedArgs& a, const int* e, const int* t, int tiles, const RingShare& share,
                                          int next, int bm, int bn, int bk) {
  int id = share.start + next, part = 0, parts = 1;
  MxItem it;
  it.block = -1;
  if (next >= share.whole) {  // a part of one of the last tiles
    const int p = next - share.whole, r = p / share.parts;
    id = share.start + share.whole + r;
    parts = share.parts;
    part = p - r * parts;
    if (parts > 1) it.block = p;
  }
  const int band = div_by((int)((uint32_t)id / kMxBand), a.cols);
  const int height = min(kMxBand, tiles - band * kMxBand);
  const int rest = id - band * kMxBand * a.cols.d, y = rest / height;
  it.n0 = y * bn;
  const int tile = band * kMxBand + rest - y * height;
  int q = 0, end = a.segments + 1;  // the first segment whose tiles end behind this one
  while (q < end) {
    const int mid = (q + end) >> 1;
    if (t[mid] <= tile) q = mid + 1;
    else end = mid;
  }
  int r0, r1;
  segment(a, e, q, r0, r1);
  const bool zero = q >= a.segments;
  it.m0 = r0 + (tile - (q ? t[q - 1] : 0)) * bm;
  it.mlim = r1 - it.m0;
  it.w = zero ? 0 : a.merged ? q : div_by(q, a.layers);
  it.kind = zero ? 2 : a.merged ? 1 : 0;
  const int steps = zero ? 0 : (int)((uint32_t)(a.K + bk - 1) / (uint32_t)bk), s0 = part_start(steps, part, parts);
  it.steps = part_start(steps, part + 1, parts) - s0;
  it.k = s0 * bk;
  return it;
}

// Template arguments as mx_kernel's; two stages of BK values, OCC workgroups to a compute unit.  SW: 16, the scales come 512 of the
// reduced index at a time, 16 bytes of a row with the first stage of them (K a multiple of 512, scales on 16-byte boundaries), in
// two slots of [row][16], and the loop over their stages is unrolled; or 4, those of a stage with it, [128 of the reduced
// index][row][4].  A row's scales are far from the next one's, so a load of 64 rows takes 64 cache lines however few bytes of
// each: 8,192 x 8,192 x 8,192 in e2m1 took 396 us with a stage's dwords, 303 with no scale loads, 359 with these.
//
// What bounds it (16,384 rows in 16 groups, K = 1,024, N = 4,096, e2m1: 62 us, 70 where the operands come from memory; the
// matrix instructions alone run at 7,400 TFLOP/s on random values and are busy for 2.3 of the 7 us of a compute unit's
// two tiles): the waits and other instructions around each stage's products, then the stores.  An earlier form that took 72 us took 54
// without its stores, 46 without loads and LDS reads, 44 without either; four stages of half the length took 71 for 66.  Non-temporal stores took 65 for 76, but what reads the result next
// then waits for memory (with a product by 2 behind it 133 to 148 us, without them 129); half of the workgroups starting
// a half tile later, to store while the others multiply, changes nothing.
//
// Products in bfloat16 (mx_exact) read a block of 32 of both operands at once and convert it, the next one's conversions
// between the products (without: 1 to 3% more): 32 of 4 cycles for 16 products of 16, 1,100 TFLOP/s at 8,192 x 8,192 x 4,096.
template <int FA, int FB, int OUT, int BM, int BN, int WM, int WN, int BK, int OCC, int SW>
__global__ __launch_bounds__(64 * WM * WN, OCC * WM * WN / 4) void mx_ring_kernel(MxArgs x) {
  constexpr bool EXACT = mx_exact(FA, FB, OUT);
  constexpr int NS = 2, NW = WM * WN, H = BK / 128, TM = BM / WM / 16, TN = BN / WN / 16;
  using OA = MxRing<FA, BM, NW, BK>;
  using OB = MxRing<FB, BN, NW, BK>;
  constexpr int SUPER = SW == 16 ? 512 / BK : 1;  // stages that share their scales' loads, and turns of the unrolled loop
  constexpr int CODES = OA::BYTES + OB::BYTES, ROWS = BM + BN;
  constexpr int SLOT = SW == 16 ? ROWS * 16 : H * ROWS * 4, SLOTS = SW == 16 ? 2 : NS;
  constexpr int UNITS = SLOT / (64 * SW), S = (UNITS + NW - 1) / NW;  // scale loads of a slot, and of a wave
  constexpr int ST = TM * TN / (OUT == ML_F32 ? 1 : 2);               // stores of a full tile
  static_assert(TN % 4 == 0 && TM % 4 == 0, "whole scale fragments");
  static_assert(BM % 64 == 0 && BN % 64 == 0, "whole scale loads of an operand");
  static_assert(SW == 4 || SUPER % NS == 0, "a stage's slot is known where the loop is unrolled");
  __shared__ __align__(1024) unsigned char lds[NS * CODES];
  __shared__ __align__(1024) unsigned char slots[SLOTS * SLOT];
  __shared__ MxItem queue[2 * kMxItems];
  extern __shared__ int e[];
  const GroupedArgs& a = x.g;

  group_edges(a, e);
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  int* t = e + a.groups + 1;
  const int tiles = segment_tiles(a, e, t, BM);
  const int xcd = (int)blockIdx.x % kXcds, turns = (int)gridDim.x / kXcds, first = (int)blockIdx.x / kXcds;
  const RingShare share = ring_share(a, tiles * a.cols.d, xcd, turns);
  const int last = share.whole + share.rest * share.parts;
  if (first >= last) return;
  const int count = (last - first + turns - 1) / turns;
  auto item = [&](int n) {
    MxItem it = queue[n % (2 * kMxItems)];
    int* f = (int*)&it;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = uniform(f[i]);
    return it;
  };

  // ---- loads
  OA oa;
  OB ob;
  const uint32_t ring = (uint32_t)(uintptr_t)(lds_void_t*)lds, sring = (uint32_t)(uintptr_t)(lds_void_t*)slots;
  int opened = 0, left = 0, kleft = 0;         // stages left of the item being loaded, and its values left
  int sslot = 0;                               // the next slot of scales
  bool whole_a = false, whole_b = false;       // oa's, ob's offsets are those of a whole tile
  const char *pa = nullptr, *pb = nullptr;     // the next stage's codes
  const char *psa = nullptr, *psb = nullptr;   // and the next scales
  uint32_t soff[S];                            // bytes of this lane's row of each of the wave's units
  auto open_item = [&]() {
    if (opened >= count) {  // nothing more: zeros
      left = INT32_MAX - 2 * SUPER;
      kleft = 0;
      return;
    }
    if (opened % kMxItems == 0) {  // (every wave for itself, the same values)
      if (lane < min(kMxItems, count - opened))
        queue[(opened + lane) % (2 * kMxItems)] = mx_item(a, e, t, tiles, share, first + (opened + lane) * turns, BM, BN, SUPER * BK);
    }
    const MxItem it = item(opened++);
    left = max(it.steps, 1) * SUPER;  // (nothing to reduce: stages of zeros)
    kleft = it.kind == 2 ? 0 : a.K - it.k;
    const bool mapped = it.kind == 1;
    pa = (const char*)a.a + (mapped ? (int64_t)0 : (int64_t)it.m0 * a.lda) * 2 + mx_bytes(FA, it.k);
    pb = (const char*)a.b + ((int64_t)it.w * a.bstride + (int64_t)it.n0 * a.ldb) * 2 + mx_bytes(FB, it.k);
    psa = (const char*)x.sa + (mapped ? (int64_t)0 : it.m0 * x.sld) + it.k / kMxBlock;
    psb = (const char*)x.sb + ((int64_t)it.w * a.N + it.n0) * x.sld + it.k / kMxBlock;
    const bool wa = !mapped && it.mlim >= BM, wb = a.N - it.n0 >= BN;
    if (wa && wb && whole_a && whole_b) return;
    if (mapped) oa.aim(a.lda, it.mlim, wave, [&](int r) { return merged_row(a, e, it.w, it.m0 + r); });
    else oa.aim(a.lda, it.mlim, wave, [](int r) { return r; });
    ob.aim(a.ldb, a.N - it.n0, wave, [](int r) { return r; });
    whole_a = wa;
    whole_b = wb;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int row = min(wave * S + i, UNITS - 1) * 64 % ROWS + lane;  // of both operands
      int r = row < BM ? min(row, it.mlim - 1) : min(row - BM, a.N - it.n0 - 1);
      if (mapped && row < BM) r = merged_row(a, e, it.w, it.m0 + r);
      soff[i] = (uint32_t)r * (uint32_t)x.sld;
    }
  };
  // The next stage's loads, into this slot of the ring (zeros where nothing is left); `scales`: it is the first one of its
  // scales, and perhaps of an item.
  auto load = [&](int stage, bool scales) {
    if (scales) {
      if (left == 0) open_item();
      left -= SUPER;
      const uint32_t to = sring + (SW == 16 ? sslot : stage) * SLOT;
      sslot ^= 1;
      if (SW == 16 ? kleft > 0 : kleft >= BK) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
          const int u = min(wave * S + i, UNITS - 1);
          const char* base = uniform((u * 64 % ROWS < BM ? psa : psb) + (SW == 16 ? 0 : 4 * (u * 64 / ROWS)));
          if constexpr (SW == 16) {
            const uint32_t o[1] = {soff[i]};
            ring_loads(base, o, to + u * 1024);
          } else {
            ring_dwords(base, soff[i], to + u * 256);
          }
        }
        psa += SUPER * BK / kMxBlock;
        psb += SUPER * BK / kMxBlock;
      } else {
#pragma unroll
        for (int i = 0; i < S; ++i) {
          const int u = min(wave * S + i, UNITS - 1), h = u * 64 / ROWS;
          if constexpr (SW == 16) ring_load((const char*)g_zeros, to + u * 1024);
          else if (h * 128 < kleft) ring_dwords(uniform((u * 64 % ROWS < BM ? psa : psb) + 4 * h), soff[i], to + u * 256);
          else ring_dwords((const char*)g_zeros, to + u * 256);
        }
      }
    }
    const uint32_t to = ring + stage * CODES;
    if (kleft >= BK) {
      ring_loads(uniform(pa), oa.off, to + wave * OA::PER * 1024);
      ring_loads(uniform(pb), ob.off, to + OA::BYTES + wave * OB::PER * 1024);
      pa += mx_bytes(FA, BK);
      pb += mx_bytes(FB, BK);
    } else {
      oa.load(pa, mx_bytes(FA, kleft) / 2, to, wave);
      ob.load(pb, mx_bytes(FB, kleft) / 2, to + OA::BYTES, wave);
    }
    kleft -= BK;
  };
#pragma unroll
  for (int s = 0; s < NS; ++s) load(s, s % SUPER == 0);

  // ---- products
  const int wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);
  const MxTurn turn;
  int at = 0;  // the slot of the scales in turn
  auto frag_a = [&](int stage, int j, int h) { return OA::frag(lds + stage * CODES, wm + 16 * j, h); };
  auto frag_b = [&](int stage, int i, int h) { return OB::frag(lds + stage * CODES + OA::BYTES, wn + 16 * i, h); };
  auto scale = [&](int stage, int part, int row0, int h) {  // lane l's: row row0 + l, its four of the sub-step
    const unsigned char* p = SW == 16 ? slots + at * SLOT + (row0 + lane) * 16 + (part * H + h) * 4
                                      : slots + stage * SLOT + (h * ROWS + row0 + lane) * 4;
    return *(const uint32_t*)p;
  };
  auto scales_of = [&](int stage, int part, int row0) {  // lane l's: row row0 + l % 16, its four of the stage
    const int row = row0 + (lane & 15);
    return *(const uint32_t*)(SW == 16 ? slots + at * SLOT + row * 16 + part * 4 : slots + stage * SLOT + row * 4);
  };
  MxFrag<FA> fa[TM];
  MxFrag<FB> fb[TN], fn[TN];
  uint32_t sa[TM / 4], sb[TN / 4];
  constexpr int P = OA::PER + OB::PER;  // loads of a stage's codes
  if constexpr (!EXACT) {
    ring_wait<P>();
#pragma unroll
    for (int i = 0; i < TN; ++i) fb[i] = frag_b(0, i, 0);
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[i] = frag_a(0, i, 0);
#pragma unroll
    for (int i = 0; i < TM / 4; ++i) sa[i] = turn(scale(0, 0, wm + 64 * i, 0));
#pragma unroll
    for (int i = 0; i < TN / 4; ++i) sb[i] = turn(scale(0, 0, BM + wn + 64 * i, 0));
  }
  int cur = 0;     // the stage in turn (SW = 4)
  bool credit = false;  // a stage's loads were issued before the last tile's stores
  for (int n = 0; n < count; ++n) {
    const MxItem it = item(n);
    f32x4_t acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    // products of the fragments in b and fa, and reads of those of the stage's sub-step h into bn and, as they
    // fall free, fa
    auto sub_step = [&](const MxFrag<FB>(&b)[TN], MxFrag<FB>(&bn)[TN], int stage, int part, int h) {
      uint32_t na[TM / 4], nb[TN / 4];
#pragma unroll
      for (int i = 0; i < TM / 4; ++i) na[i] = scale(stage, part, wm + 64 * i, h);
#pragma unroll
      for (int i = 0; i < TN / 4; ++i) nb[i] = scale(stage, part, BM + wn + 64 * i, h);
#pragma unroll
      for (int i = 0; i < TN; ++i) bn[i] = frag_b(stage, i, h);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
#pragma unroll
        for (int i = 0; i < TN; ++i) acc[i][j] = mx_mma_at(i % 4, j % 4, b[i], fa[j], sb[i / 4], sa[j / 4], acc[i][j]);
        fa[j] = frag_a(stage, j, h);
      }
#pragma unroll
      for (int i = 0; i < TM / 4; ++i) sa[i] = turn(na[i]);
#pragma unroll
      for (int i = 0; i < TN / 4; ++i) sb[i] = turn(nb[i]);
      mx_interleave<TM / 4 + TN / 4, FB == ML_MX_E4M3 ? 2 : 1, FA == ML_MX_E4M3 ? 2 : 1, TN, TM>();
    };
    for (int s = max(it.steps, 1); s > 0; --s) {
#pragma unroll
      for (int part = 0; part < SUPER; ++part) {
        const int stage = SW == 16 ? part % NS : cur, next = SW == 16 ? (part + 1) % NS : cur ^ 1;
        if constexpr (EXACT) {
          // the next stage's loads (and the last tile's stores) may be under way
          if (part == 0 && credit) ring_wait<(P + ST < 63 ? P + ST : 63)>();
          else ring_wait<P>();
          credit = credit && part != 0;
          uint32_t ra[TM], rb[TN];  // lane l's: the four scales of row l % 16
#pragma unroll
          for (int j = 0; j < TM; ++j) ra[j] = scales_of(stage, part, wm + 16 * j);
#pragma unroll
          for (int i = 0; i < TN; ++i) rb[i] = scales_of(stage, part, BM + wn + 16 * i);
          const unsigned char* ca = lds + stage * CODES;
          bf16x8_t xa[2][TM], xb[2][TN];
          auto blocks = [&](int b) {
#pragma unroll
            for (int i = 0; i < TN; ++i)
              xb[b & 1][i] = mx_block<FB, typename OB::O>(ca + OA::BYTES, wn + 16 * i, b, rb[i] >> (8 * b) & 255u);
#pragma unroll
            for (int j = 0; j < TM; ++j)
              xa[b & 1][j] = mx_block<FA, typename OA::O>(ca, wm + 16 * j, b, ra[j] >> (8 * b) & 255u);
          };
          blocks(0);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            if (b < 3) blocks(b + 1);
#pragma unroll
            for (int j = 0; j < TM; ++j)
#pragma unroll
              for (int i = 0; i < TN; ++i)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xb[b & 1][i], xa[b & 1][j], acc[i][j], 0, 0, 0);
            if (b < 3) {  // the next block's reads and conversions between the products
              __builtin_amdgcn_sched_group_barrier(0x100, TM + TN, 0);
#pragma unroll
              for (int q = 0; q < TM * TN; ++q) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, 3, 0);
              }
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          ring_wait<63>();  // (no load is waited for: every wave has read the stage)
          load(stage, (part + NS) % SUPER == 0);
          if (part + 1 == SUPER) at ^= 1;
          cur ^= 1;
          continue;
        }
        if constexpr (H == 2) sub_step(fb, fn, stage, part, 1);
        // the products so far stay on this side of the wait: sunk to the next, they would keep both fragments (nothing is
        // read here: the compiler puts the wait states of a matrix instruction in front of the result's first reader)
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int j = 0; j < TM; ++j) asm volatile("" : "+v"(acc[i][j]));
        // the next stage's loads were issued before a full tile's stores, where they came between
        if (part == 0 && credit) ring_wait<(ST < 63 ? ST : 63)>();
        else ring_wait<0>();
        if (part == 0) credit = false;
        load(stage, (part + NS) % SUPER == 0);
        if (part + 1 == SUPER) at ^= 1;
        cur ^= 1;
        if (H == 2 || part % 2 == 1) {
          sub_step(fn, fb, next, (part + 1) % SUPER, 0);
        } else {
          sub_step(fb, fn, next, (part + 1) % SUPER, 0);
          if constexpr (SUPER % 2 == 1)
#pragma unroll
            for (int i = 0; i < TN; ++i) fb[i] = fn[i];
        }
      }
    }

    // lane l holds columns 4 (l / 16) .. + 3 of row l % 16 of each 16 x 16 tile
    const int m0 = it.m0, n0 = it.n0, tm = it.mlim, iw = it.w, block = it.block;
    const bool mapped = it.kind == 1;
    const int tn = a.N - n0;
    const bool full = tm >= BM && tn >= BN && block < 0;
    int el = lane;
    asm("" : "+v"(el));  // (as in grouped_ring_kernel: not known to be the same for every tile)
    const int mr = wm + (el & 15), g = el >> 4;
    auto row_start = [&](int j) {  // of the lane's row in row tile j
      const int r = mr + 16 * j;
      return n0 + (int64_t)(mapped ? merged_row(a, e, iw, m0 + min(r, tm - 1)) : m0 + r) * a.ldc;
    };
    if (block >= 0) {  // in the order of the registers (grouped_tail_kernel)
      f32x4_t* c = (f32x4_t*)a.parts + ((int64_t)(xcd * turns + block) * NW + wave) * (TN * TM * 64) + el;
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) c[(i * TM + j) * 64] = acc[i][j];
    } else if constexpr (OUT == ML_F32) {
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        float* c = (float*)a.c + row_start(j) + wn + 4 * g;
#pragma unroll
        for (int i = 0; i < TN; ++i) {
          if (full) {
            *(f32x4_loose*)(c + 16 * i) = acc[i][j];
            continue;
          }
          const int room = mr + 16 * j < tm ? tn - (wn + 16 * i + 4 * g) : 0;
          if (room >= 4) {
            *(f32x4_loose*)(c + 16 * i) = acc[i][j];
          } else {
#pragma unroll
            for (int q4 = 0; q4 < 3; ++q4)
              if (q4 < room) c[16 * i + q4] = acc[i][j][q4];
          }
        }
      }
    } else {
      // two tiles' columns change places between lane groups 0 and 1, 2 and 3, so that a lane
      // has eight consecutive ones: of the first tile in even groups, of the second in odd ones
      const int col = wn + 16 * (g & 1) + 8 * (g >> 1);
      auto eight = [&](int i, int j) {
        const f32x4_t u = acc[i][j], v = acc[i + 1][j];
        const auto lo = __builtin_amdgcn_permlane16_swap(GMma<OUT>::pack(u[0], u[1]), GMma<OUT>::pack(v[0], v[1]), false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap(GMma<OUT>::pack(u[2], u[3]), GMma<OUT>::pack(v[2], v[3]), false, false);
        return u32x4_t{lo[0], hi[0], lo[1], hi[1]};
      };
      if (full) {
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          uint16_t* c = (uint16_t*)a.c + row_start(j) + col;
#pragma unroll
          for (int i = 0; i < TN; i += 2) *(u32x4_loose*)(c + 16 * i) = eight(i, j);
          __builtin_amdgcn_sched_barrier(0);  // one row tile's conversions at a time: registers
        }
      } else {
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          uint16_t* c = (uint16_t*)a.c + row_start(j) + col;
#pragma unroll
          for (int i = 0; i < TN; i += 2) {
            const u32x4_t o = eight(i, j);
            const int room = mr + 16 * j < tm ? tn - (col + 16 * i) : 0;
            if (room >= 8) {
              *(u32x4_loose*)(c + 16 * i) = o;
            } else {
#pragma unroll
              for (int q8 = 0; q8 < 7; ++q8)
                if (q8 < room) c[16 * i + q8] = (uint16_t)(o[q8 / 2] >> (16 * (q8 & 1)));
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    credit = full;
  }
  ring_wait<0>();  // the last loads end before the LDS goes to another workgroup
}

}  // namespace ml
