// Products of ragged groups of rows with one matrix per group (gfx950): the shared
// kernel.  See ml_grouped.hip for the entry points and the choice of tiles.
//
// Group g holds rows e[g] .. e[g + 1] of a (rows, K) operand and takes matrix
// g % matrices, so that the L * B query sets of L layers share B feature maps.
// Three products are asked for:
//
//   forward           y_r  = x_r W_g          reduces K, contiguous in x
//   input gradient    dx_r = dy_r W_g^T       reduces N, contiguous in dy
//   weight gradient   dW_w = sum x_g^T dy_g   reduces the rows of every group of w
//
// so an operand's reduced index is either contiguous in memory (KC) or the row
// index (not KC), and one kernel with both as template arguments serves all three
// and both storage orders of W.
//
// A workgroup makes a BM x BN tile: both operands pass through LDS in steps of 128
// bytes of the reduced index (64 16-bit or 32 float elements), double buffered:
// a step is loaded into registers one step ahead, written to LDS beside the
// products of the step before, one barrier a step.  Loads of 16 bytes need only
// the element's alignment, so odd row lengths take the same path; a chunk that
// the operand's edge cuts is read element by element, zeros behind it.  A reduced
// index past its end is zero in both operands (a NaN beyond it never counts).
//
// LDS images are XOR-swizzled so that the reads below meet every bank once:
//   KC      rows of 128 bytes, 16-byte chunk c of row r at c ^ (r / 2 % 8): a read of
//           16 rows at one chunk covers 256 bytes
//   not KC  rows of the tile's width, one per reduced index k.  16-bit: 32-byte unit u
//           at u ^ (k % 4 + 4 (k / 8 % 2)), read by ds_read_b64_tr_b16, which hands 16
//           lanes that address 4 k x 16 columns the 4 k of one column each; float:
//           64-byte unit u at u ^ (k / 4 % 4), read word by word
//
// The matrix instruction takes the tile's columns as its rows, so a lane ends with
// four consecutive columns of one output row and stores them at once.
#pragma once

#include <type_traits>

#include "ml_internal.h"

namespace ml {

struct GroupedArgs {
  const void *a, *b;       // row operand and matrix; weight gradient: operands by columns
  int64_t lda, ldb, ldc;   // row lengths, elements
  int64_t bstride, cstride;  // elements per matrix: of b (rows kernel), of c (weight gradient)
  const int64_t* offsets;  // null: equal groups
  int rows, groups, matrices;
  int K;                   // reduced length (rows kernel)
  int M, N;                // output rows (weight gradient) and columns
  int splits;              // parts of the reduction, each with its own float plane
  int64_t plane;           // elements of one plane (splits > 1)
  void* c;                 // output, or the planes
};

template <int DT>
struct GMma;
template <>
struct GMma<ML_BF16> {
  static __device__ __forceinline__ f32x4_t mma(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
};
template <>
struct GMma<ML_F16> {
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4_t mma(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const h2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
};
template <>
struct GMma<ML_F32> {
  // four products of 4 reduced indices: lane group g holds 4 g .. 4 g + 3 of both operands
  static __device__ __forceinline__ f32x4_t mma(const u32x4_t& a, const u32x4_t& b, f32x4_t c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
  }
};

// 16 bytes at any element's alignment (one global_load_dwordx4 / store).
typedef u32x4_t u32x4_loose __attribute__((aligned(2)));
typedef u32x2_t u32x2_loose __attribute__((aligned(2)));
typedef f32x4_t f32x4_loose __attribute__((aligned(4)));
__device__ __forceinline__ u32x4_t load16(const void* p) { return *(const u32x4_loose*)p; }

constexpr int kStepBytes = 128;  // bytes of the reduced index per step

// One operand of a tile: R rows (KC) or columns (not KC) by one step of the reduced
// index, staged by NT threads.
template <int DT, bool KC, int R, int NT>
struct Operand {
  using E = typename std::conditional<DT == ML_F32, float, uint16_t>::type;
  static constexpr int ES = sizeof(E), CH = 16 / ES;  // elements of a chunk
  static constexpr int BK = kStepBytes / ES;
  static constexpr int CPR = (KC ? BK : R) / CH;      // chunks of an LDS row
  static constexpr int ROWB = CPR * 16;
  static constexpr int BYTES = R * BK * ES;
  static constexpr int PER = BYTES / 16 / NT;
  static_assert(PER * NT * 16 == BYTES, "whole chunks per thread");
  static_assert(KC || R * ES >= 256, "a row that holds the swizzle");

  u32x4_t reg[PER];

  static __device__ __forceinline__ int chunk_row(int i) { return ((int)threadIdx.x + i * NT) / CPR; }
  static __device__ __forceinline__ int chunk_col(int i) { return ((int)threadIdx.x + i * NT) % CPR; }

  // base: the operand's element (first row, first reduced index) of this step; ld: row
  // length; lim: valid rows (KC) or columns (not KC), at least 1; kleft: valid reduced
  // indices from here on.  Offsets inside a step stay below 2^32 bytes (host check).
  __device__ __forceinline__ void load(const E* base, int64_t ld, int lim, int kleft) {
    const uint32_t ldb = (uint32_t)ld * ES;
    if (kleft >= BK && (KC || lim >= R)) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        // rows past the last read the last one (their outputs are not stored)
        const uint32_t r = KC ? (uint32_t)min(chunk_row(i), lim - 1) : (uint32_t)chunk_row(i);
        reg[i] = load16((const char*)base + (r * ldb + (uint32_t)chunk_col(i) * 16u));
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int row = chunk_row(i), col = chunk_col(i) * CH;
      const int n = KC ? (row < lim ? kleft - col : 0) : (row < kleft ? lim - col : 0);  // valid elements
      const E* p = (const E*)((const char*)base + ((uint32_t)row * ldb + (uint32_t)col * ES));
      u32x4_t v = {0u, 0u, 0u, 0u};
      if (n >= CH) {
        v = load16(p);
      } else if (n > 0) {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          if (j >= n) continue;
          if constexpr (ES == 4) v[j] = __float_as_uint(p[j]);
          else v[j / 2] |= (uint32_t)p[j] << (16 * (j & 1));
        }
      }
      reg[i] = v;
    }
  }

  __device__ __forceinline__ void store(unsigned char* lds) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = chunk_row(i), c = chunk_col(i);
      int at;
      if constexpr (KC) at = r * ROWB + ((c ^ ((r >> 1) & 7)) << 4);
      else if constexpr (ES == 2) at = r * ROWB + ((((c >> 1) ^ ((r & 3) | ((r >> 1) & 4))) << 5) | ((c & 1) << 4));
      else at = r * ROWB + ((((c >> 2) ^ ((r >> 2) & 3)) << 6) | ((c & 3) << 4));
      *(u32x4_t*)(lds + at) = reg[i];
    }
  }

  // The fragment of rows / columns row0 .. row0 + 15 (a multiple of 16) in sub-step s
  // (of two) of the step: lane l holds index row0 + l % 16 and 16 bytes of the
  // reduced index, the same ones for both operands.
  static __device__ __forceinline__ u32x4_t frag(const unsigned char* lds, int row0, int s) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    if constexpr (KC) {
      const int row = row0 + r;
      return *(const u32x4_t*)(lds + row * ROWB + (((4 * s + g) ^ ((row >> 1) & 7)) << 4));
    } else if constexpr (ES == 2) {
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s4 lds_s4;
      // lane r of a group addresses k = r / 4 of four, columns 4 (r % 4) ..
      const int k = 32 * s + 8 * g + (r >> 2);
      const int at = k * ROWB + (((row0 >> 4) ^ ((k & 3) | ((k >> 1) & 4))) << 5) + ((r & 3) << 3);
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds + at));
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds + at + 4 * ROWB));
      const u32x2_t l2 = __builtin_bit_cast(u32x2_t, lo), h2 = __builtin_bit_cast(u32x2_t, hi);
      return u32x4_t{l2[0], l2[1], h2[0], h2[1]};
    } else {
      const int k = 16 * s + 4 * g;
      const uint32_t* p = (const uint32_t*)(lds + k * ROWB + (((row0 >> 4) ^ ((k >> 2) & 3)) << 6) + r * 4);
      return u32x4_t{p[0], p[ROWB / 4], p[2 * (ROWB / 4)], p[3 * (ROWB / 4)]};
    }
  }
};

// Group edges e[0 .. groups] from the offsets, each held to 0 .. rows and to at least
// the one before, so that any offsets give disjoint groups inside the tensors.  Every
// wave writes the same values.
__device__ __forceinline__ void group_edges(const GroupedArgs& a, int* e) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0; base <= a.groups; base += 64) {
    const int i = base + lane;
    int v = 0;
    if (i <= a.groups) {
      const int64_t o = a.offsets ? a.offsets[i] : (int64_t)i * (a.rows / a.groups);
      v = o < 0 ? 0 : o > a.rows ? a.rows : (int)o;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = max(v, __shfl_up(v, d, 64));
    v = max(v, before);
    if (i <= a.groups) e[i] = v;
    before = __shfl(v, 63, 64);
  }
  __syncthreads();
}

// Rows of segment q: the groups, those that share a matrix next to each other,
// then the rows before the first group and behind the last (g = -1: zeros).
__device__ __forceinline__ void segment(const GroupedArgs& a, const int* e, int q, int& g, int& r0, int& r1) {
  g = -1;
  r0 = r1 = 0;
  if (q < a.groups) {
    const int layers = a.groups / a.matrices;
    g = (q % layers) * a.matrices + q / layers;
    r0 = e[g];
    r1 = e[g + 1];
  } else if (q == a.groups) {
    r1 = e[0];
  } else if (q == a.groups + 1) {
    r0 = e[a.groups];
    r1 = a.rows;
  }
}

constexpr int kXcds = 8;
// Consecutive workgroups go to the XCDs in turn; work item of this workgroup when
// each XCD takes one run of consecutive items (which share operands in its L2), or -1.
__device__ __forceinline__ int xcd_item(int items) {
  const int per = (items + kXcds - 1) / kXcds, at = (int)blockIdx.x / kXcds;
  const int id = ((int)blockIdx.x % kXcds) * per + at;
  return at < per && id < items ? id : -1;
}

// WG: weight gradient (both operands by rows of the tensors, the groups of one matrix
// reduced); otherwise the row operand is KC.  BKC: the matrix's reduced index is
// contiguous.  WM x WN waves make BM x BN.
template <int DT, bool WG, bool BKC, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void grouped_kernel(GroupedArgs a) {
  constexpr int NT = 64 * WM * WN;
  using OA = Operand<DT, !WG, BM, NT>;
  using OB = Operand<DT, BKC, BN, NT>;
  using E = typename OA::E;
  constexpr int BK = OA::BK, TM = BM / WM / 16, TN = BN / WN / 16;
  __shared__ __align__(1024) unsigned char lds[2 * (OA::BYTES + OB::BYTES)];
  extern __shared__ int e[];  // groups + 1 group edges, then groups + 2 tile counts (rows kernel)

  group_edges(a, e);
  const int ntiles = (a.N + BN - 1) / BN;
  const int lane = threadIdx.x & 63;
  int m0, n0, split, mlim;   // tile's first output row and column, its rows
  int w = 0;                 // matrix
  // reduced range of this workgroup: [k, kend) of segment `seg` of nseg
  int k = 0, kend = 0, seg = 0, nseg = 1, steps_left;
  if constexpr (!WG) {
    // tiles up to and with each segment
    int* t = e + a.groups + 1;
    int tiles = 0;
    for (int base = 0; base < a.groups + 2; base += 64) {
      int gg, r0, r1;
      segment(a, e, base + lane, gg, r0, r1);
      int v = (r1 - r0 + BM - 1) / BM;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(v, d, 64);
        v += lane >= d ? u : 0;
      }
      v += tiles;
      if (base + lane < a.groups + 2) t[base + lane] = v;
      tiles = __shfl(v, 63, 64);
    }
    const int id = xcd_item(tiles * ntiles * a.splits);
    if (id < 0) return;
    // bands of kBand row tiles pass over the columns together: their rows and the
    // matrix's columns are both met again while they are in the L2
    constexpr int kBand = 4;
    const int band = id / (kBand * ntiles * a.splits);
    const int height = min(kBand, tiles - band * kBand);
    int rest = id - band * kBand * ntiles * a.splits;
    split = rest / (height * ntiles);
    rest -= split * height * ntiles;
    n0 = rest / height * BN;
    const int tile = band * kBand + rest % height;
    __syncthreads();
    int q = 0;
    for (int base = 0; base < a.groups + 2; base += 64)
      q += __popcll(__ballot(base + lane < a.groups + 2 && t[base + lane] <= tile));
    int g, r0, r1;
    segment(a, e, q, g, r0, r1);
    m0 = r0 + (tile - (q ? t[q - 1] : 0)) * BM;
    mlim = r1 - m0;
    w = g < 0 ? 0 : g % a.matrices;
    const int steps = g < 0 ? 0 : (a.K + BK - 1) / BK;
    const int s0 = (int)((int64_t)steps * split / a.splits), s1 = (int)((int64_t)steps * (split + 1) / a.splits);
    k = s0 * BK;
    kend = a.K;
    steps_left = s1 - s0;
  } else {
    const int mtiles = (a.M + BM - 1) / BM;
    const int id = xcd_item(a.matrices * mtiles * ntiles * a.splits);
    if (id < 0) return;
    w = id / (mtiles * ntiles * a.splits);
    int rest = id - w * mtiles * ntiles * a.splits;
    split = rest / (mtiles * ntiles);
    rest -= split * mtiles * ntiles;
    n0 = rest / mtiles * BN;
    m0 = rest % mtiles * BM;
    mlim = a.M - m0;
    nseg = a.groups / a.matrices;
    int steps = 0;
    for (int s = 0; s < nseg; ++s) steps += (e[s * a.matrices + w + 1] - e[s * a.matrices + w] + BK - 1) / BK;
    const int s0 = (int)((int64_t)steps * split / a.splits), s1 = (int)((int64_t)steps * (split + 1) / a.splits);
    steps_left = s1 - s0;
    // the segment that holds step s0
    int skip = s0;
    for (; seg < nseg; ++seg) {
      const int lo = e[seg * a.matrices + w], hi = e[seg * a.matrices + w + 1], n = (hi - lo + BK - 1) / BK;
      if (skip < n) {
        k = lo + skip * BK;
        kend = hi;
        break;
      }
      skip -= n;
    }
  }
  m0 = __builtin_amdgcn_readfirstlane(m0);
  n0 = __builtin_amdgcn_readfirstlane(n0);
  mlim = __builtin_amdgcn_readfirstlane(mlim);
  w = __builtin_amdgcn_readfirstlane(w);
  seg = __builtin_amdgcn_readfirstlane(seg);
  k = __builtin_amdgcn_readfirstlane(k);
  kend = __builtin_amdgcn_readfirstlane(kend);
  steps_left = __builtin_amdgcn_readfirstlane(steps_left);
  const int nlim = a.N - n0;

  const E* pa = (const E*)a.a + (WG ? (int64_t)m0 : (int64_t)m0 * a.lda);
  const E* pb = (const E*)a.b + (WG ? (int64_t)n0 : (int64_t)w * a.bstride + (BKC ? (int64_t)n0 * a.ldb : n0));
  OA oa;
  OB ob;
  auto fetch = [&]() {  // the step at k
    oa.load(pa + (WG ? (int64_t)k * a.lda : (int64_t)k), a.lda, mlim, kend - k);
    ob.load(pb + (BKC ? (int64_t)k : (int64_t)k * a.ldb), a.ldb, nlim, kend - k);
  };
  auto advance = [&]() {
    k += BK;
    if constexpr (WG) {
      while (k >= kend && seg + 1 < nseg) {
        ++seg;
        k = __builtin_amdgcn_readfirstlane(e[seg * a.matrices + w]);
        kend = __builtin_amdgcn_readfirstlane(e[seg * a.matrices + w + 1]);
      }
    }
  };

  f32x4_t acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int wave = threadIdx.x >> 6, wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);

  if (steps_left > 0) {
    fetch();
    oa.store(lds);
    ob.store(lds + OA::BYTES);
    if (steps_left > 1) {
      advance();
      fetch();
    }
    __syncthreads();
    for (int s = 0; s < steps_left; ++s) {
      unsigned char* cur = lds + (s & 1) * (OA::BYTES + OB::BYTES);
      unsigned char* nxt = lds + ((s & 1) ^ 1) * (OA::BYTES + OB::BYTES);
      if (s + 1 < steps_left) {
        oa.store(nxt);
        ob.store(nxt + OA::BYTES);
        if (s + 2 < steps_left) {
          advance();
          fetch();
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4_t fa[TM], fb[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[i] = OA::frag(cur, wm + 16 * i, h);
#pragma unroll
        for (int i = 0; i < TN; ++i) fb[i] = OB::frag(cur + OA::BYTES, wn + 16 * i, h);
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int j = 0; j < TM; ++j) acc[i][j] = GMma<DT>::mma(fb[i], fa[j], acc[i][j]);
      }
      __syncthreads();
    }
  }

  // lane l holds columns 4 (l / 16) .. + 3 of row l % 16 of each 16 x 16 tile
  const int64_t first = WG ? (int64_t)w * a.cstride : 0;
  const bool planes = a.splits > 1;
  float* cf = (float*)a.c + (planes ? (int64_t)split * a.plane : 0);
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int m = wm + 16 * j + (lane & 15);
    if (m >= mlim) continue;
    const int64_t row = first + (int64_t)(m0 + m) * a.ldc;
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      const int n = wn + 16 * i + 4 * (lane >> 4);
      if (n >= nlim) continue;
      const f32x4_t v = acc[i][j];
      const int64_t at = row + n0 + n;
      if (planes || DT == ML_F32) {
        if (n + 4 <= nlim) {
          *(f32x4_loose*)(cf + at) = v;
        } else {
#pragma unroll
          for (int q = 0; q < 3; ++q)
            if (n + q < nlim) cf[at + q] = v[q];
        }
      } else if constexpr (DT != ML_F32) {
        const u32x2_t p = {GMma<DT>::pack(v[0], v[1]), GMma<DT>::pack(v[2], v[3])};
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
