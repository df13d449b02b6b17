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
//   KC      rows of 128 bytes, 16-byte chunk c of row r at c ^ (r / 2 % 8); rows of 64
//           bytes, at c ^ swizzle64(r)
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

// Division of 0 <= n < 2^31 by a positive int known to the host: (mulhi(n, mul) + n) >> shift with
// mul = floor(2^32 (2^shift - d) / d) + 1, 2^shift >= d.
struct FastDiv {
  uint32_t mul, shift;
  int d;
};
inline FastDiv fast_div(int64_t d) {
  FastDiv f;
  f.d = (int)d;
  f.shift = 0;
  while (((int64_t)1 << f.shift) < d) ++f.shift;
  f.mul = (uint32_t)(((((uint64_t)1 << f.shift) - (uint64_t)d) << 32) / (uint64_t)d + 1);
  return f;
}
__device__ __forceinline__ int div_by(int n, const FastDiv& f) {
  return (int)((__umulhi((uint32_t)n, f.mul) + (uint32_t)n) >> f.shift);
}

struct GroupedArgs {
  const void *a, *b;       // row operand and matrix; weight gradient: operands by columns
  int64_t lda, ldb, ldc;   // row lengths, elements
  int64_t bstride, cstride;  // elements per matrix: of b (rows kernel), of c (weight gradient)
  const int64_t* offsets;  // null: groups of `equal` rows
  int equal;
  int rows, groups, matrices;
  int given;               // groups of the call; groups = 1 where there is one matrix (a range of rows)
  int K;                   // reduced length (rows kernel)
  int M, N;                // output rows (weight gradient) and columns
  int splits;              // grouped_kernel: parts of each tile's reduction, float planes in `parts`;
                           // grouped_ring_kernel: most parts of a tile of the last round
  int fewest;              // parts from which on they are worth their join behind whole rounds
  int64_t plane;           // elements of one plane
  void* c;                 // output
  float* parts;
  int segments;            // row ranges with a matrix: the groups, or (merged) the matrices
  int merged;              // the rows of the groups that share a matrix make tiles together
  FastDiv layers;          // groups per matrix
  FastDiv cols;            // column tiles
  FastDiv mtiles;          // row tiles of a matrix (weight gradient)
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
  static __device__ __forceinline__ f32x4_t mma(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    // (by the compiler, which puts the wait states between a matrix instruction and its result's first
    // reader; it does not look into assembly)
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    f32x2_t f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, h2));
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

typedef __attribute__((address_space(3))) void lds_void_t;

// A ds_read_b128 passes 16 lanes at a time, lanes 0-3, 12-15 and 20-27 first, then 4-11, 16-19 and
// 28-31, and so on.  With rows of 64 bytes and chunk l / 16 of row l % 16 wanted by lane l,
// these values for the rows' fours (0, 2, 3, 1) put the 16 into different banks each time.
__device__ __forceinline__ int swizzle64(int row) {
  const int lo = (row >> 2) & 1, hi = (row >> 3) & 1;
  return ((lo ^ hi) << 1) | hi;
}

// One operand of a tile: R rows (KC) or columns (not KC) by one step of the reduced
// index (SB bytes), staged by NT threads.
template <int DT, bool KC, int R, int NT, int SB = 128>
struct Operand {
  using E = typename std::conditional<DT == ML_F32, float, uint16_t>::type;
  static constexpr int ES = sizeof(E), CH = 16 / ES;  // elements of a chunk
  static constexpr int BK = SB / ES;
  static constexpr int CPR = (KC ? BK : R) / CH;      // chunks of an LDS row
  static constexpr int ROWB = CPR * 16;
  static constexpr int BYTES = R * BK * ES;
  static constexpr int PER = BYTES / 16 / NT;
  static_assert(PER * NT * 16 == BYTES, "whole chunks per thread");
  static_assert(KC || R * ES >= 256, "a row that holds the swizzle");
  static_assert(SB == 64 || SB == 128, "the swizzles");

  // chunk c of LDS row r lies at chunk swizzled(r, c), and the other way round
  static __device__ __forceinline__ int swizzled(int r, int c) {
    if constexpr (KC) return c ^ (SB == 128 ? (r >> 1) & 7 : swizzle64(r));
    else if constexpr (ES == 2) return c ^ (((r & 3) | ((r >> 1) & 4)) << 1);
    else return c ^ (((r >> 2) & 3) << 2);
  }

  u32x4_t reg[PER];

  uint32_t off[PER];  // bytes of this thread's chunks from a step's first element

  static __device__ __forceinline__ int chunk_row(int i) { return ((int)threadIdx.x + i * NT) / CPR; }
  static __device__ __forceinline__ int chunk_col(int i) { return ((int)threadIdx.x + i * NT) % CPR; }

  // ld: row length; lim: valid rows (KC) or columns (not KC) of the tile, at least 1.  row_at(r): where
  // row r of the tile lies (KC), in rows from the base.  Offsets stay below 2^32 bytes (host check).
  template <class F>
  __device__ __forceinline__ void aim(int64_t ld, int lim, F&& row_at) {
    const uint32_t ldb = (uint32_t)ld * ES;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      // rows past the last read the last one (their outputs are not stored)
      off[i] = (uint32_t)(KC ? row_at(min(chunk_row(i), lim - 1)) : chunk_row(i)) * ldb + (uint32_t)chunk_col(i) * 16u;
  }
  // base: the step's first element; kleft: valid reduced indices from here on
  __device__ __forceinline__ void load(const E* base, int lim, int kleft) {
    if (kleft >= BK && (KC || lim >= R)) {
#pragma unroll
      for (int i = 0; i < PER; ++i) reg[i] = load16((const char*)base + off[i]);
      return;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int row = chunk_row(i), col = chunk_col(i) * CH;
      const int n = KC ? (row < lim ? kleft - col : 0) : (row < kleft ? lim - col : 0);  // valid elements
      const E* p = (const E*)((const char*)base + off[i]);
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
      *(u32x4_t*)(lds + r * ROWB + (swizzled(r, c) << 4)) = reg[i];
    }
  }

  // The fragment of rows / columns row0 .. row0 + 15 (a multiple of 16) in sub-step s
  // (64 bytes) of the step: lane l holds index row0 + l % 16 and 16 bytes of the
  // reduced index, the same ones for both operands.
  static __device__ __forceinline__ u32x4_t frag(const unsigned char* lds, int row0, int s) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    if constexpr (KC) {
      // (row0 does not change the swizzle)
      return *(const u32x4_t*)(lds + (row0 + r) * ROWB + (swizzled(r, 4 * s + g) << 4));
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

// Inclusive scans over the wave of values that are not negative, in the vector ALU: shifts by 1, 2, 4
// and 8 within 16 lanes, then the last lane of a row (of two rows) to the rows behind it.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or_zero(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int scan_max(int v) {
  v = max(v, dpp_or_zero<0x111, 0xf>(v));
  v = max(v, dpp_or_zero<0x112, 0xf>(v));
  v = max(v, dpp_or_zero<0x114, 0xf>(v));
  v = max(v, dpp_or_zero<0x118, 0xf>(v));
  v = max(v, dpp_or_zero<0x142, 0xa>(v));
  return max(v, dpp_or_zero<0x143, 0xc>(v));
}
__device__ __forceinline__ int scan_sum(int v) {
  v += dpp_or_zero<0x111, 0xf>(v);
  v += dpp_or_zero<0x112, 0xf>(v);
  v += dpp_or_zero<0x114, 0xf>(v);
  v += dpp_or_zero<0x118, 0xf>(v);
  v += dpp_or_zero<0x142, 0xa>(v);
  return v + dpp_or_zero<0x143, 0xc>(v);
}

// Group edges e[0 .. groups] from the offsets, each held to 0 .. rows and to at least
// the one before, so that any offsets give disjoint groups inside the tensors; the groups of
// one matrix are one range of rows.  Every wave writes the same values.
__device__ __forceinline__ void group_edges(const GroupedArgs& a, int* e) {
  const int lane = threadIdx.x & 63;
  const bool range = a.groups < a.given;
  int before = 0;
  for (int base = 0; base <= a.given; base += 64) {
    const int i = base + lane;
    int v = 0;
    if (i <= a.given) {
      const int64_t o = a.offsets ? a.offsets[i] : (int64_t)i * a.equal;
      v = o < 0 ? 0 : o > a.rows ? a.rows : (int)o;
    }
    v = max(scan_max(v), before);
    if (i <= (range ? 0 : a.given)) e[i] = v;
    before = __builtin_amdgcn_readlane(v, 63);
  }
  if (range) e[1] = before;
  __syncthreads();
}

// Segment q: rows r0 .. r1 that make tiles of their own.  The groups, those that share a matrix
// (q / layers) next to each other, or (merged) each matrix's rows of all its groups, counted from 0;
// then the rows before the first group and behind the last (zeros).
__device__ __forceinline__ void segment(const GroupedArgs& a, const int* e, int q, int& r0, int& r1) {
  r0 = r1 = 0;
  if (q < a.segments) {
    if (a.merged) {
      for (int g = q; g < a.groups; g += a.matrices) r1 += e[g + 1] - e[g];
    } else {
      const int w = div_by(q, a.layers), g = (q - w * a.layers.d) * a.matrices + w;
      r0 = e[g];
      r1 = e[g + 1];
    }
  } else if (q == a.segments) {
    r1 = e[0];
  } else if (q == a.segments + 1) {
    r0 = e[a.groups];
    r1 = a.rows;
  }
}
// Row v of matrix w's rows (merged).
__device__ __forceinline__ int merged_row(const GroupedArgs& a, const int* e, int w, int v) {
  int g = w;
  for (; g + a.matrices < a.groups && v >= e[g + 1] - e[g]; g += a.matrices) v -= e[g + 1] - e[g];
  return e[g] + v;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Tiles of bm rows up to and with each segment, t[0 .. segments + 1]; returns their number.  Every wave
// writes the same values.
__device__ __forceinline__ int segment_tiles(const GroupedArgs& a, const int* e, int* t, int bm) {
  const int lane = threadIdx.x & 63;
  int tiles = 0;
  for (int base = 0; base < a.segments + 2; base += 64) {
    int r0, r1;
    segment(a, e, base + lane, r0, r1);
    int v = (int)((uint32_t)(r1 - r0 + bm - 1) / (uint32_t)bm);
    v = scan_sum(v) + tiles;
    if (base + lane < a.segments + 2) t[base + lane] = v;
    tiles = __builtin_amdgcn_readlane(v, 63);
  }
  __syncthreads();
  return tiles;
}

// A work item: a tile of the output and part `part` of `parts` of its reduction, `steps` steps of bk from
// reduced index k on; k runs to kend, then (weight gradient) through the matrix's next groups.
struct Work {
  int m0, n0, mlim, w, steps;
  int seg, k, kend;
  int mapped;  // m0 counts matrix w's rows (merged_row), not the tensor's
};

// Steps of part `part` of `parts` begin at this one of n.
__device__ __forceinline__ int part_start(int n, int part, int parts) {
  if (parts == 1) return part * n;
  const int each = n / parts;
  return each * part + min(part, n - each * parts);
}

// (1, 2, 4, 8 row tiles to a band: experts' forward of ml_grouped.hip 201, 173, 163, 173 us, masks' d input
// 201, 203, 196, 275.)
constexpr int kBand = 4;
// Rows kernels, tile id of tiles * column tiles.  Bands of kBand row tiles pass over the columns
// together: their rows and the matrix's columns are both met again while they are in the L2.
__device__ __forceinline__ Work rows_work(const GroupedArgs& a, const int* e, const int* t, int tiles, int id, int part,
                                          int parts, int bm, int bn, int bk) {
  const int lane = threadIdx.x & 63;
  Work it;
  it.seg = 0;
  const int band = div_by(id >> 2, a.cols);  // kBand = 4
  const int height = min(kBand, tiles - band * kBand);
  const int rest = id - band * kBand * a.cols.d;
  const int y = height == 4 ? rest >> 2 : height == 3 ? (int)(__umulhi((uint32_t)rest, 0xAAAAAAABu) >> 1)
                                                      : rest >> (height - 1);
  it.n0 = y * bn;
  const int tile = band * kBand + rest - y * height;
  int q = 0;
  for (int base = 0; base < a.segments + 2; base += 64)
    q += __popcll(__ballot(base + lane < a.segments + 2 && t[base + lane] <= tile));
  int r0, r1;
  segment(a, e, q, r0, r1);
  it.m0 = uniform(r0 + (tile - (q ? t[q - 1] : 0)) * bm);
  it.mlim = uniform(r1) - it.m0;
  const bool zero = q >= a.segments;
  it.w = zero ? 0 : a.merged ? q : div_by(q, a.layers);
  it.mapped = a.merged && !zero;
  const int steps = zero ? 0 : (int)((uint32_t)(a.K + bk - 1) / (uint32_t)bk);
  const int s0 = part_start(steps, part, parts);
  it.steps = part_start(steps, part + 1, parts) - s0;
  it.k = s0 * bk;
  it.kend = zero ? 0 : a.K;
  return it;
}

// Weight gradient, tile id of matrices * column tiles * row tiles.
__device__ __forceinline__ Work weight_work(const GroupedArgs& a, const int* e, int id, int part, int parts, int bm,
                                            int bn, int bk) {
  Work it;
  it.mapped = 0;
  const int x = div_by(id, a.mtiles);
  it.m0 = (id - x * a.mtiles.d) * bm;
  it.mlim = a.M - it.m0;
  it.w = div_by(x, a.cols);
  it.n0 = (x - it.w * a.cols.d) * bn;
  const int* ew = e + it.w;
  // 64 groups at a time: all steps of the matrix, then the group that holds this part's first one
  const int lane = threadIdx.x & 63;
  auto steps_to = [&](int base) {  // steps of groups base .. base + lane
    const int s = base + lane;
    const int n = s < a.layers.d ? ew[s * a.matrices + 1] - ew[s * a.matrices] : 0;
    return scan_sum((int)((uint32_t)(n + bk - 1) / (uint32_t)bk));
  };
  int steps = 0;
  for (int base = 0; base < a.layers.d; base += 64) steps += __builtin_amdgcn_readlane(steps_to(base), 63);
  const int s0 = uniform(part_start(steps, part, parts));
  it.steps = part_start(steps, part + 1, parts) - s0;
  it.k = it.kend = 0;
  it.seg = a.layers.d;
  int skip = s0;
  for (int base = 0; base < a.layers.d; base += 64) {
    const int upto = steps_to(base), here = __builtin_amdgcn_readlane(upto, 63);
    if (skip < here) {
      const int i = __popcll(__ballot(upto <= skip));
      it.seg = base + i;
      it.k = uniform(ew[it.seg * a.matrices]) + (skip - (i ? __builtin_amdgcn_readlane(upto, i - 1) : 0)) * bk;
      it.kend = uniform(ew[it.seg * a.matrices + 1]);
      break;
    }
    skip -= here;
  }
  return it;
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
  const int lane = threadIdx.x & 63;
  Work it;
  int split;
  if constexpr (WG) {
    const int count = a.matrices * a.mtiles.d * a.cols.d, id = xcd_item(count * a.splits);
    if (id < 0) return;
    split = id / count;
    it = weight_work(a, e, id - split * count, split, a.splits, BM, BN, BK);
  } else {
    int* t = e + a.groups + 1;
    const int tiles = segment_tiles(a, e, t, BM), count = tiles * a.cols.d, id = xcd_item(count * a.splits);
    if (id < 0) return;
    split = id / count;
    it = rows_work(a, e, t, tiles, id - split * count, split, a.splits, BM, BN, BK);
  }
  const int m0 = uniform(it.m0), n0 = uniform(it.n0), mlim = uniform(it.mlim), w = uniform(it.w);
  const int steps_left = uniform(it.steps);
  int k = uniform(it.k), kend = uniform(it.kend), seg = uniform(it.seg);
  const int nlim = a.N - n0;

  const bool mapped = uniform(it.mapped) != 0;
  auto row_at = [&](int r) { return mapped ? merged_row(a, e, w, m0 + r) : r; };
  const E* pa = (const E*)a.a + (WG ? (int64_t)m0 : mapped ? (int64_t)0 : (int64_t)m0 * a.lda);
  const E* pb = (const E*)a.b + (WG ? (int64_t)n0 : (int64_t)w * a.bstride + (BKC ? (int64_t)n0 * a.ldb : n0));
  OA oa;
  OB ob;
  oa.aim(a.lda, mlim, row_at);
  ob.aim(a.ldb, nlim, [](int r) { return r; });
  auto fetch = [&]() {  // the step at k
    oa.load(pa + (WG ? (int64_t)k * a.lda : (int64_t)k), mlim, kend - k);
    ob.load(pb + (BKC ? (int64_t)k : (int64_t)k * a.ldb), nlim, kend - k);
  };
  auto advance = [&]() {
    k += BK;
    if constexpr (WG) {
      while (k >= kend && seg + 1 < a.layers.d) {
        ++seg;
        k = uniform(e[seg * a.matrices + w]);
        kend = uniform(e[seg * a.matrices + w + 1]);
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
  float* cf = planes ? a.parts + (int64_t)split * a.plane : (float*)a.c;
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int m = wm + 16 * j + (lane & 15);
    if (m >= mlim) continue;
    const int64_t row = first + (int64_t)(mapped ? row_at(m) : m0 + m) * a.ldc;
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

// ---- aligned operands: stages filled by direct loads into LDS ------------------------
// Where every row starts on a 16-byte boundary, global_load_lds_dwordx4 moves the operands
// straight into LDS, without registers.  The LDS images are grouped_kernel's (a load
// instruction writes 64 consecutive 16-byte slots, so the swizzle is in the lane's source
// address).  A ring of NS stages of SB bytes of the reduced index is in LDS; the workgroups
// are persistent: each XCD's take turns over one run of consecutive work items, and the
// ring runs on from item to item, so the first loads of a tile are in flight while the
// tile before is finished and stored.
//
// A turn of the loop makes the products of one stage, in sub-steps of 64 bytes whose
// fragments are read from LDS beside the products of the sub-step before (interleave()):
//
//   products of sub-step 0     beside reads of sub-step 1 (SB = 128 only)
//   wait: the next stage has landed, every wave has read all of this one; its slot takes
//   the loads NS stages on (zeros where none is left)
//   products of the last one   beside reads of the next stage's sub-step 0
//
// The loads are issued by assembly: the compiler, which cannot tell the stages apart, would
// otherwise wait for all of them before any LDS read.  They have no output registers;
// ring_wait() waits for the ones that matter and keeps LDS reads on their side of the
// barrier.
static __device__ __align__(16) unsigned char g_zeros[16];  // the reduced index past its end

// N loads of 16 bytes from base + off[i] of each lane to LDS at `lds` + 1024 i + 16 lane.  m0 is no
// register that the compiler allocates, and it warns that the clobber list cannot keep its value; with the
// list, a value of its own in m0 (a message's, an index) is set again behind the loads.  base may come right from a
// vector instruction (uniform()): five wait states until a load reads it, which the compiler does not
// put in front of assembly; once for all N (in front of each, the masks' d input took 201 us for 196).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int N>
__device__ __forceinline__ void ring_loads(const char* base, const uint32_t (&off)[N], uint32_t lds) {
  static_assert(N == 2 || N == 4, "loads of an operand");
  if constexpr (N == 2)
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %3\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3"
        :
        : "s"(lds), "v"(off[0]), "v"(off[1]), "s"(base)
        : "memory", "m0", "scc");
  else
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %5\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %5\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %5\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %5"
        :
        : "s"(lds), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base)
        : "memory", "m0", "scc");
}
// 16 bytes from p of each lane to LDS at `lds` + 16 lane.
__device__ __forceinline__ void ring_load(const char* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds), "v"(p)
               : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ const char* uniform(const char* p) {
  const uint64_t u = (uint64_t)(uintptr_t)p;
  return (const char*)(uintptr_t)((uint64_t)(uint32_t)uniform((int)(uint32_t)u) |
                                  ((uint64_t)(uint32_t)uniform((int)(uint32_t)(u >> 32)) << 32));
}
// Until at most N vector-memory operations are outstanding (they complete in order), and
// every wave of the workgroup is here with its LDS reads done.
template <int N>
__device__ __forceinline__ void ring_wait() {
  static_assert(N < 64, "vmcnt");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// An XCD's run of consecutive tiles, from `start` on, among its workgroups (gridDim.x / kXcds): whole ones in
// full rounds, and those of the last round, where they would leave half of the workgroups or
// more without work, in parts of their reduction.
// Behind whole rounds: 16 parts of 128 x 128 tiles cost more at their join than they save (32 tiles left of
// 544, bf16; 8 / 16 parts: 4,352 x 4,096 x 2,048 85 / 93 us, 8,704 x 4,096 x 1,024 78 / 85, 2,176 x 8,192 x
// 4,096 140 / 149).  The 256 x 256 tile's 32 workgroups an XCD seldom leave room for more.
constexpr int kTailParts = 8;
struct RingShare {
  int start, whole, rest, parts;
};
__device__ __forceinline__ RingShare ring_share(const GroupedArgs& a, int count, int xcd, int turns) {
  RingShare s;
  const int per = (count + kXcds - 1) / kXcds;
  s.start = xcd * per;
  const int mine = max(0, min(per, count - s.start));
  s.rest = mine % turns;
  s.whole = mine - s.rest;
  s.parts = s.rest ? min(s.whole ? min(a.splits, kTailParts) : a.splits, turns / s.rest) : 1;
  if (s.parts < (s.whole ? a.fewest : 2)) {
    s.whole = mine;
    s.rest = 0;
    s.parts = 1;
  }
  return s;
}

// One operand of a stage, filled by NW waves.
template <int DT, bool KC, int R, int NW, int SB>
struct RingOperand : Operand<DT, KC, R, 64 * NW, SB> {
  using O = Operand<DT, KC, R, 64 * NW, SB>;
  static constexpr int ES = O::ES, CH = O::CH;
  static constexpr int PER = O::BYTES / 1024 / NW;        // load instructions of a wave
  static constexpr int READS = KC ? 1 : ES == 2 ? 2 : 4;  // LDS reads of a fragment
  static_assert(PER * NW * 1024 == O::BYTES, "whole instructions per wave");

  uint32_t off[PER];  // as Operand's, for the chunks of this lane's loads

  // the chunk of load i: its row in the LDS image, and its column there before the swizzle
  static __device__ __forceinline__ void chunk(int i, int wave, int& row, int& c) {
    const int slot = (wave * PER + i) * 64 + (int)(threadIdx.x & 63), s = slot % O::CPR;
    row = slot / O::CPR;
    c = O::swizzled(row, s);
  }
  // as Operand's; lim is a multiple of CH where it counts columns, and columns past it read the last ones
  template <class F>
  __device__ __forceinline__ void aim(int64_t ld, int lim, int wave, F&& row_at) {
    const uint32_t ldb = (uint32_t)ld * ES;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int row, c;
      chunk(i, wave, row, c);
      off[i] = KC ? (uint32_t)row_at(min(row, lim - 1)) * ldb + (uint32_t)c * 16u
                  : (uint32_t)row * ldb + (uint32_t)min(c * CH, lim - CH) * ES;
    }
  }
  // base: the stage's first element; kleft: valid reduced indices from there on
  __device__ __forceinline__ void load(const char* base, int kleft, uint32_t lds, int wave) const {
    if (kleft >= O::BK) {
      ring_loads(uniform(base), off, lds + wave * PER * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        int row, c;
        chunk(i, wave, row, c);
        ring_load((KC ? c * CH : row) < kleft ? base + off[i] : (const char*)g_zeros, lds + (wave * PER + i) * 1024);
      }
    }
  }
};

// Order of a sub-step's LDS reads (RB and RA for a fragment of either operand) and products
// (N times NM for each of M fragments).
template <int RB, int RA, int N, int M, int NM>
__device__ __forceinline__ void interleave() {
  constexpr int kMfma = 0x8, kRead = 0x100;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(kRead, RB, 0);
    __builtin_amdgcn_sched_group_barrier(kMfma, NM, 0);
  }
#pragma unroll
  for (int j = 1; j < M; ++j) {
    __builtin_amdgcn_sched_group_barrier(kRead, RA, 0);
    __builtin_amdgcn_sched_group_barrier(kMfma, N * NM, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kRead, RA, 0);
}

// Template arguments and dynamic LDS as grouped_kernel's; OCC workgroups to a compute unit.
template <int DT, bool WG, bool BKC, int BM, int BN, int WM, int WN, int SB, int NS, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC * WM * WN / 4) void grouped_ring_kernel(GroupedArgs a) {
  constexpr int NW = WM * WN;
  using OA = RingOperand<DT, !WG, BM, NW, SB>;
  using OB = RingOperand<DT, BKC, BN, NW, SB>;
  constexpr int ES = OA::ES, BK = OA::BK, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int STAGE = OA::BYTES + OB::BYTES, P = OA::PER + OB::PER;
  // stores of a full tile: a lane's 16 bytes are 8 columns of two tiles, or 4 floats
  constexpr int ST = TM * TN / (DT == ML_F32 ? 1 : 2);
  static_assert(TN % 2 == 0, "tiles in pairs");
  constexpr int kQueue = 8;  // items between the loads and the products: at most NS + 2, as each has a stage
  __shared__ __align__(1024) unsigned char lds[NS * STAGE];
  __shared__ int queue[kQueue][8];
  extern __shared__ int e[];

  group_edges(a, e);
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  int* t = e + a.groups + 1;
  const int tiles = WG ? a.matrices * a.mtiles.d : segment_tiles(a, e, t, BM);
  const int xcd = (int)blockIdx.x % kXcds, turns = (int)gridDim.x / kXcds, first = (int)blockIdx.x / kXcds;
  const RingShare share = ring_share(a, tiles * a.cols.d, xcd, turns);
  const int last = share.whole + share.rest * share.parts;
  if (first >= last) return;

  // ---- loads
  OA oa;
  OB ob;
  const uint32_t ring = (uint32_t)(uintptr_t)(lds_void_t*)lds;
  // the item being loaded (next: the one after it), and the stages left of it
  int next = first, opened = 0, left = 0, k = 0, kend = 0, seg = 0, w = 0;
  const char *pa = nullptr, *pb = nullptr;  // the tile's operands at reduced index 0
  auto open_item = [&]() {
    if (next >= last) {  // nothing more: zeros
      left = INT32_MAX;
      k = kend = 0;
      seg = a.layers.d;
      return;
    }
    int tile = share.start + next, part = 0, parts = 1;
    if (next >= share.whole) {  // a part of one of the last tiles
      const int p = next - share.whole, r = p / share.parts;
      tile = share.start + share.whole + r;
      parts = share.parts;
      part = p - r * parts;
    }
    const Work it0 = WG ? weight_work(a, e, tile, part, parts, BM, BN, BK)
                        : rows_work(a, e, t, tiles, tile, part, parts, BM, BN, BK);
    Work it = it0;
    next += turns;
    it.steps = max(it.steps, 1);  // nothing to reduce: one stage of zeros
    if (lane == 0) {
      int* q = queue[opened % kQueue];
      q[0] = it.m0;
      q[1] = it.n0;
      q[2] = it.mlim;
      q[3] = it.w;
      q[4] = parts > 1 ? next - turns - share.whole : -1;
      q[5] = it.steps;
      q[6] = it.mapped;
    }
    ++opened;
    left = uniform(it.steps);
    k = uniform(it.k);
    kend = uniform(it.kend);
    seg = uniform(it.seg);
    w = uniform(it.w);
    const int m0 = uniform(it.m0), n0 = uniform(it.n0);
    const bool mapped = uniform(it.mapped) != 0;
    pa = (const char*)a.a + (WG ? (int64_t)m0 : mapped ? (int64_t)0 : (int64_t)m0 * a.lda) * ES;
    pb = (const char*)a.b + (WG ? (int64_t)n0 : (int64_t)w * a.bstride + (BKC ? (int64_t)n0 * a.ldb : (int64_t)n0)) * ES;
    if (mapped) oa.aim(a.lda, uniform(it.mlim), wave, [&](int r) { return merged_row(a, e, w, m0 + r); });
    else oa.aim(a.lda, uniform(it.mlim), wave, [](int r) { return r; });
    ob.aim(a.ldb, a.N - n0, wave, [](int r) { return r; });
  };
  auto load = [&](uint32_t at) {  // the next stage's loads, into the slot at this LDS offset
    if (left == 0) open_item();
    --left;
    if constexpr (WG) {
      while (k >= kend && seg + 1 < a.layers.d) {
        ++seg;
        k = uniform(e[seg * a.matrices + w]);
        kend = uniform(e[seg * a.matrices + w + 1]);
      }
    }
    oa.load(pa + (WG ? k * a.lda : (int64_t)k) * ES, kend - k, ring + at, wave);
    ob.load(pb + (BKC ? (int64_t)k : k * a.ldb) * ES, kend - k, ring + at + OA::BYTES, wave);
    k += BK;
  };
#pragma unroll 1
  for (int s = 0; s < NS; ++s) load(s * STAGE);

  // ---- products
  const int wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);
  u32x4_t fa[TM], fb[TN], fn[TN];
  ring_wait<(NS - 1) * P>();
#pragma unroll
  for (int i = 0; i < TN; ++i) fb[i] = OB::frag(lds + OA::BYTES, wn + 16 * i, 0);
#pragma unroll
  for (int i = 0; i < TM; ++i) fa[i] = OA::frag(lds, wm + 16 * i, 0);
  uint32_t cur = 0;  // LDS offset of the stage in turn
  int credit = 0;    // stages whose loads were issued before the last tile's stores
  const int count = (last - first + turns - 1) / turns;
  for (int n = 0; n < count; ++n) {
    const int* q = queue[n % kQueue];
    const int steps = uniform(q[5]);
    f32x4_t acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    // products of the fragments in b and fa, and reads of those of sub-step h of the stage at
    // `from` into bn and, as they fall free, fa
    auto sub_step = [&](const u32x4_t(&b)[TN], u32x4_t(&bn)[TN], const unsigned char* from, int h) {
#pragma unroll
      for (int i = 0; i < TN; ++i) bn[i] = OB::frag(from + OA::BYTES, wn + 16 * i, h);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
#pragma unroll
        for (int i = 0; i < TN; ++i) acc[i][j] = GMma<DT>::mma(b[i], fa[j], acc[i][j]);
        fa[j] = OA::frag(from, wm + 16 * j, h);
      }
      // in this order: the scheduler would put the reads behind the products
      interleave<OB::READS, OA::READS, TN, TM, DT == ML_F32 ? 4 : 1>();
    };
    for (int s = 0; s < steps; ++s) {
      if constexpr (SB == 128) sub_step(fb, fn, lds + cur, 1);
      // issued after the next stage's loads: those of NS - 2 more and, where they came between, a
      // full tile's stores
      constexpr int kLoads = (NS - 2) * P;
      if (credit > 0) {
        --credit;
        ring_wait<(kLoads + ST < 63 ? kLoads + ST : 63)>();
      } else {
        ring_wait<kLoads>();
      }
      load(cur);
      cur = cur == (NS - 1) * STAGE ? 0 : cur + STAGE;
      if constexpr (SB == 128) {
        sub_step(fn, fb, lds + cur, 0);
      } else {
        sub_step(fb, fn, lds + cur, 0);
#pragma unroll
        for (int i = 0; i < TN; ++i) fb[i] = fn[i];
      }
    }

    // lane l holds columns 4 (l / 16) .. + 3 of row l % 16 of each 16 x 16 tile; columns come in
    // whole chunks
    const int m0 = uniform(q[0]), n0 = uniform(q[1]), tm = uniform(q[2]), iw = uniform(q[3]), block = uniform(q[4]);
    const bool mapped = uniform(q[6]) != 0;
    const int tn = a.N - n0;
    const bool full = tm >= BM && tn >= BN && block < 0;
    const int64_t origin = (WG ? (int64_t)iw * a.cstride : 0) + n0;
    // (not known to the compiler as the same for every tile: it would keep what follows from it in
    // registers, 10 more of them and spilled ones on the 256 x 256 tile)
    int el = lane;
    asm("" : "+v"(el));
    const int mr = wm + (el & 15), g = el >> 4;
    auto row_start = [&](int j) {  // of the lane's row in row tile j
      const int r = mr + 16 * j;
      return origin + (int64_t)(mapped ? merged_row(a, e, iw, m0 + min(r, tm - 1)) : m0 + r) * a.ldc;
    };
    if (block >= 0) {  // in the order of the registers (grouped_tail_kernel)
      f32x4_t* c = (f32x4_t*)a.parts + ((int64_t)(xcd * turns + block) * NW + wave) * (TN * TM * 64) + el;
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) c[(i * TM + j) * 64] = acc[i][j];
    } else if constexpr (DT == ML_F32) {
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        float* c = (float*)a.c + row_start(j) + wn + 4 * g;
#pragma unroll
        for (int i = 0; i < TN; ++i)
          if (full || (mr + 16 * j < tm && wn + 16 * i + 4 * g < tn)) *(f32x4_loose*)(c + 16 * i) = acc[i][j];
      }
    } else {
      // two tiles' columns change places between lane groups 0 and 1, 2 and 3, so that a lane
      // has eight consecutive ones: of the first tile in even groups, of the second in odd ones
      const int col = wn + 16 * (g & 1) + 8 * (g >> 1);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        uint16_t* c = (uint16_t*)a.c + row_start(j) + col;
#pragma unroll
        for (int i = 0; i < TN; i += 2) {
          const f32x4_t u = acc[i][j], v = acc[i + 1][j];
          const auto x = __builtin_amdgcn_permlane16_swap(GMma<DT>::pack(u[0], u[1]), GMma<DT>::pack(v[0], v[1]), false, false);
          const auto y = __builtin_amdgcn_permlane16_swap(GMma<DT>::pack(u[2], u[3]), GMma<DT>::pack(v[2], v[3]), false, false);
          if (full || (mr + 16 * j < tm && col + 16 * i < tn))
            *(u32x4_loose*)(c + 16 * i) = u32x4_t{x[0], y[0], x[1], y[1]};
        }
        __builtin_amdgcn_sched_barrier(0);  // one row tile's conversions at a time: registers
      }
    }
    credit = full ? NS - 1 : 0;
  }
  ring_wait<0>();  // the last loads, of zeros, end before the LDS goes to another workgroup
}

// The last round's tiles of a grouped_ring_kernel launch of `turns` workgroups an XCD (same arguments):
// sums of their parts in order, by all workgroups of the XCD, turns / rest of them to a tile.  A part is
// bm * bn floats as the waves' registers hold them.
template <int DT>
__global__ __launch_bounds__(256) void grouped_tail_kernel(GroupedArgs a, int wg, int bm, int bn, int wn, int turns) {
  extern __shared__ int e[];
  group_edges(a, e);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int* t = e + a.groups + 1;
  const int tiles = wg ? a.matrices * a.mtiles.d : segment_tiles(a, e, t, bm);
  const int xcd = (int)blockIdx.x % kXcds, i = (int)blockIdx.x / kXcds;
  const RingShare share = ring_share(a, tiles * a.cols.d, xcd, turns);
  if (share.rest == 0) return;
  const int pieces = turns / share.rest, r = i / pieces, piece = i - r * pieces, tile = share.start + share.whole + r;
  if (r >= share.rest) return;
  const Work it = wg ? weight_work(a, e, tile, 0, 1, bm, bn, 1) : rows_work(a, e, t, tiles, tile, 0, 1, bm, bn, 1);
  const int tm = bm / 32, tn = bn / wn / 16, chunks = 2 * wn * tm * tn;  // 2 x wn waves; 64 x 4 values to a chunk
  const f32x4_t* p = (const f32x4_t*)a.parts + (int64_t)(xcd * turns + r * share.parts) * chunks * 64 + lane;
  const int c1 = (piece + 1) * chunks / pieces;
  for (int c = piece * chunks / pieces + wave; c < c1; c += 4) {
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    constexpr int kFlight = 8;
    for (int s = 0; s < share.parts; s += kFlight) {
      f32x4_t u[kFlight];
#pragma unroll
      for (int j = 0; j < kFlight; ++j)
        u[j] = s + j < share.parts ? p[((int64_t)(s + j) * chunks + c) * 64] : f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kFlight; ++j) v += u[j];
    }
    const int wv = c / (tm * tn), x = c - wv * tm * tn, ci = x / tm, cj = x - ci * tm;
    const int row = (wv & 1) * (bm / 2) + 16 * cj + (lane & 15), col = (wv >> 1) * (bn / wn) + 16 * ci + 4 * (lane >> 4);
    if (row >= it.mlim || col >= a.N - it.n0) continue;  // columns come in whole chunks
    const int64_t at = (wg ? (int64_t)it.w * a.cstride : 0) +
                       (int64_t)(it.mapped ? merged_row(a, e, it.w, it.m0 + row) : it.m0 + row) * a.ldc + it.n0 + col;
    if constexpr (DT == ML_F32) *(f32x4_loose*)((float*)a.c + at) = v;
    else *(u32x2_loose*)((uint16_t*)a.c + at) = u32x2_t{GMma<DT>::pack(v[0], v[1]), GMma<DT>::pack(v[2], v[3])};
  }
}

}  // namespace ml
