// Rows on their way to their experts and back: (tokens, k) expert numbers sorted by expert, the tokens' rows at their
// experts' places (what the grouped products take), and the experts' rows summed back with weights.
//
//   assignment a = t k + j of token t has the expert ids[a]; one outside 0 .. experts - 1 is dropped
//   order    the assignments by expert, those of one expert in their order, the dropped ones last
//   slots    the place of each assignment in that order;  offsets[e]  the first place of expert e, offsets[experts]
//            that of the dropped ones
//   there:   rows[slot(t, j)] = x[t], the dropped places zero       dx[t] = sum_j drows[slot(t, j)]
//   back:    out[t] = sum_j w[t, j] rows[slot(t, j)]                drows[slot] = w dout[t],  dw[t, j] = <dout[t], rows[slot]>
//
// Sums leave dropped assignments out; their gradients are zero.
//
// The sort is a counting sort: a place is the expert's first one, and the number of its assignments in the chunks before,
// in the chunk's waves before and in the wave's lanes before (lanes of the same expert find each other by a ballot for each
// bit of its number).  No atomics decide an order, so equal calls give equal bits.  Few assignments
// take one workgroup and one launch, more take two or three: counts by chunk, their sums over many chunks, places.
//
// Everything else is bound by HBM: there reads each row once and writes it k times, back and the gradients
// read or write each assignment's row once.  A token (back's gradient: an assignment) is a wave's or 16 lanes', which
// pass over the row in 16-byte chunks, at any alignment; sums are float32 in the order of j, rounded once.  8,192 tokens x 8 of 64
// experts, 1,024 wide, bf16 (17 and 134 MB): order 12 us, there 29 (5.2 TB/s), back 32, gradient of back 58 (4.9 TB/s), of there 32;
// single elements at odd widths cost more (8,192 x 4 x 1,025 bf16 back 29 / 48 us, its gradient 36 / 69; 513 f32 27 / 29, 33 / 40).
#include <algorithm>

#include "ml_rows.h"

namespace ml {
namespace {

// ---- order ---------------------------------------------------------------------
constexpr int kSortItems = 256;  // assignments of a wave, 64 at a time
constexpr int kSortRounds = kSortItems / 64;
constexpr int kManyWaves = 4;    // waves of a workgroup where there are several
constexpr int kOneWaves = 16;
constexpr int64_t kMaxExperts = 4000;  // as the grouped products' groups
constexpr int64_t kOneExperts = 1023;  // more: several workgroups, whose counts take less LDS each

__device__ __forceinline__ int expert_of(const int64_t* ids, int64_t i, int64_t n, int experts) {
  if (i >= n) return -1;  // no assignment
  const int64_t e = ids[i];
  return (uint64_t)e < (uint64_t)experts ? (int)e : experts;
}

// Sums of v over the lanes before this one.
__device__ __forceinline__ int scan_before(int v, int lane) {
  int s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(s, o, 64);
    if (lane >= o) s += u;
  }
  return s - v;
}

// first[key] = totals of the keys before it, for keys 0 .. n - 1; every thread of W waves calls it.
template <int W>
__device__ __forceinline__ void first_places(int* first, int n, int* wave_sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int carry = 0;
  for (int base = 0; base < n; base += 64 * W) {
    const int i = base + (int)threadIdx.x, v = i < n ? first[i] : 0;
    const int before = scan_before(v, lane);
    if (lane == 63) wave_sum[wave] = before + v;
    __syncthreads();
    int add = carry;
    for (int q = 0; q < W; ++q) {
      if (q < wave) add += wave_sum[q];
      carry += wave_sum[q];
    }
    if (i < n) first[i] = before + add;
    __syncthreads();
  }
}

// chunk counts, counts[chunk][experts + 1]
__global__ __launch_bounds__(64 * kManyWaves) void expert_count_kernel(const int64_t* ids, int64_t n, int experts, int* counts) {
  extern __shared__ int c[];
  for (int i = threadIdx.x; i <= experts; i += 64 * kManyWaves) c[i] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kManyWaves * kSortItems;
  for (int i = threadIdx.x; i < kManyWaves * kSortItems; i += 64 * kManyWaves) {
    const int e = expert_of(ids, base + i, n, experts);
    if (e >= 0) atomicAdd(&c[e], 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i <= experts; i += 64 * kManyWaves) counts[(int64_t)blockIdx.x * (experts + 1) + i] = c[i];
}

// counts[chunk][key] becomes the sum over the chunks before, totals[key] that over all: 64 keys to a workgroup, its
// 16 waves a run of chunks each.
constexpr int kSumWaves = 16;
__global__ __launch_bounds__(64 * kSumWaves) void expert_sum_kernel(int* counts, int chunks, int keys, int* totals) {
  __shared__ int run[kSumWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, key = (int)blockIdx.x * 64 + lane;
  const int each = (chunks + kSumWaves - 1) / kSumWaves, c0 = min(wave * each, chunks), c1 = min(c0 + each, chunks);
  int s = 0;
  if (key < keys)
    for (int c = c0; c < c1; ++c) s += counts[(int64_t)c * keys + key];
  run[wave][lane] = s;
  __syncthreads();
  if (key >= keys) return;
  int before = 0, all = 0;
  for (int q = 0; q < kSumWaves; ++q) {
    if (q < wave) before += run[q][lane];
    all += run[q][lane];
  }
  if (wave == 0) totals[key] = all;
  for (int c = c0; c < c1; ++c) {
    int* p = counts + (int64_t)c * keys + key;
    const int v = *p;
    *p = before;
    before += v;
  }
}

// Of each key, all chunks' counts and those of the chunks before `mine`: a thread for every key and slice of the chunks,
// up to eight loads in flight.
constexpr int kFewKeys = 512, kFewChunks = 256;
template <int W>
__device__ __forceinline__ void chunk_sums(const int* counts, int chunks, int mine, int keys, int* all, int* prior) {
  for (int i = threadIdx.x; i < keys; i += 64 * W) all[i] = prior[i] = 0;
  __syncthreads();
  const int slices = max(1, min(8, 64 * W / keys)), each = (chunks + slices - 1) / slices;
  for (int i = threadIdx.x; i < keys * slices; i += 64 * W) {
    const int slice = i / keys, key = i - slice * keys, c1 = min((slice + 1) * each, chunks);
    int s = 0, before = 0;
    for (int c = slice * each; c < c1; c += 8) {
      int v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < c1 ? counts[(int64_t)(c + j) * keys + key] : 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s += v[j];
        before += c + j < mine ? v[j] : 0;
      }
    }
    atomicAdd(&all[key], s);  // (whole numbers: any order)
    atomicAdd(&prior[key], before);
  }
}

// Places of a chunk's assignments, W waves of kSortItems each.  before: counts over the chunks before, and totals
// (expert_sum_kernel); or totals null: the chunks' counts themselves, of which there are few; both null where one workgroup
// has all assignments.
template <int W>
__global__ __launch_bounds__(64 * W) void expert_place_kernel(const int64_t* ids, int64_t n, int experts, const int* before,
                                                              const int* totals, int64_t* order, int64_t* slots,
                                                              int64_t* offsets) {
  extern __shared__ int lds[];
  __shared__ int wave_sum[W];
  const int keys = experts + 1, stride = (keys + 1) & ~1;
  int* first = lds;                           // first place of each key
  uint16_t* count = (uint16_t*)(lds + keys);  // [wave][key]
  __shared__ int prior[kFewKeys];             // (few chunks) counts over the chunks before
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < W * stride; i += 64 * W) count[i] = 0;
  if (totals) {
    for (int i = threadIdx.x; i < keys; i += 64 * W) first[i] = totals[i];
  } else if (before) {
    chunk_sums<W>(before, (int)gridDim.x, (int)blockIdx.x, keys, first, prior);
  }
  __syncthreads();

  const int64_t base = ((int64_t)blockIdx.x * W + wave) * kSortItems;
  uint16_t* own = count + wave * stride;
  const int bits = 32 - __builtin_clz(keys);  // of the largest key and of the number for none (keys)
  int key[kSortRounds], rank[kSortRounds];
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    key[r] = expert_of(ids, base + r * 64 + lane, n, experts);
    const int e = key[r] < 0 ? keys : key[r];
    uint64_t same = ~(uint64_t)0;
    for (int b = 0; b < bits; ++b) {
      const bool set = e >> b & 1;
      const uint64_t with = __ballot(set);
      same &= set ? with : ~with;
    }
    const int mine = __popcll(same & (((uint64_t)1 << lane) - 1));
    rank[r] = 0;
    if (key[r] >= 0) {
      rank[r] = own[e] + mine;  // (a wave's LDS operations keep their order: read before the last lane's write)
      if (mine + 1 == __popcll(same)) own[e] = (uint16_t)(rank[r] + 1);
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  // counts of the waves before, and (one workgroup) the totals
  for (int i = threadIdx.x; i < keys; i += 64 * W) {
    int s = 0;
    for (int w = 0; w < W; ++w) {
      const int v = count[w * stride + i];
      count[w * stride + i] = (uint16_t)s;
      s += v;
    }
    if (!before) first[i] = s;
  }
  __syncthreads();
  first_places<W>(first, keys, wave_sum);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < keys; i += 64 * W) offsets[i] = first[i];
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const int e = key[r];
    if (e < 0) continue;
    const int64_t i = base + r * 64 + lane;
    const int64_t at = first[e] + (totals ? before[(int64_t)blockIdx.x * keys + e] : before ? prior[e] : 0) + own[e] + rank[r];
    slots[i] = at;
    order[at] = i;
  }
}

// ---- rows ----------------------------------------------------------------------
constexpr int kRowThreads = 256;

// Places below this hold assignments' rows; the ones behind are the dropped ones'.
__device__ __forceinline__ int64_t kept_places(const int64_t* offsets, int64_t experts, int64_t n) {
  const int64_t kept = offsets[experts];
  return kept < 0 ? 0 : kept > n ? n : kept;
}

// The row that a thread's T lanes begin with: the same for the whole wave from 64 lanes on, which the compiler is told, so that
// what belongs to the row (places, weights) comes through scalar loads into scalar registers.
template <int T>
__device__ __forceinline__ int64_t first_row() {
  const int at = (int)threadIdx.x / T;
  return (int64_t)blockIdx.x * (kRowThreads / T) + (T >= 64 ? __builtin_amdgcn_readfirstlane(at) : at);
}

// Rows to their places, T lanes to a token, 16 bytes at once.
template <int T>
__global__ __launch_bounds__(kRowThreads) void to_experts_kernel(const uint8_t* x, int64_t tokens, int64_t k, int64_t bytes,
                                                                 const int64_t* slots, const int64_t* offsets,
                                                                 int64_t experts, uint8_t* rows) {
  typedef uint32_t loose __attribute__((ext_vector_type(4), aligned(1)));
  const int lane = threadIdx.x % T;
  const int64_t kept = kept_places(offsets, experts, tokens * k);
  for (int64_t t = first_row<T>(); t < tokens; t += (int64_t)gridDim.x * (kRowThreads / T)) {
    const int64_t* at = slots + t * k;
    for (int64_t c = (int64_t)lane * 16; c < bytes; c += T * 16) {
      const int64_t n = bytes - c;
      const uint8_t* from = x + t * bytes + c;
      u32x4_t v = {0u, 0u, 0u, 0u};
      if (n >= 16) v = *(const loose*)from;
      for (int64_t j = 0; j < k; ++j) {
        const int64_t p = at[j];
        // place t k + j holds zeros if it is behind the kept ones: each such place once
        for (int zero = 0; zero < 2; ++zero) {
          if (zero ? t * k + j < kept : (uint64_t)p >= (uint64_t)kept) continue;
          uint8_t* to = rows + (zero ? t * k + j : p) * bytes + c;
          if (n >= 16) {
            *(loose*)to = zero ? u32x4_t{0u, 0u, 0u, 0u} : v;
          } else {
            for (int i = 0; i < n; ++i) to[i] = zero ? 0 : from[i];
          }
        }
      }
    }
  }
}

// out[t] = sum_j w[t, j] rows[slot(t, j)] (w null: ones), T lanes to a token.  ONCE: more rows than the caches keep for the
// gradient pass, read past them: what other kernels wrote is not driven out in between (8,192 tokens x 8 x 1,024 bf16, all
// kernels of a training pass 172 -> 155 us, 16,384 x 2 x 2,048 201 -> 198; rows that fit, 20,011 x 257 f32, 57 -> 62).
template <int DT, int T, bool ONCE>
__global__ __launch_bounds__(kRowThreads) void from_experts_kernel(const void* rowsv, const void* w, int wf32, int64_t tokens,
                                                                   int64_t k, int64_t D, const int64_t* slots,
                                                                   const int64_t* offsets, int64_t experts, void* outv) {
  using R = typename Elem<DT>::raw;
  using C = RowChunk<DT>;
  constexpr int V = C::V, kFlight = 8;  // rows whose loads are in flight together
  const R* rows = (const R*)rowsv;
  R* out = (R*)outv;
  const int lane = threadIdx.x % T;
  const int64_t kept = kept_places(offsets, experts, tokens * k);
  for (int64_t t = first_row<T>(); t < tokens; t += (int64_t)gridDim.x * (kRowThreads / T)) {
    const R* from[kFlight];
    float wj[kFlight];
    auto places = [&](int64_t j0) {
#pragma unroll
      for (int q = 0; q < kFlight; ++q) {
        const int64_t a = t * k + j0 + q, p = j0 + q < k ? slots[a] : -1;
        const bool in = (uint64_t)p < (uint64_t)kept;
        wj[q] = !in ? 0.f : w ? param_at<DT>(w, wf32, a) : 1.f;
        from[q] = in ? rows + p * D : nullptr;
      }
    };
    places(0);
    for (int64_t c = (int64_t)lane * V; c < D; c += T * V) {
      float acc[V];
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = 0.f;
      for (int64_t j0 = 0; j0 < k; j0 += kFlight) {
        if (k > kFlight) places(j0);
        C v[kFlight];
#pragma unroll
        for (int q = 0; q < kFlight; ++q) {
          v[q] = C{};
          if (from[q]) v[q].template load<false, ONCE>(from[q] + c, D - c);
        }
#pragma unroll
        for (int q = 0; q < kFlight; ++q)
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] = fmaf(wj[q], to_f32<DT>(v[q].e[i]), acc[i]);
      }
      C o;
#pragma unroll
      for (int i = 0; i < V; ++i) o.e[i] = from_f32<DT>(acc[i]);
      o.store(out + t * D + c, D - c);
    }
  }
}

// drows[slot] = w dout[t] and dw = <dout[t], rows[slot]> of an assignment, T lanes to it; either may be null.
template <int DT, int T, bool ONCE>
__global__ __launch_bounds__(kRowThreads) void from_experts_backward_kernel(const void* gv, const void* rowsv, const void* w,
                                                                            int wf32, int64_t n, int64_t k, int64_t D,
                                                                            const int64_t* slots, const int64_t* offsets,
                                                                            int64_t experts, void* drowsv, void* dw) {
  using R = typename Elem<DT>::raw;
  using C = RowChunk<DT>;
  constexpr int V = C::V;
  __shared__ float red[2][16];
  const R *dout = (const R*)gv, *rows = (const R*)rowsv;
  R* drows = (R*)drowsv;
  const int lane = threadIdx.x % T;
  const int64_t kept = kept_places(offsets, experts, n);
  int flip = 0;
  // (T = 256: the workgroup makes the rounds together, for the barriers of the sum)
  for (int64_t a = first_row<T>(); a < n; a += (int64_t)gridDim.x * (kRowThreads / T), flip ^= 1) {
    const int64_t t = a / k, p = slots[a];
    const bool in = (uint64_t)p < (uint64_t)kept;
    const float wa = !in ? 0.f : w ? param_at<DT>(w, wf32, a) : 1.f;
    float s[1] = {0.f};
    for (int64_t c = (int64_t)lane * V; c < D; c += T * V) {
      if (in) {
        C g, v;
        g.load(dout + t * D + c, D - c);
        if (dw) {
          v.template load<false, ONCE>(rows + p * D + c, D - c);
#pragma unroll
          for (int i = 0; i < V; ++i) s[0] = fmaf(to_f32<DT>(g.e[i]), to_f32<DT>(v.e[i]), s[0]);
        }
        if (drows) {
          C o;
#pragma unroll
          for (int i = 0; i < V; ++i) o.e[i] = from_f32<DT>(wa * to_f32<DT>(g.e[i]));
          o.store(drows + p * D + c, D - c);
        }
      }
      if (drows && a >= kept) C{}.store(drows + a * D + c, D - c);  // each place behind them once
    }
    if (dw) {
      row_sum<T>(s, red[flip]);
      if (lane == 0) param_set<DT>(dw, wf32, a, s[0]);
    }
  }
}

// Lanes to a row of so many 16-byte chunks: 16 where they reach over it, 256 where rows are few and long (8,192 tokens of 128
// chunks, 20,011 of 65, there / back, us: 64 lanes 28 / 45, 13 / 15, 128 lanes 28 / 46, 16 / 20).
template <class F>
int by_lanes(int64_t chunks, int64_t rows, F&& f) {
  if (chunks <= 16) return f(std::integral_constant<int, 16>());
  if (chunks > 64 && rows <= 2048) return f(std::integral_constant<int, 256>());
  return f(std::integral_constant<int, 64>());
}
constexpr int64_t kOnceBytes = (int64_t)64 << 20;
template <int DT>
bool read_once(int64_t n, int64_t D) { return n * D * (int64_t)sizeof(typename Elem<DT>::raw) >= kOnceBytes; }
dim3 row_grid(int64_t rows, int T) { return dim3((unsigned)std::min<int64_t>(ceil_div(rows * T, kRowThreads), 1 << 20)); }

int experts_check(const char* who, int64_t tokens, int64_t k, int64_t experts) {
  const std::string name(who);
  if (tokens < 0 || k < 0) return fail(ML_EINVAL, name + ": tokens and k must not be negative");
  if (experts < 1) return fail(ML_EINVAL, name + ": at least one expert");
  if (experts > kMaxExperts)
    return fail(ML_EUNSUPPORTED, name + ": at most " + std::to_string(kMaxExperts) + " experts are supported");
  if (k > 0 && tokens > (((int64_t)1 << 31) - 4096) / k)
    return fail(ML_EUNSUPPORTED, name + ": at most 2^31 - 4096 assignments are supported");
  return ML_OK;
}

bool one_workgroup(int64_t n, int64_t experts) { return n <= kOneWaves * kSortItems && experts <= kOneExperts; }
// Workgroups of a sort by several, each with a row of counts in the workspace: one at least, which writes the offsets where
// there is no assignment.
int64_t sort_chunks(int64_t n) { return std::max<int64_t>(1, ceil_div(n, kManyWaves * kSortItems)); }

template <int W>
size_t place_lds(int64_t experts) {
  const size_t keys = (size_t)experts + 1;
  return keys * sizeof(int) + W * ((keys + 1) & ~(size_t)1) * sizeof(uint16_t);
}

int rows_check(const char* who, int dtype, int wdtype, int64_t tokens, int64_t k, int64_t width, int64_t experts) {
  const int rc = experts_check(who, tokens, k, experts);
  if (rc) return rc;
  const std::string name(who);
  if (dtype != ML_F32 && dtype != ML_BF16 && dtype != ML_F16) return fail(ML_EINVAL, name + ": unsupported dtype");
  if (wdtype != dtype && wdtype != ML_F32)
    return fail(ML_EINVAL, name + ": the weights must have the rows' dtype or be float32");
  if (width < 0) return fail(ML_EINVAL, name + ": width must not be negative");
  if (width > 0 && tokens * std::max<int64_t>(k, 1) > INT64_MAX / 8 / width)
    return fail(ML_EUNSUPPORTED, name + ": too many elements");
  return ML_OK;
}

template <int DT>
int from_experts(const void* rows, const void* w, int wf32, int64_t tokens, int64_t k, int64_t D, const int64_t* slots,
                 const int64_t* offsets, int64_t experts, void* out, hipStream_t st) {
  return by_lanes(ceil_div(D, RowChunk<DT>::V), tokens, [&](auto tc) {
    constexpr int T = decltype(tc)::value;
    const dim3 grid = row_grid(tokens, T), blk(kRowThreads);
    if (read_once<DT>(tokens * k, D))
      hipLaunchKernelGGL((from_experts_kernel<DT, T, true>), grid, blk, 0, st, rows, w, wf32, tokens, k, D, slots, offsets,
                         experts, out);
    else
      hipLaunchKernelGGL((from_experts_kernel<DT, T, false>), grid, blk, 0, st, rows, w, wf32, tokens, k, D, slots, offsets,
                         experts, out);
    return check_launch("from_experts");
  });
}

template <int DT>
int from_experts_backward(const void* g, const void* rows, const void* w, int wf32, int64_t n, int64_t k, int64_t D,
                          const int64_t* slots, const int64_t* offsets, int64_t experts, void* drows, void* dw,
                          hipStream_t st) {
  return by_lanes(ceil_div(D, RowChunk<DT>::V), n, [&](auto tc) {
    constexpr int T = decltype(tc)::value;
    const dim3 grid = row_grid(n, T), blk(kRowThreads);
    if (read_once<DT>(n, D))
      hipLaunchKernelGGL((from_experts_backward_kernel<DT, T, true>), grid, blk, 0, st, g, rows, w, wf32, n, k, D, slots,
                         offsets, experts, drows, dw);
    else
      hipLaunchKernelGGL((from_experts_backward_kernel<DT, T, false>), grid, blk, 0, st, g, rows, w, wf32, n, k, D, slots,
                         offsets, experts, drows, dw);
    return check_launch("from_experts_backward");
  });
}

}  // namespace
}  // namespace ml

using namespace ml;

extern "C" size_t ml_sort_by_expert_workspace_size(int64_t tokens, int64_t k, int64_t experts) {
  if (experts_check("sort_by_expert", tokens, k, experts)) return 0;
  const int64_t n = tokens * k;
  if (one_workgroup(n, experts)) return 256;
  return align256((size_t)(sort_chunks(n) + 1) * (size_t)(experts + 1) * sizeof(int));
}

extern "C" int ml_sort_by_expert(const int64_t* ids, int64_t tokens, int64_t k, int64_t experts, int64_t* order,
                                 int64_t* slots, int64_t* offsets, void* workspace, size_t workspace_bytes,
                                 ml_stream_t stream) {
  const int rc = experts_check("sort_by_expert", tokens, k, experts);
  if (rc) return rc;
  const int64_t n = tokens * k;
  if (!offsets || (n > 0 && (!ids || !order || !slots))) return fail(ML_EINVAL, "sort_by_expert: null pointer");
  hipStream_t st = (hipStream_t)stream;
  ProfScope ps("sort_by_expert", st);
  if (one_workgroup(n, experts)) {
    hipLaunchKernelGGL(expert_place_kernel<kOneWaves>, dim3(1), dim3(64 * kOneWaves), place_lds<kOneWaves>(experts), st, ids, n,
                       (int)experts, nullptr, nullptr, order, slots, offsets);
    return check_launch("sort_by_expert");
  }
  if (!workspace || workspace_bytes < ml_sort_by_expert_workspace_size(tokens, k, experts))
    return fail(ML_EWORKSPACE, "sort_by_expert: workspace too small");
  const int keys = (int)experts + 1;
  const int64_t chunks = sort_chunks(n);
  int* totals = (int*)workspace;
  int* counts = totals + keys;
  hipLaunchKernelGGL(expert_count_kernel, dim3((unsigned)chunks), dim3(64 * kManyWaves), (size_t)keys * sizeof(int), st, ids, n,
                     (int)experts, counts);
  const bool few = chunks <= kFewChunks && keys <= kFewKeys;
  if (!few)
    hipLaunchKernelGGL(expert_sum_kernel, dim3((unsigned)ceil_div(keys, 64)), dim3(64 * kSumWaves), 0, st, counts, (int)chunks,
                       keys, totals);
  hipLaunchKernelGGL(expert_place_kernel<kManyWaves>, dim3((unsigned)chunks), dim3(64 * kManyWaves),
                     place_lds<kManyWaves>(experts), st, ids, n, (int)experts, counts, few ? nullptr : totals, order, slots, offsets);
  return check_launch("sort_by_expert");
}

extern "C" int ml_to_experts(const void* x, int64_t tokens, int64_t k, int64_t row_bytes, const int64_t* slots,
                             const int64_t* offsets, int64_t experts, void* rows, ml_stream_t stream) {
  const int rc = experts_check("to_experts", tokens, k, experts);
  if (rc) return rc;
  if (row_bytes < 0) return fail(ML_EINVAL, "to_experts: row_bytes must not be negative");
  if (row_bytes > 0 && tokens * std::max<int64_t>(k, 1) > INT64_MAX / 2 / row_bytes)
    return fail(ML_EUNSUPPORTED, "to_experts: too many elements");
  if (tokens * k == 0 || row_bytes == 0) return ML_OK;
  if (!x || !slots || !offsets || !rows) return fail(ML_EINVAL, "to_experts: null pointer");
  hipStream_t st = (hipStream_t)stream;
  ProfScope ps("to_experts", st);
  return by_lanes(ceil_div(row_bytes, 16), tokens, [&](auto tc) {
    constexpr int T = decltype(tc)::value;
    hipLaunchKernelGGL(to_experts_kernel<T>, row_grid(tokens, T), dim3(kRowThreads), 0, st, (const uint8_t*)x, tokens, k,
                       row_bytes, slots, offsets, experts, (uint8_t*)rows);
    return check_launch("to_experts");
  });
}

extern "C" int ml_from_experts_forward(int dtype, int weight_dtype, const void* rows, const void* weights, int64_t tokens,
                                       int64_t k, int64_t width, const int64_t* slots, const int64_t* offsets,
                                       int64_t experts, void* out, ml_stream_t stream) {
  const int rc = rows_check("from_experts", dtype, weight_dtype, tokens, k, width, experts);
  if (rc) return rc;
  if (tokens == 0 || width == 0) return ML_OK;
  if (!out || !offsets || (k > 0 && (!rows || !slots))) return fail(ML_EINVAL, "from_experts: null pointer");
  hipStream_t st = (hipStream_t)stream;
  ProfScope ps("from_experts", st);
  const int wf32 = weight_dtype == ML_F32;
  switch (dtype) {
    case ML_F32: return from_experts<ML_F32>(rows, weights, wf32, tokens, k, width, slots, offsets, experts, out, st);
    case ML_BF16: return from_experts<ML_BF16>(rows, weights, wf32, tokens, k, width, slots, offsets, experts, out, st);
    default: return from_experts<ML_F16>(rows, weights, wf32, tokens, k, width, slots, offsets, experts, out, st);
  }
}

extern "C" int ml_from_experts_backward(int dtype, int weight_dtype, const void* grad_out, const void* rows,
                                        const void* weights, int64_t tokens, int64_t k, int64_t width, const int64_t* slots,
                                        const int64_t* offsets, int64_t experts, void* grad_rows, void* grad_weights,
                                        ml_stream_t stream) {
  const int rc = rows_check("from_experts", dtype, weight_dtype, tokens, k, width, experts);
  if (rc) return rc;
  const int64_t n = tokens * k;
  if (n == 0 || (!grad_rows && !grad_weights) || (width == 0 && !grad_weights)) return ML_OK;
  if (!slots || !offsets || (width > 0 && (!grad_out || (grad_weights && !rows))))
    return fail(ML_EINVAL, "from_experts: null pointer");
  hipStream_t st = (hipStream_t)stream;
  ProfScope ps("from_experts_backward", st);
  const int wf32 = weight_dtype == ML_F32;
  switch (dtype) {
    case ML_F32:
      return from_experts_backward<ML_F32>(grad_out, rows, weights, wf32, n, k, width, slots, offsets, experts, grad_rows,
                                           grad_weights, st);
    case ML_BF16:
      return from_experts_backward<ML_BF16>(grad_out, rows, weights, wf32, n, k, width, slots, offsets, experts, grad_rows,
                                            grad_weights, st);
    default:
      return from_experts_backward<ML_F16>(grad_out, rows, weights, wf32, n, k, width, slots, offsets, experts, grad_rows,
                                           grad_weights, st);
  }
}
