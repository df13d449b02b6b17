// Rows to microscaled values (ml_mx.h): bound by HBM, each value read once, its code written once and a byte for every
// 32 of them.  Rows are whole blocks, so the rows are one run of blocks; a lane takes 8 values (two loads of 16 bytes in
// float32), four lanes a block.  16,384 x 2,048 bf16 from memory to e4m3 (102 MB) 20 us, to e2m1 (85 MB) 17, 5.1 TB/s; 16 and 13.5
// where the 256 MB cache still holds the rows.
#include <algorithm>

#include "ml_mx.h"

namespace ml {
namespace {

constexpr int kQuantThreads = 256;

template <int DT>
__global__ __launch_bounds__(kQuantThreads) void mx_quantize_kernel(const void* xv, int64_t n, int format, uint8_t* codes,
                                                                    uint8_t* scales) {
  using R = typename Elem<DT>::raw;
  constexpr int V = DT == ML_F32 ? 4 : 8;
  for (int64_t at = ((int64_t)blockIdx.x * kQuantThreads + threadIdx.x) * 8; at < n;
       at += (int64_t)gridDim.x * kQuantThreads * 8) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8 / V; ++i) {
      const Vec<DT, V> v = *(const Vec<DT, V>*)((const R*)xv + at + i * V);
#pragma unroll
      for (int j = 0; j < V; ++j) y[i * V + j] = to_f32<DT>(v.e[j]);
    }
    // (the four lanes of a block leave the loop together)
    const uint32_t code = mx_scale(mx_lane_max<4>(mx_max(y)), format);
    mx_store(y, code, format, at, codes);
    if (at % kMxBlock == 0) scales[at / kMxBlock] = (uint8_t)code;
  }
}

}  // namespace
}  // namespace ml

using namespace ml;

extern "C" int ml_mx_quantize(int dtype, const void* x, int64_t rows, int64_t width, int format, void* codes,
                              uint8_t* scales, ml_stream_t stream) {
  if (dtype != ML_F32 && dtype != ML_BF16 && dtype != ML_F16) return fail(ML_EINVAL, "mx_quantize: unsupported dtype");
  if (!mx_format(format)) return fail(ML_EINVAL, "mx_quantize: unknown format");
  if (rows < 0 || width < 0) return fail(ML_EINVAL, "mx_quantize: rows and width must not be negative");
  if (width % kMxBlock) return fail(ML_EINVAL, "mx_quantize: width must be a multiple of 32");
  if (rows > 0 && width > INT64_MAX / 8 / rows) return fail(ML_EUNSUPPORTED, "mx_quantize: too many elements");
  const int64_t n = rows * width;
  if (n == 0) return ML_OK;
  if (!x || !codes || !scales) return fail(ML_EINVAL, "mx_quantize: null pointer");
  if (!aligned16(x) || !aligned16(codes)) return fail(ML_EINVAL, "mx_quantize: x and codes must be 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  ProfScope ps("mx_quantize", st);
  const dim3 grid((unsigned)std::min<int64_t>(ceil_div(n, 8 * kQuantThreads), 8192)), blk(kQuantThreads);
  uint8_t* c = (uint8_t*)codes;
  switch (dtype) {
    case ML_F32: hipLaunchKernelGGL(mx_quantize_kernel<ML_F32>, grid, blk, 0, st, x, n, format, c, scales); break;
    case ML_BF16: hipLaunchKernelGGL(mx_quantize_kernel<ML_BF16>, grid, blk, 0, st, x, n, format, c, scales); break;
    default: hipLaunchKernelGGL(mx_quantize_kernel<ML_F16>, grid, blk, 0, st, x, n, format, c, scales); break;
  }
  return check_launch("mx_quantize");
}
