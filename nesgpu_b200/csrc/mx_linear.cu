// Product of microscaled operands: y[t, n] = sum_k x[t, k] w[n, k] + bias[n].
//
// Both operands are rows of blocks (microscale.cuh).  Raw activations are quantised into scratch first.
#include <type_traits>
#include "microscale.cuh"

namespace nes {
namespace mx {

struct Product {
  const uint8_t *x, *x_scales, *w, *w_scales;
  const float* bias;
  void* y;
  int64_t M, N, K;
};

constexpr int TILE = 64;

// 64 x 64 outputs per block, one block of 32 elements of K per trip, operands decoded into shared memory.
template <typename T, int XF, int WF>
__global__ void __launch_bounds__(256) product_kernel(const Product p) {
  __shared__ float xs[BLOCK][TILE + 1], ws[BLOCK][TILE + 1];
  const int64_t m0 = int64_t(blockIdx.y) * TILE, n0 = int64_t(blockIdx.x) * TILE;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  const int64_t blocks = (p.K + BLOCK - 1) / BLOCK;
  const int r = threadIdx.x >> 2, u = threadIdx.x & 3;       // 64 rows, 4 units of a block each
  for (int64_t b = 0; b < blocks; ++b) {
    float v[UNIT];
    const int64_t m = m0 + r, n = n0 + r;
    float s = 0.f;
    if (m < p.M) {
      unit_elements<XF>(p.x + m * code_pitch(p.K, XF), b * 4 + u, v);
      s = scale_value(p.x_scales[m * scale_pitch(p.K) + b]);
    }
#pragma unroll
    for (int i = 0; i < UNIT; ++i) xs[u * UNIT + i][r] = m < p.M ? v[i] * s : 0.f;
    if (n < p.N) {
      unit_elements<WF>(p.w + n * code_pitch(p.K, WF), b * 4 + u, v);
      s = scale_value(p.w_scales[n * scale_pitch(p.K) + b]);
    }
#pragma unroll
    for (int i = 0; i < UNIT; ++i) ws[u * UNIT + i][r] = n < p.N ? v[i] * s : 0.f;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < BLOCK; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[k][ty * 4 + i], ws[k][tx + j * 16], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx + j * 16;
      if (m < p.M && n < p.N) static_cast<T*>(p.y)[m * p.N + n] = from_float<T>(acc[i][j] + (p.bias ? p.bias[n] : 0.f));
    }
}

template <typename T>
static void launch_product(const Product& p, int xf, int wf, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div<int64_t>(p.N, TILE), (unsigned)ceil_div<int64_t>(p.M, TILE));
  if (xf == NES_MXFP4 && wf == NES_MXFP4) product_kernel<T, NES_MXFP4, NES_MXFP4><<<grid, 256, 0, st>>>(p);
  else if (xf == NES_MXFP8 && wf == NES_MXFP4) product_kernel<T, NES_MXFP8, NES_MXFP4><<<grid, 256, 0, st>>>(p);
  else product_kernel<T, NES_MXFP8, NES_MXFP8><<<grid, 256, 0, st>>>(p);
}

static int64_t align256(int64_t v) { return (v + 255) & ~int64_t(255); }

}  // namespace mx
}  // namespace nes

using namespace nes;
using namespace nes::mx;

extern "C" int64_t nes_mx_linear_fwd_scratch_bytes(int64_t M, int64_t N, int64_t K, int x_format) {
  if (M <= 0 || N <= 0 || K <= 0 || !known_format(x_format)) return 0;
  return align256(M * code_pitch(K, x_format)) + align256(M * scale_pitch(K));
}

extern "C" int nes_mx_linear_fwd(const void* x, const uint8_t* x_scales, int x_dtype, int x_format, const void* w_codes,
                                 const uint8_t* w_scales, int w_format, const float* bias, void* y, int y_dtype, int64_t M, int64_t N,
                                 int64_t K, void* scratch, int64_t scratch_bytes, nes_stream_t stream) {
  NES_REQUIRE(M >= 0 && N >= 0 && K >= 1, NES_ERR_BAD_ARG, "mx_linear_fwd: bad extent");
  NES_REQUIRE(known_format(x_format) && known_format(w_format) && !(x_format == NES_MXFP4 && w_format == NES_MXFP8) &&
                  (x_scales || known_dtype(x_dtype)) && known_dtype(y_dtype),
              NES_ERR_UNSUPPORTED, "mx_linear_fwd: unknown dtype or combination of formats");
  if (M == 0 || N == 0) return NES_OK;
  NES_REQUIRE(x && w_codes && w_scales && y, NES_ERR_BAD_ARG, "mx_linear_fwd: null pointer");
  NES_REQUIRE(aligned16(w_codes) && (!x_scales || aligned16(x)), NES_ERR_BAD_ARG, "mx_linear_fwd: codes must be 16-byte aligned");
  NES_REQUIRE(M <= INT32_MAX && N <= INT32_MAX && K <= INT32_MAX && ceil_div<int64_t>(M, TILE) <= 65535, NES_ERR_UNSUPPORTED, "mx_linear_fwd: too large");
  cudaStream_t st = as_stream(stream);
  Product p;
  p.x = static_cast<const uint8_t*>(x); p.x_scales = x_scales;
  p.w = static_cast<const uint8_t*>(w_codes); p.w_scales = w_scales;
  p.bias = bias; p.y = y; p.M = M; p.N = N; p.K = K;
  if (!x_scales) {
    const int64_t need = nes_mx_linear_fwd_scratch_bytes(M, N, K, x_format);
    NES_REQUIRE(scratch && scratch_bytes >= need && aligned16(scratch), NES_ERR_SCRATCH,
                "mx_linear_fwd: scratch needs %lld bytes, 16-byte aligned", (long long)need);
    uint8_t* codes = static_cast<uint8_t*>(scratch);
    uint8_t* scales = codes + align256(M * code_pitch(K, x_format));
    const int rc = nes_mx_quantize(x, x_dtype, codes, scales, M, K, x_format, stream);
    if (rc != NES_OK) return rc;
    p.x = codes; p.x_scales = scales;
  }
  if (y_dtype == NES_F32) launch_product<float>(p, x_format, w_format, st);
  else if (y_dtype == NES_BF16) launch_product<__nv_bfloat16>(p, x_format, w_format, st);
  else launch_product<__half>(p, x_format, w_format, st);
  return check_launch("mx_linear_fwd");
}
