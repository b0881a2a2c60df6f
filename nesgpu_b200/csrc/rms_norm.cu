// Root-mean-square norm with the residual's addition and a plain or microscaled output.
//
//   h = x + residual                                   (fp32; stored in x's type when there is a residual)
//   y = h * rsqrt(mean(h^2) + eps) * (gain + s(r) * noise[d])     row = r * members + d
//
// One pass: a row stays in registers between the sum of squares and the scaling, so x and the residual are read once
// and h and y written once.  A group of THREADS threads owns a row (a warp for short rows, a block for longer ones)
// and holds UNITS units of eight columns per thread; rows longer than that take the looping kernel, which reads x and
// the residual a second time.
#include <type_traits>
#include "microscale.cuh"

namespace nes {
namespace mx {

struct NormArgs {
  const void* x;
  const void* residual;
  void* h;
  const float* gain;
  const float* noise;
  void* y;
  uint8_t* scales;
  int64_t rows, cols, members;
  int antithetic;
  float eps;
  double inv_cols;
  bool vec, vec_gain;
};

// 1 / sqrt(v) as hi + lo: one Newton step on the hardware's approximation.  A reciprocal root that is zero or
// infinite keeps lo = 0.
__device__ __forceinline__ float2 rsqrt_pair(double v) {
  const float r = rsqrtf(float(v));
  if (!(r > 0.f) || r > 3.0e38f) return make_float2(r, 0.f);
  return make_float2(r, 0.5f * r * float(1.0 - v * (double(r) * double(r))));
}

// h * (r.x + r.y) * g, the products' rounding errors carried along.  SHARP leaves the fp32 result rounded to odd (cut
// off, lowest bit set), so that a rounding to fewer bits afterwards decides as it would on the unrounded value; a
// value exactly on a border does not occur except for a zero.  Otherwise the result is rounded to nearest.
template <bool SHARP>
__device__ __forceinline__ float scaled(float h, float2 r, float g) {
  const float t = h * r.x, te = fmaf(h, r.y, fmaf(h, r.x, -t));
  const float p = t * g, c = fmaf(te, g, fmaf(t, g, -p));
  if (SHARP) return __uint_as_float(__float_as_uint(__fadd_rz(p, c)) | 1u);
  return fabsf(p) < 3.0e38f && fabsf(t) < 3.0e38f ? p + c : p;       // infinities have no error terms
}

__device__ __forceinline__ void load_gain(const NormArgs& a, int64_t row, int64_t c, float (&g)[UNIT]) {
  if (a.gain) {
    load_unit(a.gain, c, a.cols, a.vec_gain, g);
  } else {
#pragma unroll
    for (int i = 0; i < UNIT; ++i) g[i] = 1.f;
  }
  if (a.noise) {
    const int64_t d = row % a.members;
    const float s = anti_sign(row / a.members, a.rows / a.members, a.antithetic);
    float n[UNIT];
    load_unit(a.noise + d * a.cols, c, a.cols, a.vec_gain, n);
#pragma unroll
    for (int i = 0; i < UNIT; ++i) g[i] = fmaf(s, n[i], g[i]);
  }
}

template <typename T>
__device__ __forceinline__ void load_h(const NormArgs& a, int64_t row, int64_t c, float (&v)[UNIT]) {
  load_unit(static_cast<const T*>(a.x) + row * a.cols, c, a.cols, a.vec, v);
  if (a.residual) {
    float q[UNIT];
    load_unit(static_cast<const T*>(a.residual) + row * a.cols, c, a.cols, a.vec, q);
#pragma unroll
    for (int i = 0; i < UNIT; ++i) v[i] += q[i];
  }
}

// y of one unit; every lane of the warp calls it for a quantised output
template <typename T, int OUT>
__device__ __forceinline__ void emit(const NormArgs& a, int64_t row, int64_t unit, int64_t units, const float (&h)[UNIT], float2 r) {
  float y[UNIT];
  const bool on = unit < units;
  if (on) {
    float g[UNIT];
    load_gain(a, row, unit * UNIT, g);
#pragma unroll
    for (int i = 0; i < UNIT; ++i) y[i] = scaled<OUT != 0>(h[i], r, g[i]);
  } else {
#pragma unroll
    for (int i = 0; i < UNIT; ++i) y[i] = 0.f;
  }
  if (OUT == 0) {
    if (on) store_unit(static_cast<T*>(a.y) + row * a.cols, unit * UNIT, a.cols, a.vec, y);
  } else {
    if (on && (unit + 1) * UNIT > a.cols) {      // pad columns are zero whatever the row's scale (0 * inf is not)
#pragma unroll
      for (int i = 0; i < UNIT; ++i) if (unit * UNIT + i >= a.cols) y[i] = 0.f;
    }
    quantize_unit<OUT == 0 ? NES_MXFP8 : OUT>(y, static_cast<uint8_t*>(a.y) + row * code_pitch(a.cols, OUT),
                                              a.scales + row * scale_pitch(a.cols), unit, on);
  }
}

// Sum over the THREADS threads that share a row (all of a block unless THREADS == 32), the same in every thread.  The
// threads' partial sums are joined in 64 bits: the last few additions carry the whole row's rounding.
template <int THREADS>
__device__ __forceinline__ double row_sum(float mine) {
  double s = mine;
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (THREADS > 32) {
    __shared__ double part[THREADS / 32];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    s = part[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) s += part[i];
  }
  return s;
}

template <typename T, int OUT, int THREADS, int UNITS>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS) rms_norm_kernel(const NormArgs a) {
  constexpr int ROWS = THREADS == 32 ? 4 : 1;
  const int64_t row = int64_t(blockIdx.x) * ROWS + (ROWS > 1 ? threadIdx.x / THREADS : 0);
  if (row >= a.rows) return;
  const int t = threadIdx.x % THREADS;
  const int64_t units = OUT == 0 ? (a.cols + UNIT - 1) / UNIT : padded(a.cols) / UNIT;
  float v[UNITS][UNIT];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int64_t c = int64_t(t + u * THREADS) * UNIT;
    if (c < a.cols) {
      load_h<T>(a, row, c, v[u]);
    } else {
#pragma unroll
      for (int i = 0; i < UNIT; ++i) v[u][i] = 0.f;
    }
  }
  float s = 0.f;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < UNIT; ++i) q = fmaf(v[u][i], v[u][i], q);
    s += q;
    const int64_t c = int64_t(t + u * THREADS) * UNIT;
    if (a.h && c < a.cols) store_unit(static_cast<T*>(a.h) + row * a.cols, c, a.cols, a.vec, v[u]);
  }
  const float2 r = rsqrt_pair(row_sum<THREADS>(s) * a.inv_cols + double(a.eps));
#pragma unroll
  for (int u = 0; u < UNITS; ++u) emit<T, OUT>(a, row, t + u * THREADS, units, v[u], r);
}

// Rows of any length: the sum of squares in one loop over the row, the outputs in a second one.
template <typename T, int OUT, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_norm_long_kernel(const NormArgs a) {
  const int64_t row = blockIdx.x;
  const int64_t units = OUT == 0 ? (a.cols + UNIT - 1) / UNIT : padded(a.cols) / UNIT;
  float s = 0.f;
  for (int64_t c = int64_t(threadIdx.x) * UNIT; c < a.cols; c += THREADS * UNIT) {
    float v[UNIT];
    load_h<T>(a, row, c, v);
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < UNIT; ++i) q = fmaf(v[i], v[i], q);
    s += q;
    if (a.h) store_unit(static_cast<T*>(a.h) + row * a.cols, c, a.cols, a.vec, v);
  }
  const float2 r = rsqrt_pair(row_sum<THREADS>(s) * a.inv_cols + double(a.eps));
  for (int64_t u0 = 0; u0 < units; u0 += THREADS) {
    const int64_t unit = u0 + threadIdx.x;
    float v[UNIT];
    if (unit * UNIT < a.cols) {
      load_h<T>(a, row, unit * UNIT, v);
    } else {
#pragma unroll
      for (int i = 0; i < UNIT; ++i) v[i] = 0.f;
    }
    emit<T, OUT>(a, row, unit, units, v, r);
  }
}

template <typename T, int OUT>
static void launch_norm(const NormArgs& a, cudaStream_t st) {
  const unsigned rows = unsigned(a.rows);
  const int64_t units = padded(a.cols) / UNIT;
  if (units <= 32) rms_norm_kernel<T, OUT, 32, 1><<<(rows + 3) / 4, 128, 0, st>>>(a);
  else if (units <= 64) rms_norm_kernel<T, OUT, 32, 2><<<(rows + 3) / 4, 128, 0, st>>>(a);
  else if (units <= 128) rms_norm_kernel<T, OUT, 32, 4><<<(rows + 3) / 4, 128, 0, st>>>(a);
  else if (units <= 256) rms_norm_kernel<T, OUT, 128, 2><<<rows, 128, 0, st>>>(a);
  else if (units <= 512) rms_norm_kernel<T, OUT, 128, 4><<<rows, 128, 0, st>>>(a);
  else if (units <= 1024) rms_norm_kernel<T, OUT, 256, 4><<<rows, 256, 0, st>>>(a);
  else if (units <= 2048) rms_norm_kernel<T, OUT, 512, 4><<<rows, 512, 0, st>>>(a);
  else rms_norm_long_kernel<T, OUT, 512><<<rows, 512, 0, st>>>(a);
}

template <typename T>
static void launch_norm_out(const NormArgs& a, int format, cudaStream_t st) {
  if (format == 0) launch_norm<T, 0>(a, st);
  else if (format == NES_MXFP4) launch_norm<T, NES_MXFP4>(a, st);
  else launch_norm<T, NES_MXFP8>(a, st);
}

}  // namespace mx
}  // namespace nes

using namespace nes;
using namespace nes::mx;

extern "C" int nes_rms_norm_fwd(const void* x, const void* residual, void* residual_out, const float* gain, const float* noise,
                                void* y, uint8_t* y_scales, int64_t rows, int64_t cols, int64_t members, int antithetic,
                                int dtype, int format, float eps, nes_stream_t stream) {
  NES_REQUIRE(rows >= 0 && cols >= 0 && members >= 0, NES_ERR_BAD_ARG, "rms_norm_fwd: negative extent");
  NES_REQUIRE(known_dtype(dtype) && (format == 0 || known_format(format)), NES_ERR_UNSUPPORTED, "rms_norm_fwd: unknown dtype or format");
  if (rows == 0 || cols == 0) return NES_OK;
  NES_REQUIRE(x && y && (format == 0 || y_scales) && (!noise || members > 0) && (residual != nullptr) == (residual_out != nullptr),
              NES_ERR_BAD_ARG, "rms_norm_fwd: null pointer");
  NES_REQUIRE(!noise || rows % members == 0, NES_ERR_BAD_ARG, "rms_norm_fwd: rows must be a multiple of members");
  NES_REQUIRE(rows <= INT32_MAX, NES_ERR_UNSUPPORTED, "rms_norm_fwd: too many rows");
  NES_REQUIRE(format == 0 || aligned16(y), NES_ERR_BAD_ARG, "rms_norm_fwd: codes must be 16-byte aligned");
  const bool vec_rows = (cols * dtype_bytes(dtype)) % 16 == 0;
  NormArgs a;
  a.x = x; a.residual = residual; a.h = residual_out; a.gain = gain; a.noise = noise; a.y = y; a.scales = y_scales;
  a.rows = rows; a.cols = cols; a.members = members > 0 ? members : 1; a.antithetic = antithetic;
  a.eps = eps; a.inv_cols = 1.0 / double(cols);
  a.vec = vec_rows && aligned16(x) && (!residual || (aligned16(residual) && aligned16(residual_out))) && (format != 0 || aligned16(y));
  a.vec_gain = cols % 4 == 0 && (!gain || aligned16(gain)) && (!noise || aligned16(noise));
  cudaStream_t st = as_stream(stream);
  if (dtype == NES_F32) launch_norm_out<float>(a, format, st);
  else if (dtype == NES_BF16) launch_norm_out<__nv_bfloat16>(a, format, st);
  else launch_norm_out<__half>(a, format, st);
  return check_launch("rms_norm_fwd");
}
