// Root-mean-square norm with the residual's addition and a plain or microscaled output.
//
//   h = x + residual                                   (fp32; stored in x's type when there is a residual)
//   y = h * rsqrt(mean(h^2) + eps) * (gain + s(r) * noise[d])     row = r * members + d
//
// One pass: a row stays in registers between the sum of squares and the scaling, so x and the residual are read once
// and h and y written once.  THREADS threads own a row (a warp for short rows, a block for longer ones) and hold UNITS
// units of eight columns each; rows longer than that take the looping kernel, which reads x and the residual a second
// time.  A unit is eight consecutive columns, or (STRIPES: rows that are not whole 16-byte pieces) one column in each of
// eight consecutive blocks of 32, a lane per column, so that any row start is read and written in whole lines.
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
  const float s = r.x * g, se = fmaf(r.y, g, fmaf(r.x, g, -s));
  const float p = h * s, c = fmaf(h, se, fmaf(h, s, -p));
  if (SHARP) return __uint_as_float(__float_as_uint(__fadd_rz(p, c)) | 1u);
  return fabsf(p) < 3.0e38f && fabsf(s) < 3.0e38f ? p + c : p;       // infinities have no error terms
}

// Where a thread's unit u lies: its first column, and how the rest of the unit follows it.
template <bool STRIPES, int THREADS>
__device__ __forceinline__ int64_t unit_column(int t, int64_t u) {
  if (STRIPES) return ((t >> 5) + u * (THREADS / 32)) * (32 * UNIT) + (t & 31);
  return (t + u * THREADS) * UNIT;
}
template <bool STRIPES, typename T>
__device__ __forceinline__ void get(const T* row, int64_t c, int64_t cols, float (&v)[UNIT]) {
  if (STRIPES) load_stripes(row, c, cols, v); else load_unit(row, c, cols, v);
}
template <bool STRIPES, typename T>
__device__ __forceinline__ void put(T* row, int64_t c, int64_t cols, const float (&v)[UNIT]) {
  if (STRIPES) store_stripes(row, c, cols, v); else store_unit(row, c, cols, v);
}

// A row's member noise and its sign.
struct RowNoise { const float* p; float sign; };
__device__ __forceinline__ RowNoise row_noise(const NormArgs& a, int64_t row) {
  if (!a.noise) return RowNoise{nullptr, 0.f};
  const int64_t r = row / a.members, d = row - r * a.members;
  return RowNoise{a.noise + d * a.cols, anti_sign(r, a.rows / a.members, a.antithetic)};
}

template <typename T, bool STRIPES>
__device__ __forceinline__ void load_h(const NormArgs& a, int64_t row, int64_t c, float (&v)[UNIT]) {
  get<STRIPES>(static_cast<const T*>(a.x) + row * a.cols, c, a.cols, v);
  if (a.residual) {
    float q[UNIT];
    get<STRIPES>(static_cast<const T*>(a.residual) + row * a.cols, c, a.cols, q);
#pragma unroll
    for (int i = 0; i < UNIT; ++i) v[i] += q[i];
  }
}

// y of the unit at column c; all lanes of a warp call it
template <typename T, int OUT, bool STRIPES>
__device__ __forceinline__ void emit(const NormArgs& a, const RowNoise& noise, int64_t row, int64_t c, const float (&h)[UNIT], float2 r) {
  float g[UNIT], y[UNIT];
  if (a.gain) {
    get<STRIPES>(a.gain, c, a.cols, g);
  } else {
#pragma unroll
    for (int i = 0; i < UNIT; ++i) g[i] = 1.f;
  }
  if (noise.p) {
    float n[UNIT];
    get<STRIPES>(noise.p, c, a.cols, n);
#pragma unroll
    for (int i = 0; i < UNIT; ++i) g[i] = fmaf(noise.sign, n[i], g[i]);
  }
#pragma unroll
  for (int i = 0; i < UNIT; ++i) y[i] = scaled<OUT != 0>(h[i], r, g[i]);
  if (OUT == 0) {
    put<STRIPES>(static_cast<T*>(a.y) + row * a.cols, c, a.cols, y);
    return;
  }
  // columns of the padding are zero whatever the row's scale (0 * inf is not)
  constexpr int FORMAT = OUT == 0 ? NES_MXFP8 : OUT, APART = STRIPES ? 32 : 1;
  if (c + (UNIT - 1) * APART >= a.cols) {
#pragma unroll
    for (int i = 0; i < UNIT; ++i) if (c + i * APART >= a.cols) y[i] = 0.f;
  }
  uint8_t* codes = static_cast<uint8_t*>(a.y) + row * code_pitch(a.cols, FORMAT);
  uint8_t* scales = a.scales + row * scale_pitch(a.cols);
  if (STRIPES) quantize_stripes<FORMAT>(y, codes, scales, c / BLOCK, padded(a.cols) / BLOCK, int(c) & 31);
  else quantize_unit<FORMAT>(y, codes, scales, c / UNIT, c < padded(a.cols));
}

template <int N>
__device__ __forceinline__ double tree_sum(const double* p) {
  if constexpr (N == 1) return p[0];
  else return tree_sum<N / 2>(p) + tree_sum<N / 2>(p + N / 2);
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
    s = tree_sum<THREADS / 32>(part);
  }
  return s;
}

__device__ __forceinline__ float square_sum(const float (&v)[UNIT]) {
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < UNIT; ++i) q = fmaf(v[i], v[i], q);
  return q;
}

template <typename T, int OUT, int THREADS, int UNITS, bool STRIPES>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS) rms_norm_kernel(const NormArgs a) {
  constexpr int ROWS = THREADS == 32 ? 4 : 1;
  const int64_t row = int64_t(blockIdx.x) * ROWS + (ROWS > 1 ? threadIdx.x / THREADS : 0);
  if (row >= a.rows) return;
  const int t = threadIdx.x % THREADS;
  float v[UNITS][UNIT];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) load_h<T, STRIPES>(a, row, unit_column<STRIPES, THREADS>(t, u), v[u]);
  const RowNoise noise = row_noise(a, row);
  float s = 0.f;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) s += square_sum(v[u]);
  if (a.h) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) put<STRIPES>(static_cast<T*>(a.h) + row * a.cols, unit_column<STRIPES, THREADS>(t, u), a.cols, v[u]);
  }
  const float2 r = rsqrt_pair(row_sum<THREADS>(s) * a.inv_cols + double(a.eps));
#pragma unroll
  for (int u = 0; u < UNITS; ++u) emit<T, OUT, STRIPES>(a, noise, row, unit_column<STRIPES, THREADS>(t, u), v[u], r);
}

// Rows of any length: the sum of squares in one loop over the row, the outputs in a second one.
template <typename T, int OUT, int THREADS, bool STRIPES>
__global__ void __launch_bounds__(THREADS) rms_norm_long_kernel(const NormArgs a) {
  const int64_t row = blockIdx.x;
  const int64_t units = (padded(a.cols) + THREADS * UNIT - 1) / (THREADS * UNIT);
  const RowNoise noise = row_noise(a, row);
  float s = 0.f;
  for (int64_t u = 0; u < units; ++u) {
    float v[UNIT];
    const int64_t c = unit_column<STRIPES, THREADS>(threadIdx.x, u);
    load_h<T, STRIPES>(a, row, c, v);
    s += square_sum(v);
    if (a.h) put<STRIPES>(static_cast<T*>(a.h) + row * a.cols, c, a.cols, v);
  }
  const float2 r = rsqrt_pair(row_sum<THREADS>(s) * a.inv_cols + double(a.eps));
  for (int64_t u = 0; u < units; ++u) {
    float v[UNIT];
    const int64_t c = unit_column<STRIPES, THREADS>(threadIdx.x, u);
    load_h<T, STRIPES>(a, row, c, v);
    emit<T, OUT, STRIPES>(a, noise, row, c, v, r);
  }
}

template <typename T, int OUT, bool STRIPES>
static void launch_norm(const NormArgs& a, cudaStream_t st) {
  const unsigned rows = unsigned(a.rows);
  const int64_t cols = padded(a.cols);
  if (cols <= 256) rms_norm_kernel<T, OUT, 32, 1, STRIPES><<<(rows + 3) / 4, 128, 0, st>>>(a);
  else if (cols <= 512) rms_norm_kernel<T, OUT, 32, 2, STRIPES><<<(rows + 3) / 4, 128, 0, st>>>(a);
  else if (cols <= 1024) rms_norm_kernel<T, OUT, 32, 4, STRIPES><<<(rows + 3) / 4, 128, 0, st>>>(a);
  else if (cols <= 2048) rms_norm_kernel<T, OUT, 128, 2, STRIPES><<<rows, 128, 0, st>>>(a);
  else if (cols <= 4096) rms_norm_kernel<T, OUT, 128, 4, STRIPES><<<rows, 128, 0, st>>>(a);
  else if (cols <= 8192) rms_norm_kernel<T, OUT, 256, 4, STRIPES><<<rows, 256, 0, st>>>(a);
  else if (cols <= 16384) rms_norm_kernel<T, OUT, 512, 4, STRIPES><<<rows, 512, 0, st>>>(a);
  else rms_norm_long_kernel<T, OUT, 512, STRIPES><<<rows, 512, 0, st>>>(a);
}

template <typename T, int OUT>
static void launch_norm_rows(const NormArgs& a, bool whole, cudaStream_t st) {
  if (whole) launch_norm<T, OUT, false>(a, st); else launch_norm<T, OUT, true>(a, st);
}

template <typename T>
static void launch_norm_out(const NormArgs& a, int format, cudaStream_t st) {
  const bool whole = (a.cols * sizeof(T)) % 16 == 0 && aligned16(a.x) && aligned16(a.residual) && aligned16(a.h) && aligned16(a.gain) &&
                     aligned16(a.noise) && aligned16(a.y);
  if (format == 0) launch_norm_rows<T, 0>(a, whole, st);
  else if (format == NES_MXFP4) launch_norm_rows<T, NES_MXFP4>(a, whole, st);
  else launch_norm_rows<T, NES_MXFP8>(a, whole, st);
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
  NormArgs a;
  a.x = x; a.residual = residual; a.h = residual_out; a.gain = gain; a.noise = noise; a.y = y; a.scales = y_scales;
  a.rows = rows; a.cols = cols; a.members = members > 0 ? members : 1; a.antithetic = antithetic;
  a.eps = eps; a.inv_cols = 1.0 / double(cols);
  cudaStream_t st = as_stream(stream);
  if (dtype == NES_F32) launch_norm_out<float>(a, format, st);
  else if (dtype == NES_BF16) launch_norm_out<__nv_bfloat16>(a, format, st);
  else launch_norm_out<__half>(a, format, st);
  return check_launch("rms_norm_fwd");
}
