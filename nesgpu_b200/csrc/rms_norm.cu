// Root-mean-square norm with the residual's addition and a plain or microscaled output.
//
//   h = x + residual                                   (fp32; stored in x's type when there is a residual)
//   y = h * rsqrt(mean(h^2) + eps) * (gain + s(r) * noise[d])     row = r * members + d
//
// One pass: a row stays in registers between the sum of squares and the scaling, so x and the residual are read once
// and h and y written once.  THREADS threads own a row (a warp for short rows, a block for longer ones) and hold UNITS
// units of eight columns each; rows longer than that take the looping kernel, which reads x and the residual a second
// time.
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

// h * (r.x + r.y) * g with the products' rounding errors carried along: s + se is the row's scale times the gain to 48 bits.
// SHARP leaves the fp32 result rounded to odd (cut off, lowest bit set), so that a rounding to fewer bits afterwards
// decides as it would on the unrounded value; a value exactly on a border does not occur except for a zero.  Otherwise
// the result is rounded to nearest.
template <bool SHARP>
__device__ __forceinline__ float scaled(float h, float2 r, float g) {
  const float s = r.x * g, se = fmaf(r.y, g, fmaf(r.x, g, -s));
  if (SHARP) return __uint_as_float(__float_as_uint(__fmaf_rz(h, s, h * se)) | 1u);
  return fmaf(h, s, h * se);
}

// A row's places in memory.
template <typename T>
struct Row {
  const T *x, *residual;
  T* h;
  const float* noise;
  float sign;
  __device__ Row(const NormArgs& a, int64_t row) {
    const int64_t at = row * a.cols;
    x = static_cast<const T*>(a.x) + at;
    residual = a.residual ? static_cast<const T*>(a.residual) + at : nullptr;
    h = a.h ? static_cast<T*>(a.h) + at : nullptr;
    noise = nullptr;
    sign = 0.f;
    if (a.noise) {
      const int64_t r = row / a.members;
      noise = a.noise + (row - r * a.members) * a.cols;
      sign = anti_sign(r, a.rows / a.members, a.antithetic);
    }
  }
};

template <typename T>
__device__ __forceinline__ Span span_of(const NormArgs& a, const void* p) {
  const T* b = static_cast<const T*>(p);
  return Span{reinterpret_cast<const uint8_t*>(b), reinterpret_cast<const uint8_t*>(b + a.rows * a.cols)};
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void load_h(const NormArgs& a, const Row<T>& row, int c, float (&v)[UNIT]) {
  const Raw<T> x = load_raw<ALIGNED>(row.x, c, int(a.cols), span_of<T>(a, a.x));
  if (row.residual) {
    const Raw<T> r = load_raw<ALIGNED>(row.residual, c, int(a.cols), span_of<T>(a, a.residual));
    float q[UNIT];
    raw_values(x, v);
    raw_values(r, q);
#pragma unroll
    for (int i = 0; i < UNIT; ++i) v[i] += q[i];
  } else {
    raw_values(x, v);
  }
}

// y of the unit at column c; all lanes of a warp call it
template <typename T, int OUT, bool ALIGNED>
__device__ __forceinline__ void emit(const NormArgs& a, const Row<T>& row, int64_t index, int c, const float (&h)[UNIT], float2 r) {
  const int cols = int(a.cols);
  float g[UNIT], y[UNIT];
  if (a.gain) {
    raw_values(load_raw<ALIGNED>(a.gain, c, cols, Span{reinterpret_cast<const uint8_t*>(a.gain), reinterpret_cast<const uint8_t*>(a.gain + cols)}), g);
  } else {
#pragma unroll
    for (int i = 0; i < UNIT; ++i) g[i] = 1.f;
  }
  if (row.noise) {
    float n[UNIT];
    raw_values(load_raw<ALIGNED>(row.noise, c, cols, Span{reinterpret_cast<const uint8_t*>(a.noise),
                                                          reinterpret_cast<const uint8_t*>(a.noise + a.members * a.cols)}), n);
#pragma unroll
    for (int i = 0; i < UNIT; ++i) g[i] = fmaf(row.sign, n[i], g[i]);
  }
#pragma unroll
  for (int i = 0; i < UNIT; ++i) y[i] = scaled<OUT != 0>(h[i], r, g[i]);
  if (OUT == 0) {
    store_raw<ALIGNED, 32>(static_cast<T*>(a.y) + index * a.cols, c, cols, values_raw(y, T()));
    return;
  }
  constexpr int FORMAT = OUT == 0 ? NES_MXFP8 : OUT;
  if (c + UNIT > cols) {                          // columns of the padding are zero whatever the row's scale (0 * inf is not)
#pragma unroll
    for (int i = 0; i < UNIT; ++i) if (c + i >= cols) y[i] = 0.f;
  }
  quantize_unit<FORMAT>(y, static_cast<uint8_t*>(a.y) + index * code_pitch(cols, FORMAT), a.scales + index * scale_pitch(cols), c / UNIT,
                        c < int(padded(cols)));
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

template <typename T, int OUT, int THREADS, int UNITS, bool ALIGNED>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS) rms_norm_kernel(const NormArgs a) {
  constexpr int ROWS = THREADS == 32 ? 4 : 1;
  const int64_t index = int64_t(blockIdx.x) * ROWS + (ROWS > 1 ? threadIdx.x / THREADS : 0);
  if (index >= a.rows) return;
  const Row<T> row(a, index);
  const int t = (threadIdx.x % THREADS) * UNIT;
  float v[UNITS][UNIT];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) load_h<T, ALIGNED>(a, row, t + u * THREADS * UNIT, v[u]);
  float s = 0.f;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) s += square_sum(v[u]);
  if (row.h) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) store_raw<ALIGNED, 32>(row.h, t + u * THREADS * UNIT, int(a.cols), values_raw(v[u], T()));
  }
  const float2 r = rsqrt_pair(row_sum<THREADS>(s) * a.inv_cols + double(a.eps));
#pragma unroll
  for (int u = 0; u < UNITS; ++u) emit<T, OUT, ALIGNED>(a, row, index, t + u * THREADS * UNIT, v[u], r);
}

// Rows of any length: the sum of squares in one loop over the row, the outputs in a second one.
template <typename T, int OUT, int THREADS, bool ALIGNED>
__global__ void __launch_bounds__(THREADS) rms_norm_long_kernel(const NormArgs a) {
  const int64_t index = blockIdx.x;
  const Row<T> row(a, index);
  const int end = int(padded(a.cols));
  float s = 0.f;
  for (int c0 = 0; c0 < end; c0 += THREADS * UNIT) {
    float v[UNIT];
    const int c = c0 + threadIdx.x * UNIT;
    load_h<T, ALIGNED>(a, row, c, v);
    s += square_sum(v);
    if (row.h) store_raw<ALIGNED, 32>(row.h, c, int(a.cols), values_raw(v, T()));
  }
  const float2 r = rsqrt_pair(row_sum<THREADS>(s) * a.inv_cols + double(a.eps));
  for (int c0 = 0; c0 < end; c0 += THREADS * UNIT) {
    float v[UNIT];
    const int c = c0 + threadIdx.x * UNIT;
    load_h<T, ALIGNED>(a, row, c, v);
    emit<T, OUT, ALIGNED>(a, row, index, c, v, r);
  }
}

template <typename T, int OUT, bool ALIGNED>
static void launch_norm(const NormArgs& a, cudaStream_t st) {
  const unsigned rows = unsigned(a.rows);
  const int64_t cols = padded(a.cols);
  if (cols <= 256) rms_norm_kernel<T, OUT, 32, 1, ALIGNED><<<(rows + 3) / 4, 128, 0, st>>>(a);
  else if (cols <= 512) rms_norm_kernel<T, OUT, 32, 2, ALIGNED><<<(rows + 3) / 4, 128, 0, st>>>(a);
  else if (cols <= 1024) rms_norm_kernel<T, OUT, 32, 4, ALIGNED><<<(rows + 3) / 4, 128, 0, st>>>(a);
  else if (cols <= 2048) rms_norm_kernel<T, OUT, 128, 2, ALIGNED><<<rows, 128, 0, st>>>(a);
  else if (cols <= 4096) rms_norm_kernel<T, OUT, 128, 4, ALIGNED><<<rows, 128, 0, st>>>(a);
  else if (cols <= 8192) rms_norm_kernel<T, OUT, 256, 4, ALIGNED><<<rows, 256, 0, st>>>(a);
  else if (cols <= 16384) rms_norm_kernel<T, OUT, 512, 4, ALIGNED><<<rows, 512, 0, st>>>(a);
  else rms_norm_long_kernel<T, OUT, 512, ALIGNED><<<rows, 512, 0, st>>>(a);
}

template <typename T, int OUT>
static void launch_norm_rows(const NormArgs& a, bool whole, cudaStream_t st) {
  if (whole) launch_norm<T, OUT, true>(a, st); else launch_norm<T, OUT, false>(a, st);
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
  NES_REQUIRE(rows <= LARGEST_EXTENT && cols <= LARGEST_EXTENT, NES_ERR_UNSUPPORTED, "rms_norm_fwd: too large");
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
