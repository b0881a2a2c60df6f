// Root-mean-square norm with the residual's addition and a plain or microscaled output.
//
//   h = x + residual                                   (fp32; stored in x's type when there is a residual)
//   y = h * rsqrt(mean(h^2) + eps) * (gain + s(r) * noise[d])     row = r * members + d
//
// One pass: a row stays in registers between the sum of squares and the scaling, so x and the residual are read once
// and h and y written once.  WARPS warps own a row and hold UNITS units of eight columns per lane, a warp's units next to
// one another; rows longer than that take the looping kernel, which reads x and the residual a second time.
//
// Rows that are not whole 16-byte pieces (SHIFTED): all plain tensors start on 16 bytes, so a row begins the same number of
// elements s past such a boundary in each of them, and a unit is taken from column 8 i - s on: loads and stores stay whole
// 16-byte words, and only a row's two ends are element accesses.  For a quantised output, whose blocks begin at
// column 0, the values of h are then moved s places between neighbouring lanes.
#include <algorithm>
#include <type_traits>
#include "microscale.cuh"

namespace nes {
namespace mx {

constexpr int MOST_WARPS = 17;                   // of a row: 16384 columns, and one unit more where rows are shifted
constexpr int WARP_ROWS = 4;                     // rows of a block whose warps take one each

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
  uint32_t minus;                                  // -1
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

// h * (r.x + r.y) * (g + gl) rounded once: s + se is the row's scale times the gain to 43 bits at least.
__device__ __forceinline__ float scaled(float h, float2 r, float g) {
  const float s = r.x * g, se = fmaf(r.y, g, fmaf(r.x, g, -s));
  return fmaf(h, s, h * se);
}
__device__ __forceinline__ float scaled(float h, float2 r, float g, float gl) {
  const float s = r.x * g, se = fmaf(r.x, gl, fmaf(r.y, g, fmaf(r.x, g, -s)));
  return fmaf(h, s, h * se);
}

// A quantised output rounds y a second time.  The first rounding, to fp32, decides that one only where it ends on a border of the second:
// a number of at most five bits, whether it lies between two codes or begins the binade of a block's scale.  The low 19 bits of such a
// y are zero, and y and the exact value are told apart in 64 bits: y stays if they are equal (the border's own rule holds), else
// it becomes its neighbour on the exact value's side.  y times the root is exact where the root is a number of few bits, without
// which no value but zero can lie on a border.  One y in half a million is such a one, zeros aside: what the kernels do for them
// is to gather every y's lowest set bit; a unit in which one of these is found is worked out a second time (settle_units).  A y
// below 2^-126 has fewer bits than that and keeps its rounding to fp32.
constexpr uint32_t BORDER_BITS = 0x7ff80000u;          // of a lowest set bit; a zero has none, or the sign
// minus: -1, which the compiler does not know of: a product, unlike a negation, leaves the ALU pipe free
__device__ __forceinline__ uint32_t lowest_bits(const float (&y)[UNIT], uint32_t minus) {
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < UNIT; ++i) all |= __float_as_uint(y[i]) & (minus * __float_as_uint(y[i]));
  return all;
}
__device__ __forceinline__ float settled(float y, float h, float g, float gl, double root) {
  const uint32_t bits = __float_as_uint(y);
  if (((bits & (0u - bits)) & BORDER_BITS) == 0u) return y;
  const double past = fma(-double(y), root, double(h) * (double(g) + double(gl)));
  const int step = past > 0.0 ? 1 : past < 0.0 ? -1 : 0;                  // 0 also for a NaN: an infinite y of an infinite h
  return __uint_as_float(bits + uint32_t(y < 0.f ? -step : step));
}

// A row's places in memory.
template <typename T>
struct Row {
  const T *x, *residual;
  T *h, *y;
  const float* noise;
  float sign;
  int shift;                                       // elements past a 16-byte boundary at which the row begins
  __device__ Row(const NormArgs& a, int64_t row) {
    const int64_t at = row * a.cols;
    x = static_cast<const T*>(a.x) + at;
    residual = a.residual ? static_cast<const T*>(a.residual) + at : nullptr;
    h = a.h ? static_cast<T*>(a.h) + at : nullptr;
    y = static_cast<T*>(a.y) + at;
    shift = int(at % int64_t(16 / sizeof(T)));
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
__device__ __forceinline__ Span span_of(const T* p, int64_t elements) {
  return Span{reinterpret_cast<const uint8_t*>(p), reinterpret_cast<const uint8_t*>(p + elements)};
}

// A unit from column c on that lies on a 16-byte boundary; c may be negative, columns outside the row read as zero.
template <typename T>
__device__ __forceinline__ Raw<T> load_boundary(const T* row, int c, int cols, const Span& span) {
  constexpr int NW = UNIT * sizeof(T) / 4, PER = 4 / sizeof(T);
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < NW; ++i) r.w[i] = 0u;
  if (c >= 0 && c + UNIT <= cols) {
#pragma unroll
    for (int i = 0; i < NW; i += 4) {
      const uint4 v = fetch(reinterpret_cast<const uint4*>(row + c) + i / 4);
      r.w[i] = v.x; r.w[i + 1] = v.y; r.w[i + 2] = v.z; r.w[i + 3] = v.w;
    }
  } else if (c < cols && c + UNIT > 0) {
#pragma unroll
    for (int i = 0; i < NW; i += 4) {
      const uint4 v = load_word<T>(span, reinterpret_cast<const uint8_t*>(row + c) + 4 * i);
      r.w[i] = v.x; r.w[i + 1] = v.y; r.w[i + 2] = v.z; r.w[i + 3] = v.w;
    }
#pragma unroll
    for (int i = 0; i < UNIT; ++i)
      if (c + i < 0 || c + i >= cols) r.w[i / PER] &= PER == 1 ? 0u : i & 1 ? 0x0000ffffu : 0xffff0000u;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store_boundary(T* row, int c, int cols, const Raw<T>& r) {
  constexpr int NW = UNIT * sizeof(T) / 4;
  if (c >= 0 && c + UNIT <= cols) {
#pragma unroll
    for (int i = 0; i < NW; i += 4) reinterpret_cast<uint4*>(row + c)[i / 4] = make_uint4(r.w[i], r.w[i + 1], r.w[i + 2], r.w[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < UNIT; ++i) if (c + i >= 0 && c + i < cols) store_element(row, c, r, i);
  }
}

// SPLIT: a unit is two runs of four columns, 128 apart, so that a warp's 16-byte accesses lie next to one another (fp32 rows in
// units of eight consecutive columns reach every 32-byte sector twice, half of it each time, and so do their gains).
// FULL, SPLIT_FULL: WHOLE and SPLIT where every unit of the block lies inside the row, without checks and zeros for what does not.
// ANY: the looping kernel's, units from column 8 i on wherever they lie.
enum RowAccess { WHOLE, FULL, SPLIT, SPLIT_FULL, SHIFTED, ANY };
__host__ __device__ constexpr bool is_split(RowAccess a) { return a == SPLIT || a == SPLIT_FULL; }
__host__ __device__ constexpr bool is_full(RowAccess a) { return a == FULL || a == SPLIT_FULL; }

constexpr int HALF_APART = 128;
__device__ __forceinline__ Raw<float> load_split(const float* row, int c, int cols) {
  Raw<float> r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (inside(c + h * HALF_APART, cols)) v = fetch(reinterpret_cast<const uint4*>(row + c + h * HALF_APART));
    r.w[4 * h] = v.x; r.w[4 * h + 1] = v.y; r.w[4 * h + 2] = v.z; r.w[4 * h + 3] = v.w;
  }
  return r;
}
__device__ __forceinline__ void store_split(float* row, int c, int cols, const Raw<float>& r) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (inside(c + h * HALF_APART, cols)) *reinterpret_cast<uint4*>(row + c + h * HALF_APART) = make_uint4(r.w[4 * h], r.w[4 * h + 1], r.w[4 * h + 2], r.w[4 * h + 3]);
}
// Quantises a split unit: its halves belong to two blocks, each held by eight neighbouring lanes; columns of the padding are zero.
template <int FORMAT, bool ALL>
__device__ __forceinline__ void quantize_split(float (&v)[UNIT], uint8_t* codes_row, uint8_t* scales_row, int c, int cols) {
  const int end = int(padded(cols));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = c + h * HALF_APART;
    float* q = v + 4 * h;
    if (!ALL && at >= cols) q[0] = q[1] = q[2] = q[3] = 0.f;             // fp32 rows end on a multiple of four columns here
    uint32_t m = __float_as_uint(max_magnitude(max_magnitude(q[0], q[1], q[2]), q[3], q[3])) & 0x7fffffffu;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t code = scale_code<FORMAT>(m);
    const float inv = inverse_scale(code);
    if (!ALL && at >= end) continue;
    if (FORMAT == NES_MXFP4) {
      const float e[UNIT] = {q[0] * inv, q[1] * inv, q[2] * inv, q[3] * inv, 0.f, 0.f, 0.f, 0.f};
      *reinterpret_cast<uint16_t*>(codes_row + at / 2) = uint16_t(code == 255u ? 0u : pack_e2m1x8(e));
    } else {
      const uint32_t e = pack_e4m3x4(q[0] * inv, q[1] * inv, q[2] * inv, q[3] * inv);
      *reinterpret_cast<uint32_t*>(codes_row + at) = code == 255u ? 0u : e;
    }
    if (at % BLOCK == 0) scales_row[at / BLOCK] = uint8_t(code);
  }
}

template <RowAccess ACCESS, typename T>
__device__ __forceinline__ Raw<T> load_at(const T* row, int c, int cols, const Span& span) {
  if constexpr (is_split(ACCESS)) return load_split(row, c, ACCESS == SPLIT_FULL ? NO_END : cols);
  else if constexpr (ACCESS == SHIFTED) return load_boundary(row, c, cols, span);
  else return load_raw<ACCESS != ANY>(row, c, ACCESS == FULL ? NO_END : cols, span);
}
template <RowAccess ACCESS, typename T>
__device__ __forceinline__ void store_at(T* row, int c, int cols, const Raw<T>& r) {
  if constexpr (is_split(ACCESS)) store_split(row, c, ACCESS == SPLIT_FULL ? NO_END : cols, r);
  else if constexpr (ACCESS == SHIFTED) store_boundary(row, c, cols, r);
  else store_raw<ACCESS != ANY, 32>(row, c, ACCESS == FULL ? NO_END : cols, r);
}
// gains and noise of a unit's columns, fp32 whatever the rows' type; a quantised output's shifted units have been moved by then
template <RowAccess ACCESS, bool MOVED>
__device__ __forceinline__ void load_gain(const float* row, int c, int cols, const Span& span, bool aligned_row, float (&g)[UNIT]) {
  if constexpr (is_split(ACCESS)) raw_values(load_split(row, c, ACCESS == SPLIT_FULL ? NO_END : cols), g);
  else if constexpr (ACCESS == WHOLE || ACCESS == FULL) raw_values(load_raw<true>(row, c, ACCESS == FULL ? NO_END : cols, span), g);
  else if (MOVED && aligned_row) raw_values(load_boundary(row, c, cols, span), g);
  else raw_values(load_raw<false>(row, c, cols, span), g);
}

template <typename T, RowAccess ACCESS>
__device__ __forceinline__ void load_h(const NormArgs& a, const Row<T>& row, int c, float (&v)[UNIT]) {
  const int cols = int(a.cols);
  const int64_t n = a.rows * a.cols;
  const Raw<T> x = load_at<ACCESS>(row.x, c, cols, span_of(static_cast<const T*>(a.x), n));
  if (row.residual) {
    const Raw<T> r = load_at<ACCESS>(row.residual, c, cols, span_of(static_cast<const T*>(a.residual), n));
    float q[UNIT];
    raw_values(x, v);
    raw_values(r, q);
#pragma unroll
    for (int i = 0; i < UNIT; ++i) v[i] += q[i];
  } else {
    raw_values(x, v);
  }
}

// The sum of squares of this warp's row, kept for settle_units outside the registers.
__device__ __forceinline__ volatile double& sum_of_row() {
  __shared__ double sums[MOST_WARPS];
  return sums[threadIdx.x >> 5];
}

// y of the unit at column c; all lanes of a warp call it.  A quantised output is stored from units of whole columns 8 i, and its
// values' lowest bits are added to `lowest`.  SETTLE: values at a border are settled, with the root of mean + eps.
template <typename T, int OUT, RowAccess ACCESS, bool SETTLE = false>
__device__ __forceinline__ void emit(const NormArgs& a, const Row<T>& row, int64_t index, int c, const float (&h)[UNIT], float2 r, double root, uint32_t& lowest) {
  constexpr bool MOVED = ACCESS == SHIFTED && OUT != 0;
  const int cols = int(a.cols);
  float g[UNIT], y[UNIT];
  if (a.gain) {
    load_gain<ACCESS, MOVED>(a.gain, c, cols, span_of(a.gain, cols), true, g);
  } else {
#pragma unroll
    for (int i = 0; i < UNIT; ++i) g[i] = 1.f;
  }
  if (row.noise) {
    float n[UNIT];
    load_gain<ACCESS, MOVED>(row.noise, c, cols, span_of(a.noise, a.members * a.cols), false, n);
#pragma unroll
    for (int i = 0; i < UNIT; ++i) {
      // gain + noise as a sum and what it rounds away
      const float e = row.sign * n[i], sum = g[i] + e, back = sum - g[i], lost = (g[i] - (sum - back)) + (e - back);
      y[i] = OUT != 0 ? scaled(h[i], r, sum, lost) : scaled(h[i], r, sum);
      if (SETTLE) y[i] = settled(y[i], h[i], sum, lost, root);
    }
  } else {
#pragma unroll
    for (int i = 0; i < UNIT; ++i) {
      y[i] = scaled(h[i], r, g[i]);
      if (SETTLE) y[i] = settled(y[i], h[i], g[i], 0.f, root);
    }
  }
  if (OUT != 0 && !SETTLE) lowest |= lowest_bits(y, a.minus);
  if (OUT == 0) {
    store_at<ACCESS>(row.y, c, cols, values_raw(y, T()));
    return;
  }
  constexpr int FORMAT = OUT == 0 ? NES_MXFP8 : OUT;
  uint8_t* codes = static_cast<uint8_t*>(a.y) + index * code_pitch(cols, FORMAT);
  uint8_t* scales = a.scales + index * scale_pitch(cols);
  if (is_split(ACCESS)) {
    quantize_split<FORMAT, ACCESS == SPLIT_FULL>(y, codes, scales, c, cols);
    return;
  }
  if (ACCESS != FULL && c + UNIT > cols) {                          // columns of the padding are zero whatever the row's scale (0 * inf is not)
#pragma unroll
    for (int i = 0; i < UNIT; ++i) if (c + i >= cols) y[i] = 0.f;
  }
  quantize_unit<FORMAT>(y, codes, scales, c / UNIT, ACCESS == FULL || c < int(padded(cols)));
}

// h of columns 8 i ... from units that begin `shift` elements earlier: the end of the unit `from` and the start of the next
// lane's, for lane 31 of the unit `next` of lane 0.
__device__ __forceinline__ void unshift(const float (&from)[UNIT], const float (&next)[UNIT], int shift, float (&to)[UNIT]) {
  const int lane = threadIdx.x & 31;
  float e[2 * UNIT];
#pragma unroll
  for (int i = 0; i < UNIT; ++i) {
    e[i] = from[i];
    e[UNIT + i] = __shfl_sync(0xffffffffu, lane == 0 ? next[i] : from[i], (lane + 1) & 31);
  }
#pragma unroll
  for (int b = 4; b; b >>= 1)
#pragma unroll
    for (int i = 0; i < 2 * UNIT - b; ++i) e[i] = shift & b ? e[i + b] : e[i];
#pragma unroll
  for (int i = 0; i < UNIT; ++i) to[i] = e[i];
}

// Sum over a row's threads (all of a block, or one warp), the same in every thread.  The threads' partial sums are joined in
// 64 bits: the last few additions carry the whole row's rounding.
template <bool BLOCK_ROW>
__device__ __forceinline__ double row_sum(float mine) {
  double s = mine;
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (BLOCK_ROW) {
    __shared__ double part[32];
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    s = part[0];
    for (int i = 1; i < warps; ++i) s += part[i];
  }
  return s;
}

__device__ __forceinline__ float square_sum(const float (&v)[UNIT]) {
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < UNIT; ++i) q = fmaf(v[i], v[i], q);
  return q;
}

// 1 / sqrt(mean + eps)
template <bool QUANTISED>
__device__ __forceinline__ float2 row_scale(const NormArgs& a, double sum) {
  if (QUANTISED) sum_of_row() = sum;                                      // every lane the same: each reads what it wrote itself
  return rsqrt_pair(sum * a.inv_cols + double(a.eps));
}

// This lane's unit of 32 neighbouring ones once more, with values at a border settled; x and the residual are read again.  All lanes of
// the warp call it.
template <typename T, int OUT, RowAccess ACCESS>
__device__ __forceinline__ void settle_unit(const NormArgs& a, int64_t index, int c, float2 r) {
  const Row<T> row(a, index);
  const double root = sqrt(sum_of_row() / double(a.cols) + double(a.eps));
  uint32_t lowest = 0;
  float h[UNIT];
  if (ACCESS == SHIFTED) {
    float from[UNIT], next[UNIT];
    load_h<T, ACCESS>(a, row, c - row.shift, from);
    load_h<T, ACCESS>(a, row, c - row.shift + 32 * UNIT, next);
    unshift(from, next, row.shift, h);
  } else {
    load_h<T, ACCESS>(a, row, c, h);
  }
  emit<T, OUT, ACCESS, true>(a, row, index, c, h, r, root, lowest);
}
template <typename T, int OUT, RowAccess ACCESS>
__device__ __noinline__ void settle_unit_call(const NormArgs a, int64_t index, int c, float2 r) { settle_unit<T, OUT, ACCESS>(a, index, c, r); }

// `units`: a bit for every unit, `step` columns apart, in which a lane has a value at a border.  CALL keeps the kernel's registers
// free of what a unit takes here.
template <typename T, int OUT, RowAccess ACCESS, bool CALL>
__device__ __forceinline__ void settle_units(const NormArgs& a, int64_t index, int first, int step, uint32_t units, float2 r) {
  units = __reduce_or_sync(0xffffffffu, units);
#pragma unroll 1
  for (; units; units &= units - 1) {
    const int c = first + (__ffs(units) - 1) * step;
    if (CALL) settle_unit_call<T, OUT, ACCESS>(a, index, c, r);
    else settle_unit<T, OUT, ACCESS>(a, index, c, r);
  }
}

// Whether a kernel calls for the settling, and the blocks that an SM holds at least (0: as many as the registers allow).  Kernels of few
// units would hold fewer blocks with it in their registers.  Time relative to kernels without any of it: 65536x256 fp32 1.02 with a call
// and 12 blocks, 1.06 without the call; 16384x1023 fp32 1.12 with a call, 1.02 without; 8192x4096 bf16 1.01 and 0.97.
constexpr bool calls_settle(int bytes, int units, RowAccess access, bool block_row) {
  return !block_row && (units < 4 || (access == SHIFTED && bytes == 2));
}
constexpr int blocks_held(int out, int bytes, int units, RowAccess access, bool block_row) {
  if (out == 0 || block_row) return 0;
  if (access == SHIFTED) return units == 1 ? 10 : units == 2 ? 8 : bytes == 4 ? 6 : 0;
  return units == 1 ? 12 : units == 2 ? 10 : 7;
}

template <typename T, int OUT, int UNITS, RowAccess ACCESS, bool BLOCK_ROW>
__global__ void __launch_bounds__(BLOCK_ROW ? MOST_WARPS * 32 : WARP_ROWS * 32, blocks_held(OUT, sizeof(T), UNITS, ACCESS, BLOCK_ROW)) rms_norm_kernel(const NormArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t index = BLOCK_ROW ? int64_t(blockIdx.x) : int64_t(blockIdx.x) * WARP_ROWS + warp;
  take_turn();
  if (index >= a.rows) return;
  const Row<T> row(a, index);
  const int base = BLOCK_ROW ? warp * UNITS * 32 * UNIT : 0, first = base + lane * (is_split(ACCESS) ? 4 : UNIT);
  const int shift = ACCESS == SHIFTED ? row.shift : 0;
  const int end = OUT != 0 ? int(padded(a.cols)) : int(a.cols) + shift;
  float v[UNITS + 1][UNIT];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) load_h<T, ACCESS>(a, row, first - shift + u * 32 * UNIT, v[u]);
  constexpr bool MOVE = ACCESS == SHIFTED && OUT != 0;
  if (MOVE && lane == 0) load_h<T, ACCESS>(a, row, first - shift + UNITS * 32 * UNIT, v[UNITS]);     // the next warp's first unit
  float s = 0.f;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) s += square_sum(v[u]);
  if (row.h) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) if (is_full(ACCESS) || base + u * 32 * UNIT < int(a.cols) + shift) store_at<ACCESS>(row.h, first - shift + u * 32 * UNIT, int(a.cols), values_raw(v[u], T()));
  }
  const float2 r = row_scale<OUT != 0>(a, row_sum<BLOCK_ROW>(s));
  uint32_t units = 0;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    uint32_t lowest = 0;
    if (!is_full(ACCESS) && base + u * 32 * UNIT >= end) break;         // nothing of the row in this warp's unit u
    if (MOVE) {
      float h[UNIT];
      unshift(v[u], v[u + 1], shift, h);
      emit<T, OUT, ACCESS>(a, row, index, first + u * 32 * UNIT, h, r, 0.0, lowest);
    } else {
      emit<T, OUT, ACCESS>(a, row, index, first - shift + u * 32 * UNIT, v[u], r, 0.0, lowest);
    }
    if (lowest & BORDER_BITS) units |= 1u << u;
  }
  if (OUT != 0) settle_units<T, OUT, ACCESS, calls_settle(sizeof(T), UNITS, ACCESS, BLOCK_ROW)>(a, index, first, 32 * UNIT, units, r);
}

// Rows of any length: the sum of squares in one loop over the row, the outputs in a second one.
template <typename T, int OUT, RowAccess ACCESS>
__global__ void __launch_bounds__(512, OUT == 0 ? 0 : ACCESS == ANY ? 3 : 4) rms_norm_long_kernel(const NormArgs a) {
  const int64_t index = blockIdx.x;
  take_turn();
  const Row<T> row(a, index);
  const int end = int(padded(a.cols)), step = blockDim.x * UNIT;
  float s = 0.f;
  for (int c0 = 0; c0 < end; c0 += step) {
    float v[UNIT];
    const int c = c0 + threadIdx.x * UNIT;
    load_h<T, ACCESS>(a, row, c, v);
    s += square_sum(v);
    if (row.h) store_at<ACCESS>(row.h, c, int(a.cols), values_raw(v, T()));
  }
  const float2 r = row_scale<OUT != 0>(a, row_sum<true>(s));
  uint32_t units = 0;                                             // a bit stands for every 32nd unit
  int u = 0;
  for (int c0 = 0; c0 < end; c0 += step, ++u) {
    float v[UNIT];
    uint32_t lowest = 0;
    const int c = c0 + threadIdx.x * UNIT;
    load_h<T, ACCESS>(a, row, c, v);
    emit<T, OUT, ACCESS>(a, row, index, c, v, r, 0.0, lowest);
    if (lowest & BORDER_BITS) units |= 1u << (u & 31);
  }
  if constexpr (OUT != 0)
    for (int c0 = threadIdx.x * UNIT; c0 - int(threadIdx.x) * UNIT < end; c0 += 32 * step) settle_units<T, OUT, ACCESS, true>(a, index, c0, step, units, r);
}

// Four units per lane keep the most loads in flight where there are rows enough for all SMs; a few rows are spread over more
// warps instead (one row of 4096 bf16: 3.2 us with 4 warps, 2.5 us with 16).
template <typename T, int OUT, int UNITS, bool ALIGNED, bool BLOCK_ROW>
static void launch_rows(const NormArgs& a, int64_t units, cudaStream_t st) {
  constexpr int OF_WARP = UNITS * 32;              // units that a warp holds
  constexpr RowAccess GUARDED = !ALIGNED ? SHIFTED : sizeof(T) == 4 ? SPLIT : WHOLE, PLAIN = sizeof(T) == 4 ? SPLIT_FULL : FULL;
  const unsigned grid = unsigned(BLOCK_ROW ? a.rows : ceil_div<int64_t>(a.rows, WARP_ROWS));
  const unsigned threads = unsigned(BLOCK_ROW ? ceil_div<int64_t>(units, OF_WARP) : WARP_ROWS) * 32;
  if (ALIGNED && (BLOCK_ROW ? a.cols % (OF_WARP * UNIT) == 0 : a.cols == OF_WARP * UNIT))
    launch_in_turn(rms_norm_kernel<T, OUT, UNITS, PLAIN, BLOCK_ROW>, grid, threads, st, a);
  else
    launch_in_turn(rms_norm_kernel<T, OUT, UNITS, GUARDED, BLOCK_ROW>, grid, threads, st, a);
}

template <typename T, int OUT, bool ALIGNED>
static void launch_norm(const NormArgs& a, cudaStream_t st) {
  const int64_t units = ALIGNED ? ceil_div<int64_t>(a.cols, 32 * UNIT) * 32 : std::max<int64_t>(padded(a.cols) / UNIT, (a.cols + 2 * (UNIT - 1)) / UNIT);
  const bool few = a.rows < 2 * sm_count();
  if (units > MOST_WARPS * 32 * 4) launch_in_turn(rms_norm_long_kernel<T, OUT, ALIGNED ? WHOLE : ANY>, unsigned(a.rows), 512, st, a);
  else if (units <= 32) launch_rows<T, OUT, 1, ALIGNED, false>(a, units, st);
  else if (few && units <= MOST_WARPS * 32) launch_rows<T, OUT, 1, ALIGNED, true>(a, units, st);
  else if (units <= 64) launch_rows<T, OUT, 2, ALIGNED, false>(a, units, st);
  else if (units <= 128) launch_rows<T, OUT, 4, ALIGNED, false>(a, units, st);
  else launch_rows<T, OUT, 4, ALIGNED, true>(a, units, st);
}

template <typename T, int OUT>
static void launch_norm_rows(const NormArgs& a, bool whole, cudaStream_t st) {
  if (whole) launch_norm<T, OUT, true>(a, st); else launch_norm<T, OUT, false>(a, st);
}

template <typename T>
static void launch_norm_out(const NormArgs& a, int format, cudaStream_t st) {
  const bool whole = (a.cols * sizeof(T)) % 16 == 0;
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
  NES_REQUIRE(aligned16(x) && aligned16(residual) && aligned16(residual_out) && aligned16(gain) && aligned16(noise) && aligned16(y),
              NES_ERR_BAD_ARG, "rms_norm_fwd: tensors must be 16-byte aligned");
  const int64_t plain = rows * cols * dtype_bytes(dtype);
  const Bytes outputs[] = {{y, format ? rows * code_pitch(cols, format) : plain}, {format ? y_scales : nullptr, rows * scale_pitch(cols)}, {residual_out, plain}};
  const Bytes inputs[] = {{x, plain}, {residual, plain}, {gain, cols * 4}, {noise, members * cols * 4}};
  NES_REQUIRE(!overlap(outputs, inputs), NES_ERR_BAD_ARG, "rms_norm_fwd: an output overlaps an input or another output");
  NormArgs a;
  a.x = x; a.residual = residual; a.h = residual_out; a.gain = gain; a.noise = noise; a.y = y; a.scales = y_scales;
  a.rows = rows; a.cols = cols; a.members = members > 0 ? members : 1; a.antithetic = antithetic;
  a.minus = 0xffffffffu; a.eps = eps; a.inv_cols = 1.0 / double(cols);
  cudaStream_t st = as_stream(stream);
  if (dtype == NES_F32) launch_norm_out<float>(a, format, st);
  else if (dtype == NES_BF16) launch_norm_out<__nv_bfloat16>(a, format, st);
  else launch_norm_out<__half>(a, format, st);
  return check_launch("rms_norm_fwd");
}
