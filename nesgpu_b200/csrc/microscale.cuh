// Microscaled blocks: 32 consecutive elements of a row share one power of two.
//
//   a = max |x| over the block,  e = floor(log2 a) - EMAX clamped to >= -127,  code = e + 127
//   element = x * 2^-e rounded to nearest even, saturated to the largest element
//
// EMAX is the exponent of the largest element: 2 for e2m1 (6 = 1.5 * 2^2), 8 for e4m3 (448 = 1.75 * 2^8).  A block that
// holds a NaN or an infinity gets code 255 and zero elements: all of it reads as NaN.  A zero block gets code 0.
//
// Storage: row-major bytes, every row padded to whole groups of 128 elements (4 blocks, so that a row's codes are a
// multiple of 64 bytes and its scales of 4); e2m1 keeps the even column in the low half of a byte.  Pad codes and pad
// scales are 0.
#pragma once
#include <cuda_bf16.h>
#include "common.cuh"

namespace nes {
namespace mx {

constexpr int BLOCK = 32;
constexpr int GROUP = 128;         // row padding in elements
constexpr int UNIT = 8;            // elements a thread handles at once; 4 neighbouring lanes make a block

__host__ __device__ constexpr int64_t padded(int64_t cols) { return (cols + GROUP - 1) / GROUP * GROUP; }
__host__ __device__ constexpr int64_t code_pitch(int64_t cols, int format) { return format == NES_MXFP4 ? padded(cols) / 2 : padded(cols); }
__host__ __device__ constexpr int64_t scale_pitch(int64_t cols) { return padded(cols) / BLOCK; }

inline bool known_format(int f) { return f == NES_MXFP4 || f == NES_MXFP8; }
inline bool known_dtype(int t) { return t == NES_F32 || t == NES_BF16 || t == NES_F16; }
inline bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; }
inline int64_t dtype_bytes(int t) { return t == NES_F32 ? 4 : 2; }

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Two fp32 values from one 32-bit word of two 16-bit ones.
__device__ __forceinline__ float2 pair_to_float(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 pair_to_float(uint32_t w, __half) {
  __half2 h;
  memcpy(&h, &w, 4);
  return __half22float2(h);
}
__device__ __forceinline__ uint32_t float_to_pair(float a, float b, __nv_bfloat16) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  uint32_t w;
  memcpy(&w, &h, 4);
  return w;
}
__device__ __forceinline__ uint32_t float_to_pair(float a, float b, __half) {
  __half2 h = __floats2half2_rn(a, b);
  uint32_t w;
  memcpy(&w, &h, 4);
  return w;
}

// Eight consecutive elements starting at column c of a row whose start is 16-byte aligned and whose length is a multiple
// of 16 bytes; zeros from column `cols` on (with fp32 rows a unit may lie half inside).
__device__ __forceinline__ void load_unit(const float* row, int64_t c, int64_t cols, float (&v)[UNIT]) {
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
  if (c < cols) a = __ldg(reinterpret_cast<const float4*>(row + c));
  if (c + 4 < cols) b = __ldg(reinterpret_cast<const float4*>(row + c) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename H>
__device__ __forceinline__ void load_unit(const H* row, int64_t c, int64_t cols, float (&v)[UNIT]) {
  uint4 a = make_uint4(0u, 0u, 0u, 0u);
  if (c < cols) a = __ldg(reinterpret_cast<const uint4*>(row + c));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = pair_to_float(w[i], H());
    v[2 * i] = p.x;
    v[2 * i + 1] = p.y;
  }
}
__device__ __forceinline__ void store_unit(float* row, int64_t c, int64_t cols, const float (&v)[UNIT]) {
  if (c < cols) *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
  if (c + 4 < cols) *reinterpret_cast<float4*>(row + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
template <typename H>
__device__ __forceinline__ void store_unit(H* row, int64_t c, int64_t cols, const float (&v)[UNIT]) {
  if (c < cols)
    *reinterpret_cast<uint4*>(row + c) = make_uint4(float_to_pair(v[0], v[1], H()), float_to_pair(v[2], v[3], H()),
                                                    float_to_pair(v[4], v[5], H()), float_to_pair(v[6], v[7], H()));
}

// Rows of any length and alignment are walked the other way round: the 32 lanes take 32 consecutive columns, so that every access
// of a warp is one stretch of memory whatever its start, and a block is one such access.  v[i] is column c + 32 i.
template <typename T, int N>
__device__ __forceinline__ void load_stripes(const T* row, int64_t c, int64_t cols, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = c + 32 * i < cols ? to_float<T>(row[c + 32 * i]) : 0.f;
}
template <typename T, int N>
__device__ __forceinline__ void store_stripes(T* row, int64_t c, int64_t cols, const float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) if (c + 32 * i < cols) row[c + 32 * i] = from_float<T>(v[i]);
}

// larger magnitude of the two, NaN if either is one
__device__ __forceinline__ float max_magnitude(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

// Scale code of a block from the bits of its largest magnitude (a NaN or an infinity lies on top).
template <int FORMAT>
__device__ __forceinline__ uint32_t scale_code(uint32_t m) {
  constexpr int EMAX = FORMAT == NES_MXFP4 ? 2 : 8;
  return m >= 0x7f800000u ? 255u : uint32_t(max(int(m >> 23) - EMAX, 0));
}

// 2^-e for a scale code below 255 (at most 253: a normal number); 0 for 255
__device__ __forceinline__ float inverse_scale(uint32_t code) { return __uint_as_float(code == 255u ? 0u : (254u - code) << 23); }

// 2^(code - 127), NaN for 255
__device__ __forceinline__ float scale_value(uint32_t code) {
  return __uint_as_float(code == 255u ? 0x7fc00000u : code == 0u ? 0x00400000u : code << 23);
}

__device__ __forceinline__ uint32_t pack_e2m1x8(const float (&v)[UNIT]) {
  uint32_t r;
  asm("{\n"
      ".reg .b8 b0, b1, b2, b3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      "mov.b32 %0, {b0, b1, b2, b3};\n"
      "}\n"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// byte of two e2m1 codes, a in the low half
__device__ __forceinline__ uint32_t pack_e2m1x2(float a, float b) {
  uint32_t r;
  asm("{\n.reg .b8 b0, z;\nmov.b16 {b0, z}, 0;\ncvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\nmov.b32 %0, {b0, z, z, z};\n}\n" : "=r"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint32_t pack_e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) { return pack_e4m3x2(a, b) | (pack_e4m3x2(c, d) << 16); }

// Quantises this lane's unit of a block that four neighbouring lanes hold (all lanes of the warp call it) and stores its codes
// and, from the block's first lane, the scale.  unit: index within the padded row; `store` is false for lanes without one.
template <int FORMAT>
__device__ __forceinline__ void quantize_unit(float (&v)[UNIT], uint8_t* codes_row, uint8_t* scales_row, int64_t unit, bool store) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < UNIT; ++i) top = max_magnitude(top, v[i]);
  uint32_t m = __float_as_uint(top) & 0x7fffffffu;
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const uint32_t code = scale_code<FORMAT>(m);
  const float inv = inverse_scale(code);
#pragma unroll
  for (int i = 0; i < UNIT; ++i) v[i] *= inv;
  if (!store) return;
  if (FORMAT == NES_MXFP4) {
    const uint32_t q = pack_e2m1x8(v);
    reinterpret_cast<uint32_t*>(codes_row)[unit] = code == 255u ? 0u : q;
  } else {
    const uint32_t lo = pack_e4m3x4(v[0], v[1], v[2], v[3]), hi = pack_e4m3x4(v[4], v[5], v[6], v[7]);
    reinterpret_cast<uint2*>(codes_row)[unit] = make_uint2(code == 255u ? 0u : lo, code == 255u ? 0u : hi);
  }
  if ((unit & 3) == 0) scales_row[unit >> 2] = uint8_t(code);
}

// The same for N blocks of 32 columns, one lane per column: blocks block0 ... block0 + N - 1 of the row, of which those below
// `blocks` (the padded row's) are stored.  N is even.
template <int FORMAT, int N>
__device__ __forceinline__ void quantize_stripes(float (&v)[N], uint8_t* codes_row, uint8_t* scales_row, int64_t block0, int64_t blocks, int lane) {
  uint32_t mine = 0;                                             // lane i keeps the scale of block i
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t code = scale_code<FORMAT>(__reduce_max_sync(0xffffffffu, __float_as_uint(v[i]) & 0x7fffffffu));
    v[i] = code == 255u ? 0.f : v[i] * inverse_scale(code);
    if (lane == i) mine = code;
  }
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    if (FORMAT == NES_MXFP4) {
      // two blocks at once: even lanes store the first one's bytes, odd lanes the second one's
      const uint32_t b = pack_e2m1x2(v[i], v[i + 1]), o = __shfl_xor_sync(0xffffffffu, b, 1);
      const int64_t block = block0 + i + (lane & 1);
      if (block < blocks) codes_row[block * 16 + (lane >> 1)] = uint8_t(lane & 1 ? (o >> 4) | (b & 0xf0u) : (b & 15u) | (o << 4));
    } else {
      const uint32_t two = pack_e4m3x2(v[i], v[i + 1]);
      if (block0 + i < blocks) codes_row[(block0 + i) * 32 + lane] = uint8_t(two);
      if (block0 + i + 1 < blocks) codes_row[(block0 + i + 1) * 32 + lane] = uint8_t(two >> 8);
    }
  }
  if (lane < N && block0 + lane < blocks) scales_row[block0 + lane] = uint8_t(mine);
}

// e4m3 bytes of four e2m1 codes (the low 16 bits of c): a byte look-up in the eight magnitudes, then the signs
__device__ __forceinline__ uint32_t e2m1x4_to_e4m3(uint32_t c) {
  const uint32_t magnitude = __byte_perm(0x3c383000u, 0x4c484440u, c & 0x7777u);   // 0 .5 1 1.5 | 2 3 4 6
  const uint32_t s = c & 0x8888u;
  return magnitude | ((s << 4) & 0x80u) | ((s << 8) & 0x8000u) | ((s << 12) & 0x800000u) | ((s << 16) & 0x80000000u);
}

// value of one e4m3 byte (exact in fp16, hence in fp32)
__device__ __forceinline__ float2 e4m3x2_to_float(uint32_t two) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(uint16_t(two)));
  return pair_to_float(h2, __half());
}

// The eight elements of a unit as e4m3 bytes, and their values before the scale.
template <int FORMAT>
__device__ __forceinline__ uint2 load_codes(const uint8_t* codes_row, int64_t unit) {
  if (FORMAT == NES_MXFP8) return __ldg(reinterpret_cast<const uint2*>(codes_row) + unit);
  const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(codes_row) + unit);
  return make_uint2(e2m1x4_to_e4m3(c), e2m1x4_to_e4m3(c >> 16));
}
__device__ __forceinline__ void unit_elements(const uint2& q, float (&v)[UNIT]) {
  const uint32_t half[4] = {q.x, q.x >> 16, q.y, q.y >> 16};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = e4m3x2_to_float(half[i] & 0xffffu);
    v[2 * i] = p.x;
    v[2 * i + 1] = p.y;
  }
}

}  // namespace mx
}  // namespace nes
