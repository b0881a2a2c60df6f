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

// Eight consecutive elements starting at column c of a row, zeros from column `cols` on.  vec: rows and base are
// 16-byte aligned, so a unit that lies inside the row is one or two 128-bit loads.
template <typename T>
__device__ __forceinline__ void load_unit(const T* row, int64_t c, int64_t cols, bool vec, float (&v)[UNIT]) {
  if (vec && c + UNIT <= cols) {
    if (sizeof(T) == 4) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(row + c));
      const float4 b = __ldg(reinterpret_cast<const float4*>(row + c) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(row + c));
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
      using H = typename std::conditional<sizeof(T) == 4, __half, T>::type;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 p = pair_to_float(w[i], H());
        v[2 * i] = p.x;
        v[2 * i + 1] = p.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < UNIT; ++i) v[i] = c + i < cols ? to_float<T>(row[c + i]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store_unit(T* row, int64_t c, int64_t cols, bool vec, const float (&v)[UNIT]) {
  if (vec && c + UNIT <= cols) {
    if (sizeof(T) == 4) {
      float4* p = reinterpret_cast<float4*>(row + c);
      p[0] = make_float4(v[0], v[1], v[2], v[3]);
      p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      using H = typename std::conditional<sizeof(T) == 4, __half, T>::type;
      *reinterpret_cast<uint4*>(row + c) = make_uint4(float_to_pair(v[0], v[1], H()), float_to_pair(v[2], v[3], H()),
                                                      float_to_pair(v[4], v[5], H()), float_to_pair(v[6], v[7], H()));
    }
  } else {
#pragma unroll
    for (int i = 0; i < UNIT; ++i) if (c + i < cols) row[c + i] = from_float<T>(v[i]);
  }
}

// Scale code of the block that this lane's unit and those of its three neighbours make up (all four lanes of the
// quad take part).  The largest magnitude is found on the bit patterns, which order as the values do and put
// infinities and NaNs on top.
template <int FORMAT>
__device__ __forceinline__ uint32_t quad_scale_code(const float (&v)[UNIT]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < UNIT; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  constexpr int EMAX = FORMAT == NES_MXFP4 ? 2 : 8;
  return m >= 0x7f800000u ? 255u : uint32_t(max(int(m >> 23) - EMAX, 0));
}

// 2^-e for a scale code below 255 (at most 253: a normal number)
__device__ __forceinline__ float inverse_scale(uint32_t code) { return __uint_as_float((254u - code) << 23); }

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

__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(a), "f"(b));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(c), "f"(d));
  return uint32_t(lo) | (uint32_t(hi) << 16);
}

// Quantises this lane's unit of the block and stores its codes (4 or 8 bytes) and, from the block's first lane, the
// scale.  unit: index within the padded row.  Every lane of the warp calls it; `store` is false for lanes without a unit.
template <int FORMAT>
__device__ __forceinline__ void quantize_unit(float (&v)[UNIT], uint8_t* codes_row, uint8_t* scales_row, int64_t unit, bool store) {
  const uint32_t code = quad_scale_code<FORMAT>(v);
  const float inv = inverse_scale(code == 255u ? 127u : code);
#pragma unroll
  for (int i = 0; i < UNIT; ++i) v[i] = code == 255u ? 0.f : v[i] * inv;
  if (!store) return;
  if (FORMAT == NES_MXFP4)
    reinterpret_cast<uint32_t*>(codes_row)[unit] = pack_e2m1x8(v);
  else
    reinterpret_cast<uint2*>(codes_row)[unit] = make_uint2(pack_e4m3x4(v[0], v[1], v[2], v[3]), pack_e4m3x4(v[4], v[5], v[6], v[7]));
  if ((unit & 3) == 0) scales_row[unit >> 2] = uint8_t(code);
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

// The eight element values of a unit of codes, before the scale.
template <int FORMAT>
__device__ __forceinline__ void unit_elements(const uint8_t* codes_row, int64_t unit, float (&v)[UNIT]) {
  uint2 q;
  if (FORMAT == NES_MXFP4) {
    const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(codes_row) + unit);
    q = make_uint2(e2m1x4_to_e4m3(c), e2m1x4_to_e4m3(c >> 16));
  } else {
    q = __ldg(reinterpret_cast<const uint2*>(codes_row) + unit);
  }
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
