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
constexpr int64_t LARGEST_EXTENT = 0x3fffffff;    // of rows and of columns: both are kept in 32 bits, offsets in 64
constexpr int UNIT = 8;            // elements a thread handles at once; 4 neighbouring lanes make a block

__host__ __device__ constexpr int64_t padded(int64_t cols) { return (cols + GROUP - 1) / GROUP * GROUP; }
__host__ __device__ constexpr int64_t code_pitch(int64_t cols, int format) { return format == NES_MXFP4 ? padded(cols) / 2 : padded(cols); }
__host__ __device__ constexpr int64_t scale_pitch(int64_t cols) { return padded(cols) / BLOCK; }

inline bool known_format(int f) { return f == NES_MXFP4 || f == NES_MXFP8; }
inline bool known_dtype(int t) { return t == NES_F32 || t == NES_BF16 || t == NES_F16; }
inline bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; }
inline int64_t dtype_bytes(int t) { return t == NES_F32 ? 4 : 2; }

// What a call reads or writes.  The blocks of a kernel run in any order, so an output that lies over an input or another output is
// refused.
struct Bytes { const void* at; int64_t size; };
inline bool overlap(const Bytes& a, const Bytes& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
  return a.at && b.at && x < y + uintptr_t(b.size) && y < x + uintptr_t(a.size);
}
template <int A, int B>
inline bool overlap(const Bytes (&outputs)[A], const Bytes (&inputs)[B]) {
  for (int o = 0; o < A; ++o) {
    for (const Bytes& i : inputs)
      if (overlap(outputs[o], i)) return true;
    for (int other = 0; other < o; ++other)
      if (overlap(outputs[o], outputs[other])) return true;
  }
  return false;
}

// An ordinary load.  Not __ldg and no __restrict__ inputs in these kernels: a load of memory that is taken to be constant for the
// whole kernel could be moved ahead of the wait for the kernel before (take_turn below), which may just be writing it.
template <typename V> __device__ __forceinline__ V fetch(const V* p) { return *p; }

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Two fp32 values from one 32-bit word of two 16-bit ones, and back (rounded to nearest even).
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

// ------------------------------------------------------------------- a unit of a row in memory: UNIT elements of T
//
// ALIGNED: the tensor starts on 16 bytes and its rows are whole 16-byte pieces.  Otherwise a row may start anywhere: a unit
// is cut out of the aligned 16-byte words around it (the second of which is the neighbouring lane's first, so it comes from
// the L1 cache), and put back by shifting it against the neighbouring lane's unit into aligned words; element accesses
// remain at the ends of a run of lanes only.

// NO_END in the place of `cols`: the caller knows that the unit lies inside the row.

constexpr int NO_END = 0x7fffffff;
__device__ __forceinline__ bool inside(int c, int cols) { return cols == NO_END || c < cols; }

template <typename T> struct Raw { uint32_t w[UNIT * sizeof(T) / 4]; };
struct Span { const uint8_t *begin, *end; };                      // of a whole tensor

// the aligned 16-byte word at `at`, bytes outside the tensor read as zero without being touched
template <typename T>
__device__ __forceinline__ uint4 load_word(const Span& s, const uint8_t* at) {
  if (at >= s.begin && at + 16 <= s.end) return fetch(reinterpret_cast<const uint4*>(at));
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < int(16 / sizeof(T)); ++i) {
    const T* e = reinterpret_cast<const T*>(at) + i;
    if (reinterpret_cast<const uint8_t*>(e) < s.begin || reinterpret_cast<const uint8_t*>(e) >= s.end) continue;
    if (sizeof(T) == 4) w[i & 3] = *reinterpret_cast<const uint32_t*>(e);
    else w[i / 2] |= uint32_t(*reinterpret_cast<const uint16_t*>(e)) << (16 * (i & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Columns c ... c + 7 of a row, zeros from column `cols` on.
template <bool ALIGNED, typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* row, int c, int cols, const Span& span) {
  constexpr int NW = UNIT * sizeof(T) / 4;
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < NW; ++i) r.w[i] = 0u;
  if (!inside(c, cols)) return r;
  const uint8_t* at = reinterpret_cast<const uint8_t*>(row + c);
  if (ALIGNED) {
#pragma unroll
    for (int i = 0; i < NW; i += 4) {
      if (i && !inside(c + 4, cols)) break;                       // an fp32 unit may lie half inside
      const uint4 v = fetch(reinterpret_cast<const uint4*>(at) + i / 4);
      r.w[i] = v.x; r.w[i + 1] = v.y; r.w[i + 2] = v.z; r.w[i + 3] = v.w;
    }
    return r;
  }
  const uint32_t shift = uint32_t(reinterpret_cast<uintptr_t>(at)) & 15u;
  const bool interior = at - 16 >= span.begin && at + 4 * NW + 16 <= span.end;
  uint32_t e[NW + 4];
#pragma unroll
  for (int i = 0; i < NW + 4; i += 4) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (i < NW || shift) v = interior ? fetch(reinterpret_cast<const uint4*>(at - shift + 4 * i)) : load_word<T>(span, at - shift + 4 * i);
    e[i] = v.x; e[i + 1] = v.y; e[i + 2] = v.z; e[i + 3] = v.w;
  }
  const bool two = shift & 8u, one = shift & 4u;
#pragma unroll
  for (int i = 0; i < NW + 2; ++i) e[i] = two ? e[i + 2] : e[i];
#pragma unroll
  for (int i = 0; i < NW + 1; ++i) e[i] = one ? e[i + 1] : e[i];
#pragma unroll
  for (int i = 0; i < NW; ++i) r.w[i] = sizeof(T) == 4 ? e[i] : __funnelshift_r(e[i], e[i + 1], (shift & 2u) * 8u);
  if (c + UNIT > cols) {                                          // the row ends inside: what follows is another row's
#pragma unroll
    for (int i = 0; i < UNIT; ++i) {
      if (c + i < cols) continue;
      if (sizeof(T) == 4) r.w[i & (NW - 1)] = 0u;
      else r.w[i / 2] &= i & 1 ? 0x0000ffffu : 0u;
    }
  }
  return r;
}

__device__ __forceinline__ void raw_values(const Raw<float>& r, float (&v)[UNIT]) {
#pragma unroll
  for (int i = 0; i < UNIT; ++i) v[i] = __uint_as_float(r.w[i]);
}
template <typename H>
__device__ __forceinline__ void raw_values(const Raw<H>& r, float (&v)[UNIT]) {
#pragma unroll
  for (int i = 0; i < UNIT / 2; ++i) {
    const float2 p = pair_to_float(r.w[i], H());
    v[2 * i] = p.x;
    v[2 * i + 1] = p.y;
  }
}
__device__ __forceinline__ Raw<float> values_raw(const float (&v)[UNIT], float) {
  Raw<float> r;
#pragma unroll
  for (int i = 0; i < UNIT; ++i) r.w[i] = __float_as_uint(v[i]);
  return r;
}
template <typename H>
__device__ __forceinline__ Raw<H> values_raw(const float (&v)[UNIT], H) {
  Raw<H> r;
#pragma unroll
  for (int i = 0; i < UNIT / 2; ++i) r.w[i] = float_to_pair(v[2 * i], v[2 * i + 1], H());
  return r;
}

template <typename T>
__device__ __forceinline__ void store_element(T* row, int c, const Raw<T>& r, int i) {
  constexpr int PER = 4 / sizeof(T);
  const uint32_t w = r.w[i / PER] >> (32 / PER * (i % PER) & 31);
  if (sizeof(T) == 4) reinterpret_cast<uint32_t*>(row)[c + i] = w;
  else if (sizeof(T) == 2) reinterpret_cast<uint16_t*>(row)[c + i] = uint16_t(w);
  else reinterpret_cast<uint8_t*>(row)[c + i] = uint8_t(w);
}

// Stores columns c ... c + 7 as far as they lie below `cols` (for a lane without a unit, c >= cols).  All lanes of the warp
// call it; runs of WIDTH lanes hold neighbouring units of one row.  T is a type of 4, 2 or 1 bytes.
template <bool ALIGNED, int WIDTH, typename T>
__device__ __forceinline__ void store_raw(T* row, int c, int cols, const Raw<T>& r) {
  constexpr int NW = UNIT * sizeof(T) / 4, FRAME = NW >= 4 ? 16 : 4 * NW;      // bytes of an aligned store
  uint8_t* at = reinterpret_cast<uint8_t*>(row + c);
  if (ALIGNED) {
    if (!inside(c, cols)) return;
    if (NW == 2) {
      *reinterpret_cast<uint2*>(at) = make_uint2(r.w[0], r.w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < NW; i += 4) {
        if (i && !inside(c + 4, cols)) break;
        reinterpret_cast<uint4*>(at)[i / 4] = make_uint4(r.w[i], r.w[i + 1], r.w[i + 2], r.w[i + 3]);
      }
    }
    return;
  }
  constexpr int FW = FRAME / 4;                                   // words of a frame
  const uint32_t shift = uint32_t(reinterpret_cast<uintptr_t>(at)) & (FRAME - 1);
  const int lane = threadIdx.x & (WIDTH - 1);
  const bool full = c + UNIT <= cols;
  const unsigned fulls = __ballot_sync(0xffffffffu, full) >> ((threadIdx.x & 31) & ~(WIDTH - 1));
  const bool before = lane > 0 && (fulls >> (lane - 1) & 1u), after = lane < WIDTH - 1 && (fulls >> (lane + 1) & 1u);
  // e: the last frame of the lane before, then this lane's words; a frame to store begins `shift` bytes ahead of the unit
  uint32_t e[FW + NW];
#pragma unroll
  for (int i = 0; i < FW; ++i) e[i] = __shfl_up_sync(0xffffffffu, r.w[NW - FW + i], 1, WIDTH);
#pragma unroll
  for (int i = 0; i < NW; ++i) e[FW + i] = r.w[i];
  if (FW == 4) {
#pragma unroll
    for (int i = FW + NW - 1; i >= 2; --i) e[i] = shift & 8u ? e[i - 2] : e[i];
  }
#pragma unroll
  for (int i = FW + NW - 1; i >= 1; --i) e[i] = shift & 4u ? e[i - 1] : e[i];
  uint32_t out[NW];
#pragma unroll
  for (int i = 0; i < NW; ++i) out[i] = sizeof(T) == 4 ? e[FW + i] : __funnelshift_l(e[FW + i - 1], e[FW + i], (shift & 3u) * 8u);
  const bool first = full && (before || shift == 0);              // this lane stores its first frame as a whole
  if (NW == 2) {
    if (first) *reinterpret_cast<uint2*>(at - shift) = make_uint2(out[0], out[1]);
  } else {
#pragma unroll
    for (int i = 0; i < NW; i += 4)
      if (i ? full : first) reinterpret_cast<uint4*>(at - shift)[i / 4] = make_uint4(out[i], out[i + 1], out[i + 2], out[i + 3]);
  }
  // elements ahead of this lane's first whole frame, and those that the next lane's first frame does not take along
  const int head = int((FRAME - shift) / sizeof(T)), tail = UNIT - int(shift / sizeof(T));
#pragma unroll
  for (int i = 0; i < UNIT; ++i) {
    const bool mine = full ? (!first && i < head) || (!after && i >= tail) : c + i < cols;
    if (mine) store_element(row, c, r, i);
  }
}

// largest magnitude of the three, NaN if one is
__device__ __forceinline__ float max_magnitude(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Scale code of a block from the bits of its largest magnitude (a NaN or an infinity lies on top).
template <int FORMAT>
__device__ __forceinline__ uint32_t scale_code(uint32_t m) {
  constexpr int EMAX = FORMAT == NES_MXFP4 ? 2 : 8;
  return m >= 0x7f800000u ? 255u : uint32_t(max(int(m >> 23) - EMAX, 0));
}

// Kernels of a chain are started while the one before still runs, and wait for it before they touch memory: what is saved is the
// launch and the set-up, a microsecond or two of the few that calls on few rows take.  take_turn() waits until the kernel
// before has ended and its writes can be seen, and only then lets the next one start: what a kernel finds done when it starts
// is everything but the kernel just before it.
__device__ __forceinline__ void wait_for_kernel_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void take_turn() {
  wait_for_kernel_before();
  let_next_start();
}

// Launches a kernel that takes its turn as above; an error is left to check_launch.
template <typename... P, typename... A>
inline void launch_in_turn(void (*kernel)(P...), unsigned grid, unsigned threads, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, P(args)...);
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
__device__ __forceinline__ uint32_t pack_e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) { return pack_e4m3x2(a, b) | (pack_e4m3x2(c, d) << 16); }

// Codes (4 or, in x and y, 8 bytes) and scale of this lane's unit of a block that four neighbouring lanes hold; all lanes of the
// warp call it.
template <int FORMAT>
__device__ __forceinline__ uint2 encode_unit(float (&v)[UNIT], uint32_t& code) {
  const float top = max_magnitude(max_magnitude(v[0], v[1], v[2]), max_magnitude(v[3], v[4], v[5]), max_magnitude(v[6], v[7], v[7]));
  uint32_t m = __float_as_uint(top) & 0x7fffffffu;
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  code = scale_code<FORMAT>(m);
  const float inv = inverse_scale(code);
#pragma unroll
  for (int i = 0; i < UNIT; ++i) v[i] *= inv;
  uint2 q;
  if (FORMAT == NES_MXFP4) q = make_uint2(pack_e2m1x8(v), 0u);
  else q = make_uint2(pack_e4m3x4(v[0], v[1], v[2], v[3]), pack_e4m3x4(v[4], v[5], v[6], v[7]));
  if (code == 255u) q = make_uint2(0u, 0u);
  return q;
}

// The same, stored: codes and, from the block's first lane, the scale.  unit: index within the row, or within the whole tensor
// with its first code and scale (rows are padded to whole groups); `store` is false for lanes without one.
template <int FORMAT, typename I>
__device__ __forceinline__ void quantize_unit(float (&v)[UNIT], uint8_t* codes_row, uint8_t* scales_row, I unit, bool store) {
  uint32_t code;
  const uint2 q = encode_unit<FORMAT>(v, code);
  if (!store) return;
  if (FORMAT == NES_MXFP4) reinterpret_cast<uint32_t*>(codes_row)[unit] = q.x;
  else reinterpret_cast<uint2*>(codes_row)[unit] = q;
  if ((unit & 3) == 0) scales_row[unit >> 2] = uint8_t(code);
}

// e4m3 bytes of four e2m1 codes (the low 16 bits of c): a byte look-up in the eight magnitudes, and one that fills a byte
// with its top bit where a code's fourth bit is set (0xff, else 0x80), whose lowest bit is then the sign
__device__ __forceinline__ uint32_t e2m1x4_to_e4m3(uint32_t c) {
  const uint32_t magnitude = __byte_perm(0x3c383000u, 0x4c484440u, c & 0x7777u);   // 0 .5 1 1.5 | 2 3 4 6
  uint32_t filled;
  asm("prmt.b32 %0, %1, %1, %2;" : "=r"(filled) : "r"(0x80808080u), "r"(c));
  return magnitude | ((filled << 7) & 0x80808080u);
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
  if (FORMAT == NES_MXFP8) return fetch(reinterpret_cast<const uint2*>(codes_row) + unit);
  const uint32_t c = fetch(reinterpret_cast<const uint32_t*>(codes_row) + unit);
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
