// Quantisation to microscaled blocks and back (microscale.cuh has the format).
//
// All kernels stream: every input byte is read once, every output byte written once.  A thread holds units of eight
// consecutive elements and a block is the four neighbouring lanes of a quad, so the block maximum costs two shuffles and
// no shared memory; IN_FLIGHT units are loaded before the first is worked on, since one 16-byte load per thread does not
// cover the memory's latency.  With 16-bit inputs the kernels are near the ALU pipe's rate as well as the memory's.
#include <algorithm>
#include <type_traits>
#include "microscale.cuh"

namespace nes {
namespace mx {

constexpr int THREADS = 256;
constexpr int IN_FLIGHT = 4;

// Half-warps own 128-element groups (16 units), so a quad never straddles a row, and walk them in steps of the grid's.  Codes
// and scales follow one another without gaps, a group's at its index; the place of its columns in a plain row is kept
// as (row, group of the row), so that no trip divides.
struct Walk { int64_t total, step; int groups, step_rows, step_groups; };
struct Place {
  int64_t index;
  int row, group;
  __device__ Place(const Walk& w) : index((int64_t(blockIdx.x) * THREADS + threadIdx.x) >> 4) {
    row = int(index / w.groups);
    group = int(index - int64_t(row) * w.groups);
  }
  __device__ __forceinline__ void next(const Walk& w) {
    index += w.step;
    row += w.step_rows;
    group += w.step_groups;
    if (group >= w.groups) { group -= w.groups; ++row; }
  }
};

// Rows of whole groups have no padding: the plain matrix is one row of groups.
template <typename T, int FORMAT>
__global__ void __launch_bounds__(THREADS) quantize_groups_kernel(const T* x, uint8_t* codes, uint8_t* scales,
                                                                  int64_t total, int64_t step) {
  take_turn();
  const int lane16 = threadIdx.x & 15;
  int64_t index = (int64_t(blockIdx.x) * THREADS + threadIdx.x) >> 4;
  for (; index + (IN_FLIGHT - 1) * step < (total & ~int64_t(1)); index += IN_FLIGHT * step) {        // both half-warps, all units
    Raw<T> raw[IN_FLIGHT];
    const T* at = x + (index * GROUP + lane16 * UNIT);
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) raw[u] = load_raw<true>(at + u * step * GROUP, 0, NO_END, Span());
    const int64_t unit = index * (GROUP / UNIT) + lane16;
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) {
      float v[UNIT];
      raw_values(raw[u], v);
      quantize_unit<FORMAT>(v, codes, scales, unit + u * step * (GROUP / UNIT), true);
    }
  }
  while (__any_sync(0xffffffffu, index < total)) {
    float v[UNIT];
    raw_values(load_raw<true>(x + index * GROUP, index < total ? lane16 * UNIT : GROUP, GROUP, Span()), v);
    quantize_unit<FORMAT>(v, codes, scales, index * (GROUP / UNIT) + lane16, index < total);
    index += step;
  }
}

template <typename T, int FORMAT, bool ALIGNED>
__global__ void __launch_bounds__(THREADS) quantize_kernel(const T* x, uint8_t* codes, uint8_t* scales,
                                                           int cols, Span span, Walk w) {
  take_turn();
  Place at(w);
  const int lane16 = threadIdx.x & 15;
  // the two half-warps of a warp may differ by one trip: both run until the first one is past the end
  while (__any_sync(0xffffffffu, at.index < w.total)) {
    Raw<T> raw[IN_FLIGHT];
    const int64_t first = at.index;
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) {
      raw[u] = load_raw<ALIGNED>(x + int64_t(at.row) * cols, at.index < w.total ? at.group * GROUP + lane16 * UNIT : cols, cols, span);
      at.next(w);
    }
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) {
      float v[UNIT];
      raw_values(raw[u], v);
      const int64_t index = first + u * w.step;
      quantize_unit<FORMAT>(v, codes, scales, index * (GROUP / UNIT) + lane16, index < w.total);
    }
  }
}

template <typename T, int FORMAT, bool ALIGNED>
__global__ void __launch_bounds__(THREADS) dequantize_kernel(const uint8_t* codes, const uint8_t* scales, T* y,
                                                             int cols, Walk w) {
  take_turn();
  Place at(w);
  const int lane16 = threadIdx.x & 15;
  while (__any_sync(0xffffffffu, at.index < w.total)) {
    uint2 q[IN_FLIGHT];
    uint32_t s[IN_FLIGHT];
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) {
      const int64_t index = at.index + u * w.step, unit = index * (GROUP / UNIT) + lane16;
      q[u] = make_uint2(0u, 0u);
      s[u] = 0;
      if (index < w.total) {
        q[u] = load_codes<FORMAT>(codes, unit);
        s[u] = fetch(scales + (unit >> 2));
      }
    }
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) {
      float v[UNIT];
      unit_elements(q[u], v);
      const float scale = scale_value(s[u]);
#pragma unroll
      for (int i = 0; i < UNIT; ++i) v[i] *= scale;
      store_raw<ALIGNED, 16>(y + int64_t(at.row) * cols, at.index < w.total ? at.group * GROUP + lane16 * UNIT : cols, cols, values_raw(v, T()));
      at.next(w);
    }
  }
}

// e2m1 codes -> e4m3 bytes of the same values, where there is no padding: 16 codes of 8 bytes at a time
__global__ void __launch_bounds__(THREADS) elements_groups_kernel(const uint2* codes, uint4* y, int64_t total) {
  take_turn();
  const int64_t step = int64_t(gridDim.x) * THREADS;
  for (int64_t i = int64_t(blockIdx.x) * THREADS + threadIdx.x; i < total; i += IN_FLIGHT * step) {
    uint2 q[IN_FLIGHT];
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) if (i + u * step < total) q[u] = fetch(codes + i + u * step);
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u)
      if (i + u * step < total)
        y[i + u * step] = make_uint4(e2m1x4_to_e4m3(q[u].x), e2m1x4_to_e4m3(q[u].x >> 16), e2m1x4_to_e4m3(q[u].y), e2m1x4_to_e4m3(q[u].y >> 16));
  }
}

// e2m1 codes -> e4m3 bytes of the same values, without the padding
template <bool ALIGNED>
__global__ void __launch_bounds__(THREADS) elements_kernel(const uint8_t* codes, uint8_t* y, int cols, Walk w) {
  take_turn();
  Place at(w);
  const int lane16 = threadIdx.x & 15;
  while (__any_sync(0xffffffffu, at.index < w.total)) {
    uint2 q[IN_FLIGHT];
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) {
      const int64_t index = at.index + u * w.step;
      q[u] = index < w.total ? load_codes<NES_MXFP4>(codes, index * (GROUP / UNIT) + lane16) : make_uint2(0u, 0u);
    }
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) {
      Raw<uint8_t> r;
      r.w[0] = q[u].x;
      r.w[1] = q[u].y;
      store_raw<ALIGNED, 16>(y + int64_t(at.row) * cols, at.index < w.total ? at.group * GROUP + lane16 * UNIT : cols, cols, r);
      at.next(w);
    }
  }
}

static Walk plan(int64_t rows, int64_t cols, unsigned* grid) {
  const int64_t groups = padded(cols) / GROUP, total = rows * groups, per_block = THREADS / 16;
  int64_t blocks = ceil_div<int64_t>(total, per_block);
  const int64_t most = int64_t(sm_count()) * 8;
  if (blocks > most) blocks = most;
  *grid = unsigned(blocks);
  const int64_t step = blocks * per_block;
  return Walk{total, step, int(groups), int(step / groups), int(step % groups)};
}

template <typename T, int FORMAT>
static void launch_quantize(const void* x, void* codes, uint8_t* scales, int64_t rows, int64_t cols, cudaStream_t st) {
  unsigned grid;
  const Walk w = plan(rows, cols, &grid);
  const T* in = static_cast<const T*>(x);
  const Span span = {static_cast<const uint8_t*>(x), reinterpret_cast<const uint8_t*>(in + rows * cols)};
  uint8_t* out = static_cast<uint8_t*>(codes);
  if (aligned16(x) && cols % GROUP == 0) launch_in_turn(quantize_groups_kernel<T, FORMAT>, grid, THREADS, st, in, out, scales, w.total, w.step);
  else if (aligned16(x) && (cols * sizeof(T)) % 16 == 0) launch_in_turn(quantize_kernel<T, FORMAT, true>, grid, THREADS, st, in, out, scales, int(cols), span, w);
  else launch_in_turn(quantize_kernel<T, FORMAT, false>, grid, THREADS, st, in, out, scales, int(cols), span, w);
}

template <typename T, int FORMAT>
static void launch_dequantize(const void* codes, const uint8_t* scales, void* y, int64_t rows, int64_t cols, cudaStream_t st) {
  unsigned grid;
  const Walk w = plan(rows, cols, &grid);
  const uint8_t* in = static_cast<const uint8_t*>(codes);
  T* out = static_cast<T*>(y);
  if (aligned16(y) && (cols * sizeof(T)) % 16 == 0) launch_in_turn(dequantize_kernel<T, FORMAT, true>, grid, THREADS, st, in, scales, out, int(cols), w);
  else launch_in_turn(dequantize_kernel<T, FORMAT, false>, grid, THREADS, st, in, scales, out, int(cols), w);
}

}  // namespace mx
}  // namespace nes

using namespace nes;
using namespace nes::mx;

extern "C" int nes_mx_quantize(const void* x, int dtype, void* codes, uint8_t* scales, int64_t rows, int64_t cols, int format,
                               nes_stream_t stream) {
  NES_REQUIRE(rows >= 0 && cols >= 0, NES_ERR_BAD_ARG, "mx_quantize: negative extent");
  NES_REQUIRE(rows <= LARGEST_EXTENT && cols <= LARGEST_EXTENT, NES_ERR_UNSUPPORTED, "mx_quantize: too large");
  NES_REQUIRE(known_format(format) && known_dtype(dtype), NES_ERR_UNSUPPORTED, "mx_quantize: unknown format or dtype");
  if (rows == 0 || cols == 0) return NES_OK;
  NES_REQUIRE(x && codes && scales, NES_ERR_BAD_ARG, "mx_quantize: null pointer");
  NES_REQUIRE(aligned16(codes), NES_ERR_BAD_ARG, "mx_quantize: codes must be 16-byte aligned");
  const Bytes outputs[] = {{codes, rows * code_pitch(cols, format)}, {scales, rows * scale_pitch(cols)}}, inputs[] = {{x, rows * cols * dtype_bytes(dtype)}};
  NES_REQUIRE(!overlap(outputs, inputs), NES_ERR_BAD_ARG, "mx_quantize: the outputs overlap the input or one another");
  cudaStream_t st = as_stream(stream);
  const bool four = format == NES_MXFP4;
  if (dtype == NES_F32) (four ? launch_quantize<float, NES_MXFP4> : launch_quantize<float, NES_MXFP8>)(x, codes, scales, rows, cols, st);
  else if (dtype == NES_BF16) (four ? launch_quantize<__nv_bfloat16, NES_MXFP4> : launch_quantize<__nv_bfloat16, NES_MXFP8>)(x, codes, scales, rows, cols, st);
  else (four ? launch_quantize<__half, NES_MXFP4> : launch_quantize<__half, NES_MXFP8>)(x, codes, scales, rows, cols, st);
  return check_launch("mx_quantize");
}

extern "C" int nes_mx_dequantize(const void* codes, const uint8_t* scales, void* y, int dtype, int64_t rows, int64_t cols, int format,
                                 nes_stream_t stream) {
  NES_REQUIRE(rows >= 0 && cols >= 0, NES_ERR_BAD_ARG, "mx_dequantize: negative extent");
  NES_REQUIRE(rows <= LARGEST_EXTENT && cols <= LARGEST_EXTENT, NES_ERR_UNSUPPORTED, "mx_dequantize: too large");
  NES_REQUIRE(known_format(format) && known_dtype(dtype), NES_ERR_UNSUPPORTED, "mx_dequantize: unknown format or dtype");
  if (rows == 0 || cols == 0) return NES_OK;
  NES_REQUIRE(codes && scales && y, NES_ERR_BAD_ARG, "mx_dequantize: null pointer");
  NES_REQUIRE(aligned16(codes), NES_ERR_BAD_ARG, "mx_dequantize: codes must be 16-byte aligned");
  const Bytes outputs[] = {{y, rows * cols * dtype_bytes(dtype)}}, inputs[] = {{codes, rows * code_pitch(cols, format)}, {scales, rows * scale_pitch(cols)}};
  NES_REQUIRE(!overlap(outputs, inputs), NES_ERR_BAD_ARG, "mx_dequantize: the output overlaps an input");
  cudaStream_t st = as_stream(stream);
  const bool four = format == NES_MXFP4;
  if (dtype == NES_F32) (four ? launch_dequantize<float, NES_MXFP4> : launch_dequantize<float, NES_MXFP8>)(codes, scales, y, rows, cols, st);
  else if (dtype == NES_BF16) (four ? launch_dequantize<__nv_bfloat16, NES_MXFP4> : launch_dequantize<__nv_bfloat16, NES_MXFP8>)(codes, scales, y, rows, cols, st);
  else (four ? launch_dequantize<__half, NES_MXFP4> : launch_dequantize<__half, NES_MXFP8>)(codes, scales, y, rows, cols, st);
  return check_launch("mx_dequantize");
}

extern "C" int nes_mx_elements(const void* codes, uint8_t* y, int64_t rows, int64_t cols, nes_stream_t stream) {
  NES_REQUIRE(rows >= 0 && cols >= 0, NES_ERR_BAD_ARG, "mx_elements: negative extent");
  NES_REQUIRE(rows <= LARGEST_EXTENT && cols <= LARGEST_EXTENT, NES_ERR_UNSUPPORTED, "mx_elements: too large");
  if (rows == 0 || cols == 0) return NES_OK;
  NES_REQUIRE(codes && y, NES_ERR_BAD_ARG, "mx_elements: null pointer");
  NES_REQUIRE(aligned16(codes), NES_ERR_BAD_ARG, "mx_elements: codes must be 16-byte aligned");
  NES_REQUIRE(!overlap(Bytes{y, rows * cols}, Bytes{codes, rows * code_pitch(cols, NES_MXFP4)}), NES_ERR_BAD_ARG, "mx_elements: the output overlaps the input");
  unsigned grid;
  const Walk w = plan(rows, cols, &grid);
  const uint8_t* in = static_cast<const uint8_t*>(codes);
  if (aligned16(y) && cols % GROUP == 0) {
    const int64_t total = rows * cols / 16;
    const int64_t blocks = std::min<int64_t>(ceil_div<int64_t>(total, THREADS), int64_t(sm_count()) * 8);
    launch_in_turn(elements_groups_kernel, unsigned(blocks), THREADS, as_stream(stream), static_cast<const uint2*>(codes), reinterpret_cast<uint4*>(y), total);
  } else if ((reinterpret_cast<uintptr_t>(y) & 7u) == 0 && cols % UNIT == 0) launch_in_turn(elements_kernel<true>, grid, THREADS, as_stream(stream), in, y, int(cols), w);
  else launch_in_turn(elements_kernel<false>, grid, THREADS, as_stream(stream), in, y, int(cols), w);
  return check_launch("mx_elements");
}
