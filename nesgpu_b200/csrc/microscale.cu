// Quantisation to microscaled blocks and back (microscale.cuh has the format).
//
// All three kernels stream: every input byte is read once, every output byte written once, a thread handles units of
// eight consecutive elements and a block of 32 is the four neighbouring lanes of a quad, so the block maximum costs two
// shuffles and no shared memory.
#include <type_traits>
#include "microscale.cuh"

namespace nes {
namespace mx {

constexpr int THREADS = 256;

// Walks the units of all rows: half-warps own 128-element groups (16 units), so a quad never straddles a row.
struct Walk { int64_t rows, groups, step_rows, step_groups; };   // groups per row; the grid's stride split by division

template <typename T, int FORMAT>
__global__ void __launch_bounds__(THREADS) quantize_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                           int64_t cols, int64_t pitch, int64_t spitch, Walk w, bool vec) {
  const int64_t first = (int64_t(blockIdx.x) * THREADS + threadIdx.x) >> 4;
  int64_t row = first / w.groups, group = first - row * w.groups;
  const int lane16 = threadIdx.x & 15;
  // the two half-warps of a warp may differ by one trip: both run until the first one's row is past the end
  while (__any_sync(0xffffffffu, row < w.rows)) {
    const bool on = row < w.rows;
    const int64_t unit = group * 16 + lane16;
    float v[UNIT];
    if (on) {
      load_unit(x + row * cols, unit * UNIT, cols, vec, v);
    } else {
#pragma unroll
      for (int i = 0; i < UNIT; ++i) v[i] = 0.f;
    }
    quantize_unit<FORMAT>(v, codes + row * pitch, scales + row * spitch, unit, on);
    row += w.step_rows;
    group += w.step_groups;
    if (group >= w.groups) { group -= w.groups; ++row; }
  }
}

template <typename T, int FORMAT>
__global__ void __launch_bounds__(THREADS) dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ y,
                                                             int64_t cols, int64_t pitch, int64_t spitch, Walk w, bool vec) {
  const int64_t first = (int64_t(blockIdx.x) * THREADS + threadIdx.x) >> 4;
  int64_t row = first / w.groups, group = first - row * w.groups;
  const int lane16 = threadIdx.x & 15;
  while (row < w.rows) {
    const int64_t unit = group * 16 + lane16;
    float v[UNIT];
    unit_elements<FORMAT>(codes + row * pitch, unit, v);
    const float s = scale_value(__ldg(scales + row * spitch + (unit >> 2)));
#pragma unroll
    for (int i = 0; i < UNIT; ++i) v[i] *= s;
    store_unit(y + row * cols, unit * UNIT, cols, vec, v);
    row += w.step_rows;
    group += w.step_groups;
    if (group >= w.groups) { group -= w.groups; ++row; }
  }
}

// e2m1 codes -> e4m3 bytes of the same values, without the padding
__global__ void __launch_bounds__(THREADS) elements_kernel(const uint8_t* __restrict__ codes, uint8_t* __restrict__ y, int64_t cols, int64_t pitch,
                                                           Walk w, bool vec) {
  const int64_t first = (int64_t(blockIdx.x) * THREADS + threadIdx.x) >> 4;
  int64_t row = first / w.groups, group = first - row * w.groups;
  const int lane16 = threadIdx.x & 15;
  while (row < w.rows) {
    const int64_t unit = group * 16 + lane16, c = unit * UNIT;
    const uint32_t q = __ldg(reinterpret_cast<const uint32_t*>(codes + row * pitch) + unit);
    const uint2 e = make_uint2(e2m1x4_to_e4m3(q), e2m1x4_to_e4m3(q >> 16));
    uint8_t* out = y + row * cols;
    if (vec && c + UNIT <= cols) {
      *reinterpret_cast<uint2*>(out + c) = e;
    } else {
#pragma unroll
      for (int i = 0; i < UNIT; ++i) if (c + i < cols) out[c + i] = uint8_t((i < 4 ? e.x : e.y) >> (8 * (i & 3)));
    }
    row += w.step_rows;
    group += w.step_groups;
    if (group >= w.groups) { group -= w.groups; ++row; }
  }
}

static Walk plan(int64_t rows, int64_t cols, unsigned* grid) {
  const int64_t groups = padded(cols) / GROUP, total = rows * groups, per_block = THREADS / 16;
  int64_t blocks = ceil_div<int64_t>(total, per_block);
  const int64_t most = int64_t(sm_count()) * 8;
  if (blocks > most) blocks = most;
  *grid = unsigned(blocks);
  const int64_t step = blocks * per_block;
  return Walk{rows, groups, step / groups, step % groups};
}

template <typename T>
static void launch_quantize(const void* x, void* codes, uint8_t* scales, int64_t rows, int64_t cols, int format, cudaStream_t st) {
  unsigned grid;
  const Walk w = plan(rows, cols, &grid);
  const bool vec = aligned16(x) && (cols * sizeof(T)) % 16 == 0;
  const int64_t pitch = code_pitch(cols, format), spitch = scale_pitch(cols);
  if (format == NES_MXFP4)
    quantize_kernel<T, NES_MXFP4><<<grid, THREADS, 0, st>>>(static_cast<const T*>(x), static_cast<uint8_t*>(codes), scales, cols, pitch, spitch, w, vec);
  else
    quantize_kernel<T, NES_MXFP8><<<grid, THREADS, 0, st>>>(static_cast<const T*>(x), static_cast<uint8_t*>(codes), scales, cols, pitch, spitch, w, vec);
}

template <typename T>
static void launch_dequantize(const void* codes, const uint8_t* scales, void* y, int64_t rows, int64_t cols, int format, cudaStream_t st) {
  unsigned grid;
  const Walk w = plan(rows, cols, &grid);
  const bool vec = aligned16(y) && (cols * sizeof(T)) % 16 == 0;
  const int64_t pitch = code_pitch(cols, format), spitch = scale_pitch(cols);
  if (format == NES_MXFP4)
    dequantize_kernel<T, NES_MXFP4><<<grid, THREADS, 0, st>>>(static_cast<const uint8_t*>(codes), scales, static_cast<T*>(y), cols, pitch, spitch, w, vec);
  else
    dequantize_kernel<T, NES_MXFP8><<<grid, THREADS, 0, st>>>(static_cast<const uint8_t*>(codes), scales, static_cast<T*>(y), cols, pitch, spitch, w, vec);
}

}  // namespace mx
}  // namespace nes

using namespace nes;
using namespace nes::mx;

extern "C" int nes_mx_quantize(const void* x, int dtype, void* codes, uint8_t* scales, int64_t rows, int64_t cols, int format,
                               nes_stream_t stream) {
  NES_REQUIRE(rows >= 0 && cols >= 0, NES_ERR_BAD_ARG, "mx_quantize: negative extent");
  NES_REQUIRE(known_format(format) && known_dtype(dtype), NES_ERR_UNSUPPORTED, "mx_quantize: unknown format or dtype");
  if (rows == 0 || cols == 0) return NES_OK;
  NES_REQUIRE(x && codes && scales, NES_ERR_BAD_ARG, "mx_quantize: null pointer");
  NES_REQUIRE(aligned16(codes), NES_ERR_BAD_ARG, "mx_quantize: codes must be 16-byte aligned");
  cudaStream_t st = as_stream(stream);
  if (dtype == NES_F32) launch_quantize<float>(x, codes, scales, rows, cols, format, st);
  else if (dtype == NES_BF16) launch_quantize<__nv_bfloat16>(x, codes, scales, rows, cols, format, st);
  else launch_quantize<__half>(x, codes, scales, rows, cols, format, st);
  return check_launch("mx_quantize");
}

extern "C" int nes_mx_dequantize(const void* codes, const uint8_t* scales, void* y, int dtype, int64_t rows, int64_t cols, int format,
                                 nes_stream_t stream) {
  NES_REQUIRE(rows >= 0 && cols >= 0, NES_ERR_BAD_ARG, "mx_dequantize: negative extent");
  NES_REQUIRE(known_format(format) && known_dtype(dtype), NES_ERR_UNSUPPORTED, "mx_dequantize: unknown format or dtype");
  if (rows == 0 || cols == 0) return NES_OK;
  NES_REQUIRE(codes && scales && y, NES_ERR_BAD_ARG, "mx_dequantize: null pointer");
  NES_REQUIRE(aligned16(codes), NES_ERR_BAD_ARG, "mx_dequantize: codes must be 16-byte aligned");
  cudaStream_t st = as_stream(stream);
  if (dtype == NES_F32) launch_dequantize<float>(codes, scales, y, rows, cols, format, st);
  else if (dtype == NES_BF16) launch_dequantize<__nv_bfloat16>(codes, scales, y, rows, cols, format, st);
  else launch_dequantize<__half>(codes, scales, y, rows, cols, format, st);
  return check_launch("mx_dequantize");
}

extern "C" int nes_mx_elements(const void* codes, uint8_t* y, int64_t rows, int64_t cols, nes_stream_t stream) {
  NES_REQUIRE(rows >= 0 && cols >= 0, NES_ERR_BAD_ARG, "mx_elements: negative extent");
  if (rows == 0 || cols == 0) return NES_OK;
  NES_REQUIRE(codes && y, NES_ERR_BAD_ARG, "mx_elements: null pointer");
  NES_REQUIRE(aligned16(codes), NES_ERR_BAD_ARG, "mx_elements: codes must be 16-byte aligned");
  unsigned grid;
  const Walk w = plan(rows, cols, &grid);
  const bool vec = aligned16(y) && cols % UNIT == 0;
  elements_kernel<<<grid, THREADS, 0, as_stream(stream)>>>(static_cast<const uint8_t*>(codes), y, cols, code_pitch(cols, NES_MXFP4), w, vec);
  return check_launch("mx_elements");
}
