// Quantisation to microscaled blocks and back (microscale.cuh has the format).
//
// All kernels stream: every input byte is read once, every output byte written once.  Rows of whole 16-byte pieces: a
// thread holds units of eight consecutive elements and a block is the four neighbouring lanes of a quad, so the block
// maximum costs two shuffles and no shared memory; IN_FLIGHT units are loaded before the first is worked on, since one
// 16-byte load per thread does not cover the memory's latency.  Other rows: one lane per column (stripes).
#include <type_traits>
#include "microscale.cuh"

namespace nes {
namespace mx {

constexpr int THREADS = 256;

// Walks 128-element groups of all rows: `first` .. by a stride that is kept as (rows, groups), so that no trip divides.
struct Walk { int64_t rows, groups, step_rows, step_groups; };   // groups: per row
struct Place {
  int64_t row, group;
  __device__ Place(const Walk& w, int64_t first) : row(first / w.groups), group(0) { group = first - row * w.groups; }
  __device__ __forceinline__ void next(const Walk& w) {
    row += w.step_rows;
    group += w.step_groups;
    if (group >= w.groups) { group -= w.groups; ++row; }
  }
};

template <typename T> __host__ __device__ constexpr int in_flight() { return sizeof(T) == 4 ? 2 : 4; }

// half-warps own groups (16 units), so a quad never straddles a row
template <typename T, int FORMAT>
__global__ void __launch_bounds__(THREADS) quantize_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                           int64_t cols, int64_t pitch, int64_t spitch, Walk w) {
  Place at(w, (int64_t(blockIdx.x) * THREADS + threadIdx.x) >> 4);
  const int lane16 = threadIdx.x & 15;
  constexpr int N = in_flight<T>();
  // the two half-warps of a warp may differ by one trip: both run until the first one's row is past the end
  while (__any_sync(0xffffffffu, at.row < w.rows)) {
    float v[N][UNIT];
    int64_t row[N], unit[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      row[u] = at.row;
      unit[u] = at.group * 16 + lane16;
      load_unit(x + row[u] * cols, row[u] < w.rows ? unit[u] * UNIT : cols, cols, v[u]);
      at.next(w);
    }
#pragma unroll
    for (int u = 0; u < N; ++u) quantize_unit<FORMAT>(v[u], codes + row[u] * pitch, scales + row[u] * spitch, unit[u], row[u] < w.rows);
  }
}

// warps own groups: four blocks, one lane per column
template <typename T, int FORMAT>
__global__ void __launch_bounds__(THREADS) quantize_stripes_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                   int64_t cols, int64_t pitch, int64_t spitch, Walk w) {
  const int lane = threadIdx.x & 31;
  for (Place at(w, (int64_t(blockIdx.x) * THREADS + threadIdx.x) >> 5); at.row < w.rows;) {
    float v[2][4];
    int64_t row[2], group[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      row[u] = at.row;
      group[u] = at.group;
      load_stripes(x + row[u] * cols, row[u] < w.rows ? group[u] * GROUP + lane : cols, cols, v[u]);
      at.next(w);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (row[u] < w.rows) quantize_stripes<FORMAT>(v[u], codes + row[u] * pitch, scales + row[u] * spitch, group[u] * 4, w.groups * 4, lane);
  }
}

template <typename T, int FORMAT>
__global__ void __launch_bounds__(THREADS) dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ y,
                                                             int64_t cols, int64_t pitch, int64_t spitch, Walk w) {
  const int lane16 = threadIdx.x & 15;
  for (Place at(w, (int64_t(blockIdx.x) * THREADS + threadIdx.x) >> 4); at.row < w.rows;) {
    constexpr int N = 4;
    uint2 q[N];
    uint32_t s[N];
    int64_t row[N], unit[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      row[u] = at.row;
      unit[u] = at.group * 16 + lane16;
      if (row[u] < w.rows) {
        q[u] = load_codes<FORMAT>(codes + row[u] * pitch, unit[u]);
        s[u] = __ldg(scales + row[u] * spitch + (unit[u] >> 2));
      }
      at.next(w);
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (row[u] >= w.rows) continue;
      float v[UNIT];
      unit_elements(q[u], v);
      const float scale = scale_value(s[u]);
#pragma unroll
      for (int i = 0; i < UNIT; ++i) v[i] *= scale;
      store_unit(y + row[u] * cols, unit[u] * UNIT, cols, v);
    }
  }
}

// one e2m1 code of a row as an e4m3 byte
__device__ __forceinline__ uint32_t element_byte(const uint8_t* codes_row, int64_t c) {
  return e2m1x4_to_e4m3(uint32_t(__ldg(codes_row + (c >> 1))) >> (4 * (c & 1))) & 0xffu;
}

template <typename T, int FORMAT>
__global__ void __launch_bounds__(THREADS) dequantize_stripes_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                     T* __restrict__ y, int64_t cols, int64_t pitch, int64_t spitch, Walk w) {
  const int lane = threadIdx.x & 31;
  for (Place at(w, (int64_t(blockIdx.x) * THREADS + threadIdx.x) >> 5); at.row < w.rows; at.next(w)) {
    const uint8_t* codes_row = codes + at.row * pitch;
    const uint32_t scale4 = __ldg(reinterpret_cast<const uint32_t*>(scales + at.row * spitch) + at.group);
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t c = at.group * GROUP + i * 32 + lane;              // inside the padded row
      const uint32_t e = FORMAT == NES_MXFP4 ? element_byte(codes_row, c) : uint32_t(__ldg(codes_row + c));
      v[i] = e4m3x2_to_float(e).x * scale_value((scale4 >> (8 * i)) & 0xffu);
    }
    store_stripes(y + at.row * cols, at.group * GROUP + lane, cols, v);
  }
}

// e2m1 codes -> e4m3 bytes of the same values, without the padding
__global__ void __launch_bounds__(THREADS) elements_kernel(const uint8_t* __restrict__ codes, uint8_t* __restrict__ y, int64_t cols, int64_t pitch,
                                                           Walk w) {
  const int lane16 = threadIdx.x & 15;
  for (Place at(w, (int64_t(blockIdx.x) * THREADS + threadIdx.x) >> 4); at.row < w.rows;) {
    constexpr int N = 4;
    uint32_t q[N];
    int64_t row[N], unit[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      row[u] = at.row;
      unit[u] = at.group * 16 + lane16;
      if (row[u] < w.rows) q[u] = __ldg(reinterpret_cast<const uint32_t*>(codes + row[u] * pitch) + unit[u]);
      at.next(w);
    }
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (row[u] < w.rows && unit[u] * UNIT < cols)
        *reinterpret_cast<uint2*>(y + row[u] * cols + unit[u] * UNIT) = make_uint2(e2m1x4_to_e4m3(q[u]), e2m1x4_to_e4m3(q[u] >> 16));
  }
}
__global__ void __launch_bounds__(THREADS) elements_stripes_kernel(const uint8_t* __restrict__ codes, uint8_t* __restrict__ y, int64_t cols,
                                                                   int64_t pitch, Walk w) {
  const int lane = threadIdx.x & 31;
  for (Place at(w, (int64_t(blockIdx.x) * THREADS + threadIdx.x) >> 5); at.row < w.rows; at.next(w)) {
    uint32_t e[4];
    const int64_t c = at.group * GROUP + lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = element_byte(codes + at.row * pitch, c + i * 32);
#pragma unroll
    for (int i = 0; i < 4; ++i) if (c + i * 32 < cols) y[at.row * cols + c + i * 32] = uint8_t(e[i]);
  }
}

// per_block: groups that a block takes in one trip
static Walk plan(int64_t rows, int64_t cols, int64_t per_block, unsigned* grid) {
  const int64_t groups = padded(cols) / GROUP, total = rows * groups;
  int64_t blocks = ceil_div<int64_t>(total, per_block);
  const int64_t most = int64_t(sm_count()) * 8;
  if (blocks > most) blocks = most;
  *grid = unsigned(blocks);
  const int64_t step = blocks * per_block;
  return Walk{rows, groups, step / groups, step % groups};
}

template <typename T, int FORMAT>
static void launch_quantize(const void* x, void* codes, uint8_t* scales, int64_t rows, int64_t cols, cudaStream_t st) {
  const int64_t pitch = code_pitch(cols, FORMAT), spitch = scale_pitch(cols);
  unsigned grid;
  if (aligned16(x) && (cols * sizeof(T)) % 16 == 0) {
    const Walk w = plan(rows, cols, THREADS / 16, &grid);
    quantize_kernel<T, FORMAT><<<grid, THREADS, 0, st>>>(static_cast<const T*>(x), static_cast<uint8_t*>(codes), scales, cols, pitch, spitch, w);
  } else {
    const Walk w = plan(rows, cols, THREADS / 32, &grid);
    quantize_stripes_kernel<T, FORMAT><<<grid, THREADS, 0, st>>>(static_cast<const T*>(x), static_cast<uint8_t*>(codes), scales, cols, pitch, spitch, w);
  }
}

template <typename T, int FORMAT>
static void launch_dequantize(const void* codes, const uint8_t* scales, void* y, int64_t rows, int64_t cols, cudaStream_t st) {
  const int64_t pitch = code_pitch(cols, FORMAT), spitch = scale_pitch(cols);
  unsigned grid;
  if (aligned16(y) && (cols * sizeof(T)) % 16 == 0) {
    const Walk w = plan(rows, cols, THREADS / 16, &grid);
    dequantize_kernel<T, FORMAT><<<grid, THREADS, 0, st>>>(static_cast<const uint8_t*>(codes), scales, static_cast<T*>(y), cols, pitch, spitch, w);
  } else {
    const Walk w = plan(rows, cols, THREADS / 32, &grid);
    dequantize_stripes_kernel<T, FORMAT><<<grid, THREADS, 0, st>>>(static_cast<const uint8_t*>(codes), scales, static_cast<T*>(y), cols, pitch, spitch, w);
  }
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
  const bool four = format == NES_MXFP4;
  if (dtype == NES_F32) (four ? launch_quantize<float, NES_MXFP4> : launch_quantize<float, NES_MXFP8>)(x, codes, scales, rows, cols, st);
  else if (dtype == NES_BF16) (four ? launch_quantize<__nv_bfloat16, NES_MXFP4> : launch_quantize<__nv_bfloat16, NES_MXFP8>)(x, codes, scales, rows, cols, st);
  else (four ? launch_quantize<__half, NES_MXFP4> : launch_quantize<__half, NES_MXFP8>)(x, codes, scales, rows, cols, st);
  return check_launch("mx_quantize");
}

extern "C" int nes_mx_dequantize(const void* codes, const uint8_t* scales, void* y, int dtype, int64_t rows, int64_t cols, int format,
                                 nes_stream_t stream) {
  NES_REQUIRE(rows >= 0 && cols >= 0, NES_ERR_BAD_ARG, "mx_dequantize: negative extent");
  NES_REQUIRE(known_format(format) && known_dtype(dtype), NES_ERR_UNSUPPORTED, "mx_dequantize: unknown format or dtype");
  if (rows == 0 || cols == 0) return NES_OK;
  NES_REQUIRE(codes && scales && y, NES_ERR_BAD_ARG, "mx_dequantize: null pointer");
  NES_REQUIRE(aligned16(codes) && (reinterpret_cast<uintptr_t>(scales) & 3u) == 0, NES_ERR_BAD_ARG,
              "mx_dequantize: codes must be 16-byte and scales 4-byte aligned");
  cudaStream_t st = as_stream(stream);
  const bool four = format == NES_MXFP4;
  if (dtype == NES_F32) (four ? launch_dequantize<float, NES_MXFP4> : launch_dequantize<float, NES_MXFP8>)(codes, scales, y, rows, cols, st);
  else if (dtype == NES_BF16) (four ? launch_dequantize<__nv_bfloat16, NES_MXFP4> : launch_dequantize<__nv_bfloat16, NES_MXFP8>)(codes, scales, y, rows, cols, st);
  else (four ? launch_dequantize<__half, NES_MXFP4> : launch_dequantize<__half, NES_MXFP8>)(codes, scales, y, rows, cols, st);
  return check_launch("mx_dequantize");
}

extern "C" int nes_mx_elements(const void* codes, uint8_t* y, int64_t rows, int64_t cols, nes_stream_t stream) {
  NES_REQUIRE(rows >= 0 && cols >= 0, NES_ERR_BAD_ARG, "mx_elements: negative extent");
  if (rows == 0 || cols == 0) return NES_OK;
  NES_REQUIRE(codes && y, NES_ERR_BAD_ARG, "mx_elements: null pointer");
  NES_REQUIRE(aligned16(codes), NES_ERR_BAD_ARG, "mx_elements: codes must be 16-byte aligned");
  unsigned grid;
  const int64_t pitch = code_pitch(cols, NES_MXFP4);
  if ((reinterpret_cast<uintptr_t>(y) & 7u) == 0 && cols % UNIT == 0) {
    const Walk w = plan(rows, cols, THREADS / 16, &grid);
    elements_kernel<<<grid, THREADS, 0, as_stream(stream)>>>(static_cast<const uint8_t*>(codes), y, cols, pitch, w);
  } else {
    const Walk w = plan(rows, cols, THREADS / 32, &grid);
    elements_stripes_kernel<<<grid, THREADS, 0, as_stream(stream)>>>(static_cast<const uint8_t*>(codes), y, cols, pitch, w);
  }
  return check_launch("mx_elements");
}
