// Product of microscaled operands on the tensor cores: y[t, n] = sum_k x[t, k] w[n, k] + bias[n].
//
//   * tcgen05.mma with block scales: kind::mxf4 (both operands e2m1, K = 64 per instruction) or kind::mxf8f6f4 (e4m3
//     activations with e4m3 or e2m1 weights, K = 32).  The hardware multiplies every block's partial sum by 2^(ex + ew)
//     and accumulates in fp32.
//   * The weights are the M side of the instruction: 128 output features are the lanes of the accumulator, TOKENS
//     (16 ... 128, and 256 in the pairs below) tokens its columns.  A warp that reads a column holds 32 neighbouring
//     features of one token, so the row-major output is stored in whole lines, and few tokens cost no empty rows.
//   * Codes travel by TMA as 128-byte-swizzled rows; 4-bit weights of an 8-bit product are spread by the copy itself: 16
//     elements fill the first half of 16 bytes.
//   * Scales are stored row-major (4 bytes per 128 elements); the instruction wants them in tensor memory, one 32-bit
//     column per 32 rows and 128 elements, repeated in each quarter of the lanes.  Four warps load them for STEP = 512
//     elements of K at a time, 16 bytes per row and thread, transpose them on the way into shared memory, and tcgen05.cp
//     brings them over in the order of the products.
//   * Plain activations are quantised into scratch first, under which the product starts and loads its first weights; a few
//     tokens are quantised by the product itself, every CTA its own part of K straight into the operand's place in shared memory.
//   * Few output tiles: a cluster of up to eight CTAs splits K and adds its partial tiles in a fixed order through
//     distributed shared memory.
//
// Few tokens are bound by the latencies of one load - product - store chain and then the weights' bytes: 1 token of
// 4096x4096 with 8-bit activations takes 5.9 us with the weights in the L2 cache and 6.3 us out of HBM (8.9 MB, 1.4 us), 24 tokens of
// 8192x8192 in 4 bits, quantised before, 12.1 us out of HBM (35.7 MB, 5.5 us).  Many are bound by the operands' way from L2 in 4 bits
// (9.9 TB/s at 45 % tensor activity, where the 8-bit product has the same 9.9 TB/s at 70 %) and by the power limit back to back:
// 8192x4096x16384 in 4 bits takes 254 us in a burst (4.3 PFLOP/s) and 300 us back to back at 1.64 GHz, with 8-bit activations 394
// and 472 us (2.8 and 2.3 PFLOP/s at 1.4 GHz).
#include <type_traits>
#include "microscale.cuh"
#include "tc_ptx.cuh"

namespace nes {
namespace mx {

using namespace nes::tc;

constexpr int FEATURES = 128;                // accumulator lanes
constexpr int ROW_BYTES = 128;               // one swizzle row of an operand per stage
constexpr int STEP = 512;                    // elements of K whose scales are written at once
constexpr int CHUNKS = STEP / GROUP;         // 32-bit scale words of a row per step
constexpr int SCALE_TILE = 512;              // scales of 128 rows x 128 elements in shared memory
constexpr int THREADS_TC = 192;              // warp 0: TMA, warp 1: MMA, warps 2-5: scales, then epilogue

struct Product {
  const uint8_t *x_scales, *w_scales;
  const float* bias;
  void* y;
  int M, N, K, groups;                       // tokens, features, columns and their 128-element groups
  int y_dtype, vec_scales;
  const void* x;                             // plain activations of a product that quantises them itself
  int whole_rows;                            // their rows are whole, aligned 16-byte pieces
  bool overlap;                              // the kernel before quantises the activations: the weights have been there before it
};
struct ProductMaps { CUtensorMap w, x; };

constexpr int RAW_STEPS = 8;                 // steps of K whose quantised activations a CTA keeps

// PUSH: partial results go straight to the CTA that adds them up, which has room for them beside its stages (one barrier of the
// cluster and local reads: 1 token of 4096x4096 6.6 -> 6.0 us).  Otherwise they lie in the stages until they are fetched: of
// 128 tokens the room costs two of six stages, which pays from four CTAs to a tile on (128 tokens, 4096x1024: 9.2 -> 7.0 us;
// 1024x1024 in halves: 6.9 -> 8.0 us).
// RAW: the activations of all the CTA's stages lie behind the stages, which hold weights only; so do their scales
template <int TOKENS, bool RAW, int STAGES_PER_STEP, bool PUSH>
struct Layout {
  static constexpr int W_BYTES = FEATURES * ROW_BYTES;
  static constexpr int X_BYTES = TOKENS * ROW_BYTES;
  static constexpr int STAGE = W_BYTES + (RAW ? 0 : X_BYTES);
  static constexpr int STAGES = TOKENS >= 128 ? (PUSH ? 4 : 6) : TOKENS >= 64 ? 7 : 8;
  static constexpr int X_COLS = 4;                                         // scale columns of x per 128 elements
  static constexpr int SCALE_COLS = CHUNKS * (4 + X_COLS);                 // one buffer
  static constexpr int SCALE_BASE = TOKENS < 32 ? 32 : TOKENS;
  static constexpr int USED_COLS = SCALE_BASE + 2 * SCALE_COLS;
  static constexpr int TMEM_COLS = USED_COLS <= 128 ? 128 : USED_COLS <= 256 ? 256 : 512;
  static constexpr int STEP_SCALES = CHUNKS * SCALE_TILE;                  // of one operand
  static constexpr int SCALES = (RAW ? 1 : 2) * STEP_SCALES;               // a buffer in shared memory: w, then x
  static constexpr int RAW_X = RAW ? RAW_STEPS * STAGES_PER_STEP * X_BYTES : 0;
  static constexpr int RAW_SCALES = RAW ? RAW_STEPS * STEP_SCALES : 0;
  static constexpr int PARTS = PUSH ? TOKENS * FEATURES * 4 : 0;
  static constexpr size_t SMEM = 1024 + size_t(STAGES) * STAGE + RAW_X + RAW_SCALES + 2 * SCALES + PARTS + (2 * STAGES + 6) * sizeof(uint64_t) + 16;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// Instruction descriptor with block scales: element formats at bits 7 and 10 (kind::mxf4: 1 = e2m1; kind::mxf8f6f4: 0 = e4m3,
// 5 = e2m1), N >> 3 at bit 17, scale type 1 = E8M0 at bit 23, M >> 4 at bit 24; the byte of the scale columns that an
// instruction uses is added per instruction (bits 29 for A and 4 for B).
template <int XF, int WF>
constexpr uint32_t idesc_scaled(int m, int n) {
  constexpr uint32_t a = XF == NES_MXFP4 ? 1u : WF == NES_MXFP4 ? 5u : 0u;
  constexpr uint32_t b = XF == NES_MXFP4 ? 1u : 0u;
  return (a << 7) | (b << 10) | (uint32_t(n >> 3) << 17) | (1u << 23) | (uint32_t(m >> 4) << 24);
}
__host__ __device__ constexpr uint32_t scale_byte(uint32_t id) { return (id << 29) | (id << 4); }

// The products of one stage: four instructions (two if HALF: a last stage with one 128-element group of 4-bit codes), each 32
// bytes further along the rows.  They share one elected lane and one asm block: an instruction with an election of its own takes
// 113 cycles to issue, and the widest 4-bit one 170 to run.
// kind::mxf4: two instructions per scale word (bytes 0-1 and 2-3), words sfa / sfb and sfa1 / sfb1; otherwise four.
#define NES_MX_STAGE4(GROUP, KIND, VEC)                                                              \
  asm volatile(                                                                                      \
      "{\n"                                                                                          \
      ".reg .pred p, pe, pt;\n"                                                                      \
      ".reg .b64 a1, a2, a3, x1, x2, x3;\n"                                                          \
      "elect.sync _|pe, 0xffffffff;\n"                                                               \
      "setp.ne.b32 p, %11, 0;\n"                                                                     \
      "setp.eq.b32 pt, 0, 0;\n"                                                                      \
      "add.s64 a1, %1, 2;\n"                                                                         \
      "add.s64 a2, %1, 4;\n"                                                                         \
      "add.s64 a3, %1, 6;\n"                                                                         \
      "add.s64 x1, %2, 2;\n"                                                                         \
      "add.s64 x2, %2, 4;\n"                                                                         \
      "add.s64 x3, %2, 6;\n"                                                                         \
      "@pe tcgen05.mma." GROUP "." KIND ".block_scale." VEC " [%0], %1, %2, %3, [%7], [%8], p;\n"    \
      "@pe tcgen05.mma." GROUP "." KIND ".block_scale." VEC " [%0], a1, x1, %4, [%7], [%8], pt;\n"   \
      "@pe tcgen05.mma." GROUP "." KIND ".block_scale." VEC " [%0], a2, x2, %5, [%9], [%10], pt;\n"  \
      "@pe tcgen05.mma." GROUP "." KIND ".block_scale." VEC " [%0], a3, x3, %6, [%9], [%10], pt;\n"  \
      "}\n" ::"r"(d), "l"(a), "l"(x), "r"(i0), "r"(i1), "r"(i2), "r"(i3), "r"(sfa), "r"(sfb), "r"(sfa1), "r"(sfb1), "r"(accumulate) : "memory")
#define NES_MX_STAGE2(GROUP)                                                                         \
  asm volatile(                                                                                      \
      "{\n"                                                                                          \
      ".reg .pred p, pe, pt;\n"                                                                      \
      ".reg .b64 a1, x1;\n"                                                                          \
      "elect.sync _|pe, 0xffffffff;\n"                                                               \
      "setp.ne.b32 p, %7, 0;\n"                                                                      \
      "setp.eq.b32 pt, 0, 0;\n"                                                                      \
      "add.s64 a1, %1, 2;\n"                                                                         \
      "add.s64 x1, %2, 2;\n"                                                                         \
      "@pe tcgen05.mma." GROUP ".kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n"  \
      "@pe tcgen05.mma." GROUP ".kind::mxf4.block_scale.scale_vec::2X [%0], a1, x1, %4, [%5], [%6], pt;\n" \
      "}\n" ::"r"(d), "l"(a), "l"(x), "r"(i0), "r"(i1), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory")

template <int XF, int CTAS, bool HALF = false>
__device__ __forceinline__ void warp_mma_stage(uint32_t d, uint64_t a, uint64_t x, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t sfa1,
                                               uint32_t sfb1, uint32_t accumulate) {
  constexpr bool FOUR = XF == NES_MXFP4;
  const uint32_t i0 = idesc, i1 = idesc | scale_byte(FOUR ? 2 : 1), i2 = idesc | scale_byte(FOUR ? 0 : 2), i3 = idesc | scale_byte(FOUR ? 2 : 3);
  if (HALF) {
    if (CTAS == 2) NES_MX_STAGE2("cta_group::2"); else NES_MX_STAGE2("cta_group::1");
  } else if (FOUR) {
    if (CTAS == 2) NES_MX_STAGE4("cta_group::2", "kind::mxf4", "scale_vec::2X"); else NES_MX_STAGE4("cta_group::1", "kind::mxf4", "scale_vec::2X");
  } else {
    if (CTAS == 2) NES_MX_STAGE4("cta_group::2", "kind::mxf8f6f4", "scale_vec::1X"); else NES_MX_STAGE4("cta_group::1", "kind::mxf8f6f4", "scale_vec::1X");
  }
}

// 16 scale bytes of a row from 128-element group `group` on; zeros outside the matrix
// (through the L2 cache: the activations' may have been written while this kernel ran already)
__device__ __forceinline__ uint4 load_scale_words(const uint8_t* scales, int row, int rows, int group, int groups, bool vec) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (row >= rows) return v;
  const uint32_t* p = reinterpret_cast<const uint32_t*>(scales + int64_t(row) * groups * 4) + group;
  if (vec) return __ldcg(reinterpret_cast<const uint4*>(p));
  v.x = __ldcg(p);
  if (group + 1 < groups) v.y = __ldcg(p + 1);
  if (group + 2 < groups) v.z = __ldcg(p + 2);
  if (group + 3 < groups) v.w = __ldcg(p + 3);
  return v;
}

// Scales in shared memory: one tile of 512 bytes per 128 rows and 128 elements, the word of row 32 c + l at word 4 l + c,
// which is the order in which tcgen05.cp (32 lanes x 16 bytes, repeated for the four lane quarters) makes the four
// 32-bit columns of tensor memory that an instruction reads.  Thread t of the 128 that fill a tile owns word t, so the
// stores have no bank conflicts.
__device__ __forceinline__ int scale_row(int t) { return (t & 3) * 32 + (t >> 2); }
__device__ __forceinline__ void put_scale_words(unsigned char* tiles, int t, const uint4& v) {      // CHUNKS tiles in a row
  uint32_t* w = reinterpret_cast<uint32_t*>(tiles) + t;
  w[0] = v.x;
  w[SCALE_TILE / 4] = v.y;
  w[2 * SCALE_TILE / 4] = v.z;
  w[3 * SCALE_TILE / 4] = v.w;
}
// descriptor of a scale tile: no swizzle, 8 rows x 16 bytes per core matrix, core matrices 128 bytes apart
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
  return uint64_t((saddr & 0x3FFFFu) >> 4) | (uint64_t(1) << 16) | (uint64_t(128 >> 4) << 32) | (uint64_t(1) << 46);
}
// CHUNKS tiles, `cols` columns apart in tensor memory
#define NES_MX_COPY4(GROUP)                                            \
  asm volatile(                                                        \
      "{\n"                                                            \
      ".reg .pred pe;\n"                                               \
      ".reg .b64 s1, s2, s3;\n"                                        \
      ".reg .b32 t1, t2, t3;\n"                                        \
      "elect.sync _|pe, 0xffffffff;\n"                                 \
      "add.s64 s1, %1, 32;\n"                                          \
      "add.s64 s2, %1, 64;\n"                                          \
      "add.s64 s3, %1, 96;\n"                                          \
      "add.s32 t1, %0, %2;\n"                                          \
      "add.s32 t2, t1, %2;\n"                                          \
      "add.s32 t3, t2, %2;\n"                                          \
      "@pe tcgen05.cp." GROUP ".32x128b.warpx4 [%0], %1;\n"            \
      "@pe tcgen05.cp." GROUP ".32x128b.warpx4 [t1], s1;\n"            \
      "@pe tcgen05.cp." GROUP ".32x128b.warpx4 [t2], s2;\n"            \
      "@pe tcgen05.cp." GROUP ".32x128b.warpx4 [t3], s3;\n"            \
      "}\n" ::"r"(tmem), "l"(desc), "n"(COLS) : "memory")
template <int CTAS, int COLS>
__device__ __forceinline__ void warp_copy_scales(uint32_t tmem, uint64_t desc) {
  static_assert(CHUNKS == 4 && SCALE_TILE == 512, "the copies' offsets");
  if (CTAS == 2) NES_MX_COPY4("cta_group::2"); else NES_MX_COPY4("cta_group::1");
}

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  return remote;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t remote) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster(uint32_t remote, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
}

__device__ __forceinline__ float4 four_biases(const Product& p, int n, int left) {
  float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
  if (p.bias) {
    b.x = fetch(p.bias + n);
    if (left > 1) b.y = fetch(p.bias + n + 1);
    if (left > 2) b.z = fetch(p.bias + n + 2);
    if (left > 3) b.w = fetch(p.bias + n + 3);
  }
  return b;
}

// Four neighbouring features of one token; `left` of them exist.
template <typename T>
__device__ __forceinline__ void store_four(T* y, const float4& v, int left, bool vec) {
  if (vec && left >= 4) {
    if (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(y) = v;
    } else {
      using H = typename std::conditional<sizeof(T) == 4, __half, T>::type;
      *reinterpret_cast<uint2*>(y) = make_uint2(float_to_pair(v.x, v.y, H()), float_to_pair(v.z, v.w, H()));
    }
  } else {
    if (left > 0) y[0] = from_float<T>(v.x);
    if (left > 1) y[1] = from_float<T>(v.y);
    if (left > 2) y[2] = from_float<T>(v.z);
    if (left > 3) y[3] = from_float<T>(v.w);
  }
}

// Adds the partial tiles ([token][feature] fp32 at the same shared-memory address of every CTA of the cluster) in rank
// order and stores this CTA's share of the tokens: token = rank + splits * i, four features per lane.
template <typename T>
__device__ __forceinline__ void pull_tiles(const Product& p, uint32_t part, int n0, int m0, int tokens, int rank, int splits, int warp, int lane) {
  const int n = n0 + lane * 4, left = p.N - n;
  if (left <= 0) return;
  const float4 bias = four_biases(p, n, left);
  uint32_t source[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) source[r] = r < splits ? map_rank(part, r) : 0u;
  const bool vec = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15u) == 0;
  constexpr int AT_ONCE = 4;                                     // tokens whose loads are in flight together
  for (int t0 = rank + splits * warp; t0 < tokens; t0 += splits * 4 * AT_ONCE) {
    float4 sum[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) sum[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (r >= splits) break;
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const int t = t0 + i * splits * 4;
        if (t >= tokens) continue;
        const float4 v = ld_cluster4(source[r] + uint32_t(t * FEATURES + lane * 4) * 4u);
        sum[i].x += v.x; sum[i].y += v.y; sum[i].z += v.z; sum[i].w += v.w;
      }
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int t = t0 + i * splits * 4;
      if (t >= tokens) continue;
      sum[i].x += bias.x; sum[i].y += bias.y; sum[i].z += bias.z; sum[i].w += bias.w;
      store_four(static_cast<T*>(p.y) + int64_t(m0 + t) * p.N + n, sum[i], left, vec);
    }
  }
}

// Adds the partial results of this CTA's share of the tokens (token = rank + splits * i; [source rank][i][feature] fp32 in shared
// memory) in rank order and stores them, four features per lane.
template <typename T>
__device__ __forceinline__ void join_parts(const Product& p, const float* parts, int n0, int m0, int tokens, int share, int rank, int splits,
                                           int warp, int lane) {
  const int n = n0 + lane * 4, left = p.N - n;
  if (left <= 0) return;
  const float4 bias = four_biases(p, n, left);
  const bool vec = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15u) == 0;
  for (int i = warp; rank + i * splits < tokens; i += 4) {
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r = 0; r < splits; ++r) {
      const float4 v = *reinterpret_cast<const float4*>(parts + (r * share + i) * FEATURES + lane * 4);
      sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
    }
    sum.x += bias.x; sum.y += bias.y; sum.z += bias.z; sum.w += bias.w;
    store_four(static_cast<T*>(p.y) + int64_t(m0 + rank + i * splits) * p.N + n, sum, left, vec);
  }
}

template <typename T, bool PUSH, int TOKENS>
__device__ __forceinline__ void join(const Product& p, const float* parts, const unsigned char* tiles, int n0, int m0, int tokens, int rank, int splits,
                                     int warp, int lane) {
  if (PUSH) join_parts<T>(p, parts, n0, m0, tokens, TOKENS / splits, rank, splits, warp, lane);
  else pull_tiles<T>(p, smem_u32(tiles), n0, m0, tokens, rank, splits, warp, lane);
}

// Quantises columns c0 ... c0 + width - 1 of all (at most 16) tokens with 128 threads: codes into the 128-byte-swizzled rows of
// consecutive stages at `tiles`, scales into the tiles of consecutive steps at `scales`.  What no token fills is zero.
template <typename T, int XF>
__device__ __forceinline__ void quantize_tokens(const Product& p, int c0, int width, unsigned char* tiles, unsigned char* scales, int t) {
  constexpr int TILE = 16 * ROW_BYTES, UNIT_BYTES = XF == NES_MXFP4 ? 4 : 8, AT_ONCE = 4;
  const int row_units = width / UNIT, units = p.M * row_units;
  const T* x = static_cast<const T*>(p.x);
  const Span span = {reinterpret_cast<const uint8_t*>(x), reinterpret_cast<const uint8_t*>(x + int64_t(p.M) * p.K)};
  for (int i = t; i < width / STEP * (CHUNKS * SCALE_TILE / 16); i += 128) reinterpret_cast<uint4*>(scales)[i] = make_uint4(0u, 0u, 0u, 0u);
  for (int i = t; i < row_units * UNIT_BYTES; i += 128)                                       // = 16 rows in 16-byte pieces
    if (i / (ROW_BYTES / 16) % 16 >= p.M) reinterpret_cast<uint4*>(tiles)[i] = make_uint4(0u, 0u, 0u, 0u);
  asm volatile("bar.sync 1, 128;" ::: "memory");                                              // before scales are written
  for (int u0 = t; u0 - (t & 31) < units; u0 += 128 * AT_ONCE) {
    Raw<T> raw[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int u = u0 + 128 * i, row = u / row_units, c = c0 + (u - row * row_units) * UNIT;
      if (p.whole_rows) raw[i] = load_raw<true>(x + int64_t(row) * p.K, u < units ? c : p.K, p.K, span);
      else raw[i] = load_raw<false>(x + int64_t(row) * p.K, u < units ? c : p.K, p.K, span);
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int u = u0 + 128 * i;
      if (u - (t & 31) >= units) break;                                                       // whole warps: 64 units divide a row
      const int row = u / row_units, at = u - row * row_units;
      float v[UNIT];
      raw_values(raw[i], v);
      uint32_t code;
      const uint2 q = encode_unit<XF>(v, code);
      const int byte = at * UNIT_BYTES, stage = byte / ROW_BYTES, in_row = byte % ROW_BYTES;
      unsigned char* to = tiles + stage * TILE + row * ROW_BYTES + (((in_row >> 4) ^ (row & 7)) << 4) + (in_row & 15);
      if (XF == NES_MXFP4) *reinterpret_cast<uint32_t*>(to) = q.x;
      else *reinterpret_cast<uint2*>(to) = q;
      if ((at & 3) == 0) scales[(at / (GROUP / UNIT)) * SCALE_TILE + row * 16 + ((at >> 2) & 3)] = uint8_t(code);
    }
  }
}

// X: void for activations that are quantised already, else the type of plain ones
template <int XF, int WF, int TOKENS, typename X, bool PUSH>
__global__ void __launch_bounds__(THREADS_TC, 1) mx_product_kernel(const __grid_constant__ ProductMaps maps, const Product p, int splits) {
  constexpr bool RAW = !std::is_same<X, void>::value;
  constexpr int STAGE_GROUPS = XF == NES_MXFP4 ? 2 : 1;                  // 128-element groups per stage
  constexpr int STAGES_PER_STEP = CHUNKS / STAGE_GROUPS;
  using L = Layout<TOKENS, RAW, STAGES_PER_STEP, PUSH>;
  extern __shared__ unsigned char dyn_raw[];
  const unsigned int timeouts_at_start = timeouts_so_far();
  const uint32_t raw = smem_u32(dyn_raw);
  unsigned char* tiles = dyn_raw + (((raw + 1023u) & ~1023u) - raw);
  unsigned char* raw_tiles = tiles + size_t(L::STAGES) * L::STAGE;
  unsigned char* raw_scales = raw_tiles + L::RAW_X;
  unsigned char* scale_tiles = raw_scales + L::RAW_SCALES;
  float* parts = reinterpret_cast<float*>(scale_tiles + 2 * L::SCALES);
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<unsigned char*>(parts) + L::PARTS);
  uint64_t* empty = full + L::STAGES;
  uint64_t* sf_full = empty + L::STAGES;
  uint64_t* sf_empty = sf_full + 2;
  uint64_t* accum = sf_empty + 2;
  uint64_t* raw_full = accum + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(raw_full + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % splits, n0 = (blockIdx.x / splits) * FEATURES, m0 = blockIdx.y * TOKENS;
  const int all_steps = (p.groups + CHUNKS - 1) / CHUNKS;
  const int step0 = int(int64_t(all_steps) * rank / splits), step1 = int(int64_t(all_steps) * (rank + 1) / splits);
  const int kt0 = step0 * STAGES_PER_STEP;
  const int kt1 = min(step1 * STAGES_PER_STEP, (p.groups + STAGE_GROUPS - 1) / STAGE_GROUPS);

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&sf_full[s], 4); mbar_init(&sf_empty[s], 1); }
    mbar_init(accum, 1);
    mbar_init(raw_full, 4);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(tmem_slot, L::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  if (PUSH && splits > 1) cluster_arrive();              // waited for before the first store into another CTA's shared memory

  if (warp == 0) {
    if (lane == 0) {
      // a spreading copy counts the bytes it reads, half of those it fills
      constexpr uint32_t TX = (RAW ? 0 : L::X_BYTES) + (XF == NES_MXFP8 && WF == NES_MXFP4 ? L::W_BYTES / 2 : L::W_BYTES);
      // first coordinate: bytes of codes, or elements of a copy that spreads 4-bit codes.  The weights of the first stages do not
      // depend on the kernel before; the activations may.
      const int ready = RAW ? 0 : min(int(L::STAGES), kt1 - kt0);
      if (!p.overlap) wait_for_kernel_before();
      for (int i = 0; i < ready; ++i) {
        mbar_expect_tx(&full[i], TX);
        tma_load_2d(tiles + size_t(i) * L::STAGE, &maps.w, &full[i], (kt0 + i) * ROW_BYTES, n0);
      }
      wait_for_kernel_before();
      for (int i = 0; i < ready; ++i) tma_load_2d(tiles + size_t(i) * L::STAGE + L::W_BYTES, &maps.x, &full[i], (kt0 + i) * ROW_BYTES, m0);
      int s = ready % L::STAGES;
      uint32_t ph = ready == L::STAGES;
      for (int kt = kt0 + ready; kt < kt1; ++kt) {
        if (!mbar_wait(&empty[s], ph ^ 1, 1)) break;
        unsigned char* st = tiles + size_t(s) * L::STAGE;
        mbar_expect_tx(&full[s], TX);
        const int c = kt * ROW_BYTES;
        tma_load_2d(st, &maps.w, &full[s], c, n0);
        if (!RAW) tma_load_2d(st + L::W_BYTES, &maps.x, &full[s], c, m0);
        if (++s == L::STAGES) { s = 0; ph ^= 1u; }
      }
    }
    __syncwarp();
    if (PUSH && splits > 1) cluster_wait();
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_scaled<XF, WF>(FEATURES, TOKENS);
    const uint64_t desc0 = smem_desc_sw128(smem_u32(tiles));
    const uint64_t sdesc0 = scale_desc(smem_u32(scale_tiles)), xdesc0 = smem_desc_sw128(smem_u32(raw_tiles));
    int s = 0;
    uint32_t ph = 0, sf_ph = 0, accumulate = 0;
    int kt = kt0;
    wait_for_kernel_before();                         // the bounded waits count from here
    if (RAW) ok = warp_mbar_wait(raw_full, 0, 2);
    for (int step = step0; step < step1 && ok; ++step) {
      const int b = (step - step0) & 1;
      ok = warp_mbar_wait(&sf_full[b], sf_ph, 2);
      if (!ok) break;
      if (b) sf_ph ^= 1u;
      fence_proxy_async_smem();                         // here and not in the loading warps: it waits for loads in flight
      const uint32_t sfa = tmem + L::SCALE_BASE + b * L::SCALE_COLS, sfb = sfa + CHUNKS * 4;
      const uint64_t sdesc = sdesc0 + uint64_t((b * L::SCALES) >> 4);
      warp_copy_scales<1, 4>(sfa, sdesc);
      warp_copy_scales<1, L::X_COLS>(sfb, RAW ? scale_desc(smem_u32(raw_scales) + (step - step0) * L::STEP_SCALES) : sdesc + uint64_t(L::STEP_SCALES >> 4));
      warp_mma_commit(&sf_empty[b]);
#pragma unroll
      for (int i = 0; i < STAGES_PER_STEP; ++i, ++kt) {
        if (kt >= kt1) break;
        ok = warp_mbar_wait(&full[s], ph, 2);
        if (!ok) break;
        tc_fence_after();
        const uint64_t a = desc0 + uint64_t(uint32_t(s) * uint32_t(L::STAGE >> 4));
        const uint64_t x = RAW ? xdesc0 + uint64_t(uint32_t(kt - kt0) * uint32_t(L::X_BYTES >> 4)) : a + (L::W_BYTES >> 4);
        const int j = i * STAGE_GROUPS;
        if (STAGE_GROUPS == 1 || kt * 2 + 1 < p.groups)
          warp_mma_stage<XF, 1>(tmem, a, x, idesc, sfa + 4 * j, sfb + L::X_COLS * j, sfa + 4 * (j + STAGE_GROUPS - 1),
                                sfb + L::X_COLS * (j + STAGE_GROUPS - 1), accumulate);
        else
          warp_mma_stage<XF, 1, true>(tmem, a, x, idesc, sfa + 4 * j, sfb + L::X_COLS * j, 0u, 0u, accumulate);
        accumulate = 1;
        warp_mma_commit(&empty[s]);
        if (++s == L::STAGES) { s = 0; ph ^= 1u; }
      }
    }
    warp_mma_commit(accum);
    if (PUSH && splits > 1) cluster_wait();
  } else {
    const int q = warp & 3;
    const uint32_t lanes = uint32_t(q * 32) << 16;
    const int t = threadIdx.x - 64, row = scale_row(t);
    uint4 wv[4], xv[4];                              // four steps in flight
    take_turn();
    auto load = [&](int step, uint4& wo, uint4& xo) {
      if (step >= step1) return;
      wo = load_scale_words(p.w_scales, n0 + row, p.N, step * CHUNKS, p.groups, p.vec_scales);
      if (!RAW) xo = load_scale_words(p.x_scales, row < TOKENS ? m0 + row : p.M, p.M, step * CHUNKS, p.groups, p.vec_scales);
    };
#pragma unroll
    for (int u = 0; u < 4; ++u) load(step0 + u, wv[u], xv[u]);
    if (RAW) {
      quantize_tokens<typename std::conditional<RAW, X, float>::type, XF>(p, step0 * STEP, (step1 - step0) * STEP, raw_tiles, raw_scales, t);
      __syncwarp();
      if (lane == 0) mbar_arrive(raw_full);
    }
    for (int step = step0; step < step1 && ok; step += 4) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (step + u >= step1 || !ok) break;
        const int b = u & 1;
        ok = warp_mbar_wait(&sf_empty[b], u < 2 ? 1u : 0u, 4);
        if (!ok) break;
        unsigned char* to = scale_tiles + b * L::SCALES;
        put_scale_words(to, t, wv[u]);
        if (!RAW) put_scale_words(to + L::STEP_SCALES, t, xv[u]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sf_full[b]);
        load(step + u + 4, wv[u], xv[u]);
      }
    }
    ok = warp_mbar_wait(accum, 0, 3) && ok;
    tc_fence_after();
    const bool good = __all_sync(0xffffffffu, ok && timeouts_so_far() == timeouts_at_start);
    if (PUSH && splits > 1) cluster_wait();
    // PUSH: to the CTA that adds up the token, each rank into a part of its own
    const int share = TOKENS / splits, half = __ffs(splits) - 1;             // splits is a power of two
    const uint32_t mine = smem_u32(parts) + uint32_t(rank * share * FEATURES + q * 32 + lane) * 4u;
    float* part = reinterpret_cast<float*>(tiles) + q * 32 + lane;           // every stage has been consumed
#pragma unroll 1
    for (int c = 0; c < TOKENS; c += 16) {
      if (m0 + c >= p.M) break;
      uint32_t r[16];
      tmem_ld16_nowait(tmem + lanes + c, r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float v = good ? __uint_as_float(r[j]) : 0.f;
        if (PUSH) st_cluster(map_rank(mine + uint32_t(((c + j) >> half) * FEATURES) * 4u, (c + j) & (splits - 1)), v);
        else part[(c + j) * FEATURES] = v;
      }
    }
  }
  __syncwarp();
  if (splits > 1) cluster_sync_all(); else __syncthreads();
  if (warp >= 2 && timeouts_so_far() == timeouts_at_start) {
    const int tokens = min(TOKENS, p.M - m0);
    if (p.y_dtype == NES_F32) join<float, PUSH, TOKENS>(p, parts, tiles, n0, m0, tokens, rank, splits, warp - 2, lane);
    else if (p.y_dtype == NES_BF16) join<__nv_bfloat16, PUSH, TOKENS>(p, parts, tiles, n0, m0, tokens, rank, splits, warp - 2, lane);
    else join<__half, PUSH, TOKENS>(p, parts, tiles, n0, m0, tokens, rank, splits, warp - 2, lane);
  }
  __syncwarp();
  if (!PUSH && splits > 1) cluster_sync_all();              // partial tiles stay until everyone has read them
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------ many tokens: CTA pairs
//
// Two CTAs share a tile of 256 features x 256 tokens (tcgen05 with cta_group::2): each holds 128 weight rows and half of
// the tokens' rows and keeps the accumulator of its own features, so an SM reads 128 + 128 rows per stage where it
// would need 128 + 256 alone.  256 columns are the widest instruction and the only one near the pipe's rate: measured
// without loads and epilogue, an e2m1 product of K = 64 takes 170 cycles with 256 columns and as many with 192; an e4m3
// one of K = 32 takes 143 and 118.
//
// The grid is persistent, and the epilogue of a tile runs under the products of the next: two accumulators of 256
// columns and two buffers of scales (2 * 48) need 608 columns of the 512 there are, so the accumulators overlap by 96
// (columns 0-255 and 160-415).  The epilogue reads the shared columns first and hands them over; the rest of its
// work is done while the next tile fills the other accumulator.
// Results go through shared memory to TMA stores, which clip at the matrix's edges.

constexpr int PAIR_TOKENS = 256;
constexpr int PAIR_FEATURES = 2 * FEATURES;
constexpr int THREADS_PAIR = 320;            // warp 0: TMA, 1: MMA (leading CTA), 2-5: scales, 6-9: epilogue

struct PairLayout {
  static constexpr int W_BYTES = FEATURES * ROW_BYTES;
  static constexpr int X_BYTES = PAIR_TOKENS / 2 * ROW_BYTES;
  static constexpr int STAGE = W_BYTES + X_BYTES;
  static constexpr int STAGES = 6;
  static constexpr int X_COLS = 8;
  static constexpr int SCALE_COLS = CHUNKS * (4 + X_COLS);
  static constexpr int SCALE_BASE = 512 - 2 * SCALE_COLS;
  static constexpr int ACC_STRIDE = SCALE_BASE - PAIR_TOKENS;              // first column of the second accumulator
  static constexpr int SHARED_COLS = PAIR_TOKENS - ACC_STRIDE;             // columns both accumulators have
  static constexpr int OUT_BYTES = 32 * 64;                                // one warp's output box: 32 features x 32 (16-bit) or 16 tokens
  static constexpr int SCALES = 3 * CHUNKS * SCALE_TILE;                   // a buffer in shared memory: w, x rows 0-127, x rows 128-255
  static constexpr size_t SMEM = 1024 + size_t(STAGES) * STAGE + 8 * OUT_BYTES + 2 * SCALES + (2 * STAGES + 10) * sizeof(uint64_t) + 16;
};
static_assert(PairLayout::SHARED_COLS == 96 && PairLayout::SHARED_COLS % 32 == 0, "tensor memory");
static_assert(PairLayout::SMEM <= 227 * 1024, "shared memory");

struct PairMaps { CUtensorMap w, x, y; };

// arrives at the barrier of the same address in both CTAs once the products issued so far are done
__device__ __forceinline__ void warp_commit_pair(uint64_t* bar) {
  asm volatile(
      "{\n"
      ".reg .pred pe;\n"
      "elect.sync _|pe, 0xffffffff;\n"
      "@pe tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n"
      "}\n"
      ::"r"(smem_u32(bar)), "h"(uint16_t(3)) : "memory");
}
// load into this CTA's shared memory, counted by a barrier of the leading CTA
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t leader_bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(leader_bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(map), "r"(smem_u32(src)), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t (&r)[32]) {
  tmem_ld16_nowait(taddr, r);
  tmem_ld16_nowait(taddr + 16, r + 16);
}

// One warp's 32 tokens x 32 features: lane = feature, r[j] = token j.
template <typename T>
__device__ __forceinline__ void box_to_smem(unsigned char* box, int lane, const uint32_t* r, float bias) {
  T* out = reinterpret_cast<T*>(box) + lane;
#pragma unroll
  for (int j = 0; j < int(64 / sizeof(T)); ++j) out[j * 32] = from_float<T>(__uint_as_float(r[j]) + bias);
}
template <typename T>
__device__ __forceinline__ void box_to_global(const Product& p, int m, int n, const uint32_t (&r)[32], float bias) {
  if (n >= p.N) return;
  T* out = static_cast<T*>(p.y) + int64_t(m) * p.N + n;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    if (m + j < p.M) *out = from_float<T>(__uint_as_float(r[j]) + bias);
    out += p.N;
  }
}
// Through shared memory to a TMA store, by turns from two boxes.
template <typename T>
__device__ __forceinline__ void box_by_tma(const CUtensorMap* map, unsigned char* boxes, int& side, int lane, int m, int n0, int M,
                                           const uint32_t (&r)[32], float bias) {
  constexpr int TOKENS = 64 / sizeof(T);
#pragma unroll
  for (int h = 0; h < 32; h += TOKENS) {
    if (m + h >= M) break;
    unsigned char* out = boxes + side * PairLayout::OUT_BYTES;
    side ^= 1;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");      // the box's last store has been read
    __syncwarp();
    box_to_smem<T>(out, lane, r + h, bias);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(map, out, n0, m + h);
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
  }
}

// Order of the tiles: four feature tiles wide down all tokens, so that the pairs that run together share both operands' rows.
constexpr int RASTER = 4;
__device__ __forceinline__ int2 tile_place(int tile, int ftiles, int ttiles) {
  const int column = tile / (RASTER * ttiles), within = tile - column * RASTER * ttiles;
  const int wide = min(RASTER, ftiles - column * RASTER), t = within / wide;
  return make_int2(column * RASTER + within - t * wide, t);
}

template <int XF, int WF>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS_PAIR, 1)
mx_pair_kernel(const __grid_constant__ PairMaps maps, const Product p, int ftiles, int ttiles, int tma_out) {
  using L = PairLayout;
  extern __shared__ unsigned char dyn_raw[];
  const unsigned int timeouts_at_start = timeouts_so_far();
  const uint32_t raw = smem_u32(dyn_raw);
  unsigned char* stages = dyn_raw + (((raw + 1023u) & ~1023u) - raw);
  unsigned char* boxes = stages + size_t(L::STAGES) * L::STAGE;
  unsigned char* scale_tiles = boxes + 8 * L::OUT_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(scale_tiles + 2 * L::SCALES);
  uint64_t* empty = full + L::STAGES;
  uint64_t* sf_full = empty + L::STAGES;
  uint64_t* sf_empty = sf_full + 2;
  uint64_t* sf_peer = sf_empty + 2;
  uint64_t* acc_full = sf_peer + 2;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(cluster_rank());
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, tiles = ftiles * ttiles;
  constexpr int STAGE_GROUPS = XF == NES_MXFP4 ? 2 : 1;
  constexpr int STAGES_PER_STEP = CHUNKS / STAGE_GROUPS;
  const int steps = (p.groups + CHUNKS - 1) / CHUNKS;
  const int kts = (p.groups + STAGE_GROUPS - 1) / STAGE_GROUPS;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sf_full[s], 4); mbar_init(&sf_empty[s], 1); mbar_init(&sf_peer[s], 1);
      mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 8);     // four epilogue warps of each CTA
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                              // both CTAs' barriers exist
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      constexpr uint32_t W_TX = XF == NES_MXFP8 && WF == NES_MXFP4 ? L::W_BYTES / 2 : L::W_BYTES;   // a spreading copy counts what it reads
      const uint32_t full0 = map_rank(smem_u32(full), 0);
      // the weights of the first stages do not depend on the kernel before; the activations may
      const int ready = pair < tiles ? min(int(L::STAGES), kts) : 0;
      if (!p.overlap) wait_for_kernel_before();
      {
        const int2 at = tile_place(pair, ftiles, ttiles);
        const int n0 = at.x * PAIR_FEATURES + rank * FEATURES, m0 = at.y * PAIR_TOKENS + rank * (PAIR_TOKENS / 2);
        for (int i = 0; i < ready; ++i) {
          if (rank == 0) mbar_expect_tx(&full[i], 2 * (W_TX + L::X_BYTES));
          tma_load_pair(stages + size_t(i) * L::STAGE, &maps.w, full0 + uint32_t(i) * 8u, i * ROW_BYTES, n0);
        }
        wait_for_kernel_before();
        for (int i = 0; i < ready; ++i) tma_load_pair(stages + size_t(i) * L::STAGE + L::W_BYTES, &maps.x, full0 + uint32_t(i) * 8u, i * ROW_BYTES, m0);
      }
      int s = ready % L::STAGES;
      uint32_t ph = ready == L::STAGES;
      for (int tile = pair; tile < tiles && ok; tile += pairs) {
        const int2 at = tile_place(tile, ftiles, ttiles);
        const int n0 = at.x * PAIR_FEATURES + rank * FEATURES, m0 = at.y * PAIR_TOKENS + rank * (PAIR_TOKENS / 2);
        for (int kt = tile == pair ? ready : 0; kt < kts; ++kt) {
          ok = mbar_wait(&empty[s], ph ^ 1, 1);
          if (!ok) break;
          unsigned char* st = stages + size_t(s) * L::STAGE;
          if (rank == 0) mbar_expect_tx(&full[s], 2 * (W_TX + L::X_BYTES));
          const uint32_t bar = full0 + uint32_t(s) * 8u;
          tma_load_pair(st, &maps.w, bar, kt * ROW_BYTES, n0);
          tma_load_pair(st + L::W_BYTES, &maps.x, bar, kt * ROW_BYTES, m0);
          if (++s == L::STAGES) { s = 0; ph ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    wait_for_kernel_before();                                      // the bounded waits count from here
    if (rank == 0) {
      constexpr uint32_t idesc = idesc_scaled<XF, WF>(PAIR_FEATURES, PAIR_TOKENS);
      const uint64_t desc0 = smem_desc_sw128(smem_u32(stages));
      const uint64_t sdesc0 = scale_desc(smem_u32(scale_tiles));
      int s = 0, b = 0, acc = 0;
      uint32_t ph = 0, sf_ph = 0, acc_ph = 0;
      for (int tile = pair; tile < tiles && ok; tile += pairs) {
        // acc_empty[a]: the epilogue has read the shared columns of accumulator a, which the other one starts or ends with;
        // its own columns were read before that of the tile in between
        if (tile != pair) {
          ok = warp_mbar_wait(&acc_empty[acc ^ 1], acc_ph, 2);
          if (!ok) break;
          if (!acc) acc_ph ^= 1u;
        }
        tc_fence_after();
        const uint32_t d = tmem + acc * L::ACC_STRIDE;
        uint32_t accumulate = 0;
        int kt = 0;
        for (int step = 0; step < steps && ok; ++step) {
          ok = warp_mbar_wait(&sf_full[b], sf_ph, 2) && warp_mbar_wait(&sf_peer[b], sf_ph, 2);
          if (!ok) break;
          fence_proxy_async_smem();                     // here and not in the loading warps: it waits for loads in flight
          const uint32_t sfa = tmem + L::SCALE_BASE + b * L::SCALE_COLS, sfb = sfa + CHUNKS * 4;
          const uint64_t sdesc = sdesc0 + uint64_t((b * L::SCALES) >> 4);
          warp_copy_scales<2, 4>(sfa, sdesc);
          warp_copy_scales<2, L::X_COLS>(sfb, sdesc + uint64_t((CHUNKS * SCALE_TILE) >> 4));
          warp_copy_scales<2, L::X_COLS>(sfb + 4, sdesc + uint64_t((2 * CHUNKS * SCALE_TILE) >> 4));
          warp_commit_pair(&sf_empty[b]);
#pragma unroll
          for (int i = 0; i < STAGES_PER_STEP; ++i, ++kt) {
            if (kt >= kts) break;
            ok = warp_mbar_wait(&full[s], ph, 2);
            if (!ok) break;
            tc_fence_after();
            const uint64_t a = desc0 + uint64_t(uint32_t(s) * uint32_t(L::STAGE >> 4)), x = a + (L::W_BYTES >> 4);
            const int j = i * STAGE_GROUPS;
            if (STAGE_GROUPS == 1 || kt * 2 + 1 < p.groups)
              warp_mma_stage<XF, 2>(d, a, x, idesc, sfa + 4 * j, sfb + L::X_COLS * j, sfa + 4 * (j + STAGE_GROUPS - 1),
                                    sfb + L::X_COLS * (j + STAGE_GROUPS - 1), accumulate);
            else
              warp_mma_stage<XF, 2, true>(d, a, x, idesc, sfa + 4 * j, sfb + L::X_COLS * j, 0u, 0u, accumulate);
            accumulate = 1;
            warp_commit_pair(&empty[s]);
            if (++s == L::STAGES) { s = 0; ph ^= 1u; }
          }
          if (b) sf_ph ^= 1u;
          b ^= 1;
        }
        warp_commit_pair(&acc_full[acc]);
        acc ^= 1;
      }
    } else {
      // tells the leading CTA of this CTA's scales: a signal across CTAs also waits for its thread's loads in flight
      const uint32_t sf_peer0 = map_rank(smem_u32(sf_peer), 0);
      const int64_t total = pair < tiles ? int64_t((tiles - 1 - pair) / pairs + 1) * steps : 0;
      for (int64_t i = 0; i < total && ok; ++i) {
        ok = warp_mbar_wait(&sf_full[i & 1], uint32_t(i >> 1) & 1u, 2);
        if (!ok) break;
        fence_proxy_async_smem();
        if (lane == 0) mbar_arrive_cluster(sf_peer0 + uint32_t(i & 1) * 8u);
        __syncwarp();
      }
    }
  } else if (warp < 6) {
    const int t = threadIdx.x - 64, row = scale_row(t);
    uint4 v[4][3];                                   // four steps in flight
    int tile = pair, step = 0;                       // of the next load
    auto load = [&](uint4 (&o)[3]) {
      if (tile >= tiles) return;
      const int2 at = tile_place(tile, ftiles, ttiles);
      const int n0 = at.x * PAIR_FEATURES + rank * FEATURES, m0 = at.y * PAIR_TOKENS;
      o[0] = load_scale_words(p.w_scales, n0 + row, p.N, step * CHUNKS, p.groups, p.vec_scales);
      o[1] = load_scale_words(p.x_scales, m0 + row, p.M, step * CHUNKS, p.groups, p.vec_scales);
      o[2] = load_scale_words(p.x_scales, m0 + 128 + row, p.M, step * CHUNKS, p.groups, p.vec_scales);
      if (++step == steps) { step = 0; tile += pairs; }
    };
    take_turn();
#pragma unroll
    for (int i = 0; i < 4; ++i) load(v[i]);
    const int64_t total = pair < tiles ? int64_t((tiles - 1 - pair) / pairs + 1) * steps : 0;
    for (int64_t i = 0; i < total && ok; i += 4) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (i + u >= total) break;
        const int b = u & 1;
        ok = warp_mbar_wait(&sf_empty[b], u < 2 ? 1u : 0u, 4);
        if (!ok) break;
        unsigned char* to = scale_tiles + b * L::SCALES;
#pragma unroll
        for (int h = 0; h < 3; ++h) put_scale_words(to + h * CHUNKS * SCALE_TILE, t, v[u][h]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sf_full[b]);
        load(v[u]);
      }
    }
  } else {
    const int q = warp & 3;
    const uint32_t lanes = uint32_t(q * 32) << 16;
    const uint32_t acc_empty0 = map_rank(smem_u32(acc_empty), 0);
    unsigned char* box = boxes + (warp - 6) * 2 * L::OUT_BYTES;
    wait_for_kernel_before();
    int acc = 0, side = 0;
    uint32_t ph = 0;
    for (int tile = pair; tile < tiles; tile += pairs) {
      const int2 at = tile_place(tile, ftiles, ttiles);
      const int n0 = at.x * PAIR_FEATURES + rank * FEATURES + q * 32, m0 = at.y * PAIR_TOKENS;
      ok = warp_mbar_wait(&acc_full[acc], ph, 3);
      if (!ok) break;
      tc_fence_after();
      const bool good = __all_sync(0xffffffffu, timeouts_so_far() == timeouts_at_start);
      const float bias = p.bias && n0 + lane < p.N ? fetch(p.bias + n0 + lane) : 0.f;
      auto emit = [&](int c, const uint32_t (&r)[32]) {
        if (!good || n0 >= p.N || m0 + c >= p.M) return;
        if (tma_out) {
          if (p.y_dtype == NES_F32) box_by_tma<float>(&maps.y, box, side, lane, m0 + c, n0, p.M, r, bias);
          else if (p.y_dtype == NES_BF16) box_by_tma<__nv_bfloat16>(&maps.y, box, side, lane, m0 + c, n0, p.M, r, bias);
          else box_by_tma<__half>(&maps.y, box, side, lane, m0 + c, n0, p.M, r, bias);
        } else if (p.y_dtype == NES_F32) {
          box_to_global<float>(p, m0 + c, n0 + lane, r, bias);
        } else if (p.y_dtype == NES_BF16) {
          box_to_global<__nv_bfloat16>(p, m0 + c, n0 + lane, r, bias);
        } else {
          box_to_global<__half>(p, m0 + c, n0 + lane, r, bias);
        }
      };
      // the columns shared with the other accumulator go to registers and are handed over before anything else: the
      // last 96 of accumulator 0, the first of accumulator 1
      const uint32_t from = tmem + lanes + acc * L::ACC_STRIDE;
      const int first = acc ? 0 : L::ACC_STRIDE;
      {
        uint32_t r[3][32];
#pragma unroll
        for (int i = 0; i < 3; ++i) tmem_ld32_nowait(from + first + 32 * i, r[i]);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(acc_empty0 + acc * 8);
#pragma unroll
        for (int i = 0; i < 3; ++i) emit(first + 32 * i, r[i]);
      }
#pragma unroll 1
      for (int i = L::SHARED_COLS; i < PAIR_TOKENS; i += 32) {
        const int c = (first + i) & (PAIR_TOKENS - 1);
        if (m0 + c >= p.M) continue;
        uint32_t r[32];
        tmem_ld32_nowait(from + c, r);
        tmem_ld_wait();
        emit(c, r);
      }
      if (acc) ph ^= 1u;
      acc ^= 1;
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                              // no CTA leaves while the other may still signal it
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// Row-major byte matrix of codes as a TMA source, boxes of 128 bytes (or of 128 4-bit elements spread to bytes) x box_rows rows.
static int code_map(CUtensorMap* map, const void* base, int64_t rows, int64_t groups, bool four_bits, bool spread, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  NES_REQUIRE(fn != nullptr, NES_ERR_LAUNCH, "mx_linear_fwd: cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t pitch = cuuint64_t(groups) * (four_bits ? 64 : 128);
  cuuint64_t dims[2] = {spread ? cuuint64_t(groups) * GROUP : pitch, (cuuint64_t)rows};
  cuuint64_t strides[1] = {pitch};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, spread ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides,
                  box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  NES_REQUIRE(r == CUDA_SUCCESS, NES_ERR_LAUNCH, "mx_linear_fwd: cuTensorMapEncodeTiled failed with %d", (int)r);
  return NES_OK;
}

// CTAs that share a tile's K: as many as fill the SMs once, each with a step of its own at least.  Clusters of eight do not
// pack onto all SMs: 16 of them take two waves (1 token, 16384x2048: 14.0 us against 10.7 us in fours), 4 to 8 are faster than
// fours (8192x512: 5.4 us against 7.3 us).
static int choose_splits(int64_t tiles, int steps) {
  int splits = 1;
  while (splits < 8 && splits * 2 <= steps && tiles * splits * 2 <= (splits == 4 ? sm_count() / 2 : sm_count())) splits *= 2;
  return splits;
}

// Raises a kernel's dynamic shared memory limit once per device.
template <auto KERNEL>
static int allow_smem(size_t bytes) {
  static unsigned long long done = 0;                      // one bit per device, one word per kernel
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const unsigned long long bit = 1ULL << (dev & 63);
  if (e == cudaSuccess && (dev > 63 || !(__atomic_load_n(&done, __ATOMIC_RELAXED) & bit))) {
    e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev <= 63) __atomic_fetch_or(&done, bit, __ATOMIC_RELAXED);
  }
  NES_REQUIRE(e == cudaSuccess, NES_ERR_LAUNCH, "mx_linear_fwd: shared memory opt-in failed: %s", cudaGetErrorString(e));
  return NES_OK;
}

template <int XF, int WF, int TOKENS, typename X, bool PUSH>
static int launch_product(const Product& p, const void* x, const void* w, int splits, cudaStream_t st) {
  using L = Layout<TOKENS, !std::is_same<X, void>::value, XF == NES_MXFP4 ? 2 : 4, PUSH>;
  ProductMaps maps;
  int rc = code_map(&maps.w, w, p.N, p.groups, WF == NES_MXFP4, WF == NES_MXFP4 && XF == NES_MXFP8, FEATURES);
  if (rc != NES_OK) return rc;
  maps.x = maps.w;
  if (std::is_same<X, void>::value && (rc = code_map(&maps.x, x, p.M, p.groups, XF == NES_MXFP4, false, TOKENS)) != NES_OK) return rc;
  const int64_t ftiles = ceil_div<int64_t>(p.N, FEATURES), ttiles = ceil_div<int64_t>(p.M, TOKENS);
  NES_REQUIRE(ttiles <= 65535 && ftiles * splits <= INT32_MAX, NES_ERR_UNSUPPORTED, "mx_linear_fwd: too large");
  if ((rc = allow_smem<mx_product_kernel<XF, WF, TOKENS, X, PUSH>>(L::SMEM)) != NES_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ftiles * splits), unsigned(ttiles));
  cfg.blockDim = dim3(THREADS_TC);
  cfg.dynamicSmemBytes = L::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, mx_product_kernel<XF, WF, TOKENS, X, PUSH>, maps, p, splits);
  if (e != cudaSuccess) return fail(NES_ERR_LAUNCH, "mx_linear_fwd: %s", cudaGetErrorString(e));
  return check_launch("mx_linear_fwd");
}

template <int XF, int WF>
static int launch_pair(const Product& p, const void* x, const void* w, cudaStream_t st) {
  using L = PairLayout;
  PairMaps maps;
  int rc = code_map(&maps.w, w, p.N, p.groups, WF == NES_MXFP4, WF == NES_MXFP4 && XF == NES_MXFP8, FEATURES);
  if (rc != NES_OK) return rc;
  if ((rc = code_map(&maps.x, x, p.M, p.groups, XF == NES_MXFP4, false, PAIR_TOKENS / 2)) != NES_OK) return rc;
  const int size = int(dtype_bytes(p.y_dtype));
  const int tma_out = (int64_t(p.N) * size) % 16 == 0 && aligned16(p.y);
  maps.y = maps.x;
  if (tma_out) {
    cuuint64_t dims[2] = {(cuuint64_t)p.N, (cuuint64_t)p.M};
    cuuint64_t strides[1] = {cuuint64_t(p.N) * size};
    cuuint32_t box[2] = {32, cuuint32_t(64 / size)};
    cuuint32_t estr[2] = {1, 1};
    const CUtensorMapDataType type = p.y_dtype == NES_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : p.y_dtype == NES_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUresult r = encode_fn()(&maps.y, type, 2, p.y, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                             CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    NES_REQUIRE(r == CUDA_SUCCESS, NES_ERR_LAUNCH, "mx_linear_fwd: cuTensorMapEncodeTiled failed with %d", (int)r);
  }
  const int64_t ftiles = ceil_div<int64_t>(p.N, PAIR_FEATURES), ttiles = ceil_div<int64_t>(p.M, PAIR_TOKENS), tiles = ftiles * ttiles;
  NES_REQUIRE(tiles <= INT32_MAX / 16, NES_ERR_UNSUPPORTED, "mx_linear_fwd: too large");
  if ((rc = allow_smem<mx_pair_kernel<XF, WF>>(L::SMEM)) != NES_OK) return rc;
  const int64_t pairs = tiles < sm_count() / 2 ? tiles : sm_count() / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(pairs * 2));
  cfg.blockDim = dim3(THREADS_PAIR);
  cfg.dynamicSmemBytes = L::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, mx_pair_kernel<XF, WF>, maps, p, int(ftiles), int(ttiles), tma_out);
  if (e != cudaSuccess) return fail(NES_ERR_LAUNCH, "mx_linear_fwd: %s", cudaGetErrorString(e));
  return check_launch("mx_linear_fwd");
}

template <int XF, int WF, int TOKENS, typename X = void>
static int launch_single(const Product& p, const void* x, const void* w, cudaStream_t st) {
  const int splits = choose_splits(ceil_div<int64_t>(p.N, FEATURES) * ceil_div<int64_t>(p.M, TOKENS), ceil_div(p.groups, CHUNKS));
  if constexpr (TOKENS >= 128) {
    if (splits < 4) return launch_product<XF, WF, TOKENS, X, false>(p, x, w, splits, st);
  }
  return launch_product<XF, WF, TOKENS, X, true>(p, x, w, splits, st);
}

// Whether the product quantises its plain activations itself: few tokens, and a part of K per CTA that fits its shared memory.
// Every feature tile's CTAs do so before their first product, at about 0.23 us per 8 elements of a thread (of 128); a launch
// of its own, under which the product starts, costs the device 0.9 us and the host 2.8 us.  4096x4096, 4 bits: 1 token 5.7 us,
// with a launch of its own 6.6; 4 tokens 6.4 and 6.6; 8 tokens 7.4 and 6.7; 16 tokens 9.2 and 6.7.
static bool quantises_itself(int64_t M, int64_t N, int64_t K) {
  if (M > 16) return false;
  const int steps = int(ceil_div<int64_t>(K, STEP));
  const int64_t mine = ceil_div<int64_t>(steps, choose_splits(ceil_div<int64_t>(N, FEATURES), steps));
  return mine <= RAW_STEPS && M * mine * STEP <= 6 * 128 * UNIT;
}

template <int XF, int WF>
static int launch_raw(const Product& p, int x_dtype, const void* w, cudaStream_t st) {
  if (x_dtype == NES_F32) return launch_single<XF, WF, 16, float>(p, nullptr, w, st);
  if (x_dtype == NES_BF16) return launch_single<XF, WF, 16, __nv_bfloat16>(p, nullptr, w, st);
  return launch_single<XF, WF, 16, __half>(p, nullptr, w, st);
}

template <int XF, int WF>
static int launch_tokens(const Product& p, const void* x, const void* w, cudaStream_t st) {
  if (p.M <= 16) return launch_single<XF, WF, 16>(p, x, w, st);
  if (p.M <= 32) return launch_single<XF, WF, 32>(p, x, w, st);
  if (p.M <= 64) return launch_single<XF, WF, 64>(p, x, w, st);
  // Single CTAs on 128 x 128 tiles, or pairs on 256 x 256: what either takes in ns, from its waves over the SMs.  Measured
  // with 8-bit activations: a wave of either kind takes 2.5 us per 1024 of K, a wave of single CTAs 4.5 us besides (its
  // epilogue runs under nothing), the pairs 8 us in all.  512x4096x4096: 14.8 us single, 18.8 us in pairs; 1024x4096x4096:
  // 28.5 and 20.4 us; 4-bit activations take 1.5 us per 1024 of K.
  if (p.M > 128) {
    const int64_t sms = sm_count(), k = int64_t(p.groups) * (XF == NES_MXFP4 ? 190 : 310);
    const int64_t single = ceil_div<int64_t>(p.M, 128) * ceil_div(p.N, FEATURES), pairs = ceil_div<int64_t>(p.M, PAIR_TOKENS) * ceil_div(p.N, PAIR_FEATURES);
    const int splits = choose_splits(single, ceil_div(p.groups, CHUNKS));
    const int64_t single_ns = ceil_div<int64_t>(single * splits, sms) * (4500 + k / splits);
    if (8000 + ceil_div<int64_t>(pairs, sms / 2) * k < single_ns) return launch_pair<XF, WF>(p, x, w, st);
  }
  return launch_single<XF, WF, 128>(p, x, w, st);
}

static int64_t align256(int64_t v) { return (v + 255) & ~int64_t(255); }

}  // namespace mx

namespace tc {
int mx_linear_error_word(int* v, bool clear) { return read_error_word(v, clear, "tc_error_flag"); }
}  // namespace tc
}  // namespace nes

using namespace nes;
using namespace nes::mx;

extern "C" int64_t nes_mx_linear_fwd_scratch_bytes(int64_t M, int64_t N, int64_t K, int x_format) {
  if (M <= 0 || N <= 0 || K <= 0 || !known_format(x_format) || quantises_itself(M, N, K)) return 0;
  return align256(M * code_pitch(K, x_format)) + align256(M * scale_pitch(K));
}

extern "C" int nes_mx_linear_fwd(const void* x, const uint8_t* x_scales, int x_dtype, int x_format, const void* w_codes,
                                 const uint8_t* w_scales, int w_format, const float* bias, void* y, int y_dtype, int64_t M, int64_t N,
                                 int64_t K, void* scratch, int64_t scratch_bytes, nes_stream_t stream) {
  NES_REQUIRE(M >= 0 && N >= 0 && K >= 1, NES_ERR_BAD_ARG, "mx_linear_fwd: bad extent");
  NES_REQUIRE(known_format(x_format) && known_format(w_format) && !(x_format == NES_MXFP4 && w_format == NES_MXFP8) &&
                  (x_scales || known_dtype(x_dtype)) && known_dtype(y_dtype),
              NES_ERR_UNSUPPORTED, "mx_linear_fwd: unknown dtype or combination of formats");
  if (M == 0 || N == 0) return NES_OK;
  NES_REQUIRE(x && w_codes && w_scales && y, NES_ERR_BAD_ARG, "mx_linear_fwd: null pointer");
  NES_REQUIRE(aligned32(w_codes) && (!x_scales || aligned32(x)), NES_ERR_BAD_ARG, "mx_linear_fwd: codes must be 32-byte aligned");
  NES_REQUIRE(M <= INT32_MAX / 2 && N <= INT32_MAX / 2 && K <= INT32_MAX / 2, NES_ERR_UNSUPPORTED, "mx_linear_fwd: too large");
  NES_REQUIRE((reinterpret_cast<uintptr_t>(x_scales) & 3u) == 0 && (reinterpret_cast<uintptr_t>(w_scales) & 3u) == 0, NES_ERR_BAD_ARG,
              "mx_linear_fwd: scales must be 4-byte aligned");
  const int64_t need = x_scales ? 0 : nes_mx_linear_fwd_scratch_bytes(M, N, K, x_format);
  NES_REQUIRE(need == 0 || (scratch && scratch_bytes >= need && aligned32(scratch)), NES_ERR_SCRATCH,
              "mx_linear_fwd: scratch needs %lld bytes, 32-byte aligned", (long long)need);
  const Bytes outputs[] = {{y, M * N * dtype_bytes(y_dtype)}, {need ? scratch : nullptr, need}};
  const Bytes inputs[] = {{x, M * (x_scales ? code_pitch(K, x_format) : K * dtype_bytes(x_dtype))}, {x_scales, M * scale_pitch(K)},
                          {w_codes, N * code_pitch(K, w_format)}, {w_scales, N * scale_pitch(K)}, {bias, N * 4}};
  NES_REQUIRE(!overlap(outputs, inputs), NES_ERR_BAD_ARG, "mx_linear_fwd: the output or the scratch overlaps an input or the other");
  cudaStream_t st = as_stream(stream);
  Product p;
  p.x_scales = x_scales; p.w_scales = w_scales; p.bias = bias; p.y = y; p.x = x; p.whole_rows = 0; p.overlap = false;
  p.M = int(M); p.N = int(N); p.K = int(K); p.groups = int(padded(K) / GROUP); p.y_dtype = y_dtype;
  p.vec_scales = p.groups % CHUNKS == 0 && aligned16(x_scales) && aligned16(w_scales);
  if (!x_scales && need == 0) {
    p.whole_rows = aligned16(x) && (K * dtype_bytes(x_dtype)) % 16 == 0;
    if (x_format == NES_MXFP4) return launch_raw<NES_MXFP4, NES_MXFP4>(p, x_dtype, w_codes, st);
    if (w_format == NES_MXFP4) return launch_raw<NES_MXFP8, NES_MXFP4>(p, x_dtype, w_codes, st);
    return launch_raw<NES_MXFP8, NES_MXFP8>(p, x_dtype, w_codes, st);
  }
  if (need) {
    uint8_t* codes = static_cast<uint8_t*>(scratch);
    uint8_t* scales = codes + align256(M * code_pitch(K, x_format));
    const int rc = nes_mx_quantize(x, x_dtype, codes, scales, M, K, x_format, stream);
    if (rc != NES_OK) return rc;
    x = codes;
    p.x_scales = scales;
    p.overlap = true;
  }
  if (x_format == NES_MXFP4) return launch_tokens<NES_MXFP4, NES_MXFP4>(p, x, w_codes, st);
  if (w_format == NES_MXFP4) return launch_tokens<NES_MXFP8, NES_MXFP4>(p, x, w_codes, st);
  return launch_tokens<NES_MXFP8, NES_MXFP8>(p, x, w_codes, st);
}
