// Product of microscaled operands on the tensor cores: y[t, n] = sum_k x[t, k] w[n, k] + bias[n].
//
//   * tcgen05.mma with block scales: kind::mxf4 (both operands e2m1, K = 64 per instruction) or kind::mxf8f6f4 (e4m3
//     activations with e4m3 or e2m1 weights, K = 32).  The hardware multiplies every block's partial sum by 2^(ex + ew)
//     and accumulates in fp32.
//   * The weights are the M side of the instruction: 128 output features are the lanes of the accumulator, TOKENS
//     (16 ... 256) tokens its columns.  A warp that reads a column holds 32 neighbouring features of one token, so
//     the row-major output is stored in whole lines, and few tokens cost no empty rows.
//   * Codes travel by TMA as 128-byte-swizzled rows; 4-bit weights of an 8-bit product are spread to one element per
//     byte (16 elements and 8 empty bytes... per 16-byte piece) by the copy itself.
//   * Scales are stored row-major (4 bytes per 128 elements); the instruction wants them in tensor memory, one 32-bit
//     column per 32 rows and 128 elements, repeated in each quarter of the lanes.  Four warps load them for STEP = 512
//     elements of K at a time, 16 bytes per row, and write them with tcgen05.st: a transposition that costs no shared memory.
//   * Few output tiles: a cluster of up to eight CTAs splits K and adds its partial tiles in a fixed order through
//     distributed shared memory.
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
constexpr int THREADS_TC = 192;              // warp 0: TMA, warp 1: MMA, warps 2-5: scales, then epilogue

struct Product {
  const uint8_t *x_scales, *w_scales;
  const float* bias;
  void* y;
  int M, N, groups;                          // tokens, features, 128-element groups of K
  int y_dtype, vec_scales;
};
struct ProductMaps { CUtensorMap w, x; };

template <int TOKENS>
struct Layout {
  static constexpr int W_BYTES = FEATURES * ROW_BYTES;
  static constexpr int X_BYTES = TOKENS * ROW_BYTES;
  static constexpr int STAGE = W_BYTES + X_BYTES;
  static constexpr int STAGES = TOKENS >= 256 ? 4 : TOKENS >= 128 ? 6 : 8;
  static constexpr int X_COLS = TOKENS <= 128 ? 4 : 8;                     // scale columns of x per 128 elements
  static constexpr int SCALE_COLS = CHUNKS * (4 + X_COLS);                 // one buffer
  static constexpr int SCALE_BASE = TOKENS < 32 ? 32 : TOKENS;
  static constexpr int USED_COLS = SCALE_BASE + 2 * SCALE_COLS;
  static constexpr int TMEM_COLS = USED_COLS <= 128 ? 128 : USED_COLS <= 256 ? 256 : 512;
  static constexpr size_t SMEM = 1024 + size_t(STAGES) * STAGE + (2 * STAGES + 5) * sizeof(uint64_t) + 16;
};

template <int XF, int WF>
__device__ __forceinline__ void warp_mma_scaled(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                                uint32_t accumulate) {
  if (XF == NES_MXFP4)
    asm volatile(
        "{\n"
        ".reg .pred p, pe;\n"
        "elect.sync _|pe, 0xffffffff;\n"
        "setp.ne.b32 p, %6, 0;\n"
        "@pe tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n"
        "}\n"
        ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n"
        ".reg .pred p, pe;\n"
        "elect.sync _|pe, 0xffffffff;\n"
        "setp.ne.b32 p, %6, 0;\n"
        "@pe tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n"
        "}\n"
        ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// Instruction descriptor with block scales: element formats at bits 7 and 10 (kind::mxf4: 1 = e2m1; kind::mxf8f6f4: 0 = e4m3,
// 5 = e2m1), N >> 3 at bit 17, scale type 1 = E8M0 at bit 23, M >> 4 at bit 24; the byte of the scale columns that an
// instruction uses is added per instruction (bits 29 for A and 4 for B).
template <int XF, int WF>
constexpr uint32_t idesc_scaled(int m, int n) {
  constexpr uint32_t a = XF == NES_MXFP4 ? 1u : WF == NES_MXFP4 ? 5u : 0u;
  constexpr uint32_t b = XF == NES_MXFP4 ? 1u : 0u;
  return (a << 7) | (b << 10) | (uint32_t(n >> 3) << 17) | (1u << 23) | (uint32_t(m >> 4) << 24);
}
__device__ __forceinline__ constexpr uint32_t scale_byte(uint32_t id) { return (id << 29) | (id << 4); }

// 16 scale bytes of a row from 128-element group `group` on; zeros outside the matrix
__device__ __forceinline__ void load_scale_words(const uint8_t* scales, int row, int rows, int group, int groups, bool vec, uint32_t (&w)[CHUNKS]) {
#pragma unroll
  for (int j = 0; j < CHUNKS; ++j) w[j] = 0;
  if (row >= rows) return;
  const uint32_t* p = reinterpret_cast<const uint32_t*>(scales + int64_t(row) * groups * 4) + group;
  if (vec) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else {
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) if (group + j < groups) w[j] = __ldg(p + j);
  }
}

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

__device__ __forceinline__ void store_result(const Product& p, int64_t at, float v) {
  if (p.y_dtype == NES_F32) static_cast<float*>(p.y)[at] = v;
  else if (p.y_dtype == NES_BF16) static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p.y)[at] = __float2half_rn(v);
}

template <int XF, int WF, int TOKENS>
__global__ void __launch_bounds__(THREADS_TC, 1) mx_product_kernel(const __grid_constant__ ProductMaps maps, const Product p, int splits) {
  using L = Layout<TOKENS>;
  extern __shared__ unsigned char dyn_raw[];
  const unsigned int timeouts_at_start = timeouts_so_far();
  const uint32_t raw = smem_u32(dyn_raw);
  unsigned char* tiles = dyn_raw + (((raw + 1023u) & ~1023u) - raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + size_t(L::STAGES) * L::STAGE);
  uint64_t* empty = full + L::STAGES;
  uint64_t* sf_full = empty + L::STAGES;
  uint64_t* sf_empty = sf_full + 2;
  uint64_t* accum = sf_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accum + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % splits, n0 = (blockIdx.x / splits) * FEATURES, m0 = blockIdx.y * TOKENS;
  constexpr int STAGE_GROUPS = XF == NES_MXFP4 ? 2 : 1;                  // 128-element groups per stage
  constexpr int STAGES_PER_STEP = CHUNKS / STAGE_GROUPS;
  const int all_steps = (p.groups + CHUNKS - 1) / CHUNKS;
  const int step0 = int(int64_t(all_steps) * rank / splits), step1 = int(int64_t(all_steps) * (rank + 1) / splits);
  const int kt0 = step0 * STAGES_PER_STEP;
  const int kt1 = min(step1 * STAGES_PER_STEP, (p.groups + STAGE_GROUPS - 1) / STAGE_GROUPS);

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&sf_full[s], 4); mbar_init(&sf_empty[s], 1); }
    mbar_init(accum, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(tmem_slot, L::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      // a spreading copy counts the bytes it reads, half of those it fills
      constexpr uint32_t TX = L::X_BYTES + (XF == NES_MXFP8 && WF == NES_MXFP4 ? L::W_BYTES / 2 : L::W_BYTES);
      int s = 0;
      uint32_t ph = 0;
      for (int kt = kt0; kt < kt1; ++kt) {
        if (!mbar_wait(&empty[s], ph ^ 1, 1)) break;
        unsigned char* st = tiles + size_t(s) * L::STAGE;
        mbar_expect_tx(&full[s], TX);
        // first coordinate: bytes of codes, or elements of a copy that spreads 4-bit codes
        const int c = kt * ROW_BYTES;
        tma_load_2d(st, &maps.w, &full[s], c, n0);
        tma_load_2d(st + L::W_BYTES, &maps.x, &full[s], c, m0);
        if (++s == L::STAGES) { s = 0; ph ^= 1u; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_scaled<XF, WF>(FEATURES, TOKENS);
    const uint64_t desc0 = smem_desc_sw128(smem_u32(tiles));
    int s = 0;
    uint32_t ph = 0, sf_ph = 0, accumulate = 0;
    int kt = kt0;
    for (int step = step0; step < step1 && ok; ++step) {
      const int b = (step - step0) & 1;
      ok = warp_mbar_wait(&sf_full[b], sf_ph, 2);
      if (!ok) break;
      if (b) sf_ph ^= 1u;
      const uint32_t sfa = tmem + L::SCALE_BASE + b * L::SCALE_COLS, sfb = sfa + CHUNKS * 4;
#pragma unroll
      for (int i = 0; i < STAGES_PER_STEP; ++i, ++kt) {
        if (kt >= kt1) break;
        ok = warp_mbar_wait(&full[s], ph, 2);
        if (!ok) break;
        tc_fence_after();
        const uint64_t a = desc0 + uint64_t(uint32_t(s) * uint32_t(L::STAGE >> 4)), x = a + (L::W_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) {                 // 32 bytes of a row per instruction
          const int j = XF == NES_MXFP4 ? i * 2 + (k >> 1) : i;
          const uint32_t id = XF == NES_MXFP4 ? (k & 1) * 2 : k;
          if (XF != NES_MXFP4 || kt * 2 + (k >> 1) < p.groups)
            warp_mma_scaled<XF, WF>(tmem, a + 2 * k, x + 2 * k, idesc | scale_byte(id), sfa + 4 * j, sfb + L::X_COLS * j, accumulate);
          accumulate = 1;
        }
        warp_mma_commit(&empty[s]);
        if (++s == L::STAGES) { s = 0; ph ^= 1u; }
      }
      warp_mma_commit(&sf_empty[b]);
    }
    warp_mma_commit(accum);
  } else {
    const int q = warp & 3;
    const uint32_t lanes = uint32_t(q * 32) << 16;
    uint32_t wr[4][CHUNKS], xr[L::X_COLS][CHUNKS];
    auto load = [&](int step) {
#pragma unroll
      for (int c = 0; c < 4; ++c) load_scale_words(p.w_scales, n0 + c * 32 + lane, p.N, step * CHUNKS, p.groups, p.vec_scales, wr[c]);
#pragma unroll
      for (int c = 0; c < L::X_COLS; ++c)
        load_scale_words(p.x_scales, c * 32 < TOKENS ? m0 + c * 32 + lane : p.M, p.M, step * CHUNKS, p.groups, p.vec_scales, xr[c]);
    };
    uint32_t ph = 0;
    if (step0 < step1) load(step0);
    for (int step = step0; step < step1; ++step) {
      const int b = (step - step0) & 1;
      uint32_t r[16], t[CHUNKS * L::X_COLS];
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j) {
#pragma unroll
        for (int c = 0; c < 4; ++c) r[j * 4 + c] = wr[c][j];
#pragma unroll
        for (int c = 0; c < L::X_COLS; ++c) t[j * L::X_COLS + c] = xr[c][j];
      }
      if (step + 1 < step1) load(step + 1);
      ok = warp_mbar_wait(&sf_empty[b], ph ^ 1, 4);
      if (!ok) break;
      if (b) ph ^= 1u;
      tc_fence_after();
      const uint32_t base = tmem + lanes + L::SCALE_BASE + b * L::SCALE_COLS;
      tmem_st16(base, r);
#pragma unroll
      for (int c = 0; c < CHUNKS * L::X_COLS; c += 16) {
        uint32_t u[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) u[i] = t[c + i];
        tmem_st16(base + CHUNKS * 4 + c, u);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sf_full[b]);
    }
    ok = warp_mbar_wait(accum, 0, 3) && ok;
    tc_fence_after();
    const bool good = __all_sync(0xffffffffu, ok && timeouts_so_far() == timeouts_at_start);
    const int f = q * 32 + lane, n = n0 + f;
    if (splits == 1) {
      if (good) {
        const float bias = p.bias && n < p.N ? __ldg(p.bias + n) : 0.f;
#pragma unroll 1
        for (int c = 0; c < TOKENS; c += 16) {
          if (m0 + c >= p.M) break;
          uint32_t r[16];
          tmem_ld16_nowait(tmem + lanes + c, r);
          tmem_ld_wait();
          if (n < p.N) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (m0 + c + j < p.M) store_result(p, int64_t(m0 + c + j) * p.N + n, __uint_as_float(r[j]) + bias);
          }
        }
      }
    } else {
      float* part = reinterpret_cast<float*>(tiles);           // [token][feature]; every stage has been consumed
#pragma unroll 1
      for (int c = 0; c < TOKENS; c += 16) {
        if (m0 + c >= p.M) break;
        uint32_t r[16];
        tmem_ld16_nowait(tmem + lanes + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * FEATURES + f] = good ? __uint_as_float(r[j]) : 0.f;
      }
    }
  }
  __syncwarp();
  if (splits > 1) {
    cluster_sync_all();
    if (warp >= 2) {
      const int f = (warp & 3) * 32 + lane, n = n0 + f;
      const bool good = timeouts_so_far() == timeouts_at_start;
      const float bias = p.bias && n < p.N ? __ldg(p.bias + n) : 0.f;
      for (int t = rank; t < TOKENS && m0 + t < p.M; t += splits) {
        const uint32_t at = smem_u32(tiles) + uint32_t(t * FEATURES + f) * 4u;
        float v = 0.f;
        for (int r = 0; r < splits; ++r) v += ld_cluster(at, r);
        if (good && n < p.N) store_result(p, int64_t(m0 + t) * p.N + n, v + bias);
      }
    }
    __syncwarp();
    cluster_sync_all();                                        // partial tiles stay until everyone has read them
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::TMEM_COLS);
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

template <int XF, int WF, int TOKENS>
static int launch_product(const Product& p, const void* x, const void* w, cudaStream_t st) {
  using L = Layout<TOKENS>;
  ProductMaps maps;
  int rc = code_map(&maps.w, w, p.N, p.groups, WF == NES_MXFP4, WF == NES_MXFP4 && XF == NES_MXFP8, FEATURES);
  if (rc != NES_OK) return rc;
  if ((rc = code_map(&maps.x, x, p.M, p.groups, XF == NES_MXFP4, false, TOKENS)) != NES_OK) return rc;
  const int64_t ftiles = ceil_div<int64_t>(p.N, FEATURES), ttiles = ceil_div<int64_t>(p.M, TOKENS);
  const int steps = ceil_div(p.groups, CHUNKS);
  int splits = 1;
  if (TOKENS <= 128)
    while (splits < 8 && splits * 2 <= steps && ftiles * ttiles * splits * 2 <= sm_count()) splits *= 2;
  NES_REQUIRE(ttiles <= 65535 && ftiles * splits <= INT32_MAX, NES_ERR_UNSUPPORTED, "mx_linear_fwd: too large");
  const auto kernel = mx_product_kernel<XF, WF, TOKENS>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::SMEM);
  if (e != cudaSuccess) return fail(NES_ERR_LAUNCH, "mx_linear_fwd: shared memory opt-in failed: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ftiles * splits), unsigned(ttiles));
  cfg.blockDim = dim3(THREADS_TC);
  cfg.dynamicSmemBytes = L::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kernel, maps, p, splits);
  if (e != cudaSuccess) return fail(NES_ERR_LAUNCH, "mx_linear_fwd: %s", cudaGetErrorString(e));
  return check_launch("mx_linear_fwd");
}

template <int XF, int WF>
static int launch_tokens(const Product& p, const void* x, const void* w, cudaStream_t st) {
  if (p.M <= 16) return launch_product<XF, WF, 16>(p, x, w, st);
  if (p.M <= 32) return launch_product<XF, WF, 32>(p, x, w, st);
  if (p.M <= 64) return launch_product<XF, WF, 64>(p, x, w, st);
  if (p.M <= 128 || ceil_div(p.M, 256) * ceil_div(p.N, FEATURES) < sm_count()) return launch_product<XF, WF, 128>(p, x, w, st);
  return launch_product<XF, WF, 256>(p, x, w, st);
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
  if (M <= 0 || N <= 0 || K <= 0 || !known_format(x_format)) return 0;
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
  cudaStream_t st = as_stream(stream);
  if (!x_scales) {
    const int64_t need = nes_mx_linear_fwd_scratch_bytes(M, N, K, x_format);
    NES_REQUIRE(scratch && scratch_bytes >= need && aligned32(scratch), NES_ERR_SCRATCH,
                "mx_linear_fwd: scratch needs %lld bytes, 32-byte aligned", (long long)need);
    uint8_t* codes = static_cast<uint8_t*>(scratch);
    uint8_t* scales = codes + align256(M * code_pitch(K, x_format));
    const int rc = nes_mx_quantize(x, x_dtype, codes, scales, M, K, x_format, stream);
    if (rc != NES_OK) return rc;
    x = codes;
    x_scales = scales;
  }
  Product p;
  p.x_scales = x_scales; p.w_scales = w_scales; p.bias = bias; p.y = y;
  p.M = int(M); p.N = int(N); p.groups = int(padded(K) / GROUP); p.y_dtype = y_dtype;
  NES_REQUIRE((reinterpret_cast<uintptr_t>(x_scales) & 3u) == 0 && (reinterpret_cast<uintptr_t>(w_scales) & 3u) == 0, NES_ERR_BAD_ARG,
              "mx_linear_fwd: scales must be 4-byte aligned");
  p.vec_scales = p.groups % CHUNKS == 0 && aligned16(x_scales) && aligned16(w_scales);
  if (x_format == NES_MXFP4) return launch_tokens<NES_MXFP4, NES_MXFP4>(p, x, w_codes, st);
  if (w_format == NES_MXFP4) return launch_tokens<NES_MXFP8, NES_MXFP4>(p, x, w_codes, st);
  return launch_tokens<NES_MXFP8, NES_MXFP8>(p, x, w_codes, st);
}
