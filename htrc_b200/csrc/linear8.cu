// Matrix product in 8-bit integers with a scale per token and channel:
//   out[r][n] = (sum_k x[r][k] w[n][k]) x_scales[r] w_scales[n] + bias[n]
// on tcgen05 (kind::i8: int32 sums in TMEM, exact), the scales and the bias in float32 on the way out.
//
// Few tokens (linear8_small_kernel): the weights are what is read, so they take the product's 128-row side, a tile of
// 16 to 64 tokens its other.  Where the tiles alone leave SMs idle a cluster shares a tile, each CTA a range of the width;
// their integer sums are added over distributed shared memory, which changes no result.
//
// Many tokens (linear8_pair_kernel): two CTAs on neighbouring SMs share a tile of 256 tokens x 256 channels (cta_group::2),
// each loading half of either operand; persistent, two accumulators in TMEM, so that a tile leaves under the next one's
// products.
//
// Measured, 8-bit rows, bfloat16 out: 129,024 x 2,048 x 6,144 1,090 us after a rest (2,980 TOP/s) and 1,270 once the 1,000 W cap
// holds the SM clock at 1,290 MHz; 8,192 x 8,192 x 8,192 335 (3,280) and 395.  The tensor pipe is busy for 82 % of 16,384 x
// 2,048 x 6,144; the cap bounds the rest.  16 x 4,096 x 16,384: 14.6 us, the weights at 4.6 TB/s.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/htrc_layer.h"
#include "common.cuh"
#include "kernels.cuh"

namespace htrc {

int quantize_rows(const void* x, int dtype, int64_t batch, int64_t tokens, int width, const int64_t* stride, int8_t* codes,
                  int64_t pitch, float* scales, cudaStream_t st);

namespace {

struct Linear8Params {
  int rows, channels, blocks;               // blocks: of 128 of the width
  const float *xs, *ws;
  const void* bias;
  int bias_dtype;
  void* out;
  int* status;
  int tiles_m, tiles_n, splits;
  int stages;                               // few tokens: of the ring, behind rows_bytes of codes
  uint32_t rows_bytes;
  bool early;                               // few tokens: the kernel before this one did not write the weights
  // few float rows, quantised by the product: their elements, strides, tokens of a batch entry and width
  const void* x;
  int64_t x_stride[2], tokens;
  int width;
  bool vec;                                 // the rows are 16-byte aligned
  bool direct;                              // pair kernel: the output's rows are not 16-byte aligned
};

__device__ __forceinline__ float bias_at(const Linear8Params& p, int n) {
  if (p.bias == nullptr) return 0.f;
  if (p.bias_dtype == HTRC_LAYER_F32) return static_cast<const float*>(p.bias)[n];
  if (p.bias_dtype == HTRC_LAYER_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]);
  return __half2float(static_cast<const __half*>(p.bias)[n]);
}

template <typename O> __device__ __forceinline__ O from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

__device__ __forceinline__ float scaled(int sum, float xs, float ws, float bias) {
  return fmaf(static_cast<float>(sum) * xs, ws, bias);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of this CTA's shared-memory location in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ int load_cluster(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// ------------------------------------------------------------------------------------------------ few tokens
constexpr int kSmallChannels = 128;
constexpr int kFewTokens = 16, kFewBlocks = 32;      // rows that the product quantises itself: so many, of so many blocks a part

// X: int8_t, or the float type of rows that are quantised here.  Warps 0-3: the way out; the next two: TMA, MMA.  Of float
// rows warps 0-15 first write a row's codes each.
template <int T, typename X>
struct SmallShape {
  static constexpr bool kCodes = std::is_same<X, int8_t>::value;
  static constexpr int kRowWarps = kCodes ? 4 : 16, kThreads = 32 * (kRowWarps + 2);
  static constexpr uint32_t kW = kSmallChannels * 128, kX = T * 128, kStage = kCodes ? kW + kX : kW;
  static constexpr uint32_t kCols = T < 32 ? 32 : T;
  static constexpr uint32_t kBars = 1024;                  // then float rows' codes, block by block, then the stages
  static constexpr uint32_t kMost = 224 * 1024;            // of an SM's CTA; half of it where two share the SM
  static_assert(T * kSmallChannels * 4 <= 2 * kStage, "the parts of a split tile reuse the stages");
  static uint32_t rows(int blocks) { return kCodes ? 0 : blocks * kX; }
};
constexpr int kSmallStages = 12;                           // at most

struct SmallBars {
  uint64_t full[kSmallStages], empty[kSmallStages], done, rows;
  uint32_t tmem;
  int abort_flag;
  alignas(16) float scales[64];                            // the tokens'
};
static_assert(sizeof(SmallBars) <= 1024, "barriers");

// A float row's scale, and the codes of its elements from k0 up to k1 into blocks of [T][128] bytes, 128-byte swizzled (what
// is past the row in its last block is whatever was there: the weights are zero there).  One warp.
template <int T, typename X>
__device__ __forceinline__ float quantise_row(const X* x, int width, bool vec, int k0, int k1, uint8_t* blocks, int row, int lane) {
  constexpr int N = 16 / sizeof(X);
  auto one = [](X v) -> float {
    if constexpr (sizeof(X) == 4) return v;
    else if constexpr (std::is_same<X, __nv_bfloat16>::value) return __bfloat162float(v);
    else return __half2float(v);
  };
  auto larger = [](float a, float b) {                      // NaN if either is
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
  };
  union Sixteen {
    uint4 v;
    X e[N];
  };
  float top = 0.f;
  if (vec) {
    const int vecs = width / N;
    for (int i = lane; i < vecs; i += 8 * 32) {
      Sixteen t[8];                                         // in flight together
#pragma unroll
      for (int b = 0; b < 8; ++b) t[b].v = i + 32 * b < vecs ? reinterpret_cast<const uint4*>(x)[i + 32 * b] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int b = 0; b < 8; ++b)
#pragma unroll
        for (int j = 0; j < N; ++j) top = larger(top, fabsf(one(t[b].e[j])));
    }
  } else {
    for (int i = lane; i < width; i += 8 * 32) {
      float t[8];
#pragma unroll
      for (int b = 0; b < 8; ++b) t[b] = i + 32 * b < width ? one(x[i + 32 * b]) : 0.f;
#pragma unroll
      for (int b = 0; b < 8; ++b) top = larger(top, fabsf(t[b]));
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) top = larger(top, __shfl_xor_sync(0xffffffffu, top, d));
  // as the rows' own kernel has it
  top = top <= 3.4028235e38f ? fmaxf(top, 1e-30f) : __uint_as_float(0x7FC00000u);
  const float by = __fdiv_rn(127.f, top);
  auto code = [&](float v) { return __float_as_uint(__fadd_rn(__fmul_rn(v, by), 12582912.f)) & 0xFFu; };
  k1 = min(k1, width);
  if (vec) {
    for (int k = k0 + lane * N; k < k1; k += 8 * 32 * N) {
      Sixteen t[8];
#pragma unroll
      for (int b = 0; b < 8; ++b)
        t[b].v = k + 32 * N * b < k1 ? *reinterpret_cast<const uint4*>(x + k + 32 * N * b) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < N; ++j) w[j / 4] |= code(one(t[b].e[j])) << (8 * (j % 4));
        const uint32_t at = k + 32 * N * b - k0;
        if (k + 32 * N * b >= k1) continue;
        uint8_t* to = blocks + at / 128 * (T * 128) + sw128_off(row, at % 128 / 16) + at % 16;
        if constexpr (N == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(to) = w[0];
      }
    }
  } else {
    for (int k = k0 + lane; k < k1; k += 8 * 32) {
      float t[8];
#pragma unroll
      for (int b = 0; b < 8; ++b) t[b] = k + 32 * b < k1 ? one(x[k + 32 * b]) : 0.f;
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const uint32_t at = k + 32 * b - k0;
        if (k + 32 * b < k1) blocks[at / 128 * (T * 128) + sw128_off(row, at % 128 / 16) + at % 16] = static_cast<uint8_t>(code(t[b]));
      }
    }
  }
  return __fdiv_rn(top, 127.f);
}

// The kernel may be resident while the one before it still writes the rows, scales or bias: behind griddepcontrol.wait they are
// read by ordinary loads, since those of the read-only path want data that is constant for the kernel's whole life.
template <int T, typename O, typename X>
__global__ void __launch_bounds__(SmallShape<T, X>::kThreads, 1)
    linear8_small_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                         const __grid_constant__ Linear8Params p) {
  using SM = SmallShape<T, X>;
  constexpr int kTma = SM::kRowWarps, kMma = kTma + 1;
  extern __shared__ __align__(1024) uint8_t smem[];
  SmallBars* bars = reinterpret_cast<SmallBars*>(smem);
  uint8_t* const codes = smem + SM::kBars;
  uint8_t* const ring = codes + p.rows_bytes;
  const int stages = p.stages;
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool aligned = (smem_u32(smem) & 1023) == 0;      // the swizzled tiles need it
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    mbar_init(&bars->done, 1);
    mbar_init(&bars->rows, SM::kRowWarps);
    bars->abort_flag = !aligned;
    if (!aligned) flag_status(p.status, ST_WAIT_TIMEOUT);
    fence_barrier_init();
  }
  if (warp == kMma) tmem_alloc(&bars->tmem, SM::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int splits = p.splits, rank = blockIdx.x % splits, tile = blockIdx.x / splits;
  const int n0 = tile / p.tiles_m * kSmallChannels, row0 = tile % p.tiles_m * T;
  const int b0 = static_cast<int>(static_cast<int64_t>(p.blocks) * rank / splits);
  const int b1 = static_cast<int>(static_cast<int64_t>(p.blocks) * (rank + 1) / splits);
  const int n = n0 + 32 * (warp & 3) + lane;              // warps 0-3: the thread's channel
  float ws = 0.f, bias = 0.f;

  if (warp == kTma) {
    if (lane == 0 && aligned) {
      const uint64_t once = policy_evict_first(), keep = policy_evict_last();
      auto load_w = [&](int s, int b) {
        expect_tx(&bars->full[s], SM::kStage);
        tma_load_2d(ring + s * SM::kStage, &tm_w, &bars->full[s], b * 128, n0, p.tiles_m > 1 ? keep : once);
      };
      auto load_x = [&](int s, int b) {
        if (SM::kCodes) tma_load_2d(ring + s * SM::kStage + SM::kW, &tm_x, &bars->full[s], b * 128, row0, keep);
      };
      const int first = min(b1 - b0, stages);
      if (!p.early) asm volatile("griddepcontrol.wait;" ::: "memory");
      for (int i = 0; i < first; ++i) load_w(i, b0 + i);
      if (p.early) asm volatile("griddepcontrol.wait;" ::: "memory");
      for (int i = 0; i < first; ++i) load_x(i, b0 + i);
      int issued = first;
      for (int i = first; i < b1 - b0; ++i) {
        const int s = i % stages;
        if (!mbar_wait(&bars->empty[s], (i / stages - 1) & 1, p.status, abort_flag)) break;
        load_w(s, b0 + i);
        load_x(s, b0 + i);
        issued = i + 1;
      }
      // before the CTA leaves: every load has landed (again with a limit)
      int gave_up = 0;
      drain_ring<false>(bars->full, stages, issued, p.status, &gave_up);
    }
    __syncwarp();
  } else if (warp == kMma) {
    const uint32_t leader = elect_one();
    constexpr uint32_t idesc = idesc_i8(kSmallChannels, T);
    bool ok = aligned;
    if (!SM::kCodes) ok = ok && mbar_wait_warp(&bars->rows, 0, p.status, abort_flag);
    for (int i = 0; ok && i < b1 - b0; ++i) {
      const int s = i % stages;
      ok = mbar_wait_warp(&bars->full[s], (i / stages) & 1, p.status, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint64_t a = sw128_desc(smem_u32(ring + s * SM::kStage), 16, 1024);
      const uint64_t b = sw128_desc(smem_u32(SM::kCodes ? ring + s * SM::kStage + SM::kW : codes + i * SM::kX), 16, 1024);
#pragma unroll
      for (int k = 0; k < 4; ++k) mma_i8_by(leader, tmem, a + 2 * k, b + 2 * k, idesc, i > 0 || k > 0);
      mma_commit_by(leader, &bars->empty[s]);
    }
    mma_commit_by(leader, &bars->done);
    // the products are done before the CTA leaves, those of an aborted one too
    int gave_up = 0;
    mbar_wait_warp(&bars->done, 0, p.status, &gave_up);
    drain_ring<true>(bars->empty, stages, ok ? b1 - b0 : 0, p.status, &gave_up);
  } else {
    if constexpr (!SM::kCodes) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      if (warp < p.rows) {
        const int64_t e = warp / p.tokens, t = warp - e * p.tokens;
        const X* x = static_cast<const X*>(p.x) + e * p.x_stride[0] + t * p.x_stride[1];
        const float scale = quantise_row<T>(x, p.width, p.vec, b0 * 128, b1 * 128, codes, warp, lane);
        if (lane == 0) bars->scales[warp] = scale;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->rows);
    }
    if (warp < 4) {
      const bool in = n < p.channels;
      if (SM::kCodes) asm volatile("griddepcontrol.wait;" ::: "memory");
      if (in) {
        ws = p.ws[n];
        bias = bias_at(p, n);
      }
      O* out = static_cast<O*>(p.out) + n;
      bool ok = true;
      if constexpr (SM::kCodes) {
        if (threadIdx.x < T) bars->scales[threadIdx.x] = row0 + threadIdx.x < p.rows ? p.xs[row0 + threadIdx.x] : 0.f;
        named_bar_sync(1, 128);
      } else {
        ok = mbar_wait_warp(&bars->rows, 0, p.status, abort_flag);       // the other warps' scales
      }
      ok = mbar_wait_warp(&bars->done, 0, p.status, abort_flag) && ok && *abort_flag == 0;
      tc_fence_after();
      const uint32_t at = tmem + (static_cast<uint32_t>(32 * warp) << 16);
      int* part = reinterpret_cast<int*>(ring);
      if (__all_sync(0xffffffffu, ok)) {
        for (int t0 = 0; t0 < T && row0 + t0 < p.rows; t0 += 16) {
          uint32_t v[16];
          tmem_ld16(at + t0, v);
          tmem_ld_wait();
          if (splits > 1) {
#pragma unroll
            for (int t = 0; t < 16; ++t) part[(t0 + t) * kSmallChannels + 32 * warp + lane] = static_cast<int>(v[t]);
          } else {
#pragma unroll
            for (int t = 0; t < 16; t += 4) {
              const float4 s4 = *reinterpret_cast<const float4*>(bars->scales + t0 + t);
              const float xs[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int64_t r = row0 + t0 + t + j;
                if (in && r < p.rows) out[r * p.channels] = from_f<O>(scaled(static_cast<int>(v[t + j]), xs[j], ws, bias));
              }
            }
          }
        }
      }
    }
  }
  if (splits > 1) {
    __syncwarp();
    cluster_sync();
    if (warp < 4 && n < p.channels) {
      const int rows = min(T, p.rows - row0), share = T / splits, first = rank * share;
      constexpr int kBatch = T / 8 < 8 ? T / 8 : 8;         // tokens whose parts are in flight together
      for (int t0 = first; t0 < min(first + share, rows); t0 += kBatch) {
        const uint32_t mine = smem_u32(ring) + (t0 * kSmallChannels + 32 * warp + lane) * 4;
        int sum[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) sum[j] = 0;
        for (int c = 0; c < splits; ++c) {
          const uint32_t at = in_cta(mine, c);
          int v[kBatch];
#pragma unroll
          for (int j = 0; j < kBatch; ++j) v[j] = load_cluster(at + j * kSmallChannels * 4);
#pragma unroll
          for (int j = 0; j < kBatch; ++j) sum[j] += v[j];
        }
        O* out = static_cast<O*>(p.out) + static_cast<int64_t>(row0 + t0) * p.channels + n;
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
          if (t0 + j < rows) out[static_cast<int64_t>(j) * p.channels] = from_f<O>(scaled(sum[j], bars->scales[t0 + j], ws, bias));
      }
    }
    __syncwarp();
    cluster_sync();                        // no CTA leaves while another reads its part
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMma) tmem_dealloc(tmem, SM::kCols);
}

template <int T, typename O, typename X>
int small_launch(const CUtensorMap& mx, const CUtensorMap& mw, Linear8Params& p, cudaStream_t st) {
  using SM = SmallShape<T, X>;
  auto kernel = linear8_small_kernel<T, O, X>;
  // as many stages as there is room for: where the CTAs do not fill the SMs twice one has an SM to itself (16 x 4,096 x 16,384:
  // the loads in flight are all that counts)
  const int64_t ctas = static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.splits;
  const int part = (p.blocks + p.splits - 1) / p.splits;
  const uint32_t room = (ctas <= sm_count() ? SM::kMost : SM::kMost / 2) - 1024, fixed = SM::kBars + SM::rows(part);
  p.rows_bytes = SM::rows(part);
  p.stages = fixed + 2 * SM::kStage > room ? 2 : static_cast<int>((room - fixed) / SM::kStage);
  p.stages = std::max(2, std::min({p.stages, kSmallStages, part}));
  const uint32_t bytes = fixed + p.stages * SM::kStage;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::kMost) != cudaSuccess) return HTRC_ERR_CUDA;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(SM::kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(p.splits);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, mx, mw, p) == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
}

// ------------------------------------------------------------------------------------------------ many tokens
// Of the pair's 256 x 256 tile each CTA holds the sums of its own 128 tokens (TMEM lanes) and all 256 channels (columns),
// twice.  Warps 0-7: the way out, 32 tokens x 128 channels each; 8: TMA; 9: MMA issue (the leader's, rank 0).
constexpr int kPairThreads = 320, kPairStages = 5, kPairOuts = 2;
constexpr int kPairRows = 256, kPairChannels = 256;         // of the pair
constexpr uint32_t kPairTile = 128 * 128, kPairStage = 2 * kPairTile;
constexpr uint32_t kPairOut = kPairStages * kPairStage, kPairTable = kPairOut + 8 * kPairOuts * 4096, kPairBars = kPairTable + 2 * kPairChannels * 4;
constexpr uint32_t kPairBytes = kPairBars + 192;
constexpr int kPairGroup = 8;                               // row tiles that are walked together: their operands stay in L2

struct PairBars {
  uint64_t full[kPairStages], empty[kPairStages], sums_full[2], sums_empty[2], idle;
  uint32_t tmem;
  int abort_flag;
};
static_assert(sizeof(PairBars) <= 192 && kPairBytes <= 232448, "shared memory");

// mbarrier waits on arrivals from the other CTA
__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, int* status, volatile int* abort_flag) {
  bool ok = try_wait_cluster(bar, parity);
  if (!ok) {
    const long long t0 = clock64();
    while (!(ok = try_wait_cluster(bar, parity))) {
      if (*abort_flag) break;
      if (clock64() - t0 > kWaitCycles) {
        *abort_flag = 1;
        flag_status(status, ST_WAIT_TIMEOUT);
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ void arrive_in(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// a load into this CTA whose bytes are counted by a barrier of the pair's leader
__device__ __forceinline__ void pair_load(void* dst, const CUtensorMap* map, uint32_t cluster_bar, int x, int y, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(cluster_bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void pair_mma(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(leader)
      : "memory");
}
// an arrival on the barrier of either CTA once the products issued so far are done
__device__ __forceinline__ void pair_commit(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}" ::"r"(
          smem_u32(bar)),
      "r"(leader), "h"(static_cast<uint16_t>(3))
      : "memory");
}
__device__ __forceinline__ void store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}

// the pair's tile t: groups of kPairGroup row tiles, within one its row tiles first
__device__ __forceinline__ void pair_tile(const Linear8Params& p, int t, int& row, int& channel) {
  const int size = kPairGroup * p.tiles_n, group = t / size, first = group * kPairGroup;
  const int high = min(kPairGroup, p.tiles_m - first), rest = t - group * size;
  row = (first + rest % high) * kPairRows;
  channel = rest / high * kPairChannels;
}

template <typename O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    linear8_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                        const __grid_constant__ CUtensorMap tm_o, const __grid_constant__ Linear8Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  PairBars* bars = reinterpret_cast<PairBars*>(smem + kPairBars);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool aligned = (smem_u32(smem) & 1023) == 0;        // the same in either CTA
  if (threadIdx.x == 0) {
    for (int i = 0; i < kPairStages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->sums_full[i], 1);
      mbar_init(&bars->sums_empty[i], 16);
    }
    mbar_init(&bars->idle, 1);
    bars->abort_flag = !aligned;
    if (!aligned) flag_status(p.status, ST_WAIT_TIMEOUT);
    fence_barrier_init();
  }
  __syncthreads();
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&bars->tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  const int pairs = gridDim.x / 2, first = blockIdx.x / 2, tiles = p.tiles_m * p.tiles_n;

  if (warp == 8) {
    int issued = 0;
    if (lane == 0 && aligned) {
      const uint64_t keep = policy_evict_last(), normal = policy_evict_normal();
      bool ok = true;
      for (int t = first; ok && t < tiles; t += pairs) {
        int row, channel;
        pair_tile(p, t, row, channel);
        row += 128 * rank;
        channel += 128 * rank;
        for (int b = 0; b < p.blocks; ++b) {
          const int s = issued % kPairStages;
          if (issued >= kPairStages && !mbar_wait(&bars->empty[s], (issued / kPairStages - 1) & 1, p.status, abort_flag)) {
            ok = false;
            break;
          }
          if (rank == 0) expect_tx(&bars->full[s], 2 * kPairStage);
          const uint32_t bar = in_cta(smem_u32(&bars->full[s]), 0);
          pair_load(smem + s * kPairStage, &tm_x, bar, b * 128, row, normal);
          pair_load(smem + s * kPairStage + kPairTile, &tm_w, bar, b * 128, channel, keep);
          ++issued;
        }
      }
      // every load of the pair has landed and every stage has been read, before either CTA leaves (again with a limit)
      int gave_up = 0;
      if (rank == 0) drain_ring<false>(bars->full, kPairStages, issued, p.status, &gave_up);
      if (ok) drain_ring<false>(bars->empty, kPairStages, issued, p.status, &gave_up);
    }
    __syncwarp();
  } else if (warp == 9) {
    if (rank == 0) {
      const uint32_t leader = elect_one();
      constexpr uint32_t idesc = idesc_i8(256, 256);
      bool ok = aligned;
      int step = 0, turn = 0;
      for (int t = first; ok && t < tiles; t += pairs, ++turn) {
        const int half = turn & 1;
        if (turn >= 2) ok = wait_cluster(&bars->sums_empty[half], (turn / 2 - 1) & 1, p.status, abort_flag);
        tc_fence_after();
        for (int b = 0; ok && b < p.blocks; ++b, ++step) {
          const int s = step % kPairStages;
          ok = wait_cluster(&bars->full[s], (step / kPairStages) & 1, p.status, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint64_t a = sw128_desc(smem_u32(smem + s * kPairStage), 16, 1024);
          const uint64_t w = sw128_desc(smem_u32(smem + s * kPairStage + kPairTile), 16, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            pair_mma(leader, tmem + 256 * half, a + 2 * k, w + 2 * k, idesc, b > 0 || k > 0);
          pair_commit(leader, &bars->empty[s]);
        }
        if (ok) pair_commit(leader, &bars->sums_full[half]);
      }
      // the products are done before the CTAs leave, those of an aborted launch too
      int gave_up = 0;
      asm volatile(
          "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
          "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(&bars->idle)),
          "r"(leader)
          : "memory");
      mbar_wait_warp(&bars->idle, 0, p.status, &gave_up);
    }
  } else {
    constexpr int kCols = 128 / sizeof(O);                  // of a staged 128-byte row
    float* table = reinterpret_cast<float*>(smem + kPairTable);
    uint8_t* const stages = smem + kPairOut + warp * kPairOuts * 4096;
    const int quarter = warp & 3, side = warp >> 2;
    const uint32_t at = tmem + (static_cast<uint32_t>(32 * quarter) << 16) + 128 * side;
    const uint32_t leaders[2] = {in_cta(smem_u32(&bars->sums_empty[0]), 0), in_cta(smem_u32(&bars->sums_empty[1]), 0)};
    // a tile's scales and biases, a thread a channel, and the thread's row's scale: read one tile ahead
    float2 term = make_float2(0.f, 0.f);
    float xs = 0.f;
    auto fetch = [&](int t) {
      if (t >= tiles) return;
      int row, channel;
      pair_tile(p, t, row, channel);
      row += 128 * rank + 32 * quarter + lane;
      const int n = channel + threadIdx.x;
      term = n < p.channels ? make_float2(__ldg(p.ws + n), bias_at(p, n)) : make_float2(0.f, 0.f);
      xs = row < p.rows ? __ldg(p.xs + row) : 0.f;
    };
    fetch(first);
    bool ok = aligned;
    int turn = 0, out_turn = 0;
    // (a warp whose wait ran out goes on to the barriers that the others stand at, without work)
    for (int t = first; t < tiles; t += pairs, ++turn) {
      int row, channel;
      pair_tile(p, t, row, channel);
      row += 128 * rank + 32 * quarter;
      const int half = turn & 1;
      named_bar_sync(1, 256);
      table[threadIdx.x] = term.x;
      table[kPairChannels + threadIdx.x] = term.y;
      const float row_scale = xs;
      named_bar_sync(1, 256);
      fetch(t + pairs);
      ok = ok && wait_cluster(&bars->sums_full[half], (turn / 2) & 1, p.status, abort_flag);
      if (!ok) continue;
      tc_fence_after();
      channel += 128 * side;
      const float* ws = table + 128 * side;
#pragma unroll 1
      for (int c = 0; c < 128; c += kCols) {
        uint8_t* const stage = stages + (out_turn++ % kPairOuts) * 4096;
        asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kPairOuts - 1) : "memory");      // lane 0's: the stage has left
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kCols; i += 32) {
          uint32_t v[32];
          tmem_ld32(at + 256 * half + c + i, v);
          tmem_ld_wait();
          if (c + kCols == 128 && i + 32 == kCols) {        // the last read of these sums
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_in(leaders[half]);
          }
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(ws + c + i + j);
            const float4 b4 = *reinterpret_cast<const float4*>(ws + kPairChannels + c + i + j);
            const float y0 = scaled(static_cast<int>(v[j]), row_scale, s4.x, b4.x), y1 = scaled(static_cast<int>(v[j + 1]), row_scale, s4.y, b4.y);
            const float y2 = scaled(static_cast<int>(v[j + 2]), row_scale, s4.z, b4.z), y3 = scaled(static_cast<int>(v[j + 3]), row_scale, s4.w, b4.w);
            if constexpr (sizeof(O) == 4) {
              v[j] = __float_as_uint(y0);
              v[j + 1] = __float_as_uint(y1);
              v[j + 2] = __float_as_uint(y2);
              v[j + 3] = __float_as_uint(y3);
            } else if constexpr (std::is_same<O, __nv_bfloat16>::value) {
              v[j / 2] = pack_bf16x2(y0, y1);
              v[j / 2 + 1] = pack_bf16x2(y2, y3);
            } else {
              v[j / 2] = pack_f16x2(y0, y1);
              v[j / 2 + 1] = pack_f16x2(y2, y3);
            }
          }
          constexpr int kPieces = 32 * sizeof(O) / 16;      // 16-byte pieces of these columns
#pragma unroll
          for (int q = 0; q < kPieces; ++q)
            st_shared_v4(smem_u32(stage) + sw128_off(lane, i * sizeof(O) / 16 + q), v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        }
        if (!p.direct) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (row < p.rows && channel + c < p.channels) store_2d(&tm_o, stage, channel + c, row);
            bulk_commit_group();
          }
        } else {
          // rows of any alignment, by 4-byte words, a row's neighbours together (19,000 x 1,024 x 3,499 in bfloat16 143 us,
          // aligned 75)
          __syncwarp();
          const int cols = min(kCols, p.channels - (channel + c)), high = min(32, p.rows - row);
          O* out = static_cast<O*>(p.out) + static_cast<int64_t>(row) * p.channels + channel + c;
#pragma unroll 4
          for (int r = 0; r < high; ++r, out += p.channels) {
            const uint32_t word = *reinterpret_cast<const uint32_t*>(stage + sw128_off(r, lane / 4) + lane % 4 * 4);
            if constexpr (sizeof(O) == 4) {
              if (lane < cols) reinterpret_cast<uint32_t*>(out)[lane] = word;
            } else {
              // where the row starts inside a word its first element stands alone, and the words hold the ones after it
              const uint32_t next = __shfl_down_sync(0xffffffffu, word, 1);
              const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(out) >> 1 & 1), e = 2 * lane + odd;
              const uint32_t two = odd ? __byte_perm(word, next, 0x5432) : word;
              unsigned short* to = reinterpret_cast<unsigned short*>(out);
              if (e + 1 < cols && e + 1 < kCols) *reinterpret_cast<uint32_t*>(to + e) = two;
              else if (e < cols) to[e] = static_cast<unsigned short>(two);
              if (odd && lane == 0 && cols > 0) to[0] = static_cast<unsigned short>(word);
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) bulk_wait_group0();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();                          // neither CTA leaves while the other may still signal it
  tc_fence_after();
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <typename O>
int pair_launch(const CUtensorMap& mx, const CUtensorMap& mw, const CUtensorMap& mo, const Linear8Params& p, cudaStream_t st) {
  auto kernel = linear8_pair_kernel<O>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairBytes) != cudaSuccess) return HTRC_ERR_CUDA;
  const int pairs = std::min(sm_count() / 2, p.tiles_m * p.tiles_n);
  kernel<<<2 * pairs, kPairThreads, kPairBytes, st>>>(mx, mw, mo, p);
  return cudaGetLastError() == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
}

// ------------------------------------------------------------------------------------------------ host
bool float_type(int t) { return t == HTRC_LAYER_F32 || t == HTRC_LAYER_BF16 || t == HTRC_LAYER_F16; }

bool code_map(CUtensorMap* m, const void* base, int64_t rows, int width, int64_t pitch, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(width), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(pitch)};
  const uint32_t box[2] = {128, static_cast<uint32_t>(box_rows)};
  return make_tiled_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, true);
}

int64_t code_pitch(int width) { return (static_cast<int64_t>(width) + 15) / 16 * 16; }
size_t code_bytes(const HtrcLinear8Args* a) {
  return (static_cast<size_t>(a->batch * a->tokens) * code_pitch(a->width) + 255) / 256 * 256;
}

int linear8_validate(const HtrcLinear8Args* a) {
  if (a == nullptr || a->batch < 0 || a->tokens < 0 || a->width < 1 || a->channels < 1) return HTRC_ERR_ARG;
  const bool codes = a->dtype == HTRC_LAYER_I8;
  if ((!codes && !float_type(a->dtype)) || !float_type(a->out_dtype) || !float_type(a->bias_dtype)) return HTRC_ERR_ARG;
  const int widest = codes ? static_cast<int>(HTRC_LINEAR8_MAX_WIDTH) : static_cast<int>(HTRC_NORM_MAX_WIDTH);
  if (a->width > widest) return HTRC_ERR_UNSUPPORTED;
  constexpr int64_t kMax = (int64_t(1) << 31) - 1024;
  if (a->channels > kMax || (a->tokens > 0 && a->batch >= kMax / a->tokens)) return HTRC_ERR_UNSUPPORTED;
  // the few tokens' and the pairs' tiles are counted in 32 bits
  if ((a->batch * a->tokens + 127) / 128 * ((static_cast<int64_t>(a->channels) + 127) / 128) >= (int64_t(1) << 30))
    return HTRC_ERR_UNSUPPORTED;
  return HTRC_OK;
}

// Parts of the width that a tile of few tokens is shared out to: split while the parts are longer than 8 blocks and leave SMs
// idle.  64 x 4,096 x 4,096 10.2 us in 4 parts and 15 whole; 16 x 1,024 x 4,096 4.1 whole and 5.4 in 2; 16 x 4,096 x 16,384 14.1
// whole and 16.4 in 2.
int split_width(int64_t tiles, int blocks) {
  int splits = 1;
  while (splits < 8 && tiles * splits * 4 <= 3 * sm_count() && blocks > 8 * splits) splits *= 2;
  return splits;
}

// Whether the product quantises its float rows itself: few of them, and no more of the width to a CTA than it has room for.
// Every CTA reads all of them, which costs more than the launch that it saves where the weights take longer than that launch:
// 16 x 4,096 x 16,384 19.2 us by itself and 16.5 behind the rows' kernel; 16 x 4,096 x 4,096 10.8 either way, and one launch.
bool quantises(const HtrcLinear8Args* a) {
  if (a->dtype == HTRC_LAYER_I8 || a->batch * a->tokens > kFewTokens) return false;
  if (a->batch * a->tokens * a->width > 32768 && static_cast<int64_t>(a->width) * a->channels > (32 << 20)) return false;
  const int blocks = (a->width + 127) / 128, splits = split_width((a->channels + kSmallChannels - 1) / kSmallChannels, blocks);
  return (blocks + splits - 1) / splits <= kFewBlocks;
}

template <typename O, typename X>
int few_launch(Linear8Params& p, const HtrcLinear8Args* a, cudaStream_t st) {
  CUtensorMap mw;
  if (!code_map(&mw, a->w, p.channels, a->width, a->w_pitch, kSmallChannels)) return HTRC_ERR_CUDA;
  p.tiles_m = 1;
  p.tiles_n = (p.channels + kSmallChannels - 1) / kSmallChannels;
  p.splits = split_width(p.tiles_n, p.blocks);
  return small_launch<kFewTokens, O, X>(mw, mw, p, st);
}

template <typename O>
int linear8_launch(Linear8Params& p, const int8_t* x, int64_t pitch, const HtrcLinear8Args* a, cudaStream_t st) {
  // Pairs where their tiles occupy half of the SMs (1,024 x 4,096 x 4,096: 18.5 us, by tiles of 64 tokens 30.1), not for so few
  // tokens that most of a tile would be empty.
  const int64_t pairs = (static_cast<int64_t>(p.rows) + 255) / 256 * ((static_cast<int64_t>(p.channels) + 255) / 256);
  if (p.rows > 128 && pairs >= 32) {
    CUtensorMap mx, mw, mo;
    constexpr int es = sizeof(O);
    p.direct = p.channels * es % 16 != 0 || reinterpret_cast<uintptr_t>(p.out) % 16 != 0;
    if (!code_map(&mx, x, p.rows, a->width, pitch, 128) || !code_map(&mw, a->w, p.channels, a->width, a->w_pitch, 128))
      return HTRC_ERR_CUDA;
    mo = mx;
    if (!p.direct) {
      const uint64_t dims[2] = {static_cast<uint64_t>(p.channels), static_cast<uint64_t>(p.rows)};
      const uint64_t strides[1] = {static_cast<uint64_t>(p.channels) * es};
      const uint32_t box[2] = {128 / es, 32};
      const CUtensorMapDataType type = es == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : std::is_same<O, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                              : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
      if (!make_tiled_map(&mo, type, 2, p.out, dims, strides, box, true)) return HTRC_ERR_CUDA;
    }
    p.tiles_m = (p.rows + kPairRows - 1) / kPairRows;
    p.tiles_n = (p.channels + kPairChannels - 1) / kPairChannels;
    return pair_launch<O>(mx, mw, mo, p, st);
  }
  // tokens of a tile: 64 (512 x 1,024 x 4,096: 8.3 us, of 128 tokens 11.5, of 32 11.9), fewer where there are fewer
  const int tile = p.rows <= 16 ? 16 : p.rows <= 32 ? 32 : 64;
  CUtensorMap mx, mw;
  if (!code_map(&mx, x, p.rows, a->width, pitch, tile) || !code_map(&mw, a->w, p.channels, a->width, a->w_pitch, kSmallChannels))
    return HTRC_ERR_CUDA;
  p.tiles_m = (p.rows + tile - 1) / tile;
  p.tiles_n = (p.channels + kSmallChannels - 1) / kSmallChannels;
  p.splits = split_width(static_cast<int64_t>(p.tiles_m) * p.tiles_n, p.blocks);
  if (tile == 16) return small_launch<16, O, int8_t>(mx, mw, p, st);
  if (tile == 32) return small_launch<32, O, int8_t>(mx, mw, p, st);
  return small_launch<64, O, int8_t>(mx, mw, p, st);
}

template <typename O>
int linear8_run(Linear8Params& p, const int8_t* x, int64_t pitch, const HtrcLinear8Args* a, cudaStream_t st) {
  if (p.x == nullptr) return linear8_launch<O>(p, x, pitch, a, st);
  if (a->dtype == HTRC_LAYER_F32) return few_launch<O, float>(p, a, st);
  return a->dtype == HTRC_LAYER_BF16 ? few_launch<O, __nv_bfloat16>(p, a, st) : few_launch<O, __half>(p, a, st);
}

int linear8_forward(const HtrcLinear8Args* a, cudaStream_t st) {
  int rc = linear8_validate(a);
  if (rc != HTRC_OK) return rc;
  const int64_t rows = a->batch * a->tokens;
  const bool codes = a->dtype == HTRC_LAYER_I8;
  if (!a->w || !a->w_scales || reinterpret_cast<uintptr_t>(a->w) % 16 || a->w_pitch < a->width || a->w_pitch % 16)
    return HTRC_ERR_ARG;
  if (rows > 0) {
    if (!a->x || !a->out) return HTRC_ERR_ARG;
    if (codes) {
      const int64_t pitch = a->tokens > 1 ? a->x_stride[1] : a->x_stride[0];
      if (!a->x_scales || reinterpret_cast<uintptr_t>(a->x) % 16) return HTRC_ERR_ARG;
      if (rows > 1 && (pitch < a->width || pitch % 16)) return HTRC_ERR_ARG;
      if (a->batch > 1 && a->tokens > 1 && a->x_stride[0] != a->tokens * a->x_stride[1]) return HTRC_ERR_ARG;
    }
  }
  if (!device_is_b200()) return HTRC_ERR_DEVICE;
  if (rows == 0) return HTRC_OK;
  Linear8Params p{};
  const int8_t* x = static_cast<const int8_t*>(a->x);
  int64_t pitch = rows > 1 ? (a->tokens > 1 ? a->x_stride[1] : a->x_stride[0]) : code_pitch(a->width);
  p.xs = a->x_scales;
  if (quantises(a)) {
    const int es = a->dtype == HTRC_LAYER_F32 ? 4 : 2;
    p.x = a->x;
    p.x_stride[0] = a->x_stride[0];
    p.x_stride[1] = a->x_stride[1];
    p.tokens = a->tokens;
    p.width = a->width;
    p.vec = a->width * es % 16 == 0 && reinterpret_cast<uintptr_t>(a->x) % 16 == 0 && a->x_stride[0] * es % 16 == 0 &&
            a->x_stride[1] * es % 16 == 0;
  } else if (!codes) {
    const size_t at = code_bytes(a);
    if (a->workspace == nullptr || a->workspace_bytes < at + rows * sizeof(float) ||
        reinterpret_cast<uintptr_t>(a->workspace) % 256)
      return HTRC_ERR_WORKSPACE;
    int8_t* to = static_cast<int8_t*>(a->workspace);
    float* scales = reinterpret_cast<float*>(to + at);
    pitch = code_pitch(a->width);
    rc = quantize_rows(a->x, a->dtype, a->batch, a->tokens, a->width, a->x_stride, to, pitch, scales, st);
    if (rc != HTRC_OK) return rc;
    x = to;
    p.xs = scales;
  }
  p.rows = static_cast<int>(rows);
  p.channels = a->channels;
  p.blocks = (a->width + 127) / 128;
  p.ws = a->w_scales;
  p.bias = a->bias;
  p.bias_dtype = a->bias_dtype;
  p.out = a->out;
  p.status = a->status;
  // the rows' own kernel starts when all before it has ended, the product under the rows' kernel
  p.early = !codes && p.x == nullptr;
  if (a->out_dtype == HTRC_LAYER_F32) return linear8_run<float>(p, x, pitch, a, st);
  if (a->out_dtype == HTRC_LAYER_BF16) return linear8_run<__nv_bfloat16>(p, x, pitch, a, st);
  return linear8_run<__half>(p, x, pitch, a, st);
}

}  // namespace

}  // namespace htrc

extern "C" {

int htrc_linear8_workspace_size(const HtrcLinear8Args* args, size_t* bytes) {
  if (bytes == nullptr) return HTRC_ERR_ARG;
  const int rc = htrc::linear8_validate(args);
  if (rc != HTRC_OK) return rc;
  *bytes = args->dtype == HTRC_LAYER_I8 || htrc::quantises(args)
               ? 0
               : htrc::code_bytes(args) + static_cast<size_t>(args->batch * args->tokens) * 4;
  return HTRC_OK;
}

int htrc_linear8_forward(const HtrcLinear8Args* args, htrc_stream_t stream) {
  return htrc::linear8_forward(args, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
