// Matrix product in 8-bit integers with a scale per token and channel:
//   out[r][n] = (sum_k x[r][k] w[n][k]) x_scales[r] w_scales[n] + bias[n]
// on tcgen05 (kind::i8: int32 sums in TMEM, exact), the scales and the bias in float32 on the way out.
//
// Few tokens (linear8_small_kernel): the weights are what is read, so they take the product's 128-row side, a tile of
// 16 to 128 tokens its other.  Where the tiles alone leave SMs idle a cluster shares a tile, each CTA a range of the width;
// their integer sums are added over distributed shared memory, which changes no result.
//
// Many tokens (linear8_pair_kernel): two CTAs on neighbouring SMs share a tile of 256 tokens x 256 channels (cta_group::2),
// each loading half of either operand; persistent, two accumulators in TMEM, so that a tile leaves under the next one's
// products.
#include <algorithm>
#include <cmath>

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
  bool early;                               // few tokens: the kernel before this one did not write the weights
  bool direct;                              // pair kernel: the output's rows are not 16-byte aligned
};

__device__ __forceinline__ float bias_at(const Linear8Params& p, int n) {
  if (p.bias == nullptr) return 0.f;
  if (p.bias_dtype == HTRC_LAYER_F32) return __ldg(static_cast<const float*>(p.bias) + n);
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
constexpr int kSmallThreads = 192;          // warps 0-3: the way out; 4: TMA; 5: MMA
constexpr int kSmallChannels = 128;

template <int T>
struct SmallShape {
  static constexpr int kStages = T <= 32 ? 5 : T <= 64 ? 4 : 3;      // two CTAs per SM
  static constexpr uint32_t kW = kSmallChannels * 128, kX = T * 128, kStage = kW + kX;
  static constexpr uint32_t kCols = T < 32 ? 32 : T;
  static constexpr uint32_t kBars = kStages * kStage, kBytes = kBars + 128;
  static_assert(T * kSmallChannels * 4 <= kBars, "the parts of a split tile reuse the stages");
};

struct SmallBars {
  uint64_t full[5], empty[5], done;
  uint32_t tmem;
  int abort_flag;
};
static_assert(sizeof(SmallBars) <= 128, "barriers");

template <int T, typename O>
__global__ void __launch_bounds__(kSmallThreads)
    linear8_small_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                         const __grid_constant__ Linear8Params p) {
  using SM = SmallShape<T>;
  extern __shared__ __align__(1024) uint8_t smem[];
  SmallBars* bars = reinterpret_cast<SmallBars*>(smem + SM::kBars);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool aligned = (smem_u32(smem) & 1023) == 0;      // the swizzled tiles need it
  if (threadIdx.x == 0) {
    for (int i = 0; i < SM::kStages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    mbar_init(&bars->done, 1);
    bars->abort_flag = !aligned;
    if (!aligned) flag_status(p.status, ST_WAIT_TIMEOUT);
    fence_barrier_init();
  }
  if (warp == 5) tmem_alloc(&bars->tmem, SM::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int splits = p.splits, rank = blockIdx.x % splits, tile = blockIdx.x / splits;
  const int n0 = tile / p.tiles_m * kSmallChannels, row0 = tile % p.tiles_m * T;
  const int b0 = static_cast<int>(static_cast<int64_t>(p.blocks) * rank / splits);
  const int b1 = static_cast<int>(static_cast<int64_t>(p.blocks) * (rank + 1) / splits);

  if (warp == 4) {
    if (lane == 0 && aligned) {
      const uint64_t once = policy_evict_first(), keep = policy_evict_last();
      auto load_w = [&](int s, int b) {
        expect_tx(&bars->full[s], SM::kStage);
        tma_load_2d(smem + s * SM::kStage, &tm_w, &bars->full[s], b * 128, n0, p.tiles_m > 1 ? keep : once);
      };
      auto load_x = [&](int s, int b) {
        tma_load_2d(smem + s * SM::kStage + SM::kW, &tm_x, &bars->full[s], b * 128, row0, keep);
      };
      const int first = min(b1 - b0, SM::kStages);
      if (!p.early) asm volatile("griddepcontrol.wait;" ::: "memory");
      for (int i = 0; i < first; ++i) load_w(i, b0 + i);
      if (p.early) asm volatile("griddepcontrol.wait;" ::: "memory");
      for (int i = 0; i < first; ++i) load_x(i, b0 + i);
      int issued = first;
      for (int i = first; i < b1 - b0; ++i) {
        const int s = i % SM::kStages;
        if (!mbar_wait(&bars->empty[s], (i / SM::kStages - 1) & 1, p.status, abort_flag)) break;
        load_w(s, b0 + i);
        load_x(s, b0 + i);
        issued = i + 1;
      }
      // before the CTA leaves: every load has landed (again with a limit)
      int gave_up = 0;
      drain_ring<false>(bars->full, SM::kStages, issued, p.status, &gave_up);
    }
    __syncwarp();
  } else if (warp == 5) {
    const uint32_t leader = elect_one();
    constexpr uint32_t idesc = idesc_i8(kSmallChannels, T);
    bool ok = aligned;
    for (int i = 0; ok && i < b1 - b0; ++i) {
      const int s = i % SM::kStages;
      ok = mbar_wait_warp(&bars->full[s], (i / SM::kStages) & 1, p.status, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint64_t a = sw128_desc(smem_u32(smem + s * SM::kStage), 16, 1024);
      const uint64_t b = sw128_desc(smem_u32(smem + s * SM::kStage + SM::kW), 16, 1024);
#pragma unroll
      for (int k = 0; k < 4; ++k) mma_i8_by(leader, tmem, a + 2 * k, b + 2 * k, idesc, i > 0 || k > 0);
      mma_commit_by(leader, &bars->empty[s]);
    }
    mma_commit_by(leader, &bars->done);
    // the products are done before the CTA leaves, those of an aborted one too
    int gave_up = 0;
    mbar_wait_warp(&bars->done, 0, p.status, &gave_up);
    drain_ring<true>(bars->empty, SM::kStages, ok ? b1 - b0 : 0, p.status, &gave_up);
  } else {
    const int n = n0 + 32 * warp + lane;
    const bool in = n < p.channels;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float ws = in ? __ldg(p.ws + n) : 0.f, bias = in ? bias_at(p, n) : 0.f;
    O* out = static_cast<O*>(p.out) + n;
    const bool ok = mbar_wait_warp(&bars->done, 0, p.status, abort_flag) && *abort_flag == 0;
    tc_fence_after();
    const uint32_t at = tmem + (static_cast<uint32_t>(32 * warp) << 16);
    int* part = reinterpret_cast<int*>(smem);
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
          for (int t = 0; t < 16; ++t) {
            const int64_t r = row0 + t0 + t;
            if (in && r < p.rows) out[r * p.channels] = from_f<O>(scaled(static_cast<int>(v[t]), __ldg(p.xs + r), ws, bias));
          }
        }
      }
    }
  }
  if (splits > 1) {
    __syncwarp();
    cluster_sync();
    if (warp < 4) {
      const int n = n0 + 32 * warp + lane;
      if (n < p.channels) {
        const float ws = __ldg(p.ws + n), bias = bias_at(p, n);
        const int rows = min(T, p.rows - row0);
        for (int t = rank; t < rows; t += splits) {
          const uint32_t mine = smem_u32(smem) + (t * kSmallChannels + 32 * warp + lane) * 4;
          int sum = 0;
          for (int c = 0; c < splits; ++c) sum += load_cluster(in_cta(mine, c));
          const int64_t r = row0 + t;
          static_cast<O*>(p.out)[r * p.channels + n] = from_f<O>(scaled(sum, __ldg(p.xs + r), ws, bias));
        }
      }
    }
    __syncwarp();
    cluster_sync();                        // no CTA leaves while another reads its part
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, SM::kCols);
}

template <int T, typename O>
int small_launch(const CUtensorMap& mx, const CUtensorMap& mw, const Linear8Params& p, cudaStream_t st) {
  using SM = SmallShape<T>;
  auto kernel = linear8_small_kernel<T, O>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::kBytes) != cudaSuccess) return HTRC_ERR_CUDA;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.splits));
  cfg.blockDim = dim3(kSmallThreads);
  cfg.dynamicSmemBytes = SM::kBytes;
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

template <typename O>
int linear8_launch(Linear8Params& p, const int8_t* x, int64_t pitch, const HtrcLinear8Args* a, cudaStream_t st) {
  const int tile = p.rows <= 16 ? 16 : p.rows <= 32 ? 32 : p.rows <= 64 ? 64 : 128;
  CUtensorMap mx, mw;
  if (!code_map(&mx, x, p.rows, a->width, pitch, tile) || !code_map(&mw, a->w, p.channels, a->width, a->w_pitch, kSmallChannels))
    return HTRC_ERR_CUDA;
  p.tiles_m = (p.rows + tile - 1) / tile;
  p.tiles_n = (p.channels + kSmallChannels - 1) / kSmallChannels;
  const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  p.splits = 1;
  while (p.splits < 8 && tiles * p.splits * 2 <= 2 * sm_count() && p.blocks >= 4 * p.splits) p.splits *= 2;
  if (tile == 16) return small_launch<16, O>(mx, mw, p, st);
  if (tile == 32) return small_launch<32, O>(mx, mw, p, st);
  if (tile == 64) return small_launch<64, O>(mx, mw, p, st);
  return small_launch<128, O>(mx, mw, p, st);
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
  if (!codes) {
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
  p.early = !codes;
  if (a->out_dtype == HTRC_LAYER_F32) return linear8_launch<float>(p, x, pitch, a, st);
  if (a->out_dtype == HTRC_LAYER_BF16) return linear8_launch<__nv_bfloat16>(p, x, pitch, a, st);
  return linear8_launch<__half>(p, x, pitch, a, st);
}

}  // namespace

}  // namespace htrc

extern "C" {

int htrc_linear8_workspace_size(const HtrcLinear8Args* args, size_t* bytes) {
  if (bytes == nullptr) return HTRC_ERR_ARG;
  const int rc = htrc::linear8_validate(args);
  if (rc != HTRC_OK) return rc;
  *bytes = args->dtype == HTRC_LAYER_I8 ? 0 : htrc::code_bytes(args) + static_cast<size_t>(args->batch * args->tokens) * 4;
  return HTRC_OK;
}

int htrc_linear8_forward(const HtrcLinear8Args* args, htrc_stream_t stream) {
  return htrc::linear8_forward(args, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
