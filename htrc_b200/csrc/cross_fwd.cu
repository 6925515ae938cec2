// Cross attention to an encoder's states of another length, forward, and the checks its C entries share.
//
// A CTA owns 128 query rows of one head and walks the keys in blocks of 128:  S = Q K^T (tcgen05, float32 in TMEM),
// one thread per row takes the block's maximum and P = exp2(S scale log2 e - m), P goes back over S in TMEM as 16-bit
// words and O += P V accumulates in TMEM; the sum of P is kept in float32 from the unrounded values.  The running
// maximum is lazy: O is rescaled only when a row's maximum grew by more than 2^8 (P <= 256 until then).
//
// Two CTAs share an SM (256 TMEM columns and about 97 KB of shared memory each), so one CTA's products run under the
// other's exponentials, and prologues and epilogues hide behind the neighbour; inside a CTA the chain S -> P -> O is
// serial.  K and V are single buffers of 128 rows: K is free as soon as S is done, V as soon as O is.
//
// Rounding: P is rounded to the operands' 16-bit type for the second product (a relative 2^-9 for bfloat16, of
// weights whose errors average out over the row); out is rounded once from float32.
//
// Warps 0-3: softmax, rows 32 w ..; warp 4: TMA; warp 5: MMA issue, and the zeroing of excluded keys' values.
#include <algorithm>
#include <cmath>

#include "cross.cuh"

namespace htrc {

namespace {

constexpr int kXThreads = 192;
constexpr int kXRows = 128, kXKeys = 128;
constexpr uint32_t kXChunk = 128 * 128;            // 128 rows of 64 16-bit elements
constexpr uint32_t kXColS = 0, kXColO = 128, kXCols = 256;
constexpr float kXRescale = 8.0f;

struct CrossBars {
  uint64_t q_full, k_full, k_empty, v_full, v_empty, s_full, p_full, o_full;
  uint32_t tmem_base;
  int abort_flag;
};

template <int DP>
struct CrossFwdSmem {
  static constexpr int kChunks = DP / 64;
  static constexpr uint32_t kTile = kChunks * kXChunk;
  static constexpr uint32_t kQ = 0, kK = kTile, kV = 2 * kTile, kBias = 3 * kTile, kBars = kBias + 2 * kXKeys * 4;
  // at least a third of the SM: never more than two CTAs share its 512 TMEM columns
  static constexpr uint32_t kBytes = kBars + 256 + 1024 < 80 * 1024 ? 80 * 1024 : kBars + 256 + 1024;
};

struct CrossFwdParams {
  CrossShape s;
  float* lse;
  int tiles;
  int* status;
};

template <int DP, bool BF, int KIND>
__global__ void __launch_bounds__(kXThreads, 2)
    cross_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                     const __grid_constant__ CrossFwdParams p) {
  using SM = CrossFwdSmem<DP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  CrossBars* bars = reinterpret_cast<CrossBars*>(smem + SM::kBars);
  volatile int* abort_flag = &bars->abort_flag;
  int* status = p.status;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x % p.tiles;
  const int bh = blockIdx.x / p.tiles;
  const int h = bh % p.s.heads, b = bh / p.s.heads, hk = h / p.s.group;
  const int row0 = tile * kXRows;
  const int count = key_count(p.s, b);
  const int blocks = (count + kXKeys - 1) / kXKeys;
  const int64_t mask_at = b * p.s.mask.sb + h * p.s.mask.sh;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->k_full, 1);
    mbar_init(&bars->k_empty, 1);
    mbar_init(&bars->v_full, 1);
    mbar_init(&bars->v_empty, 1);
    mbar_init(&bars->s_full, 1);
    mbar_init(&bars->p_full, 128);
    mbar_init(&bars->o_full, 1);
    bars->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 5) tmem_alloc(&bars->tmem_base, kXCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  if (warp == 4) {
    // ------------------------------------------------------------------ TMA
    const uint64_t pol_q = policy_evict_first(), pol_kv = policy_evict_last();
    const uint32_t leader = elect_one();
    if (leader && blocks > 0) {
      mbar_arrive_expect_tx(&bars->q_full, SM::kTile);
      for (int c = 0; c < SM::kChunks; ++c)
        tma_load_4d(smem + SM::kQ + c * kXChunk, &tm_q, &bars->q_full, 64 * c, row0, h * p.s.q_h, b * p.s.q_b, pol_q);
    }
    int j = 0;
    for (; j < blocks; ++j) {
      if (j > 0 && !mbar_wait_warp(&bars->k_empty, (j - 1) & 1, status, abort_flag)) break;
      if (leader) {
        mbar_arrive_expect_tx(&bars->k_full, SM::kTile);
        for (int c = 0; c < SM::kChunks; ++c)
          tma_load_4d(smem + SM::kK + c * kXChunk, &tm_k, &bars->k_full, 64 * c, j * kXKeys, hk * p.s.k_h, b * p.s.k_b,
                      pol_kv);
      }
      __syncwarp();
      if (j > 0 && !mbar_wait_warp(&bars->v_empty, (j - 1) & 1, status, abort_flag)) break;
      if (leader) {
        mbar_arrive_expect_tx(&bars->v_full, SM::kTile);
        for (int c = 0; c < SM::kChunks; ++c)
          tma_load_4d(smem + SM::kV + c * kXChunk, &tm_v, &bars->v_full, 64 * c, j * kXKeys, hk * p.s.v_h, b * p.s.v_b,
                      pol_kv);
      }
      __syncwarp();
    }
    // the last releases have landed before the CTA leaves
    if (j == blocks && blocks > 0) {
      mbar_wait_warp(&bars->k_empty, (blocks - 1) & 1, status, abort_flag);
      mbar_wait_warp(&bars->v_empty, (blocks - 1) & 1, status, abort_flag);
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------------ MMA
    const uint32_t leader = elect_one();
    const uint32_t id_s = idesc16<BF>(128, kXKeys, false, false);
    const uint32_t id_o = idesc16<BF>(128, DP, false, true);
    const uint64_t dq = desc_k(smem_u32(smem + SM::kQ)), dk = desc_k(smem_u32(smem + SM::kK));
    const uint64_t dv = desc_mn(smem_u32(smem + SM::kV), kXChunk);
    bool ok = blocks == 0 || mbar_wait_warp(&bars->q_full, 0, status, abort_flag);
    for (int j = 0; ok && j < blocks; ++j) {
      if (!mbar_wait_warp(&bars->k_full, j & 1, status, abort_flag)) break;
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const uint32_t o = ((kk / 4) * kXChunk + (kk % 4) * 32) >> 4;
        mma_bf16_by(leader, tmem + kXColS, dq + o, dk + o, id_s, kk != 0);
      }
      mma_commit_by(leader, &bars->s_full);
      mma_commit_by(leader, &bars->k_empty);
      if (!mbar_wait_warp(&bars->v_full, j & 1, status, abort_flag)) break;
      // a block with keys that no query sees: their values may hold anything (0 * NaN), so they become zeros
      if (KIND == CROSS_KEYS || (count < p.s.keys && (j + 1) * kXKeys > count))
        zero_excluded_rows<kXKeys, SM::kChunks>(smem + SM::kV, kXChunk, j * kXKeys, count, p.s, mask_at,
                                                KIND == CROSS_KEYS, lane);
      if (!mbar_wait_warp(&bars->p_full, j & 1, status, abort_flag)) break;
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < kXKeys / 16; ++kk)
        mma_bf16_ts_by(leader, tmem + kXColO, tmem + kXColS + 8 * kk, dv + ((kk * 2048) >> 4), id_o, (j | kk) != 0);
      mma_commit_by(leader, &bars->v_empty);
      if (j == blocks - 1) mma_commit_by(leader, &bars->o_full);
    }
  } else {
    // ------------------------------------------------------------------ softmax, one thread per row
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const int row = row0 + threadIdx.x;
    const bool valid = row < p.s.queries;
    const float scale2 = p.s.scale * kCrossLog2e;
    constexpr bool NAT = KIND == CROSS_KEYS || KIND == CROSS_BIAS;   // logits kept in natural units
    float m = -INFINITY, l = 0.f;
    float* bias = reinterpret_cast<float*>(smem + SM::kBias);
    bool ok = true;
    for (int j = 0; j < blocks; ++j) {
      const int left = count - j * kXKeys;            // keys of this block
      uint32_t bits[4] = {0u, 0u, 0u, 0u};
      float* bj = bias + (j & 1) * kXKeys;
      if (KIND == CROSS_KEYS) {
        const int i = threadIdx.x;
        bj[i] = i < left ? mask_term(p.s.mask.p, p.s.mask.dtype,
                                     mask_at + static_cast<int64_t>(j * kXKeys + i) * p.s.mask.sm) : -INFINITY;
        named_bar_sync(1, 128);
      }
      if (KIND == CROSS_PAIRS) {
        // the warp's 32 rows of mask bits, a row's 128 keys by coalesced loads and four ballots
        const int rows = min(32, static_cast<int>(p.s.queries) - (row0 + warp * 32));
        const int64_t at = mask_at + static_cast<int64_t>(row0 + warp * 32) * p.s.mask.sn +
                           static_cast<int64_t>(j * kXKeys) * p.s.mask.sm;
        for (int r = 0; r < rows; ++r) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int key = 32 * q + lane;
            const bool keep = key < left && __ldg(static_cast<const uint8_t*>(p.s.mask.p) + at + r * p.s.mask.sn +
                                                  key * p.s.mask.sm) != 0;
            const uint32_t w = __ballot_sync(0xffffffffu, keep);
            if (lane == r) bits[q] = w;
          }
        }
      }
      const int64_t row_at = mask_at + (valid ? row : 0) * p.s.mask.sn + static_cast<int64_t>(j * kXKeys) * p.s.mask.sm;
      if (!mbar_wait_warp(&bars->s_full, j & 1, status, abort_flag)) { ok = false; break; }
      tc_fence_after();
      // logit of column 32 c + i: log2 units (scale2 folded in later for NONE / PAIRS), natural with a bias
      auto logits = [&](int c, uint32_t(&s)[32]) {
        tmem_ld32(tmem + lanes + kXColS + 32 * c, s);
        tmem_ld_wait();
        if (KIND == CROSS_NONE) {
          if (left < kXKeys) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (32 * c + i >= left) s[i] = __float_as_uint(-INFINITY);
          }
        } else if (KIND == CROSS_PAIRS) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(bits[c] >> i & 1u)) s[i] = __float_as_uint(-INFINITY);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float t;
            if (KIND == CROSS_KEYS)
              t = bj[32 * c + i];
            else
              t = 32 * c + i < left ? mask_term(p.s.mask.p, p.s.mask.dtype,
                                                row_at + static_cast<int64_t>(32 * c + i) * p.s.mask.sm) : -INFINITY;
            s[i] = __float_as_uint(t == -INFINITY ? t : fmaf(__uint_as_float(s[i]), p.s.scale, t));
          }
        }
      };
      float mx = -INFINITY;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t s[32];
        logits(c, s);
        float a = -INFINITY, e = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          a = max3(a, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          e = max3(e, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
        }
        mx = max3(mx, a, e);
      }
      if (!NAT) mx *= scale2;
      const float m_new = fmaxf(m, mx);
      const bool grow = m_new > m + (NAT ? kXRescale * kCrossLn2 : kXRescale);
      float alpha = 1.f;
      if (grow) {
        alpha = cross_ex2(NAT ? (m - m_new) * kCrossLog2e : m - m_new);
        l *= alpha;
        m = m_new;
      }
      // S(j) complete means O's last product is too: rescale before P(j) is handed over
      if (j > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tmem + lanes + kXColO + 32 * c, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st32(tmem + lanes + kXColO + 32 * c, o);
        }
      }
      const float mref = m == -INFINITY ? 0.f : m;      // nothing seen yet: every term is exp2(-inf) = 0
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t s[32], w[16];
        logits(c, s);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float2 e = make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          if (NAT)
            e = mul2(sub2(e, make_float2(mref, mref)), make_float2(kCrossLog2e, kCrossLog2e));
          else
            e = fma2(e, make_float2(scale2, scale2), make_float2(-mref, -mref));
          e = make_float2(cross_ex2(e.x), cross_ex2(e.y));
          sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], e);
          w[i >> 1] = pack16x2<BF>(e.x, e.y);
        }
        tmem_st16(tmem + lanes + kXColS + 16 * c, w);    // over columns this thread has already read
      }
      sum[0] = add2(sum[0], sum[1]);
      l += sum[0].x + sum[0].y;
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bars->p_full);
    }
    if (ok && valid && p.lse != nullptr)
      p.lse[static_cast<int64_t>(bh) * p.s.queries + row] = l > 0.f || l != l ? (NAT ? m : m * kCrossLn2) + logf(l) : -INFINITY;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    if (ok && blocks > 0) ok = mbar_wait_warp(&bars->o_full, 0, status, abort_flag);
    if (ok) {
      tc_fence_after();
      // rows of 64 columns through the queries' shared memory (no longer read), stored by TMA: rows past the end and
      // columns past dim are not written
      uint8_t* stage = smem + SM::kQ + warp * 32 * 128;
#pragma unroll 1
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
        if (blocks > 0) {
          tmem_ld32(tmem + lanes + kXColO + 32 * c, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        const uint32_t base = smem_u32(stage + (c / 2) * kXChunk);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = pack16x2<BF>(__uint_as_float(o[8 * g + 2 * i]) * inv, __uint_as_float(o[8 * g + 2 * i + 1]) * inv);
          st_shared_v4(base + sw128_off(lane, (c & 1) * 4 + g), w[0], w[1], w[2], w[3]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && row0 + warp * 32 < p.s.queries) {
        for (int c = 0; c < SM::kChunks; ++c)
          if (64 * c < p.s.dim) tma_store_4d(&tm_o, stage + c * kXChunk, 64 * c, row0 + warp * 32, h, b);
        bulk_commit_group();
        bulk_wait_group_read0();
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, kXCols);
}

template <int DP, bool BF, int KIND>
int launch_fwd(const CUtensorMap* maps, const CrossFwdParams& p, int64_t grid, cudaStream_t st) {
  static bool done[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return HTRC_ERR_CUDA;
  auto kernel = cross_fwd_kernel<DP, BF, KIND>;
  constexpr uint32_t bytes = CrossFwdSmem<DP>::kBytes;
  if (dev >= 64 || !done[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return HTRC_ERR_CUDA;
    if (dev < 64) done[dev] = true;
  }
  kernel<<<static_cast<unsigned>(grid), kXThreads, bytes, st>>>(maps[0], maps[1], maps[2], maps[3], p);
  return cudaGetLastError() == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
}

template <int DP, bool BF>
int launch_kind(int kind, const CUtensorMap* maps, const CrossFwdParams& p, int64_t grid, cudaStream_t st) {
  switch (kind) {
    case CROSS_NONE: return launch_fwd<DP, BF, CROSS_NONE>(maps, p, grid, st);
    case CROSS_KEYS: return launch_fwd<DP, BF, CROSS_KEYS>(maps, p, grid, st);
    case CROSS_PAIRS: return launch_fwd<DP, BF, CROSS_PAIRS>(maps, p, grid, st);
    default: return launch_fwd<DP, BF, CROSS_BIAS>(maps, p, grid, st);
  }
}

bool rows_ok(const void* p, const int64_t* stride) {
  if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (stride[i] < 0 || stride[i] % 8 || stride[i] >= (int64_t(1) << 38)) return false;
  return true;
}

int cross_forward(const HtrcCrossArgs* a, cudaStream_t st) {
  int rc = cross_validate(a, false, true);
  if (rc != HTRC_OK) return rc;
  if (!device_ok()) return HTRC_ERR_DEVICE;
  if (a->batch * a->queries == 0) return HTRC_OK;
  CrossFwdParams p{};
  p.s = cross_shape(a);
  p.lse = a->lse;
  p.status = a->status;
  p.tiles = static_cast<int>((a->queries + kXRows - 1) / kXRows);
  const int64_t grid = p.tiles * a->batch * a->heads;
  if (grid > (int64_t(1) << 31) - 1) return HTRC_ERR_UNSUPPORTED;
  CUtensorMap maps[4];
  int one;
  const bool keys = a->keys > 0;
  if (!cross_map(&maps[0], a, a->q, a->q_stride, a->queries, a->heads, kXRows, &p.s.q_b, &p.s.q_h) ||
      !cross_map(&maps[1], a, keys ? a->k : a->q, keys ? a->k_stride : a->q_stride, keys ? a->keys : a->queries,
                 keys ? a->kv_heads : a->heads, kXKeys, &p.s.k_b, &p.s.k_h) ||
      !cross_map(&maps[2], a, keys ? a->v : a->q, keys ? a->v_stride : a->q_stride, keys ? a->keys : a->queries,
                 keys ? a->kv_heads : a->heads, kXKeys, &p.s.v_b, &p.s.v_h) ||
      !cross_map(&maps[3], a, a->out, a->out_stride, a->queries, a->heads, 32, &one, &one))
    return HTRC_ERR_CUDA;
  const int kind = cross_mask_kind(a);
  const bool bf = a->dtype == HTRC_LAYER_BF16;
  if (a->dim <= 64) return bf ? launch_kind<64, true>(kind, maps, p, grid, st) : launch_kind<64, false>(kind, maps, p, grid, st);
  return bf ? launch_kind<128, true>(kind, maps, p, grid, st) : launch_kind<128, false>(kind, maps, p, grid, st);
}

}  // namespace

int cross_validate(const HtrcCrossArgs* a, bool back, bool ptrs) {
  if (a == nullptr) return HTRC_ERR_ARG;
  if (a->batch < 0 || a->queries < 0 || a->keys < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads)
    return HTRC_ERR_ARG;
  if (a->dtype != HTRC_LAYER_BF16 && a->dtype != HTRC_LAYER_F16) return HTRC_ERR_ARG;
  if (a->dim < 8 || a->dim % 8) return HTRC_ERR_ARG;
  if (a->dim > HTRC_CROSS_MAX_DIM) return HTRC_ERR_UNSUPPORTED;
  constexpr int64_t kMax = (int64_t(1) << 31) - 4096;
  if (a->batch > kMax || a->queries > kMax || a->keys > kMax || a->heads > 65536) return HTRC_ERR_UNSUPPORTED;
  if (a->batch * a->heads > kMax) return HTRC_ERR_UNSUPPORTED;
  if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return HTRC_ERR_ARG;
  if (a->mask && a->mask_dtype != HTRC_LAYER_U8 && a->mask_dtype != HTRC_LAYER_F32 && a->mask_dtype != HTRC_LAYER_BF16 &&
      a->mask_dtype != HTRC_LAYER_F16)
    return HTRC_ERR_ARG;
  if (!ptrs) return HTRC_OK;
  if (a->batch * a->queries > 0) {
    if (!a->q || !a->out || !rows_ok(a->q, a->q_stride) || !rows_ok(a->out, a->out_stride)) return HTRC_ERR_ARG;
    if (back && (!a->lse || !a->dout || !a->dq || !rows_ok(a->dout, a->dout_stride) || !rows_ok(a->dq, a->dq_stride)))
      return HTRC_ERR_ARG;
  }
  if (a->batch * a->keys > 0) {
    if (!a->k || !a->v || !rows_ok(a->k, a->k_stride) || !rows_ok(a->v, a->v_stride)) return HTRC_ERR_ARG;
    // rows of their own (TMA strides): a tensor broadcast along its tokens is laid out by the caller
    if (a->keys > 1 && (a->k_stride[1] == 0 || a->v_stride[1] == 0)) return HTRC_ERR_ARG;
    if (back && (!a->dk || !a->dv || !rows_ok(a->dk, a->dk_stride) || !rows_ok(a->dv, a->dv_stride))) return HTRC_ERR_ARG;
  }
  if (a->queries > 1 && a->batch > 0 && (a->q_stride[1] == 0 || a->out_stride[1] == 0 || (back && a->dout_stride[1] == 0)))
    return HTRC_ERR_ARG;
  return HTRC_OK;
}

CrossShape cross_shape(const HtrcCrossArgs* a) {
  CrossShape s{};
  s.batch = a->batch;
  s.queries = a->queries;
  s.keys = a->keys;
  s.heads = a->heads;
  s.kv_heads = a->kv_heads;
  s.group = a->heads / a->kv_heads;
  s.dim = a->dim;
  s.scale = a->scale;
  s.lengths = a->key_lengths;
  s.mask = CrossMaskView{a->mask, a->mask_stride[0], a->mask_stride[1], a->mask_stride[2], a->mask_stride[3], a->mask_dtype};
  return s;
}

int cross_mask_kind(const HtrcCrossArgs* a) {
  if (a->mask == nullptr) return CROSS_NONE;
  if (a->mask_stride[2] == 0 || a->queries == 1) return CROSS_KEYS;
  return a->mask_dtype == HTRC_LAYER_U8 ? CROSS_PAIRS : CROSS_BIAS;
}

bool cross_map(CUtensorMap* m, const HtrcCrossArgs* a, const void* base, const int64_t* stride, int64_t rows, int heads,
               int box_rows, int* b, int* h) {
  const bool in_b = a->batch > 1 && stride[0] != 0, in_h = heads > 1 && stride[2] != 0;
  *b = in_b;
  *h = in_h;
  const uint64_t dims[4] = {static_cast<uint64_t>(a->dim), static_cast<uint64_t>(rows),
                            in_h ? static_cast<uint64_t>(heads) : 1, in_b ? static_cast<uint64_t>(a->batch) : 1};
  // a dimension of one is never stepped along: any valid stride
  const uint64_t strides[3] = {rows > 1 ? static_cast<uint64_t>(stride[1]) * 2 : 256,
                               in_h ? static_cast<uint64_t>(stride[2]) * 2 : 256,
                               in_b ? static_cast<uint64_t>(stride[0]) * 2 : 256};
  const uint32_t box[4] = {64, static_cast<uint32_t>(box_rows), 1, 1};
  return make_tiled_map(m, a->dtype == HTRC_LAYER_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        4, base, dims, strides, box, true);
}

}  // namespace htrc

extern "C" int htrc_cross_forward(const HtrcCrossArgs* args, htrc_stream_t stream) {
  return htrc::cross_forward(args, reinterpret_cast<cudaStream_t>(stream));
}
