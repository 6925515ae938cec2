// Cross attention, backward.  With P = exp(S scale + mask - lse), dP = dO V^T, delta = rowsum(dO out) - dlse and
// dS = P (dP - delta):   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO;  the gradients of a shared key head are
// summed over its query heads.
//
// Two passes, each recomputing S and dP on tcgen05, so that no gradient needs an atomic and every sum has a fixed order:
//
// cross_dq_kernel: a CTA owns 128 query rows and walks the keys in blocks of 64, dQ accumulating in TMEM (S 64, dP 64
// and dQ 128 columns: two CTAs per SM, one's products under the other's exponentials).  It also forms delta from the
// rows of dO and out that it holds and leaves (lse, delta) for the second pass.
//
// cross_dkv_kernel: a CTA owns 128 keys of one key head (rows of S^T = K Q^T and dP^T = V dO^T) and a range of the
// query blocks of 64 of every head that shares it; dK and dV accumulate in TMEM (256 columns), S^T and dP^T are double
// buffered beside them, and two softmax warpgroups take alternate steps, so a step's exponentials run under the
// neighbouring steps' products.  P^T and dS^T never leave TMEM: they are the A operands of the products with dO and Q.
// Where the key blocks alone do not fill the device evenly, the query range is split and the float32 partial sums are
// added by cross_dkv_sum_kernel in order.
//
// Rounding: P and dS enter their products in the operands' 16-bit type, the gradients are rounded once from float32.
#include <algorithm>
#include <cmath>

#include "cross.cuh"

namespace htrc {

namespace {

constexpr float kHuge = 1e30f;        // a |log sum| above this is a mask's lowest value: the logits are lost in it

// ------------------------------------------------------------------------------------------------ dQ
constexpr int kDqThreads = 192;
constexpr int kDqRows = 128, kDqKeys = 64;
constexpr uint32_t kDqColS = 0, kDqColP = 64, kDqColQ = 128, kDqCols = 256;

struct DqBars {
  uint64_t q_full, k_full[2], k_empty[2], v_full, v_empty, s_full, ds_full, dq_full;
  uint32_t tmem_base;
  int abort_flag;
};

template <int DP>
struct DqSmem {
  static constexpr int kChunks = DP / 64;
  static constexpr uint32_t kRowChunk = 128 * 128, kKeyChunk = 64 * 128;
  static constexpr uint32_t kTile = kChunks * kRowChunk, kSlot = kChunks * kKeyChunk;
  static constexpr uint32_t kQ = 0, kDo = kTile, kK = 2 * kTile, kV = kK + 2 * kSlot, kBias = kV + kSlot;
  static constexpr uint32_t kBars = kBias + 2 * kDqKeys * 4, kUsed = kBars + 256;
  static_assert(sizeof(DqBars) <= 256 && kUsed <= 115712, "two CTAs per SM");
  // never more than two CTAs on an SM's 512 TMEM columns
  static constexpr uint32_t kBytes = kUsed < 80 * 1024 ? 80 * 1024 : kUsed;
};

struct DqParams {
  CrossShape s;
  const float* lse;
  const float* dlse;
  const uint16_t* out;
  int64_t out_stride[3];
  float* stat;              // [batch * heads][padded rows / 64][3][64]: lse in the pass's units, log2 of tied keys, delta
  int64_t stat_rows;
  int tiles;
  int* status;
};

template <int DP, bool BF, int KIND>
__global__ void __launch_bounds__(kDqThreads, 2)
    cross_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                    const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ CUtensorMap tm_dq, const __grid_constant__ DqParams p, int do_b, int do_h) {
  using SM = DqSmem<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023) {          // the swizzled tiles need it; two CTAs leave no room to round up
    flag_status(p.status, ST_WAIT_TIMEOUT);
    return;
  }
  DqBars* bars = reinterpret_cast<DqBars*>(smem + SM::kBars);
  volatile int* abort_flag = &bars->abort_flag;
  int* status = p.status;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x % p.tiles;
  const int bh = blockIdx.x / p.tiles;
  const int h = bh % p.s.heads, b = bh / p.s.heads, hk = h / p.s.group;
  const int row0 = tile * kDqRows;
  const int count = key_count(p.s, b);
  const int blocks = (count + kDqKeys - 1) / kDqKeys;
  const int64_t mask_at = b * p.s.mask.sb + h * p.s.mask.sh;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->k_full[i], 1);
      mbar_init(&bars->k_empty[i], 1);
    }
    mbar_init(&bars->v_full, 1);
    mbar_init(&bars->v_empty, 1);
    mbar_init(&bars->s_full, 1);
    mbar_init(&bars->ds_full, 128);
    mbar_init(&bars->dq_full, 1);
    bars->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 5) tmem_alloc(&bars->tmem_base, kDqCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  if (warp == 4) {
    // ------------------------------------------------------------------ TMA
    const uint64_t pol_q = policy_evict_first(), pol_kv = policy_evict_last();
    const uint32_t leader = elect_one();
    if (leader && blocks > 0) {
      mbar_arrive_expect_tx(&bars->q_full, 2 * SM::kTile);
      for (int c = 0; c < SM::kChunks; ++c) {
        tma_load_4d(smem + SM::kQ + c * SM::kRowChunk, &tm_q, &bars->q_full, 64 * c, row0, h * p.s.q_h, b * p.s.q_b, pol_q);
        tma_load_4d(smem + SM::kDo + c * SM::kRowChunk, &tm_do, &bars->q_full, 64 * c, row0, h * do_h, b * do_b, pol_q);
      }
    }
    int j = 0;
    for (; j < blocks; ++j) {
      const int s = j & 1;
      if (j > 1 && !mbar_wait_warp(&bars->k_empty[s], ((j >> 1) - 1) & 1, status, abort_flag)) break;
      if (leader) {
        mbar_arrive_expect_tx(&bars->k_full[s], SM::kSlot);
        for (int c = 0; c < SM::kChunks; ++c)
          tma_load_4d(smem + SM::kK + s * SM::kSlot + c * SM::kKeyChunk, &tm_k, &bars->k_full[s], 64 * c, j * kDqKeys,
                      hk * p.s.k_h, b * p.s.k_b, pol_kv);
      }
      __syncwarp();
      if (j > 0 && !mbar_wait_warp(&bars->v_empty, (j - 1) & 1, status, abort_flag)) break;
      if (leader) {
        mbar_arrive_expect_tx(&bars->v_full, SM::kSlot);
        for (int c = 0; c < SM::kChunks; ++c)
          tma_load_4d(smem + SM::kV + c * SM::kKeyChunk, &tm_v, &bars->v_full, 64 * c, j * kDqKeys, hk * p.s.v_h,
                      b * p.s.v_b, pol_kv);
      }
      __syncwarp();
    }
    if (j == blocks && blocks > 0) {      // the last releases have landed before the CTA leaves
      drain_ring<true>(bars->k_empty, 2, blocks, status, abort_flag);
      mbar_wait_warp(&bars->v_empty, (blocks - 1) & 1, status, abort_flag);
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------------ MMA
    const uint32_t leader = elect_one();
    const uint32_t id_s = idesc16<BF>(128, kDqKeys, false, false);
    const uint32_t id_q = idesc16<BF>(128, DP, false, true);
    const uint64_t dq = desc_k(smem_u32(smem + SM::kQ)), ddo = desc_k(smem_u32(smem + SM::kDo));
    const uint64_t dk0 = desc_k(smem_u32(smem + SM::kK)), dv = desc_k(smem_u32(smem + SM::kV));
    const uint64_t dkn0 = desc_mn(smem_u32(smem + SM::kK), SM::kKeyChunk);
    bool ok = blocks == 0 || mbar_wait_warp(&bars->q_full, 0, status, abort_flag);
    for (int j = 0; ok && j < blocks; ++j) {
      const int s = j & 1;
      // excluded keys may hold anything: their rows of K (0 * NaN in dS K) and V become zeros
      const bool dirty = KIND == CROSS_KEYS || (count < p.s.keys && (j + 1) * kDqKeys > count);
      if (!mbar_wait_warp(&bars->k_full[s], (j >> 1) & 1, status, abort_flag)) break;
      if (dirty)
        zero_excluded_rows<kDqKeys, SM::kChunks>(smem + SM::kK + s * SM::kSlot, SM::kKeyChunk, j * kDqKeys, count, p.s,
                                                 mask_at, KIND == CROSS_KEYS, lane);
      if (!mbar_wait_warp(&bars->v_full, j & 1, status, abort_flag)) break;
      if (dirty)
        zero_excluded_rows<kDqKeys, SM::kChunks>(smem + SM::kV, SM::kKeyChunk, j * kDqKeys, count, p.s, mask_at,
                                                 KIND == CROSS_KEYS, lane);
      tc_fence_after();
      const uint64_t so = (s * SM::kSlot) >> 4;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const uint32_t a = ((kk / 4) * SM::kRowChunk + (kk % 4) * 32) >> 4, o = ((kk / 4) * SM::kKeyChunk + (kk % 4) * 32) >> 4;
        mma_bf16_by(leader, tmem + kDqColS, dq + a, dk0 + so + o, id_s, kk != 0);
      }
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const uint32_t a = ((kk / 4) * SM::kRowChunk + (kk % 4) * 32) >> 4, o = ((kk / 4) * SM::kKeyChunk + (kk % 4) * 32) >> 4;
        mma_bf16_by(leader, tmem + kDqColP, ddo + a, dv + o, id_s, kk != 0);
      }
      mma_commit_by(leader, &bars->s_full);
      mma_commit_by(leader, &bars->v_empty);
      if (!mbar_wait_warp(&bars->ds_full, j & 1, status, abort_flag)) break;
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < kDqKeys / 16; ++kk)
        mma_bf16_ts_by(leader, tmem + kDqColQ, tmem + kDqColS + 8 * kk, dkn0 + so + ((kk * 2048) >> 4), id_q, (j | kk) != 0);
      mma_commit_by(leader, &bars->k_empty[s]);
      if (j == blocks - 1) mma_commit_by(leader, &bars->dq_full);
    }
  } else {
    // ------------------------------------------------------------------ one thread per row
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const int row = row0 + threadIdx.x;
    const bool valid = row < p.s.queries;
    const float scale2 = p.s.scale * kCrossLog2e;
    constexpr bool NAT = KIND == CROSS_KEYS || KIND == CROSS_BIAS;
    float* bias = reinterpret_cast<float*>(smem + SM::kBias);
    const int64_t at = static_cast<int64_t>(bh) * p.s.queries + row;
    const int64_t row_mask = mask_at + (valid ? row : 0) * p.s.mask.sn;
    // a row with nothing in it (or none): every weight exp2(-inf)
    float lse = valid ? __ldg(p.lse + at) : -INFINITY, ties = 0.f, delta = 0.f;
    if (NAT && fabsf(lse) > kHuge && lse != -INFINITY) {
      // every logit of the row is a mask's lowest value and the log of their count is lost in lse: count them
      int n = 0;
      for (int i = 0; i < count; ++i)
        n += mask_term(p.s.mask.p, p.s.mask.dtype, row_mask + static_cast<int64_t>(i) * p.s.mask.sm) == lse;
      ties = n > 1 ? log2f(static_cast<float>(n)) : 0.f;
    }
    if (lse == -INFINITY) lse = INFINITY;
    if (!NAT) lse *= kCrossLog2e;
    bool ok = true;
    if (blocks > 0) {
      ok = mbar_wait_warp(&bars->q_full, 0, status, abort_flag);
      if (ok && valid) {
        const uint16_t* o = p.out + b * p.out_stride[0] + row * p.out_stride[1] + h * p.out_stride[2];
        float2 acc = make_float2(0.f, 0.f);
        for (int c = 0; 8 * c < p.s.dim; ++c) {
          const uint4 x = __ldg(reinterpret_cast<const uint4*>(o + 8 * c));
          const uint4 y = *reinterpret_cast<const uint4*>(smem + SM::kDo + (c / 8) * SM::kRowChunk +
                                                          sw128_off(threadIdx.x, c & 7));
          acc = fma2(unpack16x2<BF>(x.x), unpack16x2<BF>(y.x), acc);
          acc = fma2(unpack16x2<BF>(x.y), unpack16x2<BF>(y.y), acc);
          acc = fma2(unpack16x2<BF>(x.z), unpack16x2<BF>(y.z), acc);
          acc = fma2(unpack16x2<BF>(x.w), unpack16x2<BF>(y.w), acc);
        }
        delta = acc.x + acc.y - (p.dlse != nullptr ? __ldg(p.dlse + at) : 0.f);
        if (lse == INFINITY) delta = 0.f;
      }
    }
    float* stat = p.stat + (static_cast<int64_t>(bh) * p.stat_rows + row / 64 * 64) * 3 + row % 64;
    stat[0] = lse;
    stat[64] = ties;
    stat[128] = delta;
    for (int j = 0; ok && j < blocks; ++j) {
      const int left = count - j * kDqKeys;
      uint32_t bits[2] = {0u, 0u};
      float* bj = bias + (j & 1) * kDqKeys;
      if (KIND == CROSS_KEYS) {
        const int i = threadIdx.x;
        if (i < kDqKeys)
          bj[i] = i < left ? mask_term(p.s.mask.p, p.s.mask.dtype,
                                       mask_at + static_cast<int64_t>(j * kDqKeys + i) * p.s.mask.sm) : -INFINITY;
        named_bar_sync(1, 128);
      }
      if (KIND == CROSS_PAIRS) {
        const int rows = min(32, static_cast<int>(p.s.queries) - (row0 + warp * 32));
        const int64_t ma = mask_at + static_cast<int64_t>(row0 + warp * 32) * p.s.mask.sn +
                           static_cast<int64_t>(j * kDqKeys) * p.s.mask.sm;
        for (int r = 0; r < rows; ++r) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int key = 32 * q + lane;
            const bool keep = key < left && __ldg(static_cast<const uint8_t*>(p.s.mask.p) + ma + r * p.s.mask.sn +
                                                  key * p.s.mask.sm) != 0;
            const uint32_t w = __ballot_sync(0xffffffffu, keep);
            if (lane == r) bits[q] = w;
          }
        }
      }
      if (!mbar_wait_warp(&bars->s_full, j & 1, status, abort_flag)) { ok = false; break; }
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        uint32_t s[32], g[32], w[16];
        tmem_ld32(tmem + lanes + kDqColS + 32 * c, s);
        tmem_ld32(tmem + lanes + kDqColP + 32 * c, g);
        tmem_ld_wait();
        if (KIND == CROSS_NONE) {
          if (left < kDqKeys) {
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
                                                row_mask + static_cast<int64_t>(j * kDqKeys + 32 * c + i) * p.s.mask.sm)
                                    : -INFINITY;
            s[i] = __float_as_uint(t == -INFINITY ? t : fmaf(__uint_as_float(s[i]), p.s.scale, t));
          }
        }
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float2 e = make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          if (NAT)
            e = fma2(sub2(e, make_float2(lse, lse)), make_float2(kCrossLog2e, kCrossLog2e), make_float2(-ties, -ties));
          else
            e = fma2(e, make_float2(scale2, scale2), make_float2(-lse, -lse));
          e = make_float2(cross_ex2(e.x), cross_ex2(e.y));
          e = mul2(e, sub2(make_float2(__uint_as_float(g[i]), __uint_as_float(g[i + 1])), make_float2(delta, delta)));
          w[i >> 1] = pack16x2<BF>(e.x, e.y);
        }
        tmem_st16(tmem + lanes + kDqColS + 16 * c, w);      // dS over columns of S this thread has already read
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bars->ds_full);
    }
    if (ok && blocks > 0) ok = mbar_wait_warp(&bars->dq_full, 0, status, abort_flag);
    if (ok) {
      tc_fence_after();
      uint8_t* stage = smem + SM::kQ + warp * 32 * 128;
#pragma unroll 1
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
        if (blocks > 0) {
          tmem_ld32(tmem + lanes + kDqColQ + 32 * c, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        const uint32_t base = smem_u32(stage + (c / 2) * SM::kRowChunk);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = pack16x2<BF>(__uint_as_float(o[8 * g + 2 * i]) * p.s.scale, __uint_as_float(o[8 * g + 2 * i + 1]) * p.s.scale);
          st_shared_v4(base + sw128_off(lane, (c & 1) * 4 + g), w[0], w[1], w[2], w[3]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && row0 + warp * 32 < p.s.queries) {
        for (int c = 0; c < SM::kChunks; ++c)
          if (64 * c < p.s.dim) tma_store_4d(&tm_dq, stage + c * SM::kRowChunk, 64 * c, row0 + warp * 32, h, b);
        bulk_commit_group();
        bulk_wait_group_read0();
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, kDqCols);
}

// ------------------------------------------------------------------------------------------------ dK, dV
constexpr int kDkvThreads = 320;
constexpr int kDkvKeys = 128, kDkvRows = 64, kDkvStages = 4;
constexpr uint32_t kDkvColK = 0, kDkvColV = 128, kDkvColS = 256, kDkvBuf = 128, kDkvCols = 512;

struct DkvBars {
  uint64_t kv_full, full[kDkvStages], empty[kDkvStages], s_full[2], dp_full[2], p_full[2], ds_full[2], acc_full;
  uint32_t tmem_base;
  int abort_flag;
};

template <int DP>
struct DkvSmem {
  static constexpr int kChunks = DP / 64;
  static constexpr uint32_t kKeyChunk = 128 * 128, kRowChunk = 64 * 128;
  static constexpr uint32_t kTile = kChunks * kKeyChunk, kRows = kChunks * kRowChunk;
  static constexpr uint32_t kK = 0, kV = kTile, kRing = 2 * kTile, kStat = kDkvRows * 3 * 4,
                            kStage = 2 * kRows + 1024;
  static constexpr uint32_t kBars = kRing + kDkvStages * kStage;
  static constexpr uint32_t kUsed = kBars + 256 + 1024;
  // one CTA per SM: it takes all 512 TMEM columns
  static constexpr uint32_t kBytes = kUsed < 120 * 1024 ? 120 * 1024 : kUsed;
};

struct DkvParams {
  CrossShape s;
  const float* stat;
  int64_t stat_rows;
  int key_blocks, splits, row_blocks;
  float* partial;           // splits > 1: [2 (dk, dv)][split][batch * kv_heads][keys][DP]
  int* status;
};

template <int DP, bool BF, int KIND>
__global__ void __launch_bounds__(kDkvThreads, 1)
    cross_dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                     const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ CUtensorMap tm_dk, const __grid_constant__ CUtensorMap tm_dv,
                     const __grid_constant__ DkvParams p, int do_b, int do_h) {
  using SM = DkvSmem<DP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  DkvBars* bars = reinterpret_cast<DkvBars*>(smem + SM::kBars);
  volatile int* abort_flag = &bars->abort_flag;
  int* status = p.status;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kb = blockIdx.x % p.key_blocks;
  const int rest = blockIdx.x / p.key_blocks;
  const int split = rest % p.splits, bk = rest / p.splits;
  const int hk = bk % p.s.kv_heads, b = bk / p.s.kv_heads;
  const int key0 = kb * kDkvKeys;
  const int count = key_count(p.s, b);
  const int64_t total = static_cast<int64_t>(p.s.group) * p.row_blocks;
  const int64_t first = total * split / p.splits;
  const int steps = key0 < count ? static_cast<int>(total * (split + 1) / p.splits - first) : 0;

  if (threadIdx.x == 0) {
    mbar_init(&bars->kv_full, 1);
    for (int i = 0; i < kDkvStages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->dp_full[i], 1);
      mbar_init(&bars->p_full[i], 128);
      mbar_init(&bars->ds_full[i], 128);
    }
    mbar_init(&bars->acc_full, 1);
    bars->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(&bars->tmem_base, kDkvCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  if (warp == 8) {
    // ------------------------------------------------------------------ TMA
    const uint64_t pol = policy_evict_normal();
    const uint32_t leader = elect_one();
    if (leader && steps > 0) {
      mbar_arrive_expect_tx(&bars->kv_full, 2 * SM::kTile);
      for (int c = 0; c < SM::kChunks; ++c) {
        tma_load_4d(smem + SM::kK + c * SM::kKeyChunk, &tm_k, &bars->kv_full, 64 * c, key0, hk * p.s.k_h, b * p.s.k_b, pol);
        tma_load_4d(smem + SM::kV + c * SM::kKeyChunk, &tm_v, &bars->kv_full, 64 * c, key0, hk * p.s.v_h, b * p.s.v_b, pol);
      }
    }
    int i = 0;
    for (; i < steps; ++i) {
      const int s = i % kDkvStages;
      if (i >= kDkvStages && !mbar_wait_warp(&bars->empty[s], ((i / kDkvStages) - 1) & 1, status, abort_flag)) break;
      if (leader) {
        const int64_t at = first + i;
        const int h = hk * p.s.group + static_cast<int>(at / p.row_blocks), row = static_cast<int>(at % p.row_blocks) * kDkvRows;
        uint8_t* st = smem + SM::kRing + s * SM::kStage;
        mbar_arrive_expect_tx(&bars->full[s], 2 * SM::kRows + SM::kStat);
        for (int c = 0; c < SM::kChunks; ++c) {
          tma_load_4d(st + c * SM::kRowChunk, &tm_q, &bars->full[s], 64 * c, row, h * p.s.q_h, b * p.s.q_b, pol);
          tma_load_4d(st + SM::kRows + c * SM::kRowChunk, &tm_do, &bars->full[s], 64 * c, row, h * do_h, b * do_b, pol);
        }
        bulk_load(st + 2 * SM::kRows, p.stat + ((static_cast<int64_t>(b) * p.s.heads + h) * p.stat_rows + row) * 3, SM::kStat,
                  &bars->full[s], pol);
      }
      __syncwarp();
    }
    if (i == steps) drain_ring<true>(bars->empty, kDkvStages, steps, status, abort_flag);
  } else if (warp == 9) {
    // ------------------------------------------------------------------ MMA
    const uint32_t leader = elect_one();
    const uint32_t id_s = idesc16<BF>(128, kDkvRows, false, false);
    const uint32_t id_g = idesc16<BF>(128, DP, false, true);
    const uint64_t dk = desc_k(smem_u32(smem + SM::kK)), dv = desc_k(smem_u32(smem + SM::kV));
    const uint32_t ring = smem_u32(smem + SM::kRing);
    const uint64_t qk0 = desc_k(ring), dok0 = desc_k(ring + SM::kRows);
    const uint64_t qn0 = desc_mn(ring, SM::kRowChunk), don0 = desc_mn(ring + SM::kRows, SM::kRowChunk);
    auto scores = [&](int i) -> bool {
      const int s = i % kDkvStages;
      if (!mbar_wait_warp(&bars->full[s], (i / kDkvStages) & 1, status, abort_flag)) return false;
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const uint32_t a = ((kk / 4) * SM::kKeyChunk + (kk % 4) * 32) >> 4, o = ((kk / 4) * SM::kRowChunk + (kk % 4) * 32) >> 4;
        mma_bf16_by(leader, tmem + kDkvColS + (i & 1) * kDkvBuf, dk + a, qk0 + ((s * SM::kStage) >> 4) + o, id_s, kk != 0);
      }
      mma_commit_by(leader, &bars->s_full[i & 1]);
      return true;
    };
    auto products = [&](int i) {          // dP^T, of a stage that scores() waited for
      const int s = i % kDkvStages;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const uint32_t a = ((kk / 4) * SM::kKeyChunk + (kk % 4) * 32) >> 4, o = ((kk / 4) * SM::kRowChunk + (kk % 4) * 32) >> 4;
        mma_bf16_by(leader, tmem + kDkvColS + (i & 1) * kDkvBuf + 64, dv + a, dok0 + ((s * SM::kStage) >> 4) + o, id_s, kk != 0);
      }
      mma_commit_by(leader, &bars->dp_full[i & 1]);
    };
    bool ok = steps == 0 || mbar_wait_warp(&bars->kv_full, 0, status, abort_flag);
    // keys past the entry's count may hold anything: their rows become zeros (with a bias the softmax threads select)
    if (ok && steps > 0 && (KIND == CROSS_NONE || KIND == CROSS_PAIRS) && count < p.s.keys && key0 + kDkvKeys > count) {
      zero_excluded_rows<kDkvKeys, SM::kChunks>(smem + SM::kK, SM::kKeyChunk, key0, count, p.s, 0, false, lane);
      zero_excluded_rows<kDkvKeys, SM::kChunks>(smem + SM::kV, SM::kKeyChunk, key0, count, p.s, 0, false, lane);
    }
    for (int i = 0; ok && i < 2 && i < steps; ++i) {
      ok = scores(i);
      if (ok) products(i);
    }
    for (int i = 0; ok && i < steps; ++i) {
      const int s = i % kDkvStages;
      // P^T first: its product and the next S^T of this buffer run while the threads form dS^T
      ok = mbar_wait_warp(&bars->p_full[i & 1], (i >> 1) & 1, status, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint64_t so = (s * SM::kStage) >> 4;
      const uint32_t a = tmem + kDkvColS + (i & 1) * kDkvBuf;
#pragma unroll
      for (int kk = 0; kk < kDkvRows / 16; ++kk)
        mma_bf16_ts_by(leader, tmem + kDkvColV, a + 8 * kk, don0 + so + ((kk * 2048) >> 4), id_g, (i | kk) != 0);
      if (i + 2 < steps) ok = scores(i + 2);
      ok = ok && mbar_wait_warp(&bars->ds_full[i & 1], (i >> 1) & 1, status, abort_flag);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < kDkvRows / 16; ++kk)
        mma_bf16_ts_by(leader, tmem + kDkvColK, a + 64 + 8 * kk, qn0 + so + ((kk * 2048) >> 4), id_g, (i | kk) != 0);
      mma_commit_by(leader, &bars->empty[s]);
      if (i == steps - 1) mma_commit_by(leader, &bars->acc_full);
      if (i + 2 < steps) products(i + 2);
    }
  } else {
    // ------------------------------------------------------------------ two warpgroups, one thread per key
    const int wg = warp >> 2, quarter = warp & 3;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const int r = quarter * 32 + lane, key = key0 + r;
    constexpr bool NAT = KIND == CROSS_KEYS || KIND == CROSS_BIAS;
    const float scale = NAT ? p.s.scale : p.s.scale * kCrossLog2e;
    const bool in = key < count;
    int head = -1;
    float kbias = in ? 0.f : -INFINITY;           // this key's term: -inf where it is excluded
    bool ok = true;
    for (int i = wg; i < steps; i += 2) {
      const int s = i % kDkvStages;
      const int64_t at = first + i;
      const int hg = static_cast<int>(at / p.row_blocks), row = static_cast<int>(at % p.row_blocks) * kDkvRows;
      const int h = hk * p.s.group + hg;
      const int64_t mask_at = b * p.s.mask.sb + h * p.s.mask.sh + static_cast<int64_t>(key) * p.s.mask.sm;
      if (KIND == CROSS_KEYS && hg != head) {
        head = hg;
        if (in) kbias = mask_term(p.s.mask.p, p.s.mask.dtype, mask_at);
      }
      if (!mbar_wait_warp(&bars->s_full[wg], (i >> 1) & 1, status, abort_flag)) { ok = false; break; }
      tc_fence_after();
      // the queries' statistics: [lse][ties][delta], 64 each
      const float* st = reinterpret_cast<const float*>(smem + SM::kRing + s * SM::kStage + 2 * SM::kRows);
      const uint32_t buf = tmem + lanes + kDkvColS + wg * kDkvBuf;
      float2 w[32];                         // P, kept for dS
      uint32_t out = 0u, out_hi = 0u;       // queries this key is excluded from (with a mask per query)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t x[32], pw[16];
        tmem_ld32(buf + 32 * c, x);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 ls = *reinterpret_cast<const float4*>(st + 32 * c + k);
          const float4 ti = NAT ? *reinterpret_cast<const float4*>(st + 64 + 32 * c + k) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int h2 = 0; h2 < 2; ++h2) {
            const float l0 = h2 ? ls.z : ls.x, l1 = h2 ? ls.w : ls.y;
            const int kk = k + 2 * h2, q = row + 32 * c + kk;
            float2 e = make_float2(__uint_as_float(x[kk]), __uint_as_float(x[kk + 1]));
            if (!NAT) {
              float2 off = make_float2(kbias - l0, kbias - l1);
              if (KIND == CROSS_PAIRS) {
                const uint8_t* mk = static_cast<const uint8_t*>(p.s.mask.p) + mask_at;
                if (!(in && q < p.s.queries && __ldg(mk + q * p.s.mask.sn) != 0)) off.x = -INFINITY;
                if (!(in && q + 1 < p.s.queries && __ldg(mk + (q + 1) * p.s.mask.sn) != 0)) off.y = -INFINITY;
              }
              e = fma2(e, make_float2(scale, scale), off);
            } else {
              float b0 = kbias, b1 = kbias;
              if (KIND == CROSS_BIAS) {
                b0 = in && q < p.s.queries ? mask_term(p.s.mask.p, p.s.mask.dtype, mask_at + q * p.s.mask.sn) : -INFINITY;
                b1 = in && q + 1 < p.s.queries ? mask_term(p.s.mask.p, p.s.mask.dtype, mask_at + (q + 1) * p.s.mask.sn) : -INFINITY;
              }
              e = fma2(e, make_float2(scale, scale), make_float2(b0, b1));
              e = fma2(sub2(e, make_float2(l0, l1)), make_float2(kCrossLog2e, kCrossLog2e),
                       h2 ? make_float2(-ti.z, -ti.w) : make_float2(-ti.x, -ti.y));
              // an excluded key's weight and gradient are zero whatever its row holds
              if (b0 == -INFINITY) {
                e.x = -INFINITY;
                (c ? out_hi : out) |= 1u << kk;
              }
              if (b1 == -INFINITY) {
                e.y = -INFINITY;
                (c ? out_hi : out) |= 2u << kk;
              }
            }
            e = make_float2(cross_ex2(e.x), cross_ex2(e.y));
            w[16 * c + kk / 2] = e;
            pw[kk / 2] = pack16x2<BF>(e.x, e.y);
          }
        }
        tmem_st16(buf + 16 * c, pw);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bars->p_full[wg]);
      if (!mbar_wait_warp(&bars->dp_full[wg], (i >> 1) & 1, status, abort_flag)) { ok = false; break; }
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t y[32], dw[16];
        tmem_ld32(buf + 64 + 32 * c, y);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 de = *reinterpret_cast<const float4*>(st + 128 + 32 * c + k);
#pragma unroll
          for (int h2 = 0; h2 < 2; ++h2) {
            const int kk = k + 2 * h2;
            float2 g = make_float2(__uint_as_float(y[kk]), __uint_as_float(y[kk + 1]));
            if (NAT) {
              if ((c ? out_hi : out) >> kk & 1u) g.x = 0.f;
              if ((c ? out_hi : out) >> kk & 2u) g.y = 0.f;
            }
            const float2 d = mul2(w[16 * c + kk / 2], sub2(g, h2 ? make_float2(de.z, de.w) : make_float2(de.x, de.y)));
            dw[kk / 2] = pack16x2<BF>(d.x, d.y);
          }
        }
        tmem_st16(buf + 64 + 16 * c, dw);
      }
      tmem_st_wait();
      fence_proxy_async_smem();             // generic reads of a stage that TMA refills
      tc_fence_before();
      mbar_arrive(&bars->ds_full[wg]);
    }
    if (ok && steps > 0) ok = mbar_wait_warp(&bars->acc_full, 0, status, abort_flag);
    if (ok) {
      // warpgroup 0 writes dV, 1 dK
      tc_fence_after();
      const uint32_t acc = tmem + lanes + (wg == 0 ? kDkvColV : kDkvColK);
      const float mul = wg == 0 ? 1.0f : p.s.scale;
      uint8_t* stage = smem + (wg == 0 ? SM::kV : SM::kK) + quarter * 32 * 128;
      const int64_t parts = static_cast<int64_t>(p.splits) * p.s.batch * p.s.kv_heads;
      float* dst = p.splits > 1 ? p.partial + (((wg == 0 ? parts : 0) + (static_cast<int64_t>(split) * p.s.batch * p.s.kv_heads + bk)) *
                                               p.s.keys + key) * DP : nullptr;
#pragma unroll 1
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
        if (steps > 0) {
          tmem_ld32(acc + 32 * c, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0u;
        }
        if (p.splits > 1) {
          if (key < p.s.keys) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<float4*>(dst + 32 * c + k) =
                  make_float4(__uint_as_float(o[k]) * mul, __uint_as_float(o[k + 1]) * mul, __uint_as_float(o[k + 2]) * mul,
                              __uint_as_float(o[k + 3]) * mul);
          }
        } else {
          const uint32_t base = smem_u32(stage + (c / 2) * SM::kKeyChunk);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = pack16x2<BF>(__uint_as_float(o[8 * g + 2 * k]) * mul, __uint_as_float(o[8 * g + 2 * k + 1]) * mul);
            st_shared_v4(base + sw128_off(lane, (c & 1) * 4 + g), w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (p.splits == 1) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && key0 + quarter * 32 < p.s.keys) {
          for (int c = 0; c < SM::kChunks; ++c)
            if (64 * c < p.s.dim)
              tma_store_4d(wg == 0 ? &tm_dv : &tm_dk, stage + c * SM::kKeyChunk, 64 * c, key0 + quarter * 32, hk, b);
          bulk_commit_group();
          bulk_wait_group_read0();
        }
        __syncwarp();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, kDkvCols);
}

struct DkvSumParams {
  const float* partial;
  uint16_t *dk, *dv;
  int64_t dk_stride[3], dv_stride[3];
  int64_t keys, rows;               // rows = batch * kv_heads * keys
  int kv_heads, dim, splits;
};

// the splits' partial sums added in order; 8 elements per thread, blockIdx.y: dK, dV
template <int DP, bool BF>
__global__ void __launch_bounds__(256) cross_dkv_sum_kernel(const __grid_constant__ DkvSumParams p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = i / (DP / 8);
  const int e = static_cast<int>(i % (DP / 8)) * 8;
  if (row >= p.rows || e >= p.dim) return;
  const float* src = p.partial + (blockIdx.y * p.splits * p.rows + row) * DP + e;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), c = a;
  for (int s = 0; s < p.splits; ++s, src += p.rows * DP) {
    const float4 x = __ldcs(reinterpret_cast<const float4*>(src)), y = __ldcs(reinterpret_cast<const float4*>(src + 4));
    a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
    c.x += y.x; c.y += y.y; c.z += y.z; c.w += y.w;
  }
  const int64_t key = row % p.keys, bk = row / p.keys, hk = bk % p.kv_heads, b = bk / p.kv_heads;
  const int64_t* st = blockIdx.y ? p.dv_stride : p.dk_stride;
  uint16_t* dst = (blockIdx.y ? p.dv : p.dk) + b * st[0] + key * st[1] + hk * st[2] + e;
  *reinterpret_cast<uint4*>(dst) = make_uint4(pack16x2<BF>(a.x, a.y), pack16x2<BF>(a.z, a.w), pack16x2<BF>(c.x, c.y),
                                              pack16x2<BF>(c.z, c.w));
}

// Query-range splits of the dK / dV pass: the fewest rounds of CTAs times steps, each CTA's prologue and epilogue
// counted as a dozen steps.
int dkv_splits(const HtrcCrossArgs* a) {
  const int64_t units = a->batch * a->kv_heads * ((a->keys + kDkvKeys - 1) / kDkvKeys);
  const int64_t steps = (a->heads / a->kv_heads) * ((a->queries + kDkvRows - 1) / kDkvRows);
  const int64_t sms = sm_count();
  int best = 1;
  int64_t cost = INT64_MAX;
  for (int s = 1; s <= 16 && s <= std::max<int64_t>(steps, 1); ++s) {
    const int64_t c = ((units * s + sms - 1) / sms) * ((steps + s - 1) / s + 12);
    if (c < cost) {
      cost = c;
      best = s;
    }
  }
  return best;
}

int64_t stat_rows(const HtrcCrossArgs* a) { return (a->queries + kDqRows - 1) / kDqRows * kDqRows; }
size_t stat_bytes(const HtrcCrossArgs* a) { return (static_cast<size_t>(a->batch * a->heads * stat_rows(a)) * 12 + 255) / 256 * 256; }

template <typename K>
bool ready(K kernel, uint32_t bytes, bool (&done)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (dev < 64 && done[dev]) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  if (dev < 64) done[dev] = true;
  return true;
}

template <int DP, bool BF, int KIND>
int launch_bwd(const HtrcCrossArgs* a, cudaStream_t st) {
  static bool done_q[64] = {}, done_kv[64] = {};
  auto kq = cross_dq_kernel<DP, BF, KIND>;
  auto kkv = cross_dkv_kernel<DP, BF, KIND>;
  if (!ready(kq, DqSmem<DP>::kBytes, done_q) || !ready(kkv, DkvSmem<DP>::kBytes, done_kv)) return HTRC_ERR_CUDA;
  const CrossShape s = cross_shape(a);
  float* stat = static_cast<float*>(a->workspace);
  const bool keys = a->keys > 0, rows = a->queries > 0;
  // an empty side's maps are never read: the other side's rows stand in
  const void *k = keys ? a->k : a->q, *v = keys ? a->v : a->q, *q = rows ? a->q : a->k, *o = rows ? a->dout : a->k;
  const int64_t *ks = keys ? a->k_stride : a->q_stride, *vs = keys ? a->v_stride : a->q_stride;
  const int64_t *qs = rows ? a->q_stride : a->k_stride, *os = rows ? a->dout_stride : a->k_stride;
  const int64_t nk = keys ? a->keys : a->queries, nq = rows ? a->queries : a->keys;
  const int hk = keys ? a->kv_heads : a->heads, hq = rows ? a->heads : a->kv_heads;
  int do_b = 0, do_h = 0, one;
  if (rows) {
    CUtensorMap mq, mo, mk, mv, mdq;
    DqParams p{};
    p.s = s;
    if (!cross_map(&mq, a, q, qs, nq, hq, kDqRows, &p.s.q_b, &p.s.q_h) || !cross_map(&mo, a, o, os, nq, hq, kDqRows, &do_b, &do_h) ||
        !cross_map(&mk, a, k, ks, nk, hk, kDqKeys, &p.s.k_b, &p.s.k_h) || !cross_map(&mv, a, v, vs, nk, hk, kDqKeys, &p.s.v_b, &p.s.v_h) ||
        !cross_map(&mdq, a, a->dq, a->dq_stride, nq, hq, 32, &one, &one))
      return HTRC_ERR_CUDA;
    p.lse = a->lse;
    p.dlse = a->dlse;
    p.out = static_cast<const uint16_t*>(a->out);
    for (int i = 0; i < 3; ++i) p.out_stride[i] = a->out_stride[i];
    p.stat = stat;
    p.stat_rows = stat_rows(a);
    p.tiles = static_cast<int>(stat_rows(a) / kDqRows);
    p.status = a->status;
    kq<<<static_cast<unsigned>(p.tiles * a->batch * a->heads), kDqThreads, DqSmem<DP>::kBytes, st>>>(mq, mo, mk, mv, mdq, p, do_b, do_h);
    if (cudaGetLastError() != cudaSuccess) return HTRC_ERR_CUDA;
  }
  if (!keys) return HTRC_OK;
  CUtensorMap mq, mo, mk, mv, mdk, mdv;
  DkvParams p{};
  p.s = s;
  if (!cross_map(&mq, a, q, qs, nq, hq, kDkvRows, &p.s.q_b, &p.s.q_h) || !cross_map(&mo, a, o, os, nq, hq, kDkvRows, &do_b, &do_h) ||
      !cross_map(&mk, a, k, ks, nk, hk, kDkvKeys, &p.s.k_b, &p.s.k_h) || !cross_map(&mv, a, v, vs, nk, hk, kDkvKeys, &p.s.v_b, &p.s.v_h) ||
      !cross_map(&mdk, a, a->dk, a->dk_stride, nk, hk, 32, &one, &one) || !cross_map(&mdv, a, a->dv, a->dv_stride, nk, hk, 32, &one, &one))
    return HTRC_ERR_CUDA;
  p.stat = stat;
  p.stat_rows = stat_rows(a);
  p.key_blocks = static_cast<int>((a->keys + kDkvKeys - 1) / kDkvKeys);
  p.row_blocks = static_cast<int>((a->queries + kDkvRows - 1) / kDkvRows);
  p.splits = dkv_splits(a);
  p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + stat_bytes(a));
  p.status = a->status;
  const int64_t grid = a->batch * a->kv_heads * p.splits * p.key_blocks;
  kkv<<<static_cast<unsigned>(grid), kDkvThreads, DkvSmem<DP>::kBytes, st>>>(mq, mo, mk, mv, mdk, mdv, p, do_b, do_h);
  if (cudaGetLastError() != cudaSuccess) return HTRC_ERR_CUDA;
  if (p.splits > 1) {
    DkvSumParams r{};
    r.partial = p.partial;
    r.dk = static_cast<uint16_t*>(a->dk);
    r.dv = static_cast<uint16_t*>(a->dv);
    for (int i = 0; i < 3; ++i) {
      r.dk_stride[i] = a->dk_stride[i];
      r.dv_stride[i] = a->dv_stride[i];
    }
    r.keys = a->keys;
    r.rows = a->batch * a->kv_heads * a->keys;
    r.kv_heads = a->kv_heads;
    r.dim = a->dim;
    r.splits = p.splits;
    const int64_t blocks = (r.rows * (DP / 8) + 255) / 256;
    cross_dkv_sum_kernel<DP, BF><<<dim3(static_cast<unsigned>(blocks), 2), 256, 0, st>>>(r);
    if (cudaGetLastError() != cudaSuccess) return HTRC_ERR_CUDA;
  }
  return HTRC_OK;
}

template <int DP, bool BF>
int launch_bwd_kind(const HtrcCrossArgs* a, cudaStream_t st) {
  switch (cross_mask_kind(a)) {
    case CROSS_NONE: return launch_bwd<DP, BF, CROSS_NONE>(a, st);
    case CROSS_KEYS: return launch_bwd<DP, BF, CROSS_KEYS>(a, st);
    case CROSS_PAIRS: return launch_bwd<DP, BF, CROSS_PAIRS>(a, st);
    default: return launch_bwd<DP, BF, CROSS_BIAS>(a, st);
  }
}

int cross_sizes(const HtrcCrossArgs* a, size_t* bytes) {
  const int rc = cross_validate(a, true, false);
  if (rc != HTRC_OK) return rc;
  // the grids, and the workspace as a whole
  const int64_t limit = (int64_t(1) << 31) - 1;
  const int64_t tiles = stat_rows(a) / kDqRows, blocks = (a->keys + kDkvKeys - 1) / kDkvKeys;
  if (tiles * a->batch * a->heads > limit || blocks > limit / (16 * std::max<int64_t>(1, a->batch * a->kv_heads)))
    return HTRC_ERR_UNSUPPORTED;
  const int dp = a->dim <= 64 ? 64 : 128, splits = dkv_splits(a);
  *bytes = stat_bytes(a) + (splits > 1 ? static_cast<size_t>(2) * splits * a->batch * a->kv_heads * a->keys * dp * 4 : 0);
  return HTRC_OK;
}

int cross_backward(const HtrcCrossArgs* a, cudaStream_t st) {
  int rc = cross_validate(a, true, true);
  if (rc != HTRC_OK) return rc;
  size_t need = 0;
  rc = cross_sizes(a, &need);
  if (rc != HTRC_OK) return rc;
  if (!device_ok()) return HTRC_ERR_DEVICE;
  if (a->batch == 0 || (a->queries == 0 && a->keys == 0)) return HTRC_OK;
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 256))
    return HTRC_ERR_WORKSPACE;
  const bool bf = a->dtype == HTRC_LAYER_BF16;
  if (a->dim <= 64) return bf ? launch_bwd_kind<64, true>(a, st) : launch_bwd_kind<64, false>(a, st);
  return bf ? launch_bwd_kind<128, true>(a, st) : launch_bwd_kind<128, false>(a, st);
}

}  // namespace

}  // namespace htrc

extern "C" {

int htrc_cross_backward_workspace_size(const HtrcCrossArgs* args, size_t* bytes) {
  if (bytes == nullptr) return HTRC_ERR_ARG;
  return htrc::cross_sizes(args, bytes);
}

int htrc_cross_backward(const HtrcCrossArgs* args, htrc_stream_t stream) {
  return htrc::cross_backward(args, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
