// Cross attention to an encoder's states of another length, forward, and the checks its C entries share.
//
// A unit of work is 256 query rows of one head (two tiles of 128, one per softmax warpgroup) and a range of its keys; a
// persistent CTA per SM walks the units.  Per block of 128 keys and tile:  S = Q K^T (tcgen05, float32 in TMEM), one
// thread per row takes the block's maximum and P = exp2(S scale log2 e - m), P goes back over S in TMEM as 16-bit words
// and O += P V accumulates in TMEM; the sum of P is kept in float32 from the unrounded values.  The running maximum is
// lazy: O is rescaled only when a row's maximum grew by more than 2^8 (P <= 256 until then).
//
// The two tiles share each block of K and V and run under one another's exponentials, each with an MMA warp of its own
// (TMEM: two S and two O, 512 columns).  Within a tile the next block's S starts early: S stands in two halves of 64
// keys, P covers the columns of the second, and the first half's columns are free once the threads hold S in registers,
// so its product for the next block runs under this block's exponentials, and only the second half's follows P V.  P is
// handed over a quarter at a time.  The K / V ring runs on into the next unit, whose first S is ready before a
// warpgroup has finished the last one's epilogue.
//
// Where there are few units the keys are split; the parts' float32 O, maxima and sums are joined by cross_join_kernel.
//
// Rounding: P is rounded to the operands' 16-bit type for the second product (a relative 2^-9 for bfloat16, of
// weights whose errors average out over the row); out is rounded once from float32.
//
// Measured, bfloat16, 24 heads of 128, device time of 20 passes: 129,024 queries x 512 keys 839 us after a second's rest (968
// TFLOP/s) and 972 once the power cap holds the SM clock, at 1,605 MHz (836); 4,096 x 16,384 761 and 851 (1,725 MHz).  Times
// beside variants below are after a rest.  The exponentials' turns bound it: 1,700 clocks for a tile's block, of which the special function units need
// 1,024 and the products, under the other tile's turn, 1,280.
//
// Warps 0-3 and 4-7: softmax of tile A and B, rows 32 w ..; warp 8: TMA; warps 9 and 10: MMA issue of tile A and B, and
// the zeroing of excluded keys' values.
#include <algorithm>
#include <cmath>

#include "cross.cuh"

namespace htrc {

namespace {

constexpr int kXThreads = 352;
constexpr int kXRows = 128, kXUnit = 256, kXKeys = 128;
constexpr uint32_t kXChunk = 128 * 128;            // 128 rows of 64 16-bit elements
constexpr uint32_t kXColS = 0, kXColO = 256, kXCols = 512;   // tile t: S at 128 t, O at 256 + 128 t
constexpr float kXRescale = 8.0f;

template <int DP>
struct CrossFwdSmem {
  static constexpr int kChunks = DP / 64, kSlots = 4;
  static constexpr uint32_t kTile = kChunks * kXChunk, kStage = 32 * 128;      // a warp's 32 output rows of 64 columns
  static constexpr uint32_t kQ = 0, kKV = 2 * kTile, kOut = kKV + kSlots * kTile, kBias = kOut + 8 * kStage;
  static constexpr uint32_t kBars = kBias + 4 * kXKeys * 4, kBytes = kBars + 320;
};

struct CrossBars {
  uint64_t q_full[2], q_empty[2], kv_full[4], kv_empty[4], s_full[2][2], s_read[2], p_full[2][4], o_full[2], turn[2], idle[2];
  uint32_t tmem_base;
  int abort_flag, loads[3];           // of the TMA warp in all: K / V, Q of either tile
};
static_assert(sizeof(CrossBars) <= 320, "barriers");

struct CrossFwdParams {
  CrossShape s;
  float* lse;
  void* out;
  int64_t os[3];
  uint32_t units, pairs;      // pairs of tiles per head
  int splits;
  float* part;                // splits > 1: O [split][batch * heads][queries][DP], not divided by the sum
  float2* part_ml;            // (maximum, sum) [split][batch * heads][queries]
  int* status;
};

// A CTA's units, and within one its blocks of keys
struct Walk {
  uint32_t unit;
  int b, h, row0, split, count, j, j1;
  __device__ __forceinline__ void open(const CrossFwdParams& p, uint32_t u) {
    unit = u;
    if (u >= p.units) return;
    const uint32_t rest = u / p.pairs, pair = u - rest * p.pairs;
    uint32_t bh = rest;
    split = 0;
    if (p.splits > 1) {
      bh = rest / p.splits;
      split = static_cast<int>(rest - bh * p.splits);
    }
    b = static_cast<int>(bh / static_cast<uint32_t>(p.s.heads));
    h = static_cast<int>(bh - b * static_cast<uint32_t>(p.s.heads));
    row0 = static_cast<int>(pair) * kXUnit;
    count = key_count(p.s, b);
    j = 0;
    j1 = (count + kXKeys - 1) / kXKeys;
    if (p.splits > 1) {
      const int64_t nb = j1;
      j = static_cast<int>(nb * split / p.splits);
      j1 = static_cast<int>(nb * (split + 1) / p.splits);
    }
  }
  __device__ __forceinline__ bool done(const CrossFwdParams& p) const { return unit >= p.units; }
  // the first unit from u on that has a block
  __device__ __forceinline__ void open_live(const CrossFwdParams& p, uint32_t u) {
    for (open(p, u); !done(p) && j >= j1;) open(p, unit + gridDim.x);
  }
  __device__ __forceinline__ void next(const CrossFwdParams& p) {
    if (++j >= j1) open_live(p, unit + gridDim.x);
  }
};

template <int DP, bool BF, int KIND>
__global__ void __launch_bounds__(kXThreads, 1)
    cross_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                     const __grid_constant__ CrossFwdParams p) {
  using SM = CrossFwdSmem<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023) {          // the swizzled tiles need it; there is no room to round up
    flag_status(p.status, ST_WAIT_TIMEOUT);
    return;
  }
  CrossBars* bars = reinterpret_cast<CrossBars*>(smem + SM::kBars);
  volatile int* abort_flag = &bars->abort_flag;
  int* status = p.status;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars->q_full[t], 1);
      mbar_init(&bars->q_empty[t], 1);
      mbar_init(&bars->s_full[t][0], 1);
      mbar_init(&bars->s_full[t][1], 1);
      mbar_init(&bars->s_read[t], 128);
      for (int c = 0; c < 4; ++c) mbar_init(&bars->p_full[t][c], 128);
      mbar_init(&bars->o_full[t], 1);
      mbar_init(&bars->turn[t], 4);
      mbar_init(&bars->idle[t], 1);
    }
    for (int i = 0; i < SM::kSlots; ++i) {
      mbar_init(&bars->kv_full[i], 1);
      mbar_init(&bars->kv_empty[i], 2);
    }
    bars->abort_flag = bars->loads[0] = bars->loads[1] = bars->loads[2] = 0;
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(&bars->tmem_base, kXCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  Walk w{};

  if (warp == 8) {
    // ------------------------------------------------------------------ TMA
    const uint64_t pol_q = policy_evict_first(), pol_kv = policy_evict_last();
    const uint32_t leader = elect_one();
    int slots = 0, units[2] = {0, 0};   // ring slots filled, tiles of queries loaded
    auto load = [&](const Walk& at, int j, int kv) -> bool {
      const int s = slots % SM::kSlots, hk = at.h / p.s.group;
      if (slots >= SM::kSlots && !mbar_wait_warp(&bars->kv_empty[s], ((slots / SM::kSlots) - 1) & 1, status, abort_flag))
        return false;
      if (leader) {
        mbar_arrive_expect_tx(&bars->kv_full[s], SM::kTile);
        for (int c = 0; c < SM::kChunks; ++c)
          tma_load_4d(smem + SM::kKV + s * SM::kTile + c * kXChunk, kv ? &tm_v : &tm_k, &bars->kv_full[s], 64 * c,
                      j * kXKeys, hk * (kv ? p.s.v_h : p.s.k_h), at.b * (kv ? p.s.v_b : p.s.k_b), pol_kv);
      }
      __syncwarp();
      ++slots;
      return true;
    };
    bool ok = true;
    for (w.open_live(p, blockIdx.x); ok && !w.done(p); w.open_live(p, w.unit + gridDim.x)) {
      ok = load(w, w.j, 0);
      for (int t = 0; t < 2 && ok; ++t) {
        if (w.row0 + t * kXRows >= p.s.queries) continue;
        ok = units[t] == 0 || mbar_wait_warp(&bars->q_empty[t], (units[t] - 1) & 1, status, abort_flag);
        if (!ok) break;
        if (leader) {
          mbar_arrive_expect_tx(&bars->q_full[t], SM::kTile);
          for (int c = 0; c < SM::kChunks; ++c)
            tma_load_4d(smem + SM::kQ + t * SM::kTile + c * kXChunk, &tm_q, &bars->q_full[t], 64 * c, w.row0 + t * kXRows,
                        w.h * p.s.q_h, w.b * p.s.q_b, pol_q);
        }
        __syncwarp();
        ++units[t];
      }
      ok = ok && load(w, w.j, 1);
      for (int j = w.j + 1; ok && j < w.j1; ++j) ok = load(w, j, 0) && load(w, j, 1);
    }
    if (ok) {      // the last releases have landed before the CTA leaves
      drain_ring<true>(bars->kv_empty, SM::kSlots, slots, status, abort_flag);
      for (int t = 0; t < 2; ++t)
        if (units[t] > 0) mbar_wait_warp(&bars->q_empty[t], (units[t] - 1) & 1, status, abort_flag);
    }
    if (lane == 0) {
      bars->loads[0] = slots;
      bars->loads[1] = units[0];
      bars->loads[2] = units[1];
    }
  } else if (warp >= 9) {
    // ------------------------------------------------------------------ MMA of tile t
    const int t = warp - 9;
    const uint32_t leader = elect_one();
    const uint32_t id_s = idesc16<BF>(128, kXKeys / 2, false, false);
    const uint32_t id_o = idesc16<BF>(128, DP, false, true);
    const uint64_t dq = desc_k(smem_u32(smem + SM::kQ + t * SM::kTile)), dk = desc_k(smem_u32(smem + SM::kKV));
    const uint64_t dv = desc_mn(smem_u32(smem + SM::kKV), kXChunk);
    const uint32_t col_s = tmem + kXColS + 128 * t, col_o = tmem + kXColO + 128 * t;
    Walk a;                             // one step ahead of w
    a.open_live(p, blockIdx.x);
    int ahead = 0, units = 0;           // a's step, and its unit among those with this tile
    bool opened = false;                // a's queries have been waited for
    // half of S of a's step (K in ring slot 2 * ahead): keys 0-63 to columns 64-127, keys 64-127 to columns 0-63
    auto scores = [&](int half) -> bool {
      const int at = 2 * ahead, s = at % SM::kSlots;
      if (half == 0) {
        if (!mbar_wait_warp(&bars->kv_full[s], (at / SM::kSlots) & 1, status, abort_flag)) return false;
        if (!opened) {
          if (!mbar_wait_warp(&bars->q_full[t], units & 1, status, abort_flag)) return false;
          opened = true;
        }
        tc_fence_after();
      }
      const uint64_t ko = (s * SM::kTile + half * 64 * 128) >> 4;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const uint32_t o = ((kk / 4) * kXChunk + (kk % 4) * 32) >> 4;
        mma_bf16_by(leader, col_s + (half ? 0 : 64), dq + o, dk + ko + o, id_s, kk != 0);
      }
      mma_commit_by(leader, &bars->s_full[t][half]);
      if (half == 1) {
        mma_commit_by(leader, &bars->kv_empty[s]);
        if (a.j + 1 == a.j1) {
          mma_commit_by(leader, &bars->q_empty[t]);
          ++units;
          opened = false;
        }
        ++ahead;
        a.next(p);
      }
      return true;
    };
    // the ring's slots of a unit without this tile are released as they fill
    auto skip = [&](int slot) -> bool {
      const int s = slot % SM::kSlots;
      if (!mbar_wait_warp(&bars->kv_full[s], (slot / SM::kSlots) & 1, status, abort_flag)) return false;
      if (leader) mbar_arrive(&bars->kv_empty[s]);
      __syncwarp();
      return true;
    };
    auto mine = [&](const Walk& x) { return x.row0 + t * kXRows < p.s.queries; };
    bool ok = true, first = true;
    int n = 0, own = 0;                 // steps, and those of this tile
    for (w.open_live(p, blockIdx.x); ok && !w.done(p); ++n) {
      if (!mine(w)) {
        ok = skip(2 * n) && skip(2 * n + 1);
        w.next(p);
        if (ahead == n) {
          ++ahead;
          a.next(p);
        }
        continue;
      }
      if (ahead == n) ok = scores(0) && scores(1);      // nothing was under way: the first step, or one after a unit without this tile
      const bool more = !a.done(p) && mine(a), last = w.j + 1 == w.j1;
      if (ok && more) {
        // the columns of the next S's first half are free once S is in the threads' registers
        ok = mbar_wait_warp(&bars->s_read[t], own & 1, status, abort_flag) && scores(0);
      }
      const int at = 2 * n + 1, s = at % SM::kSlots;
      ok = ok && mbar_wait_warp(&bars->kv_full[s], (at / SM::kSlots) & 1, status, abort_flag);
      if (!ok) break;
      // a block with keys that no query sees: their values may hold anything (0 * NaN), so they become zeros
      if (KIND == CROSS_KEYS || (w.count < p.s.keys && (w.j + 1) * kXKeys > w.count))
        zero_excluded_rows<kXKeys, SM::kChunks>(smem + SM::kKV + s * SM::kTile, kXChunk, w.j * kXKeys, w.count, p.s,
                                                w.b * p.s.mask.sb + w.h * p.s.mask.sh, KIND == CROSS_KEYS, lane);
      const uint64_t vo = (s * SM::kTile) >> 4;
      for (int c = 0; c < 4; ++c) {
        ok = mbar_wait_warp(&bars->p_full[t][c], own & 1, status, abort_flag);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int kk = 2 * c + i;
          mma_bf16_ts_by(leader, col_o, col_s + 8 * kk, dv + vo + ((kk * 2048) >> 4), id_o, !first || kk != 0);
        }
      }
      if (!ok) break;
      if (last) mma_commit_by(leader, &bars->o_full[t]);
      mma_commit_by(leader, &bars->kv_empty[s]);
      if (more) ok = scores(1);
      first = last;
      ++own;
      w.next(p);
    }
  } else {
    // ------------------------------------------------------------------ softmax, one thread per row
    const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t col_s = tmem + lanes + kXColS + 128 * t, col_o = tmem + lanes + kXColO + 128 * t;
    const float scale2 = p.s.scale * kCrossLog2e;
    constexpr bool NAT = KIND == CROSS_KEYS || KIND == CROSS_BIAS;   // logits kept in natural units
    float* bias = reinterpret_cast<float*>(smem + SM::kBias) + t * 2 * kXKeys;
    int steps = 0, units = 0, turns = 0;      // of this tile; steps taken in turns
    bool ok = true;
    for (w.open(p, blockIdx.x); ok && !w.done(p); w.open(p, w.unit + gridDim.x)) {
      const bool live = w.j < w.j1, mine = w.row0 + t * kXRows < p.s.queries;
      const int row0 = w.row0 + t * kXRows, row = row0 + r;
      const bool valid = row < p.s.queries;
      const int64_t at = (static_cast<int64_t>(w.b) * p.s.heads + w.h) * p.s.queries + row;
      const int64_t mask_at = w.b * p.s.mask.sb + w.h * p.s.mask.sh;
      float m = -INFINITY, l = 0.f;
      for (int j = w.j; mine && j < w.j1; ++j, ++steps) {
        const int left = w.count - j * kXKeys;            // keys of this block
        uint32_t bits[4] = {0u, 0u, 0u, 0u};
        float* bj = bias + (steps & 1) * kXKeys;
        if (KIND == CROSS_KEYS) {
          bj[r] = r < left ? mask_term(p.s.mask.p, p.s.mask.dtype,
                                       mask_at + static_cast<int64_t>(j * kXKeys + r) * p.s.mask.sm) : -INFINITY;
          named_bar_sync(1 + t, 128);
        }
        if ((KIND == CROSS_PAIRS || KIND == CROSS_BIAS) && valid && left > kXKeys)      // the next block's terms of this row
          prefetch_mask(p.s.mask, mask_at + row * p.s.mask.sn + static_cast<int64_t>((j + 1) * kXKeys) * p.s.mask.sm);
        if (KIND == CROSS_PAIRS) {
          // the warp's 32 rows of mask bits: a lane's four keys of each row, by one load where all rows are aligned
          // to it, else a byte each, and ballots: bit k of word q is key 4 k + q.  (5 x 52 queries x 260 keys x 6 heads: 15.6
          // us, consecutive bytes 22.1; 2 x 29,540 x 1,151 x 2, by bytes: 302 us, 284 with a word of consecutive keys; two
          // aligned words shifted together: 437)
          const int rows = min(32, static_cast<int>(p.s.queries) - (row0 + quarter * 32)), mine4 = left - 4 * lane;
          const uint32_t keep = mine4 >= 4 ? 0xffffffffu : mine4 <= 0 ? 0u : (1u << 8 * mine4) - 1u;
          const uint8_t* mk = static_cast<const uint8_t*>(p.s.mask.p) + mask_at + static_cast<int64_t>(row0 + quarter * 32) * p.s.mask.sn +
                              static_cast<int64_t>(j * kXKeys + 4 * lane) * p.s.mask.sm;
          auto vote = [&](int row, uint32_t v) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t word = __ballot_sync(0xffffffffu, (v >> 8 * q & 0xffu) != 0);
              if (lane == row) bits[q] = word;
            }
          };
          if (p.s.mask.sm == 1 && !((reinterpret_cast<uintptr_t>(p.s.mask.p) + mask_at) & 3) && !(p.s.mask.sn & 3)) {
            // (a word with one of the row's keys in it lies in the mask's allocation as a whole)
            for (int g = 0; g < rows; g += 16) {
              uint32_t v[16];
#pragma unroll
              for (int i = 0; i < 16; ++i)
                v[i] = g + i < rows && keep ? __ldg(reinterpret_cast<const uint32_t*>(mk + i * p.s.mask.sn)) & keep : 0u;
#pragma unroll
              for (int i = 0; i < 16; ++i) vote(g + i, v[i]);
              mk += 16 * p.s.mask.sn;
            }
          } else {
            for (int g = 0; g < rows; g += 8) {
              uint32_t v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                v[i] = 0;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  if (g + i < rows && q < mine4) v[i] |= static_cast<uint32_t>(__ldg(mk + i * p.s.mask.sn + q * p.s.mask.sm)) << 8 * q;
              }
#pragma unroll
              for (int i = 0; i < 8; ++i) vote(g + i, v[i]);
              mk += 8 * p.s.mask.sn;
            }
          }
        }
        // the block's logits: times scale2 in the exponent for NONE / PAIRS, natural units with a bias
        uint32_t s[4][32];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          ok = mbar_wait_warp(&bars->s_full[t][half], steps & 1, status, abort_flag);
          if (!ok) break;
          tc_fence_after();
          tmem_ld32(col_s + (half ? 0 : 64), s[2 * half]);
          tmem_ld32(col_s + (half ? 32 : 96), s[2 * half + 1]);
        }
        if (!ok) break;
        tmem_ld_wait();
        tc_fence_before();
        mbar_arrive(&bars->s_read[t]);
        if (KIND == CROSS_NONE) {
          if (left < kXKeys) {
#pragma unroll
            for (int i = 0; i < kXKeys; ++i)
              if (i >= left) s[i / 32][i % 32] = __float_as_uint(-INFINITY);
          }
        } else if (KIND == CROSS_PAIRS) {
#pragma unroll
          for (int i = 0; i < kXKeys; ++i)
            if (!(bits[i % 4] >> (i / 4) & 1u)) s[i / 32][i % 32] = __float_as_uint(-INFINITY);
        } else if (KIND == CROSS_KEYS) {
#pragma unroll
          for (int i = 0; i < kXKeys; ++i) {
            uint32_t& x = s[i / 32][i % 32];
            x = __float_as_uint(bj[i] == -INFINITY ? bj[i] : fmaf(__uint_as_float(x), p.s.scale, bj[i]));
          }
        } else {
          const int64_t row_at = mask_at + (valid ? row : 0) * p.s.mask.sn + static_cast<int64_t>(j * kXKeys) * p.s.mask.sm;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            float b[16];
            mask_terms<16>(p.s.mask.p, p.s.mask.dtype, row_at + static_cast<int64_t>(16 * c) * p.s.mask.sm, p.s.mask.sm, left - 16 * c, b);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              uint32_t& x = s[c / 2][16 * (c & 1) + i];
              x = __float_as_uint(b[i] == -INFINITY ? b[i] : fmaf(__uint_as_float(x), p.s.scale, b[i]));
            }
          }
        }
        float mxs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 32; i += 2)
#pragma unroll
          for (int c = 0; c < 4; ++c) mxs[c] = max3(mxs[c], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
        float mx = fmaxf(fmaxf(mxs[0], mxs[1]), fmaxf(mxs[2], mxs[3]));
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
        if (j > w.j && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
          for (int c = 0; c < DP / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(col_o + 16 * c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st16(col_o + 16 * c, o);
          }
        }
        // The two tiles' exponentials take turns: each then has the special function units to itself, and the other's
        // loads, maxima and products run meanwhile (together, both would wait for the units and then both leave them:
        // 4,115 clocks a pair of steps, 3,900 in turns).  The turn passes on before the last quarter has landed
        const bool two = w.row0 + kXRows < p.s.queries;
        if (two && (t == 1 || turns > 0)) {
          ok = mbar_wait_warp(&bars->turn[t], (turns - (t == 0)) & 1, status, abort_flag);
          if (!ok) break;
        }
        const float mref = m == -INFINITY ? 0.f : m;      // nothing seen yet: every term is exp2(-inf) = 0
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        auto weights = [&]() {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pw[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float2 e = make_float2(__uint_as_float(s[c][2 * i]), __uint_as_float(s[c][2 * i + 1]));
              if (NAT)
                e = mul2(sub2(e, make_float2(mref, mref)), make_float2(kCrossLog2e, kCrossLog2e));
              else
                e = fma2(e, make_float2(scale2, scale2), make_float2(-mref, -mref));
              e = make_float2(cross_ex2(e.x), cross_ex2(e.y));
              sum[i & 1] = add2(sum[i & 1], e);
              pw[i] = pack16x2<BF>(e.x, e.y);
            }
            tmem_st16(col_s + 16 * c, pw);
            if (two && c == 3 && lane == 0) mbar_arrive(&bars->turn[t ^ 1]);
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&bars->p_full[t][c]);
          }
        };
        // without a mask whole blocks have a copy of their own: one copy for these and the ragged last ones spills more
        // (129,024 queries x 512 keys x 24 heads: 840 us, 837 with two; 4,096 x 16,384: 763 and 758)
        if (KIND == CROSS_NONE && left >= kXKeys)
          weights();
        else
          weights();
        turns += two;
        sum[0] = add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
      }
      if (!ok) break;
      if (live && mine) {
        ok = mbar_wait_warp(&bars->o_full[t], units & 1, status, abort_flag);
        if (!ok) break;
        tc_fence_after();
        ++units;
      }
      if (mine && p.splits > 1) {
        // a part: O as it is, the maximum and the sum
        const int64_t rows = p.s.batch * p.s.heads * p.s.queries;
        if (valid) p.part_ml[w.split * rows + at] = make_float2(m, l);
        float* dst = p.part + (w.split * rows + at) * DP;
        if (live) {
#pragma unroll 1
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(col_o + 32 * c, o);
            tmem_ld_wait();
            if (valid) {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<uint4*>(dst + 32 * c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
          }
        }
      } else if (mine) {
        if (valid && p.lse != nullptr)
          p.lse[at] = l > 0.f || l != l ? (NAT ? m : m * kCrossLn2) + logf(l) : -INFINITY;
        if (live) {
          const float inv = l == 0.f ? 0.f : 1.0f / l;
          // 64 columns at a time through the warp's staging rows, stored by TMA: rows past the end and columns past dim
          // are not written
          uint8_t* stage = smem + SM::kOut + warp * SM::kStage;
#pragma unroll 1
          for (int c = 0; c < SM::kChunks; ++c) {
            uint32_t x[32];
            {
              uint32_t o[2][32];
              tmem_ld32(col_o + 64 * c, o[0]);
              tmem_ld32(col_o + 64 * c + 32, o[1]);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i)
                x[i] = pack16x2<BF>(__uint_as_float(o[i / 16][2 * (i % 16)]) * inv, __uint_as_float(o[i / 16][2 * (i % 16) + 1]) * inv);
            }
            if (lane == 0) bulk_wait_group_read0();         // the last rows have left
            __syncwarp();
#pragma unroll
            for (int g = 0; g < 8; ++g)
              st_shared_v4(smem_u32(stage) + sw128_off(lane, g), x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && row0 + quarter * 32 < p.s.queries && 64 * c < p.s.dim) {
              tma_store_4d(&tm_o, stage, 64 * c, row0 + quarter * 32, w.h, w.b);
              bulk_commit_group();
            }
          }
        } else if (valid) {
          // no keys at all: zeros
          uint16_t* dst = static_cast<uint16_t*>(p.out) + w.b * p.os[0] + row * p.os[1] + w.h * p.os[2];
          for (int c = 0; c < p.s.dim; c += 8) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0, 0, 0, 0);
        }
      }
    }
    if (lane == 0) bulk_wait_group_read0();                 // the staging rows outlive the CTA's last stores
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (warp == 8) {
      settle_loads(bars->kv_full, SM::kSlots, bars->loads[0], status);
      settle_loads(&bars->q_full[0], 1, bars->loads[1], status);
      settle_loads(&bars->q_full[1], 1, bars->loads[2], status);
    } else if (warp >= 9) {
      settle_products(&bars->idle[warp - 9], status);
    }
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, kXCols);
}

struct CrossJoinParams {
  const float* part;
  const float2* ml;
  float* lse;
  uint16_t* out;
  int64_t os[3], rows, queries;
  int heads, dim, splits;
  bool natural;             // the maxima are in natural units
};

// out and lse of the rows whose keys were split; 8 elements per thread
template <int DP, bool BF>
__global__ void __launch_bounds__(256) cross_join_kernel(const __grid_constant__ CrossJoinParams p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = i / (DP / 8);
  const int e = static_cast<int>(i % (DP / 8)) * 8;
  if (row >= p.rows) return;
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.ml[s * p.rows + row].x);
  const float unit = p.natural ? kCrossLog2e : 1.0f;
  float l = 0.f, acc[8] = {};
  for (int s = 0; s < p.splits; ++s) {
    const float2 ml = p.ml[s * p.rows + row];
    if (ml.x == -INFINITY && ml.y == 0.f) continue;         // a part with no key: its O was not written
    const float w = cross_ex2((ml.x - m) * unit);
    l = fmaf(ml.y, w, l);
    const float4* src = reinterpret_cast<const float4*>(p.part + (s * p.rows + row) * DP + e);
    const float4 x = __ldcs(src), y = __ldcs(src + 1);
    acc[0] = fmaf(x.x, w, acc[0]); acc[1] = fmaf(x.y, w, acc[1]); acc[2] = fmaf(x.z, w, acc[2]); acc[3] = fmaf(x.w, w, acc[3]);
    acc[4] = fmaf(y.x, w, acc[4]); acc[5] = fmaf(y.y, w, acc[5]); acc[6] = fmaf(y.z, w, acc[6]); acc[7] = fmaf(y.w, w, acc[7]);
  }
  if (e == 0 && p.lse != nullptr) p.lse[row] = l > 0.f || l != l ? (p.natural ? m : m * kCrossLn2) + logf(l) : -INFINITY;
  if (e >= p.dim) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const int64_t n = row % p.queries, bh = row / p.queries, h = bh % p.heads, b = bh / p.heads;
  *reinterpret_cast<uint4*>(p.out + b * p.os[0] + n * p.os[1] + h * p.os[2] + e) =
      make_uint4(pack16x2<BF>(acc[0] * inv, acc[1] * inv), pack16x2<BF>(acc[2] * inv, acc[3] * inv),
                 pack16x2<BF>(acc[4] * inv, acc[5] * inv), pack16x2<BF>(acc[6] * inv, acc[7] * inv));
}

template <int DP, bool BF, int KIND>
int launch_fwd(const CUtensorMap* maps, const CrossFwdParams& p, cudaStream_t st) {
  static bool done[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return HTRC_ERR_CUDA;
  auto kernel = cross_fwd_kernel<DP, BF, KIND>;
  constexpr uint32_t bytes = CrossFwdSmem<DP>::kBytes;
  static_assert(bytes <= 232448, "shared memory of one CTA");
  if (dev >= 64 || !done[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return HTRC_ERR_CUDA;
    if (dev < 64) done[dev] = true;
  }
  const unsigned grid = std::min<uint32_t>(p.units, static_cast<uint32_t>(sm_count()));
  kernel<<<grid, kXThreads, bytes, st>>>(maps[0], maps[1], maps[2], maps[3], p);
  if (cudaGetLastError() != cudaSuccess) return HTRC_ERR_CUDA;
  if (p.splits > 1) {
    CrossJoinParams j{};
    j.part = p.part;
    j.ml = p.part_ml;
    j.lse = p.lse;
    j.out = static_cast<uint16_t*>(p.out);
    for (int i = 0; i < 3; ++i) j.os[i] = p.os[i];
    j.rows = p.s.batch * p.s.heads * p.s.queries;
    j.queries = p.s.queries;
    j.heads = p.s.heads;
    j.dim = p.s.dim;
    j.splits = p.splits;
    j.natural = KIND == CROSS_KEYS || KIND == CROSS_BIAS;
    const int64_t blocks = (j.rows * (DP / 8) + 255) / 256;
    cross_join_kernel<DP, BF><<<static_cast<unsigned>(blocks), 256, 0, st>>>(j);
    if (cudaGetLastError() != cudaSuccess) return HTRC_ERR_CUDA;
  }
  return HTRC_OK;
}

template <int DP, bool BF>
int launch_kind(int kind, const CUtensorMap* maps, const CrossFwdParams& p, cudaStream_t st) {
  switch (kind) {
    case CROSS_NONE: return launch_fwd<DP, BF, CROSS_NONE>(maps, p, st);
    case CROSS_KEYS: return launch_fwd<DP, BF, CROSS_KEYS>(maps, p, st);
    case CROSS_PAIRS: return launch_fwd<DP, BF, CROSS_PAIRS>(maps, p, st);
    default: return launch_fwd<DP, BF, CROSS_BIAS>(maps, p, st);
  }
}

bool rows_ok(const void* p, const int64_t* stride) {
  if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (stride[i] < 0 || stride[i] % 8 || stride[i] >= (int64_t(1) << 38)) return false;
  return true;
}

// Whether the rows that share a key head go without matrix tiles (cross_few.cu): 16 at most, a chunk of its products, or
// two chunks where this file's units alone fill the SMs, so that it would not split their keys.  4 entries x 24 heads x
// 1,000 keys: 16 rows 22.4 us there and 20.2 here, 24 rows 29.3 and 20.3; 16 x 24 heads on 8 key heads of 1,000 keys: 24
// rows 35.9 and 53.9; 64 x 24 x 500: 16 rows 67 and 112, 32 rows 87 and 112, 64 rows 155 and 112.
bool few_rows(const HtrcCrossArgs* a) {
  const int64_t rows = a->heads / a->kv_heads * a->queries;
  return rows <= kCrossFewRows || (rows <= 2 * kCrossFewRows && a->batch * a->heads >= sm_count());
}

// Parts the keys are split into: the fewest rounds of CTAs times blocks (1.2 us each), with about two blocks' time for a
// unit's ends and, for any split, four for the second launch and the time that the parts' bytes take at 5 TB/s.

int fwd_splits(const HtrcCrossArgs* a) {
  if (few_rows(a)) return 1;
  const int64_t units = a->batch * a->heads * ((a->queries + kXUnit - 1) / kXUnit), sms = sm_count();
  const int64_t blocks = (a->keys + kXKeys - 1) / kXKeys;
  if (units == 0 || units >= 4 * sms) return 1;
  int best = 1;
  int64_t cost = INT64_MAX;
  const int64_t row_bytes = a->batch * a->heads * a->queries * (a->dim <= 64 ? 64 : 128) * 8;     // written and read
  for (int s = 1; s <= 64 && s <= std::max<int64_t>(blocks, 1); ++s) {
    const int64_t c = ((units * s + sms - 1) / sms) * ((blocks + s - 1) / s + 2) + (s > 1 ? 4 + row_bytes * s / 6000000 : 0);
    if (c < cost) {
      cost = c;
      best = s;
    }
  }
  return best;
}

size_t fwd_rows_bytes(const HtrcCrossArgs* a, int splits) {
  return (static_cast<size_t>(splits) * a->batch * a->heads * a->queries * 8 + 255) / 256 * 256;
}

size_t fwd_bytes(const HtrcCrossArgs* a, int splits) {
  if (splits == 1) return 0;
  const int dp = a->dim <= 64 ? 64 : 128;
  return fwd_rows_bytes(a, splits) + static_cast<size_t>(splits) * a->batch * a->heads * a->queries * dp * 4;
}

int fwd_sizes(const HtrcCrossArgs* a, int* splits, size_t* bytes) {
  const int rc = cross_validate(a, false, false);
  if (rc != HTRC_OK) return rc;
  *splits = fwd_splits(a);
  const int64_t units = a->batch * a->heads * ((a->queries + kXUnit - 1) / kXUnit) * *splits;
  if (units > (int64_t(1) << 31) - 1) return HTRC_ERR_UNSUPPORTED;
  *bytes = few_rows(a) ? cross_few_bytes(a) : fwd_bytes(a, *splits);
  return HTRC_OK;
}

int cross_forward(const HtrcCrossArgs* a, cudaStream_t st) {
  int rc = cross_validate(a, false, true);
  if (rc != HTRC_OK) return rc;
  int splits = 1;
  size_t need = 0;
  rc = fwd_sizes(a, &splits, &need);
  if (rc != HTRC_OK) return rc;
  if (!device_is_b200()) return HTRC_ERR_DEVICE;
  if (a->batch * a->queries == 0) return HTRC_OK;
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 256))
    return HTRC_ERR_WORKSPACE;
  if (few_rows(a)) return cross_forward_few(a, st);
  CrossFwdParams p{};
  p.s = cross_shape(a);
  p.lse = a->lse;
  p.out = a->out;
  for (int i = 0; i < 3; ++i) p.os[i] = a->out_stride[i];
  p.status = a->status;
  p.pairs = static_cast<uint32_t>((a->queries + kXUnit - 1) / kXUnit);
  p.splits = splits;
  p.units = static_cast<uint32_t>(p.pairs * a->batch * a->heads * splits);
  if (need > 0) {
    p.part_ml = static_cast<float2*>(a->workspace);
    p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + fwd_rows_bytes(a, splits));
  }
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
  if (a->dim <= 64) return bf ? launch_kind<64, true>(kind, maps, p, st) : launch_kind<64, false>(kind, maps, p, st);
  return bf ? launch_kind<128, true>(kind, maps, p, st) : launch_kind<128, false>(kind, maps, p, st);
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

extern "C" int htrc_cross_forward_workspace_size(const HtrcCrossArgs* args, size_t* bytes) {
  if (bytes == nullptr) return HTRC_ERR_ARG;
  int splits = 1;
  return htrc::fwd_sizes(args, &splits, bytes);
}

extern "C" int htrc_cross_forward(const HtrcCrossArgs* args, htrc_stream_t stream) {
  return htrc::cross_forward(args, reinterpret_cast<cudaStream_t>(stream));
}
