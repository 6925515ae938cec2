// Cross attention, backward.  With P = exp(S scale + mask - lse), dP = dO V^T, delta = rowsum(dO out) - dlse and
// dS = P (dP - delta):   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO;  the gradients of a shared key head are
// summed over its query heads.
//
// Two passes, each recomputing S and dP on tcgen05, so that no gradient needs an atomic and every sum has a fixed order:
//
// cross_dq_kernel: persistent, one CTA per SM; a unit is 128 query rows of one head, walked over the keys in blocks of
// 128, dQ accumulating in TMEM (128 columns).  S is double buffered (256 columns), so the next block's S runs under this
// block's exponentials; dP (128 columns) is freed when the threads have read it, so its next product runs before dQ's.
// dS overwrites S.  Two threads per row, 64 keys each: nothing passes between them (no maximum here) but delta's halves.
// Where there are few units the keys are split and cross_grad_sum_kernel adds the parts' float32 dQ in order.
// delta comes from the rows of dO and out while the unit's first weights are formed; (lse, delta) are left for the second
// pass.  The K / V ring runs on into the next unit, and its Q and dO follow as soon as the last products have read these.
//
// cross_dkv_kernel: a CTA owns 128 keys of one key head (rows of S^T = K Q^T and dP^T = V dO^T) and a range of the
// query blocks of 64 of every head that shares it; dK and dV accumulate in TMEM (256 columns), S^T and dP^T are double
// buffered beside them, and two softmax warpgroups take alternate steps, so a step's exponentials run under the
// neighbouring steps' products.  P^T and dS^T never leave TMEM: they are the A operands of the products with dO and Q.
// Where the key blocks alone do not fill the device evenly, the query range is split and the float32 partial sums are
// added by cross_grad_sum_kernel in order.
//
// Measured: 16,384 queries x 512 keys x 24 heads of 128, bfloat16, device time of 20 passes: 376 us after a second's rest, 435
// once the power cap holds the SM clock (1,635 MHz), of which the dQ pass a little over half; the chain
// S, dP -> threads -> dS -> product bounds both (tensor pipe 39 % and 60 % busy).
//
// Rounding: P and dS enter their products in the operands' 16-bit type (a relative 2^-9 for bfloat16, about what the
// result's own rounding adds; carrying the rest would take a second product each), the gradients are rounded once from
// float32.
//
// With an added mask lse is no full account of a row's sum: float32 near a mask of -1e9 is spaced 64 apart, so the log of
// the sum is lost in it (a row of 256 such keys: exp(x - lse) = 1 for each instead of 1 / 256), and from -1e4 on it costs
// more than the gradients' rounding.  x - lse itself is exact there.  So the first pass adds the row's weights up as lse
// gives them, divides dQ by the sum, and leaves its log2 for the second pass.  (They are at most 1: lse, the rounding
// of something no less than the row's maximum, is no less than that either.)
//
// float16 has no room below: with an upstream gradient of 1e-5 dS would be among its subnormals, and so are the weights of
// many keys.  There P enters its product times 2^12 and dS times 2^t, both taken out of the float32 results.  t goes by
// |dS| <= 2 max|dP| + max|dlse| <= 2 dim max|dO| max|v| + max|dlse|, of a tile of rows in the first pass and of all rows
// that share a key head in the second: 2^t times that stays below 2^15, half of what float16 holds.  It only ever
// enlarges.  cross_vmax_kernel finds max|v| ahead; the first pass has dO at hand.  (4,096 x 512 x 2 heads of 128, upstream
// 1e-5: dK's relative error 0.0017, the rounding of the result itself, in place of 0.0157.  In a row, 16,384 x 512 x 24
// heads 425 -> 440 us, 3 x 777 x 130 x 12 heads 42.9 -> 44.7.)
#include <algorithm>
#include <cmath>

#include "cross.cuh"

namespace htrc {

namespace {

// With a bool mask per query the first pass leaves its ballots for the second: word w of a row holds keys 32 w .. (set:
// kept), laid out [entry][head (one where the mask has none)][word][padded row], words padded to the second pass's blocks
struct CrossBits {
  uint32_t* p;
  int words;
  bool heads;
  __device__ __forceinline__ int64_t at(const CrossShape& s, int64_t rows, int b, int h, int word) const {
    return ((static_cast<int64_t>(b) * (heads ? s.heads : 1) + (heads ? h : 0)) * words + word) * rows;
  }
};

// ------------------------------------------------------------------------------------------------ float16's room
constexpr int kVmaxParts = 32;        // CTAs per entry and key head, at most
template <bool BF>
__host__ __device__ constexpr float p_room() { return BF ? 0.f : 12.f; }     // P enters its product times 2^this
__device__ __forceinline__ float two_to(int t) { return __int_as_float((127 + t) << 23); }
// t for a bound on |dS|: bound < 2^(e + 1)
__device__ __forceinline__ int room(float bound) {
  const int e = static_cast<int>(__float_as_uint(bound) >> 23) - 127;
  return max(0, min(40, 14 - e));
}
// two float16 magnitudes of each word, those that are not finite as 0 (they make the results they reach not finite
// whatever t is)
__device__ __forceinline__ uint32_t magnitudes(uint32_t x) {
  x &= 0x7fff7fffu;
  return x & ~__vcmpgeu2(x, 0x7c007c00u);
}
__device__ __forceinline__ uint32_t most(uint32_t to, const uint4& x) {
  return __vmaxu2(__vmaxu2(to, __vmaxu2(magnitudes(x.x), magnitudes(x.y))), __vmaxu2(magnitudes(x.z), magnitudes(x.w)));
}
// the larger of two float16 magnitudes, as the bits of a float32 (which compare as they do)
__device__ __forceinline__ uint32_t wide(uint32_t x) {
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(max(x & 0xffffu, x >> 16)))));
}

struct VmaxParams {
  CrossShape s;
  const uint16_t* v;
  int64_t vs[3];
  uint32_t* vmax;             // [batch * kv_heads][parts], float32 bits
  int parts;
};

// max|v| of the keys that a query may see; 8 or 16 lanes per row
template <int DP, bool KEYED>
__global__ void __launch_bounds__(256) cross_vmax_kernel(const __grid_constant__ VmaxParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");          // the dQ pass waits for this kernel's end itself
  constexpr int LPR = DP / 8, RPC = 256 / LPR;
  __shared__ uint32_t part[8];
  const int bk = blockIdx.x / p.parts, first = (blockIdx.x - bk * p.parts) * RPC + threadIdx.x / LPR, step = p.parts * RPC;
  const int b = bk / p.s.kv_heads, hk = bk - b * p.s.kv_heads, e = threadIdx.x % LPR * 8;
  const int count = key_count(p.s, b);
  const uint16_t* src = p.v + b * p.vs[0] + hk * p.vs[2] + e;
  uint32_t m = 0;
#pragma unroll 4
  for (int64_t key = first; key < count; key += step) {
    const uint4 x = e < p.s.dim ? __ldg(reinterpret_cast<const uint4*>(src + key * p.vs[1])) : make_uint4(0, 0, 0, 0);
    bool seen = !KEYED;
    if (KEYED)
      for (int g = 0; g < (p.s.mask.sh != 0 ? p.s.group : 1) && !seen; ++g)
        seen = mask_term(p.s.mask.p, p.s.mask.dtype, b * p.s.mask.sb + (hk * p.s.group + g) * p.s.mask.sh + key * p.s.mask.sm) != -INFINITY;
    if (seen) m = most(m, x);
  }
  m = __reduce_max_sync(0xffffffffu, wide(m));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) m = max(m, part[w]);
    p.vmax[blockIdx.x] = m;
  }
}

// ------------------------------------------------------------------------------------------------ dQ
constexpr int kDqThreads = 320;
constexpr int kDqRows = 128, kDqKeys = 128;
constexpr uint32_t kDqColS = 0, kDqColP = 256, kDqColQ = 384, kDqCols = 512;      // S: two buffers

struct DqBars {
  uint64_t q_full, q_empty, do_full, do_empty, kv_full[5], kv_empty[5], s_full[2], ds_full[2], dp_full, dp_read, dq_full, idle;
  uint32_t tmem_base;
  int abort_flag, loads[3];           // of the TMA warp in all: K / V, Q, dO
};

template <int DP>
struct DqSmem {
  // five slots: with four, a block's K waited for the K two blocks before it to leave, a step later
  static constexpr int kChunks = DP / 64, kSlots = 5;
  static constexpr uint32_t kChunk = 128 * 128, kTile = kChunks * kChunk;
  static constexpr uint32_t kQ = 0, kDo = kTile, kKV = 2 * kTile, kBias = kKV + kSlots * kTile;
  static constexpr uint32_t kDelta = kBias + 2 * kDqKeys * 4, kMax = kDelta + 2 * kDqRows * 4, kBars = kMax + 64, kBytes = kBars + 224;
  static_assert(sizeof(DqBars) <= 224 && kBytes <= 232448, "shared memory of one CTA");
};

struct DqParams {
  CrossShape s;
  const float* lse;
  const float* dlse;
  const uint16_t* out;
  int64_t out_stride[3];
  uint16_t* dq;
  int64_t dq_stride[3];
  // [batch * heads][padded rows / 64][3][64]: minus lse in the pass's units, log2 of the weights' sum by it, delta.  (p_room
  // is in the second with an added mask, else in the first)
  float* stat;
  int64_t stat_rows;
  CrossBits bits;
  const uint32_t* vmax;     // float16: [batch * kv_heads][vmax_parts]
  float* bounds;            // float16, left for the second pass: the bound on |dS| of each tile [batch * heads][tiles]
  int vmax_parts;
  uint32_t units, tiles;    // tiles of 128 rows per head
  int splits;               // parts of the keys
  float* part;              // splits > 1: [split][batch * heads][queries][DP], not divided by the weights' sums
  float* part_sum;          // with an added mask: [split][batch * heads][queries]
  int do_b, do_h;
  int* status;
};

// A CTA's units, and within one its blocks of keys.  SPLIT: its part of them (a kernel of its own: with both in one, the
// unsplit pass lost 6 to 16 %)
template <bool SPLIT>
struct DqWalk {
  uint32_t unit;
  int b, h, row0, split, count, j, j0, j1;
  __device__ __forceinline__ void open(const DqParams& p, uint32_t u) {
    unit = u;
    if (u >= p.units) return;
    const uint32_t rest = u / p.tiles;
    uint32_t bh = rest;
    split = 0;
    if (SPLIT) {
      bh = rest / p.splits;
      split = static_cast<int>(rest - bh * p.splits);
    }
    b = static_cast<int>(bh / static_cast<uint32_t>(p.s.heads));
    h = static_cast<int>(bh - b * static_cast<uint32_t>(p.s.heads));
    row0 = static_cast<int>(u - rest * p.tiles) * kDqRows;
    count = key_count(p.s, b);
    j1 = (count + kDqKeys - 1) / kDqKeys;
    if (SPLIT) {
      const int64_t nb = j1;
      j0 = static_cast<int>(nb * split / p.splits);
      j1 = static_cast<int>(nb * (split + 1) / p.splits);
    }
    j = from();
  }
  // the part that leaves the rows' statistics: the last, which has a block wherever the entry has a key
  __device__ __forceinline__ bool leaves_stat(const DqParams& p) const { return !SPLIT || split == p.splits - 1; }
  __device__ __forceinline__ int from() const { return SPLIT ? j0 : 0; }
  __device__ __forceinline__ bool done(const DqParams& p) const { return unit >= p.units; }
  // the first unit from u on that has a block
  __device__ __forceinline__ void open_live(const DqParams& p, uint32_t u) {
    for (open(p, u); !done(p) && j >= j1;) open(p, unit + gridDim.x);
  }
  __device__ __forceinline__ void next(const DqParams& p) {
    if (++j >= j1) open_live(p, unit + gridDim.x);
  }
};

template <int DP, bool BF, int KIND, bool SPLIT>
__global__ void __launch_bounds__(kDqThreads, 1)
    cross_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                    const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ DqParams p) {
  using SM = DqSmem<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023) {          // the swizzled tiles need it; there is no room to round up
    flag_status(p.status, ST_WAIT_TIMEOUT);
    return;
  }
  DqBars* bars = reinterpret_cast<DqBars*>(smem + SM::kBars);
  volatile int* abort_flag = &bars->abort_flag;
  int* status = p.status;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->q_empty, 1);
    mbar_init(&bars->do_full, 1);
    mbar_init(&bars->do_empty, 1 + 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->ds_full[i], 256);
    }
    mbar_init(&bars->idle, 1);
    for (int i = 0; i < SM::kSlots; ++i) {
      mbar_init(&bars->kv_full[i], 1);
      mbar_init(&bars->kv_empty[i], 1);
    }
    mbar_init(&bars->dp_full, 1);
    mbar_init(&bars->dp_read, 256);
    mbar_init(&bars->dq_full, 1);
    bars->abort_flag = bars->loads[0] = bars->loads[1] = bars->loads[2] = 0;
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(&bars->tmem_base, kDqCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  DqWalk<SPLIT> w{};

  if (warp == 8) {
    // ------------------------------------------------------------------ TMA: ring slots K, V, K, V, ...
    const uint64_t pol_q = policy_evict_first(), pol_kv = policy_evict_last();
    const uint32_t leader = elect_one();
    int slots = 0, units = 0, q_loads = 0, do_loads = 0;
    auto load = [&](int j, int kv) -> bool {
      const int s = slots % SM::kSlots, hk = w.h / p.s.group;
      if (slots >= SM::kSlots && !mbar_wait_warp(&bars->kv_empty[s], ((slots / SM::kSlots) - 1) & 1, status, abort_flag))
        return false;
      if (leader) {
        mbar_arrive_expect_tx(&bars->kv_full[s], SM::kTile);
        for (int c = 0; c < SM::kChunks; ++c)
          tma_load_4d(smem + SM::kKV + s * SM::kTile + c * SM::kChunk, kv ? &tm_v : &tm_k, &bars->kv_full[s], 64 * c,
                      j * kDqKeys, hk * (kv ? p.s.v_h : p.s.k_h), w.b * (kv ? p.s.v_b : p.s.k_b), pol_kv);
      }
      __syncwarp();
      ++slots;
      return true;
    };
    bool ok = true;
    auto rows = [&](const CUtensorMap* map, uint32_t at, uint64_t* full, uint64_t* empty, int in_h, int in_b, int& loads) -> bool {
      if (units > 0 && !mbar_wait_warp(empty, (units - 1) & 1, status, abort_flag)) return false;
      if (leader) {
        mbar_arrive_expect_tx(full, SM::kTile);
        for (int c = 0; c < SM::kChunks; ++c)
          tma_load_4d(smem + at + c * SM::kChunk, map, full, 64 * c, w.row0, w.h * in_h, w.b * in_b, pol_q);
      }
      __syncwarp();
      ++loads;
      return true;
    };
    for (w.open_live(p, blockIdx.x); ok && !w.done(p); w.open_live(p, w.unit + gridDim.x), ++units) {
      ok = load(w.j, 0) && rows(&tm_q, SM::kQ, &bars->q_full, &bars->q_empty, p.s.q_h, p.s.q_b, q_loads) &&
           rows(&tm_do, SM::kDo, &bars->do_full, &bars->do_empty, p.do_h, p.do_b, do_loads) && load(w.j, 1);
      for (int j = w.j + 1; ok && j < w.j1; ++j) ok = load(j, 0) && load(j, 1);
    }
    if (ok && units > 0) {                // the last releases have landed before the CTA leaves
      mbar_wait_warp(&bars->q_empty, (units - 1) & 1, status, abort_flag);
      mbar_wait_warp(&bars->do_empty, (units - 1) & 1, status, abort_flag);
    }
    if (ok) drain_ring<true>(bars->kv_empty, SM::kSlots, slots, status, abort_flag);   // before the CTA leaves
    if (lane == 0) {
      bars->loads[0] = slots;
      bars->loads[1] = q_loads;
      bars->loads[2] = do_loads;
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------ MMA
    const uint32_t leader = elect_one();
    const uint32_t id_s = idesc16<BF>(128, kDqKeys, false, false);
    const uint32_t id_q = idesc16<BF>(128, DP, false, true);
    const uint64_t dq = desc_k(smem_u32(smem + SM::kQ)), ddo = desc_k(smem_u32(smem + SM::kDo));
    const uint64_t ring_k = desc_k(smem_u32(smem + SM::kKV)), ring_n = desc_mn(smem_u32(smem + SM::kKV), SM::kChunk);
    DqWalk<SPLIT> a;                           // the step whose S and dP are next
    a.open_live(p, blockIdx.x);
    int ahead = 0, units = 0;
    // excluded keys may hold anything: their rows of K (0 * NaN in dS K) and V become zeros
    auto slot = [&](int at) -> int {
      const int s = at % SM::kSlots;
      if (!mbar_wait_warp(&bars->kv_full[s], (at / SM::kSlots) & 1, status, abort_flag)) return -1;
      if (KIND == CROSS_KEYS || (a.count < p.s.keys && (a.j + 1) * kDqKeys > a.count))
        zero_excluded_rows<kDqKeys, SM::kChunks>(smem + SM::kKV + s * SM::kTile, SM::kChunk, a.j * kDqKeys, a.count, p.s,
                                                 a.b * p.s.mask.sb + a.h * p.s.mask.sh, KIND == CROSS_KEYS, lane);
      return s;
    };
    auto product = [&](uint32_t d, uint64_t rows, int s) {
      tc_fence_after();
      const uint64_t so = (s * SM::kTile) >> 4;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const uint32_t o = ((kk / 4) * SM::kChunk + (kk % 4) * 32) >> 4;
        mma_bf16_by(leader, d, rows + o, ring_k + so + o, id_s, kk != 0);
      }
    };
    auto scores = [&]() -> bool {         // S of a's step
      if (a.j == a.from() && !mbar_wait_warp(&bars->q_full, units & 1, status, abort_flag)) return false;
      const int s = slot(2 * ahead);
      if (s < 0) return false;
      product(tmem + kDqColS + 128 * (ahead & 1), dq, s);
      mma_commit_by(leader, &bars->s_full[ahead & 1]);
      if (a.j + 1 == a.j1) mma_commit_by(leader, &bars->q_empty);
      return true;
    };
    auto gradients = [&]() -> bool {      // dP of the same step, which it ends
      if (a.j == a.from() && !mbar_wait_warp(&bars->do_full, units & 1, status, abort_flag)) return false;
      const int s = slot(2 * ahead + 1);
      if (s < 0) return false;
      product(tmem + kDqColP, ddo, s);
      mma_commit_by(leader, &bars->dp_full);
      mma_commit_by(leader, &bars->kv_empty[s]);
      if (a.j + 1 == a.j1) {
        mma_commit_by(leader, &bars->do_empty);
        ++units;
      }
      ++ahead;
      a.next(p);
      return true;
    };
    bool ok = true, first = true;
    if (!a.done(p)) ok = scores() && gradients();
    int n = 0;
    for (w.open_live(p, blockIdx.x); ok && !w.done(p); ++n) {
      const int s = (2 * n) % SM::kSlots;
      const bool last = w.j + 1 == w.j1;
      // the unit's next S and dP go before this dQ; the next unit's, whose rows come later, behind it
      if (!last) ok = scores() && mbar_wait_warp(&bars->dp_read, n & 1, status, abort_flag) && gradients();
      // (two barriers: the threads may finish the next step before this wait)
      ok = ok && mbar_wait_warp(&bars->ds_full[n & 1], (n >> 1) & 1, status, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint64_t ko = (s * SM::kTile) >> 4;
      const uint32_t ds = tmem + kDqColS + 128 * (n & 1);        // keys 0-63 in columns 0-31, 64-127 in 64-95
#pragma unroll
      for (int kk = 0; kk < kDqKeys / 16; ++kk)
        mma_bf16_ts_by(leader, tmem + kDqColQ, ds + (kk / 4) * 64 + (kk % 4) * 8, ring_n + ko + ((kk * 2048) >> 4), id_q,
                       !first || kk != 0);
      mma_commit_by(leader, &bars->kv_empty[s]);
      if (last) mma_commit_by(leader, &bars->dq_full);
      if (last && !a.done(p)) ok = scores() && mbar_wait_warp(&bars->dp_read, n & 1, status, abort_flag) && gradients();
      first = last;
      w.next(p);
    }
  } else {
    // ------------------------------------------------------------------ two threads per row, 64 keys (columns) each
    const int half = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane, key0 = 64 * half;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const float scale2 = p.s.scale * kCrossLog2e;
    constexpr bool NAT = KIND == CROSS_KEYS || KIND == CROSS_BIAS;
    float* bias = reinterpret_cast<float*>(smem + SM::kBias);
    float* delta_s = reinterpret_cast<float*>(smem + SM::kDelta);
    uint2* max_s = reinterpret_cast<uint2*>(smem + SM::kMax);
    bool ok = true;
    int n = 0, units = 0;
    // the row's lse and its gradient: loaded a unit ahead, as this half's columns of out into L2 (float16: and vmax's parts,
    // once the first unit with a block has waited for cross_vmax_kernel)
    float lse, dlse;
    uint32_t vmax = 0;
    auto ask_vmax = [&]() {
      if (lane < p.vmax_parts) vmax = p.vmax[(static_cast<int64_t>(w.b) * p.s.kv_heads + w.h / p.s.group) * p.vmax_parts + lane];
    };
    auto out_row = [&]() {
      return p.out + w.b * p.out_stride[0] + static_cast<int64_t>(w.row0 + r) * p.out_stride[1] + w.h * p.out_stride[2] + half * (DP / 2);
    };
    auto ask = [&](bool waited) {
      const int row = w.row0 + r;
      const bool valid = !w.done(p) && row < p.s.queries;
      const int64_t at = (static_cast<int64_t>(w.b) * p.s.heads + w.h) * p.s.queries + row;
      lse = -INFINITY;
      dlse = 0.f;
      if (valid) {
        lse = __ldg(p.lse + at);
        if (p.dlse != nullptr) dlse = __ldg(p.dlse + at);
        if (half * (DP / 2) < p.s.dim) asm volatile("prefetch.global.L2 [%0];" ::"l"(out_row()));
      }
      if (!BF && waited && !w.done(p)) ask_vmax();
    };
    w.open(p, blockIdx.x);
    ask(false);
    while (ok && !w.done(p)) {
      const int row = w.row0 + r;
      const bool valid = row < p.s.queries, live = w.from() < w.j1;
      const int64_t bh = static_cast<int64_t>(w.b) * p.s.heads + w.h;
      const int64_t mask_at = w.b * p.s.mask.sb + w.h * p.s.mask.sh;
      const int64_t row_mask = mask_at + (valid ? row : 0) * p.s.mask.sn;
      float delta = 0.f, shift = 0.f;         // shift: t, once it is known
      float2 sum = make_float2(0.f, 0.f);
      if (lse == -INFINITY) lse = INFINITY;     // a row with nothing in it (or none): every weight exp2(-inf)
      if (!NAT) lse *= kCrossLog2e;
      for (int j = w.from(); j < w.j1; ++j, ++n) {
        const int first = j * kDqKeys + key0, left = w.count - first;      // this thread's keys of the block
        uint32_t bits[2] = {0u, 0u};
        float* bj = bias + (n & 1) * kDqKeys + key0;
        if (KIND == CROSS_KEYS) {
          if (r < 64)
            bj[r] = r < left ? mask_term(p.s.mask.p, p.s.mask.dtype, mask_at + static_cast<int64_t>(first + r) * p.s.mask.sm) : -INFINITY;
          named_bar_sync(1 + half, 128);
        }
        if ((KIND == CROSS_PAIRS || KIND == CROSS_BIAS) && valid && left > kDqKeys)     // the next block's terms of this row
          prefetch_mask(p.s.mask, row_mask + static_cast<int64_t>(first + kDqKeys) * p.s.mask.sm);
        if (KIND == CROSS_PAIRS) {
          // the warp's 32 rows of mask bits: a row's 64 keys by coalesced loads, sixteen rows in flight, and ballots
          const int rows = min(32, static_cast<int>(p.s.queries) - (w.row0 + quarter * 32));
          const uint8_t* mk = static_cast<const uint8_t*>(p.s.mask.p) + mask_at +
                              static_cast<int64_t>(w.row0 + quarter * 32) * p.s.mask.sn + static_cast<int64_t>(first + lane) * p.s.mask.sm;
          for (int g = 0; g < rows; g += 16) {
            uint8_t v[16][2];
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
              for (int q = 0; q < 2; ++q)
                v[i][q] = g + i < rows && 32 * q + lane < left ? __ldg(mk + i * p.s.mask.sn + 32 * q * p.s.mask.sm) : 0;
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const uint32_t word = __ballot_sync(0xffffffffu, v[i][q] != 0);
                if (lane == g + i) bits[q] = word;
              }
            mk += 16 * p.s.mask.sn;
          }
          if (p.bits.heads || w.h == 0) {
#pragma unroll
            for (int q = 0; q < 2; ++q) p.bits.p[p.bits.at(p.s, p.stat_rows, w.b, w.h, first / 32 + q) + row] = bits[q];
          }
        }
        // this half's columns of out, asked for before the unit's first weights are formed
        uint4 o[DP / 16];
        if (j == w.from()) {
          const uint16_t* src = out_row();
#pragma unroll
          for (int c = 0; c < DP / 16; ++c) {
            o[c] = make_uint4(0, 0, 0, 0);
            if (valid && half * (DP / 2) + 8 * c < p.s.dim) o[c] = __ldg(reinterpret_cast<const uint4*>(src + 8 * c));
          }
        }
        const uint32_t col_s = tmem + lanes + kDqColS + 128 * (n & 1) + key0, col_p = tmem + lanes + kDqColP + key0;
        if (!mbar_wait_warp(&bars->s_full[n & 1], (n >> 1) & 1, status, abort_flag)) { ok = false; break; }
        tc_fence_after();
        float2 e[32];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t s[32];
          tmem_ld32(col_s + 32 * c, s);
          tmem_ld_wait();
          if (KIND == CROSS_NONE) {
            if (left < 64) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (32 * c + i >= left) s[i] = __float_as_uint(-INFINITY);
            }
          } else if (KIND == CROSS_PAIRS) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(bits[c] >> i & 1u)) s[i] = __float_as_uint(-INFINITY);
          } else {
            float t[32];
            if (KIND == CROSS_KEYS) {
#pragma unroll
              for (int i = 0; i < 32; ++i) t[i] = bj[32 * c + i];
            } else {
              mask_terms<32>(p.s.mask.p, p.s.mask.dtype, row_mask + static_cast<int64_t>(first + 32 * c) * p.s.mask.sm, p.s.mask.sm,
                             left - 32 * c, t);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i)
              s[i] = __float_as_uint(t[i] == -INFINITY ? t[i] : fmaf(__uint_as_float(s[i]), p.s.scale, t[i]));
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float2 x = make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
            if (NAT)
              x = BF ? mul2(sub2(x, make_float2(lse, lse)), make_float2(kCrossLog2e, kCrossLog2e))
                     : fma2(sub2(x, make_float2(lse, lse)), make_float2(kCrossLog2e, kCrossLog2e), make_float2(shift, shift));
            else
              x = fma2(x, make_float2(scale2, scale2), make_float2(-lse, -lse));
            x = make_float2(cross_ex2(x.x), cross_ex2(x.y));
            if (NAT) sum = add2(sum, x);
            e[16 * c + i / 2] = x;
          }
        }
        if (j == w.from()) {
          if (!BF && units == 0) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            ask_vmax();
          }
          // delta: each half of the row's columns, then both
          ok = mbar_wait_warp(&bars->do_full, units & 1, status, abort_flag);
          if (!ok) break;
          float2 acc = make_float2(0.f, 0.f);
          __half2 top = __float2half2_rn(0.f);
#pragma unroll
          for (int c = 0; c < DP / 16; ++c) {
            const int piece = half * (DP / 16) + c;
            const uint4 y = *reinterpret_cast<const uint4*>(smem + SM::kDo + (piece / 8) * SM::kChunk + sw128_off(r, piece & 7));
            acc = fma2(unpack16x2<BF>(o[c].x), unpack16x2<BF>(y.x), acc);
            acc = fma2(unpack16x2<BF>(o[c].y), unpack16x2<BF>(y.y), acc);
            acc = fma2(unpack16x2<BF>(o[c].z), unpack16x2<BF>(y.z), acc);
            acc = fma2(unpack16x2<BF>(o[c].w), unpack16x2<BF>(y.w), acc);
            if (!BF) {
              // (a gradient that is not finite: NaN is passed over, an infinity makes t 0)
              const uint32_t words[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) top = __hmax2(top, __habs2(*reinterpret_cast<const __half2*>(&words[i])));
            }
          }
          delta_s[half * kDqRows + r] = acc.x + acc.y;
          if (!BF) {
            // max|dO| and max|dlse| of the warp's rows that see a key
            const uint32_t z = __float_as_uint(dlse) & 0x7fffffffu;
            const uint32_t most_do = __reduce_max_sync(0xffffffffu, lse == INFINITY ? 0u : wide(*reinterpret_cast<const uint32_t*>(&top)));
            const uint32_t most_z = __reduce_max_sync(0xffffffffu, lse == INFINITY || z >= 0x7f800000u ? 0u : z);
            if (lane == 0) max_s[warp] = make_uint2(most_do, most_z);
          }
          fence_proxy_async_smem();           // generic reads of rows that TMA refills
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->do_empty);
          named_bar_sync(3, 256);
          delta = delta_s[r] + delta_s[kDqRows + r] - dlse;
          if (lse == INFINITY) delta = 0.f;
          if (half == 0 && w.leaves_stat(p)) {
            float* stat = p.stat + (bh * p.stat_rows + row / 64 * 64) * 3 + row % 64;
            stat[0] = NAT ? -lse : p_room<BF>() - lse;
            if (!NAT || SPLIT) stat[64] = NAT ? -p_room<BF>() : 0.f;
            stat[128] = delta;
          }
          if (!BF) {
            uint2 m = max_s[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) m = make_uint2(max(m.x, max_s[i].x), max(m.y, max_s[i].y));
            const float bound = 2.f * p.s.dim * __uint_as_float(m.x) * __uint_as_float(__reduce_max_sync(0xffffffffu, vmax)) + __uint_as_float(m.y);
            if (threadIdx.x == 0 && w.leaves_stat(p)) p.bounds[bh * p.tiles + w.row0 / kDqRows] = bound;
            // the weights of this first block are there already
            const int t = room(bound);
            shift = static_cast<float>(t);
            const float2 up = make_float2(two_to(t), two_to(t));
#pragma unroll
            for (int i = 0; i < 32; ++i) e[i] = mul2(e[i], up);
            sum = mul2(sum, up);
            if (!NAT) lse -= shift;
          }
        }
        if (!mbar_wait_warp(&bars->dp_full, n & 1, status, abort_flag)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t g[32], x[16];
          tmem_ld32(col_p + 32 * c, g);
          tmem_ld_wait();
          if (c == 1) {
            tc_fence_before();
            mbar_arrive(&bars->dp_read);
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 d = mul2(e[16 * c + i / 2], sub2(make_float2(__uint_as_float(g[i]), __uint_as_float(g[i + 1])), make_float2(delta, delta)));
            x[i / 2] = pack16x2<BF>(d.x, d.y);
          }
          tmem_st16(col_s + 16 * c, x);       // dS over columns of S this thread has read
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bars->ds_full[n & 1]);
      }
      if (!ok) break;
      if (!live) {
        // no keys at all, or none for this part: zeros
        if (half == 0) {
          if (w.leaves_stat(p)) {
            float* stat = p.stat + (bh * p.stat_rows + row / 64 * 64) * 3 + row % 64;
            stat[0] = -lse;
            stat[64] = 0.f;
            stat[128] = 0.f;
          }
          if (SPLIT && valid) {
            float* dst = p.part + ((w.split * p.s.batch * p.s.heads + bh) * p.s.queries + row) * DP;
            for (int c = 0; c < DP; c += 4) *reinterpret_cast<float4*>(dst + c) = make_float4(0.f, 0.f, 0.f, 0.f);
            if (NAT) p.part_sum[(w.split * p.s.batch * p.s.heads + bh) * p.s.queries + row] = 0.f;
          } else if (valid) {
            uint16_t* dst = p.dq + w.b * p.dq_stride[0] + row * p.dq_stride[1] + w.h * p.dq_stride[2];
            for (int c = 0; c < p.s.dim; c += 8) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0, 0, 0, 0);
          }
        }
        w.open(p, w.unit + gridDim.x);
        ask(units > 0);
        continue;
      }
      uint16_t* const dst0 = p.dq + w.b * p.dq_stride[0] + static_cast<int64_t>(w.row0 + quarter * 32) * p.dq_stride[1] +
                             w.h * p.dq_stride[2] + half * (DP / 2);
      float* const part = SPLIT ? p.part + ((w.split * p.s.batch * p.s.heads + bh) * p.s.queries + row) * DP + half * (DP / 2) : nullptr;
      const int rows = static_cast<int>(p.s.queries) - (w.row0 + quarter * 32);
      const int64_t sum_at = SPLIT ? (w.split * p.s.batch * p.s.heads + bh) * p.s.queries + row : 0;
      float* const stat = p.stat + (bh * p.stat_rows + row / 64 * 64) * 3 + row % 64;
      w.open(p, w.unit + gridDim.x);
      ask(true);
      ok = mbar_wait_warp(&bars->dq_full, units & 1, status, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const float down = BF ? 1.f : two_to(-static_cast<int>(shift));
      float mul = p.s.scale * down;
      if (NAT) {
        // the weights' sum, of both halves of the row: by way of delta_s, which every thread has read before its last dS
        delta_s[half * kDqRows + r] = sum.x + sum.y;
        named_bar_sync(3, 256);
        const float total = delta_s[r] + delta_s[kDqRows + r];
        named_bar_sync(3, 256);               // before the next unit's delta is written there
        if constexpr (SPLIT) {
          if (half == 0 && valid) p.part_sum[sum_at] = total * down;
        } else {
          // (none: a row with nothing in it, whose dQ is zero)
          if (half == 0) stat[64] = total == 0.f ? 0.f : log2f(total) - shift - p_room<BF>();
          if (total != 0.f) mul = p.s.scale / total;
        }
      }
      if constexpr (SPLIT) {
#pragma unroll 1
        for (int c = 0; c < DP / 64; ++c) {
          uint32_t a[32];
          tmem_ld32(tmem + lanes + kDqColQ + half * (DP / 2) + 32 * c, a);
          tmem_ld_wait();
          if (valid) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(part + 32 * c + i) =
                  make_float4(__uint_as_float(a[i]) * mul, __uint_as_float(a[i + 1]) * mul, __uint_as_float(a[i + 2]) * mul,
                              __uint_as_float(a[i + 3]) * mul);
          }
        }
        tc_fence_before();
        ++units;
        continue;
      }
      constexpr int PIECES = DP / 16;
      uint32_t x[PIECES][4];
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        uint32_t a[32];
        tmem_ld32(tmem + lanes + kDqColQ + half * (DP / 2) + 32 * c, a);
        tmem_ld_wait();
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x[4 * c + g][i] = pack16x2<BF>(__uint_as_float(a[8 * g + 2 * i]) * mul, __uint_as_float(a[8 * g + 2 * i + 1]) * mul);
      }
      tc_fence_before();
      exchange_pieces<PIECES>(x, lane);
      const int piece = lane % PIECES, row8 = lane / PIECES * PIECES;
      if (half * (DP / 2) + 8 * piece < p.s.dim) {
#pragma unroll
        for (int g = 0; g < PIECES; ++g)
          if (row8 + g < rows)
            *reinterpret_cast<uint4*>(dst0 + (row8 + g) * p.dq_stride[1] + 8 * piece) = make_uint4(x[g][0], x[g][1], x[g][2], x[g][3]);
      }
      ++units;
    }
    if (!BF && units == 0) asm volatile("griddepcontrol.wait;" ::: "memory");        // this kernel's end is that one's too
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (warp == 8) {
      settle_loads(bars->kv_full, SM::kSlots, bars->loads[0], status);
      settle_loads(&bars->q_full, 1, bars->loads[1], status);
      settle_loads(&bars->do_full, 1, bars->loads[2], status);
    } else if (warp == 9) {
      settle_products(&bars->idle, status);
    }
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, kDqCols);
}

// ------------------------------------------------------------------------------------------------ dK, dV
constexpr int kDkvThreads = 320;
constexpr int kDkvKeys = 128, kDkvRows = 64, kDkvStages = 4;
constexpr uint32_t kDkvColK = 0, kDkvColV = 128, kDkvColS = 256, kDkvBuf = 128, kDkvCols = 512;

struct DkvBars {
  uint64_t kv_full, full[kDkvStages], empty[kDkvStages], s_full[2], dp_full[2], p_full[2], ds_full[2], acc_full, idle;
  uint32_t tmem_base;
  int abort_flag, loads;              // of the TMA warp in all: stages
};

template <int DP>
struct DkvSmem {
  static constexpr int kChunks = DP / 64;
  static constexpr uint32_t kKeyChunk = 128 * 128, kRowChunk = 64 * 128;
  static constexpr uint32_t kTile = kChunks * kKeyChunk, kRows = kChunks * kRowChunk;
  static constexpr uint32_t kK = 0, kV = kTile, kRing = 2 * kTile, kStat = kDkvRows * 3 * 4,
                            kBits = 2 * kRows + 1024, kStage = kBits + 1024;      // rows, statistics, 4 words of bits per row
  static constexpr uint32_t kBars = kRing + kDkvStages * kStage;
  static constexpr uint32_t kUsed = kBars + 256 + 1024;
  // one CTA per SM: it takes all 512 TMEM columns
  static constexpr uint32_t kBytes = kUsed < 120 * 1024 ? 120 * 1024 : kUsed;
};

struct DkvParams {
  CrossShape s;
  const float* stat;
  int64_t stat_rows;
  CrossBits bits;
  const float* bounds;      // float16: [batch * heads][tiles]
  int tiles;
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
    mbar_init(&bars->idle, 1);
    bars->abort_flag = bars->loads = 0;
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
        mbar_arrive_expect_tx(&bars->full[s], 2 * SM::kRows + SM::kStat + (KIND == CROSS_PAIRS ? 4 * kDkvRows * 4 : 0));
        for (int c = 0; c < SM::kChunks; ++c) {
          tma_load_4d(st + c * SM::kRowChunk, &tm_q, &bars->full[s], 64 * c, row, h * p.s.q_h, b * p.s.q_b, pol);
          tma_load_4d(st + SM::kRows + c * SM::kRowChunk, &tm_do, &bars->full[s], 64 * c, row, h * do_h, b * do_b, pol);
        }
        bulk_load(st + 2 * SM::kRows, p.stat + ((static_cast<int64_t>(b) * p.s.heads + h) * p.stat_rows + row) * 3, SM::kStat,
                  &bars->full[s], pol);
        if (KIND == CROSS_PAIRS)
          for (int q = 0; q < 4; ++q)
            bulk_load(st + SM::kBits + q * kDkvRows * 4, p.bits.p + p.bits.at(p.s, p.stat_rows, b, h, key0 / 32 + q) + row,
                      kDkvRows * 4, &bars->full[s], pol);
      }
      __syncwarp();
    }
    if (i == steps) drain_ring<true>(bars->empty, kDkvStages, steps, status, abort_flag);
    if (lane == 0) bars->loads = i;
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
    int t = 0;
    if (!BF && steps > 0) {
      const float* bound = p.bounds + (static_cast<int64_t>(b) * p.s.heads + hk * p.s.group) * p.tiles;
      uint32_t m = 0;
#pragma unroll 4
      for (int64_t i = lane; i < static_cast<int64_t>(p.s.group) * p.tiles; i += 32) m = max(m, __float_as_uint(__ldg(bound + i)));
      t = room(__uint_as_float(__reduce_max_sync(0xffffffffu, m)));
    }
    const float2 up = make_float2(two_to(t - static_cast<int>(p_room<BF>())), two_to(t - static_cast<int>(p_room<BF>())));
    int head = -1;
    float kbias = in ? 0.f : -INFINITY;           // with a bias: this key's term, -inf where it is excluded
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
      if (KIND == CROSS_BIAS) {
        // the terms of this warp's keys that its next step reads (lane: query)
        const int64_t then = at + 2;
        if (i + 2 < steps && key0 + quarter * 32 < count) {
          const int row2 = static_cast<int>(then % p.row_blocks) * kDkvRows + lane, h2 = hk * p.s.group + static_cast<int>(then / p.row_blocks);
          const int64_t m0 = b * p.s.mask.sb + h2 * p.s.mask.sh + static_cast<int64_t>(key0 + quarter * 32) * p.s.mask.sm;
          if (row2 < p.s.queries) prefetch_mask(p.s.mask, m0 + row2 * p.s.mask.sn);
          if (row2 + 32 < p.s.queries) prefetch_mask(p.s.mask, m0 + (row2 + 32) * p.s.mask.sn);
        }
      }
      uint32_t out[2] = {0u, 0u};           // queries this key is excluded from (of a bias: found with its terms)
      if (!mbar_wait_warp(&bars->s_full[wg], (i >> 1) & 1, status, abort_flag)) { ok = false; break; }
      tc_fence_after();
      // the queries' statistics: [-lse][log2 of the weights' sum by it][delta], 64 each
      const float* st = reinterpret_cast<const float*>(smem + SM::kRing + s * SM::kStage + 2 * SM::kRows);
      const uint32_t buf = tmem + lanes + kDkvColS + wg * kDkvBuf;
      const uint4* words = reinterpret_cast<const uint4*>(smem + SM::kRing + s * SM::kStage + SM::kBits + quarter * kDkvRows * 4);
      float2 w[32];                         // P, kept for dS
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t x[32], pw[16];
        tmem_ld32(buf + 32 * c, x);
        tmem_ld_wait();
        float terms[32];
        if (KIND == CROSS_PAIRS) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint4 x4 = words[8 * c + k];
            out[c] |= (~x4.x >> lane & 1u) << (4 * k) | (~x4.y >> lane & 1u) << (4 * k + 1) | (~x4.z >> lane & 1u) << (4 * k + 2) |
                      (~x4.w >> lane & 1u) << (4 * k + 3);
          }
        }
        if (KIND == CROSS_BIAS)
          mask_terms<32>(p.s.mask.p, p.s.mask.dtype, mask_at + (row + 32 * c) * p.s.mask.sn, p.s.mask.sn,
                         in ? static_cast<int>(p.s.queries) - row - 32 * c : 0, terms);
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 ls = *reinterpret_cast<const float4*>(st + 32 * c + k);
          const float4 ls2 = NAT ? *reinterpret_cast<const float4*>(st + 64 + 32 * c + k) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int h2 = 0; h2 < 2; ++h2) {
            const float l0 = h2 ? ls.z : ls.x, l1 = h2 ? ls.w : ls.y;
            const int kk = k + 2 * h2;
            float2 e = make_float2(__uint_as_float(x[kk]), __uint_as_float(x[kk + 1]));
            if (!NAT) {
              // (a key past the entry's count: zero rows here, its gradients are not taken in the end)
              float2 off = make_float2(l0, l1);
              if (KIND == CROSS_PAIRS) {
                if (out[c] >> kk & 1u) off.x = -INFINITY;
                if (out[c] >> kk & 2u) off.y = -INFINITY;
              }
              e = fma2(e, make_float2(scale, scale), off);
            } else {
              float b0 = kbias, b1 = kbias;
              if (KIND == CROSS_BIAS) {
                b0 = terms[kk];
                b1 = terms[kk + 1];
              }
              e = fma2(e, make_float2(scale, scale), make_float2(b0, b1));
              e = fma2(add2(e, make_float2(l0, l1)), make_float2(kCrossLog2e, kCrossLog2e),
                       h2 ? make_float2(-ls2.z, -ls2.w) : make_float2(-ls2.x, -ls2.y));
              // an excluded key's weight and gradient are zero whatever its row holds
              if (b0 == -INFINITY) {
                e.x = -INFINITY;
                out[c] |= 1u << kk;
              }
              if (b1 == -INFINITY) {
                e.y = -INFINITY;
                out[c] |= 2u << kk;
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
              if (out[c] >> kk & 1u) g.x = 0.f;
              if (out[c] >> kk & 2u) g.y = 0.f;
            }
            float2 d = mul2(w[16 * c + kk / 2], sub2(g, h2 ? make_float2(de.z, de.w) : make_float2(de.x, de.y)));
            if (!BF) d = mul2(d, up);
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
      const float mul = wg == 0 ? two_to(-static_cast<int>(p_room<BF>())) : p.s.scale * two_to(-t);
      uint8_t* stage = smem + (wg == 0 ? SM::kV : SM::kK) + quarter * 32 * 128;
      const int64_t parts = static_cast<int64_t>(p.splits) * p.s.batch * p.s.kv_heads;
      // splits > 1: this warp's 32 keys' rows
      float* dst = p.partial + (((wg == 0 ? parts : 0) + (static_cast<int64_t>(split) * p.s.batch * p.s.kv_heads + bk)) * p.s.keys +
                                key0 + quarter * 32) * DP;
      const int rows = static_cast<int>(p.s.keys) - (key0 + quarter * 32);
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
          uint32_t x[8][4];
#pragma unroll
          for (int k = 0; k < 32; ++k) x[k / 4][k % 4] = in ? __float_as_uint(__uint_as_float(o[k]) * mul) : 0u;
          exchange_pieces<8>(x, lane);
#pragma unroll
          for (int g = 0; g < 8; ++g)
            if ((lane & ~7) + g < rows)
              *reinterpret_cast<uint4*>(dst + ((lane & ~7) + g) * DP + 32 * c + 4 * (lane & 7)) = make_uint4(x[g][0], x[g][1], x[g][2], x[g][3]);
        } else {
          const uint32_t base = smem_u32(stage + (c / 2) * SM::kKeyChunk);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = in ? pack16x2<BF>(__uint_as_float(o[8 * g + 2 * k]) * mul, __uint_as_float(o[8 * g + 2 * k + 1]) * mul) : 0u;
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
  if (*abort_flag) {
    if (warp == 8) {
      settle_loads(bars->full, kDkvStages, bars->loads, status);
      settle_loads(&bars->kv_full, 1, steps > 0, status);
    } else if (warp == 9) {
      settle_products(&bars->idle, status);
    }
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, kDkvCols);
}

struct GradSumParams {
  const float* partial;             // [tensor][split][batch * heads][tokens][DP]
  uint16_t* out[2];
  int64_t stride[2][3];
  int64_t tokens, rows;             // rows = batch * heads * tokens
  int heads, dim, splits;
  // SUMS (dQ with an added mask): the parts' sums of weights, which dQ is divided by, and the statistics their log2 goes to
  const float* sums;
  float* stat;
  int64_t stat_rows;
};

// the splits' partial sums added in order; 8 elements per thread, blockIdx.y: the tensor (dQ; dK, dV)
template <int DP, bool BF, bool SUMS>
__global__ void __launch_bounds__(256) cross_grad_sum_kernel(const __grid_constant__ GradSumParams p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = i / (DP / 8);
  const int e = static_cast<int>(i % (DP / 8)) * 8;
  if (row >= p.rows || e >= p.dim) return;
  const float* src = p.partial + (blockIdx.y * p.splits * p.rows + row) * DP + e;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), c = a;
  float total = 0.f;
  for (int s = 0; s < p.splits; ++s, src += p.rows * DP) {
    if (SUMS) total += __ldg(p.sums + s * p.rows + row);
    const float4 x = __ldcs(reinterpret_cast<const float4*>(src)), y = __ldcs(reinterpret_cast<const float4*>(src + 4));
    a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
    c.x += y.x; c.y += y.y; c.z += y.z; c.w += y.w;
  }
  const int64_t token = row % p.tokens, bh = row / p.tokens, h = bh % p.heads, b = bh / p.heads;
  if (SUMS) {
    if (e == 0 && total != 0.f) p.stat[(bh * p.stat_rows + token / 64 * 64) * 3 + 64 + token % 64] += log2f(total);    // to -p_room
    const float inv = total == 0.f ? 1.f : 1.f / total;
    a.x *= inv; a.y *= inv; a.z *= inv; a.w *= inv;
    c.x *= inv; c.y *= inv; c.z *= inv; c.w *= inv;
  }
  const int64_t* st = p.stride[blockIdx.y];
  uint16_t* dst = p.out[blockIdx.y] + b * st[0] + token * st[1] + h * st[2] + e;
  *reinterpret_cast<uint4*>(dst) = make_uint4(pack16x2<BF>(a.x, a.y), pack16x2<BF>(a.z, a.w), pack16x2<BF>(c.x, c.y),
                                              pack16x2<BF>(c.z, c.w));
}

template <int DP, bool BF>
int launch_sum(GradSumParams r, const float* partial, int tensors, int64_t batch, int heads, int64_t tokens, int dim, int splits,
               cudaStream_t st) {
  r.partial = partial;
  r.tokens = tokens;
  r.rows = batch * heads * tokens;
  r.heads = heads;
  r.dim = dim;
  r.splits = splits;
  const int64_t blocks = (r.rows * (DP / 8) + 255) / 256;
  const dim3 grid(static_cast<unsigned>(blocks), tensors);
  if (r.sums != nullptr) cross_grad_sum_kernel<DP, BF, true><<<grid, 256, 0, st>>>(r);
  else cross_grad_sum_kernel<DP, BF, false><<<grid, 256, 0, st>>>(r);
  return cudaGetLastError() == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
}

// Parts of the keys in the dQ pass: the fewest rounds of CTAs times blocks (about 1.7 us each), with three blocks' time
// for a unit's ends and, for any split, three for the sum's launch and the time the parts' bytes take at 5 TB/s.
int dq_splits(const HtrcCrossArgs* a) {
  const int64_t units = a->batch * a->heads * ((a->queries + kDqRows - 1) / kDqRows);
  const int64_t steps = (a->keys + kDqKeys - 1) / kDqKeys, sms = sm_count();
  const double part_steps = static_cast<double>(a->batch) * a->heads * a->queries * (a->dim <= 64 ? 64 : 128) * 8 / 5e12 / 1.7e-6;
  int best = 1;
  double cost = 1e300;
  for (int s = 1; s <= 64 && s <= std::max<int64_t>(steps, 1); ++s) {
    const double c = static_cast<double>((units * s + sms - 1) / sms) * ((steps + s - 1) / s + 3) + (s > 1 ? 3 + s * part_steps : 0);
    if (c < cost) {
      cost = c;
      best = s;
    }
  }
  return best;
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

// words of a row's bits: whole blocks of either pass
int bit_words(const HtrcCrossArgs* a) { return static_cast<int>((a->keys + 127) / 128 * 4); }
size_t bits_bytes(const HtrcCrossArgs* a) {
  if (cross_mask_kind(a) != CROSS_PAIRS) return 0;
  const int64_t heads = a->mask_stride[1] != 0 ? a->heads : 1;
  return (static_cast<size_t>(a->batch) * heads * bit_words(a) * stat_rows(a) * 4 + 255) / 256 * 256;
}

// float16: CTAs per entry and key head that look for max|v|, and the bytes of their finds and the tiles' bounds
int vmax_parts(const HtrcCrossArgs* a) {
  const int64_t units = std::max<int64_t>(1, a->batch * a->kv_heads);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({kVmaxParts, (4 * sm_count() + units - 1) / units, (a->keys + 63) / 64})));
}
size_t vmax_bytes(const HtrcCrossArgs* a) {
  return a->dtype == HTRC_LAYER_F16 ? (static_cast<size_t>(a->batch) * a->kv_heads * vmax_parts(a) * 4 + 255) / 256 * 256 : 0;
}
size_t bounds_bytes(const HtrcCrossArgs* a) {
  return a->dtype == HTRC_LAYER_F16 ? (static_cast<size_t>(a->batch) * a->heads * (stat_rows(a) / kDqRows) * 4 + 255) / 256 * 256 : 0;
}

template <int DP, bool KEYED>
int launch_vmax(const HtrcCrossArgs* a, const CrossShape& s, uint32_t* vmax, cudaStream_t st) {
  VmaxParams m{};
  m.s = s;
  m.v = static_cast<const uint16_t*>(a->v);
  for (int i = 0; i < 3; ++i) m.vs[i] = a->v_stride[i];
  m.vmax = vmax;
  m.parts = vmax_parts(a);
  cross_vmax_kernel<DP, KEYED><<<static_cast<unsigned>(a->batch * a->kv_heads * m.parts), 256, 0, st>>>(m);
  return cudaGetLastError() == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
}

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
  static bool done_q[64] = {}, done_qs[64] = {}, done_kv[64] = {};
  auto kq = cross_dq_kernel<DP, BF, KIND, false>;
  auto kqs = cross_dq_kernel<DP, BF, KIND, true>;
  auto kkv = cross_dkv_kernel<DP, BF, KIND>;
  if (!ready(kq, DqSmem<DP>::kBytes, done_q) || !ready(kqs, DqSmem<DP>::kBytes, done_qs) || !ready(kkv, DkvSmem<DP>::kBytes, done_kv)) return HTRC_ERR_CUDA;
  const CrossShape s = cross_shape(a);
  float* stat = static_cast<float*>(a->workspace);
  const CrossBits bits{reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a->workspace) + stat_bytes(a)), bit_words(a), a->mask_stride[1] != 0};
  uint8_t* rest = static_cast<uint8_t*>(a->workspace) + stat_bytes(a) + bits_bytes(a);
  uint32_t* vmax = reinterpret_cast<uint32_t*>(rest);
  float* bounds = reinterpret_cast<float*>(rest + vmax_bytes(a));
  // the two passes' partial sums, one after the other
  float* partial = reinterpret_cast<float*>(rest + vmax_bytes(a) + bounds_bytes(a));
  const bool keys = a->keys > 0, rows = a->queries > 0;
  // an empty side's maps are never read: the other side's rows stand in
  const void *k = keys ? a->k : a->q, *v = keys ? a->v : a->q, *q = rows ? a->q : a->k, *o = rows ? a->dout : a->k;
  const int64_t *ks = keys ? a->k_stride : a->q_stride, *vs = keys ? a->v_stride : a->q_stride;
  const int64_t *qs = rows ? a->q_stride : a->k_stride, *os = rows ? a->dout_stride : a->k_stride;
  const int64_t nk = keys ? a->keys : a->queries, nq = rows ? a->queries : a->keys;
  const int hk = keys ? a->kv_heads : a->heads, hq = rows ? a->heads : a->kv_heads;
  int do_b = 0, do_h = 0, one;
  if (rows) {
    CUtensorMap mq, mo, mk, mv;
    DqParams p{};
    p.s = s;
    if (!cross_map(&mq, a, q, qs, nq, hq, kDqRows, &p.s.q_b, &p.s.q_h) || !cross_map(&mo, a, o, os, nq, hq, kDqRows, &do_b, &do_h) ||
        !cross_map(&mk, a, k, ks, nk, hk, kDqKeys, &p.s.k_b, &p.s.k_h) || !cross_map(&mv, a, v, vs, nk, hk, kDqKeys, &p.s.v_b, &p.s.v_h))
      return HTRC_ERR_CUDA;
    p.lse = a->lse;
    p.dlse = a->dlse;
    p.out = static_cast<const uint16_t*>(a->out);
    p.dq = static_cast<uint16_t*>(a->dq);
    for (int i = 0; i < 3; ++i) {
      p.out_stride[i] = a->out_stride[i];
      p.dq_stride[i] = a->dq_stride[i];
    }
    p.stat = stat;
    p.stat_rows = stat_rows(a);
    p.bits = bits;
    p.tiles = static_cast<uint32_t>(stat_rows(a) / kDqRows);
    p.splits = dq_splits(a);
    p.part = partial;
    constexpr bool natural = KIND == CROSS_KEYS || KIND == CROSS_BIAS;
    if (natural && p.splits > 1) p.part_sum = partial + static_cast<int64_t>(p.splits) * a->batch * a->heads * a->queries * DP;
    p.units = static_cast<uint32_t>(p.tiles * a->batch * a->heads * p.splits);
    p.do_b = do_b;
    p.do_h = do_h;
    p.status = a->status;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(std::min<uint32_t>(p.units, static_cast<uint32_t>(sm_count())));
    cfg.blockDim = dim3(kDqThreads);
    cfg.dynamicSmemBytes = DqSmem<DP>::kBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    if (!BF) {
      p.vmax = vmax;
      p.vmax_parts = vmax_parts(a);
      p.bounds = bounds;
      const int rc = launch_vmax<DP, KIND == CROSS_KEYS>(a, s, vmax, st);
      if (rc != HTRC_OK) return rc;
      // the launch, the first tiles and the first scores under that kernel, which itself started after all before it
      attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr.val.programmaticStreamSerializationAllowed = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
    }
    if (cudaLaunchKernelEx(&cfg, p.splits > 1 ? kqs : kq, mq, mo, mk, mv, p) != cudaSuccess) return HTRC_ERR_CUDA;
    if (p.splits > 1) {
      GradSumParams r{};
      r.out[0] = p.dq;
      for (int i = 0; i < 3; ++i) r.stride[0][i] = a->dq_stride[i];
      r.sums = p.part_sum;
      r.stat = stat;
      r.stat_rows = p.stat_rows;
      const int rc = launch_sum<DP, BF>(r, partial, 1, a->batch, a->heads, a->queries, a->dim, p.splits, st);
      if (rc != HTRC_OK) return rc;
    }
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
  p.bits = bits;
  p.bounds = bounds;
  p.tiles = static_cast<int>(stat_rows(a) / kDqRows);
  p.key_blocks = static_cast<int>((a->keys + kDkvKeys - 1) / kDkvKeys);
  p.row_blocks = static_cast<int>((a->queries + kDkvRows - 1) / kDkvRows);
  p.splits = dkv_splits(a);
  p.partial = partial;
  p.status = a->status;
  const int64_t grid = a->batch * a->kv_heads * p.splits * p.key_blocks;
  kkv<<<static_cast<unsigned>(grid), kDkvThreads, DkvSmem<DP>::kBytes, st>>>(mq, mo, mk, mv, mdk, mdv, p, do_b, do_h);
  if (cudaGetLastError() != cudaSuccess) return HTRC_ERR_CUDA;
  if (p.splits > 1) {
    GradSumParams r{};
    r.out[0] = static_cast<uint16_t*>(a->dk);
    r.out[1] = static_cast<uint16_t*>(a->dv);
    for (int i = 0; i < 3; ++i) {
      r.stride[0][i] = a->dk_stride[i];
      r.stride[1][i] = a->dv_stride[i];
    }
    return launch_sum<DP, BF>(r, p.partial, 2, a->batch, a->kv_heads, a->keys, a->dim, p.splits, st);
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
  if (tiles * a->batch * a->heads > limit || tiles * a->batch * a->heads * dq_splits(a) > limit || blocks > limit / (16 * std::max<int64_t>(1, a->batch * a->kv_heads)))
    return HTRC_ERR_UNSUPPORTED;
  const int dp = a->dim <= 64 ? 64 : 128, sq = dq_splits(a), sk = dkv_splits(a);
  const size_t of_dq = sq > 1 ? static_cast<size_t>(sq) * a->batch * a->heads * a->queries : 0;
  const size_t of_dkv = sk > 1 ? static_cast<size_t>(2) * sk * a->batch * a->kv_heads * a->keys : 0;
  // (a part's row of dQ: its elements and its sum of weights)
  *bytes = stat_bytes(a) + bits_bytes(a) + vmax_bytes(a) + bounds_bytes(a) + std::max(of_dq * (dp + 1), of_dkv * dp) * 4;
  return HTRC_OK;
}

int cross_backward(const HtrcCrossArgs* a, cudaStream_t st) {
  int rc = cross_validate(a, true, true);
  if (rc != HTRC_OK) return rc;
  size_t need = 0;
  rc = cross_sizes(a, &need);
  if (rc != HTRC_OK) return rc;
  if (!device_is_b200()) return HTRC_ERR_DEVICE;
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
