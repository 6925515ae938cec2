// Shared by the cross-attention kernels (cross_fwd.cu, cross_bwd.cu): the masks, the element types, the shapes that
// the C entries check, and the tensor maps of [batch][token][head][dim] operands.
#pragma once
#include "../../include/htrc_layer.h"
#include "common.cuh"
#include "kernels.cuh"

namespace htrc {

// How a launch's mask is read; the key lengths apply in every kind.
enum CrossMask : int {
  CROSS_NONE = 0,       // no mask
  CROSS_KEYS = 1,       // the same for every query: a bias per key (0 / -inf from a bool mask)
  CROSS_PAIRS = 2,      // bool, per query and key
  CROSS_BIAS = 3,       // added, per query and key
};

struct CrossMaskView {
  const void* p;
  int64_t sb, sh, sn, sm;
  int dtype;
};

// the mask's term at element offset i: -inf excludes
__device__ __forceinline__ float mask_term(const void* p, int dtype, int64_t i) {
  if (dtype == HTRC_LAYER_U8) return __ldg(static_cast<const uint8_t*>(p) + i) ? 0.f : -INFINITY;
  if (dtype == HTRC_LAYER_F32) return __ldg(static_cast<const float*>(p) + i);
  if (dtype == HTRC_LAYER_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// N terms from element offset `at` on, `step` apart; those from n on are excluded.  The type is looked at once, so that
// the loads are in flight together.
template <int N>
__device__ __forceinline__ void mask_terms(const void* p, int dtype, int64_t at, int64_t step, int n, float (&t)[N]) {
  if (dtype == HTRC_LAYER_U8) {
    const uint8_t* x = static_cast<const uint8_t*>(p) + at;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = i < n ? static_cast<float>(__ldg(x + i * step)) : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = t[i] != 0.f ? 0.f : -INFINITY;
  } else if (dtype == HTRC_LAYER_F32) {
    const float* x = static_cast<const float*>(p) + at;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = i < n ? __ldg(x + i * step) : -INFINITY;
  } else if (dtype == HTRC_LAYER_BF16) {
    const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p) + at;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = i < n ? __bfloat162float(x[i * step]) : -INFINITY;
  } else {
    const __half* x = static_cast<const __half*>(p) + at;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = i < n ? __half2float(x[i * step]) : -INFINITY;
  }
}

struct CrossShape {
  int64_t batch, queries, keys;
  int heads, kv_heads, group, dim;
  float scale;                          // of the natural logits
  const int32_t* lengths;
  CrossMaskView mask;
  // 1 where a tensor has that batch / head dimension, 0 where it is broadcast along it (the map then has one)
  int q_b, q_h, k_b, k_h, v_b, v_h;
};

// keys of batch entry b
__device__ __forceinline__ int key_count(const CrossShape& s, int b) {
  if (s.lengths == nullptr) return static_cast<int>(s.keys);
  const int n = __ldg(s.lengths + b);
  return max(0, min(n, static_cast<int>(s.keys)));
}

template <bool BF>
__device__ __forceinline__ uint32_t pack16x2(float lo, float hi) {
  return BF ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}
template <bool BF>
__device__ __forceinline__ float2 unpack16x2(uint32_t w) {
  if (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
template <bool BF>
__host__ __device__ constexpr uint32_t idesc16(int M, int N, bool a_mn, bool b_mn) {
  return BF ? idesc_bf16(M, N, a_mn, b_mn) : idesc_f16(M, N, a_mn, b_mn);
}

// After a wait that ran out, before the CTA leaves (each again with a limit of its own): the last fills of a ring of loads
// have landed, and the products that this warp issued are done.  Calls at the kernels' ends: inlined in their roles they
// took 6 % of the forward's time (129,024 x 512 keys) for code that does not run.
static __noinline__ __device__ void settle_loads(uint64_t* full, int slots, int fills, int* status) {
  int gave_up = 0;
  drain_ring<true>(full, slots, fills, status, &gave_up);
}
static __noinline__ __device__ void settle_products(uint64_t* idle, int* status) {
  int gave_up = 0;
  mma_commit_by(elect_one(), idle);
  mbar_wait_warp(idle, 0, status, &gave_up);
}

constexpr float kCrossLog2e = 1.4426950408889634f;
constexpr float kCrossLn2 = 0.6931471805599453f;

__device__ __forceinline__ float cross_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, const void* src, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}

// Groups of P lanes hold P 16-byte pieces of a row each; they exchange them so that lane i holds piece i % P of the
// group's rows, and a store instruction then writes P * 16 contiguous bytes of a few rows instead of 16 of 32 rows (which
// takes a pass of the store path per row).
template <int P>
__device__ __forceinline__ void exchange_pieces(uint32_t (&x)[P][4], int lane) {
#pragma unroll
  for (int d = 1; d < P; d *= 2) {
    const bool up = lane & d;
#pragma unroll
    for (int g = 0; g < P; ++g) {
      if (g & d) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // the lower lane keeps its piece g and takes the upper's g; the upper lane keeps g + d and takes the lower's
        const uint32_t give = up ? x[g][i] : x[g + d][i];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, give, d);
        if (up) x[g][i] = got;
        else x[g + d][i] = got;
      }
    }
  }
}

__device__ __forceinline__ void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }
__host__ __device__ constexpr int mask_bytes(int dtype) { return dtype == HTRC_LAYER_U8 ? 1 : dtype == HTRC_LAYER_F32 ? 4 : 2; }
// a mask's terms at element offset i and what shares their line
__device__ __forceinline__ void prefetch_mask(const CrossMaskView& m, int64_t i) {
  prefetch_l1(static_cast<const uint8_t*>(m.p) + i * mask_bytes(m.dtype));
}

// A descriptor's constant words: K-major operand (LBO unused) and MN-major operand with 64-element chunks lbo apart
__device__ __forceinline__ uint64_t desc_k(uint32_t smem) { return sw128_desc(smem, 16, 1024); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t smem, uint32_t lbo) { return sw128_desc(smem, lbo, 1024); }

// Zeroes the rows of a staged [chunks][rows][64] tile (chunk_bytes apart) whose key is excluded for every query: past
// the entry's keys or -inf in a per-key mask.  One warp; the writes are made visible to the tensor cores' reads.
// Lane i decides keys key0 + 32 r + i.
template <int ROWS, int CHUNKS>
__device__ __forceinline__ void zero_excluded_rows(uint8_t* tile, uint32_t chunk_bytes, int key0, int count,
                                                   const CrossShape& s, int64_t mask_at, bool keyed, int lane) {
#pragma unroll
  for (int r = 0; r < ROWS / 32; ++r) {
    const int key = key0 + 32 * r + lane;
    bool out = key >= count;
    if (!out && keyed) out = mask_term(s.mask.p, s.mask.dtype, mask_at + static_cast<int64_t>(key) * s.mask.sm) == -INFINITY;
    uint32_t todo = __ballot_sync(0xffffffffu, out);
    while (todo) {
      // four rows at a time: 8 lanes per 128-byte row
      int row = -1;
      uint32_t rest = todo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int f = rest ? __ffs(rest) - 1 : -1;
        if (rest) rest &= rest - 1;
        if (lane / 8 == i) row = f;
      }
      todo = rest;
      if (row >= 0) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
          *reinterpret_cast<uint4*>(tile + c * chunk_bytes + (32 * r + row) * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

int cross_validate(const HtrcCrossArgs* a, bool back, bool ptrs);
CrossShape cross_shape(const HtrcCrossArgs* a);
int cross_mask_kind(const HtrcCrossArgs* a);
// [batch][token][head][dim] as a 4-d map (dim, token, head, batch), box (64, box_rows, 1, 1), 128-byte swizzle; *b and
// *h are cleared for a dimension the tensor is broadcast along
bool cross_map(CUtensorMap* m, const HtrcCrossArgs* a, const void* base, const int64_t* stride, int64_t rows, int heads,
               int box_rows, int* b, int* h);

// few rows that share a key head, computed without matrix tiles (cross_few.cu)
int cross_forward_few(const HtrcCrossArgs* a, cudaStream_t st);
size_t cross_few_bytes(const HtrcCrossArgs* a);              // its workspace
constexpr int kCrossFewRows = 16;                            // a chunk of them

}  // namespace htrc
