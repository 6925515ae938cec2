// Cross attention of few rows (single tokens): the query rows that share a key head, up to 16 at a time, against that
// head's keys and values.  The keys and values are read once and nothing else matters: a tcgen05 tile of 128 rows would
// load the same bytes behind a much longer chain of steps (87 us where this takes 19 for the 65 MB of 16 tokens,
// 24 heads on 8 key heads of 1,000 keys on average), so the products run on warp-level m16n8k16 instructions, whose rate
// is far above what the bytes ask for.
//
// All units' tiles of 32 keys (a unit: one entry, key head and up to 16 rows) form one line that the warps share evenly,
// 12 per SM, whatever the entries' lengths; what a warp has of a unit is a segment, and cross_few_join_kernel joins the
// units' segments.  (A cluster of up to 8 CTAs per unit, joined in place, took 28 us for the case above: the longest
// entry's clusters ran on while the others' SMs were idle.)  Units of two tiles or less, or as many units as half the
// warps, get a warp each and no second launch.
//
// A warp has buffers of its own in shared memory (16-byte asynchronous copies: the next tile's keys land while this
// tile's values are used, its values while its scores are formed; 192 KB per SM) and waits on no other.  S = Q K^T has the
// layout of the second product's left operand, so P stays in registers; running maximum and sum in float32; P enters P V
// in the operands' 16-bit type as on the larger path.  Every sum has a fixed order.
//
// With a key mask per query head a unit has one head's rows: a key that this head excludes and another one sees may hold
// anything (0 * NaN in P V), and its values become zeros only where no row of the unit sees it.  (Three heads to a key
// head then read it three times: 16 tokens x 24 heads on 8 key heads of 2,000 keys 70 us, 36 with one mask for all.)
#include <algorithm>

#include "cross.cuh"

namespace htrc {

namespace {

constexpr int kFewWarps = 6, kFewRows = 16, kFewBatch = 192;
constexpr int kFewAlone = 2;                 // tiles of a unit that a warp takes whole
constexpr int kFewSegments = 64;             // warps of a unit, at most about

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// four 8 x 8 matrices of 16-bit elements; lane i gives the address of row i % 8 of matrix i / 8
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// d += a b, 16 x 8 (float32) += 16 x 16 times 16 x 8
template <bool BF>
__device__ __forceinline__ void mma_16x8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int DP>
struct FewSmem {
  static constexpr uint32_t kTile = 32 * DP * 2;                 // 32 rows of keys, or of values
  static constexpr uint32_t kTiles = 0, kStarts = kFewWarps * 2 * kTile;          // [warp][keys, values]
  static constexpr uint32_t kBytes = kStarts + (kFewBatch + 1) * 8 + kFewWarps * 8;
};

struct CrossFewParams {
  CrossShape s;
  const uint16_t *q, *k, *v;
  uint16_t* out;
  float* lse;
  int64_t qs[3], ks[3], vs[3], os[3];
  int chunks;               // of 16 rows of (head in the group, query)
  int span;                 // rows of a head: its queries, or whole chunks of them
  bool line;                // the warps share the line of all units' tiles (else a warp has a unit)
  int64_t units;
  // line: the entries' starts (in tiles of one key head and chunk) [batch + 1], then each segment's rows
  int64_t* starts;
  float2* part_ml;          // (maximum, sum) [segment][16]
  float* part;              // [segment][16][DP]
};

// Segment of unit u in warp i: segments in order step i, u or both, so the sum numbers them
__device__ __forceinline__ int64_t few_slot(int64_t u, int64_t i) { return u + i; }

// a row's place: index = head in the group * span + query; n and h mean something where it is live
struct FewRow {
  int n, h;
  bool live;
  __device__ __forceinline__ FewRow(const CrossFewParams& p, int unit, int r) {
    const int queries = static_cast<int>(p.s.queries), at = unit % p.chunks * kFewRows + r;
    const int g = at / p.span;
    n = at - g * p.span;
    live = g < p.s.group && n < queries;
    h = unit / p.chunks % p.s.kv_heads * p.s.group + g;
  }
};

__device__ __forceinline__ void few_lse(const CrossFewParams& p, int b, const FewRow& w, float m, float l) {
  if (p.lse != nullptr)
    p.lse[(static_cast<int64_t>(b) * p.s.heads + w.h) * p.s.queries + w.n] = l > 0.f || l != l ? m + logf(l) : -INFINITY;
}

// A tile of 32 keys on the line
struct FewCursor {
  int b, unit, t, tiles, count;       // tiles and keys of the unit's entry
};

// i / w of a line of `all` tiles; the products fit 32 bits unless the line is very long
__device__ __forceinline__ int64_t few_start(int64_t all, int64_t i, int64_t w) {
  const int64_t x = all * i;
  return x >> 32 ? x / w : static_cast<int64_t>(static_cast<uint32_t>(x) / static_cast<uint32_t>(w));
}

// MASKED: there is a mask.  WIDE: units of more than 8 rows (else a lane's second row is not computed).
template <int DP, bool BF, bool MASKED, bool WIDE>
__global__ void __launch_bounds__(kFewWarps * 32, 2)
    cross_few_kernel(const __grid_constant__ CrossFewParams p) {
  using SM = FewSmem<DP>;
  constexpr int R = kFewRows, U = WIDE ? 2 : 1;
  constexpr int PCS = DP / 8, KPI = 32 / PCS;                       // 16-byte pieces of a row, rows per copy instruction
  extern __shared__ __align__(128) uint8_t smem[];
  int64_t* starts = reinterpret_cast<int64_t*>(smem + SM::kStarts);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, t4 = lane & 3;
  const int per_entry = p.s.kv_heads * p.chunks;
  const int64_t self = static_cast<int64_t>(blockIdx.x) * kFewWarps + warp;
  int64_t left;                           // tiles of this warp, the first at cur
  FewCursor cur;
  if (p.line) {
    // tiles before each entry: a scan over the CTA's threads
    const int batch = static_cast<int>(p.s.batch);
    int64_t* sums = starts + kFewBatch + 1;
    int64_t mine = static_cast<int>(threadIdx.x) < batch ? (key_count(p.s, threadIdx.x) + 31) / 32 : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, mine, o);
      if (lane >= o) mine += y;
    }
    if (lane == 31) sums[warp] = mine;
    __syncthreads();
    for (int w = 0; w < warp; ++w) mine += sums[w];
    if (static_cast<int>(threadIdx.x) < batch) {
      starts[threadIdx.x + 1] = mine;
      if (blockIdx.x == 0) p.starts[threadIdx.x + 1] = mine;
    }
    if (threadIdx.x == 0) {
      starts[0] = 0;
      if (blockIdx.x == 0) p.starts[0] = 0;
    }
    __syncthreads();
    const int64_t all = starts[batch] * per_entry, warps = min(all, static_cast<int64_t>(gridDim.x) * kFewWarps);
    if (self >= warps) return;
    const int64_t x = few_start(all, self, warps);
    left = few_start(all, self + 1, warps) - x;
    int lo = 0, hi = batch;
    while (hi - lo > 1) {                 // the last entry that starts at or before x (one without keys starts where the next does)
      const int mid = (lo + hi) / 2;
      if (starts[mid] * per_entry <= x) lo = mid;
      else hi = mid;
    }
    cur.b = lo;
    cur.tiles = static_cast<int>(starts[lo + 1] - starts[lo]);
    const int64_t in = x - starts[lo] * per_entry;
    const int u = static_cast<int>(in / cur.tiles);
    cur.t = static_cast<int>(in - static_cast<int64_t>(u) * cur.tiles);
    cur.unit = lo * per_entry + u;
    cur.count = key_count(p.s, lo);
  } else {
    if (self >= p.units) return;
    cur.unit = static_cast<int>(self);
    cur.b = cur.unit / per_entry;
    cur.count = key_count(p.s, cur.b);
    cur.t = 0;
    left = cur.tiles = (cur.count + 31) / 32;
  }
  auto advance = [&](FewCursor& c) {      // only where the line goes on
    if (++c.t < c.tiles) return;
    c.t = 0;
    if (++c.unit < (c.b + 1) * per_entry) return;
    do {
      ++c.b;
      c.tiles = static_cast<int>(starts[c.b + 1] - starts[c.b]);
    } while (c.tiles == 0);
    c.unit = c.b * per_entry;
    c.count = key_count(p.s, c.b);
  };

  uint8_t* tile = smem + SM::kTiles + warp * 2 * SM::kTile;
  const uint32_t tile_k = smem_u32(tile), tile_v = tile_k + SM::kTile;
  // a tile's keys (values): row r's piece c at piece c ^ (r & 7); rows past the entry's keys and pieces past dim are zeros
  auto fetch = [&](const FewCursor& at, bool values) {
    const int hk = at.unit / p.chunks % p.s.kv_heads;
    const uint16_t* src = values ? p.v + at.b * p.vs[0] + hk * p.vs[2] : p.k + at.b * p.ks[0] + hk * p.ks[2];
    const int64_t step = values ? p.vs[1] : p.ks[1];
    const uint32_t base = (values ? tile_v : tile_k) + lane / PCS * (DP * 2);
    const int r0 = lane / PCS, c = lane % PCS;
    src += static_cast<int64_t>(at.t * 32 + r0) * step + 8 * c;
    if (at.t * 32 + 32 <= at.count && p.s.dim == DP) {
#pragma unroll
      for (int i = 0; i < PCS; ++i) {
        copy16(base + i * KPI * (DP * 2) + ((c ^ ((i * KPI + r0) & 7)) << 4), src, true);
        src += KPI * step;
      }
    } else {
#pragma unroll
      for (int i = 0; i < PCS; ++i) {
        const bool in = at.t * 32 + i * KPI + r0 < at.count && 8 * c < p.s.dim;
        copy16(base + i * KPI * (DP * 2) + ((c ^ ((i * KPI + r0) & 7)) << 4), in ? src : p.k, in);
        src += KPI * step;
      }
    }
  };
  if (left > 0) fetch(cur, false);
  copy_commit();
  if (left > 0) fetch(cur, true);
  copy_commit();

  // this lane's rows of S and O: g4 and g4 + 8 of the unit
  uint32_t q[DP / 16][4];
  int64_t mask_row[U];
  bool live[U];
  float m[U], l[U], acc[DP / 8][4];
  int first = cur.t;                      // of the segment
  bool opened = false;
  FewCursor nxt = cur;
  do {
    if (!opened) {
      opened = true;
      first = cur.t;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const FewRow w(p, cur.unit, g4 + 8 * u);
        live[u] = w.live;
        mask_row[u] = cur.b * p.s.mask.sb + w.h * p.s.mask.sh + w.n * p.s.mask.sn;
        const uint16_t* row = p.q + cur.b * p.qs[0] + w.n * p.qs[1] + w.h * p.qs[2];
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const int e = 16 * kk + 8 * v + 2 * t4;
            q[kk][u + 2 * v] = w.live && e < p.s.dim ? __ldg(reinterpret_cast<const uint32_t*>(row + e)) : 0u;
            if (!WIDE) q[kk][1 + 2 * v] = 0u;
          }
        m[u] = -INFINITY;
        l[u] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < DP / 8; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[i][v] = 0.f;
    }
    const bool more = left > 1;
    if (left > 0) {
      if (more) advance(nxt);
      copy_wait<1>();
      __syncwarp();
      float s[4][4];                        // keys 8 i + 2 t4, + 1 of rows g4 (0, 1) and g4 + 8 (2, 3)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int v = 0; v < 4; ++v) s[i][v] = 0.f;
        const int r = 8 * i + (lane & 7);
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk += 2) {
          uint32_t x[4];
          ldsm4(tile_k + r * (DP * 2) + (((2 * kk + (lane >> 3)) ^ (r & 7)) << 4), x);
          mma_16x8<BF>(s[i], q[kk], x[0], x[1]);
          mma_16x8<BF>(s[i], q[kk + 1], x[2], x[3]);
        }
      }
      __syncwarp();
      if (more) fetch(nxt, false);
      copy_commit();
      // natural logits where there is a mask, else in log2 units; U rows of 8 keys per lane
      const float scale = MASKED ? p.s.scale : p.s.scale * kCrossLog2e;
      const bool full = cur.t * 32 + 32 <= cur.count;
      uint32_t seen = 0;
      float mx[U];
#pragma unroll
      for (int u = 0; u < U; ++u) mx[u] = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < 2 * U; ++v) {
          const int u = v >> 1, bit = 8 * i + 2 * t4 + (v & 1), key = cur.t * 32 + bit;
          float x = s[i][v] * scale;
          if (MASKED) {
            x = -INFINITY;
            if (key < cur.count && live[u]) {
              const float bias = mask_term(p.s.mask.p, p.s.mask.dtype, mask_row[u] + static_cast<int64_t>(key) * p.s.mask.sm);
              if (bias != -INFINITY) {
                x = fmaf(s[i][v], scale, bias);
                seen |= 1u << bit;
              }
            }
          } else if (!full && key >= cur.count) {
            x = -INFINITY;
          }
          s[i][v] = x;
          mx[u] = fmaxf(mx[u], x);
        }
      float alpha[U];
      bool grow = false;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 1));
        mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 2));
        const float mn = fmaxf(m[u], mx[u]);
        mx[u] = mn == -INFINITY ? 0.f : mn;                        // the reference
        alpha[u] = cross_ex2(MASKED ? (m[u] - mx[u]) * kCrossLog2e : m[u] - mx[u]);
        grow |= mn != m[u];
        m[u] = mn;
        l[u] *= alpha[u];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          if (v >= 2 * U) {
            s[i][v] = 0.f;
            continue;
          }
          s[i][v] = cross_ex2(MASKED ? (s[i][v] - mx[v >> 1]) * kCrossLog2e : s[i][v] - mx[v >> 1]);
          l[v >> 1] += s[i][v];
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
#pragma unroll
          for (int v = 0; v < 2 * U; ++v) acc[i][v] *= alpha[v >> 1];
      }
      copy_wait<1>();
      __syncwarp();
      if (MASKED) {
        // the values of keys that no row sees may hold anything (0 * NaN): they become zeros
        seen = __reduce_or_sync(0xffffffffu, seen);
        if (seen != 0xffffffffu) {
          for (uint32_t todo = ~seen; todo; todo &= todo - 1)
            if (lane < PCS) *reinterpret_cast<uint4*>(tile + SM::kTile + (__ffs(todo) - 1) * (DP * 2) + lane * 16) = make_uint4(0, 0, 0, 0);
          __syncwarp();
        }
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const uint32_t a[4] = {pack16x2<BF>(s[2 * kk][0], s[2 * kk][1]), pack16x2<BF>(s[2 * kk][2], s[2 * kk][3]),
                               pack16x2<BF>(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack16x2<BF>(s[2 * kk + 1][2], s[2 * kk + 1][3])};
        const int r = 16 * kk + (lane & 15);
#pragma unroll
        for (int i = 0; i < DP / 8; i += 2) {
          uint32_t x[4];
          ldsm4_t(tile_v + r * (DP * 2) + (((i + (lane >> 4)) ^ (r & 7)) << 4), x);
          mma_16x8<BF>(acc[i], a, x[0], x[1]);
          mma_16x8<BF>(acc[i + 1], a, x[2], x[3]);
        }
      }
      __syncwarp();
      if (more) fetch(nxt, true);
      copy_commit();
    }
    if (!more || nxt.unit != cur.unit) {
      // the segment ends; maxima leave in natural units
      const bool whole = !p.line || (first == 0 && cur.t + 1 == cur.tiles);
      const int64_t slot = few_slot(cur.unit, self) * R;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
        const float top = MASKED ? m[u] : m[u] * kCrossLn2;
        const int r = g4 + 8 * u;
        if (!live[u]) continue;
        if (whole) {
          const FewRow w(p, cur.unit, r);
          const float inv = l[u] == 0.f ? 0.f : 1.0f / l[u];
          uint16_t* dst = p.out + cur.b * p.os[0] + w.n * p.os[1] + w.h * p.os[2];
#pragma unroll
          for (int i = 0; i < DP / 8; ++i)
            if (8 * i + 2 * t4 < p.s.dim)
              *reinterpret_cast<uint32_t*>(dst + 8 * i + 2 * t4) = pack16x2<BF>(acc[i][2 * u] * inv, acc[i][2 * u + 1] * inv);
          if (t4 == 0) few_lse(p, cur.b, w, top, l[u]);
        } else {
          float* dst = p.part + (slot + r) * DP;
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) *reinterpret_cast<float2*>(dst + 8 * i + 2 * t4) = make_float2(acc[i][2 * u], acc[i][2 * u + 1]);
          if (t4 == 0) p.part_ml[slot + r] = make_float2(top, l[u]);
        }
      }
      opened = false;
    }
    cur = nxt;
  } while (--left > 0);
  copy_wait<0>();
}

// units of several segments (or none): a CTA per row, a group of DP / 4 threads per segment
template <int DP, bool BF>
__global__ void __launch_bounds__(256) cross_few_join_kernel(const __grid_constant__ CrossFewParams p, int64_t most) {
  asm volatile("griddepcontrol.wait;" ::: "memory");               // the first kernel's results
  constexpr int T = DP / 4, G = 256 / T;                            // threads per row (4 columns each), groups
  __shared__ float4 acc_s[G][T];
  __shared__ float ml_s[G][2];
  const int unit = blockIdx.x, per_entry = p.s.kv_heads * p.chunks, b = unit / per_entry;
  const int g = threadIdx.x / T, c = threadIdx.x % T;
  const int64_t all = p.starts[p.s.batch] * per_entry, tiles = p.starts[b + 1] - p.starts[b], warps = min(all, most);
  const int64_t first = p.starts[b] * per_entry + (unit - static_cast<int64_t>(b) * per_entry) * tiles;
  int i0 = 0, n = 0;                      // the warps that have some of it
  if (tiles > 0) {
    i0 = static_cast<int>(((first + 1) * warps - 1) / all);
    n = static_cast<int>(((first + tiles) * warps - 1) / all) - i0 + 1;
    if (n == 1) return;
  }
  const int64_t slot0 = few_slot(unit, i0) * kFewRows;
  const int r = blockIdx.y;
  const FewRow w(p, unit, r);
  if (!w.live) return;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = g; i < n; i += 4 * G) {
    // four segments' loads together
    float2 ml[4];
    float4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t slot = slot0 + static_cast<int64_t>(i + k * G) * kFewRows + r;
      const bool in = i + k * G < n;
      ml[k] = in ? p.part_ml[slot] : make_float2(-INFINITY, 0.f);
      x[k] = in ? *reinterpret_cast<const float4*>(p.part + slot * DP + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float mn = fmaxf(m, ml[k].x), ref = mn == -INFINITY ? 0.f : mn;
      const float f0 = cross_ex2((m - ref) * kCrossLog2e), f1 = cross_ex2((ml[k].x - ref) * kCrossLog2e);
      m = mn;
      l = l * f0 + ml[k].y * f1;
      acc.x = acc.x * f0 + x[k].x * f1;
      acc.y = acc.y * f0 + x[k].y * f1;
      acc.z = acc.z * f0 + x[k].z * f1;
      acc.w = acc.w * f0 + x[k].w * f1;
    }
  }
  acc_s[g][c] = acc;
  if (c == 0) {
    ml_s[g][0] = m;
    ml_s[g][1] = l;
  }
  __syncthreads();
  if (threadIdx.x < DP) {
    const int d = threadIdx.x;
    float mm = -INFINITY;
#pragma unroll
    for (int i = 0; i < G; ++i) mm = fmaxf(mm, ml_s[i][0]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    float a = 0.f, ll = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const float f = cross_ex2((ml_s[i][0] - ref) * kCrossLog2e);
      a = fmaf(reinterpret_cast<const float*>(acc_s[i])[d], f, a);
      ll = fmaf(ml_s[i][1], f, ll);
    }
    if (d < p.s.dim) {
      const float x = ll == 0.f ? 0.f : a / ll;
      uint16_t* dst = p.out + b * p.os[0] + w.n * p.os[1] + w.h * p.os[2] + d;
      if (BF) *reinterpret_cast<__nv_bfloat16*>(dst) = __float2bfloat16_rn(x);
      else *reinterpret_cast<__half*>(dst) = __float2half_rn(x);
    }
    if (d == 0) few_lse(p, b, w, mm, ll);
  }
}

template <int DP, bool BF, bool MASKED, bool WIDE>
int launch_few_main(const CrossFewParams& p, int ctas, cudaStream_t st) {
  static bool done[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return HTRC_ERR_CUDA;
  constexpr uint32_t bytes = FewSmem<DP>::kBytes;
  if (dev >= 64 || !done[dev]) {
    if (cudaFuncSetAttribute(cross_few_kernel<DP, BF, MASKED, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return HTRC_ERR_CUDA;
    if (dev < 64) done[dev] = true;
  }
  cross_few_kernel<DP, BF, MASKED, WIDE><<<ctas, kFewWarps * 32, bytes, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
}

struct FewPlan {
  int64_t units;
  int rows, span, chunks, ctas;   // rows: of a unit, at most
  bool line;
  size_t starts, ml, bytes;       // workspace: where the segments' parts begin, and its size
};

template <int DP, bool BF>
int launch_few(const CrossFewParams& p, const FewPlan& f, cudaStream_t st) {
  const bool wide = f.rows > 8;
  const int rc = p.s.mask.p ? (wide ? launch_few_main<DP, BF, true, true>(p, f.ctas, st) : launch_few_main<DP, BF, true, false>(p, f.ctas, st))
                            : (wide ? launch_few_main<DP, BF, false, true>(p, f.ctas, st) : launch_few_main<DP, BF, false, false>(p, f.ctas, st));
  if (rc != HTRC_OK) return rc;
  if (!p.line) return HTRC_OK;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(f.units), static_cast<unsigned>(f.rows));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;     // its launch under the first kernel's end
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, cross_few_join_kernel<DP, BF>, p, static_cast<int64_t>(f.ctas) * kFewWarps) == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
}

FewPlan few_plan(const HtrcCrossArgs* a) {
  FewPlan f{};
  const int64_t group = a->heads / a->kv_heads, tiles = (a->keys + 31) / 32;
  const bool apart = group > 1 && cross_mask_kind(a) == CROSS_KEYS && a->mask_stride[1] != 0;      // a key mask per head
  f.span = static_cast<int>(apart ? (a->queries + kFewRows - 1) / kFewRows * kFewRows : a->queries);
  f.rows = static_cast<int>(std::min<int64_t>(kFewRows, apart ? a->queries : group * a->queries));
  f.chunks = static_cast<int>((group * f.span + kFewRows - 1) / kFewRows);
  f.units = a->batch * a->kv_heads * f.chunks;
  // The line evens out the entries' lengths for the price of the segments' rows and the join.  Ragged entries, 8 key heads
  // of up to 1,000 keys: 512 units of 3 rows 36.5 us in line and 52.2 apart, of 15 rows 62.7 and 59.1; 1,024 units of 3
  // rows 64.7 either way, of 15 rows 107 and 71.  (Its starts are found by one CTA: kFewBatch entries.)
  f.line = tiles > kFewAlone && a->batch <= kFewBatch && f.units < int64_t(sm_count()) * kFewWarps;
  const int64_t most = f.line ? std::min(f.units * std::min<int64_t>(tiles, kFewSegments), int64_t(2) * sm_count() * kFewWarps) : f.units;
  f.ctas = static_cast<int>((most + kFewWarps - 1) / kFewWarps);
  if (!f.line) return f;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const int64_t slots = f.units + static_cast<int64_t>(f.ctas) * kFewWarps;
  f.starts = up((a->batch + 1) * 8);
  f.ml = f.starts + up(slots * kFewRows * 8);
  f.bytes = f.ml + static_cast<size_t>(slots) * kFewRows * (a->dim <= 64 ? 64 : 128) * 4;
  return f;
}

}  // namespace

size_t cross_few_bytes(const HtrcCrossArgs* a) { return few_plan(a).bytes; }

int cross_forward_few(const HtrcCrossArgs* a, cudaStream_t st) {
  const FewPlan f = few_plan(a);
  if (f.units > (int64_t(1) << 31) - 1) return HTRC_ERR_UNSUPPORTED;
  CrossFewParams p{};
  p.s = cross_shape(a);
  p.q = static_cast<const uint16_t*>(a->q);
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.out = static_cast<uint16_t*>(a->out);
  p.lse = a->lse;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = a->q_stride[i];
    p.ks[i] = a->k_stride[i];
    p.vs[i] = a->v_stride[i];
    p.os[i] = a->out_stride[i];
  }
  p.chunks = f.chunks;
  p.span = f.span;
  p.line = f.line;
  p.units = f.units;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  if (f.line) {
    p.starts = reinterpret_cast<int64_t*>(ws);
    p.part_ml = reinterpret_cast<float2*>(ws + f.starts);
    p.part = reinterpret_cast<float*>(ws + f.ml);
  }
  const bool bf = a->dtype == HTRC_LAYER_BF16;
  if (a->dim <= 64) return bf ? launch_few<64, true>(p, f, st) : launch_few<64, false>(p, f, st);
  return bf ? launch_few<128, true>(p, f, st) : launch_few<128, false>(p, f, st);
}

}  // namespace htrc
