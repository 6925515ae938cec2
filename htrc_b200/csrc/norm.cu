// Layer norm with a learned affine and a modulation per batch entry, forward and backward, and rows in 8-bit integers
// with a scale each (of a norm's result, or of the rows as they are) for the product in linear8.cu.
//
//   u = (x - mean) rstd,   y = (u weight + bias) (1 + scale) + shift = u A + B
//   codes = rint(y (127 / top)), scales = top / 127, top = max |y| of the row
//
// Forward: a row is read once and stays in registers as it was read, W warps to a row and rows to the CTA's warps; mean,
// then the squared deviations from it (no cancellation under a large mean), then the result, all float32.  A and B are
// formed once per batch entry in shared memory.  HBM bounds it: 4 bytes per 16-bit element, 3 to 8-bit rows.
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "../../include/htrc_layer.h"
#include "common.cuh"
#include "kernels.cuh"

namespace htrc {

namespace {

constexpr int kNormThreads = 256;           // of a CTA with a warp per row; wider rows: 32 W
constexpr int kNormMaxWarps = 16;           // per row
constexpr float kRoundMagic = 12582912.f;   // 1.5 * 2^23: adding it rounds to the nearest integer, ties to even
constexpr float kLeastTop = 1e-30f;         // of a quantised row: 127 / top stays finite

enum NormMode : int { NORM_ROWS = 0, NORM_CODES = 1, QUANT_CODES = 2 };

struct TermView {                           // a vector of the width, per batch entry where stride is not 0
  const void* p;
  int64_t stride;
  int dtype;
};

struct NormParams {
  const void* x;
  int64_t xs[2];                            // entry, row
  void* out;
  int64_t os[2];
  int8_t* codes;
  int64_t pitch;                            // codes: rows in order, whatever the entry
  float* scales;
  float *mean, *rstd;
  int64_t entries, rows;                    // rows per entry
  int width, nvec, warps;                   // vectors per row, warps per row
  int64_t chunk, chunks;                    // rows of a task, tasks per entry
  float eps, inv_width;
  bool affine, modulated;
  TermView weight, bias, scale, shift;
};

__device__ __forceinline__ float term_at(const void* p, int dtype, int64_t i) {
  if (dtype == HTRC_LAYER_F32) return __ldg(static_cast<const float*>(p) + i);
  if (dtype == HTRC_LAYER_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// N neighbouring elements as they were read: 16 bytes, or two elements by themselves where rows are not 16-byte aligned
// (`both`: the second is within the row; it is 0 where not)
template <typename T, bool VEC>
struct Piece {
  static constexpr int N = VEC ? 16 / sizeof(T) : 2, W = VEC ? 4 : 2;
  uint32_t w[W];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0;
  }
  // makes the next use unpack the elements again, rather than keep each in a register of its own
  __device__ __forceinline__ void packed() {
#pragma unroll
    for (int i = 0; i < W; ++i) asm volatile("" : "+r"(w[i]));
  }
  __device__ __forceinline__ void load(const T* p, bool both) {
    if constexpr (VEC) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (sizeof(T) == 4) {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
      w[1] = both ? __ldg(reinterpret_cast<const uint32_t*>(p) + 1) : 0;
    } else {
      w[0] = __ldg(reinterpret_cast<const unsigned short*>(p));
      w[1] = both ? __ldg(reinterpret_cast<const unsigned short*>(p) + 1) : 0;
    }
  }
  __device__ __forceinline__ static float one(uint32_t bits) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(bits);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(bits << 16);
    else return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  }
  // elements 2 i and 2 i + 1
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (!VEC || sizeof(T) == 4) {
      return make_float2(one(w[2 * i]), one(w[2 * i + 1]));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    } else {
      return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    }
  }
  __device__ __forceinline__ void set(int i, float2 v) {
    if constexpr (sizeof(T) == 4) {
      w[2 * i] = __float_as_uint(v.x);
      w[2 * i + 1] = __float_as_uint(v.y);
    } else {
      const uint32_t two = std::is_same<T, __nv_bfloat16>::value ? pack_bf16x2(v.x, v.y) : pack_f16x2(v.x, v.y);
      if constexpr (VEC) {
        w[i] = two;
      } else {
        w[0] = two & 0xFFFFu;
        w[1] = two >> 16;
      }
    }
  }
  __device__ __forceinline__ void store(T* p, bool both) const {
    if constexpr (VEC) {
      __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<uint32_t*>(p) = w[0];
      if (both) reinterpret_cast<uint32_t*>(p)[1] = w[1];
    } else {
      *reinterpret_cast<unsigned short*>(p) = static_cast<unsigned short>(w[0]);
      if (both) reinterpret_cast<unsigned short*>(p)[1] = static_cast<unsigned short>(w[1]);
    }
  }
};

// Where element e of A or B stands in shared memory: a lane's 8 elements as two planes of 4, each read without bank
// conflicts by 16-byte loads
template <int N>
__device__ __forceinline__ int term_slot(int e, int nvec) {
  if constexpr (N == 8) return ((e >> 2 & 1) * nvec + (e >> 3)) * 4 + (e & 3);
  return e;
}
template <int N>
__device__ __forceinline__ void term_load(const float* s, int vec, int nvec, float2 (&t)[N / 2]) {
  if constexpr (N == 2) {
    t[0] = *reinterpret_cast<const float2*>(s + 2 * vec);
  } else {
#pragma unroll
    for (int h = 0; h < N / 4; ++h) {
      const float4 v = *reinterpret_cast<const float4*>(s + (h * nvec + vec) * 4);
      t[2 * h] = make_float2(v.x, v.y);
      t[2 * h + 1] = make_float2(v.z, v.w);
    }
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// the row's sum / maximum over its W warps (W > 1: the CTA is one row's; slots alternate, so one barrier each)
__device__ __forceinline__ float row_add(float v, int warps, float* slots, int& turn) {
  v = warp_sum(v);
  if (warps == 1) return v;
  float* s = slots + (turn ^= 1) * kNormMaxWarps;
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
  for (int i = 1; i < warps; ++i) v += s[i];
  return v;
}
__device__ __forceinline__ uint32_t row_most(uint32_t v, int warps, float* slots, int& turn) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (warps == 1) return v;
  uint32_t* s = reinterpret_cast<uint32_t*>(slots + (turn ^= 1) * kNormMaxWarps);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
  for (int i = 1; i < warps; ++i) v = max(v, s[i]);
  return v;
}

template <typename T, bool VEC, int V, int MODE>
__global__ void __launch_bounds__(kNormMaxWarps * 32) norm_rows_kernel(const __grid_constant__ NormParams p) {
  using P = Piece<T, VEC>;
  constexpr int N = P::N, H = N / 2;
  extern __shared__ __align__(16) float terms[];
  __shared__ float slots[2 * kNormMaxWarps];
  const int W = p.warps, L = 32 * W;
  const int group = threadIdx.x / L, at = threadIdx.x % L, groups = blockDim.x / L;
  const int room = p.nvec * N;
  const float *sa = terms, *sb = terms + room;
  int turn = 0;
  int64_t held = -1;                                        // the entry whose A and B are in shared memory
  const int64_t tasks = p.entries * p.chunks;
  if (MODE != NORM_ROWS) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");     // a product waits for this kernel's end itself
  for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int64_t e = task / p.chunks, r0 = (task - e * p.chunks) * p.chunk, r1 = min(r0 + p.chunk, p.rows);
    if (MODE != QUANT_CODES && p.affine && held != (p.modulated ? e : 0)) {
      if (held >= 0) __syncthreads();
      held = p.modulated ? e : 0;
      for (int i = threadIdx.x; i < room; i += blockDim.x) {
        float a = 0.f, b = 0.f;
        if (i < p.width) {
          a = p.weight.p ? term_at(p.weight.p, p.weight.dtype, i) : 1.f;
          b = p.bias.p ? term_at(p.bias.p, p.bias.dtype, i) : 0.f;
        }
        if (i < p.width && p.scale.p) {
          const float s = 1.f + term_at(p.scale.p, p.scale.dtype, e * p.scale.stride + i);
          a *= s;
          b *= s;
        }
        if (i < p.width && p.shift.p) b += term_at(p.shift.p, p.shift.dtype, e * p.shift.stride + i);
        const int slot = term_slot<N>(i, p.nvec);
        terms[slot] = a;
        terms[room + slot] = b;
      }
      __syncthreads();
    }
    for (int64_t r = r0 + group; r < r1; r += groups) {
      const T* x = static_cast<const T*>(p.x) + e * p.xs[0] + r * p.xs[1];
      P v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int vec = at + i * L;
        if (vec < p.nvec) v[i].load(x + vec * N, N > 2 || 2 * vec + 1 < p.width);
        else v[i].clear();
      }
      const int64_t row = e * p.rows + r;
      float mean = 0.f, rstd = 1.f;
      if (MODE != QUANT_CODES) {
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int h = 0; h < H; ++h) sum = add2(sum, v[i].pair(h));
        mean = row_add(sum.x + sum.y, W, slots, turn) * p.inv_width;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i].packed();
        float2 ss = make_float2(0.f, 0.f);
        const float2 m2 = make_float2(mean, mean);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (at + i * L < p.nvec) {
#pragma unroll
            for (int h = 0; h < H; ++h) {
              float2 d = sub2(v[i].pair(h), m2);
              if (N == 2 && 2 * (at + i * L) + 1 >= p.width) d.y = 0.f;
              ss = fma2(d, d, ss);
            }
          }
        }
        rstd = rsqrtf(row_add(ss.x + ss.y, W, slots, turn) * p.inv_width + p.eps);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i].packed();
        if (at == 0) {
          if (p.mean) p.mean[row] = mean;
          if (p.rstd) p.rstd[row] = rstd;
        }
      }
      const float2 m2 = make_float2(mean, mean), r2 = make_float2(rstd, rstd);
      auto result = [&](int i, int vec, float2 (&y)[H]) {
        float2 a[H], b[H];
        if (p.affine) {
          term_load<N>(sa, vec, p.nvec, a);
          term_load<N>(sb, vec, p.nvec, b);
        }
#pragma unroll
        for (int h = 0; h < H; ++h) {
          y[h] = mul2(sub2(v[i].pair(h), m2), r2);
          if (p.affine) y[h] = fma2(y[h], a[h], b[h]);
        }
      };
      if (MODE == NORM_ROWS) {
        T* out = static_cast<T*>(p.out) + e * p.os[0] + r * p.os[1];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int vec = at + i * L;
          if (vec < p.nvec) {
            float2 y[H];
            result(i, vec, y);
#pragma unroll
            for (int h = 0; h < H; ++h) v[i].set(h, y[h]);
            v[i].store(out + vec * N, N > 2 || 2 * vec + 1 < p.width);
          }
        }
      } else {
        // a norm's results stay in float32 until the row's largest is known
        float2 y[MODE == NORM_CODES ? V : 1][H];
        uint32_t top = 0;             // as bits: of magnitudes they are ordered, NaN above infinity
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int vec = at + i * L;
          if (vec < p.nvec) {
            if (MODE == NORM_CODES) result(i, vec, y[MODE == NORM_CODES ? i : 0]);
#pragma unroll
            for (int h = 0; h < H; ++h) {
              const float2 t = MODE == NORM_CODES ? y[MODE == NORM_CODES ? i : 0][h] : v[i].pair(h);
              top = max(top, __float_as_uint(t.x) & 0x7FFFFFFFu);
              if (N > 2 || 2 * vec + 1 < p.width) top = max(top, __float_as_uint(t.y) & 0x7FFFFFFFu);
            }
          }
        }
        top = row_most(top, W, slots, turn);
        if (MODE == QUANT_CODES) {
#pragma unroll
          for (int i = 0; i < V; ++i) v[i].packed();
        }
        // a row with a NaN or an infinity has no codes: its scale is NaN, and with it what is made of it
        const float most = top >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : fmaxf(__uint_as_float(top), kLeastTop);
        const float by = __fdiv_rn(127.f, most);
        if (at == 0) p.scales[row] = __fdiv_rn(most, 127.f);
        int8_t* codes = p.codes + row * p.pitch;
        const float2 by2 = make_float2(by, by);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int vec = at + i * L;
          if (vec < p.nvec) {
            uint32_t c[2 * H];
#pragma unroll
            for (int h = 0; h < H; ++h) {
              // rounded to float32 by the product and to an integer by the sum: two roundings, as the definition has them
              // (elements of half the largest stand on a border; a paired sum would be fused with the paired product)
              const float2 z = mul2(MODE == NORM_CODES ? y[MODE == NORM_CODES ? i : 0][h] : v[i].pair(h), by2);
              c[2 * h] = __float_as_uint(__fadd_rn(z.x, kRoundMagic));
              c[2 * h + 1] = __float_as_uint(__fadd_rn(z.y, kRoundMagic));
            }
            if constexpr (N == 2) {             // an odd row's last store reaches into the pitch
              *reinterpret_cast<unsigned short*>(codes + 2 * vec) = static_cast<unsigned short>(__byte_perm(c[0], c[1], 0x0040));
            } else {
              uint32_t w[N / 4];
#pragma unroll
              for (int k = 0; k < N / 4; ++k)
                w[k] = __byte_perm(__byte_perm(c[4 * k], c[4 * k + 1], 0x0040), __byte_perm(c[4 * k + 2], c[4 * k + 3], 0x0040),
                                   0x5410);
              if constexpr (N == 8) *reinterpret_cast<uint2*>(codes + vec * 8) = make_uint2(w[0], w[1]);
              else *reinterpret_cast<uint32_t*>(codes + vec * 4) = w[0];
            }
          }
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ backward
// A thread keeps its columns: C vectors of them, over R rows at a time, so that the columns' sums P = sum dy u and
// Q = sum dy stay in registers over all of the CTA's rows; the rows' two sums go over the CTA.
//   g = dy A,  dx = rstd (g - mean(g) - u mean(g u))
// The parts' P and Q are added in order by norm_terms_kernel.  HBM bounds it: 6 bytes per 16-bit element.
struct NormBackParams {
  const void *dy, *x;
  int64_t gs[2], xs[2];
  void* dx;
  int64_t os[2];
  const float *mean, *rstd;
  int64_t entries, rows;
  int width, nvec;
  int64_t chunk, chunks;
  float inv_width;
  bool sums, affine;                        // sums: P and Q are wanted
  TermView weight, scale;
  float* part;                              // [entry * chunks][2][width]
};

// RELOAD: rows too wide for the registers are read again (from L2) once their sums are known.
template <typename T, bool VEC, int C, int R, bool RELOAD>
__global__ void __launch_bounds__(512) norm_back_kernel(const __grid_constant__ NormBackParams p) {
  using P = Piece<T, VEC>;
  constexpr int N = P::N, H = N / 2, HELD = RELOAD ? 1 : C;
  __shared__ float slots[2][16][2 * R];
  extern __shared__ __align__(16) float gain[];          // A, as term_slot() has it
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, L = blockDim.x;
  int turn = 0;
  const int64_t e = blockIdx.x / p.chunks, c0 = blockIdx.x - e * p.chunks;
  const int64_t r0 = c0 * p.chunk, r1 = min(r0 + p.chunk, p.rows);
  if (p.affine) {
    for (int i = threadIdx.x; i < p.nvec * N; i += L) {
      float t = i >= p.width ? 0.f : p.weight.p ? term_at(p.weight.p, p.weight.dtype, i) : 1.f;
      if (i < p.width && p.scale.p) t *= 1.f + term_at(p.scale.p, p.scale.dtype, e * p.scale.stride + i);
      gain[term_slot<N>(i, p.nvec)] = t;
    }
    __syncthreads();
  }
  float2 sp[C][H], sq[C][H];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int h = 0; h < H; ++h) sp[c][h] = sq[c][h] = make_float2(0.f, 0.f);
  auto gains = [&](int vec, float2 (&a)[H]) {
#pragma unroll
    for (int h = 0; h < H; ++h) a[h] = make_float2(1.f, 1.f);
    if (p.affine) term_load<N>(gain, vec, p.nvec, a);
  };
  const T* dy = static_cast<const T*>(p.dy) + e * p.gs[0];
  const T* x = static_cast<const T*>(p.x) + e * p.xs[0];
  T* dx = static_cast<T*>(p.dx) + e * p.os[0];
  for (int64_t r = r0; r < r1; r += R) {
    P vg[R][HELD], vx[R][HELD];
    float mean[R], rstd[R];
    auto fetch = [&](int k, int c, int to) {
      const int vec = threadIdx.x + c * L;
      if (r + k < r1 && vec < p.nvec) {
        const bool both = N > 2 || 2 * vec + 1 < p.width;
        vg[k][to].load(dy + (r + k) * p.gs[1] + vec * N, both);
        vx[k][to].load(x + (r + k) * p.xs[1] + vec * N, both);
      } else {
        vg[k][to].clear();
        vx[k][to].clear();
      }
    };
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if (!RELOAD) {
#pragma unroll
        for (int c = 0; c < C; ++c) fetch(k, c, c);
      }
      const bool in = r + k < r1;
      mean[k] = in ? __ldg(p.mean + e * p.rows + r + k) : 0.f;
      rstd[k] = in ? __ldg(p.rstd + e * p.rows + r + k) : 0.f;
    }
    float2 s0[R], s1[R];
#pragma unroll
    for (int k = 0; k < R; ++k) s0[k] = s1[k] = make_float2(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int vec = threadIdx.x + c * L, at = RELOAD ? 0 : c;
      if (vec >= p.nvec) break;
      float2 a[H];
      gains(vec, a);
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (RELOAD) fetch(k, c, 0);
        const float2 r2 = make_float2(rstd[k], rstd[k]), m2 = make_float2(mean[k], mean[k]);
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const float2 d = vg[k][at].pair(h), u = mul2(sub2(vx[k][at].pair(h), m2), r2), g = mul2(d, a[h]);
          sq[c][h] = add2(sq[c][h], d);
          sp[c][h] = fma2(d, u, sp[c][h]);
          s0[k] = add2(s0[k], g);
          s1[k] = fma2(g, u, s1[k]);
        }
        vg[k][at].packed();
        vx[k][at].packed();
      }
    }
    turn ^= 1;
    float sum[2 * R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      sum[2 * k] = warp_sum(s0[k].x + s0[k].y);
      sum[2 * k + 1] = warp_sum(s1[k].x + s1[k].y);
    }
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < 2 * R; ++k) slots[turn][warp][k] = sum[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2 * R; ++k) {
      sum[k] = slots[turn][0][k];
      for (int w = 1; w < warps; ++w) sum[k] += slots[turn][w][k];
      sum[k] *= p.inv_width;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int vec = threadIdx.x + c * L, at = RELOAD ? 0 : c;
      if (vec >= p.nvec) break;
      float2 a[H];
      gains(vec, a);
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (r + k >= r1) break;
        if (RELOAD) fetch(k, c, 0);
        const float2 r2 = make_float2(rstd[k], rstd[k]), m2 = make_float2(mean[k], mean[k]);
        const float2 g0 = make_float2(sum[2 * k], sum[2 * k]), g1 = make_float2(-sum[2 * k + 1], -sum[2 * k + 1]);
        P o;
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const float2 u = mul2(sub2(vx[k][at].pair(h), m2), r2), g = mul2(vg[k][at].pair(h), a[h]);
          o.set(h, mul2(fma2(u, g1, sub2(g, g0)), r2));
        }
        o.store(dx + (r + k) * p.os[1] + vec * N, N > 2 || 2 * vec + 1 < p.width);
      }
    }
  }
  if (p.sums) {
    float* part = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.width;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const int i = (threadIdx.x + c * L) * N + 2 * h;
        if (i < p.width) {
          part[i] = sp[c][h].x;
          part[p.width + i] = sq[c][h].x;
          if (i + 1 < p.width) {
            part[i + 1] = sp[c][h].y;
            part[p.width + i + 1] = sq[c][h].y;
          }
        }
      }
  }
}

struct NormTermsParams {
  const float* part;
  int64_t entries, chunks;
  int width;
  TermView weight, bias, scale;             // scale: of the modulation
  void *dweight, *dbias, *dscale, *dshift;
  int weight_dtype, bias_dtype, scale_dtype, shift_dtype;
};

__device__ __forceinline__ void term_store(void* p, int dtype, int64_t i, float v) {
  if (dtype == HTRC_LAYER_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == HTRC_LAYER_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// 32 columns per CTA: an entry's parts in 32 interleaved sums and those in order, then the entries in order
__global__ void __launch_bounds__(1024) norm_terms_kernel(const __grid_constant__ NormTermsParams p) {
  __shared__ float part[2][32][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + lane;
  const bool in = i < p.width;
  const float w = in && p.weight.p ? term_at(p.weight.p, p.weight.dtype, i) : 1.f;
  const float b = in && p.bias.p ? term_at(p.bias.p, p.bias.dtype, i) : 0.f;
  float dw = 0.f, db = 0.f;
  for (int64_t e = 0; e < p.entries; ++e) {
    float sp = 0.f, sq = 0.f;
    if (in) {
      const float* src = p.part + e * p.chunks * 2 * p.width + i;
      for (int64_t c = row; c < p.chunks; c += 32) {
        sp += src[c * 2 * p.width];
        sq += src[c * 2 * p.width + p.width];
      }
    }
    part[0][row][lane] = sp;
    part[1][row][lane] = sq;
    __syncthreads();
    if (row == 0 && in) {
      sp = sq = 0.f;
      for (int k = 0; k < 32; ++k) {
        sp += part[0][k][lane];
        sq += part[1][k][lane];
      }
      const float s = p.scale.p ? 1.f + term_at(p.scale.p, p.scale.dtype, e * p.scale.stride + i) : 1.f;
      dw = fmaf(sp, s, dw);
      db = fmaf(sq, s, db);
      if (p.dscale) term_store(p.dscale, p.scale_dtype, e * p.width + i, fmaf(sp, w, sq * b));
      if (p.dshift) term_store(p.dshift, p.shift_dtype, e * p.width + i, sq);
    }
    __syncthreads();
  }
  if (row == 0 && in) {
    if (p.dweight) term_store(p.dweight, p.weight_dtype, i, dw);
    if (p.dbias) term_store(p.dbias, p.bias_dtype, i, db);
  }
}

// ------------------------------------------------------------------------------------------------ host
bool float_type(int t) { return t == HTRC_LAYER_F32 || t == HTRC_LAYER_BF16 || t == HTRC_LAYER_F16; }
int type_size(int t) { return t == HTRC_LAYER_F32 ? 4 : 2; }

constexpr int64_t kMaxRows = int64_t(1) << 31;

int rows_validate(int64_t batch, int64_t tokens, int width, int dtype) {
  if (!float_type(dtype) || batch < 0 || tokens < 0 || width < 1) return HTRC_ERR_ARG;
  if (width > HTRC_NORM_MAX_WIDTH) return HTRC_ERR_UNSUPPORTED;
  if (tokens > 0 && batch >= kMaxRows / tokens) return HTRC_ERR_UNSUPPORTED;
  return HTRC_OK;
}

int norm_validate(const HtrcNormArgs* a) {
  if (a == nullptr) return HTRC_ERR_ARG;
  const int rc = rows_validate(a->batch, a->tokens, a->width, a->dtype);
  if (rc != HTRC_OK) return rc;
  if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return HTRC_ERR_ARG;
  if (!float_type(a->weight_dtype) || !float_type(a->bias_dtype) || !float_type(a->scale_dtype) || !float_type(a->shift_dtype))
    return HTRC_ERR_ARG;
  return HTRC_OK;
}

bool rows16(const void* p, const int64_t* s, int es) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] * es % 16 == 0 && s[1] * es % 16 == 0;
}

// Entries and rows of a launch, and how a tensor's (batch, token) strides step over them: one entry where neither terms
// nor strides tell the batch's entries apart.
struct RowShape {
  int64_t entries, rows;
  int kind;                                 // 0: as they are, 1: one entry of evenly spaced rows, 2: one of single rows
  RowShape(int64_t batch, int64_t tokens, bool modulated, std::initializer_list<const int64_t*> strides) {
    bool even = true;
    for (const int64_t* s : strides) even = even && (batch <= 1 || s[0] == tokens * s[1]);
    kind = modulated ? 0 : even ? 1 : tokens == 1 ? 2 : 0;
    entries = kind ? 1 : batch;
    rows = kind ? batch * tokens : tokens;
  }
  void set(const int64_t* s, int64_t (&to)[2]) const {
    to[0] = kind ? 0 : s[0];
    to[1] = kind == 2 ? s[0] : s[1];
  }
};

template <typename T, bool VEC, int MODE>
int norm_launch(NormParams& p, cudaStream_t st) {
  constexpr int N = Piece<T, VEC>::N;
  p.nvec = (p.width + N - 1) / N;
  const int64_t rows = p.entries * p.rows;
  int w = 1;
  while (w < kNormMaxWarps && p.nvec > 32 * w * (VEC ? 8 : 4)) w *= 2;
  // few rows: more warps to each, as long as a lane has more than two pieces
  while (w < kNormMaxWarps && p.nvec > 32 * w * 2 && rows * w * 2 <= 4 * sm_count()) w *= 2;
  p.warps = w;
  const int threads = w > 1 ? 32 * w : kNormThreads, groups = threads / (32 * w);
  const size_t smem = MODE != QUANT_CODES && p.affine ? static_cast<size_t>(p.nvec) * N * 2 * sizeof(float) : 0;
  const int resident = std::max<int>(1, std::min<int64_t>(MODE == NORM_CODES ? 512 / threads : 1024 / threads,
                                                          smem > 0 ? 220 * 1024 / (smem + 1024) : 32));
  const int64_t ctas = static_cast<int64_t>(sm_count()) * resident;
  p.chunks = std::max<int64_t>(1, std::min((p.rows + groups - 1) / groups, ctas / std::max<int64_t>(1, p.entries)));
  p.chunk = (p.rows + p.chunks - 1) / p.chunks;
  p.chunks = (p.rows + p.chunk - 1) / p.chunk;
  const unsigned grid = static_cast<unsigned>(std::min(p.entries * p.chunks, ctas));
  const int per = (p.nvec + 32 * w - 1) / (32 * w);
  auto go = [&](auto kernel) {
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
      return HTRC_ERR_CUDA;
    kernel<<<grid, threads, smem, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
  };
  if constexpr (VEC) {
    if (per <= 2) return go(norm_rows_kernel<T, VEC, 2, MODE>);
    if (per <= 4) return go(norm_rows_kernel<T, VEC, 4, MODE>);
    return go(norm_rows_kernel<T, VEC, 8, MODE>);
  } else {
    if (per <= 4) return go(norm_rows_kernel<T, VEC, 4, MODE>);
    return go(norm_rows_kernel<T, VEC, 16, MODE>);
  }
}

template <int MODE>
int norm_types(NormParams& p, int dtype, bool vec, cudaStream_t st) {
  if (dtype == HTRC_LAYER_F32) return vec ? norm_launch<float, true, MODE>(p, st) : norm_launch<float, false, MODE>(p, st);
  if (dtype == HTRC_LAYER_BF16)
    return vec ? norm_launch<__nv_bfloat16, true, MODE>(p, st) : norm_launch<__nv_bfloat16, false, MODE>(p, st);
  return vec ? norm_launch<__half, true, MODE>(p, st) : norm_launch<__half, false, MODE>(p, st);
}

int norm_forward(const HtrcNormArgs* a, cudaStream_t st) {
  int rc = norm_validate(a);
  if (rc != HTRC_OK) return rc;
  const bool codes = a->codes != nullptr;
  const bool some = a->batch * a->tokens > 0;
  if (some && (a->x == nullptr || (codes ? a->scales == nullptr : a->out == nullptr))) return HTRC_ERR_ARG;
  if (codes && (a->codes_pitch < a->width || a->codes_pitch % 16 || reinterpret_cast<uintptr_t>(a->codes) % 16)) return HTRC_ERR_ARG;
  if (!device_is_b200()) return HTRC_ERR_DEVICE;
  if (!some) return HTRC_OK;
  NormParams p{};
  p.x = a->x;
  p.out = a->out;
  p.codes = a->codes;
  p.pitch = a->codes_pitch;
  p.scales = a->scales;
  p.mean = a->mean;
  p.rstd = a->rstd;
  p.width = a->width;
  p.eps = a->eps;
  p.inv_width = 1.0f / static_cast<float>(a->width);
  p.weight = TermView{a->weight, 0, a->weight_dtype};
  p.bias = TermView{a->bias, 0, a->bias_dtype};
  p.scale = TermView{a->scale, a->scale_stride, a->scale_dtype};
  p.shift = TermView{a->shift, a->shift_stride, a->shift_dtype};
  p.modulated = a->scale || a->shift;
  p.affine = p.modulated || a->weight || a->bias;
  const int es = type_size(a->dtype);
  bool vec = a->width * es % 16 == 0 && rows16(a->x, a->x_stride, es);
  if (!codes) vec = vec && rows16(a->out, a->out_stride, es);
  const RowShape shape = codes ? RowShape(a->batch, a->tokens, p.modulated, {a->x_stride})
                               : RowShape(a->batch, a->tokens, p.modulated, {a->x_stride, a->out_stride});
  p.entries = shape.entries;
  p.rows = shape.rows;
  shape.set(a->x_stride, p.xs);
  if (!codes) shape.set(a->out_stride, p.os);
  return codes ? norm_types<NORM_CODES>(p, a->dtype, vec, st) : norm_types<NORM_ROWS>(p, a->dtype, vec, st);
}

int64_t norm_back_chunks(int64_t entries, int64_t rows, int64_t* chunk) {
  // two CTAs per SM, and no chunk of less than four rows
  const int64_t want = std::max<int64_t>(1, 2 * sm_count() / std::max<int64_t>(1, entries));
  const int64_t chunks = std::max<int64_t>(1, std::min(want, (rows + 3) / 4));
  *chunk = std::max<int64_t>(1, (rows + chunks - 1) / chunks);
  return std::max<int64_t>(1, (rows + *chunk - 1) / *chunk);
}

bool norm_sums(const HtrcNormArgs* a) { return a->dweight || a->dbias || a->dscale || a->dshift; }

RowShape norm_back_shape(const HtrcNormArgs* a) {
  return RowShape(a->batch, a->tokens, a->scale || a->shift, {a->dy_stride, a->x_stride, a->dx_stride});
}

template <typename T, bool VEC>
int norm_back_launch(NormBackParams& p, unsigned grid, cudaStream_t st) {
  constexpr int N = Piece<T, VEC>::N;
  p.nvec = (p.width + N - 1) / N;
  const int per = (p.nvec + 511) / 512;
  const size_t smem = p.affine ? static_cast<size_t>(p.nvec) * N * sizeof(float) : 0;
  auto go = [&](auto kernel, int c) {
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
      return HTRC_ERR_CUDA;
    kernel<<<grid, ((p.nvec + c - 1) / c + 31) / 32 * 32, smem, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
  };
  if constexpr (VEC) {
    if (per <= 1) return go(norm_back_kernel<T, VEC, 1, 4, false>, 1);
    if (per <= 2) return go(norm_back_kernel<T, VEC, 2, 2, false>, 2);
    if constexpr (N == 8) return go(norm_back_kernel<T, VEC, 4, 1, true>, 4);
    else return per <= 4 ? go(norm_back_kernel<T, VEC, 4, 1, true>, 4) : go(norm_back_kernel<T, VEC, 8, 1, true>, 8);
  } else {
    if (per <= 2) return go(norm_back_kernel<T, VEC, 2, 4, false>, 2);
    if (per <= 4) return go(norm_back_kernel<T, VEC, 4, 2, false>, 4);
    return go(norm_back_kernel<T, VEC, 16, 1, true>, 16);
  }
}

int norm_back_size(const HtrcNormArgs* a, size_t* bytes) {
  if (bytes == nullptr) return HTRC_ERR_ARG;
  const int rc = norm_validate(a);
  if (rc != HTRC_OK) return rc;
  int64_t chunk;
  const RowShape shape = norm_back_shape(a);
  const int64_t chunks = norm_back_chunks(shape.entries, shape.rows, &chunk);
  *bytes = norm_sums(a) ? static_cast<size_t>(shape.entries) * chunks * 2 * a->width * sizeof(float) : 0;
  return HTRC_OK;
}

int norm_backward(const HtrcNormArgs* a, cudaStream_t st) {
  size_t need = 0;
  int rc = norm_back_size(a, &need);
  if (rc != HTRC_OK) return rc;
  const bool some = a->batch * a->tokens > 0;
  if (some && (!a->x || !a->dy || !a->dx || !a->mean || !a->rstd)) return HTRC_ERR_ARG;
  if ((a->dscale && !a->scale) || (a->dshift && !a->shift) || (a->dweight && !a->weight) || (a->dbias && !a->bias))
    return HTRC_ERR_ARG;
  if (!device_is_b200()) return HTRC_ERR_DEVICE;
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16))
    return HTRC_ERR_WORKSPACE;
  if (a->batch == 0 && !norm_sums(a)) return HTRC_OK;
  NormBackParams p{};
  p.dy = a->dy;
  p.x = a->x;
  p.dx = a->dx;
  const RowShape shape = norm_back_shape(a);
  p.entries = shape.entries;
  p.rows = shape.rows;
  shape.set(a->dy_stride, p.gs);
  shape.set(a->x_stride, p.xs);
  shape.set(a->dx_stride, p.os);
  p.mean = a->mean;
  p.rstd = a->rstd;
  p.width = a->width;
  p.inv_width = 1.0f / static_cast<float>(a->width);
  p.weight = TermView{a->weight, 0, a->weight_dtype};
  p.scale = TermView{a->scale, a->scale_stride, a->scale_dtype};
  p.sums = norm_sums(a);
  p.affine = a->weight || a->scale;
  p.part = static_cast<float*>(a->workspace);
  p.chunks = norm_back_chunks(p.entries, p.rows, &p.chunk);
  if (p.entries * p.chunks >= kMaxRows) return HTRC_ERR_UNSUPPORTED;
  const unsigned grid = static_cast<unsigned>(p.entries * p.chunks);
  const int es = type_size(a->dtype);
  const bool vec = a->width * es % 16 == 0 && rows16(a->x, a->x_stride, es) && rows16(a->dy, a->dy_stride, es) &&
                   rows16(a->dx, a->dx_stride, es);
  if (grid > 0) {
    if (a->dtype == HTRC_LAYER_F32)
      rc = vec ? norm_back_launch<float, true>(p, grid, st) : norm_back_launch<float, false>(p, grid, st);
    else if (a->dtype == HTRC_LAYER_BF16)
      rc = vec ? norm_back_launch<__nv_bfloat16, true>(p, grid, st) : norm_back_launch<__nv_bfloat16, false>(p, grid, st);
    else
      rc = vec ? norm_back_launch<__half, true>(p, grid, st) : norm_back_launch<__half, false>(p, grid, st);
    if (rc != HTRC_OK) return rc;
  }
  if (p.sums) {
    NormTermsParams t{};
    t.part = p.part;
    t.entries = p.entries;
    t.chunks = p.chunks;
    t.width = a->width;
    t.weight = p.weight;
    t.bias = TermView{a->bias, 0, a->bias_dtype};
    t.scale = p.scale;
    t.dweight = a->dweight;
    t.dbias = a->dbias;
    t.dscale = a->dscale;
    t.dshift = a->dshift;
    t.weight_dtype = a->weight_dtype;
    t.bias_dtype = a->bias_dtype;
    t.scale_dtype = a->scale_dtype;
    t.shift_dtype = a->shift_dtype;
    norm_terms_kernel<<<(a->width + 31) / 32, 1024, 0, st>>>(t);
  }
  return cudaGetLastError() == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
}

}  // namespace

int quantize_rows(const void* x, int dtype, int64_t batch, int64_t tokens, int width, const int64_t* stride, int8_t* codes,
                  int64_t pitch, float* scales, cudaStream_t st) {
  const int rc = rows_validate(batch, tokens, width, dtype);
  if (rc != HTRC_OK) return rc;
  const bool some = batch * tokens > 0;
  if (some && (!x || !codes || !scales || !stride)) return HTRC_ERR_ARG;
  if (some && (pitch < width || pitch % 16 || reinterpret_cast<uintptr_t>(codes) % 16)) return HTRC_ERR_ARG;
  if (!device_is_b200()) return HTRC_ERR_DEVICE;
  if (!some) return HTRC_OK;
  NormParams p{};
  p.x = x;
  p.codes = codes;
  p.pitch = pitch;
  p.scales = scales;
  p.width = width;
  const int es = type_size(dtype);
  const bool vec = static_cast<int64_t>(width) * es % 16 == 0 && rows16(x, stride, es);
  const RowShape shape(batch, tokens, false, {stride});
  p.entries = shape.entries;
  p.rows = shape.rows;
  shape.set(stride, p.xs);
  return norm_types<QUANT_CODES>(p, dtype, vec, st);
}

}  // namespace htrc

extern "C" {

int htrc_norm_forward(const HtrcNormArgs* args, htrc_stream_t stream) {
  return htrc::norm_forward(args, reinterpret_cast<cudaStream_t>(stream));
}

int htrc_norm_workspace_size(const HtrcNormArgs* args, size_t* bytes) { return htrc::norm_back_size(args, bytes); }

int htrc_norm_backward(const HtrcNormArgs* args, htrc_stream_t stream) {
  return htrc::norm_backward(args, reinterpret_cast<cudaStream_t>(stream));
}

int htrc_quantize_rows(const void* x, int32_t dtype, int64_t batch, int64_t tokens, int32_t width, const int64_t* stride,
                       int8_t* codes, int64_t pitch, float* scales, htrc_stream_t stream) {
  return htrc::quantize_rows(x, dtype, batch, tokens, width, stride, codes, pitch, scales,
                             reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
