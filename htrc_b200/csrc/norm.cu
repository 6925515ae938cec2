// Layer norm with a learned affine and a modulation per batch entry, forward and backward, and rows in 8-bit integers
// with a scale each (of a norm's result, or of the rows as they are) for the product in linear8.cu.
//
//   u = (x - mean) rstd,   y = (u weight + bias) (1 + scale) + shift = u A + B
//   codes = rint(y (127 / top)), scales = top / 127, top = max |y| of the row
//
// Forward: a row is read once and stays in registers as it was read, 8 lanes to 16 warps to a row, up to four rows to a lane,
// which share the reading of A and B.  The mean, then the squared deviations from it (no cancellation under a large mean),
// then the result, all float32.  A and B are formed once per batch entry in shared memory.  An entry's CTAs sweep its rows
// together: each with rows of its own far from the others' cost 10 % (129,024 x 2,048: 188 us, 168).
//
// HBM bounds it: 4 bytes per 16-bit element, 3 to 8-bit rows.  129,024 x 2,048 in bfloat16, device time after a rest: plain
// 170 us (6.2 TB/s), modulated 177 (5.9), its 8-bit rows 160 (4.9; issue and 16 warps of 128 registers), 8-bit rows of x
// itself 131 (6.0).
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "../../include/htrc_layer.h"
#include "common.cuh"
#include "kernels.cuh"

namespace htrc {

namespace {

constexpr int kNormThreads = 256;           // of a CTA; of rows that take more: those lanes
constexpr int kNormMaxWarps = 16;           // per row
constexpr int kNormSms = 228 * 1024;        // shared memory of an SM
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
  int width, nvec, lanes;                   // pieces per row, lanes per row (a power of two)
  int64_t chunks;                           // CTAs that share an entry
  float eps, inv_width;
  bool affine, modulated;
  TermView weight, bias, scale, shift;
};

__device__ __forceinline__ float term_at(const void* p, int dtype, int64_t i) {
  if (dtype == HTRC_LAYER_F32) return __ldg(static_cast<const float*>(p) + i);
  if (dtype == HTRC_LAYER_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// How a row's elements are read: 16 bytes at a time, two neighbours by one load (an even width, rows at multiples of two
// elements), or two neighbours by themselves
enum Reads : int { BY_ELEMENT = 0, BY_PAIR = 1, BY_16 = 2 };

// N neighbouring elements as they were read (`both`: the second of two is within the row; it is 0 where not)
template <typename T, int READ>
struct Piece {
  static constexpr int N = READ == BY_16 ? 16 / sizeof(T) : 2, W = READ == BY_16 ? 4 : READ == BY_PAIR ? sizeof(T) / 2 : 2;
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
    if constexpr (READ == BY_16) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (READ == BY_PAIR && sizeof(T) == 4) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = v.x; w[1] = v.y;
    } else if constexpr (READ == BY_PAIR) {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
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
    if constexpr (READ == BY_ELEMENT || sizeof(T) == 4) {
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
      if constexpr (READ != BY_ELEMENT) {
        w[i] = two;
      } else {
        w[0] = two & 0xFFFFu;
        w[1] = two >> 16;
      }
    }
  }
  __device__ __forceinline__ void store(T* p, bool both) const {
    if constexpr (READ == BY_16) {
      __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
    } else if constexpr (READ == BY_PAIR && sizeof(T) == 4) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else if constexpr (READ == BY_PAIR) {
      *reinterpret_cast<uint32_t*>(p) = w[0];
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
// a lane's view of them: piece i of it is `at + i * L`
template <int N>
struct Terms {
  const float *lo, *hi;
  __device__ __forceinline__ Terms(const float* s, int at, int nvec) : lo(s + at * (N == 2 ? 2 : 4)), hi(lo + nvec * 4) {}
  __device__ __forceinline__ void load(int off, float2 (&t)[N / 2]) const {
    if constexpr (N == 2) {
      t[0] = *reinterpret_cast<const float2*>(lo + off * 2);
    } else {
      const float4 v = *reinterpret_cast<const float4*>(lo + off * 4);
      t[0] = make_float2(v.x, v.y);
      t[1] = make_float2(v.z, v.w);
      if constexpr (N == 8) {
        const float4 u = *reinterpret_cast<const float4*>(hi + off * 4);
        t[2] = make_float2(u.x, u.y);
        t[3] = make_float2(u.z, u.w);
      }
    }
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

__device__ __forceinline__ float larger(float a, float b) {      // NaN if either is
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// R rows' sums (or maxima) over their L lanes.  L > 32: through the group's slots, which alternate, so that one barrier of
// the group (of its L threads) does for each.
template <int R, bool MOST>
__device__ __forceinline__ void over_lanes(float (&v)[R], int L, int group, float (*slots)[kNormMaxWarps][4], int& turn) {
  auto step = [&](int d) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const float o = __shfl_xor_sync(0xffffffffu, v[k], d);
      v[k] = MOST ? larger(v[k], o) : v[k] + o;
    }
  };
  if (L >= 32) step(16);
  if (L >= 16) step(8);
  step(4);
  step(2);
  step(1);
  if (L <= 32) return;
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int k = 0; k < R; ++k) slots[turn][threadIdx.x >> 5][k] = v[k];
  }
  named_bar_sync(1 + group, L);
  const int warps = L >> 5, first = group * warps;
#pragma unroll
  for (int k = 0; k < R; ++k) v[k] = slots[turn][first][k];
  for (int i = 1; i < warps; ++i) {
#pragma unroll
    for (int k = 0; k < R; ++k) v[k] = MOST ? larger(v[k], slots[turn][first + i][k]) : v[k] + slots[turn][first + i][k];
  }
}

// Rows to a lane of V pieces of each.  Two 16-bit rows of several warps share the reading of A and B (16,384 x 5,120: 85 us one by
// one, 66 so; a warp's: 129,024 x 2,048 171 and 190; float32, 32,768 x 1,536: 69 and 73).  A norm's 8-bit rows, whose results stay
// in registers, do better one by one with more warps (16 bits, 65,536 x 1,024: 57 us by two, 50 so; 100,000 x 512: 52 by four,
// 42; float32, 65,536 x 512: 34 by four, 37).
template <typename T, int READ, int V, int LANES, int MODE>
constexpr int rows_of() {
  if (V == 8 && LANES >= 64 && MODE == NORM_ROWS && READ == BY_16 && sizeof(T) == 2) return 2;
  if ((V == 2 || V == 4) && MODE == NORM_CODES && READ == BY_16 && sizeof(T) == 2) return 1;
  return V >= 8 ? 1 : V == 1 ? 4 : 8 / V;
}
// (-Xptxas -v: 8-bit rows from two and four 16-byte pieces of 16-bit elements spill 32 bytes in their 64 and 80 registers, from
// eight 52 to 64 in 128; results of sixteen unaligned pieces 156 in 80)
template <typename T, int READ, int V, int MODE>
constexpr int registers_of() {
  if (MODE == QUANT_CODES) return 64;
  if (MODE == NORM_CODES) return READ != BY_16 || sizeof(T) == 4 || V == 1 || V == 8 ? 128 : V == 4 ? 80 : 64;
  return V == 8 ? 128 : 80;
}

// LANES: lanes to a row, or 0 for any number (p.lanes); fixed ones have the pieces' offsets in the instructions (8,192 x
// 8,192, a row at a time: 61 us, 79 by runtime offsets).  Registers: eight pieces of a row want the 128 that 16 warps leave (129,024 x 2,048 in
// 80 of them, spilling: 322 us); fewer pieces, and rows that only look for their largest, do better with more warps.
template <typename T, int READ, int V, int LANES, int MODE>
__global__ void __maxnreg__((registers_of<T, READ, V, MODE>())) norm_rows_kernel(const __grid_constant__ NormParams p) {
  using P = Piece<T, READ>;
  constexpr int N = P::N, H = N / 2, R = rows_of<T, READ, V, LANES, MODE>();
  extern __shared__ __align__(16) float terms[];
  __shared__ float slots[2][kNormMaxWarps][4];
  const int L = LANES ? LANES : p.lanes, at = threadIdx.x & (L - 1), G = blockDim.x / L, group = threadIdx.x / L;
  const int room = p.nvec * N;
  const Terms<N> ta(terms, at, p.nvec), tb(terms + room, at, p.nvec);
  // a fixed number of lanes: V is the least power of two that holds a row, so that half of the pieces are whole
  auto has = [&](int i) { return (LANES && i < V / 2) || at + i * L < p.nvec; };
  auto two = [&](int i) { return READ != BY_ELEMENT || 2 * (at + i * L) + 1 < p.width; };
  int turn = 0;
  int64_t held = -1;                                        // the entry whose A and B are in shared memory
  const int64_t tasks = p.entries * p.chunks;
  if (MODE != NORM_ROWS) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");     // a product waits for this kernel's end itself
  for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    // an entry's CTAs sweep its rows together: neighbouring CTAs at neighbouring rows
    // (fewer than 2^31 rows and 2^20 to a step: unsigned 32 bits hold the row after the last)
    const int64_t e = task / p.chunks;
    const uint32_t chunk = static_cast<uint32_t>(task - e * p.chunks), r1 = static_cast<uint32_t>(p.rows);
    const uint32_t r0 = chunk * G * R, step = static_cast<uint32_t>(p.chunks) * G * R;
    // row r + group, and what leads from it to the lane's other rows and to the next step's
    const T* x = static_cast<const T*>(p.x) + e * p.xs[0] + (static_cast<int64_t>(r0) + group) * p.xs[1] + at * N;
    const int64_t x_step = step * p.xs[1], x_row = G * p.xs[1];
    auto fetch = [&](P (&v)[R][V], uint32_t r) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const T* from = x + k * x_row;
        const bool in = r + k * G + group < r1;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[k][i].clear();
          if (in && has(i)) v[k][i].load(from + i * L * N, two(i));
        }
      }
    };
    P v[R][V];
    fetch(v, r0);
    x += x_step;
    if (MODE != QUANT_CODES && p.affine && held != (p.modulated ? e : 0)) {
      if (held >= 0) __syncthreads();
      held = p.modulated ? e : 0;
      for (int i = threadIdx.x; i < room; i += blockDim.x) {
        float a = 0.f, b = 0.f;
        if (i < p.width) {
          a = p.weight.p ? term_at(p.weight.p, p.weight.dtype, i) : 1.f;
          b = p.bias.p ? term_at(p.bias.p, p.bias.dtype, i) : 0.f;
          if (p.scale.p) {
            const float s = 1.f + term_at(p.scale.p, p.scale.dtype, e * p.scale.stride + i);
            a *= s;
            b *= s;
          }
          if (p.shift.p) b += term_at(p.shift.p, p.shift.dtype, e * p.shift.stride + i);
        }
        const int slot = term_slot<N>(i, p.nvec);
        terms[slot] = a;
        terms[room + slot] = b;
      }
      __syncthreads();
    }
    const int64_t row0 = e * p.rows + r0 + group;           // in the statistics and among the 8-bit rows
    T* out = static_cast<T*>(p.out) + e * p.os[0] + (static_cast<int64_t>(r0) + group) * p.os[1] + at * N;
    int8_t* codes = p.codes + row0 * p.pitch + at * N;
    for (uint32_t r = r0; r < r1; r += step) {
      if (MODE != NORM_CODES && r > r0) {
        fetch(v, r);
        x += x_step;
      }
      float mean[R], rstd[R];
      if (MODE != QUANT_CODES) {
#pragma unroll
        for (int k = 0; k < R; ++k) {
          float2 sum = make_float2(0.f, 0.f);
          if (r + k * G < r1) {                             // the same for all of the CTA
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
              for (int h = 0; h < H; ++h) sum = add2(sum, v[k][i].pair(h));
          }
          mean[k] = sum.x + sum.y;
#pragma unroll
          for (int i = 0; i < V; ++i) v[k][i].packed();
        }
        over_lanes<R, false>(mean, L, group, slots, turn);
#pragma unroll
        for (int k = 0; k < R; ++k) {
          mean[k] *= p.inv_width;
          float2 ss = make_float2(0.f, 0.f);
          const float2 m2 = make_float2(mean[k], mean[k]);
          if (r + k * G < r1) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              if (has(i)) {
#pragma unroll
                for (int h = 0; h < H; ++h) {
                  float2 d = sub2(v[k][i].pair(h), m2);
                  if (!two(i)) d.y = 0.f;
                  ss = fma2(d, d, ss);
                }
              }
            }
          }
          rstd[k] = ss.x + ss.y;
#pragma unroll
          for (int i = 0; i < V; ++i) v[k][i].packed();
        }
        over_lanes<R, false>(rstd, L, group, slots, turn);
#pragma unroll
        for (int k = 0; k < R; ++k) {
          rstd[k] = rsqrtf(rstd[k] * p.inv_width + p.eps);
          if (at == 0 && r + k * G + group < r1) {
            const int64_t row = row0 + (r - r0) + k * G;
            if (p.mean) p.mean[row] = mean[k];
            if (p.rstd) p.rstd[row] = rstd[k];
          }
        }
      }
      // the results of piece i of every row, which share its A and B
      auto results = [&](int i, auto use) {
        float2 a[H], b[H];
        if (p.affine) {
          ta.load(i * L, a);
          tb.load(i * L, b);
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
          if (r + k * G >= r1) break;
          const float2 m2 = make_float2(mean[k], mean[k]), r2 = make_float2(rstd[k], rstd[k]);
          float2 y[H];
#pragma unroll
          for (int h = 0; h < H; ++h) {
            y[h] = mul2(sub2(v[k][i].pair(h), m2), r2);
            if (p.affine) y[h] = fma2(y[h], a[h], b[h]);
          }
          use(k, y);
        }
      };
      if constexpr (MODE == NORM_ROWS) {
        T* to[R];
        bool in[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
          to[k] = out + k * G * p.os[1];
          in[k] = r + k * G + group < r1;
        }
        out += step * p.os[1];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (has(i)) {
            results(i, [&](int k, float2 (&y)[H]) {
              P o;
#pragma unroll
              for (int h = 0; h < H; ++h) o.set(h, y[h]);
              if (in[k]) o.store(to[k] + i * L * N, two(i));
            });
          }
        }
      } else {
        // a norm's results stay in float32 until the row's largest is known (129,024 x 2,048: 157 us; formed again then: 267)
        float2 y[MODE == NORM_CODES ? R : 1][MODE == NORM_CODES ? V : 1][H];
        float top[R];
#pragma unroll
        for (int k = 0; k < R; ++k) top[k] = 0.f;
        auto most = [&](int k, float2 t, bool both) {
          top[k] = larger(top[k], fabsf(t.x));
          if (both) top[k] = larger(top[k], fabsf(t.y));
        };
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const bool both = two(i);
          if (has(i)) {
            if constexpr (MODE == NORM_CODES) {
              results(i, [&](int k, float2 (&t)[H]) {
#pragma unroll
                for (int h = 0; h < H; ++h) {
                  y[k][i][h] = t[h];
                  most(k, t[h], both);
                }
              });
            } else {
#pragma unroll
              for (int k = 0; k < R; ++k)
#pragma unroll
                for (int h = 0; h < H; ++h) most(k, v[k][i].pair(h), both);
            }
          }
        }
        // the rows as they were read are done with: the next ones arrive while these are quantised
        if (MODE == NORM_CODES) {
          fetch(v, r + step);
          x += x_step;
        }
        over_lanes<R, true>(top, L, group, slots, turn);
        // the lane's rows' factors 127 / top and scales top / 127 by one division in 2 R lanes.  A row with a NaN or an
        // infinity has no codes: its scale is NaN, and with it what is made of it
        float factor[R];
        {
          const int lane = threadIdx.x & 31, which = lane >> 1 & (R - 1), width = L < 32 ? L : 32;
          float full = top[0];
#pragma unroll
          for (int k = 1; k < R; ++k) full = which == k ? top[k] : full;
          full = full <= 3.4028235e38f ? fmaxf(full, kLeastTop) : __uint_as_float(0x7FC00000u);
          const float q = __fdiv_rn(lane & 1 ? full : 127.f, lane & 1 ? 127.f : full);
#pragma unroll
          for (int k = 0; k < R; ++k) factor[k] = __shfl_sync(0xffffffffu, q, 2 * k, width);
          if ((at & 1) && at < 2 * R && r + which * G + group < r1) p.scales[row0 + (r - r0) + which * G] = q;
        }
        int8_t* base = codes;
        codes += step * p.pitch;
#pragma unroll
        for (int k = 0; k < R; ++k) {
          if (r + k * G >= r1) break;
          const float2 by2 = make_float2(factor[k], factor[k]);
          int8_t* to = base + k * G * p.pitch;
          const bool in = r + k * G + group < r1;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            if (MODE == QUANT_CODES) v[k][i].packed();
            if (has(i) && in) {
              uint32_t c[2 * H];
#pragma unroll
              for (int h = 0; h < H; ++h) {
                // rounded to float32 by the product and to an integer by the sum: two roundings, as the definition has
                // them (elements of half the largest stand on a border; a paired sum would be fused with the product)
                float2 z;
                if constexpr (MODE == NORM_CODES) z = mul2(y[k][i][h], by2);
                else z = mul2(v[k][i].pair(h), by2);
                c[2 * h] = __float_as_uint(__fadd_rn(z.x, kRoundMagic));
                c[2 * h + 1] = __float_as_uint(__fadd_rn(z.y, kRoundMagic));
              }
              if constexpr (N == 2) {             // an odd row's last store reaches into the pitch
                *reinterpret_cast<unsigned short*>(to + i * L * N) = static_cast<unsigned short>(__byte_perm(c[0], c[1], 0x0040));
              } else {
                uint32_t w[N / 4];
#pragma unroll
                for (int q = 0; q < N / 4; ++q)
                  w[q] = __byte_perm(__byte_perm(c[4 * q], c[4 * q + 1], 0x0040), __byte_perm(c[4 * q + 2], c[4 * q + 3], 0x0040),
                                     0x5410);
                if constexpr (N == 8) *reinterpret_cast<uint2*>(to + i * L * N) = make_uint2(w[0], w[1]);
                else *reinterpret_cast<uint32_t*>(to + i * L * N) = w[0];
              }
            }
          }
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ backward
//   g = dy A,  dx = rstd (g - mean(g) - u mean(g u)),  P = sum over rows of dy u,  Q = sum over rows of dy
// A thread keeps its columns over all of the CTA's rows, so that their P and Q stay in registers; the rows' two sums go over
// the lanes.  Rows of up to two pieces to a lane of a warp (norm_back_narrow_kernel) need no barrier.  A wider row is the
// whole CTA's (norm_back_ring_kernel): rows arrive in shared memory by bulk copies several stages ahead, since a barrier per
// four rows leaves loads by the threads themselves no time in flight (32,768 x 2,048: 120 us by such loads).  Rows that are
// not 16-byte aligned arrive as the 16-byte pieces that cover them (16,384 x 4,999: 1,062 us by elements, 252 so).  The
// parts' P and Q are added in a fixed order by norm_terms_kernel.
//
// HBM bounds it: 6 bytes per 16-bit element.  32,768 x 2,048 in bfloat16, modulated: 79 us, 5.1 TB/s; the barriers are the
// largest stall.  In float32 133 us, 6.1 TB/s.  Rows to warps and columns to other warps that meet at mbarriers alone, without
// any, took 93 us.
struct NormBackParams {
  const void *dy, *x;
  int64_t gs[2], xs[2];
  void* dx;
  int64_t os[2];
  const float *mean, *rstd;
  int64_t entries, rows;
  int width, nvec;
  int64_t chunks;                           // CTAs that share an entry
  float inv_width;
  bool sums, affine;                        // sums: P and Q are wanted
  int lanes, stages;
  int* status;
  TermView weight, scale;
  float* part;                              // [entry * chunks][2][width]
};

// 8 values over a warp: afterwards lane 4 i' holds one of them, value_of(lane)
__device__ __forceinline__ float warp_sum8(float (&v)[8], int lane) {
#pragma unroll
  for (int n = 4; n; n >>= 1) {
    const bool up = lane & (4 * n);
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, 4 * n);
    }
  }
  float t = v[0];
  t += __shfl_xor_sync(0xffffffffu, t, 2);
  return t + __shfl_xor_sync(0xffffffffu, t, 1);
}
__device__ __forceinline__ int value_of(int lane) { return lane >> 2; }

// rows of a ring's stage with C pieces of each to a thread
template <typename T, int READ>
__host__ __device__ constexpr int ring_rows(int c) {
  return READ == BY_16 ? (c >= 4 ? 1 : 4 / c) : sizeof(T) == 4 ? (c >= 8 ? 1 : 8 / c) : c <= 4 ? 4 : 16 / c;
}
// bytes between the rows of a stage: a row that starts inside a 16-byte piece begins with what is before it there
__host__ __device__ inline uint32_t ring_pitch(uint32_t row_bytes, int read) {
  return read == BY_16 ? row_bytes : (row_bytes + 15 + 15) / 16 * 16;
}

// C pieces of each of R rows to a thread, the CTA one row wide
template <typename T, int READ, int C>
__global__ void __launch_bounds__(512, 1) norm_back_ring_kernel(const __grid_constant__ NormBackParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");     // the sums' kernel waits for this one's end itself
  using P = Piece<T, READ == BY_16 ? BY_16 : BY_PAIR>;        // in registers two elements stand together
  constexpr int N = P::N, H = N / 2, R = ring_rows<T, READ>(C), kStages = 4;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) uint64_t full[kStages];
  __shared__ float slots[2][8][16];
  __shared__ __align__(16) float stats[2][2][4];            // the rows' means and reciprocal deviations
  __shared__ int abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, L = blockDim.x;
  const uint32_t row_bytes = p.width * sizeof(T), pitch = ring_pitch(row_bytes, READ), stage_bytes = 2 * R * pitch;
  float* gain = reinterpret_cast<float*>(ring + p.stages * stage_bytes);       // C > 1: A, as term_slot() has it
  int turn = 0;
  const int64_t e = blockIdx.x / p.chunks, r1 = p.rows, r0 = (blockIdx.x - e * p.chunks) * R, step = p.chunks * R;
  const T* dy = static_cast<const T*>(p.dy) + e * p.gs[0];
  const T* x = static_cast<const T*>(p.x) + e * p.xs[0];
  T* dx = static_cast<T*>(p.dx) + e * p.os[0];
  const uint64_t policy = policy_evict_first();
  auto fill = [&](int s, int64_t r) {
    const int n = static_cast<int>(min(static_cast<int64_t>(R), r1 - r));
    // the 16-byte pieces that cover a row
    auto start = [](const T* row) { return reinterpret_cast<uintptr_t>(row) & ~static_cast<uintptr_t>(READ == BY_16 ? 0 : 15); };
    auto bytes = [&](const T* row) {
      if (READ == BY_16) return row_bytes;
      return static_cast<uint32_t>((reinterpret_cast<uintptr_t>(row) + row_bytes + 15 & ~static_cast<uintptr_t>(15)) - start(row));
    };
    uint32_t all = 2 * n * row_bytes;
    if (READ != BY_16) {
      all = 0;
      for (int k = 0; k < n; ++k) all += bytes(dy + (r + k) * p.gs[1]) + bytes(x + (r + k) * p.xs[1]);
    }
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(&full[s])), "r"(all) : "memory");
    for (int k = 0; k < n; ++k) {
      uint8_t* to = ring + s * stage_bytes + 2 * k * pitch;
      const T *g = dy + (r + k) * p.gs[1], *v = x + (r + k) * p.xs[1];
      bulk_load(to, reinterpret_cast<const void*>(start(g)), bytes(g), &full[s], policy);
      bulk_load(to + pitch, reinterpret_cast<const void*>(start(v)), bytes(v), &full[s], policy);
    }
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], 1);
    abort_flag = 0;
    fence_barrier_init();
    for (int s = 0; s < p.stages && r0 + s * step < r1; ++s) fill(s, r0 + s * step);
  }
  auto gain_of = [&](int i) {
    float t = i >= p.width ? 0.f : p.weight.p ? term_at(p.weight.p, p.weight.dtype, i) : 1.f;
    if (i < p.width && p.scale.p) t *= 1.f + term_at(p.scale.p, p.scale.dtype, e * p.scale.stride + i);
    return t;
  };
  float2 own[H];
  if (C == 1) {
#pragma unroll
    for (int h = 0; h < H; ++h) own[h] = make_float2(gain_of(threadIdx.x * N + 2 * h), gain_of(threadIdx.x * N + 2 * h + 1));
  } else if (p.affine) {
    for (int i = threadIdx.x; i < p.nvec * N; i += L) gain[term_slot<N>(i, p.nvec)] = gain_of(i);
  }
  float2 sp[C][H], sq[C][H];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int h = 0; h < H; ++h) sp[c][h] = sq[c][h] = make_float2(0.f, 0.f);
  auto gains = [&](int vec, float2 (&a)[H]) {
    if (C == 1) {
#pragma unroll
      for (int h = 0; h < H; ++h) a[h] = own[h];
    } else if (p.affine) {
      Terms<N>(gain, vec, p.nvec).load(0, a);
    } else {
#pragma unroll
      for (int h = 0; h < H; ++h) a[h] = make_float2(1.f, 1.f);
    }
  };
  // threads 0 .. 2 R - 1 each fetch one of the next rows' statistics
  const bool keeps = threadIdx.x < 2 * R;
  const int64_t ahead = threadIdx.x % R;
  const float* stat = (threadIdx.x < R ? p.mean : p.rstd) + e * p.rows + ahead;
  if (keeps) stats[0][threadIdx.x / R][ahead] = r0 + ahead < r1 ? __ldg(stat + r0) : 0.f;
  auto two = [&](int vec) { return READ != BY_ELEMENT || 2 * vec + 1 < p.width; };
  auto take = [](P& v, const uint8_t* at, bool both) {
    if constexpr (READ == BY_16) {
      const uint4 w = *reinterpret_cast<const uint4*>(at);
      v.w[0] = w.x; v.w[1] = w.y; v.w[2] = w.z; v.w[3] = w.w;
    } else if constexpr (sizeof(T) == 4) {
      v.w[0] = *reinterpret_cast<const uint32_t*>(at);
      if (both) v.w[1] = *reinterpret_cast<const uint32_t*>(at + 4);
    } else if constexpr (READ == BY_PAIR) {
      v.w[0] = *reinterpret_cast<const uint32_t*>(at);
    } else {
      uint32_t w = *reinterpret_cast<const unsigned short*>(at);
      if (both) w |= static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(at + 2)) << 16;
      v.w[0] = w;
    }
  };
  __syncthreads();
  bool ok = true;
  int it = 0;
  for (int64_t r = r0; r < r1; r += step, ++it) {
    const int s = it % p.stages;
    // (a wait that ran out: the launch ends without further waits, its status says so)
    ok = ok && mbar_wait(&full[s], (it / p.stages) & 1, p.status, &abort_flag);
    const uint8_t* from = ring + s * stage_bytes + threadIdx.x * N * sizeof(T);
    const float later = keeps && r + step + ahead < r1 ? __ldg(stat + r + step) : 0.f;
    const int rows = static_cast<int>(min(static_cast<int64_t>(R), r1 - r));
    // where row k begins in its first 16 bytes
    auto skip = [&](const T* base, int64_t stride, int k) -> uint32_t {
      if (READ == BY_16) return 0;
      return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base)) + (static_cast<uint32_t>(r) + k) * static_cast<uint32_t>(stride * sizeof(T)) & 15u;
    };
    P vg[R][C], vx[R][C];
    float mean[4], rstd[4], sum[8];
    {
      const float4 m4 = *reinterpret_cast<const float4*>(stats[it & 1][0]), d4 = *reinterpret_cast<const float4*>(stats[it & 1][1]);
      mean[0] = m4.x; mean[1] = m4.y; mean[2] = m4.z; mean[3] = m4.w;
      rstd[0] = d4.x; rstd[1] = d4.y; rstd[2] = d4.z; rstd[3] = d4.w;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sum[k] = 0.f;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const bool in = k < rows;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int vec = threadIdx.x + c * L;
        vg[k][c].clear();
        vx[k][c].clear();
        if (in && vec < p.nvec) {
          const int off = c * L * N * sizeof(T);
          take(vg[k][c], from + 2 * k * pitch + skip(dy, p.gs[1], k) + off, two(vec));
          take(vx[k][c], from + (2 * k + 1) * pitch + skip(x, p.xs[1], k) + off, two(vec));
        }
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int vec = threadIdx.x + c * L;
      if (vec >= p.nvec) break;
      float2 a[H];
      gains(vec, a);
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const float2 r2 = make_float2(rstd[k], rstd[k]), m2 = make_float2(mean[k], mean[k]);
        float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const float2 d = vg[k][c].pair(h), dl = mul2(d, sub2(vx[k][c].pair(h), m2));
          sq[c][h] = add2(sq[c][h], d);
          sp[c][h] = fma2(dl, r2, sp[c][h]);
          s0 = fma2(d, a[h], s0);
          s1 = fma2(dl, a[h], s1);
        }
        sum[2 * k] += s0.x + s0.y;
        sum[2 * k + 1] += s1.x + s1.y;
      }
    }
    turn ^= 1;
    const float mine = warp_sum8(sum, lane);
    if ((lane & 3) == 0) slots[turn][value_of(lane)][warp] = mine;
    if (keeps) stats[(it + 1) & 1][threadIdx.x / R][ahead] = later;
    __syncthreads();
    // the stage has been read: its next rows
    if (threadIdx.x == 0 && ok && r + p.stages * step < r1) fill(s, r + p.stages * step);
    // lane 4 i + j adds warps j, j + 4, .. of value i
    float t = 0.f;
    for (int w = lane & 3; w < warps; w += 4) t += slots[turn][lane >> 2][w];
    t += __shfl_xor_sync(0xffffffffu, t, 1);
    t += __shfl_xor_sync(0xffffffffu, t, 2);
    t *= p.inv_width;
#pragma unroll
    for (int k = 0; k < 2 * R; ++k) sum[k] = __shfl_sync(0xffffffffu, t, 4 * k);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int vec = threadIdx.x + c * L;
      if (vec >= p.nvec) break;
      float2 a[H];
      gains(vec, a);
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (k >= rows) break;
        // dx = (x - mean) (-rstd^3 mean(g (x - mean))) + dy (A rstd) - rstd mean(g)
        const float f0 = -rstd[k] * sum[2 * k], f1 = -rstd[k] * (rstd[k] * (rstd[k] * sum[2 * k + 1]));
        const float2 r2 = make_float2(rstd[k], rstd[k]), m2 = make_float2(mean[k], mean[k]);
        const float2 g0 = make_float2(f0, f0), g1 = make_float2(f1, f1);
        Piece<T, READ> o;
#pragma unroll
        for (int h = 0; h < H; ++h)
          o.set(h, fma2(sub2(vx[k][c].pair(h), m2), g1, fma2(vg[k][c].pair(h), mul2(a[h], r2), g0)));
        o.store(dx + (r + k) * p.os[1] + vec * N, two(vec));
      }
    }
  }
  if (!ok && threadIdx.x == 0) {          // the copies in flight have landed before the CTA leaves (again with a limit)
    int gave_up = 0;
    drain_ring<false>(full, p.stages, it, p.status, &gave_up);
  }
  if (p.sums) {
    float* part = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.width;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int vec = threadIdx.x + c * L;
      if (vec >= p.nvec) break;
#pragma unroll
      for (int h = 0; h < H; ++h) {
        if constexpr (READ == BY_ELEMENT) {
          part[2 * vec] = sp[c][h].x;
          part[p.width + 2 * vec] = sq[c][h].x;
          if (two(vec)) {
            part[2 * vec + 1] = sp[c][h].y;
            part[p.width + 2 * vec + 1] = sq[c][h].y;
          }
        } else {
          *reinterpret_cast<float2*>(part + vec * N + 2 * h) = sp[c][h];
          *reinterpret_cast<float2*>(part + p.width + vec * N + 2 * h) = sq[c][h];
        }
      }
    }
  }
}

// 8 to 32 lanes to a row, V pieces of R = 2 / V rows to a lane, the next rows fetched before these are used
template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 2) norm_back_narrow_kernel(const __grid_constant__ NormBackParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");     // the sums' kernel waits for this one's end itself
  using P = Piece<T, BY_16>;
  constexpr int N = P::N, H = N / 2, R = 2 / V;
  extern __shared__ __align__(16) float sums[];             // [group][2][nvec * N]
  const int L = p.lanes, at = threadIdx.x & (L - 1), G = kNormThreads / L, group = threadIdx.x / L;
  const int64_t e = blockIdx.x / p.chunks, r1 = p.rows, r0 = (blockIdx.x - e * p.chunks) * G * R, step = p.chunks * G * R;
  float2 a[V][H], sp[V][H], sq[V][H];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int h = 0; h < H; ++h) {
      float t[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = (at + i * L) * N + 2 * h + j;
        t[j] = n >= p.width ? 0.f : p.weight.p ? term_at(p.weight.p, p.weight.dtype, n) : 1.f;
        if (n < p.width && p.scale.p) t[j] *= 1.f + term_at(p.scale.p, p.scale.dtype, e * p.scale.stride + n);
      }
      a[i][h] = make_float2(t[0], t[1]);
      sp[i][h] = sq[i][h] = make_float2(0.f, 0.f);
    }
  const T* dy = static_cast<const T*>(p.dy) + e * p.gs[0] + at * N;
  const T* x = static_cast<const T*>(p.x) + e * p.xs[0] + at * N;
  T* dx = static_cast<T*>(p.dx) + e * p.os[0] + at * N;
  struct Rows {
    P g[R][V], x[R][V];
    float mean[R], rstd[R];
  };
  auto fetch = [&](Rows& v, int64_t r) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t row = r + k * G + group;
      const bool in = row < r1;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v.g[k][i].clear();
        v.x[k][i].clear();
        if (in && at + i * L < p.nvec) {
          v.g[k][i].load(dy + row * p.gs[1] + i * L * N, true);
          v.x[k][i].load(x + row * p.xs[1] + i * L * N, true);
        }
      }
      v.mean[k] = in ? __ldg(p.mean + e * p.rows + row) : 0.f;
      v.rstd[k] = in ? __ldg(p.rstd + e * p.rows + row) : 0.f;
    }
  };
  Rows v;
  fetch(v, r0);
  for (int64_t r = r0; r < r1; r += step) {
    Rows next;
    fetch(next, r + step);
    float s0[R], s1[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const float2 r2 = make_float2(v.rstd[k], v.rstd[k]), m2 = make_float2(v.mean[k], v.mean[k]);
      float2 t0 = make_float2(0.f, 0.f), t1 = t0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const float2 d = v.g[k][i].pair(h), u = mul2(sub2(v.x[k][i].pair(h), m2), r2), g = mul2(d, a[i][h]);
          sq[i][h] = add2(sq[i][h], d);
          sp[i][h] = fma2(d, u, sp[i][h]);
          t0 = add2(t0, g);
          t1 = fma2(g, u, t1);
        }
        v.g[k][i].packed();
        v.x[k][i].packed();
      }
      s0[k] = t0.x + t0.y;
      s1[k] = t1.x + t1.y;
    }
    auto step = [&](int d) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        s0[k] += __shfl_xor_sync(0xffffffffu, s0[k], d);
        s1[k] += __shfl_xor_sync(0xffffffffu, s1[k], d);
      }
    };
    if (L >= 32) step(16);
    if (L >= 16) step(8);
    step(4);
    step(2);
    step(1);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t row = r + k * G + group;
      const float2 r2 = make_float2(v.rstd[k], v.rstd[k]), m2 = make_float2(v.mean[k], v.mean[k]);
      const float m0 = s0[k] * p.inv_width, m1 = -s1[k] * p.inv_width;
      const float2 g0 = make_float2(m0, m0), g1 = make_float2(m1, m1);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        P o;
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const float2 u = mul2(sub2(v.x[k][i].pair(h), m2), r2), g = mul2(v.g[k][i].pair(h), a[i][h]);
          o.set(h, mul2(fma2(u, g1, sub2(g, g0)), r2));
        }
        if (row < r1 && at + i * L < p.nvec) o.store(dx + row * p.os[1] + i * L * N, true);
      }
    }
    v = next;
  }
  if (!p.sums) return;
  const int room = p.nvec * N;
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (at + i * L < p.nvec) {
        float* to = sums + group * 2 * room + (at + i * L) * N + 2 * h;
        *reinterpret_cast<float2*>(to) = sp[i][h];
        *reinterpret_cast<float2*>(to + room) = sq[i][h];
      }
  __syncthreads();
  float* part = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.width;
  for (int n = threadIdx.x; n < 2 * p.width; n += kNormThreads) {
    float t = 0.f;
    for (int g = 0; g < G; ++g) t += sums[g * 2 * room + (n < p.width ? n : room + n - p.width)];
    part[n] = t;
  }
}

struct NormTermsParams {
  float* part;                              // P and Q of a part: [2][width]
  int64_t lists, count, list_stride, part_stride;    // lists of `count` parts
  int width, columns;                       // columns: CTAs to a list
  bool entries;                             // a list is a batch entry's, else all of the entries' weighted sums
  TermView weight, bias, scale;             // scale: of the modulation
  void *dweight, *dbias, *dscale, *dshift;
  int weight_dtype, bias_dtype, scale_dtype, shift_dtype;
  bool keep;                                // an entry's sums times its modulation, for the sum over entries, in its first part
};

__device__ __forceinline__ void term_store(void* p, int dtype, int64_t i, float v) {
  if (dtype == HTRC_LAYER_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == HTRC_LAYER_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// A list's parts added up, 32 columns to a CTA: each warp every blockDim / 32th part, the warps' sums by a tree
__global__ void __launch_bounds__(1024, 1) norm_terms_kernel(const __grid_constant__ NormTermsParams p) {
  __shared__ float part[2][32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int64_t list = blockIdx.x / p.columns;
  const int first = static_cast<int>(blockIdx.x - list * p.columns) * 32;
  float* base = p.part + list * p.list_stride;
  asm volatile("griddepcontrol.wait;" ::: "memory");        // the kernel that writes the parts has ended
  float sp = 0.f, sq = 0.f;
  if (first + lane < p.width) {
    const float* src = base + warp * p.part_stride + first + lane;
    const int64_t step = warps * p.part_stride;
    int64_t c = warp;
    for (; c + 3 * warps < p.count; c += 4 * warps, src += 4 * step) {
      float a[4], b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a[k] = __ldcg(src + k * step);
        b[k] = __ldcg(src + k * step + p.width);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        sp += a[k];
        sq += b[k];
      }
    }
    float a[3] = {0.f, 0.f, 0.f}, b[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (c + k * warps < p.count) {
        a[k] = __ldcg(src + k * step);
        b[k] = __ldcg(src + k * step + p.width);
      }
    sp += a[0] + a[1] + a[2];
    sq += b[0] + b[1] + b[2];
  }
  part[0][warp][lane] = sp;
  part[1][warp][lane] = sq;
  __syncthreads();
  for (int col = warp; col < 32; col += warps) {
    sp = warp_sum(lane < warps ? part[0][lane][col] : 0.f);
    sq = warp_sum(lane < warps ? part[1][lane][col] : 0.f);
    const int i = first + col;
    if (lane != 0 || i >= p.width) continue;
    if (p.entries) {
      const float w = p.weight.p ? term_at(p.weight.p, p.weight.dtype, i) : 1.f;
      const float b = p.bias.p ? term_at(p.bias.p, p.bias.dtype, i) : 0.f;
      if (p.dscale) term_store(p.dscale, p.scale_dtype, list * p.width + i, fmaf(sp, w, sq * b));
      if (p.dshift) term_store(p.dshift, p.shift_dtype, list * p.width + i, sq);
      const float s = p.scale.p ? 1.f + term_at(p.scale.p, p.scale.dtype, list * p.scale.stride + i) : 1.f;
      sp *= s;
      sq *= s;
      if (p.keep) {                         // (this column of this part is read by this CTA alone, before the barrier)
        base[i] = sp;
        base[p.width + i] = sq;
        continue;
      }
    }
    if (p.dweight) term_store(p.dweight, p.weight_dtype, i, sp);
    if (p.dbias) term_store(p.dbias, p.bias_dtype, i, sq);
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

// how the rows of a tensor may be read
Reads reads_of(const void* p, const int64_t* s, int width, int es) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  if (width * es % 16 == 0 && at % 16 == 0 && s[0] * es % 16 == 0 && s[1] * es % 16 == 0) return BY_16;
  return width % 2 == 0 && at % (2 * es) == 0 && s[0] % 2 == 0 && s[1] % 2 == 0 ? BY_PAIR : BY_ELEMENT;
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

// CTAs of a kernel that an SM holds at once
template <typename K>
int resident_ctas(K kernel, int threads, size_t smem, int* registers) {
  if (*registers == 0) {
    cudaFuncAttributes attr{};
    if (cudaFuncGetAttributes(&attr, kernel) != cudaSuccess) return 0;
    *registers = attr.numRegs;
  }
  const int by_registers = 65536 / ((*registers + 7) / 8 * 8 * threads), by_smem = static_cast<int>(kNormSms / (smem + 3 * 1024));
  return std::max(1, std::min({by_registers, by_smem, 2048 / threads, 32}));
}

bool allow_smem(const void* kernel, size_t smem) {
  return smem <= 40 * 1024 ||
         cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) == cudaSuccess;
}

template <typename T, int READ, int MODE, int V, int LANES>
int norm_run(NormParams& p, cudaStream_t st) {
  constexpr int N = Piece<T, READ>::N, R = rows_of<T, READ, V, LANES, MODE>();
  auto kernel = norm_rows_kernel<T, READ, V, LANES, MODE>;
  if (LANES) p.lanes = LANES;
  const size_t smem = MODE != QUANT_CODES && p.affine ? static_cast<size_t>(p.nvec) * N * 2 * sizeof(float) : 0;
  // rows so wide that an SM holds one CTA's A and B: twice the warps share them
  const int threads = std::max(p.lanes, smem > kNormSms / 2 - 4096 ? 2 * kNormThreads : kNormThreads), groups = threads / p.lanes;
  static int registers = 0;
  const int resident = resident_ctas(kernel, threads, smem, &registers);
  if (resident == 0 || !allow_smem(reinterpret_cast<const void*>(kernel), smem)) return HTRC_ERR_CUDA;
  const int64_t ctas = static_cast<int64_t>(sm_count()) * resident;
  p.chunks = std::min(std::max<int64_t>(1, ctas / p.entries), (p.rows + groups * R - 1) / (groups * R));
  kernel<<<static_cast<unsigned>(std::min(p.entries * p.chunks, ctas)), threads, smem, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
}

template <typename T, int READ, int MODE>
int norm_launch(NormParams& p, cudaStream_t st) {
  constexpr int N = Piece<T, READ>::N;
  p.nvec = (p.width + N - 1) / N;
  const int64_t rows = p.entries * p.rows;
  // a warp to a row of up to 16 words to a lane (narrower rows: as many lanes as they have pieces, from eight on), more warps
  // to a wider one
  constexpr int kMost = READ == BY_16 ? 8 : 16;
  int lanes = 8;
  while (lanes < 32 * kNormMaxWarps && p.nvec > lanes * (lanes >= 32 ? kMost : 1)) lanes *= 2;
  // few rows: as many lanes as a row has pieces (1 x 4,096: 5.4 us, 6.3 by a warp for eight of them; more rows the same)
  int most = lanes;
  while (most < p.nvec) most *= 2;
  if (most <= 32 * kNormMaxWarps && rows * most <= 256 * sm_count()) lanes = most;
  p.lanes = lanes;
  if (p.nvec <= lanes) return norm_run<T, READ, MODE, 1, 0>(p, st);
  if constexpr (READ == BY_16) {
    if (lanes == 32 && p.nvec <= 64) return norm_run<T, READ, MODE, 2, 32>(p, st);
    if (lanes == 32 && p.nvec <= 128) return norm_run<T, READ, MODE, 4, 32>(p, st);
    if (lanes == 32) return norm_run<T, READ, MODE, 8, 32>(p, st);
    if (lanes == 64) return norm_run<T, READ, MODE, 8, 64>(p, st);
    if (lanes == 128) return norm_run<T, READ, MODE, 8, 128>(p, st);
    if constexpr (sizeof(T) == 4) return lanes == 256 ? norm_run<T, READ, MODE, 8, 256>(p, st) : norm_run<T, READ, MODE, 8, 512>(p, st);
    else return norm_run<T, READ, MODE, 8, 256>(p, st);
  } else {
    if (p.nvec > 64 && p.nvec <= 128) return norm_run<T, READ, MODE, 4, 32>(p, st);
    if (p.nvec > 256 && p.nvec <= 512) return norm_run<T, READ, MODE, 16, 32>(p, st);
    return norm_run<T, READ, MODE, 16, 0>(p, st);
  }
}

template <int MODE, typename T>
int norm_reads(NormParams& p, Reads reads, cudaStream_t st) {
  if (reads == BY_16) return norm_launch<T, BY_16, MODE>(p, st);
  return reads == BY_PAIR ? norm_launch<T, BY_PAIR, MODE>(p, st) : norm_launch<T, BY_ELEMENT, MODE>(p, st);
}
template <int MODE>
int norm_types(NormParams& p, int dtype, Reads reads, cudaStream_t st) {
  if (dtype == HTRC_LAYER_F32) return norm_reads<MODE, float>(p, reads, st);
  return dtype == HTRC_LAYER_BF16 ? norm_reads<MODE, __nv_bfloat16>(p, reads, st) : norm_reads<MODE, __half>(p, reads, st);
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
  Reads reads = reads_of(a->x, a->x_stride, a->width, es);
  if (!codes) reads = std::min(reads, reads_of(a->out, a->out_stride, a->width, es));
  const RowShape shape = codes ? RowShape(a->batch, a->tokens, p.modulated, {a->x_stride})
                               : RowShape(a->batch, a->tokens, p.modulated, {a->x_stride, a->out_stride});
  p.entries = shape.entries;
  p.rows = shape.rows;
  shape.set(a->x_stride, p.xs);
  if (!codes) shape.set(a->out_stride, p.os);
  return codes ? norm_types<NORM_CODES>(p, a->dtype, reads, st) : norm_types<NORM_ROWS>(p, a->dtype, reads, st);
}

// How the backward's rows are shared out: the kernel, its CTAs' threads, shared memory and rows
struct NormBackPlan {
  Reads reads;
  bool narrow;
  int per, lanes, threads, stages;          // per: pieces of a row to a thread
  size_t smem;
  int64_t chunks;                           // CTAs of an entry
  NormBackPlan(int width, int es, Reads by, bool affine, int64_t entries, int64_t rows) : reads(by) {
    // float32 rows of more 16-byte pieces than a thread has registers for
    if (reads == BY_16 && width * es > 2048 * 16) reads = BY_PAIR;
    const int n = reads == BY_16 ? 16 / es : 2, nvec = (width + n - 1) / n;
    int resident, least;                    // CTAs of an SM, rows that a CTA takes at a time
    lanes = stages = 0;
    // rows to warps: 200,000 x 128 in 16 bits 38 us, by the ring 68; 200,000 x 256 66 and 70; 100,000 x 512 70 and 68; float32,
    // 200,000 x 128 63 and 63, 100,000 x 256 60 and 58
    narrow = reads == BY_16 && nvec <= 64;
    if (narrow) {
      lanes = nvec <= 8 ? 8 : nvec <= 16 ? 16 : 32;
      per = nvec <= lanes ? 1 : 2;
      threads = kNormThreads;
      smem = static_cast<size_t>(threads / lanes) * 2 * nvec * n * sizeof(float);
      resident = 2;
      least = threads / lanes * (2 / per);
    } else {
      if (reads == BY_16) per = nvec <= 512 ? 1 : nvec <= 1024 ? 2 : 4;
      else per = nvec <= 128 ? 2 : nvec <= 2048 ? 4 : nvec <= 4096 ? 8 : 16;
      threads = ((nvec + per - 1) / per + 31) / 32 * 32;
      resident = std::max(1, 512 / threads);
      least = es == 4 ? (reads == BY_16 ? ring_rows<float, BY_16>(per) : ring_rows<float, BY_PAIR>(per))
                      : (reads == BY_16 ? ring_rows<__half, BY_16>(per) : ring_rows<__half, BY_PAIR>(per));
      const size_t stage = 2 * static_cast<size_t>(least) * ring_pitch(width * es, reads);
      const size_t gain = per > 1 && affine ? static_cast<size_t>(nvec) * n * 4 : 0, room = 216 * 1024 / resident - gain - 2048;
      stages = static_cast<int>(std::max<size_t>(1, std::min<size_t>(4, room / stage)));
      smem = stages * stage + gain;
    }
    const int64_t share = std::max<int64_t>(1, static_cast<int64_t>(resident) * sm_count() / std::max<int64_t>(1, entries));
    chunks = std::max<int64_t>(1, std::min(share, (rows + least - 1) / least));
  }
};

bool norm_sums(const HtrcNormArgs* a) { return a->dweight || a->dbias || a->dscale || a->dshift; }

RowShape norm_back_shape(const HtrcNormArgs* a) {
  return RowShape(a->batch, a->tokens, a->scale || a->shift, {a->dy_stride, a->x_stride, a->dx_stride});
}

template <typename T>
int norm_back_launch(NormBackParams& p, const NormBackPlan& plan, cudaStream_t st) {
  const int n = plan.reads == BY_16 ? static_cast<int>(16 / sizeof(T)) : 2;
  p.nvec = (p.width + n - 1) / n;
  p.lanes = plan.lanes;
  p.stages = plan.stages;
  p.chunks = plan.chunks;
  const unsigned grid = static_cast<unsigned>(p.entries * p.chunks);
  if (grid == 0) return HTRC_OK;
  auto go = [&](auto kernel) {
    if (!allow_smem(reinterpret_cast<const void*>(kernel), plan.smem)) return HTRC_ERR_CUDA;
    kernel<<<grid, plan.threads, plan.smem, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
  };
  if (plan.narrow) return plan.per == 1 ? go(norm_back_narrow_kernel<T, 1>) : go(norm_back_narrow_kernel<T, 2>);
  if (plan.reads == BY_16) {
    if (plan.per == 1) return go(norm_back_ring_kernel<T, BY_16, 1>);
    return plan.per == 2 ? go(norm_back_ring_kernel<T, BY_16, 2>) : go(norm_back_ring_kernel<T, BY_16, 4>);
  }
  auto by = [&](auto read) {
    constexpr int READ = decltype(read)::value;
    if (plan.per == 2) return go(norm_back_ring_kernel<T, READ, 2>);
    if (plan.per == 4) return go(norm_back_ring_kernel<T, READ, 4>);
    return plan.per == 8 ? go(norm_back_ring_kernel<T, READ, 8>) : go(norm_back_ring_kernel<T, READ, 16>);
  };
  return plan.reads == BY_PAIR ? by(std::integral_constant<int, BY_PAIR>{}) : by(std::integral_constant<int, BY_ELEMENT>{});
}

Reads back_reads(const HtrcNormArgs* a) {
  const int es = type_size(a->dtype);
  return std::min({reads_of(a->x, a->x_stride, a->width, es), reads_of(a->dy, a->dy_stride, a->width, es),
                   reads_of(a->dx, a->dx_stride, a->width, es)});
}

int norm_back_size(const HtrcNormArgs* a, size_t* bytes) {
  if (bytes == nullptr) return HTRC_ERR_ARG;
  const int rc = norm_validate(a);
  if (rc != HTRC_OK) return rc;
  const RowShape shape = norm_back_shape(a);
  const NormBackPlan plan(a->width, type_size(a->dtype), back_reads(a), a->weight || a->scale, shape.entries, shape.rows);
  *bytes = norm_sums(a) ? static_cast<size_t>(shape.entries) * plan.chunks * 2 * a->width * sizeof(float) : 0;
  return HTRC_OK;
}

int norm_terms(const NormTermsParams& t, cudaStream_t st) {
  if (t.lists == 0) return HTRC_OK;
  if (t.lists * t.columns >= kMaxRows) return HTRC_ERR_UNSUPPORTED;
  int warps = 1;
  while (warps < 32 && warps * 4 < t.count) warps *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(t.lists * t.columns));
  cfg.blockDim = dim3(32 * warps);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, norm_terms_kernel, t) == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
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
  p.status = a->status;
  const NormBackPlan plan(a->width, type_size(a->dtype), back_reads(a), p.affine, p.entries, p.rows);
  if (p.entries * plan.chunks >= kMaxRows) return HTRC_ERR_UNSUPPORTED;
  rc = a->dtype == HTRC_LAYER_F32    ? norm_back_launch<float>(p, plan, st)
       : a->dtype == HTRC_LAYER_BF16 ? norm_back_launch<__nv_bfloat16>(p, plan, st)
                                     : norm_back_launch<__half>(p, plan, st);
  if (rc != HTRC_OK) return rc;
  if (p.sums) {
    NormTermsParams t{};
    t.part = p.part;
    t.width = a->width;
    t.columns = (a->width + 31) / 32;
    t.part_stride = 2 * static_cast<int64_t>(a->width);
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
    // an entry's parts with a modulation, and then the entries' sums where a weight or bias wants them; without one all
    // parts are alike
    t.entries = a->scale || a->shift;
    t.lists = t.entries ? p.entries : 1;
    t.count = t.entries ? p.chunks : p.entries * p.chunks;
    t.list_stride = t.count * t.part_stride;
    t.keep = t.entries && p.entries != 1 && (a->dweight || a->dbias);
    rc = norm_terms(t, st);
    if (rc != HTRC_OK) return rc;
    if (t.keep) {
      t.entries = t.keep = false;
      t.part_stride = t.list_stride;
      t.count = t.lists;
      t.lists = 1;
      rc = norm_terms(t, st);
      if (rc != HTRC_OK) return rc;
    }
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
  const RowShape shape(batch, tokens, false, {stride});
  p.entries = shape.entries;
  p.rows = shape.rows;
  shape.set(stride, p.xs);
  return norm_types<QUANT_CODES>(p, dtype, reads_of(x, stride, width, type_size(dtype)), st);
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
