// Rotary positions over several axes, with the per-head RMS norm before them, forward and backward, and the
// C entries of include/htrc_layer.h for them.
//
// Forward, per row of dim elements (one token, one head):  u = x * rsqrt(mean(x^2) + eps) * w  (or u = x), then
// every pair (a, b) of the rotated width becomes (a cos - b sin, a sin + b cos).  Backward:  g = the transposed
// rotation of dy;  dw = sum g x r;  h = g w;  dx = r (h - x r^2 mean(h x)),  r = rsqrt(mean(x^2) + eps).
//
// Both only move bytes: a row is read once and written once (backward with a norm: two reads), all arithmetic is
// float32 in registers.  A warp holds 32 / LPR rows of one token at a time, LPR lanes of 8 elements each, and walks
// the heads of its token, so the 4 cosines and sines that a lane needs are computed once per token and stay in
// registers.  The output's strides carry the token-major -> head-major reorder.
//
// Angles: an int32 position times the frequency in revolutions as a 64-bit fixed-point fraction, modulo 2^64, is the
// exactly reduced turn for every int32 position (float32 positions: the product in two floats, its whole turns
// dropped), so late positions lose no accuracy.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <limits>

#include "../../include/htrc_layer.h"
#include "common.cuh"
#include "kernels.cuh"

namespace htrc {

namespace {

constexpr int kRotWarps = 8;
constexpr int kRotMaxPairs = HTRC_ROTARY_MAX_DIM / 2;
// Row batches that a warp fetches together (one more set is in flight while they are used), and CTAs per SM the
// registers are held to.  q and k of 129,024 tokens x 24 heads x 128, bfloat16, after a rest: forward 504 us (2, 4), 529
// (3, 3), 571 (2, 2), 576 (2, 3), 618 (1, 4); backward of 32,768 tokens 233 us (3, 2), 239 (4, 2), 247 (2, 2), 266 (1, 3), 320
// (2, 3).
constexpr int rot_unroll(bool back) { return back ? 3 : 2; }
constexpr int rot_ctas(bool back, int bytes) { return back || bytes == 4 ? 2 : 4; }

struct RotaryRows {
  const void* in;
  void* out;
  const void* x;
  const void* weight;
  int64_t is[3], os[3], xs[3];
  int heads, weight_dtype;
  int chunk, chunks;                  // heads per task, tasks per token
};

struct RotaryParams {
  RotaryRows t[2];
  const void* positions;
  int64_t ps[3];
  int64_t batch, tokens;
  int dim, npairs;
  float eps;
  bool float_positions;
  uint64_t turn[kRotMaxPairs];        // frequency in revolutions: 0.64 fixed point, or (hi, lo) floats
  uint8_t axis[kRotMaxPairs];
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float load_weight(const void* w, int dtype, int i) {
  if (dtype == HTRC_LAYER_F32) return __ldg(static_cast<const float*>(w) + i);
  if (dtype == HTRC_LAYER_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(static_cast<const __half*>(w)[i]);
}

// A CTA's copies of what its lanes index: a kernel parameter read at an index that differs by lane takes a pass for each
// (32,768 tokens x 24 heads: 154 us with the parameters themselves, 136 so)
struct RotaryShared {
  uint64_t turn[kRotMaxPairs];
  int64_t axis[kRotMaxPairs];           // element offset of the pair's position
  float weight[2 * kRotMaxPairs];       // 1 without a norm
  __device__ __forceinline__ void fill(const RotaryParams& p, const RotaryRows& r) {
    for (int i = threadIdx.x; i < p.npairs; i += blockDim.x) {
      turn[i] = p.turn[i];
      axis[i] = p.axis[i] * p.ps[2];
    }
    for (int i = threadIdx.x; i < p.dim; i += blockDim.x) weight[i] = r.weight ? load_weight(r.weight, r.weight_dtype, i) : 1.f;
    __syncthreads();
  }
};

// cosine and sine of pair i of a token whose positions start at pos.  QUICK (16-bit rows): by the special function units,
// absolute error 2^-21 on the reduced angle, against a rounding of 2^-9 or 2^-12; float32 rows take the 2-ulp functions.
template <bool QUICK>
__device__ __forceinline__ float2 pair_turn(const RotaryParams& p, const RotaryShared& sh, int64_t pos, int i) {
  const int64_t at = pos + sh.axis[i];
  const uint64_t f = sh.turn[i];
  float turns;
  if (!p.float_positions) {
    const int32_t n = __ldg(static_cast<const int32_t*>(p.positions) + at);
    const uint64_t frac = static_cast<uint64_t>(static_cast<int64_t>(n)) * f;      // modulo one revolution
    turns = static_cast<float>(static_cast<int32_t>(frac >> 32)) * 0x1p-32f;
  } else {
    const float n = __ldg(static_cast<const float*>(p.positions) + at);
    const float hi = __uint_as_float(static_cast<uint32_t>(f >> 32)), lo = __uint_as_float(static_cast<uint32_t>(f));
    const float t = n * hi;
    turns = (t - rintf(t)) + fmaf(n, lo, fmaf(n, hi, -t));
  }
  float s, c;
  if constexpr (QUICK) __sincosf(6.283185307179586f * turns, &s, &c);
  else sincospif(2.0f * turns, &s, &c);
  return make_float2(c, s);
}

// A lane's 8 elements of a row: two groups of 4 at off0 and off1 (16-bit types: 8 bytes each, float32: 16).
// Interleaved pairs: off1 = off0 + 4, one contiguous piece.
template <typename T>
struct Raw {
  uint4 a;
};
template <>
struct Raw<float> {
  uint4 a, b;
};
template <typename T, bool HALF>
__device__ __forceinline__ Raw<T> load_raw(const T* row, int off0, int off1) {
  Raw<T> r;
  if constexpr (sizeof(T) == 4) {
    r.a = __ldg(reinterpret_cast<const uint4*>(row + off0));
    r.b = __ldg(reinterpret_cast<const uint4*>(row + off1));
  } else if constexpr (HALF) {
    const uint2 lo = __ldg(reinterpret_cast<const uint2*>(row + off0));
    const uint2 hi = __ldg(reinterpret_cast<const uint2*>(row + off1));
    r.a = make_uint4(lo.x, lo.y, hi.x, hi.y);
  } else {
    r.a = __ldg(reinterpret_cast<const uint4*>(row + off0));
  }
  return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) { return pack_f16x2(a, b); }

// A lane's elements as the firsts and seconds of its four pairs, two pairs per register pair: paired float32
// instructions then do two pairs at once, whatever the pairs' layout in memory.
struct Pairs {
  float2 f[2], s[2];
};

template <typename T, bool HALF>
__device__ __forceinline__ Pairs unpack(const Raw<T>& r) {
  Pairs v;
  if constexpr (sizeof(T) == 4) {
    const float a[8] = {__uint_as_float(r.a.x), __uint_as_float(r.a.y), __uint_as_float(r.a.z), __uint_as_float(r.a.w),
                        __uint_as_float(r.b.x), __uint_as_float(r.b.y), __uint_as_float(r.b.z), __uint_as_float(r.b.w)};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v.f[i] = HALF ? make_float2(a[2 * i], a[2 * i + 1]) : make_float2(a[4 * i], a[4 * i + 2]);
      v.s[i] = HALF ? make_float2(a[4 + 2 * i], a[5 + 2 * i]) : make_float2(a[4 * i + 1], a[4 * i + 3]);
    }
  } else {
    const float2 w[4] = {unpack2<T>(r.a.x), unpack2<T>(r.a.y), unpack2<T>(r.a.z), unpack2<T>(r.a.w)};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v.f[i] = HALF ? w[i] : make_float2(w[2 * i].x, w[2 * i + 1].x);
      v.s[i] = HALF ? w[2 + i] : make_float2(w[2 * i].y, w[2 * i + 1].y);
    }
  }
  return v;
}
template <typename T, bool HALF>
__device__ __forceinline__ void store8(T* row, int off0, int off1, const Pairs& v) {
  if constexpr (sizeof(T) == 4) {
    const float4 lo = HALF ? make_float4(v.f[0].x, v.f[0].y, v.f[1].x, v.f[1].y) : make_float4(v.f[0].x, v.s[0].x, v.f[0].y, v.s[0].y);
    const float4 hi = HALF ? make_float4(v.s[0].x, v.s[0].y, v.s[1].x, v.s[1].y) : make_float4(v.f[1].x, v.s[1].x, v.f[1].y, v.s[1].y);
    *reinterpret_cast<float4*>(row + off0) = lo;
    *reinterpret_cast<float4*>(row + off1) = hi;
  } else if constexpr (HALF) {
    *reinterpret_cast<uint2*>(row + off0) = make_uint2(pack2<T>(v.f[0].x, v.f[0].y), pack2<T>(v.f[1].x, v.f[1].y));
    *reinterpret_cast<uint2*>(row + off1) = make_uint2(pack2<T>(v.s[0].x, v.s[0].y), pack2<T>(v.s[1].x, v.s[1].y));
  } else {
    *reinterpret_cast<uint4*>(row + off0) = make_uint4(pack2<T>(v.f[0].x, v.s[0].x), pack2<T>(v.f[0].y, v.s[0].y),
                                                       pack2<T>(v.f[1].x, v.s[1].x), pack2<T>(v.f[1].y, v.s[1].y));
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// the sums of two values over the LPR lanes of a row, in one exchange more than one of them takes
template <int LPR>
__device__ __forceinline__ float2 row_sums(float a, float b, int lane) {
  const bool odd = lane & 1;
  float v = odd ? b : a;
  v += __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
#pragma unroll
  for (int o = LPR / 2; o > 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const float t = __shfl_xor_sync(0xffffffffu, v, 1);
  return odd ? make_float2(t, v) : make_float2(v, t);
}

// Rows whose pieces are 16-byte aligned, dim a multiple of 8 (HALF: the rotated width too).  blockIdx.y names the
// tensor; a warp's task is a token and `chunk` of its heads or, FLAT, rows of any tokens.  The norm's weight is folded
// into the cosines and sines.  BACK with a weight leaves the CTA's weight-gradient sums at partial[(blockIdx.y * gridDim.x + blockIdx.x) * dim].
template <typename T, int LPR, bool HALF, bool BACK, bool FLAT>
__global__ void __launch_bounds__(kRotWarps * 32, rot_ctas(BACK, sizeof(T)))
    rotary_kernel(const __grid_constant__ RotaryParams p, float* __restrict__ partial) {
  __shared__ float sums[BACK ? kRotWarps * 32 * 8 : 1];
  __shared__ RotaryShared sh;
  const RotaryRows& r = p.t[blockIdx.y];
  sh.fill(p, r);
  constexpr int RPW = 32 / LPR, kRotUnroll = rot_unroll(BACK);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int u = lane % LPR, sub = lane / LPR;
  const int units = p.dim / 8;
  const bool on = u < units;
  // the lane's elements (off0 .. + 3, off1 .. + 3) and the pairs they make, the first `turned` of them rotated
  int off0 = 8 * u, off1 = 8 * u + 4, pair0 = 4 * u, turned;
  if (HALF) {
    const int rot = p.npairs / 4;
    turned = u < rot ? 4 : 0;
    if (u < rot) {
      off0 = 4 * u;
      off1 = p.npairs + 4 * u;
    }
  } else {
    turned = min(4, max(0, p.npairs - pair0));
  }
  if (!on) turned = 0;
  const bool norm = r.weight != nullptr, whole = 2 * p.npairs == p.dim;
  // offsets of element e of the firsts (0 .. 3) and seconds
  auto first_at = [&](int e) { return HALF ? off0 + e : off0 + 2 * e; };
  auto second_at = [&](int e) { return HALF ? off1 + e : off0 + 2 * e + 1; };
  auto weights = [&]() {
    Pairs w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w.f[i] = w.s[i] = make_float2(1.f, 1.f);
      if (on) {
        w.f[i] = make_float2(sh.weight[first_at(2 * i)], sh.weight[first_at(2 * i + 1)]);
        w.s[i] = make_float2(sh.weight[second_at(2 * i)], sh.weight[second_at(2 * i + 1)]);
      }
    }
    return w;
  };
  Pairs dw;
#pragma unroll
  for (int i = 0; i < 2; ++i) dw.f[i] = dw.s[i] = make_float2(0.f, 0.f);
  const float inv_dim = 1.0f / static_cast<float>(p.dim);
  // forward: (f, s) -> (f fc - s ss, f fs + s sc), the weight folded in; backward: (f fc + s fs, s fc - f fs)
  float2 fc[2], fs[2], sc[2], ss[2];
  auto angles = [&](int64_t pos) {
    const Pairs w = weights();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 t0 = 2 * i < turned ? pair_turn<sizeof(T) == 2>(p, sh, pos, pair0 + 2 * i) : make_float2(1.f, 0.f);
      const float2 t1 = 2 * i + 1 < turned ? pair_turn<sizeof(T) == 2>(p, sh, pos, pair0 + 2 * i + 1) : make_float2(1.f, 0.f);
      fc[i] = make_float2(t0.x, t1.x);
      fs[i] = make_float2(t0.y, t1.y);
      if (!BACK) {
        sc[i] = mul2(fc[i], w.s[i]);
        ss[i] = mul2(make_float2(-t0.y, -t1.y), w.s[i]);
        fc[i] = mul2(fc[i], w.f[i]);
        fs[i] = mul2(fs[i], w.f[i]);
      } else {
        ss[i] = make_float2(-t0.y, -t1.y);
      }
    }
  };
  // one row's elements of this lane: what was read (backward: the gradient, and x with a norm) to what is written
  auto turn = [&](const Raw<T>& now, const Raw<T>& nowx) {
    Pairs v = unpack<T, HALF>(now), y;
    if (!BACK) {
      if (norm) {
        float2 q = mul2(v.f[0], v.f[0]);
        q = fma2(v.f[1], v.f[1], q);
        q = fma2(v.s[0], v.s[0], q);
        q = fma2(v.s[1], v.s[1], q);
        const float rs = rsqrtf(fmaf(row_sum<LPR>(q.x + q.y), inv_dim, p.eps));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          v.f[i] = mul2(v.f[i], make_float2(rs, rs));
          v.s[i] = mul2(v.s[i], make_float2(rs, rs));
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        y.f[i] = fma2(v.f[i], fc[i], mul2(v.s[i], ss[i]));
        y.s[i] = fma2(v.f[i], fs[i], mul2(v.s[i], sc[i]));
      }
      if (!whole) {      // a pair past the rotated width keeps its elements apart, whatever they hold
        const Pairs w = weights();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (2 * i >= turned) {
            y.f[i].x = v.f[i].x * w.f[i].x;
            y.s[i].x = v.s[i].x * w.s[i].x;
          }
          if (2 * i + 1 >= turned) {
            y.f[i].y = v.f[i].y * w.f[i].y;
            y.s[i].y = v.s[i].y * w.s[i].y;
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        y.f[i] = fma2(v.f[i], fc[i], mul2(v.s[i], fs[i]));
        y.s[i] = fma2(v.s[i], fc[i], mul2(v.f[i], ss[i]));
      }
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (2 * i >= turned) {
            y.f[i].x = v.f[i].x;
            y.s[i].x = v.s[i].x;
          }
          if (2 * i + 1 >= turned) {
            y.f[i].y = v.f[i].y;
            y.s[i].y = v.s[i].y;
          }
        }
      }
      if (norm) {
        const Pairs w = weights(), xv = unpack<T, HALF>(nowx);
        float2 q = mul2(xv.f[0], xv.f[0]), hx;
        q = fma2(xv.f[1], xv.f[1], q);
        q = fma2(xv.s[0], xv.s[0], q);
        q = fma2(xv.s[1], xv.s[1], q);
        Pairs g;         // the gradient of the normalised row, times the weight
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          g.f[i] = mul2(y.f[i], w.f[i]);
          g.s[i] = mul2(y.s[i], w.s[i]);
        }
        hx = mul2(g.f[0], xv.f[0]);
        hx = fma2(g.f[1], xv.f[1], hx);
        hx = fma2(g.s[0], xv.s[0], hx);
        hx = fma2(g.s[1], xv.s[1], hx);
        const float2 t = row_sums<LPR>(q.x + q.y, hx.x + hx.y, lane);
        const float rs = rsqrtf(fmaf(t.x, inv_dim, p.eps));
        const float back = -t.y * inv_dim * rs * rs;
        const float2 rs2 = make_float2(rs, rs), back2 = make_float2(back, back);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 xf = mul2(xv.f[i], rs2), xs = mul2(xv.s[i], rs2);
          dw.f[i] = fma2(y.f[i], xf, dw.f[i]);
          dw.s[i] = fma2(y.s[i], xs, dw.s[i]);
          y.f[i] = fma2(xf, back2, mul2(g.f[i], rs2));
          y.s[i] = fma2(xs, back2, mul2(g.s[i], rs2));
        }
      }
    }
    return y;
  };
  const uint32_t tokens = static_cast<uint32_t>(p.tokens);
  if constexpr (FLAT) {
    // a task is RPW * kRotUnroll rows, each with a token of its own
    const uint32_t rows = static_cast<uint32_t>(p.batch) * tokens * r.heads, per = RPW * kRotUnroll;
    for (uint32_t task = blockIdx.x * kRotWarps + warp; task * static_cast<uint64_t>(per) < rows; task += gridDim.x * kRotWarps) {
      Raw<T> raw[kRotUnroll], rawx[BACK ? kRotUnroll : 1];
      T* out[kRotUnroll];
      int64_t pos[kRotUnroll];
#pragma unroll
      for (int k = 0; k < kRotUnroll; ++k) {
        const uint32_t row = task * per + k * RPW + sub;
        const bool in_k = row < rows;
        const uint32_t at = in_k ? row : 0, tok = at / r.heads, h = at - tok * r.heads, b = tok / tokens, n = tok - b * tokens;
        raw[k] = Raw<T>{};
        if (BACK) rawx[k] = Raw<T>{};
        if (on && in_k) {
          raw[k] = load_raw<T, HALF>(static_cast<const T*>(r.in) + b * r.is[0] + n * r.is[1] + h * r.is[2], off0, off1);
          if (BACK && norm) rawx[k] = load_raw<T, HALF>(static_cast<const T*>(r.x) + b * r.xs[0] + n * r.xs[1] + h * r.xs[2], off0, off1);
        }
        out[k] = on && in_k ? static_cast<T*>(r.out) + b * r.os[0] + n * r.os[1] + h * r.os[2] : nullptr;
        pos[k] = b * p.ps[0] + n * p.ps[1];
      }
#pragma unroll
      for (int k = 0; k < kRotUnroll; ++k) {
        angles(pos[k]);
        const Pairs y = turn(raw[k], rawx[BACK ? k : 0]);
        if (out[k] != nullptr) store8<T, HALF>(out[k], off0, off1, y);
      }
    }
  } else {
    const uint32_t tasks = static_cast<uint32_t>(p.batch) * tokens * r.chunks;
    for (uint32_t task = blockIdx.x * kRotWarps + warp; task < tasks; task += gridDim.x * kRotWarps) {
      const uint32_t tok = task / r.chunks, b = tok / tokens, n = tok - b * tokens;
      const int h0 = static_cast<int>(task - tok * r.chunks) * r.chunk, h1 = min(r.heads, h0 + r.chunk);
      const T* in = static_cast<const T*>(r.in) + b * r.is[0] + n * r.is[1] + (h0 + sub) * r.is[2];
      const T* x = BACK && norm ? static_cast<const T*>(r.x) + b * r.xs[0] + n * r.xs[1] + (h0 + sub) * r.xs[2] : nullptr;
      T* out = static_cast<T*>(r.out) + b * r.os[0] + n * r.os[1] + (h0 + sub) * r.os[2];
      // rows in flight: the first ones are asked for before the angles are formed, the next ones before these are used
      Raw<T> raw[kRotUnroll], rawx[BACK ? kRotUnroll : 1];
      auto fetch = [&](int h) {
#pragma unroll
        for (int k = 0; k < kRotUnroll; ++k) {
          raw[k] = Raw<T>{};
          if (BACK) rawx[k] = Raw<T>{};
          if (on && h + k * RPW < h1) {
            raw[k] = load_raw<T, HALF>(in + k * RPW * r.is[2], off0, off1);
            if (BACK && norm) rawx[k] = load_raw<T, HALF>(x + k * RPW * r.xs[2], off0, off1);
          }
        }
        in += RPW * kRotUnroll * r.is[2];
        if (BACK && norm) x += RPW * kRotUnroll * r.xs[2];
      };
      fetch(h0 + sub);
      angles(b * p.ps[0] + n * p.ps[1]);
      for (int h = h0 + sub; h - sub < h1; h += RPW * kRotUnroll) {
        Raw<T> now[kRotUnroll], nowx[BACK ? kRotUnroll : 1];
#pragma unroll
        for (int k = 0; k < kRotUnroll; ++k) {
          now[k] = raw[k];
          if (BACK) nowx[k] = rawx[k];
        }
        if (h - sub + RPW * kRotUnroll < h1) fetch(h + RPW * kRotUnroll);
#pragma unroll
        for (int k = 0; k < kRotUnroll; ++k) {
          const Pairs y = turn(now[k], nowx[BACK ? k : 0]);
          if (on && h + k * RPW < h1) store8<T, HALF>(out + k * RPW * r.os[2], off0, off1, y);
        }
        out += RPW * kRotUnroll * r.os[2];
      }
    }
  }
  if (BACK && norm) {
    // the CTA's sums, rows of a warp and then warps in order
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<float2*>(sums + threadIdx.x * 8 + 2 * i) = dw.f[i];
      *reinterpret_cast<float2*>(sums + threadIdx.x * 8 + 4 + 2 * i) = dw.s[i];
    }
    __syncthreads();
    float* dst = partial + (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * p.dim;
    if (threadIdx.x < LPR && on) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float s = 0.f;
        for (int g = 0; g < kRotWarps * RPW; ++g) s += sums[(g * LPR + u) * 8 + i];
        dst[i < 4 ? first_at(i) : second_at(i - 4)] = s;
      }
    }
  }
}

// Any dim, alignment and rotated width: a warp per row, one element per lane and step, the normalised row in shared
// memory while its pairs are formed.
template <typename T, bool BACK>
__global__ void __launch_bounds__(kRotWarps * 32)
    rotary_any_kernel(const __grid_constant__ RotaryParams p, bool half, float* __restrict__ partial) {
  constexpr int kMax = HTRC_ROTARY_MAX_DIM, kEl = kMax / 32;
  __shared__ float rows[kRotWarps][kMax];
  __shared__ RotaryShared sh;
  const RotaryRows& r = p.t[blockIdx.y];
  sh.fill(p, r);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool norm = r.weight != nullptr;
  float dw[kEl];
#pragma unroll
  for (int k = 0; k < kEl; ++k) dw[k] = 0.f;
  const float inv_dim = 1.0f / static_cast<float>(p.dim);
  const int64_t tasks = p.batch * p.tokens * r.heads;
  for (int64_t task = static_cast<int64_t>(blockIdx.x) * kRotWarps + warp; task < tasks;
       task += static_cast<int64_t>(gridDim.x) * kRotWarps) {
    const int64_t tok = task / r.heads, h = task - tok * r.heads, b = tok / p.tokens, n = tok - b * p.tokens;
    const T* in = static_cast<const T*>(r.in) + b * r.is[0] + n * r.is[1] + h * r.is[2];
    T* out = static_cast<T*>(r.out) + b * r.os[0] + n * r.os[1] + h * r.os[2];
    const int64_t pos = b * p.ps[0] + n * p.ps[1];
    float v[kEl], ss = 0.f;
#pragma unroll
    for (int k = 0; k < kEl; ++k) {
      const int e = lane + 32 * k;
      v[k] = e < p.dim ? to_f<T>(in[e]) : 0.f;
      ss = fmaf(v[k], v[k], ss);
    }
    if (!BACK && norm) {
      const float rs = rsqrtf(row_sum<32>(ss) * inv_dim + p.eps);
#pragma unroll
      for (int k = 0; k < kEl; ++k) {
        const int e = lane + 32 * k;
        if (e < p.dim) v[k] *= rs * sh.weight[e];
      }
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kEl; ++k) rows[warp][lane + 32 * k] = v[k];
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kEl; ++k) {
      const int e = lane + 32 * k;
      if (e < 2 * p.npairs) {
        const int i = half ? (e < p.npairs ? e : e - p.npairs) : e >> 1;
        const bool second = half ? e >= p.npairs : (e & 1);
        const float other = rows[warp][half ? (second ? i : i + p.npairs) : e ^ 1];
        const float2 cs = pair_turn<sizeof(T) == 2>(p, sh, pos, i);
        const float s = (BACK != second) ? cs.y : -cs.y;     // forward: a c - b s and b c + a s
        v[k] = fmaf(v[k], cs.x, other * s);
      }
    }
    if (BACK && norm) {
      const T* x = static_cast<const T*>(r.x) + b * r.xs[0] + n * r.xs[1] + h * r.xs[2];
      float xv[kEl], hx = 0.f;
      ss = 0.f;
#pragma unroll
      for (int k = 0; k < kEl; ++k) {
        const int e = lane + 32 * k;
        xv[k] = e < p.dim ? to_f<T>(x[e]) : 0.f;
        ss = fmaf(xv[k], xv[k], ss);
        if (e < p.dim) hx = fmaf(v[k] * sh.weight[e], xv[k], hx);
      }
      const float rs = rsqrtf(row_sum<32>(ss) * inv_dim + p.eps);
      const float back = row_sum<32>(hx) * inv_dim * rs * rs;
#pragma unroll
      for (int k = 0; k < kEl; ++k) {
        const int e = lane + 32 * k;
        if (e < p.dim) {
          dw[k] = fmaf(v[k], xv[k] * rs, dw[k]);
          v[k] = rs * fmaf(-xv[k], back, v[k] * sh.weight[e]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kEl; ++k) {
      const int e = lane + 32 * k;
      if (e < p.dim) out[e] = from_f<T>(v[k]);
    }
  }
  if (BACK && norm) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kEl; ++k) rows[warp][lane + 32 * k] = dw[k];
    __syncthreads();
    float* dst = partial + (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * p.dim;
    for (int e = threadIdx.x; e < p.dim; e += blockDim.x) {
      float s = 0.f;
      for (int g = 0; g < kRotWarps; ++g) s += rows[g][e];
      dst[e] = s;
    }
  }
}

// dweight[e] = the CTAs' partial sums in a fixed order: 32 interleaved sums, then those
__global__ void __launch_bounds__(1024)
    rotary_weight_kernel(const float* __restrict__ partial, int blocks, int dim, void* dw0, int dt0, void* dw1, int dt1) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int e = blockIdx.x * 32 + lane;
  void* dst = blockIdx.y ? dw1 : dw0;
  const int dt = blockIdx.y ? dt1 : dt0;
  if (dst == nullptr) return;
  const float* src = partial + static_cast<int64_t>(blockIdx.y) * blocks * dim;
  float s = 0.f;
  if (e < dim)
    for (int g = row; g < blocks; g += 32) s += src[static_cast<int64_t>(g) * dim + e];
  part[row][lane] = s;
  __syncthreads();
  if (row == 0 && e < dim) {
    s = 0.f;
    for (int g = 0; g < 32; ++g) s += part[g][lane];
    if (dt == HTRC_LAYER_F32) static_cast<float*>(dst)[e] = s;
    else if (dt == HTRC_LAYER_BF16) static_cast<__nv_bfloat16*>(dst)[e] = __float2bfloat16_rn(s);
    else static_cast<__half*>(dst)[e] = __float2half_rn(s);
  }
}

constexpr int kRotFlatHeads = 2;       // FLAT: see rotary_run
constexpr int kRotBlocksPerSm = 8;      // 256-thread CTAs per SM the grids are sized for

int rotary_max_blocks() { return sm_count() * kRotBlocksPerSm; }

int rotary_validate(const HtrcRotaryArgs* a, bool back, bool ptrs) {
  if (a == nullptr || a->n_tensors < 1 || a->n_tensors > 2) return HTRC_ERR_ARG;
  if (a->dtype < HTRC_LAYER_F32 || a->dtype > HTRC_LAYER_F16) return HTRC_ERR_ARG;
  if (a->batch < 0 || a->tokens < 0) return HTRC_ERR_ARG;
  constexpr int64_t kMaxRows = int64_t(1) << 32;      // more would not fit the device: the products below cannot overflow
  if (a->tokens > 0 && a->batch > kMaxRows / a->tokens) return HTRC_ERR_UNSUPPORTED;
  if (a->dim < 2 || a->n_axes < 1) return HTRC_ERR_ARG;
  if (a->dim > HTRC_ROTARY_MAX_DIM || a->n_axes > HTRC_ROTARY_MAX_AXES) return HTRC_ERR_UNSUPPORTED;
  int64_t width = 0;
  for (int i = 0; i < a->n_axes; ++i) {
    if (a->axis_width[i] < 0 || a->axis_width[i] % 2) return HTRC_ERR_ARG;
    width += a->axis_width[i];
  }
  if (width > a->dim) return HTRC_ERR_ARG;
  if (a->pairs != HTRC_ROTARY_INTERLEAVED && a->pairs != HTRC_ROTARY_HALF) return HTRC_ERR_ARG;
  if (a->position_dtype != HTRC_LAYER_I32 && a->position_dtype != HTRC_LAYER_F32) return HTRC_ERR_ARG;
  if (a->freqs == nullptr && !(a->theta > 0.0 && std::isfinite(a->theta))) return HTRC_ERR_ARG;
  if (!(a->eps >= 0.0f) || !std::isfinite(a->eps)) return HTRC_ERR_ARG;
  for (int i = 0; i < a->n_tensors; ++i) {
    const HtrcRotaryTensor& t = a->tensor[i];
    if (t.heads < 1) return HTRC_ERR_ARG;
    if (t.heads > HTRC_ROTARY_MAX_HEADS || a->batch * a->tokens * t.heads >= kMaxRows) return HTRC_ERR_UNSUPPORTED;
    if (t.weight_dtype < HTRC_LAYER_F32 || t.weight_dtype > HTRC_LAYER_F16) return HTRC_ERR_ARG;
    if (!ptrs || a->batch * a->tokens == 0) continue;
    if (!t.in || !t.out || !a->positions) return HTRC_ERR_ARG;
    if (back && t.weight && (!t.x || !t.dweight)) return HTRC_ERR_ARG;
  }
  return HTRC_OK;
}

bool aligned16(const void* p, const int64_t* s, int es) {
  if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (s[i] * es % 16) return false;
  return true;
}

// The pairs' axes and turns per position.  The last table without frequencies of the caller's own is kept per thread:
// its 64 powers cost more host time than the rest of a small call.
bool rotary_table(const HtrcRotaryArgs* a, RotaryParams* p) {
  struct Kept {
    double theta = 0.0;
    int n_axes = 0, width[HTRC_ROTARY_MAX_AXES] = {}, npairs = 0;
    bool floats = false;
    uint64_t turn[kRotMaxPairs];
    uint8_t axis[kRotMaxPairs];
  };
  static thread_local Kept kept;
  bool same = a->freqs == nullptr && kept.theta == a->theta && kept.n_axes == a->n_axes && kept.floats == p->float_positions;
  for (int x = 0; same && x < a->n_axes; ++x) same = kept.width[x] == a->axis_width[x];
  if (!same) {
    kept.theta = 0.0;                                               // no caller's theta: not kept until complete
    kept.npairs = 0;
    kept.floats = p->float_positions;
    for (int x = 0; x < a->n_axes; ++x) {
      kept.width[x] = a->axis_width[x];
      for (int i = 0; i < a->axis_width[x] / 2; ++i, ++kept.npairs) {
        const double f = (a->freqs ? a->freqs[kept.npairs] : std::pow(a->theta, -2.0 * i / a->axis_width[x])) *
                         0.15915494309189533577;                    // 1 / (2 pi): revolutions per position
        if (!std::isfinite(f)) return false;
        kept.axis[kept.npairs] = static_cast<uint8_t>(x);
        uint64_t& t = kept.turn[kept.npairs];
        if (kept.floats) {
          const float hi = static_cast<float>(f), lo = static_cast<float>(f - hi);
          uint32_t h, l;
          memcpy(&h, &hi, 4);
          memcpy(&l, &lo, 4);
          t = static_cast<uint64_t>(h) << 32 | l;
        } else {
          // the fraction of a revolution in 64 bits; whole revolutions per position turn nothing
          const double top = (f - std::floor(f)) * 0x1p32, hi = std::floor(top);
          t = (static_cast<uint64_t>(hi) << 32) + static_cast<uint64_t>((top - hi) * 0x1p32);
        }
      }
    }
    kept.n_axes = a->n_axes;
    if (a->freqs == nullptr) kept.theta = a->theta;
  }
  p->npairs = kept.npairs;
  memcpy(p->turn, kept.turn, kept.npairs * sizeof(kept.turn[0]));
  memcpy(p->axis, kept.axis, kept.npairs * sizeof(kept.axis[0]));
  return true;
}

template <typename T, int LPR, bool BACK, bool FLAT>
void run_rows(const RotaryParams& p, bool half, dim3 grid, float* partial, cudaStream_t st) {
  if (half) rotary_kernel<T, LPR, true, BACK, FLAT><<<grid, kRotWarps * 32, 0, st>>>(p, partial);
  else rotary_kernel<T, LPR, false, BACK, FLAT><<<grid, kRotWarps * 32, 0, st>>>(p, partial);
}

template <typename T, bool BACK, bool FLAT>
void run_dim(const RotaryParams& p, bool half, dim3 grid, float* partial, cudaStream_t st) {
  if (p.dim <= 64) run_rows<T, 8, BACK, FLAT>(p, half, grid, partial, st);
  else if (p.dim <= 128) run_rows<T, 16, BACK, FLAT>(p, half, grid, partial, st);
  else run_rows<T, 32, BACK, FLAT>(p, half, grid, partial, st);
}

template <bool BACK>
int rotary_run(const HtrcRotaryArgs* a, cudaStream_t st) {
  int rc = rotary_validate(a, BACK, true);
  if (rc != HTRC_OK) return rc;
  if (!device_is_b200()) return HTRC_ERR_DEVICE;
  RotaryParams p{};
  p.batch = a->batch;
  p.tokens = a->tokens;
  p.dim = a->dim;
  // The backward's warps are filled up with rows of zeros, which must add nothing to the weight's gradient: with eps = 0
  // their rsqrt(0) would make 0 * inf of it.  The smallest float instead, which changes no mean square that is a normal
  // number, costs nothing; leaving such rows out by a select in the loop took 237.6 us for 232.6 (32,768 tokens x 24 heads).
  p.eps = BACK ? std::max(a->eps, std::numeric_limits<float>::denorm_min()) : a->eps;
  p.positions = a->positions;
  p.float_positions = a->position_dtype == HTRC_LAYER_F32;
  for (int i = 0; i < 3; ++i) p.ps[i] = a->position_stride[i];
  if (!rotary_table(a, &p)) return HTRC_ERR_ARG;
  const int es = a->dtype == HTRC_LAYER_F32 ? 4 : 2;
  const bool half = a->pairs == HTRC_ROTARY_HALF;
  bool vec = a->dim % 8 == 0 && (!half || p.npairs % 4 == 0), any_weight = false;
  int64_t rows = a->batch * a->tokens;
  for (int i = 0; i < a->n_tensors; ++i) {
    const HtrcRotaryTensor& t = a->tensor[i];
    RotaryRows& r = p.t[i];
    r.in = t.in;
    r.out = t.out;
    r.x = t.x;
    r.weight = t.weight;
    r.weight_dtype = t.weight_dtype;
    r.heads = t.heads;
    for (int s = 0; s < 3; ++s) {
      r.is[s] = t.in_stride[s];
      r.os[s] = t.out_stride[s];
      r.xs[s] = t.x_stride[s];
    }
    any_weight |= t.weight != nullptr;
    vec = vec && aligned16(t.in, t.in_stride, es) && aligned16(t.out, t.out_stride, es) &&
          (!(BACK && t.weight) || aligned16(t.x, t.x_stride, es));
  }
  const bool partials = BACK && any_weight;
  size_t need = 0;
  if (partials) {
    htrc_rotary_workspace_size(a, &need);
    if (a->workspace == nullptr || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16)
      return HTRC_ERR_WORKSPACE;
  }
  const int lpr = a->dim <= 64 ? 8 : a->dim <= 128 ? 16 : 32;
  // few heads: a warp's rows come from several tokens, each with angles of its own, rather than leave lanes idle.
  // q and k of 32,768 tokens x 128, bfloat16: 1 head 17.9 us against 40.3, 4 heads 58.1 against 44.3; of 16,384 tokens
  // x 2 heads 17.9 against 22.6, backward of 32,768 x 2 58.9 against 89.1
  bool flat = true;
  for (int i = 0; i < a->n_tensors; ++i) {
    flat = flat && a->tensor[i].heads <= kRotFlatHeads;
    vec = vec && rows * a->tensor[i].heads < int64_t{1} << 31;      // its task numbers are 32-bit
  }
  int64_t blocks = 1;
  for (int i = 0; i < a->n_tensors; ++i) {
    RotaryRows& r = p.t[i];
    // heads per warp: all of a token's, whose angles are then formed once, where the tokens alone give every SM 8
    // warps; else the token's heads are shared out until they do.  1,024 tokens x 24 heads: 7.8 us shared out, 31.5 not;
    // 16,384 tokens: 83 us shared out twice as far, 72 not
    const int batch_rows = 32 / lpr;
    const int64_t most = (r.heads + batch_rows - 1) / batch_rows, want = 8 * sm_count();
    const int64_t parts = rows > 0 ? std::min(most, (want + rows - 1) / rows) : 1;
    r.chunk = static_cast<int>((most + parts - 1) / parts) * batch_rows;
    r.chunks = (r.heads + r.chunk - 1) / r.chunk;
    const int64_t per = 32 / lpr * rot_unroll(BACK);
    const int64_t tasks = !vec ? rows * r.heads : flat ? (rows * r.heads + per - 1) / per : rows * r.chunks;
    blocks = std::max(blocks, (tasks + kRotWarps - 1) / kRotWarps);
  }
  blocks = std::min<int64_t>(blocks, rotary_max_blocks());
  float* partial = static_cast<float*>(a->workspace);
  const dim3 grid(static_cast<unsigned>(blocks), a->n_tensors);
  if (rows > 0 || partials) {
    auto go = [&](auto tag) {
      using T = decltype(tag);
      if (vec && flat) run_dim<T, BACK, true>(p, half, grid, partial, st);
      else if (vec) run_dim<T, BACK, false>(p, half, grid, partial, st);
      else rotary_any_kernel<T, BACK><<<grid, kRotWarps * 32, 0, st>>>(p, half, partial);
    };
    if (a->dtype == HTRC_LAYER_F32) go(float{});
    else if (a->dtype == HTRC_LAYER_BF16) go(__nv_bfloat16{});
    else go(__half{});
    if (partials) {
      const HtrcRotaryTensor &t0 = a->tensor[0], &t1 = a->tensor[a->n_tensors - 1];
      rotary_weight_kernel<<<dim3((a->dim + 31) / 32, a->n_tensors), 1024, 0, st>>>(
          partial, static_cast<int>(blocks), a->dim, t0.weight ? t0.dweight : nullptr, t0.weight_dtype,
          t1.weight ? t1.dweight : nullptr, t1.weight_dtype);
    }
  }
  return cudaGetLastError() == cudaSuccess ? HTRC_OK : HTRC_ERR_CUDA;
}

}  // namespace

}  // namespace htrc

extern "C" {

int htrc_rotary_forward(const HtrcRotaryArgs* args, htrc_stream_t stream) {
  return htrc::rotary_run<false>(args, reinterpret_cast<cudaStream_t>(stream));
}

int htrc_rotary_workspace_size(const HtrcRotaryArgs* args, size_t* bytes) {
  if (bytes == nullptr) return HTRC_ERR_ARG;
  const int rc = htrc::rotary_validate(args, false, false);
  if (rc != HTRC_OK) return rc;
  *bytes = static_cast<size_t>(2) * htrc::rotary_max_blocks() * args->dim * sizeof(float);
  return HTRC_OK;
}

int htrc_rotary_backward(const HtrcRotaryArgs* args, htrc_stream_t stream) {
  return htrc::rotary_run<true>(args, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
