// Layer norm over the last axis, with the residual sum in front of it, and its backward.
//   s = x (+ r), mu = mean s, rstd = (mean (s - mu)^2 + eps)^-1/2, xh = (s - mu) rstd, y = xh w + b
//   t = gy w, gs = rstd (t - mean t - xh mean(t xh)) (+ g_sum), gw = sum_rows gy xh, gb = sum_rows gy
// DROP: s = drop(x) + r with the mask of egnn_random.h, and in the backward gx = drop(gs) beside gs, the residual's gradient:
// two tensors fewer to write and read again than with a dropout of its own, and the mask is made in registers, twice.  40,961 x
// 259 fp32, forward and backward 37.6 and 48.4 us, 4.5 and 4.4 TB/s; 19,456 x 128 bf16 8.4 and 8.1 us, launches; 2,000,000 x 128
// bf16, with what the sum's rounding loses (Low), forward and backward 906 us, and 943 beside fp32 parameters, 5.7 and 6.0 TB/s.
// A row lives in the registers of LPR lanes, so it is read once and the variance is taken around the mean.  The backward's
// blocks walk the rows with a fixed stride; a lane keeps the sums of gw and gb of its columns in fp32 registers, a
// block's row groups are joined in LDS and its sums leave as one partial row, which a second launch adds up in order.
// y is made from the sum as it is, before it is rounded to the type it is stored in.  The backward reads the stored one, so
// where the mean exceeds the deviation the statistics kept for it are those of the stored one: with the others a row whose
// values differ by less than their rounding would get any gradient (one column of bf16: hundreds of times too large, instead
// of 0).  Elsewhere the two agree to 2^-8 of the deviation.  (For every row: 402 us instead of 360, 2,000,000 x 128 bf16.)
// Bound by HBM where the tensors are large: 2,000,000 x 128 bf16 with a residual, forward 337 us and backward 323 us, 6.1 and
// 6.3 TB/s (each kernel alone, called back to back); 40,961 x 259 fp32, rows that cross lines, 18.4 and 23.6 us, 4.6 and 5.4
// TB/s.  By its launches where they are small: 2,432 x 128 fp32, forward, 2.8 us.  Rows wider than a wave's registers are read
// value by value, twice or three times: 20,000 x 4,096 bf16, forward and backward, 265 and 395 us, floors 64 and 95.
#pragma once
#include "egnn_device.h"
#include "egnn_internal.h"
#include "egnn_random.h"
#include "egnn_rows.h"

namespace egnn {
namespace norm {

struct Args {
  const void *x, *r, *w, *b, *gy, *gsum;
  void *y, *s, *gx, *gw, *gb;
  float *mean, *rstd, *part;
  int64_t N, ldx, ldr, ldg, ldgs;
  int32_t C;
  float eps;
  bool f32_params;                           // w, b, gw and gb are fp32 beside bf16 rows
  void* gr;                                  // DROP: the residual's gradient, gs
  void* low;                                 // DROP: what the stored sum's rounding lost (Low), or NULL
  int64_t row0;                              // DROP: the first row's number
  DropArgs d;
};

constexpr int NT = 256;

// What a bf16 sum's rounding lost: the fp32 value's bits less those of the rounded one, -32,768 to 32,768 of them, in full (L =
// int16_t: the two make the value again, but for one unit in 2^23 at ties) or in steps of 256 (int8_t: to 128 units, 2^-16 of
// the value at most, and to 256 in the one of 512 values that lie past the byte's 127 steps; in steps of 257 none would, but sums
// that cancelled, whose last 8 bits are 0, would no longer come back whole).  From the rounded sum alone the gradients would
// carry its rounding, up to 2^-8: as much again as their own where they are bf16 (errors of gw 2.5e-3 to 3.9e-3 of its norm,
// 1.7e-3 with the byte), and 10^4 times as much where the parameters are fp32.
template <typename L, bool TAIL> struct Low {
  typedef L type __attribute__((ext_vector_type(8), aligned(sizeof(L))));
  typedef L piece __attribute__((ext_vector_type(8)));
  static constexpr int kShift = sizeof(L) == 2 ? 0 : 8, kMost = sizeof(L) == 2 ? 32767 : 127;
  static __device__ __forceinline__ L of(float v) {
    const int32_t d = (int32_t)(__float_as_uint(v) - __float_as_uint((float)(bf16)v));
    return (L)min(max(kShift ? (d + 128) >> kShift : d, -kMost - 1), kMost);
  }
  static __device__ __forceinline__ float with(float rounded, L d) {
    return __uint_as_float(__float_as_uint(rounded) + ((uint32_t)(int32_t)d << kShift));
  }
  template <bool PAST> static __device__ __forceinline__ piece load(const L* p, int f, int C) {
    piece t;
    if (!TAIL || C >= 8) {
      if constexpr (PAST) t = __builtin_nontemporal_load(reinterpret_cast<const type*>(p + f));
      else t = *reinterpret_cast<const type*>(p + f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = i < C ? p[i] : (L)0;
    }
    return t;
  }
  static __device__ __forceinline__ void store(L* p, int f, int C, const float* v) {
    if (!TAIL || C >= 8) {
      type t;
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = of(v[i]);
      *reinterpret_cast<type*>(p + f) = t;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < C) p[i] = of(v[i]);
    }
  }
};
// Without dropout, with it, and with what the sum's rounding lost in 16 or 8 bits
enum { kPlain, kDrop, kDropLow, kDropByte };
template <int D> struct LowOf { typedef int16_t type; };
template <> struct LowOf<kDropByte> { typedef int8_t type; };

template <typename T, typename P, int LPR, int VPL, bool TAIL, int D>
__global__ __launch_bounds__(NT) void fwd_kernel(Args a) {
  typedef Vec<T, TAIL> V;
  constexpr bool DROP = D != kPlain, LOW = D >= kDropLow;
  typedef typename LowOf<D>::type L;
  constexpr int VEC = V::N;
  const int lane = threadIdx.x % LPR;
  const int64_t n = (int64_t)blockIdx.x * (NT / LPR) + threadIdx.x / LPR;
  const bool live = n < a.N;
  float v[VPL][VEC];
  Piece c[VPL];
#pragma unroll
  for (int p = 0; p < VPL; ++p) {
    c[p] = piece_of<VEC, TAIL>(p * LPR + lane, a.C);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[p][i] = 0.f;
    if (!DROP && live && c[p].in) V::load((const T*)a.x + n * a.ldx, c[p].f, a.C, v[p]);
  }
  if constexpr (DROP) {
    typename V::piece x[VPL], r[VPL];
#pragma unroll
    for (int p = 0; p < VPL; ++p)
      if (live && c[p].in) {
        x[p] = V::load((const T*)a.x + n * a.ldx, c[p].f, a.C);
        r[p] = V::load((const T*)a.r + n * a.ldr, c[p].f, a.C);
      }
    const Mask m = mask_of(a.d);
#pragma unroll
    for (int p = 0; p < VPL; ++p)
      if (live && c[p].in) {
        float e[VEC];
        V::floats(x[p], v[p]);
        V::floats(r[p], e);
        drop<VEC, TAIL>(m, (uint32_t)(a.row0 + n), c[p].f, v[p]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[p][i] += e[i];
        V::store((T*)a.s + n * a.C, c[p].f, a.C, v[p]);
        if constexpr (LOW) Low<L, TAIL>::store((L*)a.low + n * a.C, c[p].f, a.C, v[p]);
      }
  } else if (a.r) {
    typename V::piece r[VPL];
#pragma unroll
    for (int p = 0; p < VPL; ++p)
      if (live && c[p].in) r[p] = V::load((const T*)a.r + n * a.ldr, c[p].f, a.C);
#pragma unroll
    for (int p = 0; p < VPL; ++p)
      if (live && c[p].in) {
        float x[VEC];
        V::floats(r[p], x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[p][i] += x[i];
        V::store((T*)a.s + n * a.C, c[p].f, a.C, v[p]);
      }
  }
  // mean and rstd of the row, or (ROUND) of the row as it is stored
  float mean, rstd;
  auto stats = [&](auto round, float& mean, float& rstd) {
    constexpr bool ROUND = decltype(round)::value;
    auto at = [&](int p, int i) {
      if (!ROUND) return v[p][i];
      const float h = to_f32(from_f32<T>(v[p][i]));
      return LOW ? Low<L, TAIL>::with(h, Low<L, TAIL>::of(v[p][i])) : h;
    };
    float sum = 0.f;
#pragma unroll
    for (int p = 0; p < VPL; ++p)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += (!TAIL || i >= c[p].skip) ? at(p, i) : 0.f;
    mean = row_sum<LPR>(sum) / a.C;
    float sq = 0.f;
#pragma unroll
    for (int p = 0; p < VPL; ++p)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = at(p, i) - mean;
        if (c[p].in && (!TAIL || (i >= c[p].skip && i < a.C))) sq = __builtin_fmaf(d, d, sq);
      }
    rstd = 1.0f / sqrtf(row_sum<LPR>(sq) / a.C + a.eps);
  };
  stats(std::false_type{}, mean, rstd);
  if (a.mean) {
    float m = mean, rs = rstd;
    if (sizeof(T) == 2 && a.r) {
      const bool far = mean * mean * rstd * rstd > 1.f;
      if (__ballot(far)) {
        stats(std::true_type{}, m, rs);
        if (!far) { m = mean; rs = rstd; }
      }
    }
    if (live && lane == 0) { a.mean[n] = m; a.rstd[n] = rs; }
  }
  if (!live) return;
#pragma unroll
  for (int p = 0; p < VPL; ++p) {
    if (c[p].in) {
      float w[VEC], b[VEC], y[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) { w[i] = 1.f; b[i] = 0.f; }
      if (a.w) load_params<T, P, TAIL>(a.w, c[p].f, a.C, w);
      if (a.b) load_params<T, P, TAIL>(a.b, c[p].f, a.C, b);
#pragma unroll
      for (int i = 0; i < VEC; ++i) y[i] = __builtin_fmaf((v[p][i] - mean) * rstd, w[i], b[i]);
      V::store((T*)a.y + n * a.C, c[p].f, a.C, y);
    }
  }
}

// PAST: 1: the result is stored past the cache, 2: the operands are read past it too (egnn_rows.h).  60,000 x 512 fp32, 123 MB:
// 71, 58 and 67 us at 0, 1 and 2; 40,961 x 259, 42 MB: 32.0 and 33.3 at 0 and 1; 2,000,000 x 128 bf16: 347 and 325 at 1 and 2.
template <typename T, int LPR, int VPL, int PAST, bool TAIL, int D>
__global__ __launch_bounds__(NT) void bwd_kernel(Args a) {
  typedef Vec<T, TAIL> V;
  constexpr bool DROP = D != kPlain, LOW = D >= kDropLow;
  typedef typename LowOf<D>::type L;
  constexpr int VEC = V::N, RG = NT / LPR, W = LPR * VPL * VEC;
  __shared__ float red[RG][W];
  const int lane = threadIdx.x % LPR, rg = threadIdx.x / LPR;
  float gw[VPL][VEC], gb[VPL][VEC], w[VPL][VEC];
  Piece c[VPL];
#pragma unroll
  for (int p = 0; p < VPL; ++p) {
    c[p] = piece_of<VEC, TAIL>(p * LPR + lane, a.C);
#pragma unroll
    for (int i = 0; i < VEC; ++i) { gw[p][i] = 0.f; gb[p][i] = 0.f; w[p][i] = 1.f; }
    if (a.w && c[p].in) {                    // (once a block: no kernel of its own for fp32 parameters)
      if (sizeof(T) == 2 && a.f32_params) load_params<T, float, TAIL>(a.w, c[p].f, a.C, w[p]);
      else load_params<T, T, TAIL>(a.w, c[p].f, a.C, w[p]);
    }
  }
  const Mask m = DROP ? mask_of(a.d) : Mask{};
  const int64_t step = (int64_t)gridDim.x * RG;
  typename V::piece pg[VPL], px[VPL], pe[VPL];
  typename Low<L, TAIL>::piece pl[LOW ? VPL : 1];
  float mean = 0.f, rstd = 0.f;
  // everything a row needs, requested at once; without branches, which would make the loop wait for the loads they join
  // (2,000,000 x 128 bf16: 409 us, and 326 without).  Past the rows, and in lanes without a piece, what is there is read
  // again.
  auto fetch = [&](int64_t n) {
    n = n < a.N ? n : a.N - 1;
    mean = a.mean[n];
    rstd = a.rstd[n];
#pragma unroll
    for (int p = 0; p < VPL; ++p) {
      pg[p] = V::template load<PAST == 2>((const T*)a.gy + n * a.ldg, c[p].f, a.C);
      px[p] = V::template load<PAST == 2>((const T*)a.x + n * a.ldx, c[p].f, a.C);
      if (a.gsum) pe[p] = V::template load<PAST == 2>((const T*)a.gsum + n * a.ldgs, c[p].f, a.C);
      if constexpr (LOW) pl[p] = Low<L, TAIL>::template load<PAST == 2>((const L*)a.low + n * a.C, c[p].f, a.C);
    }
  };
  int64_t n = (int64_t)blockIdx.x * RG + rg;
  fetch(n);
  for (; n - rg < a.N; n += step) {
    const bool live = n < a.N;
    float xh[VPL][VEC], t[VPL][VEC], e[VPL][VEC];
    float s1 = 0.f, s2 = 0.f;
    const float mu = mean, rs = rstd;
#pragma unroll
    for (int p = 0; p < VPL; ++p) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) { t[p][i] = 0.f; xh[p][i] = mu; e[p][i] = 0.f; }
      if (live && c[p].in) {
        V::floats(pg[p], t[p]);
        V::floats(px[p], xh[p]);
        if constexpr (LOW)
#pragma unroll
          for (int i = 0; i < VEC; ++i) xh[p][i] = Low<L, TAIL>::with(xh[p][i], (L)pl[p][i]);
        if (a.gsum) V::floats(pe[p], e[p]);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        xh[p][i] = (xh[p][i] - mu) * rs;
        gw[p][i] = __builtin_fmaf(t[p][i], xh[p][i], gw[p][i]);
        gb[p][i] += t[p][i];
        t[p][i] *= w[p][i];
        const float own = (!TAIL || i >= c[p].skip) ? t[p][i] : 0.f;
        s1 += own;
        s2 = __builtin_fmaf(own, xh[p][i], s2);
      }
    }
    fetch(n + step);
    const float m1 = row_sum<LPR>(s1) / a.C, m2 = row_sum<LPR>(s2) / a.C;
#pragma unroll
    for (int p = 0; p < VPL; ++p) {
      if (live && c[p].in) {
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = __builtin_fmaf(rs, t[p][i] - m1 - xh[p][i] * m2, e[p][i]);
        if constexpr (DROP) {
          V::template store<(PAST > 0)>((T*)a.gr + n * a.C, c[p].f, a.C, o);
          drop<VEC, TAIL>(m, (uint32_t)n, c[p].f, o);
        }
        V::template store<(PAST > 0)>((T*)a.gx + n * a.C, c[p].f, a.C, o);
      }
    }
  }
  if (!a.part) return;
  float* out = a.part + (int64_t)blockIdx.x * 2 * a.C;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    __syncthreads();
#pragma unroll
    for (int p = 0; p < VPL; ++p)
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (c[p].in && (!TAIL || i >= c[p].skip)) red[rg][c[p].f + i] = half ? gb[p][i] : gw[p][i];
    __syncthreads();
    for (int f = threadIdx.x; f < a.C; f += NT) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < RG; ++k) s += red[k][f];
      out[half * a.C + f] = s;
    }
  }
}

// rows wider than a wave's registers: one block a row, the row read again (from cache) for each pass
__device__ __forceinline__ float block_sum(float v, float* buf) {
  v = row_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  return buf[0] + buf[1] + buf[2] + buf[3];
}
// (DROP: a thread takes 4 columns in a row, half of what one run of the generator makes; else one)
template <int S, typename F> __device__ __forceinline__ void columns(int C, F go) {
  for (int f = S * threadIdx.x; f < C; f += S * NT) go(f);
}
template <typename T, typename P, int D>
__global__ __launch_bounds__(NT) void fwd_wide_kernel(Args a) {
  __shared__ float buf[4];
  constexpr bool DROP = D != kPlain, LOW = D >= kDropLow;
  typedef typename LowOf<D>::type L;
  constexpr int S = DROP ? 4 : 1;
  const int64_t n = blockIdx.x;
  const T *x = (const T*)a.x + n * a.ldx, *r = a.r ? (const T*)a.r + n * a.ldr : nullptr;
  const Mask m = DROP ? mask_of(a.d) : Mask{};
  // the sums of columns f .. f + S - 1, and how many of them there are
  auto vals = [&](int f, float* v) {
#pragma unroll
    for (int i = 0; i < S; ++i) v[i] = f + i < a.C ? to_f32(x[f + i]) : 0.f;
    if constexpr (DROP) drop<4, false>(m, (uint32_t)(a.row0 + n), f, v);
#pragma unroll
    for (int i = 0; i < S; ++i) v[i] += r && f + i < a.C ? to_f32(r[f + i]) : 0.f;
    return a.C - f < S ? a.C - f : S;
  };
  auto stored = [&](float x) {
    const float h = to_f32(from_f32<T>(x));
    return LOW ? Low<L, true>::with(h, Low<L, true>::of(x)) : h;
  };
  auto stats = [&](bool round, float& mean, float& rstd) {
    float s = 0.f;
    columns<S>(a.C, [&](int f) {
      float v[S];
      const int k = vals(f, v);
#pragma unroll
      for (int i = 0; i < S; ++i)
        if (i < k) s += round ? stored(v[i]) : v[i];
    });
    mean = block_sum(s, buf) / a.C;
    float q = 0.f;
    columns<S>(a.C, [&](int f) {
      float v[S];
      const int k = vals(f, v);
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const float d = (round ? stored(v[i]) : v[i]) - mean;
        if (i < k) q = __builtin_fmaf(d, d, q);
      }
    });
    rstd = 1.0f / sqrtf(block_sum(q, buf) / a.C + a.eps);
  };
  float mean, rstd;
  stats(false, mean, rstd);
  if (a.mean) {
    float m = mean, rs = rstd;
    if (sizeof(T) == 2 && r && mean * mean * rstd * rstd > 1.f) stats(true, m, rs);
    if (threadIdx.x == 0) { a.mean[n] = m; a.rstd[n] = rs; }
  }
  columns<S>(a.C, [&](int f) {
    float v[S];
    const int k = vals(f, v);
#pragma unroll
    for (int i = 0; i < S; ++i) {
      if (i >= k) break;
      const float w = a.w ? param<P>(a.w, f + i) : 1.f, b = a.b ? param<P>(a.b, f + i) : 0.f;
      if (r) ((T*)a.s)[n * a.C + f + i] = from_f32<T>(v[i]);
      if (LOW) ((L*)a.low)[n * a.C + f + i] = Low<L, true>::of(v[i]);
      ((T*)a.y)[n * a.C + f + i] = from_f32<T>(__builtin_fmaf((v[i] - mean) * rstd, w, b));
    }
  });
}
template <typename T, typename P, int D>
__global__ __launch_bounds__(NT) void bwd_wide_kernel(Args a) {
  __shared__ float buf[4];
  constexpr bool DROP = D != kPlain, LOW = D >= kDropLow;
  typedef typename LowOf<D>::type L;
  const int64_t n = blockIdx.x;
  const T *x = (const T*)a.x + n * a.ldx, *g = (const T*)a.gy + n * a.ldg;
  const float mean = a.mean[n], rstd = a.rstd[n];
  auto sum_at = [&](int f) { return LOW ? Low<L, true>::with(to_f32(x[f]), ((const L*)a.low)[n * a.C + f]) : to_f32(x[f]); };
  float s1 = 0.f, s2 = 0.f;
  for (int f = threadIdx.x; f < a.C; f += NT) {
    const float t = to_f32(g[f]) * (a.w ? param<P>(a.w, f) : 1.f);
    s1 += t;
    s2 = __builtin_fmaf(t, (sum_at(f) - mean) * rstd, s2);
  }
  const float m1 = block_sum(s1, buf) / a.C, m2 = block_sum(s2, buf) / a.C;
  constexpr int S = DROP ? 4 : 1;
  const Mask m = DROP ? mask_of(a.d) : Mask{};
  columns<S>(a.C, [&](int f) {
    float o[S];
    const int k = a.C - f < S ? a.C - f : S;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      o[i] = 0.f;
      if (i >= k) break;
      const float t = to_f32(g[f + i]) * (a.w ? param<P>(a.w, f + i) : 1.f);
      o[i] = rstd * (t - m1 - (sum_at(f + i) - mean) * rstd * m2);
      if (a.gsum) o[i] += to_f32(((const T*)a.gsum)[n * a.ldgs + f + i]);
      if (DROP) ((T*)a.gr)[n * a.C + f + i] = from_f32<T>(o[i]);
    }
    if constexpr (DROP) drop<4, false>(m, (uint32_t)(a.row0 + n), f, o);
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (i < k) ((T*)a.gx)[n * a.C + f + i] = from_f32<T>(o[i]);
  });
}
// gw and gb of wide rows: a thread a column, rows of one of gridDim.y parts
template <typename T, int D>
__global__ __launch_bounds__(NT) void bwd_wide_weights_kernel(Args a) {
  const int f = blockIdx.x * NT + threadIdx.x;
  if (f >= a.C) return;
  float gw = 0.f, gb = 0.f;
  for (int64_t n = blockIdx.y; n < a.N; n += gridDim.y) {
    const float g = to_f32(((const T*)a.gy)[n * a.ldg + f]);
    float v = to_f32(((const T*)a.x)[n * a.ldx + f]);
    if (D >= kDropLow) v = Low<typename LowOf<D>::type, true>::with(v, ((const typename LowOf<D>::type*)a.low)[n * a.C + f]);
    gw = __builtin_fmaf(g, (v - a.mean[n]) * a.rstd[n], gw);
    gb += g;
  }
  float* out = a.part + (int64_t)blockIdx.y * 2 * a.C;
  out[f] = gw;
  out[a.C + f] = gb;
}

// gw, gb = sums of the partial rows: 16 columns a block, 64 row groups joined in order
template <typename T>
__global__ __launch_bounds__(1024) void sum_kernel(const float* part, int nblk, int C, T* gw, T* gb) {
  __shared__ float red[64][17];
  const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
  const int f = blockIdx.x * 16 + c;
  float s = 0.f;
  if (f < 2 * C) {
#pragma unroll 8
    for (int b = k; b < nblk; b += 64) s += part[(int64_t)b * 2 * C + f];
  }
  red[k][c] = s;
  __syncthreads();
  for (int h = 32; h; h >>= 1) {
    if (k < h) red[k][c] += red[k + h][c];
    __syncthreads();
  }
  if (k || f >= 2 * C) return;
  s = red[0][c];
  if (f < C) { if (gw) gw[f] = from_f32<T>(s); }
  else if (gb) gb[f - C] = from_f32<T>(s);
}

// Blocks of the backward, and partial rows of the weight gradients: two a CU.  2,000,000 x 128 bf16 with a sum's gradient:
// 434, 368, 414 and 475 us at 256, 512, 1,024 and 4,096 blocks.
constexpr int kMaxBlocks = 512;

// Lanes and pieces of a row: the fewest lane slots that hold it.  Three pieces a lane instead of idle lanes only where the
// rows are many (the next power of two and three pieces, forward + backward in us: 300,000 x 160 fp32 242 and 176;
// 1,351,820 x 164 bf16 700 and 558; 20,000 x 164 19.3 and 21.3).
constexpr int64_t kManyRows = 65536;
struct Shape { int lpr, vpl; };
static bool shape_of(int pieces, int64_t rows, Shape* s) {
  static const Shape all[] = {{4, 1},  {8, 1},  {4, 3},  {16, 1}, {8, 3},  {32, 1}, {16, 3},
                              {64, 1}, {32, 3}, {64, 2}, {64, 3}, {64, 4}, {64, 6}};
  for (const Shape& x : all)
    if (x.lpr * x.vpl >= pieces && (x.vpl == 1 || x.lpr >= 32 || rows >= kManyRows)) { *s = x; return true; }
  return false;
}
// Partial rows of the backward: a block makes several rounds over its row groups where there are enough rows, so that
// the sums over the partial rows stay small
static int64_t part_rows(int64_t N) {
  const int64_t n = cdiv(N, 32);
  return n < 1 ? 1 : (n < kMaxBlocks ? n : kMaxBlocks);
}

// A launch may have fewer than 2^32 threads, and there may be more rows than that leaves room for (2^24 of the wide ones):
// at most kMaxGrid blocks at a time, go(args, blocks) of the rows from one launch's first on.  A part is 1 GB of rows or
// more, beside which its launch does not show.
constexpr int64_t kMaxGrid = int64_t(1) << 20;
template <typename T, typename Go>
static void in_parts(const Args& a, int rows_per_block, Go go) {
  const int64_t most = kMaxGrid * rows_per_block;
  for (int64_t n = 0; n < a.N; n += most) {
    Args x = a;
    auto at = [&](const void* p, int64_t ld) -> const void* { return p ? (const T*)p + n * ld : nullptr; };
    x.x = at(a.x, a.ldx); x.r = at(a.r, a.ldr); x.gy = at(a.gy, a.ldg); x.gsum = at(a.gsum, a.ldgs);
    x.y = (void*)at(a.y, a.C); x.s = (void*)at(a.s, a.C); x.gx = (void*)at(a.gx, a.C); x.gr = (void*)at(a.gr, a.C);
    x.low = a.low ? (char*)a.low + n * a.C * (a.f32_params ? 2 : 1) : nullptr;
    x.row0 = n;
    x.mean = a.mean ? a.mean + n : nullptr; x.rstd = a.rstd ? a.rstd + n : nullptr;
    x.N = a.N - n < most ? a.N - n : most;
    go(x, (uint32_t)cdiv(x.N, rows_per_block));
  }
}

template <typename T, int LPR, int VPL, bool TAIL, int D>
static void launch_tail(const Args& a, bool bwd, hipStream_t st, int* nblk) {
  if (!bwd) {
    in_parts<T>(a, NT / LPR, [&](const Args& x, uint32_t blocks) {
      if (sizeof(T) == 2 && a.f32_params) fwd_kernel<T, float, LPR, VPL, TAIL, D><<<blocks, NT, 0, st>>>(x);
      else fwd_kernel<T, T, LPR, VPL, TAIL, D><<<blocks, NT, 0, st>>>(x);
    });
    return;
  }
  const int64_t n = cdiv(a.N, NT / LPR);
  *nblk = (int)(n < part_rows(a.N) ? n : part_rows(a.N));
  const int64_t bytes = a.N * a.C * (int64_t)sizeof(T);
  if (bytes >= kPastLoad) bwd_kernel<T, LPR, VPL, 2, TAIL, D><<<(uint32_t)*nblk, NT, 0, st>>>(a);
  else if (bytes >= kPastStore) bwd_kernel<T, LPR, VPL, 1, TAIL, D><<<(uint32_t)*nblk, NT, 0, st>>>(a);
  else bwd_kernel<T, LPR, VPL, 0, TAIL, D><<<(uint32_t)*nblk, NT, 0, st>>>(a);
}
template <typename T, int LPR, int VPL, int D>
static void launch_shape(const Args& a, bool bwd, hipStream_t st, int* nblk) {
  if (a.C % Vec<T>::N) launch_tail<T, LPR, VPL, true, D>(a, bwd, st, nblk);
  else launch_tail<T, LPR, VPL, false, D>(a, bwd, st, nblk);
}
template <typename T, int D>
static void launch_rows(const Args& a, const Shape& s, bool bwd, hipStream_t st, int* nblk) {
  switch (s.lpr * 8 + s.vpl - 1) {
    case 32: return launch_shape<T, 4, 1, D>(a, bwd, st, nblk);
    case 34: return launch_shape<T, 4, 3, D>(a, bwd, st, nblk);
    case 64: return launch_shape<T, 8, 1, D>(a, bwd, st, nblk);
    case 128: return launch_shape<T, 16, 1, D>(a, bwd, st, nblk);
    case 256: return launch_shape<T, 32, 1, D>(a, bwd, st, nblk);
    case 66: return launch_shape<T, 8, 3, D>(a, bwd, st, nblk);
    case 130: return launch_shape<T, 16, 3, D>(a, bwd, st, nblk);
    case 258: return launch_shape<T, 32, 3, D>(a, bwd, st, nblk);
    case 512: return launch_shape<T, 64, 1, D>(a, bwd, st, nblk);
    case 513: return launch_shape<T, 64, 2, D>(a, bwd, st, nblk);
    case 514: return launch_shape<T, 64, 3, D>(a, bwd, st, nblk);
    case 515: return launch_shape<T, 64, 4, D>(a, bwd, st, nblk);
    default: return launch_shape<T, 64, 6, D>(a, bwd, st, nblk);
  }
}

template <typename T, typename P, int D>
static void launch_wide(const Args& a, bool bwd, hipStream_t st) {
  in_parts<T>(a, 1, [&](const Args& x, uint32_t blocks) {
    if (bwd) bwd_wide_kernel<T, P, D><<<blocks, NT, 0, st>>>(x);
    else fwd_wide_kernel<T, P, D><<<blocks, NT, 0, st>>>(x);
  });
}
template <typename T, int D>
static int launch(const Args& a, bool bwd, hipStream_t st) {
  Shape s;
  int nblk = 0;
  if (a.N) {
    const bool narrow = shape_of((int)cdiv(a.C, Vec<T>::N), a.N, &s);
    if (narrow) launch_rows<T, D>(a, s, bwd, st, &nblk);
    else if (a.f32_params) launch_wide<T, float, D>(a, bwd, st);
    else launch_wide<T, T, D>(a, bwd, st);
    if (!narrow && bwd && a.part) {
      nblk = (int)(part_rows(a.N) < 128 ? part_rows(a.N) : 128);
      bwd_wide_weights_kernel<T, D><<<dim3((uint32_t)cdiv(a.C, NT), (uint32_t)nblk), NT, 0, st>>>(a);
    }
  }
  if (bwd && a.part) {
    const uint32_t blocks = (uint32_t)cdiv(2 * (int64_t)a.C, 16);
    if (a.f32_params) sum_kernel<float><<<blocks, 1024, 0, st>>>(a.part, nblk, a.C, (float*)a.gw, (float*)a.gb);
    else sum_kernel<T><<<blocks, 1024, 0, st>>>(a.part, nblk, a.C, (T*)a.gw, (T*)a.gb);
  }
  return hipGetLastError() == hipSuccess ? EGNN_OK : EGNN_ERR_HIP;
}

inline bool dims_ok(const EgnnNormDims* d) {
  return d->N >= 0 && d->N <= INT32_MAX && d->C >= 1 && d->C <= 1 << 20 && (d->dtype == EGNN_F32 || d->dtype == EGNN_BF16) &&
         d->eps >= 0.f && d->eps - d->eps == 0.f && (d->f32_params == 0 || d->f32_params == 1);
}

}  // namespace norm
}  // namespace egnn
