// Layer norm over the last axis, with the residual sum in front of it, and its backward.
//   s = x (+ r), mu = mean s, rstd = (mean (s - mu)^2 + eps)^-1/2, xh = (s - mu) rstd, y = xh w + b
//   t = gy w, gs = rstd (t - mean t - xh mean(t xh)) (+ g_sum), gw = sum_rows gy xh, gb = sum_rows gy
// A row lives in the registers of LPR lanes, so it is read once and the variance is taken around the mean.  The backward's
// blocks walk the rows with a fixed stride; a lane keeps the sums of gw and gb of its columns in fp32 registers, a
// block's row groups are joined in LDS and its sums leave as one partial row, which a second launch adds up in order.
// y is made from the sum as it is, before it is rounded to the type it is stored in.  The backward reads the stored one, so
// where the mean exceeds the deviation the statistics kept for it are those of the stored one: with the others a row whose
// values differ by less than their rounding would get any gradient (one column of bf16: hundreds of times too large, instead
// of 0).  Elsewhere the two agree to 2^-9 of the deviation.  (For every row: 402 us instead of 360, 2,000,000 x 128 bf16.)
// Bound by HBM where the tensors are large: 2,000,000 x 128 bf16 with a residual, forward 337 us and backward 323 us, 6.1 and
// 6.3 TB/s (each kernel alone, called back to back); 40,961 x 259 fp32, rows that cross lines, 18.4 and 23.6 us, 4.6 and 5.4
// TB/s.  By its launches where they are small: 2,432 x 128 fp32, forward, 2.8 us.  Rows wider than a wave's registers are read
// value by value, twice or three times: 20,000 x 4,096 bf16, forward and backward, 265 and 395 us, floors 64 and 95.
#include "egnn_device.h"
#include "egnn_internal.h"
#include <type_traits>

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
};

// A piece: 16 bytes of values from column f on.  Rows need no alignment but their values': the type says so, and the
// compiler still makes one 16-byte access of it.  The last piece of a row that is not a multiple of them wide ends with the
// row and overlaps the one before: its first `skip` columns enter no sum and are stored twice, with the same bits (value by
// value instead: 1,351,820 x 164 bf16, forward and backward, 1,154 us where it takes 700).  A row narrower than a piece goes
// value by value.  A piece stays as it was loaded until it is used, so that the next row's can be on their way.
// TAIL: the row is not a multiple of pieces wide
template <typename T, bool TAIL = true> struct Vec {
  static constexpr int N = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  typedef T piece __attribute__((ext_vector_type(N)));
  // PAST: of a tensor so large that it has left the cache when it is used again
  template <bool PAST = false> static __device__ __forceinline__ piece load(const T* p, int f, int C) {
    piece t;
    if (!TAIL || C >= N) {
      if constexpr (PAST) t = __builtin_nontemporal_load(reinterpret_cast<const type*>(p + f));
      else t = *reinterpret_cast<const type*>(p + f);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) t[i] = i < C ? p[i] : (T)0.f;
    }
    return t;
  }
  static __device__ __forceinline__ void floats(const piece& t, float* v) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f32((T)t[i]);
  }
  static __device__ __forceinline__ void load(const T* p, int f, int C, float* v) { floats(load(p, f, C), v); }
  template <bool PAST = false> static __device__ __forceinline__ void store(T* p, int f, int C, const float* v) {
    if (!TAIL || C >= N) {
      type t;
#pragma unroll
      for (int i = 0; i < N; ++i) t[i] = from_f32<T>(v[i]);
      if constexpr (PAST) __builtin_nontemporal_store(t, reinterpret_cast<type*>(p + f));
      else *reinterpret_cast<type*>(p + f) = t;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < C) p[i] = from_f32<T>(v[i]);
    }
  }
};
// A piece of the weight or the bias, of type P: T, or float beside bf16 rows (rounded to bf16 they would lose what training
// accumulates in them).
template <typename T, typename P, bool TAIL> __device__ __forceinline__ void load_params(const void* p, int f, int C, float* v) {
  constexpr int N = Vec<T, TAIL>::N;
  if constexpr (std::is_same<T, P>::value) Vec<T, TAIL>::load((const T*)p, f, C, v);
  else {
    const P* q = (const P*)p;
    if (!TAIL || C >= N) {
      Vec<P, false>::load(q, f, C, v);
      Vec<P, false>::load(q, f + N / 2, C, v + N / 2);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = i < C ? q[i] : 0.f;
    }
  }
}
template <typename P> __device__ __forceinline__ float param(const void* p, int f) { return to_f32(((const P*)p)[f]); }
// the lane's piece number k of a row: its first column, and how many of its columns another piece has (all of them: no
// such piece)
struct Piece {
  int f, skip;
  bool in;
};
template <int VEC, bool TAIL> __device__ __forceinline__ Piece piece_of(int k, int C) {
  const int f = k * VEC;
  Piece p{f < C ? f : 0, 0, f < C};
  if (TAIL && f + VEC > C && C >= VEC) {
    p.f = p.in ? C - VEC : 0;
    p.skip = p.in ? f - p.f : VEC;
  }
  return p;
}

template <int LPR> __device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int x = LPR / 2; x; x >>= 1) v += shfl_xor(v, x);
  return v;
}

constexpr int NT = 256;

template <typename T, typename P, int LPR, int VPL, bool TAIL>
__global__ __launch_bounds__(NT) void fwd_kernel(Args a) {
  typedef Vec<T, TAIL> V;
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
    if (live && c[p].in) V::load((const T*)a.x + n * a.ldx, c[p].f, a.C, v[p]);
  }
  if (a.r) {
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
    auto at = [&](int p, int i) { return ROUND ? to_f32(from_f32<T>(v[p][i])) : v[p][i]; };
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

// PAST: 1: the result is stored past the cache, 2: the operands are read past it too.  By the size of one tensor (the
// cache holds 256 MB): from 64 MB on storing past it is the faster (60,000 x 512 fp32, 123 MB: 71 -> 58 us; 40,961 x 259,
// 42 MB: 32.0 -> 33.3), from 256 MB on reading too (2,000,000 x 128 bf16: 347 -> 325 us; the 123 MB: 58 -> 67).
constexpr int64_t kPastStore = int64_t(64) << 20, kPastLoad = int64_t(256) << 20;

template <typename T, int LPR, int VPL, int PAST, bool TAIL>
__global__ __launch_bounds__(NT) void bwd_kernel(Args a) {
  typedef Vec<T, TAIL> V;
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
  const int64_t step = (int64_t)gridDim.x * RG;
  typename V::piece pg[VPL], px[VPL], pe[VPL];
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
template <typename T, typename P>
__global__ __launch_bounds__(NT) void fwd_wide_kernel(Args a) {
  __shared__ float buf[4];
  const int64_t n = blockIdx.x;
  const T *x = (const T*)a.x + n * a.ldx, *r = a.r ? (const T*)a.r + n * a.ldr : nullptr;
  auto val = [&](int f) { return to_f32(x[f]) + (r ? to_f32(r[f]) : 0.f); };
  auto stats = [&](bool round, float& mean, float& rstd) {
    auto at = [&](int f) { return round ? to_f32(from_f32<T>(val(f))) : val(f); };
    float s = 0.f;
    for (int f = threadIdx.x; f < a.C; f += NT) s += at(f);
    mean = block_sum(s, buf) / a.C;
    float q = 0.f;
    for (int f = threadIdx.x; f < a.C; f += NT) { const float d = at(f) - mean; q = __builtin_fmaf(d, d, q); }
    rstd = 1.0f / sqrtf(block_sum(q, buf) / a.C + a.eps);
  };
  float mean, rstd;
  stats(false, mean, rstd);
  if (a.mean) {
    float m = mean, rs = rstd;
    if (sizeof(T) == 2 && r && mean * mean * rstd * rstd > 1.f) stats(true, m, rs);
    if (threadIdx.x == 0) { a.mean[n] = m; a.rstd[n] = rs; }
  }
  for (int f = threadIdx.x; f < a.C; f += NT) {
    const float v = val(f), w = a.w ? param<P>(a.w, f) : 1.f, b = a.b ? param<P>(a.b, f) : 0.f;
    if (r) ((T*)a.s)[n * a.C + f] = from_f32<T>(v);
    ((T*)a.y)[n * a.C + f] = from_f32<T>(__builtin_fmaf((v - mean) * rstd, w, b));
  }
}
template <typename T, typename P>
__global__ __launch_bounds__(NT) void bwd_wide_kernel(Args a) {
  __shared__ float buf[4];
  const int64_t n = blockIdx.x;
  const T *x = (const T*)a.x + n * a.ldx, *g = (const T*)a.gy + n * a.ldg;
  const float mean = a.mean[n], rstd = a.rstd[n];
  float s1 = 0.f, s2 = 0.f;
  for (int f = threadIdx.x; f < a.C; f += NT) {
    const float t = to_f32(g[f]) * (a.w ? param<P>(a.w, f) : 1.f);
    s1 += t;
    s2 = __builtin_fmaf(t, (to_f32(x[f]) - mean) * rstd, s2);
  }
  const float m1 = block_sum(s1, buf) / a.C, m2 = block_sum(s2, buf) / a.C;
  for (int f = threadIdx.x; f < a.C; f += NT) {
    const float t = to_f32(g[f]) * (a.w ? param<P>(a.w, f) : 1.f);
    float o = rstd * (t - m1 - (to_f32(x[f]) - mean) * rstd * m2);
    if (a.gsum) o += to_f32(((const T*)a.gsum)[n * a.ldgs + f]);
    ((T*)a.gx)[n * a.C + f] = from_f32<T>(o);
  }
}
// gw and gb of wide rows: a thread a column, rows of one of gridDim.y parts
template <typename T>
__global__ __launch_bounds__(NT) void bwd_wide_weights_kernel(Args a) {
  const int f = blockIdx.x * NT + threadIdx.x;
  if (f >= a.C) return;
  float gw = 0.f, gb = 0.f;
  for (int64_t n = blockIdx.y; n < a.N; n += gridDim.y) {
    const float g = to_f32(((const T*)a.gy)[n * a.ldg + f]);
    gw = __builtin_fmaf(g, (to_f32(((const T*)a.x)[n * a.ldx + f]) - a.mean[n]) * a.rstd[n], gw);
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
    x.y = (void*)at(a.y, a.C); x.s = (void*)at(a.s, a.C); x.gx = (void*)at(a.gx, a.C);
    x.mean = a.mean ? a.mean + n : nullptr; x.rstd = a.rstd ? a.rstd + n : nullptr;
    x.N = a.N - n < most ? a.N - n : most;
    go(x, (uint32_t)cdiv(x.N, rows_per_block));
  }
}

template <typename T, int LPR, int VPL, bool TAIL>
static void launch_tail(const Args& a, bool bwd, hipStream_t st, int* nblk) {
  if (!bwd) {
    in_parts<T>(a, NT / LPR, [&](const Args& x, uint32_t blocks) {
      if (sizeof(T) == 2 && a.f32_params) fwd_kernel<T, float, LPR, VPL, TAIL><<<blocks, NT, 0, st>>>(x);
      else fwd_kernel<T, T, LPR, VPL, TAIL><<<blocks, NT, 0, st>>>(x);
    });
    return;
  }
  const int64_t n = cdiv(a.N, NT / LPR);
  *nblk = (int)(n < part_rows(a.N) ? n : part_rows(a.N));
  const int64_t bytes = a.N * a.C * (int64_t)sizeof(T);
  if (bytes >= kPastLoad) bwd_kernel<T, LPR, VPL, 2, TAIL><<<(uint32_t)*nblk, NT, 0, st>>>(a);
  else if (bytes >= kPastStore) bwd_kernel<T, LPR, VPL, 1, TAIL><<<(uint32_t)*nblk, NT, 0, st>>>(a);
  else bwd_kernel<T, LPR, VPL, 0, TAIL><<<(uint32_t)*nblk, NT, 0, st>>>(a);
}
template <typename T, int LPR, int VPL>
static void launch_shape(const Args& a, bool bwd, hipStream_t st, int* nblk) {
  if (a.C % Vec<T>::N) launch_tail<T, LPR, VPL, true>(a, bwd, st, nblk);
  else launch_tail<T, LPR, VPL, false>(a, bwd, st, nblk);
}
template <typename T>
static void launch_rows(const Args& a, const Shape& s, bool bwd, hipStream_t st, int* nblk) {
  switch (s.lpr * 8 + s.vpl - 1) {
    case 32: return launch_shape<T, 4, 1>(a, bwd, st, nblk);
    case 34: return launch_shape<T, 4, 3>(a, bwd, st, nblk);
    case 64: return launch_shape<T, 8, 1>(a, bwd, st, nblk);
    case 128: return launch_shape<T, 16, 1>(a, bwd, st, nblk);
    case 256: return launch_shape<T, 32, 1>(a, bwd, st, nblk);
    case 66: return launch_shape<T, 8, 3>(a, bwd, st, nblk);
    case 130: return launch_shape<T, 16, 3>(a, bwd, st, nblk);
    case 258: return launch_shape<T, 32, 3>(a, bwd, st, nblk);
    case 512: return launch_shape<T, 64, 1>(a, bwd, st, nblk);
    case 513: return launch_shape<T, 64, 2>(a, bwd, st, nblk);
    case 514: return launch_shape<T, 64, 3>(a, bwd, st, nblk);
    case 515: return launch_shape<T, 64, 4>(a, bwd, st, nblk);
    default: return launch_shape<T, 64, 6>(a, bwd, st, nblk);
  }
}

template <typename T, typename P>
static void launch_wide(const Args& a, bool bwd, hipStream_t st) {
  in_parts<T>(a, 1, [&](const Args& x, uint32_t blocks) {
    if (bwd) bwd_wide_kernel<T, P><<<blocks, NT, 0, st>>>(x);
    else fwd_wide_kernel<T, P><<<blocks, NT, 0, st>>>(x);
  });
}
template <typename T>
static int launch(const Args& a, bool bwd, hipStream_t st) {
  Shape s;
  int nblk = 0;
  if (a.N) {
    const bool narrow = shape_of((int)cdiv(a.C, Vec<T>::N), a.N, &s);
    if (narrow) launch_rows<T>(a, s, bwd, st, &nblk);
    else if (a.f32_params) launch_wide<T, float>(a, bwd, st);
    else launch_wide<T, T>(a, bwd, st);
    if (!narrow && bwd && a.part) {
      nblk = (int)(part_rows(a.N) < 128 ? part_rows(a.N) : 128);
      bwd_wide_weights_kernel<T><<<dim3((uint32_t)cdiv(a.C, NT), (uint32_t)nblk), NT, 0, st>>>(a);
    }
  }
  if (bwd && a.part) {
    const uint32_t blocks = (uint32_t)cdiv(2 * (int64_t)a.C, 16);
    if (a.f32_params) sum_kernel<float><<<blocks, 1024, 0, st>>>(a.part, nblk, a.C, (float*)a.gw, (float*)a.gb);
    else sum_kernel<T><<<blocks, 1024, 0, st>>>(a.part, nblk, a.C, (T*)a.gw, (T*)a.gb);
  }
  return hipGetLastError() == hipSuccess ? EGNN_OK : EGNN_ERR_HIP;
}

static bool dims_ok(const EgnnNormDims* d) {
  return d->N >= 0 && d->N <= INT32_MAX && d->C >= 1 && d->C <= 1 << 20 && (d->dtype == EGNN_F32 || d->dtype == EGNN_BF16) &&
         d->eps >= 0.f && d->eps - d->eps == 0.f && (d->f32_params == 0 || d->f32_params == 1);
}

}  // namespace norm
}  // namespace egnn

using namespace egnn::norm;

extern "C" {

size_t egnn_norm_bwd_workspace_bytes(const EgnnNormDims* d) {
  return d && dims_ok(d) ? (size_t)part_rows(d->N) * 2 * d->C * 4 : 0;
}

int32_t egnn_norm_fwd(const EgnnNormDims* d, const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight,
                      const void* bias, void* y, void* sum, float* mean, float* rstd, void* stream) {
  if (!d) return EGNN_ERR_NULL;
  if (!dims_ok(d)) return EGNN_ERR_DIMS;
  if (!mean != !rstd || (residual && !sum) || (d->N && (!x || !y))) return EGNN_ERR_NULL;
  if (ldx < 0 || (residual && ldr < 0)) return EGNN_ERR_STRIDE;
  const uintptr_t e = d->dtype == EGNN_F32 ? 4 : 2, ep = d->f32_params ? 4 : e;
  if ((uintptr_t)x % e || (uintptr_t)residual % e || (uintptr_t)weight % ep || (uintptr_t)bias % ep || (uintptr_t)y % e ||
      (uintptr_t)sum % e || (uintptr_t)mean % 4 || (uintptr_t)rstd % 4)
    return EGNN_ERR_ALIGN;
  Args a{};
  a.x = x; a.ldx = ldx; a.r = residual; a.ldr = ldr; a.w = weight; a.b = bias; a.y = y; a.s = residual ? sum : nullptr;
  a.mean = mean; a.rstd = rstd; a.N = d->N; a.C = d->C; a.eps = d->eps; a.f32_params = d->f32_params != 0;
  return d->dtype == EGNN_BF16 ? launch<egnn::bf16>(a, false, (hipStream_t)stream) : launch<float>(a, false, (hipStream_t)stream);
}

int32_t egnn_norm_bwd(const EgnnNormDims* d, const void* grad_y, int64_t ldg, const void* sum, int64_t lds, const void* weight,
                      const float* mean, const float* rstd, const void* grad_sum, int64_t ldgs, void* grad_x, void* grad_weight,
                      void* grad_bias, void* workspace, size_t workspace_bytes, void* stream) {
  if (!d) return EGNN_ERR_NULL;
  if (!dims_ok(d)) return EGNN_ERR_DIMS;
  if (d->N && (!grad_y || !sum || !mean || !rstd || !grad_x)) return EGNN_ERR_NULL;
  if (ldg < 0 || lds < 0 || (grad_sum && ldgs < 0)) return EGNN_ERR_STRIDE;
  const uintptr_t e = d->dtype == EGNN_F32 ? 4 : 2, ep = d->f32_params ? 4 : e;
  if ((uintptr_t)grad_y % e || (uintptr_t)sum % e || (uintptr_t)weight % ep || (uintptr_t)grad_sum % e || (uintptr_t)grad_x % e ||
      (uintptr_t)grad_weight % ep || (uintptr_t)grad_bias % ep || (uintptr_t)mean % 4 || (uintptr_t)rstd % 4 || (uintptr_t)workspace % 16)
    return EGNN_ERR_ALIGN;
  const bool weights = grad_weight || grad_bias;
  if (weights && (!workspace || workspace_bytes < egnn_norm_bwd_workspace_bytes(d))) return EGNN_ERR_WORKSPACE;
  Args a{};
  a.gy = grad_y; a.ldg = ldg; a.x = sum; a.ldx = lds; a.w = weight; a.mean = (float*)mean; a.rstd = (float*)rstd;
  a.gsum = grad_sum; a.ldgs = ldgs; a.gx = grad_x; a.gw = grad_weight; a.gb = grad_bias;
  a.part = weights ? (float*)workspace : nullptr; a.N = d->N; a.C = d->C; a.eps = d->eps; a.f32_params = d->f32_params != 0;
  return d->dtype == EGNN_BF16 ? launch<egnn::bf16>(a, true, (hipStream_t)stream) : launch<float>(a, true, (hipStream_t)stream);
}

}  // extern "C"
