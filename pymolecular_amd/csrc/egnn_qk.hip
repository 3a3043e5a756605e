// Norm of every head of queries and keys and their rotation by position, and the backward.
//   r = (mean x^2 + eps)^-1/2, xh = x r, y = xh w, out = turn(y): pairs (a, b) -> (a cos - b sin, b cos + a sin)
//   backward: gn = turn^-1(g), gw = sum over rows and heads of gn xh, t = gn w, gx = r (t - xh mean(t xh))
// One pass: a head lives in the registers of a few lanes, each of which holds both values of its pairs, so that nothing but
// the two row sums crosses lanes.  The angles depend on the row alone: a workgroup makes cos and sin of its rows once, in LDS,
// for all its heads, queries' and keys'; a thread has one pair's frequency and takes every so many rows.  An angle is position
// times frequency in turns, as a 64-bit fixed-point product whose overflow is the whole turns, so there is no large argument to
// reduce; the frequency is rounded to such a fixed-point number, and the position multiplies what that loses (frequencies()).
// cos and sin come from their Taylor series on an eighth of a turn to either side.
// Bound by HBM where there are many rows: 2,000,000 x 8 heads of 32 bf16, forward 394 us and backward 686 us, 5.2 and 4.5 TB/s (a
// large copy 5.3; queries and keys in workgroups of their own, which makes the angles twice, 600 and 783).  The backward holds
// weights and their gradients of both sides, 104 to 121 registers: four waves a SIMD; two heads at once instead of one take 138,
// three waves, and 445 instead of 356 us for 1,000,000 rows.  Loads and stores past the cache are slower here (476 us forward):
// a head's pieces are half lines.  Small calls are bound by the launch, the positions, the barrier behind the angles and the rows:
// 64 x 10 heads of 64, forward 5.8 us.
#include "egnn_internal.h"
#include "egnn_qk_plan.h"
#include "egnn_rows.h"

namespace egnn {
namespace qk {

struct Side {
  const void *x, *w, *g;
  void* y;                                   // the output, or the gradient of x
  void* gw;
  float* part;                               // [blocks][D] sums of gw
  int64_t xr, xh, gr, gh, yr, yh;            // strides of rows and heads
  int32_t H;                                 // heads
  uint32_t magic;                            // reciprocal(H)
};
struct Args {
  Side s[2];
  const void* pos;
  int64_t N;
  int32_t TB, blocks;                        // rows of a tile, workgroups
  int32_t D, rot, lanes, act;                // lanes of a head (a power of two), and those of them with values
  float eps, inv;                            // inv = 1 / D
  bool il, f32, i64;
  uint64_t freq[kPairs];                     // turns a position, in units of 2^-64
};

// cos and sin of t 2^-32 turns
__device__ __forceinline__ float2 cos_sin(uint32_t t) {
  const uint32_t q = (t + (1u << 29)) >> 30; // quarter turns, rounded
  const float x = (float)(int32_t)(t - (q << 30)) * (float)(6.283185307179586 / 4294967296.0);
  const float z = x * x;
  const float s = __builtin_fmaf(x * z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
  const float c = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const float u = q & 1 ? s : c, v = q & 1 ? c : s;
  return float2{(q + 1) & 2 ? -u : u, q & 2 ? -v : v};
}

template <typename T, int VEC> struct Piece {
  typedef T type __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  typedef T vals __attribute__((ext_vector_type(VEC)));
  static __device__ __forceinline__ vals load(const T* p) { return *reinterpret_cast<const type*>(p); }
  static __device__ __forceinline__ void store(T* p, const float* v) {
    type t;
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = from_f32<T>(v[i]);
    *reinterpret_cast<type*>(p) = t;
  }
};
// (pairs of bf16 stay words until they are used: vectors of bf16 that live across the loop take a register a value)
template <int VEC> struct Piece<bf16, VEC> {
  typedef bf16 type __attribute__((ext_vector_type(VEC), aligned(2)));
  typedef uint32_t words __attribute__((ext_vector_type(VEC / 2), aligned(2)));
  struct vals {
    uint32_t w[VEC / 2];
    __device__ __forceinline__ float operator[](int i) const { return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16); }
  };
  static __device__ __forceinline__ vals load(const bf16* p) {
    vals v;
    const words t = *reinterpret_cast<const words*>(p);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) v.w[i] = t[i];
    return v;
  }
  static __device__ __forceinline__ void store(bf16* p, const float* v) {
    type t;
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = (bf16)v[i];
    *reinterpret_cast<type*>(p) = t;
  }
};
template <> struct Piece<bf16, 1> {
  struct vals { bf16 x; __device__ __forceinline__ float operator[](int) const { return (float)x; } };
  static __device__ __forceinline__ vals load(const bf16* p) { return vals{*p}; }
  static __device__ __forceinline__ void store(bf16* p, const float* v) { *p = (bf16)v[0]; }
};
template <typename T> struct Piece<T, 1> {
  struct vals { T x; __device__ __forceinline__ T operator[](int) const { return x; } };
  static __device__ __forceinline__ vals load(const T* p) { return vals{*p}; }
  static __device__ __forceinline__ void store(T* p, const float* v) { *p = from_f32<T>(v[0]); }
};

// The two pieces a lane holds of a head, as values a[i] and b[i] of its pairs
template <int VEC, bool IL, typename V> __device__ __forceinline__ void to_pairs(const V& p0, const V& p1, float* a, float* b) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    if (IL) {
      a[i] = to_f32(2 * i < VEC ? p0[(2 * i) % VEC] : p1[(2 * i) % VEC]);
      b[i] = to_f32(2 * i + 1 < VEC ? p0[(2 * i + 1) % VEC] : p1[(2 * i + 1) % VEC]);
    } else {
      a[i] = to_f32(p0[i]);
      b[i] = to_f32(p1[i]);
    }
  }
}
template <int VEC, bool IL> __device__ __forceinline__ void from_pairs(const float* a, const float* b, float* p0, float* p1) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    p0[i] = !IL ? a[i] : i & 1 ? b[i / 2] : a[i / 2];
    p1[i] = !IL ? b[i] : (VEC + i) & 1 ? b[(VEC + i) / 2] : a[(VEC + i) / 2];
  }
}

// What a lane has of a side: the weights of its pairs and, in the backward, their gradient
template <int VEC> struct Weights {
  float a[VEC], b[VEC], ga[VEC], gb[VEC];
};
// the pairs' cos and sin: rows of the table are an even number of pairs apart where VEC is even
template <int VEC> __device__ __forceinline__ void angles(const float2* t, float* c, float* s) {
  if constexpr (VEC == 1) {
    c[0] = t->x;
    s[0] = t->y;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const float4 v = *reinterpret_cast<const float4*>(t + i);
      c[i] = v.x; s[i] = v.y; c[i + 1] = v.z; s[i + 1] = v.w;
    }
  }
}

template <typename T, int VEC, bool IL, bool BWD>
__global__ __launch_bounds__(NT) void qk_kernel(Args a) {
  typedef Piece<T, VEC> P;
  constexpr int U = BWD ? 1 : 2;             // heads that a group of lanes loads at once
  __shared__ __align__(16) float2 table[kTable];
  const int half = a.D / 2, apart = half + 2;   // (rows of the table 16 bytes further apart: fewer of them in one bank)
  const int lanes = a.lanes, groups = NT / lanes, group = threadIdx.x / lanes, lane = threadIdx.x & (lanes - 1);
  const bool lives = lane < a.act;
  const int j0 = lives ? lane * VEC : 0;     // the lane's first pair
  int f0, f1;                                // the columns of its two pieces
  if (IL) { f0 = 2 * j0; f1 = f0 + VEC; }
  else if (j0 < a.rot / 2) { f0 = j0; f1 = j0 + a.rot / 2; }
  else { f0 = a.rot + j0 - a.rot / 2; f1 = f0 + (a.D - a.rot) / 2; }
  // a thread makes cos and sin of one pair (past the turned ones: of angle 0), for every per-th row
  const int per = NT / half, tr = (int)threadIdx.x < per * half ? threadIdx.x / half : 1 << 30, tj = threadIdx.x % half;
  const uint64_t freq = tj < a.rot / 2 ? a.freq[tj] : 0;
  Weights<VEC> ws[2];
  const int64_t tiles = (a.N + a.TB - 1) / a.TB;
  struct Raw { typename P::vals x0, x1, g0, g1; };
  auto fetch = [&](const Side& s, int64_t n0, int units, int base, Raw* raw) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(base + u * groups + group, units - 1);
      const int row = s.H > 1 ? (int)__umulhi(k, s.magic) : k;
      const T* x = (const T*)s.x + (n0 + row) * s.xr + (k - row * s.H) * s.xh;
      raw[u].x0 = P::load(x + f0);
      raw[u].x1 = P::load(x + f1);
      if (BWD) {
        const T* g = (const T*)s.g + (n0 + row) * s.gr + (k - row * s.H) * s.gh;
        raw[u].g0 = P::load(g + f0);
        raw[u].g1 = P::load(g + f1);
      }
    }
  };
  auto compute = [&](const Side& s, Weights<VEC>& w, int64_t n0, int units, int base, const Raw* raw) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = base + u * groups + group, kk = min(k, units - 1);
      const bool in = k < units && lives;
      const int row = s.H > 1 ? (int)__umulhi(kk, s.magic) : kk, head = kk - row * s.H;
      float va[VEC], vb[VEC], c[VEC], sn[VEC];
      to_pairs<VEC, IL>(raw[u].x0, raw[u].x1, va, vb);
      angles<VEC>(table + row * apart + j0, c, sn);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        sum = __builtin_fmaf(va[i], va[i], sum);
        sum = __builtin_fmaf(vb[i], vb[i], sum);
      }
      sum = lives ? sum : 0.f;
      for (int m = lanes / 2; m; m >>= 1) sum += shfl_xor(sum, m);
      float r = __builtin_amdgcn_rsqf(__builtin_fmaf(sum, a.inv, a.eps));   // (to one unit of 2^-23)
      float oa[VEC], ob[VEC];
      if constexpr (!BWD) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float ya = va[i] * r * w.a[i], yb = vb[i] * r * w.b[i];
          oa[i] = ya * c[i] - yb * sn[i];
          ob[i] = yb * c[i] + ya * sn[i];
        }
      } else {
        float ta[VEC], tb[VEC], dot = 0.f;
        to_pairs<VEC, IL>(raw[u].g0, raw[u].g1, ta, tb);
        // A head whose gradient is 0 throughout takes no part, NaN and infinities of it neither: what an attention leaves out may
        // hold anything.  (0 times a finite head is 0 anyway, but for one of zeros without eps, whose r is infinite; that of NaN is
        // NaN, that of infinities 0.)
        if (__ballot(!(r > 0.f && r < __builtin_inff()))) {
          float some = 0.f;                   // (how many of the gradient's pairs are not 0)
#pragma unroll
          for (int i = 0; i < VEC; ++i) some += (ta[i] != 0.f || tb[i] != 0.f) ? 1.f : 0.f;
          some = lives ? some : 0.f;
          for (int m = lanes / 2; m; m >>= 1) some += shfl_xor(some, m);
          if (some == 0.f) {
            r = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) va[i] = vb[i] = 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float na = ta[i] * c[i] + tb[i] * sn[i], nb = tb[i] * c[i] - ta[i] * sn[i];
          va[i] *= r;
          vb[i] *= r;
          if (in) {
            w.ga[i] = __builtin_fmaf(na, va[i], w.ga[i]);
            w.gb[i] = __builtin_fmaf(nb, vb[i], w.gb[i]);
          }
          ta[i] = na * w.a[i];
          tb[i] = nb * w.b[i];
          dot = __builtin_fmaf(ta[i], va[i], dot);
          dot = __builtin_fmaf(tb[i], vb[i], dot);
        }
        dot = lives ? dot : 0.f;
        for (int m = lanes / 2; m; m >>= 1) dot += shfl_xor(dot, m);
        dot *= a.inv;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          oa[i] = r * (ta[i] - va[i] * dot);
          ob[i] = r * (tb[i] - vb[i] * dot);
        }
      }
      if (in) {
        float p0[VEC], p1[VEC];
        from_pairs<VEC, IL>(oa, ob, p0, p1);
        T* y = (T*)s.y + (n0 + row) * s.yr + head * s.yh;
        P::store(y + f0, p0);
        P::store(y + f1, p1);
      }
    }
  };
  bool first = true;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += a.blocks) {
    const int64_t n0 = tile * a.TB;
    const int rows = (int)(a.N - n0 < a.TB ? a.N - n0 : a.TB);
    Raw raw[U];
    fetch(a.s[0], n0, rows * a.s[0].H, 0, raw);
    if (first) {                             // (behind the first rows' loads, which take longest)
      first = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const void* w = a.s[i].w;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          ws[i].a[v] = ws[i].b[v] = 1.f;
          ws[i].ga[v] = ws[i].gb[v] = 0.f;
        }
        if (!w) continue;
        if (sizeof(T) == 2 && a.f32) {
          typedef Piece<float, VEC> F;
          to_pairs<VEC, IL>(F::load((const float*)w + f0), F::load((const float*)w + f1), ws[i].a, ws[i].b);
        } else {
          to_pairs<VEC, IL>(P::load((const T*)w + f0), P::load((const T*)w + f1), ws[i].a, ws[i].b);
        }
      }
    } else {
      __syncthreads();                       // the table is read no more
    }
    for (int row0 = tr; row0 < rows; row0 += 4 * per) {
      int64_t p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t n = n0 + min(row0 + u * per, rows - 1);
        p[u] = !a.rot ? 0 : a.i64 ? ((const int64_t*)a.pos)[n] : ((const int32_t*)a.pos)[n];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (row0 + u * per < rows) table[(row0 + u * per) * apart + tj] = cos_sin((uint32_t)(((uint64_t)p[u] * freq) >> 32));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int units = rows * a.s[i].H;
      for (int base = 0; base < units; base += U * groups) {
        if (i || base) fetch(a.s[i], n0, units, base, raw);
        compute(a.s[i], ws[i], n0, units, base, raw);
      }
    }
  }
  if (!BWD) return;
  // the groups' sums of a column, in order, by all threads: parts of the groups first, [group][D] in the table's place
  float* red = (float*)table;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (!a.s[i].part) continue;
    float p0[VEC], p1[VEC];
    from_pairs<VEC, IL>(ws[i].ga, ws[i].gb, p0, p1);
    __syncthreads();
    if (lives)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        red[group * a.D + f0 + v] = p0[v];
        red[group * a.D + f1 + v] = p1[v];
      }
    __syncthreads();
    const int parts = NT / a.D, part = threadIdx.x / a.D, f = threadIdx.x - part * a.D;
    float t = 0.f;
    if (part < parts) {
#pragma unroll 8
      for (int g = part; g < groups; g += parts) t += red[g * a.D + f];
    }
    __syncthreads();
    red[threadIdx.x] = t;
    __syncthreads();
    if (part == 0) {
      for (int k = 1; k < parts; ++k) t += red[k * a.D + f];
      a.s[i].part[(int64_t)blockIdx.x * a.D + f] = t;
    }
  }
}

// gw = the sums over the workgroups: 16 columns of one side a workgroup, 64 groups joined in order
template <typename P> __global__ __launch_bounds__(1024) void sum_kernel(Args a) {
  __shared__ float red[64][17];
  const Side s = a.s[blockIdx.y];
  const int c = threadIdx.x & 15, k = threadIdx.x >> 4, f = blockIdx.x * 16 + c;
  float t = 0.f;
  if (f < a.D && s.gw) {
#pragma unroll 8
    for (int b = k; b < a.blocks; b += 64) t += s.part[(int64_t)b * a.D + f];
  }
  red[k][c] = t;
  __syncthreads();
  for (int h = 32; h; h >>= 1) {
    if (k < h) red[k][c] += red[k + h][c];
    __syncthreads();
  }
  if (!k && f < a.D && s.gw) ((P*)s.gw)[f] = from_f32<P>(red[0][c]);
}

template <typename T, int VEC>
static void launch(const Args& a, bool bwd, hipStream_t st) {
  const uint32_t grid = (uint32_t)a.blocks;
  if (!grid) return;
  if constexpr (VEC <= 4) {
    if (bwd) {
      if (a.il) qk_kernel<T, VEC, true, true><<<grid, NT, 0, st>>>(a);
      else qk_kernel<T, VEC, false, true><<<grid, NT, 0, st>>>(a);
      return;
    }
  }
  if (a.il) qk_kernel<T, VEC, true, false><<<grid, NT, 0, st>>>(a);
  else qk_kernel<T, VEC, false, false><<<grid, NT, 0, st>>>(a);
}
static int run(const EgnnQkDims* d, Args& a, bool bwd, hipStream_t st) {
  const int vec = piece_of(d, bwd), half = d->D / 2;
  a.N = d->N; a.D = d->D; a.rot = d->rotary; a.lanes = lanes_of(d, bwd); a.act = half / vec; a.eps = d->eps;
  a.il = d->interleaved; a.f32 = d->f32_params; a.i64 = d->index64;
  frequencies(d, a.freq);
  for (int i = 0; i < 2; ++i) {
    Side& s = a.s[i];
    s.H = i ? d->Hk : d->Hq;
    s.magic = reciprocal(s.H);
  }
  a.inv = 1.f / d->D;
  a.TB = tile_rows(d, bwd);
  a.blocks = blocks_of(d, bwd);
  if (d->dtype == EGNN_F32) {
    if (vec == 4) launch<float, 4>(a, bwd, st);
    else if (vec == 2) launch<float, 2>(a, bwd, st);
    else launch<float, 1>(a, bwd, st);
  } else {
    if (vec == 8) launch<bf16, 8>(a, bwd, st);
    else if (vec == 4) launch<bf16, 4>(a, bwd, st);
    else if (vec == 2) launch<bf16, 2>(a, bwd, st);
    else launch<bf16, 1>(a, bwd, st);
  }
  if (bwd && (a.s[0].gw || a.s[1].gw)) {  // (without rows: sums of nothing)
    const dim3 grid((uint32_t)cdiv(d->D, 16), 2);
    if (d->dtype == EGNN_F32 || d->f32_params) sum_kernel<float><<<grid, 1024, 0, st>>>(a);
    else sum_kernel<bf16><<<grid, 1024, 0, st>>>(a);
  }
  return hipGetLastError() == hipSuccess ? EGNN_OK : EGNN_ERR_HIP;
}

static bool dims_ok(const EgnnQkDims* d) {
  return d->N >= 0 && d->N <= INT32_MAX && d->Hq >= 1 && d->Hq <= kHeads && d->Hk >= 1 && d->Hk <= kHeads && d->D >= 2 &&
         d->D <= 2 * kPairs && d->D % 2 == 0 && d->rotary >= 0 && d->rotary <= d->D && d->rotary % 2 == 0 &&
         (d->interleaved == 0 || d->interleaved == 1) && (d->dtype == EGNN_F32 || d->dtype == EGNN_BF16) &&
         (d->f32_params == 0 || d->f32_params == 1) && (d->index64 == 0 || d->index64 == 1) && d->eps >= 0.f &&
         d->eps - d->eps == 0.f && d->base >= 1.0 && d->base - d->base == 0.0;
}

}  // namespace qk
}  // namespace egnn

using namespace egnn::qk;

extern "C" {

int32_t egnn_qk_fwd(const EgnnQkDims* d, const EgnnQkStrides* st, const void* q, const void* k, const void* q_weight,
                    const void* k_weight, const void* positions, void* q_out, void* k_out, void* stream) {
  if (!d || !st) return EGNN_ERR_NULL;
  if (!dims_ok(d)) return EGNN_ERR_DIMS;
  if (d->N && (!q || !k || !q_out || !k_out || (d->rotary && !positions))) return EGNN_ERR_NULL;
  if (st->q_row < 0 || st->q_head < 0 || st->k_row < 0 || st->k_head < 0 || st->q_out_head < d->D || st->k_out_head < d->D ||
      st->q_out_row < d->Hq * (int64_t)d->D || st->k_out_row < d->Hk * (int64_t)d->D)
    return EGNN_ERR_STRIDE;
  const uintptr_t e = d->dtype == EGNN_F32 ? 4 : 2, ep = d->f32_params ? 4 : e, ei = d->index64 ? 8 : 4;
  if ((uintptr_t)q % e || (uintptr_t)k % e || (uintptr_t)q_out % e || (uintptr_t)k_out % e || (uintptr_t)q_weight % ep ||
      (uintptr_t)k_weight % ep || (uintptr_t)positions % ei)
    return EGNN_ERR_ALIGN;
  Args a{};
  a.pos = positions;
  Side &x = a.s[0], &y = a.s[1];
  x.x = q; x.w = q_weight; x.y = q_out; x.xr = st->q_row; x.xh = st->q_head; x.yr = st->q_out_row; x.yh = st->q_out_head;
  y.x = k; y.w = k_weight; y.y = k_out; y.xr = st->k_row; y.xh = st->k_head; y.yr = st->k_out_row; y.yh = st->k_out_head;
  return run(d, a, false, (hipStream_t)stream);
}

size_t egnn_qk_bwd_workspace_bytes(const EgnnQkDims* d) {
  if (!d || !dims_ok(d)) return 0;
  return (size_t)blocks_of(d, true) * 2 * d->D * 4;
}

int32_t egnn_qk_bwd(const EgnnQkDims* d, const EgnnQkStrides* st, const void* grad_q_out, const void* grad_k_out,
                    const void* q, const void* k, const void* q_weight, const void* k_weight, const void* positions,
                    void* grad_q, void* grad_k, void* grad_q_weight, void* grad_k_weight, void* workspace,
                    size_t workspace_bytes, void* stream) {
  if (!d || !st) return EGNN_ERR_NULL;
  if (!dims_ok(d)) return EGNN_ERR_DIMS;
  if (d->N && (!grad_q_out || !grad_k_out || !q || !k || !grad_q || !grad_k || (d->rotary && !positions))) return EGNN_ERR_NULL;
  if (st->q_row < 0 || st->q_head < 0 || st->k_row < 0 || st->k_head < 0 || st->grad_q_out_row < 0 || st->grad_q_out_head < 0 ||
      st->grad_k_out_row < 0 || st->grad_k_out_head < 0 || st->grad_q_head < d->D || st->grad_k_head < d->D ||
      st->grad_q_row < d->Hq * (int64_t)d->D || st->grad_k_row < d->Hk * (int64_t)d->D)
    return EGNN_ERR_STRIDE;
  const uintptr_t e = d->dtype == EGNN_F32 ? 4 : 2, ep = d->f32_params ? 4 : e, ei = d->index64 ? 8 : 4;
  if ((uintptr_t)grad_q_out % e || (uintptr_t)grad_k_out % e || (uintptr_t)q % e || (uintptr_t)k % e || (uintptr_t)grad_q % e ||
      (uintptr_t)grad_k % e || (uintptr_t)q_weight % ep || (uintptr_t)k_weight % ep || (uintptr_t)grad_q_weight % ep ||
      (uintptr_t)grad_k_weight % ep || (uintptr_t)positions % ei || (uintptr_t)workspace % 16)
    return EGNN_ERR_ALIGN;
  const size_t need = egnn_qk_bwd_workspace_bytes(d);
  if ((grad_q_weight || grad_k_weight) && need && (!workspace || workspace_bytes < need)) return EGNN_ERR_WORKSPACE;
  Args a{};
  a.pos = positions;
  Side &x = a.s[0], &y = a.s[1];
  x.x = q; x.w = q_weight; x.g = grad_q_out; x.y = grad_q; x.gw = grad_q_weight;
  x.xr = st->q_row; x.xh = st->q_head; x.gr = st->grad_q_out_row; x.gh = st->grad_q_out_head; x.yr = st->grad_q_row; x.yh = st->grad_q_head;
  y.x = k; y.w = k_weight; y.g = grad_k_out; y.y = grad_k; y.gw = grad_k_weight;
  y.xr = st->k_row; y.xh = st->k_head; y.gr = st->grad_k_out_row; y.gh = st->grad_k_out_head; y.yr = st->grad_k_row; y.yh = st->grad_k_head;
  x.part = grad_q_weight ? (float*)workspace : nullptr;
  y.part = grad_k_weight ? (float*)workspace + (int64_t)blocks_of(d, true) * d->D : nullptr;
  return run(d, a, true, (hipStream_t)stream);
}

}  // extern "C"
