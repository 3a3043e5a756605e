// Segment attention, forward: o_i = sum_j softmax_j(scale q_i k_j) v_j over the keys of i's segment, in one pass over
// the keys with the running maximum and sum.
//
// The maximum is lazy: a column keeps its reference m while the probabilities against it stay below 2^10, which costs no
// precision in floating point, so that a step costs no maximum, no shuffle and no rescaling of the output.  A step whose
// sum passes 2^10 (the first one always: m starts at the lowest float) is made again with its maximum as the reference.
// The sum takes the unrounded probabilities (one more product, against ones, would sum the rounded ones at less
// cost, and put up to 2^-9 into lse).
//
// Measured (the kernel alone, called back to back): 12,289 rows, 4 heads of 64, bf16, 196 us, 0.79 PFLOP/s, bound by vector
// and MFMA issue, which do not overlap (0.50 and 0.32 of the cycles); one query of 8 heads on 2 over 2,000,000 keys 183 us,
// 5.6 TB/s, bound by HBM; 128 molecules in fp32 4.9 us, bound by three round trips to memory.
#include "egnn_attn.h"

namespace egnn {
namespace attn {

constexpr float kLazy = 1024.0f, kLowest = -3.40282347e+38f;

// Partial results of a split call: [split][row of q, head] sums of DP values, then (m, l)
__device__ __forceinline__ float* part_o(const Args& a, int dp, int s, int64_t r) { return a.part + ((int64_t)s * a.Nq * a.Hq + r) * dp; }
__device__ __forceinline__ float* part_ml(const Args& a, int dp, int s, int64_t r) {
  return a.part + (int64_t)a.nsplit * a.Nq * a.Hq * dp + ((int64_t)s * a.Nq * a.Hq + r) * 2;
}

// R: blocks of 16 columns a wave.  W waves, on one tile (SH) or each on its own.  KT: steps of 32 keys between barriers,
// KC of them at a time in registers.
template <typename T, int DP, int R, int W, bool SH, int KT, int KC>
__device__ __forceinline__ void fwd_tile(const Args& a, const Item& it, int e, int vq0, const Seg& qs, bf16* sK, bf16* sV, int w) {
  typedef Tile<T, DP, KT> TL;
  typedef typename Num<T>::Frag Frag;
  constexpr int NT = SH ? 64 * W : 64, KS = TK * KT;
  const int l = lane_id(), c = l & 15, g = l >> 4;
  const Seg ks = other_rows(a.kv_ptr, e, a.B, a.Nk, a.same, qs);
  const int nv = (qs.hi - qs.lo) * a.G, v0 = vq0 + (SH ? 16 * R * w : 0);
  const bool act = v0 < nv;                  // a wave without rows still loads tiles for the others
  int j = ks.lo + it.sp * KS;
  const int j1 = ks.hi, stride = KS * a.nsplit;

  Stage<T, DP, KT, NT, TK * KC> stK, stV;
  uint32_t offK[stK.PER], offV[stV.PER];
  const int64_t krb = a.k_r * (int64_t)sizeof(T), vrb = a.v_r * (int64_t)sizeof(T);
  stK.offsets(offK, krb, a.D);
  stV.offsets(offV, vrb, a.D);
  const T *kb = (const T*)a.k + it.kvh * a.k_h, *vb = (const T*)a.v + it.kvh * a.v_h;
  uint8_t mb[Bits<KT>::N];
  const bool masked = a.mask || a.v_r == 0;
  auto rows_at = [&](int j) { return j1 - j < KS ? j1 - j : KS; };
  auto fetch = [&](int j) {
    const int n = rows_at(j);
    stK.load(rows_buffer(kb + j * a.k_r, n, krb, a.D * (int)sizeof(T)), offK, n);
    stV.load(rows_buffer(vb + j * a.v_r, n, vrb, a.D * (int)sizeof(T)), offV, n);
    if (a.mask) {
#pragma unroll
      for (int k = 0; k < Bits<KT>::N; ++k) mb[k] = 64 * k + l < n ? a.mask[j + 64 * k + l] : 0;
    }
  };
  if (j < j1) fetch(j);

  // the lane's columns of Q^T
  typename TL::Feat Q[R][TL::NK];
  int row[R], head[R];
  bool live[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int v = v0 + 16 * r + c;
    live[r] = v < nv;
    const uint32_t i = live[r] ? a.by_g(v) : 0;
    row[r] = qs.lo + (int)i;
    head[r] = it.kvh * a.G + (live[r] ? v - (int)i * a.G : 0);
    const T* qp = live[r] ? (const T*)a.q + row[r] * a.q_r + head[r] * a.q_h : nullptr;
#pragma unroll
    for (int kk = 0; kk < TL::NK; ++kk) {
      Q[r][kk] = TL::column(qp, kk, g, a.D, a.flip);
      landed(Q[r][kk]);
    }
  }
  Sum<T> O[R][TL::NB];
  float m[R], sum[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = kLowest;
    sum[r] = 0.f;
  }

  for (; j < j1; j += stride) {
    const int n = rows_at(j);
    Bits<KT> bits = step_bits<KT>(n);
    // what a masked value holds must not meet a probability of 0, nor what the one row of a broadcast v does past the last
    // key (other rows there read as zeros)
    if (masked) {
      if (a.mask) {
#pragma unroll
        for (int k = 0; k < Bits<KT>::N; ++k) bits.w[k] &= __ballot(mb[k] != 0);
      }
      stV.keep(bits);
    }
    tile_sync<SH>();                         // the step before has read the tile
    stK.store(sK, n);
    stV.store(sV, n);
    tile_sync<SH>();
    if (j + stride < j1) fetch(j + stride);
    if (!act) continue;
    if constexpr (KT > 1) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int b = 0; b < TL::NB; ++b) O[r][b].begin();
    }
#pragma unroll
    for (int t0 = 0; t0 < KT; t0 += KC) {
      if (KT > KC && TK * t0 >= n) break;
      f32x4 S[R][2 * KC];
      float ps[R];
      for (bool again = false;; again = true) {
#pragma unroll
        for (int h = 0; h < 2 * KC; ++h) {
          f32x4 hi[R], lo[R];
#pragma unroll
          for (int r = 0; r < R; ++r) { hi[r] = zero4(); lo[r] = zero4(); }
#pragma unroll
          for (int kk = 0; kk < TL::NK; ++kk) {
            const auto A = TL::rows(sK, 2 * t0 + h, kk, c, g);
#pragma unroll
            for (int r = 0; r < R; ++r) product1(hi[r], lo[r], A, Q[r][kk]);
          }
#pragma unroll
          for (int r = 0; r < R; ++r) S[r][h] = result<T>(hi[r], lo[r]);
        }
#pragma unroll
        for (int t = 0; t < KC; ++t) {
          const uint32_t b = bits.step(t0 + t);
          if (b != 0xffffffffu) {
            const uint32_t x = b >> (4 * g);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const bool ok = (x >> (16 * h + i)) & 1;
#pragma unroll
                for (int r = 0; r < R; ++r) S[r][2 * t + h][i] = ok ? S[r][2 * t + h][i] : -INFINITY;
              }
          }
        }
        if (again) {                         // the step's maximum as the new reference
#pragma unroll
          for (int r = 0; r < R; ++r) {
            float top = S[r][0][0];
#pragma unroll
            for (int h = 0; h < 2 * KC; ++h)
#pragma unroll
              for (int i = 0; i < 4; ++i) top = fmaxf(top, S[r][h][i]);
            const float mn = fmaxf(m[r], col_max(top) * a.c2), alpha = __builtin_amdgcn_exp2f(m[r] - mn);
            m[r] = mn;
            sum[r] *= alpha;
#pragma unroll
            for (int b = 0; b < TL::NB; ++b) O[r][b].scale(alpha, KT > KC && t0 > 0);
          }
        }
        bool over = false;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          ps[r] = 0.f;
#pragma unroll
          for (int h = 0; h < 2 * KC; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              S[r][h][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[r][h][i], a.c2, -m[r]));
              ps[r] += S[r][h][i];
            }
          over |= ps[r] > kLazy;
        }
        if (again || !__ballot(over)) break;
      }
      Frag P[R][KC];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        sum[r] += ps[r];
#pragma unroll
        for (int t = 0; t < KC; ++t) P[r][t] = chain_frag<T>(S[r][2 * t], S[r][2 * t + 1]);
      }
#pragma unroll
      for (int t = 0; t < KC; ++t)
#pragma unroll
        for (int b = 0; b < TL::NB; ++b) {
          const Frag A = TL::cols(sV, t0 + t, b, c, g);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if constexpr (KT == 1) O[r][b].one(A, P[r][t]);
            else O[r][b].add(A, P[r][t]);
          }
        }
    }
    if constexpr (KT > 1) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int b = 0; b < TL::NB; ++b) O[r][b].end();
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float s = col_sum(sum[r]);
    if (!live[r]) continue;
    if (a.nsplit > 1) {
      const int64_t x = (int64_t)row[r] * a.Hq + head[r];
      float* p = part_o(a, DP, it.sp, x);
#pragma unroll
      for (int b = 0; b < TL::NB; ++b) store4(p + 16 * b + 4 * g, O[r][b].v);
      p = part_ml(a, DP, it.sp, x);
      if (g == 0) { p[0] = m[r]; p[1] = s; }
      continue;
    }
    // no key left: the sum is 0 (a NaN is not), the output 0 and lse -inf
    const float inv = s == 0.f ? 0.f : 1.0f / s;
    T* op = (T*)a.out + row[r] * a.o_r + head[r] * a.o_h;
#pragma unroll
    for (int b = 0; b < TL::NB; ++b)
      if (16 * b + 4 * g < a.D) store4(op + 16 * b + 4 * g, O[r][b].v * inv);
    if (a.lse && g == 0) a.lse[(int64_t)head[r] * a.Nq + row[r]] = (m[r] + __builtin_amdgcn_logf(s)) * kLn2;
  }
}

template <typename T, int DP, int R, int W, bool SH, int KT, int KC>
__global__ __launch_bounds__(64 * W, (SH ? group_occupancy<T, DP, R>() : 1)) void fwd_kernel(Args a, uint32_t n_items) {
  typedef Tile<T, DP, KT> TL;
  constexpr int BQ = 16 * R * (SH ? W : 1);
  __shared__ __attribute__((aligned(16))) bf16 lds[SH ? 1 : W][2][TL::elems];
  Item it;
  if (!item_of<W, SH>(a, n_items, it)) return;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  int vq0;
  Seg qs;
  const int e = find_tile<BQ>(a.q_ptr, a.B, a.Nq, a.G, a.guess, it.slot, vq0, qs);
  if (vq0 < 0) return;
  fwd_tile<T, DP, R, W, SH, KT, KC>(a, it, e, vq0, qs, lds[SH ? 0 : w][0], lds[SH ? 0 : w][1], w);
}

// A segment with at most 32 virtual rows and 32 keys (a molecule): each row of q, k and v read once, in rows as they lie,
// and one softmax over all keys.  One wave, or two (P) with 16 virtual rows each.
template <typename T, int DP, int P>
__device__ __forceinline__ void small_segment(const Args& a, int kvh, const Seg& qs, const Seg& ks, bf16* lds, int w) {
  typedef Tile<T, DP> TL;
  typedef typename Num<T>::Frag Frag;
  const int l = lane_id(), c = l & 15, g = l >> 4;
  const int nv = (qs.hi - qs.lo) * a.G, nk = ks.hi - ks.lo;
  bf16 *sQ = lds, *sK = sQ + TL::elems, *sV = sK + TL::elems;
  const int64_t e = sizeof(T);
  const int last = a.D * (int)e;
  uint32_t kbits;
  {
    // of two waves the first brings q, the second k and v
    const bool bq = P == 1 || w == 0, bk = (P == 1 || w == 1) && nk;
    Stage<T, DP, 1, 64> stQ, stK, stV;
    if (bq) {
      uint32_t offQ[stQ.PER];
      if (a.G == 1) stQ.offsets(offQ, a.q_r * e, a.D);
      else {
#pragma unroll
        for (int p = 0; p < stQ.PER; ++p) {
          const uint32_t u = stQ.row(p), i = a.by_g(u), h = u - i * a.G, f = stQ.feature(p);
          offQ[p] = stQ.in(p) && (int)u < nv && (int)f < a.D ? (uint32_t)((i * a.q_r + h * a.q_h + f) * e) : kOob;
        }
      }
      stQ.load(rows_buffer((const T*)a.q + qs.lo * a.q_r + (int64_t)kvh * a.G * a.q_h, qs.hi - qs.lo, a.q_r * e, last + (int)((a.G - 1) * a.q_h * e)), offQ, nv);
    }
    if (bk) {
      uint32_t offK[stK.PER], offV[stV.PER];
      stK.offsets(offK, a.k_r * e, a.D);
      stV.offsets(offV, a.v_r * e, a.D);
      stK.load(rows_buffer((const T*)a.k + ks.lo * a.k_r + kvh * a.k_h, nk, a.k_r * e, last), offK, nk);
      stV.load(rows_buffer((const T*)a.v + ks.lo * a.v_r + kvh * a.v_h, nk, a.v_r * e, last), offV, nk);
    }
    bool key = l < nk;
    if (key && a.mask) key = a.mask[ks.lo + l] != 0;
    kbits = (uint32_t)__ballot(key);
    if (bq) stQ.store(sQ, TK);
    if (bk) {
      if (a.mask || a.v_r == 0) {            // as in fwd_tile
        Bits<1> bits;
        bits.w[0] = kbits;
        stV.keep(bits);
      }
      stK.store(sK, nk);
      stV.store(sV, nk);
    }
  }
  tile_sync<(P > 1)>();
  const float c2 = a.flip ? -a.c2 : a.c2;
#pragma unroll
  for (int q = 0; q < 2; q += P) {
    if (P == 2) q = w;
    if (P == 1 ? q && nv <= 16 : 16 * q >= nv) break;
    typename TL::Feat Qc[TL::NK];
#pragma unroll
    for (int kk = 0; kk < TL::NK; ++kk) Qc[kk] = TL::rows(sQ, q, kk, c, g);
    f32x4 S[2] = {zero4(), zero4()};
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k ? nk <= 16 : nk == 0) break;
      S[k] = TL::product(sK, k, Qc, c, g, zero4());
      const uint32_t b = kbits >> (16 * k + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        S[k][i] = (b >> i) & 1 ? S[k][i] * c2 : -INFINITY;
        top = fmaxf(top, S[k][i]);
      }
    }
    top = col_max(top);
    const float m = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (k ? nk > 16 : nk > 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { S[k][i] = __builtin_amdgcn_exp2f(S[k][i] - m); sum += S[k][i]; }
      }
    sum = col_sum(sum);
    const Frag F = chain_frag<T>(S[0], S[1]);
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    const int v = 16 * q + c;
    const uint32_t i = a.by_g(v);
    const int row = qs.lo + (int)i, head = kvh * a.G + (v - (int)i * a.G);
    T* op = (T*)a.out + row * a.o_r + head * a.o_h;
    f32x4 o[TL::NB];
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) {
      Sum<T> O;
      O.begin();
      if (nk) O.add(TL::cols(sV, 0, b, c, g), F);
      O.end();
      o[b] = O.v * inv;
    }
    if (v >= nv) continue;
    store_row<TL::NB>(op, o, g, a.D);
    if (a.lse && g == 0) a.lse[(int64_t)head * a.Nq + row] = (m + __builtin_amdgcn_logf(sum)) * kLn2;
  }
}

// Tiles of 32 virtual rows, P waves each and W a workgroup: the whole segment where it is small
template <typename T, int DP, int P, int W>
__global__ __launch_bounds__(64 * W) void short_kernel(Args a, uint32_t n_items) {
  typedef Tile<T, DP> TL;
  static_assert(P == 1 || W == P, "");
  __shared__ __attribute__((aligned(16))) bf16 lds[W / P][P == 1 ? 3 : 4][TL::elems];
  Item it;
  if (!item_of<W, (P > 1)>(a, n_items, it)) return;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  int vq0;
  Seg qs;
  const int e = find_tile<TK>(a.q_ptr, a.B, a.Nq, a.G, a.guess, it.slot, vq0, qs);
  if (vq0 < 0) return;
  const Seg ks = other_rows(a.kv_ptr, e, a.B, a.Nk, a.same, qs);
  const int nv = (qs.hi - qs.lo) * a.G;
  if (nv <= TK && ks.hi - ks.lo <= TK) {
    small_segment<T, DP, P>(a, it.kvh, qs, ks, lds[P == 1 ? w : 0][0], w);
    return;
  }
  bf16* t = P == 1 ? lds[w][0] : lds[0][2 * w];   // of a wave by itself
  for (int x = P == 2 ? 16 * w : 0; x < TK && vq0 + x < nv; x += 16 * P) {
    wave_sync();
    fwd_tile<T, DP, 1, W, false, 1, 1>(a, it, e, vq0 + x, qs, t, t + TL::elems, 0);
  }
}

// Joins many splits of a row and head: their weights first, then 4 features a thread over 64 groups of splits, whose sums
// are added in order.  16 features a block: with all of a row's in one, the few rows that are split this often kept few
// CUs busy (8 rows of 2,048 splits: 24.8 us against 13.3).
constexpr int kMaxSplit = 2048;
template <typename T, int DP>
__global__ __launch_bounds__(256) void fwd_join_many_kernel(Args a) {
  __shared__ float wt[kMaxSplit], red[4];
  __shared__ f32x4 part[64][4];
  const uint32_t r = blockIdx.x;
  const int head = (int)(r % (uint32_t)a.Hq), t = threadIdx.x;
  const int64_t row = r / (uint32_t)a.Hq;
  float m = kLowest;
  for (int s = t; s < a.nsplit; s += 256) m = fmaxf(m, part_ml(a, DP, s, r)[0]);
  for (int x = 32; x; x >>= 1) m = fmaxf(m, shfl_xor(m, x));
  if ((t & 63) == 0) red[t >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  __syncthreads();
  float sum = 0.f;
  for (int s = t; s < a.nsplit; s += 256) {
    const float* p = part_ml(a, DP, s, r);
    wt[s] = __builtin_amdgcn_exp2f(p[0] - m);
    sum = __builtin_fmaf(p[1], wt[s], sum);
  }
  for (int x = 32; x; x >>= 1) sum += shfl_xor(sum, x);
  if ((t & 63) == 0) red[t >> 6] = sum;
  __syncthreads();
  sum = (red[0] + red[1]) + (red[2] + red[3]);
  const int f = 16 * (int)blockIdx.y + 4 * (t & 3), gr = t >> 2;
  f32x4 o = zero4();
#pragma unroll 8
  for (int s = gr; s < a.nsplit; s += 64) o += load4_f32(part_o(a, DP, s, r) + f) * wt[s];
  part[gr][t & 3] = o;
  __syncthreads();
  for (int h = 32; h; h >>= 1) {
    if (gr < h) part[gr][t & 3] += part[gr + h][t & 3];
    __syncthreads();
  }
  if (gr) return;
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  if (f < a.D) store4((T*)a.out + row * a.o_r + head * a.o_h + f, part[0][t & 3] * inv);
  if (a.lse && t == 0 && blockIdx.y == 0) a.lse[(int64_t)head * a.Nq + row] = (m + __builtin_amdgcn_logf(sum)) * kLn2;
}
// Joins few splits, or those of many rows: 4 features a thread
constexpr int kFewSplits = 16;
template <typename T, int DP>
__global__ __launch_bounds__(256) void fwd_join_kernel(Args a) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, r = t / (DP / 4);
  const int f = 4 * (int)(t % (DP / 4));
  if (r >= (int64_t)a.Nq * a.Hq) return;
  const int head = (int)((uint32_t)r % (uint32_t)a.Hq);
  const int64_t row = (uint32_t)r / (uint32_t)a.Hq;
  float m = kLowest, sum = 0.f;
  for (int s = 0; s < a.nsplit; ++s) m = fmaxf(m, part_ml(a, DP, s, r)[0]);
  f32x4 o = zero4();
#pragma unroll 4
  for (int s = 0; s < a.nsplit; ++s) {
    const float* p = part_ml(a, DP, s, r);
    const float x = __builtin_amdgcn_exp2f(p[0] - m);
    sum = __builtin_fmaf(p[1], x, sum);
    o += load4_f32(part_o(a, DP, s, r) + f) * x;
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  if (f < a.D) store4((T*)a.out + row * a.o_r + head * a.o_h + f, o * inv);
  if (a.lse && f == 0) a.lse[(int64_t)head * a.Nq + row] = (m + __builtin_amdgcn_logf(sum)) * kLn2;
}

template <typename T, int DP, int R, int W, bool SH, int KT, int KC>
static void go(const Args& a, const Plan& p, hipStream_t st) {
  const int64_t n = p.slots * a.Hkv * a.nsplit;
  in_parts(a, SH ? n : cdiv(n, W), [&](const Args& x, uint32_t blocks) {
    fwd_kernel<T, DP, R, W, SH, KT, KC><<<blocks, 64 * W, 0, st>>>(x, (uint32_t)n);
  });
}
template <typename T, int DP>
static int launch_t(const Args& a, const Plan& p, hipStream_t st) {
  constexpr int tile = 2 * Tile<T, DP>::elems * 2, W = 4 * tile <= 65536 ? 4 : 2 * tile <= 65536 ? 2 : 1;
  constexpr bool f32 = Num<T>::planes == 3;
  constexpr int KT = f32 ? (DP <= 32 ? 2 : 1) : 2, KC = f32 || DP == 128 ? 1 : 2;
  if constexpr (DP <= (f32 ? 32 : 64)) {
    // short segments on both axes
    if (p.form == 0 && a.nsplit == 1 && a.Nk <= kShortMean * (int64_t)(a.B > 0 ? a.B : 1)) {
      constexpr int tile3 = 3 * Tile<T, DP>::elems * 2, W3 = 4 * tile3 <= 65536 ? 4 : 2;
      Args x = a;
      const int64_t slots = (int64_t)a.Nq * a.G / TK + a.B + 2, n = slots * a.Hkv;
      x.slots = (uint32_t)slots;
      x.guess = (float)(a.B + 2) / (float)slots;
      x.by_slots = Div::of(x.slots);
      // Two waves a segment where its products take long (one and two waves, 10 .. 30 rows a segment, 4 heads: fp32, D = 32,
      // 4,000 segments 59 and 51 us; bf16, D = 64 41 and 32), not where they do not (bf16, D = 32: 18.6 and 20.6)
      constexpr int P = f32 || DP == 64 ? 2 : 1, WS = P == 2 ? 2 : W3;
      in_parts(x, cdiv(n, WS / P), [&](const Args& y, uint32_t blocks) {
        short_kernel<T, DP, P, WS><<<blocks, 64 * WS, 0, st>>>(y, (uint32_t)n);
      });
      return (int)hipGetLastError();
    }
  }
  if constexpr (f32 && DP == 128) go<T, DP, 1, 4, true, KT, KC>(a, p, st);
  else if (p.form == 0) go<T, DP, 1, W, false, 1, 1>(a, p, st);
  else if (p.form == 1) go<T, DP, 1, 4, true, f32 ? KT : 1, 1>(a, p, st);
  else go<T, DP, 2, 4, true, KT, KC>(a, p, st);
  const int64_t rows = (int64_t)a.Nq * a.Hq;
  if (a.nsplit > kFewSplits && rows * (DP / 4) < 65536) fwd_join_many_kernel<T, DP><<<dim3((uint32_t)rows, DP / 16), 256, 0, st>>>(a);
  else if (a.nsplit > 1) fwd_join_kernel<T, DP><<<(uint32_t)cdiv(rows * (DP / 4), 256), 256, 0, st>>>(a);
  return (int)hipGetLastError();
}
template <typename T>
static int launch_d(const Args& a, const Plan& p, hipStream_t st) {
  switch (padded(a.D)) {
    case 16: return launch_t<T, 16>(a, p, st);
    case 32: return launch_t<T, 32>(a, p, st);
    case 64: return launch_t<T, 64>(a, p, st);
    default: return launch_t<T, 128>(a, p, st);
  }
}
int launch_fwd(const Args& a, bool is_bf16, const Plan& p, hipStream_t st) {
  return is_bf16 ? launch_d<bf16>(a, p, st) : launch_d<float>(a, p, st);
}

}  // namespace attn
}  // namespace egnn
