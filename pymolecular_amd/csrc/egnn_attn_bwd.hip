// Segment attention, backward.  With p = e^{s - lse} recomputed from the forward's statistics,
//   delta_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i.
// dq's kernel owns tiles of queries and walks the keys, dk and dv's owns tiles of keys and walks the queries (of all
// heads of the group); each sum is made by one owner in a fixed order, so there are no atomics.  That takes seven products
// where one kernel with atomics on dq would take five.
//
// delta.  o is the rounded output, so in bf16 do . o is off by up to 2^-9 |do| |o|, which shows where a row has few keys.
// As sum_j p_ij = 1, delta is also sum_j p_ij dp_ij: where a wave has all keys of its rows in one step (molecules) it
// takes that, and reads no o; on a longer axis it starts from do . o and adds what the ds sum to before dk's kernel reads it.
#include "egnn_attn.h"

namespace egnn {
namespace attn {

template <typename T, int DP, int R, int W, bool SH>
__global__ __launch_bounds__(64 * W, SH ? 2 : 1) void dq_kernel(Args a, uint32_t n_items) {
  typedef Tile<T, DP> TL;
  typedef typename Num<T>::Frag Frag;
  constexpr int NT = SH ? 64 * W : 64, BQ = 16 * R * (SH ? W : 1);
  __shared__ __attribute__((aligned(16))) bf16 lds[SH ? 1 : W][2][TL::elems];
  Item it;
  if (!item_of<W, SH>(a, n_items, it)) return;
  const int l = lane_id(), c = l & 15, g = l >> 4, w = threadIdx.x >> 6;
  bf16 *sK = lds[SH ? 0 : w][0], *sV = lds[SH ? 0 : w][1];
  int vq0;
  Seg qs;
  const int e = find_tile<BQ>(a.q_ptr, a.B, a.Nq, a.G, it.slot, vq0, qs);
  if (vq0 < 0) return;
  const Seg ks = other_rows(a.kv_ptr, e, a.B, a.Nk);
  const int nv = (qs.hi - qs.lo) * a.G, v0 = vq0 + (SH ? 16 * R * w : 0);
  const bool act = v0 < nv;
  int j, j1;
  split_range<TK>(ks.lo, ks.hi, a.nsplit, it.sp, j, j1);
  const bool one = !SH && a.nsplit == 1 && j1 - j <= TK;   // all keys in one step

  Stage<T, DP, 1, NT> stK, stV;
  uint32_t offK[stK.PER], offV[stV.PER];
  const int64_t krb = a.k_r * (int64_t)sizeof(T), vrb = a.v_r * (int64_t)sizeof(T);
  stK.offsets(offK, krb, a.D);
  stV.offsets(offV, vrb, a.D);
  const T *kb = (const T*)a.k + it.kvh * a.k_h, *vb = (const T*)a.v + it.kvh * a.v_h;
  uint8_t mb = 1;
  auto fetch = [&](int j) {
    const int n = j1 - j < TK ? j1 - j : TK;
    stK.load(rows_buffer(kb + j * a.k_r, n, krb, a.D * (int)sizeof(T)), offK);
    stV.load(rows_buffer(vb + j * a.v_r, n, vrb, a.D * (int)sizeof(T)), offV);
    if (a.mask) mb = l < n ? a.mask[j + l] : 0;
  };
  if (j < j1) fetch(j);

  typename TL::Feat Q[R][TL::NK], GO[R][TL::NK];
  int row[R], head[R];
  bool live[R], none[R];
  float delta[R], ref[R], sum[R];
  f32x4 dQ[R][TL::NB];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int v = v0 + 16 * r + c;
    live[r] = v < nv;
    const uint32_t i = live[r] ? a.by_g(v) : 0;
    row[r] = qs.lo + (int)i;
    head[r] = it.kvh * a.G + (live[r] ? v - (int)i * a.G : 0);
    const T *qp = live[r] ? (const T*)a.q + row[r] * a.q_r + head[r] * a.q_h : nullptr,
            *gp = live[r] ? (const T*)a.go + row[r] * a.go_r + head[r] * a.go_h : nullptr,
            *op = (const T*)a.o + row[r] * a.o_r + head[r] * a.o_h;
    const float lse = live[r] ? a.lse[(int64_t)head[r] * a.Nq + row[r]] * kLog2e : INFINITY;
    delta[r] = 0.f;
#pragma unroll
    for (int kk = 0; kk < TL::NK; ++kk) {
      Q[r][kk] = TL::column(qp, kk, g, a.D, a.flip);
      GO[r][kk] = TL::column(gp, kk, g, a.D, 0);
      if (!one && live[r]) delta[r] += TL::dot(gp, op, kk, g, a.D);
    }
    if (!one) delta[r] = col_sum(delta[r]);
    none[r] = lse == -INFINITY;              // a row without keys: no gradient from it or to it
    ref[r] = none[r] ? INFINITY : lse;
    sum[r] = 0.f;
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) dQ[r][b] = zero4();
  }

  for (; j < j1; j += TK) {
    uint64_t bits = first_bits(j1 - j < TK ? j1 - j : TK);
    if (a.mask) {                            // what a masked key holds must not meet a ds of 0
      bits &= __ballot(mb != 0);
      stK.keep(bits);
    }
    tile_sync<SH>();
    stK.store(sK);
    stV.store(sV);
    tile_sync<SH>();
    if (j + TK < j1) fetch(j + TK);
    if (!act) continue;
    f32x4 P[R][2], dS[R][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4 hi[R], lo[R], dhi[R], dlo[R];
#pragma unroll
      for (int r = 0; r < R; ++r) { hi[r] = zero4(); lo[r] = zero4(); dhi[r] = zero4(); dlo[r] = zero4(); }
#pragma unroll
      for (int kk = 0; kk < TL::NK; ++kk) {
        const auto A = TL::rows(sK, h, kk, c, g), B = TL::rows(sV, h, kk, c, g);
#pragma unroll
        for (int r = 0; r < R; ++r) { product1(hi[r], lo[r], A, Q[r][kk]); product1(dhi[r], dlo[r], B, GO[r][kk]); }
      }
      const uint32_t hb = (uint32_t)bits >> (16 * h + 4 * g);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        P[r][h] = result<T>(hi[r], lo[r]);
        dS[r][h] = result<T>(dhi[r], dlo[r]);
#pragma unroll
        for (int i = 0; i < 4; ++i) P[r][h][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(P[r][h][i], a.c2, -ref[r]));
        if (bits != 0xffffffffu) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            P[r][h][i] = (hb >> i) & 1 ? P[r][h][i] : 0.f;
            dS[r][h][i] = (hb >> i) & 1 ? dS[r][h][i] : 0.f;
          }
        }
      }
    }
    if (one) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) delta[r] = __builtin_fmaf(P[r][h][i], dS[r][h][i], delta[r]);
        delta[r] = col_sum(delta[r]);
      }
    }
    Frag F[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          dS[r][h][i] = P[r][h][i] * (dS[r][h][i] - delta[r]);
          if constexpr (!SH) sum[r] += dS[r][h][i];
        }
      F[r] = chain_frag<T>(dS[r][0], dS[r][1]);
    }
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) {
      const Frag A = TL::cols(sK, 0, b, c, g);
#pragma unroll
      for (int r = 0; r < R; ++r) accumulate(dQ[r][b], A, F[r]);
    }
  }
  const float sc = a.flip ? -a.scale : a.scale;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (!SH && !one && a.nsplit == 1) delta[r] += col_sum(sum[r]);
    if (!live[r]) continue;
    if (it.sp == 0 && g == 0) a.delta[(int64_t)head[r] * a.Nq + row[r]] = none[r] ? 0.f : delta[r];
    if (a.nsplit > 1) {
      float* p = a.part + ((int64_t)it.sp * a.Nq * a.Hq + (int64_t)row[r] * a.Hq + head[r]) * DP;
#pragma unroll
      for (int b = 0; b < TL::NB; ++b) store4(p + 16 * b + 4 * g, none[r] ? zero4() : dQ[r][b]);
      continue;
    }
    T* out = (T*)a.gq + row[r] * a.gq_r + head[r] * a.gq_h;
#pragma unroll
    for (int b = 0; b < TL::NB; ++b)
      if (16 * b + 4 * g < a.D) store4(out + 16 * b + 4 * g, none[r] ? zero4() : dQ[r][b] * sc);
  }
}

template <typename T, int DP, int R, int W, bool SH>
__global__ __launch_bounds__(64 * W, SH ? 2 : 1) void dkv_kernel(Args a, uint32_t n_items) {
  typedef Tile<T, DP> TL;
  typedef typename Num<T>::Frag Frag;
  constexpr int NT = SH ? 64 * W : 64, BK = 16 * R * (SH ? W : 1);
  __shared__ __attribute__((aligned(16))) bf16 lds[SH ? 1 : W][2][TL::elems];
  __shared__ __attribute__((aligned(16))) float stat[SH ? 1 : W][2][TK];
  Item it;
  if (!item_of<W, SH>(a, n_items, it)) return;
  const int l = lane_id(), c = l & 15, g = l >> 4, w = threadIdx.x >> 6;
  bf16 *sQ = lds[SH ? 0 : w][0], *sG = lds[SH ? 0 : w][1];
  float *sL = stat[SH ? 0 : w][0], *sD = stat[SH ? 0 : w][1];
  int k0;
  Seg ks;
  const int e = find_tile<BK>(a.kv_ptr, a.B, a.Nk, 1, it.slot, k0, ks);
  if (k0 < 0) return;
  const Seg qs = other_rows(a.q_ptr, e, a.B, a.Nq);
  const int key0 = ks.lo + k0 + (SH ? 16 * R * w : 0);
  const bool act = key0 < ks.hi;
  int j, j1;                                 // virtual rows of the segment
  split_range<TK>(0, (qs.hi - qs.lo) * a.G, a.nsplit, it.sp, j, j1);

  Stage<T, DP, 1, NT> stQ, stG;
  uint32_t offQ[stQ.PER], offG[stG.PER];
  const int64_t qrb = a.q_r * (int64_t)sizeof(T), grb = a.go_r * (int64_t)sizeof(T);
  stQ.offsets(offQ, qrb, a.D);
  stG.offsets(offG, grb, a.D);
  const T *qb = (const T*)a.q + (int64_t)it.kvh * a.G * a.q_h, *gb = (const T*)a.go + (int64_t)it.kvh * a.G * a.go_h;
  float lse = INFINITY, delta = 0.f;
  auto fetch = [&](int j) {
    const int n = j1 - j < TK ? j1 - j : TK, r0 = (int)a.by_g(j), first = qs.lo + r0;
    int rows = n;
    if (a.G > 1) {                           // rows and heads of the step's virtual rows
      const int u0 = j - r0 * a.G;           // head of the first one
      rows = (int)a.by_g(u0 + n - 1) + 1;
#pragma unroll
      for (int p = 0; p < stQ.PER; ++p) {
        const uint32_t u = u0 + stQ.row(p), i = a.by_g(u), h = u - i * a.G, f = stQ.feature(p);
        const bool ok = stQ.in(p) && stQ.row(p) < n && (int)f < a.D;
        offQ[p] = ok ? (uint32_t)((i * a.q_r + h * a.q_h + f) * (int64_t)sizeof(T)) : kOob;
        offG[p] = ok ? (uint32_t)((i * a.go_r + h * a.go_h + f) * (int64_t)sizeof(T)) : kOob;
      }
    }
    const int more = a.D * (int)sizeof(T);
    stQ.load(rows_buffer(qb + first * a.q_r, rows, qrb, more + (int)((a.G - 1) * a.q_h * (int64_t)sizeof(T))), offQ);
    stG.load(rows_buffer(gb + first * a.go_r, rows, grb, more + (int)((a.G - 1) * a.go_h * (int64_t)sizeof(T))), offG);
    // a row without keys, and one past the end, takes no part: its p is e^-inf
    lse = INFINITY;
    delta = 0.f;
    if (l < n) {
      const uint32_t v = j + l, i = a.by_g(v);
      const int64_t x = (int64_t)(it.kvh * a.G + (int)(v - i * a.G)) * a.Nq + qs.lo + (int)i;
      lse = a.lse[x];
      delta = a.delta[x];
    }
  };
  if (j < j1) fetch(j);

  typename TL::Feat K[R][TL::NK], V[R][TL::NK];
  int key[R];
  bool in[R], live[R];
  f32x4 dK[R][TL::NB], dV[R][TL::NB];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    key[r] = key0 + 16 * r + c;
    in[r] = key[r] < ks.hi;
    live[r] = in[r] && (!a.mask || a.mask[key[r]] != 0);
    const T *kp = live[r] ? (const T*)a.k + key[r] * a.k_r + it.kvh * a.k_h : nullptr,
            *vp = live[r] ? (const T*)a.v + key[r] * a.v_r + it.kvh * a.v_h : nullptr;
#pragma unroll
    for (int kk = 0; kk < TL::NK; ++kk) {
      K[r][kk] = TL::column(kp, kk, g, a.D, a.flip);   // the scale's sign
      V[r][kk] = TL::column(vp, kk, g, a.D, 0);
    }
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) { dK[r][b] = zero4(); dV[r][b] = zero4(); }
  }

  for (; j < j1; j += TK) {
    const float ref = lse == -INFINITY ? INFINITY : lse * kLog2e;
    const uint64_t bits = __ballot(ref != INFINITY);   // lanes 0 .. 31
    if (bits != 0xffffffffu) { stQ.keep(bits); stG.keep(bits); }
    tile_sync<SH>();
    stQ.store(sQ);
    stG.store(sG);
    if ((!SH || w == 0) && l < TK) { sL[l] = ref; sD[l] = delta; }
    tile_sync<SH>();
    if (j + TK < j1) fetch(j + TK);
    if (!act) continue;
    f32x4 P[R][2], dS[R][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4 hi[R], lo[R], dhi[R], dlo[R];
#pragma unroll
      for (int r = 0; r < R; ++r) { hi[r] = zero4(); lo[r] = zero4(); dhi[r] = zero4(); dlo[r] = zero4(); }
#pragma unroll
      for (int kk = 0; kk < TL::NK; ++kk) {
        const auto A = TL::rows(sQ, h, kk, c, g), B = TL::rows(sG, h, kk, c, g);
#pragma unroll
        for (int r = 0; r < R; ++r) { product1(hi[r], lo[r], A, K[r][kk]); product1(dhi[r], dlo[r], B, V[r][kk]); }
      }
      const f32x4 Lr = load4_f32(sL + 16 * h + 4 * g), D = load4_f32(sD + 16 * h + 4 * g);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        P[r][h] = result<T>(hi[r], lo[r]);
        dS[r][h] = result<T>(dhi[r], dlo[r]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          P[r][h][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(P[r][h][i], a.c2, -Lr[i]));
          dS[r][h][i] = P[r][h][i] * (dS[r][h][i] - D[i]);
        }
      }
    }
    Frag FP[R], FS[R];
#pragma unroll
    for (int r = 0; r < R; ++r) { FP[r] = chain_frag<T>(P[r][0], P[r][1]); FS[r] = chain_frag<T>(dS[r][0], dS[r][1]); }
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) {
      const Frag A = TL::cols(sG, 0, b, c, g), B = TL::cols(sQ, 0, b, c, g);
#pragma unroll
      for (int r = 0; r < R; ++r) { accumulate(dV[r][b], A, FP[r]); accumulate(dK[r][b], B, FS[r]); }
    }
  }
  const float sc = a.flip ? -a.scale : a.scale;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (!in[r]) continue;
    if (a.nsplit > 1) {
      float* p = a.part + ((int64_t)it.sp * a.Nk * a.Hkv + (int64_t)key[r] * a.Hkv + it.kvh) * (2 * DP);
#pragma unroll
      for (int b = 0; b < TL::NB; ++b) {
        store4(p + 16 * b + 4 * g, live[r] ? dK[r][b] : zero4());
        store4(p + DP + 16 * b + 4 * g, live[r] ? dV[r][b] : zero4());
      }
      continue;
    }
    T *gk = (T*)a.gk + key[r] * a.gk_r + it.kvh * a.gk_h, *gv = (T*)a.gv + key[r] * a.gv_r + it.kvh * a.gv_h;
#pragma unroll
    for (int b = 0; b < TL::NB; ++b)
      if (16 * b + 4 * g < a.D) {
        store4(gk + 16 * b + 4 * g, live[r] ? dK[r][b] * sc : zero4());
        store4(gv + 16 * b + 4 * g, live[r] ? dV[r][b] : zero4());
      }
  }
}

// out[row][head][f] = mul * sum over the splits: 32 values a block, 8 groups of splits, added in order; the partial rows
// are `width` values apart, the values from `off` on
template <typename T>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* part, int nsplit, int64_t rows, int heads, int D, int width, int off,
                                                        float mul, T* out, int64_t rs, int64_t hs) {
  __shared__ float red[8][32];
  const int x = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int64_t t = (int64_t)blockIdx.x * 32 + x, r = t / D, n = rows * heads;
  const int f = (int)(t - r * D);
  float s = 0.f;
  if (r < n) {
#pragma unroll 4
    for (int i = k; i < nsplit; i += 8) s += part[(i * n + r) * width + off + f];
  }
  red[k][x] = s;
  __syncthreads();
  if (k || r >= n) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += red[i][x];
  out[(r / heads) * rs + (r % heads) * hs + f] = from_f32<T>(s * mul);
}

template <typename T, int DP, int R, int W, bool SH>
static void go_q(const Args& a, const Plan& p, hipStream_t st) {
  const int64_t n = p.slots * a.Hkv * a.nsplit;
  dq_kernel<T, DP, R, W, SH><<<(uint32_t)(SH ? n : cdiv(n, W)), 64 * W, 0, st>>>(a, (uint32_t)n);
}
template <typename T, int DP, int R, int W, bool SH>
static void go_k(const Args& a, const Plan& p, hipStream_t st) {
  const int64_t n = p.slots * a.Hkv * a.nsplit;
  dkv_kernel<T, DP, R, W, SH><<<(uint32_t)(SH ? n : cdiv(n, W)), 64 * W, 0, st>>>(a, (uint32_t)n);
}
template <typename T, int DP>
static int launch_t(Args a, const Plan& pq, const Plan& pk, hipStream_t st) {
  constexpr int tile = 2 * Tile<T, DP>::elems * 2 + 256, W = 4 * tile <= 65536 ? 4 : 2 * tile <= 65536 ? 2 : 1;
  constexpr bool wide = Num<T>::planes == 3 && DP == 128;
  auto blocks = [&](int64_t n) { return (uint32_t)cdiv(n * a.D, 32); };
  a.nsplit = pq.nsplit;
  a.by_split = Div::of(a.nsplit);
  if (a.Nq) {
    if constexpr (wide) go_q<T, DP, 1, 4, true>(a, pq, st);
    else if (pq.form == 0) go_q<T, DP, 1, W, false>(a, pq, st);
    else if (pq.form == 1) go_q<T, DP, 1, 4, true>(a, pq, st);
    else go_q<T, DP, 2, 4, true>(a, pq, st);
    if (a.nsplit > 1)
      sum_parts_kernel<T><<<blocks((int64_t)a.Nq * a.Hq), 256, 0, st>>>(a.part, a.nsplit, a.Nq, a.Hq, a.D, DP, 0,
                                                                        a.flip ? -a.scale : a.scale, (T*)a.gq, a.gq_r, a.gq_h);
  }
  a.nsplit = pk.nsplit;
  a.by_split = Div::of(a.nsplit);
  if (a.Nk) {
    if constexpr (wide) go_k<T, DP, 1, 4, true>(a, pk, st);
    else if (pk.form == 0) go_k<T, DP, 1, W, false>(a, pk, st);
    else if (pk.form == 1) go_k<T, DP, 1, 4, true>(a, pk, st);
    else if constexpr (DP <= (Num<T>::planes == 1 ? 64 : 32)) go_k<T, DP, 2, 4, true>(a, pk, st);
    if (a.nsplit > 1) {
      const uint32_t nb = blocks((int64_t)a.Nk * a.Hkv);
      const float sc = a.flip ? -a.scale : a.scale;
      sum_parts_kernel<T><<<nb, 256, 0, st>>>(a.part, a.nsplit, a.Nk, a.Hkv, a.D, 2 * DP, 0, sc, (T*)a.gk, a.gk_r, a.gk_h);
      sum_parts_kernel<T><<<nb, 256, 0, st>>>(a.part, a.nsplit, a.Nk, a.Hkv, a.D, 2 * DP, DP, 1.0f, (T*)a.gv, a.gv_r, a.gv_h);
    }
  }
  return (int)hipGetLastError();
}
template <typename T>
static int launch_d(const Args& a, const Plan& pq, const Plan& pk, hipStream_t st) {
  switch (padded(a.D)) {
    case 16: return launch_t<T, 16>(a, pq, pk, st);
    case 32: return launch_t<T, 32>(a, pq, pk, st);
    case 64: return launch_t<T, 64>(a, pq, pk, st);
    default: return launch_t<T, 128>(a, pq, pk, st);
  }
}
int launch_bwd(const Args& a, bool is_bf16, const Plan& pq, const Plan& pk, hipStream_t st) {
  return is_bf16 ? launch_d<bf16>(a, pq, pk, st) : launch_d<float>(a, pq, pk, st);
}

}  // namespace attn
}  // namespace egnn
