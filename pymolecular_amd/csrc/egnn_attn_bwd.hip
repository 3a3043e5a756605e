// Segment attention, backward.  With p = e^{s - lse} recomputed from the forward's statistics,
//   delta_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i.
// dq's kernel owns tiles of queries and walks the keys, dk and dv's owns tiles of keys and walks the queries (of all
// heads of the group); each sum is made by one owner in a fixed order, so there are no atomics.  That takes seven products
// (eight in bf16, below) where one kernel with atomics on dq would take five.
//
// delta.  o is the rounded output, so in bf16 do . o is off by up to 2^-9 |do| |o|, and the ds made with it sum to that
// instead of 0.  Where keys and values have a common part (a projection's bias), o has it too and dq takes the error times
// that of the keys: with three times the spread of the values in both, dq was off by 7 % of its norm at 512 keys and by 13 %
// at 4,000, with ten times by as much as it is long.  As sum_j p_ij = 1, delta is also sum_j p_ij dp_ij, and the ds made with
// a delta' sum to delta - delta'.  So in bf16 dq's kernel also sums p_ij k_j (one product more) and takes
// (delta - delta') sum_j p_ij k_j off dq, and dk's kernel reads the corrected delta; a wave that has all keys of its rows in
// one step (molecules) makes delta from p and dp at once and reads no o.  Left is the rounding of ds: errors of dq against
// 64 bits with 0, 1, 3 and 10 times the spread 2.4e-3, 2.9e-3, 5.2e-3 and 1.6e-2 of its norm.  The cost, backward alone:
// 64 x 512 rows, D = 32, 53.6 -> 59.9 us; 12,289 rows, D = 64, 600 -> 680; 80-row slabs and molecules 0 to 1 %.
// One case keeps do . o for dk: segments of more than 32 rows or keys in batches of short ones (launch_short), where dk's
// workgroups run beside dq's in one launch (a launch more: 14.2 -> 16.6 us, 1,024 molecules).  There dk takes the error times
// p_ij q_i: 2.6e-3 instead of 2.3e-3, and 6.7e-3 with three times the spread.  fp32 keeps do . o, whose error is one of fp32.
//
// Measured (each kernel alone, called back to back): 12,289 rows, 4 heads of 64, bf16, dq 315 us and dk, dv 338 us, 0.98 and
// 0.91 PFLOP/s of the four products each makes, bound by vector and MFMA issue (0.42 and 0.41, 0.36 and 0.38 of the cycles)
// and by two waves a SIMD; 128 molecules in fp32 8.2 us, bound by latency.
#include "egnn_attn.h"

namespace egnn {
namespace attn {

// The S and dp products of a step are made with the scale's sign in the exponent's factor.
__device__ __forceinline__ float signed_c2(const Args& a) { return a.flip ? -a.c2 : a.c2; }
__host__ __device__ __forceinline__ float signed_scale(const Args& a) { return a.flip ? -a.scale : a.scale; }

// dq of the tile from virtual row vq0 of segment e on; sK, sV: tiles of the wave's (SH: the workgroup's) own.  EX: exact
// delta (above)
template <typename T, int DP, int R, int W, bool SH, int KT, bool EX>
__device__ __forceinline__ void dq_tile(const Args& a, const Item& it, int e, int vq0, const Seg& qs, bf16* sK, bf16* sV, int w) {
  typedef Tile<T, DP, KT> TL;
  typedef typename Num<T>::Frag Frag;
  constexpr int NT = SH ? 64 * W : 64, KS = TK * KT;
  const int l = lane_id(), c = l & 15, g = l >> 4;
  const float c2 = signed_c2(a);
  const Seg ks = other_rows(a.kv_ptr, e, a.B, a.Nk, a.same, qs);
  const int nv = (qs.hi - qs.lo) * a.G, v0 = vq0 + (SH ? 16 * R * w : 0);
  const bool act = v0 < nv;
  int j = ks.lo + it.sp * KS;
  const int j1 = ks.hi, stride = KS * a.nsplit;
  const bool one = !SH && a.nsplit == 1 && j1 - j <= KS;   // all keys in one step

  Stage<T, DP, KT, NT> stK, stV;
  uint32_t offK[stK.PER], offV[stV.PER];
  const int64_t krb = a.k_r * (int64_t)sizeof(T), vrb = a.v_r * (int64_t)sizeof(T);
  stK.offsets(offK, krb, a.D);
  stV.offsets(offV, vrb, a.D);
  const T *kb = (const T*)a.k + it.kvh * a.k_h, *vb = (const T*)a.v + it.kvh * a.v_h;
  uint8_t mb[Bits<KT>::N];
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

  typename TL::Feat Q[R][TL::NK], GO[R][TL::NK];
  int row[R], head[R];
  bool live[R], none[R];
  float delta[R], ref[R], sum[R];
  Sum<T> dQ[R][TL::NB], PK[R][EX ? TL::NB : 1];   // PK: sum_j p_j k_j
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
      Q[r][kk] = TL::column(qp, kk, g, a.D, 0);
      GO[r][kk] = TL::column(gp, kk, g, a.D, 0);
      landed(Q[r][kk]);
      landed(GO[r][kk]);
      if (!one && live[r]) delta[r] += TL::dot(gp, op, kk, g, a.D);
    }
    if (!one) delta[r] = col_sum(delta[r]);
    none[r] = lse == -INFINITY;              // a row without keys: no gradient from it or to it
    ref[r] = none[r] ? INFINITY : lse;
    sum[r] = 0.f;
  }

  for (; j < j1; j += stride) {
    const int n = rows_at(j);
    Bits<KT> bits = step_bits<KT>(n);
    if (a.mask) {                            // what a masked key holds must not meet a ds of 0
#pragma unroll
      for (int k = 0; k < Bits<KT>::N; ++k) bits.w[k] &= __ballot(mb[k] != 0);
      stK.keep(bits);
    }
    tile_sync<SH>();
    stK.store(sK, n);
    stV.store(sV, n);
    tile_sync<SH>();
    if (j + stride < j1) fetch(j + stride);
    if (!act) continue;
    if constexpr (KT > 1) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int b = 0; b < TL::NB; ++b) dQ[r][b].begin();
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      if (KT > 1 && TK * t >= n) break;
      f32x4 P[R][2], dS[R][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x4 hi[R], lo[R], dhi[R], dlo[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          hi[r] = zero4();
          lo[r] = zero4();
          dhi[r] = f32x4{-delta[r], -delta[r], -delta[r], -delta[r]};   // dp - delta
          dlo[r] = zero4();
        }
#pragma unroll
        for (int kk = 0; kk < TL::NK; ++kk) {
          const auto A = TL::rows(sK, 2 * t + h, kk, c, g), B = TL::rows(sV, 2 * t + h, kk, c, g);
#pragma unroll
          for (int r = 0; r < R; ++r) { product1(hi[r], lo[r], A, Q[r][kk]); product1(dhi[r], dlo[r], B, GO[r][kk]); }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          P[r][h] = result<T>(hi[r], lo[r]);
          dS[r][h] = result<T>(dhi[r], dlo[r]);
#pragma unroll
          for (int i = 0; i < 4; ++i) P[r][h][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(P[r][h][i], c2, -ref[r]));
        }
      }
      if (const uint32_t b = bits.step(t); b != 0xffffffffu) {
        const uint32_t tb = b >> (4 * g);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool ok = (tb >> (16 * h + i)) & 1;
#pragma unroll
            for (int r = 0; r < R; ++r) {
              P[r][h][i] = ok ? P[r][h][i] : 0.f;
              dS[r][h][i] = ok ? dS[r][h][i] : 0.f;
            }
          }
      }
      if (one) {                             // delta was 0 so far
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) delta[r] = __builtin_fmaf(P[r][h][i], dS[r][h][i], delta[r]);
          delta[r] = col_sum(delta[r]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) dS[r][h][i] -= delta[r];
        }
      }
      Frag F[R], FP[EX ? R : 1];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if constexpr (EX) if (!one) FP[r] = chain_frag<T>(P[r][0], P[r][1]);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dS[r][h][i] *= P[r][h][i];
            if constexpr (EX) sum[r] += dS[r][h][i];
          }
        F[r] = chain_frag<T>(dS[r][0], dS[r][1]);
      }
#pragma unroll
      for (int b = 0; b < TL::NB; ++b) {
        const Frag A = TL::cols(sK, t, b, c, g);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if constexpr (KT == 1) dQ[r][b].one(A, F[r]);
          else dQ[r][b].add(A, F[r]);
          if constexpr (EX) if (!one) PK[r][b].add(A, FP[r]);
        }
      }
    }
    if constexpr (KT > 1) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int b = 0; b < TL::NB; ++b) dQ[r][b].end();
    }
  }
  const float sc = signed_scale(a);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float off = 0.f;                         // of these keys: delta less the one that the ds were made with
    if constexpr (EX) {
      if (!one) off = col_sum(sum[r]);
      if (a.nsplit == 1) {
        delta[r] += off;
#pragma unroll
        for (int b = 0; b < TL::NB; ++b) dQ[r][b].v -= PK[r][b].v * off;
      }
    }
    if (!live[r]) continue;
    if (a.delta && it.sp == 0 && g == 0) a.delta[(int64_t)head[r] * a.Nq + row[r]] = none[r] ? 0.f : delta[r];
    if (a.nsplit > 1) {
      const int64_t rows = (int64_t)a.Nq * a.Hq, x = (int64_t)it.sp * rows + (int64_t)row[r] * a.Hq + head[r];
      float* p = a.part + x * ((EX ? 2 : 1) * DP);
#pragma unroll
      for (int b = 0; b < TL::NB; ++b) {
        store4(p + 16 * b + 4 * g, none[r] ? zero4() : dQ[r][b].v);
        if constexpr (EX) store4(p + DP + 16 * b + 4 * g, none[r] ? zero4() : PK[r][b].v);
      }
      if constexpr (EX) if (g == 0) a.part[a.nsplit * rows * (2 * DP) + x] = none[r] ? 0.f : off;
      continue;
    }
    T* out = (T*)a.gq + row[r] * a.gq_r + head[r] * a.gq_h;
    f32x4 o[TL::NB];
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) o[b] = none[r] ? zero4() : dQ[r][b].v * sc;
    store_row<TL::NB>(out, o, g, a.D);
  }
}

// dk and dv of the tile from key k0 of segment e on.  OD: delta is made from o here, not read (no launch before this one
// has written it).
template <typename T, int DP, int R, int W, bool SH, int KT, bool OD>
__device__ __forceinline__ void dkv_tile(const Args& a, const Item& it, int e, int k0, const Seg& ks, bf16* sQ, bf16* sG, float* sL,
                                         float* sD, int w) {
  typedef Tile<T, DP, KT> TL;
  typedef typename Num<T>::Frag Frag;
  constexpr int NT = SH ? 64 * W : 64, KS = TK * KT;
  const int l = lane_id(), c = l & 15, g = l >> 4;
  const float c2 = signed_c2(a);
  const Seg qs = other_rows(a.q_ptr, e, a.B, a.Nq, a.same, ks);
  const int key0 = ks.lo + k0 + (SH ? 16 * R * w : 0);
  const bool act = key0 < ks.hi;
  int j = it.sp * KS;                        // virtual rows of the segment
  const int j1 = (qs.hi - qs.lo) * a.G, stride = KS * a.nsplit;

  Stage<T, DP, KT, NT> stQ, stG, stO;
  uint32_t offQ[stQ.PER], offG[stG.PER], offO[stO.PER];
  const int64_t qrb = a.q_r * (int64_t)sizeof(T), grb = a.go_r * (int64_t)sizeof(T);
  stQ.offsets(offQ, qrb, a.D);
  stG.offsets(offG, grb, a.D);
  const int64_t orb = a.o_r * (int64_t)sizeof(T);
  if constexpr (OD) stO.offsets(offO, orb, a.D);
  const T *qb = (const T*)a.q + (int64_t)it.kvh * a.G * a.q_h, *gb = (const T*)a.go + (int64_t)it.kvh * a.G * a.go_h,
          *ob = (const T*)a.o + (int64_t)it.kvh * a.G * a.o_h;
  constexpr int NL = Bits<KT>::N;
  float lse[NL], delta[NL];                  // of row 64 k + lane
  auto rows_at = [&](int j) { return j1 - j < KS ? j1 - j : KS; };
  auto fetch = [&](int j) {
    const int n = rows_at(j), r0 = (int)a.by_g(j), first = qs.lo + r0;
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
        if constexpr (OD) offO[p] = ok ? (uint32_t)((i * a.o_r + h * a.o_h + f) * (int64_t)sizeof(T)) : kOob;
      }
    }
    const int more = a.D * (int)sizeof(T);
    stQ.load(rows_buffer(qb + first * a.q_r, rows, qrb, more + (int)((a.G - 1) * a.q_h * (int64_t)sizeof(T))), offQ, n);
    stG.load(rows_buffer(gb + first * a.go_r, rows, grb, more + (int)((a.G - 1) * a.go_h * (int64_t)sizeof(T))), offG, n);
    if constexpr (OD)
      stO.load(rows_buffer(ob + first * a.o_r, rows, orb, more + (int)((a.G - 1) * a.o_h * (int64_t)sizeof(T))), offO, n);
    // a row without keys, and one past the end, takes no part: its p is e^-inf
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      lse[k] = INFINITY;
      delta[k] = 0.f;
      if (64 * k + l < n) {
        const uint32_t v = j + 64 * k + l, i = a.by_g(v);
        const int64_t x = (int64_t)(it.kvh * a.G + (int)(v - i * a.G)) * a.Nq + qs.lo + (int)i;
        lse[k] = a.lse[x];
        if constexpr (!OD) delta[k] = a.delta[x];
      }
    }
  };
  if (j < j1) fetch(j);

  typename TL::Feat K[R][TL::NK], V[R][TL::NK];
  int key[R];
  bool in[R], live[R];
  Sum<T> dK[R][TL::NB], dV[R][TL::NB];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    key[r] = key0 + 16 * r + c;
    in[r] = key[r] < ks.hi;
    live[r] = in[r] && (!a.mask || a.mask[key[r]] != 0);
    const T *kp = live[r] ? (const T*)a.k + key[r] * a.k_r + it.kvh * a.k_h : nullptr,
            *vp = live[r] ? (const T*)a.v + key[r] * a.v_r + it.kvh * a.v_h : nullptr;
#pragma unroll
    for (int kk = 0; kk < TL::NK; ++kk) {
      K[r][kk] = TL::column(kp, kk, g, a.D, 0);
      V[r][kk] = TL::column(vp, kk, g, a.D, 0);
      landed(K[r][kk]);
      landed(V[r][kk]);
    }
  }

  for (; j < j1; j += stride) {
    const int n = rows_at(j);
    Bits<KT> bits;
    bool all = true;
    float ref[NL];
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      ref[k] = lse[k] == -INFINITY ? INFINITY : lse[k] * kLog2e;
      bits.w[k] = __ballot(ref[k] != INFINITY);
      all &= bits.w[k] == step_bits<KT>(KS).w[k];
    }
    if (!all) { stQ.keep(bits); stG.keep(bits); }
    tile_sync<SH>();
    stQ.store(sQ, n);
    stG.store(sG, n);
    if (!SH || w == 0) {
#pragma unroll
      for (int k = 0; k < NL; ++k)
        if (64 * k + l < KS) {
          sL[64 * k + l] = ref[k];
          if constexpr (!OD) sD[64 * k + l] = -delta[k];
        }
    }
    if constexpr (OD) {                      // the threads of a row are neighbours
#pragma unroll
      for (int p = 0; p < stG.PER; ++p) {
        float d = dot8(stG.r[p], stO.r[p]);
#pragma unroll
        for (int x = 1; x < stG.CH; x <<= 1) d += shfl_xor(d, x);
        if (stG.in(p) && stG.feature(p) == 0) sD[stG.row(p)] = -d;
      }
    }
    tile_sync<SH>();
    if (j + stride < j1) fetch(j + stride);
    if (!act) continue;
    if constexpr (KT > 1) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int b = 0; b < TL::NB; ++b) { dK[r][b].begin(); dV[r][b].begin(); }
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      if (KT > 1 && TK * t >= n) break;
      f32x4 P[R][2], dS[R][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int b = 2 * t + h;
        const f32x4 Lr = load4_f32(sL + 16 * b + 4 * g), nD = load4_f32(sD + 16 * b + 4 * g);
        f32x4 hi[R], lo[R], dhi[R], dlo[R];
#pragma unroll
        for (int r = 0; r < R; ++r) { hi[r] = zero4(); lo[r] = zero4(); dhi[r] = nD; dlo[r] = zero4(); }   // dp - delta
#pragma unroll
        for (int kk = 0; kk < TL::NK; ++kk) {
          const auto A = TL::rows(sQ, b, kk, c, g), B = TL::rows(sG, b, kk, c, g);
#pragma unroll
          for (int r = 0; r < R; ++r) { product1(hi[r], lo[r], A, K[r][kk]); product1(dhi[r], dlo[r], B, V[r][kk]); }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          P[r][h] = result<T>(hi[r], lo[r]);
          dS[r][h] = result<T>(dhi[r], dlo[r]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            P[r][h][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(P[r][h][i], c2, -Lr[i]));
            dS[r][h][i] *= P[r][h][i];
          }
        }
      }
      Frag FP[R], FS[R];
#pragma unroll
      for (int r = 0; r < R; ++r) { FP[r] = chain_frag<T>(P[r][0], P[r][1]); FS[r] = chain_frag<T>(dS[r][0], dS[r][1]); }
      // rows that take no part are zeros, and 0 times an infinity of a key is NaN
      if (const uint32_t b = bits.step(t); b != 0xffffffffu) {
        const u32x4 m = chain_rows(b >> (4 * g));
#pragma unroll
        for (int r = 0; r < R; ++r) { FP[r] = masked(FP[r], m); FS[r] = masked(FS[r], m); }
      }
#pragma unroll
      for (int b = 0; b < TL::NB; ++b) {
        const Frag A = TL::cols(sG, t, b, c, g), B = TL::cols(sQ, t, b, c, g);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if constexpr (KT == 1) { dV[r][b].one(A, FP[r]); dK[r][b].one(B, FS[r]); }
          else { dV[r][b].add(A, FP[r]); dK[r][b].add(B, FS[r]); }
        }
      }
    }
    if constexpr (KT > 1) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int b = 0; b < TL::NB; ++b) { dK[r][b].end(); dV[r][b].end(); }
    }
  }
  const float sc = signed_scale(a);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (!in[r]) continue;
    if (a.nsplit > 1) {
      float* p = a.part + ((int64_t)it.sp * a.Nk * a.Hkv + (int64_t)key[r] * a.Hkv + it.kvh) * (2 * DP);
#pragma unroll
      for (int b = 0; b < TL::NB; ++b) {
        store4(p + 16 * b + 4 * g, live[r] ? dK[r][b].v : zero4());
        store4(p + DP + 16 * b + 4 * g, live[r] ? dV[r][b].v : zero4());
      }
      continue;
    }
    f32x4 o[TL::NB];
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) o[b] = live[r] ? dK[r][b].v * sc : zero4();
    store_row<TL::NB>((T*)a.gk + key[r] * a.gk_r + it.kvh * a.gk_h, o, g, a.D);
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) o[b] = live[r] ? dV[r][b].v : zero4();
    store_row<TL::NB>((T*)a.gv + key[r] * a.gv_r + it.kvh * a.gv_h, o, g, a.D);
  }
}

// Waves a SIMD that dq's registers leave room for: the sums of p k take its 128-row tiles to 143 registers at D = 32 and 219
// at D = 64.  (D = 64 held to three waves spills 50.  The backward of 12,289 rows: as here 680 us, in steps of 32 keys 691, in
// 64-row tiles 772.)
template <typename T, int DP, int R> constexpr int dq_occupancy() {
  return Num<T>::planes == 1 ? (R == 2 ? (DP <= 16 ? 4 : DP == 32 ? 3 : 2) : DP <= 64 ? 4 : 3) : 2;
}
template <typename T, int DP, int R, int W, bool SH, int KT, bool EX>
__global__ __launch_bounds__(64 * W, (SH ? dq_occupancy<T, DP, R>() : 1)) void dq_kernel(Args a, uint32_t n_items) {
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
  dq_tile<T, DP, R, W, SH, KT, EX>(a, it, e, vq0, qs, lds[SH ? 0 : w][0], lds[SH ? 0 : w][1], w);
}

// (bf16, D = 32, 128 rows: 128 registers, four waves a SIMD; 136 took 64 chains of 512 rows from 68 to 72 us)
template <typename T, int DP, int R, int W, bool SH, int KT>
__global__ __launch_bounds__(64 * W, SH ? (Num<T>::planes == 1 && DP <= 32 ? 4 : 2) : 1) void dkv_kernel(Args a, uint32_t n_items) {
  typedef Tile<T, DP, KT> TL;
  constexpr int BK = 16 * R * (SH ? W : 1);
  __shared__ __attribute__((aligned(16))) bf16 lds[SH ? 1 : W][2][TL::elems];
  __shared__ __attribute__((aligned(16))) float stat[SH ? 1 : W][2][TK * KT];
  Item it;
  if (!item_of<W, SH>(a, n_items, it)) return;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), x = SH ? 0 : w;
  int k0;
  Seg ks;
  const int e = find_tile<BK>(a.kv_ptr, a.B, a.Nk, 1, a.guess, it.slot, k0, ks);
  if (k0 < 0) return;
  dkv_tile<T, DP, R, W, SH, KT, false>(a, it, e, k0, ks, lds[x][0], lds[x][1], stat[x][0], stat[x][1], w);
}

// ---- short segments: one launch -------------------------------------------------------
// A segment with at most 32 virtual rows and 32 keys (a molecule) is one wave's, or two waves' (P): its q, k, v and do are
// read once, its gradients written once, delta is exact, and neither o nor a statistic of another launch is read.  Both
// orientations of the scores are made from the same LDS tiles, the second for the sums over the queries.  Two waves take
// 16 columns each, first of the queries, then of the keys.
template <typename T, int DP, int P>
__device__ __forceinline__ void small_segment(const Args& a, int kvh, const Seg& qs, const Seg& ks, bf16* lds, float* sL, float* sD, int w) {
  typedef Tile<T, DP> TL;
  typedef typename Num<T>::Frag Frag;
  const int l = lane_id(), c = l & 15, g = l >> 4;
  const int nv = (qs.hi - qs.lo) * a.G, nk = ks.hi - ks.lo;
  bf16 *sQ = lds, *sG = sQ + TL::elems, *sK = sG + TL::elems, *sV = sK + TL::elems;
  const int64_t e = sizeof(T);
  const int last = a.D * (int)e;
  uint32_t kbits;                            // keys that exist, and are not masked
  {
    // of two waves the first brings q, do and lse, the second k and v
    const bool bq = P == 1 || w == 0, bk = (P == 1 || w == 1) && nk;
    Stage<T, DP, 1, 64> stQ, stG, stK, stV;
    float ref = INFINITY;                    // of row l
    if (bq) {
      uint32_t offQ[stQ.PER], offG[stQ.PER];
      if (a.G == 1) {
        stQ.offsets(offQ, a.q_r * e, a.D);
        stG.offsets(offG, a.go_r * e, a.D);
      } else {
#pragma unroll
        for (int p = 0; p < stQ.PER; ++p) {
          const uint32_t u = stQ.row(p), i = a.by_g(u), h = u - i * a.G, f = stQ.feature(p);
          const bool ok = stQ.in(p) && (int)u < nv && (int)f < a.D;
          offQ[p] = ok ? (uint32_t)((i * a.q_r + h * a.q_h + f) * e) : kOob;
          offG[p] = ok ? (uint32_t)((i * a.go_r + h * a.go_h + f) * e) : kOob;
        }
      }
      const int rows = qs.hi - qs.lo;
      stQ.load(rows_buffer((const T*)a.q + qs.lo * a.q_r + (int64_t)kvh * a.G * a.q_h, rows, a.q_r * e, last + (int)((a.G - 1) * a.q_h * e)), offQ, nv);
      stG.load(rows_buffer((const T*)a.go + qs.lo * a.go_r + (int64_t)kvh * a.G * a.go_h, rows, a.go_r * e, last + (int)((a.G - 1) * a.go_h * e)), offG, nv);
      if (l < nv) {
        const uint32_t i = a.by_g(l);
        ref = a.lse[(int64_t)(kvh * a.G + (l - (int)i * a.G)) * a.Nq + qs.lo + (int)i] * kLog2e;
        if (ref == -INFINITY) ref = INFINITY;   // a row without keys: no gradient from it or to it
      }
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
    Bits<1> bits;
    if (bq) {
      bits.w[0] = __ballot(ref != INFINITY);
      // (past the last row the one row of a broadcast gradient would be read again)
      if (bits.w[0] != (nv >= 32 ? 0xffffffffull : (1ull << nv) - 1) || a.go_r == 0) { stQ.keep(bits); stG.keep(bits); }
      stQ.store(sQ, TK);
      stG.store(sG, TK);
      if (l < TK) sL[l] = ref;
    }
    if (bk) {
      if (a.mask) {
        bits.w[0] = kbits;
        stK.keep(bits);
        stV.keep(bits);
      }
      stK.store(sK, nk);
      stV.store(sV, nk);
    }
  }
  tile_sync<(P > 1)>();
  const bool q2 = nv > 16, k2 = nk > 16;     // second blocks of 16 rows
  const float c2 = signed_c2(a), sc = signed_scale(a);
  // scores with the queries on the columns: delta and dq
#pragma unroll
  for (int q = 0; q < 2; q += P) {
    if (P == 2) q = w;
    if (P == 1 ? q && nv <= 16 : 16 * q >= nv) break;
    typename TL::Feat Qc[TL::NK], Gc[TL::NK];
#pragma unroll
    for (int kk = 0; kk < TL::NK; ++kk) { Qc[kk] = TL::rows(sQ, q, kk, c, g); Gc[kk] = TL::rows(sG, q, kk, c, g); }
    const float ref = sL[16 * q + c];
    f32x4 S[2] = {zero4(), zero4()}, dS[2] = {zero4(), zero4()};
    float delta = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k ? !k2 : nk == 0) break;
      S[k] = TL::product(sK, k, Qc, c, g, zero4());
      dS[k] = TL::product(sV, k, Gc, c, g, zero4());
      const uint32_t b = kbits >> (16 * k + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        S[k][i] = (b >> i) & 1 ? __builtin_amdgcn_exp2f(__builtin_fmaf(S[k][i], c2, -ref)) : 0.f;
        delta = __builtin_fmaf(S[k][i], dS[k][i], delta);
      }
    }
    delta = col_sum(delta);
    if (g == 0) sD[16 * q + c] = ref == INFINITY ? 0.f : -delta;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) dS[k][i] = S[k][i] * (dS[k][i] - delta);
    const Frag F = chain_frag<T>(dS[0], dS[1]);
    const int v = 16 * q + c;
    const uint32_t i = a.by_g(v);
    T* out = (T*)a.gq + (qs.lo + (int)i) * a.gq_r + (kvh * a.G + (v - (int)i * a.G)) * a.gq_h;
    f32x4 o[TL::NB];
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) {
      Sum<T> d;
      d.begin();
      if (nk) d.add(TL::cols(sK, 0, b, c, g), F);
      d.end();
      o[b] = d.v * sc;
    }
    if (v < nv) store_row<TL::NB>(out, o, g, a.D);
  }
  if (nk == 0) return;
  tile_sync<(P > 1)>();
  // and with the keys on the columns: dk and dv
#pragma unroll
  for (int k = 0; k < 2; k += P) {
    if (P == 2) k = w;
    if (P == 1 ? k && nk <= 16 : 16 * k >= nk) break;
    typename TL::Feat Kc[TL::NK], Vc[TL::NK];
#pragma unroll
    for (int kk = 0; kk < TL::NK; ++kk) { Kc[kk] = TL::rows(sK, k, kk, c, g); Vc[kk] = TL::rows(sV, k, kk, c, g); }
    f32x4 S[2] = {zero4(), zero4()}, dS[2] = {zero4(), zero4()};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (q && !q2) break;
      const f32x4 Lr = load4_f32(sL + 16 * q + 4 * g), nD = load4_f32(sD + 16 * q + 4 * g);
      S[q] = TL::product(sQ, q, Kc, c, g, zero4());
      dS[q] = TL::product(sG, q, Vc, c, g, nD);
#pragma unroll
      for (int i = 0; i < 4; ++i) {        // rows that take no part are zeros, and 0 times an infinity of a key is NaN
        S[q][i] = Lr[i] == INFINITY ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(S[q][i], c2, -Lr[i]));
        dS[q][i] *= S[q][i];
      }
    }
    const Frag FP = chain_frag<T>(S[0], S[1]), FS = chain_frag<T>(dS[0], dS[1]);
    const int key0 = 16 * k + c;
    const bool live = (kbits >> key0) & 1;
    f32x4 ok[TL::NB], ov[TL::NB];
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) {
      Sum<T> dK, dV;
      dK.begin();
      dV.begin();
      dV.add(TL::cols(sG, 0, b, c, g), FP);
      dK.add(TL::cols(sQ, 0, b, c, g), FS);
      dK.end();
      dV.end();
      ok[b] = live ? dK.v * sc : zero4();
      ov[b] = live ? dV.v : zero4();
    }
    if (key0 < nk) {
      store_row<TL::NB>((T*)a.gk + (ks.lo + key0) * a.gk_r + kvh * a.gk_h, ok, g, a.D);
      store_row<TL::NB>((T*)a.gv + (ks.lo + key0) * a.gv_r + kvh * a.gv_h, ov, g, a.D);
    }
  }
}

// Items 0 .. n_q - 1: a tile of 32 virtual rows and a key head: the whole segment where it is small, else its dq (and with
// n_k = 0, where queries and keys are the same rows, the dk and dv of those).  The others: a tile of 32 keys and heads_per
// key heads, their dk and dv where the segment is not small.  P waves an item, W a workgroup.
//
// Waves a SIMD that its registers leave room for: the tiles of long segments would take those of two or three waves, where
// the small segments, which are most, gain by four or five (left to the compiler and as here: bf16, D = 32, 4,000 segments
// of 2 .. 10 rows 32.6 and 23.9 us; D = 16, 1,024 molecules and 8 heads 15.7 and 14.6; fp32, D = 16, 2,000 segments and 8
// heads 58 and 52), although at D = 16 that spills 18 registers in bf16 and 9 in fp32.  The other widths would spill more, or
// have no room for more waves in LDS.
template <typename T, int DP> constexpr int short_occupancy() {
  return Num<T>::planes == 1 ? (DP == 16 ? 5 : DP == 32 ? 3 : 1) : DP == 16 ? 4 : 1;
}
template <typename T, int DP, int P, int W>
__global__ __launch_bounds__(64 * W, (short_occupancy<T, DP>())) void short_kernel(Args a, uint32_t n_q, uint32_t n_k, uint32_t slots_k,
                                                                                   Div by_heads_k, int heads_per) {
  typedef Tile<T, DP> TL;
  static_assert(P == 1 || W == P, "");
  __shared__ __attribute__((aligned(16))) bf16 lds[W / P][4][TL::elems];
  __shared__ __attribute__((aligned(16))) float stat[W][2][TK];
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), x0 = P == 2 ? 16 * w : 0;
  uint32_t i = a.first + xcd_order(blockIdx.x, gridDim.x);
  if (P == 1) i = i * W + w;
  bf16* t = lds[P == 1 ? w : 0][0];
  bf16* t2 = P == 1 ? t : lds[0][2 * w];     // of a wave by itself
  Seg own;
  int r0, e, h0, h1;
  // tiles of 16 where the segment is not small: of 32 rows the registers would cost waves
  if (i < n_q) {
    const uint32_t slot = a.by_heads(i);
    h0 = (int)(i - slot * (uint32_t)a.Hkv);
    h1 = h0 + 1;
    e = find_tile<TK>(a.q_ptr, a.B, a.Nq, a.G, a.guess, slot, r0, own);
    if (r0 < 0) return;
    const Seg ks = other_rows(a.kv_ptr, e, a.B, a.Nk, a.same, own);
    const int nv = (own.hi - own.lo) * a.G;
    if (nv <= TK && ks.hi - ks.lo <= TK && (n_k || (e >= 1 && e <= a.B))) {   // (keys outside every segment: zeros, below)
      small_segment<T, DP, P>(a, h0, own, ks, t, stat[P == 1 ? w : 0][0], stat[P == 1 ? w : 0][1], w);
      return;
    }
    for (int x = x0; x < TK && r0 + x < nv; x += 16 * P) {
      wave_sync();
      dq_tile<T, DP, 1, W, false, 1, Num<T>::planes == 1>(a, Item{slot, h0, 0}, e, r0 + x, own, t2, t2 + TL::elems, 0);
    }
    if (n_k) return;
  } else {
    i -= n_q;
    if (i >= n_k) return;
    const uint32_t slot = by_heads_k(i);
    h0 = (int)(i - slot * (uint32_t)(a.Hkv / heads_per)) * heads_per;
    h1 = h0 + heads_per;
    e = find_tile<TK>(a.kv_ptr, a.B, a.Nk, 1, (float)(a.B + 2) / (float)slots_k, slot, r0, own);
    if (r0 < 0) return;
    const Seg qs = other_rows(a.q_ptr, e, a.B, a.Nq, a.same, own);
    const int nv = (qs.hi - qs.lo) * a.G;
    if (nv >= 1 && nv <= TK && own.hi - own.lo <= TK) return;   // a query's item has it
  }
  for (int h = h0; h < h1; ++h)
    for (int x = x0; x < TK && r0 + x < own.hi - own.lo; x += 16 * P) {
      wave_sync();
      dkv_tile<T, DP, 1, W, false, 1, true>(a, Item{0, h, 0}, e, r0 + x, own, t2, t2 + TL::elems, stat[w][0], stat[w][1], 0);
    }
}

// out[row][head][f] = mul * sum over the splits, 4 features a thread: GR groups of splits a block, whose sums are added in
// order.  The partial rows are `width` values apart and hold one output's DP values, or two's.
template <typename T> struct Out { T* p; int64_t rs, hs; float mul; };
template <typename T, int GR>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* part, int nsplit, int64_t rows, int heads, int D, int DP, int width,
                                                        Out<T> one, Out<T> two) {
  const Out<T> o = blockIdx.y ? two : one;
  const int off = blockIdx.y * DP;
  constexpr int PB = 256 / GR;
  __shared__ f32x4 red[GR][PB];
  const int x = threadIdx.x % PB, k = threadIdx.x / PB;
  const int64_t n = rows * heads, t = (int64_t)blockIdx.x * PB + x;
  const int64_t r = t / (D / 4);
  const int f = 4 * (int)(t - r * (D / 4));
  f32x4 s = zero4();
  if (r < n) {
#pragma unroll 4
    for (int i = k; i < nsplit; i += GR) s += load4_f32(part + (i * n + r) * width + off + f);
  }
  if constexpr (GR > 1) {
    red[k][x] = s;
    __syncthreads();
    if (k) return;
#pragma unroll
    for (int i = 1; i < GR; ++i) s += red[i][x];
  }
  if (r < n) store4(o.p + (r / heads) * o.rs + (r % heads) * o.hs + f, s * o.mul);
}
// dq of the splits whose rows hold sum_j ds_j k_j and sum_j p_j k_j, DP values each, and behind all rows sum_j ds_j: the last
// is what delta lacked, over all splits.  It is added to the row's delta, which dk's kernel reads.
template <typename T, int GR>
__global__ __launch_bounds__(256) void join_dq_kernel(const float* part, int nsplit, int64_t rows, int heads, int D, int DP, Out<T> o,
                                                      float* delta) {
  constexpr int PB = 256 / GR;
  __shared__ f32x4 red[2][GR][PB];
  __shared__ float reds[GR][PB];
  const int x = threadIdx.x % PB, k = threadIdx.x / PB;
  const int64_t n = rows * heads, t = (int64_t)blockIdx.x * PB + x;
  const int64_t r = t / (D / 4);
  const int f = 4 * (int)(t - r * (D / 4));
  const float* offs = part + nsplit * n * (2 * DP);
  f32x4 s = zero4(), pk = zero4();
  float off = 0.f;
  if (r < n) {
#pragma unroll 4
    for (int i = k; i < nsplit; i += GR) {
      const float* p = part + (i * n + r) * (2 * DP) + f;
      s += load4_f32(p);
      pk += load4_f32(p + DP);
      off += offs[i * n + r];
    }
  }
  if constexpr (GR > 1) {
    red[0][k][x] = s;
    red[1][k][x] = pk;
    reds[k][x] = off;
    __syncthreads();
    if (k) return;
#pragma unroll 4
    for (int i = 1; i < GR; ++i) { s += red[0][i][x]; pk += red[1][i][x]; off += reds[i][x]; }
  }
  if (r >= n) return;
  const int64_t row = r / heads, head = r % heads;
  store4(o.p + row * o.rs + head * o.hs + f, (s - pk * off) * o.mul);
  if (f == 0) delta[head * rows + row] += off;
}
template <typename T>
static void sum_parts(const float* part, int nsplit, int64_t rows, int heads, int D, int DP, Out<T> one, Out<T> two, hipStream_t st) {
  const int64_t n = rows * heads * (D / 4);
  const int outs = two.p ? 2 : 1, width = outs * DP;
  // (17 .. 128 parts in 32 groups, 128 bytes of a part at a time: 44.8 us where 8 groups take
  // 8.6, 3 graphs of 1,000 to 1,400 rows, 8 heads on 2)
  if (nsplit <= 16) sum_parts_kernel<T, 1><<<dim3((uint32_t)cdiv(n, 256), outs), 256, 0, st>>>(part, nsplit, rows, heads, D, DP, width, one, two);
  else if (nsplit <= 128) sum_parts_kernel<T, 8><<<dim3((uint32_t)cdiv(n, 32), outs), 256, 0, st>>>(part, nsplit, rows, heads, D, DP, width, one, two);
  else sum_parts_kernel<T, 32><<<dim3((uint32_t)cdiv(n, 8), outs), 256, 0, st>>>(part, nsplit, rows, heads, D, DP, width, one, two);
}

template <typename T>
static void join_dq(const Args& a, int DP, Out<T> o, hipStream_t st) {
  const int64_t n = (int64_t)a.Nq * a.Hq * (a.D / 4);
  if (a.nsplit <= 16) join_dq_kernel<T, 1><<<(uint32_t)cdiv(n, 256), 256, 0, st>>>(a.part, a.nsplit, a.Nq, a.Hq, a.D, DP, o, a.delta);
  else if (a.nsplit <= 128) join_dq_kernel<T, 8><<<(uint32_t)cdiv(n, 32), 256, 0, st>>>(a.part, a.nsplit, a.Nq, a.Hq, a.D, DP, o, a.delta);
  else join_dq_kernel<T, 32><<<(uint32_t)cdiv(n, 8), 256, 0, st>>>(a.part, a.nsplit, a.Nq, a.Hq, a.D, DP, o, a.delta);
}

template <typename T, int DP, int R, int W, bool SH, int KT>
static void go_q(const Args& a, const Plan& p, hipStream_t st) {
  const int64_t n = p.slots * a.Hkv * a.nsplit;
  in_parts(a, SH ? n : cdiv(n, W), [&](const Args& x, uint32_t blocks) {
    dq_kernel<T, DP, R, W, SH, KT, Num<T>::planes == 1><<<blocks, 64 * W, 0, st>>>(x, (uint32_t)n);
  });
}
template <typename T, int DP, int R, int W, bool SH, int KT>
static void go_k(const Args& a, const Plan& p, hipStream_t st) {
  const int64_t n = p.slots * a.Hkv * a.nsplit;
  in_parts(a, SH ? n : cdiv(n, W), [&](const Args& x, uint32_t blocks) {
    dkv_kernel<T, DP, R, W, SH, KT><<<blocks, 64 * W, 0, st>>>(x, (uint32_t)n);
  });
}
// One launch for both axes in short segments: both plans say waves, without splits
template <typename T, int DP>
static bool launch_short(Args a, const Plan& pq, const Plan& pk, hipStream_t st) {
  constexpr bool f32 = Num<T>::planes == 3;
  if constexpr (DP > (f32 ? 32 : 64)) return false;
  else {
    if (pq.form != 0 || pk.form != 0 || pq.nsplit > 1 || pk.nsplit > 1 || !a.Nq || !a.Nk) return false;
    const int64_t sq = ((int64_t)a.Nq * a.G) / TK + a.B + 2, sk = a.Nk / TK + a.B + 2;
    const int per = sk >= 1024 ? a.Hkv : 1;
    const int64_t nq = sq * a.Hkv, nk = a.same && a.G == 1 ? 0 : sk * (a.Hkv / per);
    if (nq + nk > INT32_MAX) return false;
    a.delta = nullptr;
    a.nsplit = 1;
    a.slots = (uint32_t)sq;
    a.guess = (float)(a.B + 2) / (float)sq;
    constexpr int tile = 4 * Tile<T, DP>::elems * 2, W = 4 * tile <= 65536 ? 4 : 2;
    const Div by = Div::of(a.Hkv / per);
    // Two waves a segment in fp32, whose products are six (one and two waves, 10 .. 30 rows a segment, D = 32, 4 heads: 27
    // and 18 us for 512 segments, 165 and 101 for 4,000); not in bf16 (4,000 segments: 46 and 44; D = 64: 78 and 85;
    // D = 16, 1,024 molecules and 8 heads: 15.6 and 19).
    constexpr int P = f32 ? 2 : 1, WS = f32 ? 2 : W;
    in_parts(a, cdiv(nq + nk, WS / P), [&](const Args& x, uint32_t blocks) {
      short_kernel<T, DP, P, WS><<<blocks, 64 * WS, 0, st>>>(x, (uint32_t)nq, (uint32_t)nk, (uint32_t)sk, by, per);
    });
    return true;
  }
}

template <typename T, int DP>
static int launch_t(Args a, const Plan& pq, const Plan& pk, hipStream_t st) {
  constexpr int tile = 2 * Tile<T, DP>::elems * 2 + 256, W = 4 * tile <= 65536 ? 4 : 2 * tile <= 65536 ? 2 : 1;
  if (launch_short<T, DP>(a, pq, pk, st)) return (int)hipGetLastError();
  constexpr bool wide = Num<T>::planes == 3 && DP == 128;
  constexpr int KT = Num<T>::planes == 1 ? (DP < 128 ? 2 : 1) : DP <= 32 ? 2 : 1, KT1 = Num<T>::planes == 1 ? 1 : KT;
  a.nsplit = pq.nsplit;
  a.slots = (uint32_t)pq.slots;
  a.guess = (float)(a.B + 2) / (float)a.slots;
  a.by_slots = Div::of(a.slots);
  if (a.Nq) {
    if constexpr (wide) go_q<T, DP, 1, 4, true, KT>(a, pq, st);
    else if (pq.form == 0) go_q<T, DP, 1, W, false, 1>(a, pq, st);
    else if (pq.form == 1) go_q<T, DP, 1, 4, true, KT1>(a, pq, st);
    else if constexpr (Num<T>::planes == 3 || DP <= 64) go_q<T, DP, 2, 4, true, KT>(a, pq, st);
    if (a.nsplit > 1) {
      const Out<T> gq{(T*)a.gq, a.gq_r, a.gq_h, signed_scale(a)};
      if constexpr (Num<T>::planes == 1) join_dq<T>(a, DP, gq, st);
      else sum_parts<T>(a.part, a.nsplit, a.Nq, a.Hq, a.D, DP, gq, Out<T>{}, st);
    }
  }
  a.nsplit = pk.nsplit;
  a.slots = (uint32_t)pk.slots;
  a.guess = (float)(a.B + 2) / (float)a.slots;
  a.by_slots = Div::of(a.slots);
  if (a.Nk) {
    if constexpr (wide) go_k<T, DP, 1, 4, true, KT>(a, pk, st);
    else if (pk.form == 0) go_k<T, DP, 1, W, false, 1>(a, pk, st);
    else if (pk.form == 1) go_k<T, DP, 1, 4, true, KT1>(a, pk, st);
    else if constexpr (DP <= (Num<T>::planes == 1 ? 64 : 32)) go_k<T, DP, 2, 4, true, KT>(a, pk, st);
    if (a.nsplit > 1)
      sum_parts<T>(a.part, a.nsplit, a.Nk, a.Hkv, a.D, DP, Out<T>{(T*)a.gk, a.gk_r, a.gk_h, signed_scale(a)}, Out<T>{(T*)a.gv, a.gv_r, a.gv_h, 1.0f}, st);
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
