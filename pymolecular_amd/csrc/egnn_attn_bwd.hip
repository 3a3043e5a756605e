// Segment attention, backward.  With p = e^{s - lse} recomputed from the forward's statistics,
//   delta_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i.
// dq's kernel owns tiles of queries and walks the keys, dk and dv's owns tiles of keys and walks the queries (of all
// heads of the group); each sum is made by one owner in a fixed order, so there are no atomics.
#include "egnn_attn.h"

namespace egnn {
namespace attn {

template <typename T, int DP, int W>
__global__ __launch_bounds__(64 * W) void dq_kernel(Args a, int64_t n_items) {
  typedef Tile<T, DP> TL;
  typedef typename Num<T>::Frag Frag;
  constexpr int NT = 64 * W, BQ = 16 * W;
  __shared__ __attribute__((aligned(16))) bf16 sK[TL::elems], sV[TL::elems];
  int64_t item = item_of(blockIdx.x, n_items);
  const int kvh = (int)(item % a.Hkv);
  item /= a.Hkv;
  const int sp = (int)(item % a.nsplit);
  const int64_t slot = item / a.nsplit;
  const int l = lane_id(), c = l & 15, g = l >> 4, w = threadIdx.x >> 6;
  int vq0;
  Seg qs;
  const int e = find_tile(a.q_ptr, a.B, a.Nq, a.G, BQ, slot, vq0, qs);
  if (vq0 < 0) return;
  const Seg ks = other_rows(a.kv_ptr, e, a.B, a.Nk);
  const int nv = (qs.hi - qs.lo) * a.G, vq = vq0 + 16 * w + c;
  const bool live = vq < nv;
  const int row = qs.lo + (live ? vq / a.G : 0), head = kvh * a.G + (live ? vq % a.G : 0);
  const T *qp = (const T*)a.q + row * a.q_r + head * a.q_h, *gp = (const T*)a.go + row * a.go_r + head * a.go_h,
          *op = (const T*)a.o + row * a.o_r + head * a.o_h;
  Frag Q[TL::NK], GO[TL::NK];
  float delta = 0.f;
#pragma unroll
  for (int kk = 0; kk < TL::NK; ++kk) {
    const int f = 32 * kk + 8 * g;
    typename Num<T>::Raw r = zero_chunk<T>(), go = r;
    if (live && f < a.D) {
      r = negate(load_chunk(qp + f), a.flip);
      go = load_chunk(gp + f);
      delta += dot8(go, load_chunk(op + f));
    }
    Q[kk] = to_frag(r);
    GO[kk] = to_frag(go);
  }
  delta = col_sum(delta);
  const float lse = live ? a.lse[(int64_t)head * a.Nq + row] * kLog2e : INFINITY;
  const bool none = lse == -INFINITY;   // a row without keys: no gradient from it or to it
  const float ref = none ? INFINITY : lse;
  if (sp == 0 && live && g == 0) a.delta[(int64_t)head * a.Nq + row] = none ? 0.f : delta;
  int64_t j0, j1;
  split_range(ks.lo, ks.hi, a.nsplit, sp, j0, j1);
  const T *kb = (const T*)a.k + kvh * a.k_h, *vb = (const T*)a.v + kvh * a.v_h;
  f32x4 dQ[TL::NB];
#pragma unroll
  for (int b = 0; b < TL::NB; ++b) dQ[b] = zero4();

  for (int64_t j = j0; j < j1; j += TK) {
    const uint32_t bits = key_bits(a.mask, (int)j, (int)j1);
    Stage<T, DP, NT> st;
    st.load([&](int i) { return (bits >> i) & 1 ? kb + (j + i) * a.k_r : nullptr; }, a.D);
    __syncthreads();
    st.store(sK);
    st.load([&](int i) { return (bits >> i) & 1 ? vb + (j + i) * a.v_r : nullptr; }, a.D);
    st.store(sV);
    __syncthreads();
    f32x4 dS[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4 S = product<TL::NK>(Q, [&](int kk) { return TL::rows(sK, h, kk, c, g); });
      const f32x4 dP = product<TL::NK>(GO, [&](int kk) { return TL::rows(sV, h, kk, c, g); });
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], a.c2, -ref));
        const float d = p * (dP[i] - delta);
        dS[h][i] = (bits >> (16 * h + 4 * g + i)) & 1 ? d : 0.f;
      }
    }
    const Frag F = chain_frag<T>(dS[0], dS[1]);
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) accumulate(dQ[b], TL::cols(sK, b, c, g), F);
  }
  if (!live) return;
  if (a.nsplit > 1) {
    float* p = a.part + ((int64_t)sp * a.Nq * a.Hq + (int64_t)row * a.Hq + head) * DP;
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) store4(p + 16 * b + 4 * g, none ? zero4() : dQ[b]);
    return;
  }
  const float sc = a.flip ? -a.scale : a.scale;
  T* out = (T*)a.gq + row * a.gq_r + head * a.gq_h;
#pragma unroll
  for (int b = 0; b < TL::NB; ++b)
    if (16 * b + 4 * g < a.D) store4(out + 16 * b + 4 * g, none ? zero4() : dQ[b] * sc);
}

template <typename T, int DP, int W>
__global__ __launch_bounds__(64 * W) void dkv_kernel(Args a, int64_t n_items) {
  typedef Tile<T, DP> TL;
  typedef typename Num<T>::Frag Frag;
  constexpr int NT = 64 * W, BK = 16 * W;
  __shared__ __attribute__((aligned(16))) bf16 sQ[TL::elems], sG[TL::elems];
  __shared__ float sL[TK], sD[TK];
  int64_t item = item_of(blockIdx.x, n_items);
  const int kvh = (int)(item % a.Hkv);
  item /= a.Hkv;
  const int sp = (int)(item % a.nsplit);
  const int64_t slot = item / a.nsplit;
  const int l = lane_id(), c = l & 15, g = l >> 4, w = threadIdx.x >> 6;
  int k0;
  Seg ks;
  const int e = find_tile(a.kv_ptr, a.B, a.Nk, 1, BK, slot, k0, ks);
  if (k0 < 0) return;
  const Seg qs = other_rows(a.q_ptr, e, a.B, a.Nq);
  const int key = ks.lo + k0 + 16 * w + c;
  const bool in = key < ks.hi, live = in && (!a.mask || a.mask[key] != 0);
  Frag K[TL::NK], V[TL::NK];
#pragma unroll
  for (int kk = 0; kk < TL::NK; ++kk) {
    const int f = 32 * kk + 8 * g;
    typename Num<T>::Raw k = zero_chunk<T>(), v = k;
    if (live && f < a.D) {
      k = load_chunk((const T*)a.k + key * a.k_r + kvh * a.k_h + f);
      v = load_chunk((const T*)a.v + key * a.v_r + kvh * a.v_h + f);
    }
    K[kk] = to_frag(k);
    V[kk] = to_frag(v);
  }
  int64_t v0, v1;
  split_range(0, (int64_t)(qs.hi - qs.lo) * a.G, a.nsplit, sp, v0, v1);
  f32x4 dK[TL::NB], dV[TL::NB];
#pragma unroll
  for (int b = 0; b < TL::NB; ++b) { dK[b] = zero4(); dV[b] = zero4(); }

  for (int64_t j = v0; j < v1; j += TK) {
    // statistics of the step's rows; a row without keys (or past the end) takes no part: its p is e^-inf
    const int i = l & 31, vq = (int)j + i;
    float lse = INFINITY, delta = 0.f;
    if (vq < v1) {
      const int64_t r = (int64_t)(kvh * a.G + vq % a.G) * a.Nq + qs.lo + vq / a.G;
      lse = a.lse[r] * kLog2e;
      delta = a.delta[r];
      if (lse == -INFINITY) lse = INFINITY;
    }
    const uint32_t bits = (uint32_t)__ballot(lse != INFINITY);
    auto at = [&](const void* p, int64_t rs, int64_t hs, int i) -> const T* {
      const int v = (int)j + i;
      return (bits >> i) & 1 ? (const T*)p + (qs.lo + v / a.G) * rs + (kvh * a.G + v % a.G) * hs : nullptr;
    };
    Stage<T, DP, NT> st;
    st.load([&](int i) { return at(a.q, a.q_r, a.q_h, i); }, a.D);
    st.flip(a.flip);
    __syncthreads();
    st.store(sQ);
    st.load([&](int i) { return at(a.go, a.go_r, a.go_h, i); }, a.D);
    st.store(sG);
    if (w == 0 && l < TK) { sL[l] = lse; sD[l] = delta; }
    __syncthreads();
    f32x4 P[2], dS[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 S = product<TL::NK>(K, [&](int kk) { return TL::rows(sQ, h, kk, c, g); });
      const f32x4 dP = product<TL::NK>(V, [&](int kk) { return TL::rows(sG, h, kk, c, g); });
      const f32x4 L = load4_f32(sL + 16 * h + 4 * g), D = load4_f32(sD + 16 * h + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        P[h][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], a.c2, -L[i]));
        dS[h][i] = P[h][i] * (dP[i] - D[i]);
      }
    }
    const Frag FP = chain_frag<T>(P[0], P[1]), FS = chain_frag<T>(dS[0], dS[1]);
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) {
      accumulate(dV[b], TL::cols(sG, b, c, g), FP);
      accumulate(dK[b], TL::cols(sQ, b, c, g), FS);
    }
  }
  if (!in) return;
  if (a.nsplit > 1) {
    float* p = a.part + ((int64_t)sp * a.Nk * a.Hkv + (int64_t)key * a.Hkv + kvh) * (2 * DP);
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) {
      store4(p + 16 * b + 4 * g, live ? dK[b] : zero4());
      store4(p + DP + 16 * b + 4 * g, live ? dV[b] : zero4());
    }
    return;
  }
  // q entered with the scale's sign
  T *gk = (T*)a.gk + key * a.gk_r + kvh * a.gk_h, *gv = (T*)a.gv + key * a.gv_r + kvh * a.gv_h;
#pragma unroll
  for (int b = 0; b < TL::NB; ++b)
    if (16 * b + 4 * g < a.D) {
      store4(gk + 16 * b + 4 * g, live ? dK[b] * a.scale : zero4());
      store4(gv + 16 * b + 4 * g, live ? dV[b] : zero4());
    }
}

// out[row][head][f] = mul * sum over the splits, in order; width fp32 values a row, at offset off
template <typename T>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* part, int nsplit, int64_t rows, int heads, int D, int width, int off,
                                                        float mul, T* out, int64_t rs, int64_t hs) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int f = (int)(t % D);
  const int64_t r = t / D;
  if (r >= rows * heads) return;
  float s = 0.f;
  for (int x = 0; x < nsplit; ++x) s += part[((int64_t)x * rows * heads + r) * width + off + f];
  out[(r / heads) * rs + (r % heads) * hs + f] = from_f32<T>(s * mul);
}

template <typename T, int DP>
static int launch_t(Args a, const Plan& pq, const Plan& pk, hipStream_t st) {
  auto blocks = [&](int64_t n) { return (uint32_t)((n * a.D + 255) / 256); };
  a.nsplit = pq.nsplit;
  if (a.Nq) {
    const int64_t n = pq.slots * a.Hkv * a.nsplit;
    if (pq.waves == 1) dq_kernel<T, DP, 1><<<(uint32_t)n, 64, 0, st>>>(a, n);
    else dq_kernel<T, DP, 4><<<(uint32_t)n, 256, 0, st>>>(a, n);
    if (a.nsplit > 1)
      sum_parts_kernel<T><<<blocks((int64_t)a.Nq * a.Hq), 256, 0, st>>>(a.part, a.nsplit, a.Nq, a.Hq, a.D, DP, 0,
                                                                        a.flip ? -a.scale : a.scale, (T*)a.gq, a.gq_r, a.gq_h);
  }
  a.nsplit = pk.nsplit;
  if (a.Nk) {
    const int64_t n = pk.slots * a.Hkv * a.nsplit;
    if (pk.waves == 1) dkv_kernel<T, DP, 1><<<(uint32_t)n, 64, 0, st>>>(a, n);
    else dkv_kernel<T, DP, 4><<<(uint32_t)n, 256, 0, st>>>(a, n);
    if (a.nsplit > 1) {
      const uint32_t nb = blocks((int64_t)a.Nk * a.Hkv);
      sum_parts_kernel<T><<<nb, 256, 0, st>>>(a.part, a.nsplit, a.Nk, a.Hkv, a.D, 2 * DP, 0, a.scale, (T*)a.gk, a.gk_r, a.gk_h);
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
