// Segment attention, forward: o_i = sum_j softmax_j(scale q_i k_j) v_j over the keys of i's segment.
#include "egnn_attn.h"

namespace egnn {
namespace attn {

// Workspace of a split call: per split and virtual output row [D padded to DP] sums, then (m, l)
__device__ __forceinline__ float* part_row(const Args& a, int dp, int s, int64_t r) {
  return a.part + ((int64_t)s * a.Nq * a.Hq + r) * (dp + 2);
}

template <typename T, int DP, int W>
__global__ __launch_bounds__(64 * W) void fwd_kernel(Args a, int64_t n_items) {
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
  // the lane's column of Q^T
  Frag Q[TL::NK];
  const T* qp = (const T*)a.q + row * a.q_r + head * a.q_h;
#pragma unroll
  for (int kk = 0; kk < TL::NK; ++kk) {
    const int f = 32 * kk + 8 * g;
    typename Num<T>::Raw r = zero_chunk<T>();
    if (live && f < a.D) r = negate(load_chunk(qp + f), a.flip);
    Q[kk] = to_frag(r);
  }
  int64_t j0, j1;
  split_range(ks.lo, ks.hi, a.nsplit, sp, j0, j1);
  const T *kb = (const T*)a.k + kvh * a.k_h, *vb = (const T*)a.v + kvh * a.v_h;
  f32x4 O[TL::NB];
#pragma unroll
  for (int b = 0; b < TL::NB; ++b) O[b] = zero4();
  float m = -INFINITY, sum = 0.f;

  for (int64_t j = j0; j < j1; j += TK) {
    const uint32_t bits = key_bits(a.mask, (int)j, (int)j1);
    Stage<T, DP, NT> st;
    st.load([&](int i) { return (bits >> i) & 1 ? kb + (j + i) * a.k_r : nullptr; }, a.D);
    __syncthreads();   // the step before has read the tile
    st.store(sK);
    st.load([&](int i) { return (bits >> i) & 1 ? vb + (j + i) * a.v_r : nullptr; }, a.D);
    st.store(sV);
    __syncthreads();
    f32x4 S[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      S[h] = product<TL::NK>(Q, [&](int kk) { return TL::rows(sK, h, kk, c, g); });
      if (bits != 0xffffffffu) {
#pragma unroll
        for (int i = 0; i < 4; ++i) S[h][i] = (bits >> (16 * h + 4 * g + i)) & 1 ? S[h][i] : -INFINITY;
      }
    }
    float mx = fmaxf(fmaxf(fmaxf(S[0][0], S[0][1]), fmaxf(S[0][2], S[0][3])), fmaxf(fmaxf(S[1][0], S[1][1]), fmaxf(S[1][2], S[1][3])));
    const float mn = fmaxf(m, col_max(mx) * a.c2);
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = mn;
    float ps = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        S[h][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[h][i], a.c2, -ref));
        ps += S[h][i];
      }
    sum = __builtin_fmaf(sum, alpha, ps);
    const Frag P = chain_frag<T>(S[0], S[1]);
#pragma unroll
    for (int b = 0; b < TL::NB; ++b) {
      O[b] *= alpha;
      accumulate(O[b], TL::cols(sV, b, c, g), P);
    }
  }
  sum = col_sum(sum);
  if (!live) return;
  if (a.nsplit > 1) {
    float* p = part_row(a, DP, sp, (int64_t)row * a.Hq + head);
#pragma unroll
    for (int b = 0; b < TL::NB; ++b)
      if (16 * b + 4 * g < a.D) {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[16 * b + 4 * g + i] = O[b][i];
      }
    if (g == 0) { p[DP] = m; p[DP + 1] = sum; }
    return;
  }
  // no key left: the sum is 0 (a NaN is not), the output 0
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  T* op = (T*)a.out + row * a.o_r + head * a.o_h;
#pragma unroll
  for (int b = 0; b < TL::NB; ++b)
    if (16 * b + 4 * g < a.D) store4(op + 16 * b + 4 * g, O[b] * inv);
  if (a.lse && g == 0) a.lse[(int64_t)head * a.Nq + row] = (m + __builtin_amdgcn_logf(sum)) * kLn2;
}

// Joins the splits of one row and head: one wave each, in split order
template <typename T, int DP>
__global__ __launch_bounds__(64) void fwd_join_kernel(Args a) {
  const int64_t r = blockIdx.x;
  const int head = (int)(r % a.Hq), l = lane_id();
  const int64_t row = r / a.Hq;
  float m = -INFINITY;
  for (int s = l; s < a.nsplit; s += 64) m = fmaxf(m, part_row(a, DP, s, r)[DP]);
  for (int x = 32; x; x >>= 1) m = fmaxf(m, shfl_xor(m, x));
  const float ref = m == -INFINITY ? 0.f : m;
  float sum = 0.f, o0 = 0.f, o1 = 0.f;
  for (int s = 0; s < a.nsplit; ++s) {
    const float* p = part_row(a, DP, s, r);
    const float f = __builtin_amdgcn_exp2f(p[DP] - ref);
    sum = __builtin_fmaf(p[DP + 1], f, sum);
    if (l < a.D) o0 = __builtin_fmaf(p[l], f, o0);
    if (l + 64 < a.D) o1 = __builtin_fmaf(p[l + 64], f, o1);
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  T* op = (T*)a.out + row * a.o_r + head * a.o_h;
  if (l < a.D) op[l] = from_f32<T>(o0 * inv);
  if (l + 64 < a.D) op[l + 64] = from_f32<T>(o1 * inv);
  if (a.lse && l == 0) a.lse[(int64_t)head * a.Nq + row] = (m + __builtin_amdgcn_logf(sum)) * kLn2;
}

template <typename T, int DP>
static int launch_t(const Args& a, const Plan& p, hipStream_t st) {
  const int64_t n = p.slots * a.Hkv * a.nsplit;
  if (p.waves == 1) fwd_kernel<T, DP, 1><<<(uint32_t)n, 64, 0, st>>>(a, n);
  else fwd_kernel<T, DP, 4><<<(uint32_t)n, 256, 0, st>>>(a, n);
  if (a.nsplit > 1) fwd_join_kernel<T, DP><<<(uint32_t)((int64_t)a.Nq * a.Hq), 64, 0, st>>>(a);
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
