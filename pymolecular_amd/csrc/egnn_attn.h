// Attention over the nodes of ragged segments (gfx950): what the forward and the backward kernels share.
//
// Segments.  Rows of q (k) lie back to back; ptr[b] .. ptr[b + 1] are those of segment b.  Two segments without keys are
// added, the rows before ptr[0] and those from ptr[n_seg] on, so that every row belongs to one.  Offsets are clamped to
// [0, N] wherever they are read, so whatever they hold no access leaves the tensors.
//
// Virtual rows.  The G = Hq / Hkv query heads of a key head run as G rows of the same axis: row vq of a segment is query
// vq / G, head vq % G of the group.  A tile of 16 columns is then full with four queries of four heads, keys and values
// are read once per key head, and the gradients of shared heads are sums over one axis.
//
// Tiles.  Segments are cut into tiles of BQ virtual rows.  Slot b + floor(ptr[b] G / BQ) starts segment b: the next
// segment's slot is never inside the ceil(n G / BQ) slots this one needs, since floor(x + y) + 1 >= floor(x) + ceil(y).
// So a slot finds its segment by a search in ptr and no scan over the segments is needed; at most one slot a segment
// stays empty.
//
// Operands (egnn_device.h): products run with the tile's own axis (queries in the forward and in dq, keys in dk and dv)
// on the MFMA columns and the other axis, 32 at a time, on its rows: S^T = K Q^T gives a lane four rows of one column
// per C-block, so softmax statistics belong to a lane's column and the two C-blocks of 32 rows are the B operand of the
// second product (O^T = V^T P^T) without leaving the registers.  Its A operand is read transposed from LDS.
// fp32 values are held as three bf16 parts in LDS and registers (egnn_split.h).
#pragma once
#include "egnn_device.h"
#include "egnn_internal.h"
#include "egnn_split.h"

namespace egnn {
namespace attn {

constexpr int TK = 32;                       // rows of the other axis in one step
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

struct Args {
  const void *q, *k, *v, *go;
  const void* o;                             // backward: the forward's output
  void *out, *gq, *gk, *gv;
  float* lse;                                // [Hq][Nq], natural logarithm
  float* delta;                              // [Hq][Nq], backward
  int64_t q_r, q_h, k_r, k_h, v_r, v_h, o_r, o_h, go_r, go_h, gq_r, gq_h, gk_r, gk_h, gv_r, gv_h;   // elements
  const int32_t *q_ptr, *kv_ptr;
  const uint8_t* mask;                       // [Nk] or null
  int32_t Nq, Nk, B, Hq, Hkv, G, D;
  float c2;                                  // |scale| log2 e
  float scale;                               // |scale|
  uint32_t flip;                             // sign bit of a negative scale: q enters negated
  int32_t nsplit;
  float* part;                               // split partials
};

// How one axis is cut: slots of 16 waves rows, and the parts the other axis is walked in
struct Plan { int64_t slots; int waves, nsplit; };
inline int padded(int D) { return D <= 16 ? 16 : D <= 32 ? 32 : D <= 64 ? 64 : 128; }
int launch_fwd(const Args& a, bool is_bf16, const Plan& p, hipStream_t st);
int launch_bwd(const Args& a, bool is_bf16, const Plan& pq, const Plan& pk, hipStream_t st);

// ---- operand fragments ----------------------------------------------------------
template <typename T> struct Num;
template <> struct Num<bf16> { static constexpr int planes = 1; typedef bf16x8 Frag; typedef bf16x8 Raw; };
template <> struct Num<float> { static constexpr int planes = 3; typedef split::Chunk3 Frag; typedef f32x8 Raw; };

__device__ __forceinline__ bf16x8 to_frag(const bf16x8& r) { return r; }
__device__ __forceinline__ split::Chunk3 to_frag(const f32x8& r) { return split::split_chunk(r.lo, r.hi); }
template <typename T> __device__ __forceinline__ typename Num<T>::Frag chain_frag(const f32x4& lo, const f32x4& hi);
template <> __device__ __forceinline__ bf16x8 chain_frag<bf16>(const f32x4& lo, const f32x4& hi) { return pack_chunk_bf16(lo, hi); }
template <> __device__ __forceinline__ split::Chunk3 chain_frag<float>(const f32x4& lo, const f32x4& hi) { return split::split_chunk(lo, hi); }

__device__ __forceinline__ bf16x8 negate(const bf16x8& r, uint32_t flip) {
  u32x4 u = __builtin_bit_cast(u32x4, r);
  const uint32_t f = flip | (flip >> 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] ^= f;
  return __builtin_bit_cast(bf16x8, u);
}
__device__ __forceinline__ f32x8 negate(const f32x8& r, uint32_t flip) {
  return f32x8{split::flip_sign(r.lo, flip), split::flip_sign(r.hi, flip)};
}

// sum over NK 32-deep slices of a(kk) b(kk)
template <int NK, typename FA> __device__ __forceinline__ f32x4 product(const bf16x8* b, FA a) {
  f32x4 s = zero4();
#pragma unroll
  for (int kk = 0; kk < NK; ++kk) mma(s, a(kk), b[kk]);
  return s;
}
template <int NK, typename FA> __device__ __forceinline__ f32x4 product(const split::Chunk3* b, FA a) {
  f32x4 hi = zero4(), lo = zero4();
#pragma unroll
  for (int kk = 0; kk < NK; ++kk) split::mma3(hi, lo, a(kk), b[kk]);
  return split::joined(hi, lo);
}
// acc += a b, one slice.  fp32: the slice's sum is made apart and added in fp32, so a long axis is not summed by the
// matrix unit, which rounds to one side
__device__ __forceinline__ void accumulate(f32x4& acc, const bf16x8& a, const bf16x8& b) { mma(acc, a, b); }
__device__ __forceinline__ void accumulate(f32x4& acc, const split::Chunk3& a, const split::Chunk3& b) {
  f32x4 hi = zero4(), lo = zero4();
  split::mma3(hi, lo, a, b);
  acc += split::joined(hi, lo);
}

// ---- a tile of TK rows in LDS -----------------------------------------------------
// [plane][row][KP + 8] bf16, features past D zero.  The pitch is an odd number of 16-byte units: the 16 rows that one
// row read touches start on different banks, and so do the rows of a transposing read.
template <typename T, int DP> struct Tile {
  static constexpr int KP = DP < 32 ? 32 : DP, NK = KP / 32, NB = DP / 16, pitch = KP + 8, plane = TK * pitch;
  static constexpr int elems = Num<T>::planes * plane;

  // A[r][k] = tile[16 blk + r][32 kk + 8g + s]
  static __device__ __forceinline__ typename Num<T>::Frag rows(const bf16* t, int blk, int kk, int c, int g) {
    const bf16* p = t + (16 * blk + c) * pitch + 32 * kk + 8 * g;
    if constexpr (Num<T>::planes == 1) return load_chunk(p);
    else return split::Chunk3{load_chunk(p), load_chunk(p + plane), load_chunk(p + 2 * plane)};
  }
  // A[r][k] = tile[kappa_chain(g, s)][16 blk + r]
  static __device__ __forceinline__ bf16x8 tr(const bf16* p) {
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)p);
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(p + 16 * pitch));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ typename Num<T>::Frag cols(const bf16* t, int blk, int c, int g) {
    const bf16* p = t + (4 * g + (c >> 2)) * pitch + 16 * blk + 4 * (c & 3);
    if constexpr (Num<T>::planes == 1) return tr(p);
    else return split::Chunk3{tr(p), tr(p + plane), tr(p + 2 * plane)};
  }
};

// The rows of a tile on their way to LDS: NT threads, 8 values each and step
template <typename T, int DP, int NT> struct Stage {
  typedef Tile<T, DP> TL;
  static constexpr int CH = TL::KP / 8, N = TK * CH, PER = (N + NT - 1) / NT;
  typename Num<T>::Raw r[PER];
  // row(i): address of row i of the tile, or null for a row of zeros
  template <typename F> __device__ __forceinline__ void load(F row, int D) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int t = p * NT + (int)threadIdx.x, i = t / CH, f = 8 * (t % CH);
      r[p] = zero_chunk<T>();
      if (t < N && f < D) {
        const T* a = row(i);
        if (a) r[p] = load_chunk(a + f);
      }
    }
  }
  __device__ __forceinline__ void flip(uint32_t f) {
#pragma unroll
    for (int p = 0; p < PER; ++p) r[p] = negate(r[p], f);
  }
  __device__ __forceinline__ void store(bf16* t) const {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int x = p * NT + (int)threadIdx.x;
      if (x < N) {
        bf16* d = t + (x / CH) * TL::pitch + 8 * (x % CH);
        const auto v = to_frag(r[p]);
        if constexpr (Num<T>::planes == 1) store_chunk(d, v);
        else { store_chunk(d, v.p0); store_chunk(d + TL::plane, v.p1); store_chunk(d + 2 * TL::plane, v.p2); }
      }
    }
  }
};

// ---- work items -------------------------------------------------------------------
struct Seg { int lo, hi; };                  // rows of one axis
__device__ __forceinline__ int edge_of(const int32_t* ptr, int e, int B, int N) {   // start of extended segment e
  if (e <= 0) return 0;
  if (e > B + 1) return N;
  const int p = ptr[e - 1];
  return p < 0 ? 0 : (p > N ? N : p);
}
// The extended segment of a slot and the slot's first virtual row in it (-1: an empty slot).  Every lane probes one
// segment and step, so 64 segments take one round and 4,096 two.
__device__ __forceinline__ int find_tile(const int32_t* ptr, int B, int N, int G, int BQ, int64_t slot, int& vq0, Seg& s) {
  int lo = 0, hi = B + 2;
  const int lane = lane_id();
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int64_t e = lo + (int64_t)lane * step;
    const bool le = e < hi && (int64_t)edge_of(ptr, (int)e, B, N) * G / BQ + e <= slot;
    const int n = __builtin_popcountll(__ballot(le));
    lo += (n > 0 ? n - 1 : 0) * step;
    hi = hi < lo + step ? hi : lo + step;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  s.lo = edge_of(ptr, lo, B, N);
  s.hi = edge_of(ptr, lo + 1, B, N);
  if (s.hi < s.lo) s.hi = s.lo;
  const int64_t v = (slot - ((int64_t)s.lo * G / BQ + lo)) * BQ;
  vq0 = v >= 0 && v < (int64_t)(s.hi - s.lo) * G ? (int)v : -1;
  return lo;
}
// Rows of the other axis of extended segment e
__device__ __forceinline__ Seg other_rows(const int32_t* ptr, int e, int B, int N) {
  if (e < 1 || e > B) return Seg{0, 0};
  Seg s{edge_of(ptr, e, B, N), edge_of(ptr, e + 1, B, N)};
  if (s.hi < s.lo) s.hi = s.lo;
  return s;
}
// part s of n of [lo, hi), in whole steps
__device__ __forceinline__ void split_range(int64_t lo, int64_t hi, int n, int s, int64_t& a, int64_t& b) {
  const int64_t per = ((hi - lo + n - 1) / n + TK - 1) / TK * TK;
  a = lo + s * per < hi ? lo + s * per : hi;
  b = a + per < hi ? a + per : hi;
}
// Consecutive items on one XCD (workgroups go to the 8 XCDs in turn, each has an L2 of its own): neighbouring heads of a
// tile share the lines of its rows
__device__ __forceinline__ int64_t item_of(int64_t bid, int64_t n) {
  const int64_t per = n / 8, rest = n % 8, x = bid % 8, y = bid / 8;
  return x * per + (x < rest ? x : rest) + y;
}

// max and sum over the four lanes of a column
__device__ __forceinline__ float col_max(float v) { v = fmaxf(v, shfl_xor(v, 16)); return fmaxf(v, shfl_xor(v, 32)); }
__device__ __forceinline__ float col_sum(float v) { v += shfl_xor(v, 16); return v + shfl_xor(v, 32); }

// four features of one row
__device__ __forceinline__ void store4(float* p, const f32x4& v) { *reinterpret_cast<f32x4*>(p) = v; }
__device__ __forceinline__ void store4(bf16* p, const f32x4& v) {
  bf16x4 r;
  r[0] = (bf16)v[0]; r[1] = (bf16)v[1]; r[2] = (bf16)v[2]; r[3] = (bf16)v[3];
  *reinterpret_cast<bf16x4*>(p) = r;
}
__device__ __forceinline__ float dot8(const bf16x8& a, const bf16x8& b) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = __builtin_fmaf((float)a[i], (float)b[i], s);
  return s;
}
__device__ __forceinline__ float dot8(const f32x8& a, const f32x8& b) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) s = __builtin_fmaf(a.hi[i], b.hi[i], __builtin_fmaf(a.lo[i], b.lo[i], s));
  return s;
}

// 32 rows j0 .. of the key axis that exist and are not masked, as bits; the same in every wave
__device__ __forceinline__ uint32_t key_bits(const uint8_t* mask, int j0, int hi) {
  const int j = j0 + (lane_id() & 31);
  bool ok = j < hi;
  if (ok && mask) ok = mask[j] != 0;
  return (uint32_t)__ballot(ok);
}

}  // namespace attn
}  // namespace egnn
