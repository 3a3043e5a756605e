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
#include <type_traits>

namespace egnn {
namespace attn {

constexpr int TK = 32;                       // rows of the other axis that one product contracts
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

// n / d by a multiplication, for n < 2^31 (m = 0: d is 1)
struct Div {
  uint32_t m, s;
  __host__ static Div of(uint32_t d) {
    if (d <= 1) return Div{0, 0};
    uint32_t s = 0;
    while ((1u << s) < d) ++s;             // 2^(s-1) < d <= 2^s
    return Div{(uint32_t)((((uint64_t)1 << (31 + s)) + d - 1) / d), s - 1};
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return m ? __umulhi(n, m) >> s : n; }
};

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
  uint32_t slots;
  float guess;                               // segments per slot
  bool same;                                 // q_ptr is kv_ptr and there are as many queries as keys
  Div by_g, by_heads, by_slots;              // divisions by G, Hkv and slots
  float c2;                                  // |scale| log2 e
  float scale;                               // |scale|
  uint32_t flip;                             // sign bit of a negative scale: q enters negated
  int32_t nsplit;
  uint32_t first;                            // workgroups of the call before this launch's
  float* part;                               // split partials
};

// A launch may have fewer than 2^32 threads, a call more workgroups than that leaves room for (2^24 of 256 threads: a
// batch of 8 million graphs with 8 key heads): at most kMaxGrid at a time, go(args, workgroups) of each part.
constexpr uint32_t kMaxGrid = 1u << 20;
template <typename Go> void in_parts(Args a, int64_t blocks, Go go) {
  for (int64_t n = 0; n < blocks; n += kMaxGrid) {
    a.first = (uint32_t)n;
    go(a, (uint32_t)(blocks - n < kMaxGrid ? blocks - n : kMaxGrid));
  }
}

constexpr int kShortMean = 28;               // rows a segment up to which a wave takes a tile

// How one axis is cut into tiles; the other axis is walked in nsplit parts, part s taking every nsplit-th step from s on
struct Plan {
  int64_t slots;
  int form;                                  // 0: a wave a tile of 16 rows; 1, 2: a workgroup of 4 waves, 64 or 128 rows
  int nsplit;
  int rows() const { return form == 0 ? 16 : 64 * form; }
};
inline int padded(int D) { return D <= 16 ? 16 : D <= 32 ? 32 : D <= 64 ? 64 : 128; }
int launch_fwd(const Args& a, bool is_bf16, const Plan& p, hipStream_t st);
int launch_bwd(const Args& a, bool is_bf16, const Plan& pq, const Plan& pk, hipStream_t st);

// ---- operand fragments ----------------------------------------------------------
// Frag: 8 values a lane, a 32-deep slice of an operand.  Half: 4 values, a 16-deep slice (head widths up to 16).
// Raw: 8 values as they lie in memory.
typedef short s16x4 __attribute__((ext_vector_type(4)));
struct Half3 { bf16x4 p0, p1, p2; };
template <typename T> struct Num;
template <> struct Num<bf16> { static constexpr int planes = 1; typedef bf16x8 Frag; typedef bf16x4 Half; typedef bf16x8 Raw; };
template <> struct Num<float> { static constexpr int planes = 3; typedef split::Chunk3 Frag; typedef Half3 Half; typedef f32x8 Raw; };

__device__ __forceinline__ void mma16(f32x4& acc, const bf16x4& a, const bf16x4& b) {   // A[r][k], B[k][n]: k = 4g + s
  acc = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), acc, 0, 0, 0);
}

__device__ __forceinline__ bf16x8 to_frag(const bf16x8& r) { return r; }
__device__ __forceinline__ split::Chunk3 to_frag(const f32x8& r) { return split::split_chunk(r.lo, r.hi); }
template <typename T> __device__ __forceinline__ typename Num<T>::Frag chain_frag(const f32x4& lo, const f32x4& hi);
template <> __device__ __forceinline__ bf16x8 chain_frag<bf16>(const f32x4& lo, const f32x4& hi) { return pack_chunk_bf16(lo, hi); }
template <> __device__ __forceinline__ split::Chunk3 chain_frag<float>(const f32x4& lo, const f32x4& hi) { return split::split_chunk(lo, hi); }

// the bits of chain_frag's values whose row's bit is set: rows 0 .. 3 and 16 .. 19
__device__ __forceinline__ u32x4 chain_rows(uint32_t b) {
  u32x4 m;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = b >> (16 * (i / 2) + 2 * (i & 1));
    m[i] = ((x & 1) ? 0xffffu : 0u) | ((x & 2) ? 0xffff0000u : 0u);
  }
  return m;
}
__device__ __forceinline__ bf16x8 masked(const bf16x8& r, const u32x4& m) {
  return __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, r) & m);
}
__device__ __forceinline__ split::Chunk3 masked(const split::Chunk3& r, const u32x4& m) {
  return split::Chunk3{masked(r.p0, m), masked(r.p1, m), masked(r.p2, m)};
}

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

__device__ __forceinline__ void product1(f32x4& hi, f32x4&, const bf16x8& a, const bf16x8& b) { mma(hi, a, b); }
__device__ __forceinline__ void product1(f32x4& hi, f32x4&, const bf16x4& a, const bf16x4& b) { mma16(hi, a, b); }
__device__ __forceinline__ void product1(f32x4& hi, f32x4& lo, const split::Chunk3& a, const split::Chunk3& b) { split::mma3(hi, lo, a, b); }
__device__ __forceinline__ void product1(f32x4& hi, f32x4& lo, const Half3& a, const Half3& b) {
  mma16(lo, a.p2, b.p0);
  mma16(hi, a.p0, b.p0);
  mma16(lo, a.p0, b.p2);
  mma16(lo, a.p1, b.p1);
  mma16(lo, a.p1, b.p0);
  mma16(lo, a.p0, b.p1);
}
template <typename T> __device__ __forceinline__ f32x4 result(const f32x4& hi, const f32x4& lo);
template <> __device__ __forceinline__ f32x4 result<bf16>(const f32x4& hi, const f32x4&) { return hi; }
template <> __device__ __forceinline__ f32x4 result<float>(const f32x4& hi, const f32x4& lo) { return split::joined(hi, lo); }
// A sum over the steps of an axis.  fp32: the matrix unit sums the steps between begin() and end(), whose result is added
// in fp32, so that a long axis is not summed by the matrix unit, which rounds to one side.  (Two steps at a time: 162 us
// against 184 one at a time, 37 chains of 301, forward and backward.)
template <typename T> struct Sum;
template <> struct Sum<bf16> {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void begin() {}
  __device__ __forceinline__ void add(const bf16x8& a, const bf16x8& b) { mma(v, a, b); }
  __device__ __forceinline__ void one(const bf16x8& a, const bf16x8& b) { mma(v, a, b); }
  __device__ __forceinline__ void scale(float x, bool) { v *= x; }
  __device__ __forceinline__ void end() {}
};
template <> struct Sum<float> {
  f32x4 v = {0.f, 0.f, 0.f, 0.f}, hi, lo;
  __device__ __forceinline__ void begin() { hi = zero4(); lo = zero4(); }
  __device__ __forceinline__ void add(const split::Chunk3& a, const split::Chunk3& b) { split::mma3(hi, lo, a, b); }
  __device__ __forceinline__ void one(const split::Chunk3& a, const split::Chunk3& b) { begin(); add(a, b); end(); }   // one step
  __device__ __forceinline__ void scale(float x, bool added) {                    // added: since begin()
    v *= x;
    if (added) { hi *= x; lo *= x; }
  }
  __device__ __forceinline__ void end() { v += split::joined(hi, lo); }
};

// ---- buffer loads -------------------------------------------------------------------
// Rows 0 .. n - 1 of a tensor part (n >= 1), the last one `last` bytes wide, as a range-checked buffer: rows past them
// read as zeros, and so do features past the head's width, which get the offset kOob.  (64 rows of at most 2^24 bytes
// and a group's heads of at most 2^29 stay below 2^31.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_buffer(const void* base, int n, int64_t row_bytes, int last) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)((n - 1) * row_bytes) + last, kBufFlags);
}
__device__ __forceinline__ bf16x8 load8(const bf16*, __amdgpu_buffer_rsrc_t b, uint32_t off) {
  return __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(b, (int)off, 0, 0));
}
__device__ __forceinline__ f32x8 load8(const float*, __amdgpu_buffer_rsrc_t b, uint32_t off) {
  f32x8 r;
  r.lo = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(b, (int)off, 0, 0));
  r.hi = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(b, (int)off, 16, 0));
  return r;
}

// ---- a tile of rows in LDS ------------------------------------------------------------
// [plane][row][DP + 8] bf16, features past D zero.  The pitch is an odd number of 16-byte units: the 16 rows that one
// row read touches start on different banks, and so do the rows of a transposing read.  KT: steps of TK rows.
template <typename T, int DP, int KT = 1> struct Tile {
  static constexpr bool half = DP == 16;
  static constexpr int NK = half ? 1 : DP / 32, NB = DP / 16, pitch = DP + 8, plane = KT * TK * pitch;
  static constexpr int elems = Num<T>::planes * plane;
  typedef typename std::conditional<half, typename Num<T>::Half, typename Num<T>::Frag>::type Feat;   // over features

  // A[r][k] = tile[16 blk + r][features of slice kk]
  static __device__ __forceinline__ Feat rows(const bf16* t, int blk, int kk, int c, int g) {
    typedef typename std::conditional<half, bf16x4, bf16x8>::type V;
    const bf16* p = t + (16 * blk + c) * pitch + (half ? 4 * g : 32 * kk + 8 * g);
    auto at = [](const bf16* q) { return *reinterpret_cast<const V*>(q); };
    if constexpr (Num<T>::planes == 1) return at(p);
    else return Feat{at(p), at(p + plane), at(p + 2 * plane)};
  }
  // A[r][k] = tile[32 step + kappa_chain(g, s)][16 blk + r]
  static __device__ __forceinline__ bf16x8 tr(const bf16* p) {
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)p);
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(p + 16 * pitch));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ typename Num<T>::Frag cols(const bf16* t, int step, int blk, int c, int g) {
    const bf16* p = t + (TK * step + 4 * g + (c >> 2)) * pitch + 16 * blk + 4 * (c & 3);
    if constexpr (Num<T>::planes == 1) return tr(p);
    else return split::Chunk3{tr(p), tr(p + plane), tr(p + 2 * plane)};
  }
  // the lane's B[k][n] of column n: features of one row of a tensor, from p (null: zeros), negated by flip
  static __device__ __forceinline__ Feat column(const T* p, int kk, int g, int D, uint32_t flip) {
    const int f = half ? 4 * g : 32 * kk + 8 * g;
    if constexpr (half) {
      f32x4 v = zero4();
      if (p && f < D) v = split::flip_sign(load4_f32(p + f), flip);
      if constexpr (Num<T>::planes == 1) {
        bf16x4 r;
        r[0] = (bf16)v[0]; r[1] = (bf16)v[1]; r[2] = (bf16)v[2]; r[3] = (bf16)v[3];
        return r;
      } else {
        const split::Chunk3 x = split::split_chunk(v, v);
        return Half3{__builtin_shufflevector(x.p0, x.p0, 0, 1, 2, 3), __builtin_shufflevector(x.p1, x.p1, 0, 1, 2, 3),
                     __builtin_shufflevector(x.p2, x.p2, 0, 1, 2, 3)};
      }
    } else {
      typename Num<T>::Raw r = zero_chunk<T>();
      if (p && f < D) r = negate(load_chunk(p + f), flip);
      return to_frag(r);
    }
  }
  // the lane's part of the dot product of two rows
  static __device__ __forceinline__ float dot(const T* p, const T* q, int kk, int g, int D) {
    const int f = half ? 4 * g : 32 * kk + 8 * g;
    if (f >= D) return 0.f;
    f32x4 a = load4_f32(p + f), b = load4_f32(q + f);
    float s = a[0] * b[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) s = __builtin_fmaf(a[i], b[i], s);
    if constexpr (!half) {
      a = load4_f32(p + f + 4); b = load4_f32(q + f + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) s = __builtin_fmaf(a[i], b[i], s);
    }
    return s;
  }
  // C[row][col] = init + sum over the features of tile[16 blk + row] b[col]
  static __device__ __forceinline__ f32x4 product(const bf16* t, int blk, const Feat* b, int c, int g, const f32x4& init) {
    f32x4 hi = init, lo = zero4();
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) product1(hi, lo, rows(t, blk, kk, c, g), b[kk]);
    return result<T>(hi, lo);
  }
};

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

// bits of a step's rows, 64 a word
template <int KT> struct Bits {
  static constexpr int N = (KT * TK + 63) / 64;
  uint64_t w[N];
  __device__ __forceinline__ uint32_t step(int t) const { return (uint32_t)(w[t / 2] >> (32 * (t & 1))); }
  __device__ __forceinline__ bool row(int i) const {
    uint64_t x = w[0];
#pragma unroll
    for (int k = 1; k < N; ++k) x = i >= 64 * k ? w[k] : x;
    return (x >> (i & 63)) & 1;
  }
};

// The rows of a tile on their way to LDS: NT threads, 8 values each and piece.  n: the rows there are; pieces past them
// are left out, up to a whole number of UNIT rows, which are computed together: their zeros are written too.
template <typename T, int DP, int KT, int NT, int UNIT = TK> struct Stage {
  typedef Tile<T, DP, KT> TL;
  static constexpr int CH = DP / 8, N = KT * TK * CH, PER = (N + NT - 1) / NT;
  typename Num<T>::Raw r[PER];
  static __device__ __forceinline__ int row(int p) { return (p * NT + (int)threadIdx.x % NT) / CH; }
  static __device__ __forceinline__ int feature(int p) { return 8 * ((p * NT + (int)threadIdx.x % NT) % CH); }
  static __device__ __forceinline__ bool in(int p) { return N % NT == 0 || p * NT + (int)threadIdx.x % NT < N; }
  static __device__ __forceinline__ bool needed(int p, int n) { return p * NT / CH < (n + UNIT - 1) / UNIT * UNIT; }   // uniform
  // byte offsets of the lane's pieces in a buffer of rows
  static __device__ __forceinline__ void offsets(uint32_t* off, int64_t row_bytes, int D) {
#pragma unroll
    for (int p = 0; p < PER; ++p)
      off[p] = in(p) && feature(p) < D ? (uint32_t)(row(p) * (uint32_t)row_bytes + feature(p) * (uint32_t)sizeof(T)) : kOob;
  }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t b, const uint32_t* off, int n) {
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if (needed(p, n)) r[p] = load8((const T*)nullptr, b, off[p]);
  }
  // zeros in the rows whose bit is not set
  __device__ __forceinline__ void keep(const Bits<KT>& bits) {
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if (!bits.row(row(p))) r[p] = zero_chunk<T>();
  }
  __device__ __forceinline__ void store(bf16* t, int n) const {
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if (needed(p, n) && in(p)) {
        bf16* d = t + row(p) * TL::pitch + feature(p);
        const auto v = to_frag(r[p]);
        if constexpr (Num<T>::planes == 1) store_chunk(d, v);
        else { store_chunk(d, v.p0); store_chunk(d + TL::plane, v.p1); store_chunk(d + 2 * TL::plane, v.p2); }
      }
  }
};

// ---- work items -------------------------------------------------------------------
struct Seg { int lo, hi; };                  // rows of one axis
__device__ __forceinline__ int edge_of(const int32_t* ptr, int e, int B, int N) {   // start of extended segment e
  const int i = e - 1 < 0 ? 0 : (e - 1 > B ? B : e - 1);
  int p = ptr[i];
  p = p < 0 ? 0 : (p > N ? N : p);
  return e <= 0 ? 0 : (e > B + 1 ? N : p);
}
// The extended segment of a slot and the slot's first virtual row in it (-1: an empty slot).  Segments of like lengths are
// found in one round: 64 lanes look at the segments around slot x guess (segments per slot).  Where that misses, every
// lane probes one of 63 steps, 3,969 segments in two more rounds.  The last round's lanes also hold the segment's ends.
template <int BQ>
__device__ __forceinline__ int find_tile(const int32_t* ptr, int B, int N, int G, float guess, uint32_t slot, int& vq0, Seg& s) {
  uint32_t lo = 0, hi = (uint32_t)B + 2;     // the slot is at or after segment lo's first, before hi's
  const uint32_t lane = lane_id();
  uint32_t step = 1, base = (uint32_t)((float)slot * guess);
  base = base > 31 ? base - 31 : 0;
  base = base + 63 < hi ? base : (hi > 63 ? hi - 63 : 0);
  for (bool first = true;; first = false) {
    if (!first) {
      step = (hi - lo + 62) / 63;
      base = lo;
    }
    const uint32_t e = base + lane * step;
    const int p = edge_of(ptr, (int)(e < hi ? e : hi), B, N);
    const uint64_t le = __ballot(e < hi && (uint32_t)p * (uint32_t)G / BQ + e <= slot);
    const int n = __builtin_popcountll(le);
    if (first ? n >= 1 && n < 64 : step == 1) {   // (offsets that decrease may give n = 0 here)
      const int i = n < 1 ? 1 : (n > 63 ? 63 : n);
      lo = base + i - 1;
      s.lo = __builtin_amdgcn_readlane(p, i - 1);
      s.hi = __builtin_amdgcn_readlane(p, i);
      break;
    }
    if (first) {                             // n is 0 or 64
      lo = n ? base + 63 : 0;
      hi = n ? hi : base;
    } else {
      lo = base + (n > 0 ? n - 1 : 0) * step;
      hi = hi < lo + step ? hi : lo + step;
    }
  }
  if (s.hi < s.lo) s.hi = s.lo;
  const int64_t v = ((int64_t)slot - (uint32_t)s.lo * (uint32_t)G / BQ - lo) * BQ;
  vq0 = v >= 0 && v < (int64_t)(s.hi - s.lo) * G ? (int)v : -1;
  return (int)lo;
}
// Rows of the other axis of extended segment e
__device__ __forceinline__ Seg other_rows(const int32_t* ptr, int e, int B, int N, bool same, const Seg& own) {
  if (e < 1 || e > B) return Seg{0, 0};
  if (same) return own;                      // one set of offsets for both axes
  Seg s{edge_of(ptr, e, B, N), edge_of(ptr, e + 1, B, N)};
  if (s.hi < s.lo) s.hi = s.lo;
  return s;
}
// Workgroups go to the 8 XCDs in turn, each with an L2 of its own.  Runs of 16 consecutive items stay on one XCD:
// neighbouring heads of a tile share the lines of its rows, and the tiles of a segment its keys.  (An eighth of all items
// each would do that too, but the work is not even along the items: of one graph's three slots two are empty, and one
// query over 2,000,000 keys in 2,048 parts took 297 us on three XCDs against 186 on all.)
constexpr uint32_t kRun = 16;
__device__ __forceinline__ uint32_t xcd_order(uint32_t bid, uint32_t n) {
  if (bid >= n / (8 * kRun) * (8 * kRun)) return bid;
  const uint32_t x = bid % 8, y = bid / 8;
  return (y / kRun * 8 + x) * kRun + y % kRun;
}
// One wave's (SH: one workgroup's) part of the work: key heads of a slot side by side, then slots, then parts
struct Item { uint32_t slot; int kvh, sp; };
template <int W, bool SH>
__device__ __forceinline__ bool item_of(const Args& a, uint32_t n_items, Item& it) {
  uint32_t i = a.first + xcd_order(blockIdx.x, gridDim.x);
  if constexpr (!SH && W > 1) i = i * W + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  if (i >= n_items) return false;
  const uint32_t j = a.by_heads(i), k = a.by_slots(j);
  it.kvh = (int)(i - j * (uint32_t)a.Hkv);
  it.slot = j - k * a.slots;
  it.sp = (int)k;
  return true;
}
// between a tile's writes and its reads
template <bool SH> __device__ __forceinline__ void tile_sync() {
  if constexpr (SH) __syncthreads();
  else wave_sync();
}

// Waves a SIMD that a workgroup kernel's registers have to leave room for.  The allocation is in steps that a change of a
// register or two can cross: 169 instead of 167 (bf16, D = 64, 32 columns a wave) took the forward of 12,289 rows from 197
// to 210 us.
template <typename T, int DP, int R> constexpr int group_occupancy() {
  return Num<T>::planes == 1 ? (R == 2 ? (DP <= 32 ? 4 : DP == 64 ? 3 : 2) : (DP <= 64 ? 4 : 3)) : 2;
}

// max and sum over the four lanes of a column
__device__ __forceinline__ float col_max(float v) { v = fmaxf(v, shfl_xor(v, 16)); return fmaxf(v, shfl_xor(v, 32)); }
__device__ __forceinline__ float col_sum(float v) { v += shfl_xor(v, 16); return v + shfl_xor(v, 32); }

// four features of one row
__device__ __forceinline__ void store4(float* p, const f32x4& v) { *reinterpret_cast<f32x4*>(p) = v; }
__device__ __forceinline__ bf16x4 pack4(const f32x4& v) {
  bf16x4 r;
  r[0] = (bf16)v[0]; r[1] = (bf16)v[1]; r[2] = (bf16)v[2]; r[3] = (bf16)v[3];
  return r;
}
__device__ __forceinline__ void store4(bf16* p, const f32x4& v) { *reinterpret_cast<bf16x4*>(p) = pack4(v); }
// values that a loop reads: waited for here, or every round of the loop would wait for its own prefetch as well
__device__ __forceinline__ void landed(bf16x4& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void landed(bf16x8& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void landed(Half3& v) { landed(v.p0); landed(v.p1); landed(v.p2); }
__device__ __forceinline__ void landed(split::Chunk3& v) { landed(v.p0); landed(v.p1); landed(v.p2); }

// Stores a column's features, NB blocks of 16: a lane has four of each block, 4g .. of it.  bf16: two blocks' four are
// exchanged with the neighbouring lane group's, so that a lane stores 8 neighbouring values and 64 bytes of a row are
// written at once instead of 32.
template <int NB> __device__ __forceinline__ void store_row(float* p, const f32x4* v, int g, int D) {
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (16 * b + 4 * g < D) store4(p + 16 * b + 4 * g, v[b]);
}
template <int NB> __device__ __forceinline__ void store_row(bf16* p, const f32x4* v, int g, int D) {
  if constexpr (NB == 1) {
    if (4 * g < D) store4(p + 4 * g, v[0]);
  } else {
#pragma unroll
    for (int b = 0; b < NB; b += 2) {
      const u32x2 x = __builtin_bit_cast(u32x2, pack4(v[b])), y = __builtin_bit_cast(u32x2, pack4(v[b + 1]));
      // groups 1, 3 of the first change places with groups 0, 2 of the second
      const u32x2 s0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(x[0], y[0], false, false));
      const u32x2 s1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(x[1], y[1], false, false));
      const int f = 16 * (b + (g & 1)) + 4 * (g & 2);
      if (f < D) *reinterpret_cast<u32x4*>(p + f) = u32x4{s0[0], s1[0], s0[1], s1[1]};
    }
  }
}

// the first n rows of a step, and of those the ones whose flag (of row 64 k + lane) is set
template <int KT>
__device__ __forceinline__ Bits<KT> step_bits(int n) {
  Bits<KT> b;
#pragma unroll
  for (int k = 0; k < Bits<KT>::N; ++k) {
    const int x = n - 64 * k;
    b.w[k] = x >= 64 ? ~0ull : x > 0 ? (1ull << x) - 1 : 0;
  }
  return b;
}

}  // namespace attn
}  // namespace egnn
