// Pieces of a row: what a lane of the kernels over rows (norms, table rows, heads) loads and stores at once.
#pragma once
#include "egnn_device.h"
#include <type_traits>

namespace egnn {

// From which size of one tensor on it is written, and read, past the cache (which holds 256 MB) where the next kernel reads it,
// or this one reads it once.  The norm's backward and the table rows were measured on both sides, see there.
constexpr int64_t kPastStore = int64_t(64) << 20, kPastLoad = int64_t(256) << 20;


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

}  // namespace egnn
