// The mask of the dropout: which values of a row stay, from a counter-based generator, so that it is made again in the
// backward instead of being stored.
//   value (row n, column f) stays where its 16 bits u >= cut = round(65536 p), and is scaled by up = 65536 / (65536 - cut)
// u is halfword f % 8 (lower half of a word first) of the four words that Philox4x32 (Salmon, Moraes, Dror, Shaw: Parallel
// random numbers: as easy as 1, 2, 3, 2011) makes of the counter (f / 8, n, offset low, offset high) and the key (seed low,
// seed high).  Seven rounds, the fewest with which its authors found it to pass every test of BigCrush: the products of 32
// bits run at a quarter of the vector rate, and ten rounds would bound the kernels.  16 bits a value halve that again; p is
// met to 2^-17 and the scale belongs to the p that is met, so the expectation is exact.  The mask depends on neither the
// dtype nor the strides nor the launch.
#pragma once
#include "../../include/egnn.h"
#include "egnn_device.h"
#include <cmath>

namespace egnn {

struct DropArgs {
  const int64_t* rng;                        // device: seed, offset
  int64_t site;
  uint32_t cut;
  float up;
};

inline bool drop_ok(const EgnnDropout* d) { return d->p >= 0.0 && d->p <= 1.0; }   // (not a NaN)
inline DropArgs drop_args(const EgnnDropout* d) {
  DropArgs a{};
  a.rng = d->rng; a.site = d->site;
  a.cut = (uint32_t)std::nearbyint(d->p * 65536.0);
  a.up = a.cut < 65536 ? (float)(65536.0 / (65536.0 - a.cut)) : 0.f;
  return a;
}

struct Mask {
  uint32_t k0, k1, c2, c3, cut;
  float up;
};
__device__ __forceinline__ Mask mask_of(const DropArgs& a) {
  const uint64_t s = (uint64_t)a.rng[0], o = (uint64_t)a.rng[1] + (uint64_t)a.site;
  return Mask{(uint32_t)s, (uint32_t)(s >> 32), (uint32_t)o, (uint32_t)(o >> 32), a.cut, a.up};
}

// the 128 bits of columns 8 g .. 8 g + 7 of row n
__device__ __forceinline__ u32x4 mask_words(const Mask& m, uint32_t n, uint32_t g) {
  uint32_t c0 = g, c1 = n, c2 = m.c2, c3 = m.c3, k0 = m.k0, k1 = m.k1;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return u32x4{c0, c1, c2, c3};
}

// bit i: column f + i stays, for the N columns (4 or 8) from any column f on
template <int N> __device__ __forceinline__ uint32_t keep_bits(const Mask& m, uint32_t n, int f) {
  uint32_t bits = 0;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    if (part && (f & 7) + N <= 8) break;
    const u32x4 w = mask_words(m, n, (uint32_t)(f >> 3) + part);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu;
      bits |= (u >= m.cut ? 1u : 0u) << (8 * part + i);
    }
  }
  return bits >> (f & 7);
}

// v[i] *= up where column f + i of row n stays, else 0 (whatever it was).  ANY: f need not be a multiple of N.
template <int N, bool ANY> __device__ __forceinline__ void drop(const Mask& m, uint32_t n, int f, float* v) {
  static_assert(N == 4 || N == 8, "pieces of 16 bytes");
  if (ANY && f % N) {
    const uint32_t bits = keep_bits<N>(m, n, f);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = bits >> i & 1 ? v[i] * m.up : 0.f;
    return;
  }
  const u32x4 w = mask_words(m, n, (uint32_t)f >> 3);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint32_t x = w[i / 2];
    if (N == 4 && (f & 4)) x = w[2 + i / 2];
    const uint32_t u = i & 1 ? x >> 16 : x & 0xffffu;
    v[i] = u >= m.cut ? v[i] * m.up : 0.f;
  }
}

}  // namespace egnn
