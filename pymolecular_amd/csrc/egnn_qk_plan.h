// How a call of the head norm with rotation is cut into pieces, tiles and workgroups: host arithmetic alone.
#pragma once
#include "../../include/egnn.h"
#include <cmath>

namespace egnn {
namespace qk {

constexpr int NT = 256;
constexpr int kPairs = 64;                   // pairs of a head at most
constexpr int kTable = 2304;                 // cos and sin of a tile at most: 18 KB
constexpr int kHeads = 4096;
constexpr int64_t kMaxGrid = int64_t(1) << 20;

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// k / H = the high word of k reciprocal(H), for H > 1.  The reciprocal is rounded up, by less than H units of 2^-32 / H, so
// the quotient is exact where k H <= 2^32: the number of a head in a tile stays below rows times heads (tile_rows).
inline uint32_t reciprocal(int32_t H) { return H > 1 ? (uint32_t)(((uint64_t(1) << 32) + H - 1) / H) : 0; }

// Widest piece that fits 16 bytes (8 in the backward) and never lies across the rotated part's middle or end.  The backward
// with pieces of 8 bf16 holds 184 registers, two waves a SIMD, with 4 it holds 116: 32,768 x 8 heads of 32, 24.5 and 16.3 us;
// 1,048,576 x 3 heads of 128, 757 and 613; only the largest tensors of narrow heads lose, 2,000,000 x 8 heads of 32, 660 and 712.
inline int piece_of(const EgnnQkDims* d, bool bwd) {
  int v = d->dtype == EGNN_F32 || bwd ? 4 : 8;
  const int half = d->D / 2, r = d->rotary / 2;
  while (v > 1 && (half % v || (!d->interleaved && r % v))) v /= 2;
  return v;
}
inline int lanes_of(const EgnnQkDims* d, bool bwd) {
  int l = 1;
  while (l * piece_of(d, bwd) < d->D / 2) l *= 2;
  return l;
}
// Workgroups that small calls are spread over, and partial rows of the weight gradients.  Each costs its start, about 4 ns:
// with 512, 1,024, 2,048 and 4,096, forward of 4,096 x 8 heads of 32 bf16 5.6, 6.6, 10.8 and 19.0 us, of 32,768 x 10 heads of 64
// 18.1, 16.7, 19.4 and 25.8; backward with 512, 1,024 and 2,048 10.8, 13.2 and 21.8 us, and 35.0, 29.1 and 34.5.
inline int blocks_for(const EgnnQkDims* d, bool bwd) {
  const int64_t values = d->N * (d->Hq + d->Hk) * d->D;
  return values < 1 << 20 ? 256 : values < (bwd ? 4 : 8) << 20 ? 512 : 1024;
}
// Rows of a tile: enough heads of the side with fewer of them for two of each group of lanes, but a tile for each workgroup first
inline int tile_rows(const EgnnQkDims* d, bool bwd) {
  const int H = d->Hq < d->Hk ? d->Hq : d->Hk;
  const int groups = NT / lanes_of(d, bwd);
  int64_t tb = groups * 2 / H;
  if (tb > kTable / (d->D / 2 + 2)) tb = kTable / (d->D / 2 + 2);
  const int64_t big = d->Hq < d->Hk ? d->Hk : d->Hq;
  if (tb > (int64_t(1) << 32) / (big * big)) tb = (int64_t(1) << 32) / (big * big);   // (reciprocal(); 256 at 4,096 heads)
  if (tb > ceil_div(d->N, blocks_for(d, bwd))) tb = ceil_div(d->N, blocks_for(d, bwd));
  int m = groups;                            // whole rounds of the groups over the heads
  for (int h = H; h % 2 == 0 && m > 1; h /= 2) m /= 2;
  if (tb > m) tb = tb / m * m;
  return tb < 1 ? 1 : (int)tb;
}
inline int32_t blocks_of(const EgnnQkDims* d, bool bwd) {
  const int64_t most = bwd ? blocks_for(d, true) : kMaxGrid;
  const int64_t tiles = ceil_div(d->N, tile_rows(d, bwd));
  return (int32_t)(tiles < most ? tiles : most);
}

// base^(-2 i / rotary) / 2 pi for the rotary / 2 pairs, turns a position, in units of 2^-64: by repeated multiplication in
// extended precision (one power instead of 64), whose roundings make them wrong by up to 5 units for bases near 1, by less than
// one from 100 on.  A position of 2^32 makes 2^-29 turns of the 5, one of 2^20 2^-41.
inline void frequencies(const EgnnQkDims* d, uint64_t* freq) {
  const long double step = d->rotary ? powl((long double)d->base, -2.0L / d->rotary) : 1.0L;
  long double f = 18446744073709551616.0L / 6.283185307179586476925286766559L;
  for (int i = 0; i < d->rotary / 2; ++i, f *= step) freq[i] = (uint64_t)(f + 0.5L);
}

}  // namespace qk
}  // namespace egnn
