// Rows of a table by token, times a scale, and the table's gradient.
//   out_i = scale W[t_i],   gW[v] = scale sum_{i: t_i = v} g_i,   tokens outside the table: rows of zeros, no gradient
// Forward: a lane takes one or four pieces of 16 bytes, whose tokens and then table pieces are on their way together.  Bound by
// the rows it writes: 2,000,000 x 128 bf16 81 us, 6.3 TB/s.
// Backward: tokens are sorted first (stably, so every sum has a fixed order), then each row of the gradient is read once, in
// the sorted order, by a group of lanes that sums a span of it in fp32 registers and writes a table row where a run of one
// token ends.  Spans that share a run are joined in LDS, in order; no value goes through an atomic.  A group has as many lanes as a
// row has pieces (up to 64), so odd widths leave few of them idle.  Two forms:
//  - local: a workgroup sorts a chunk of tokens by counting, in LDS, for a range of table rows.  One chunk: it writes the table;
//    several chunks: a partial table each, added up in order by a second launch.  2,000,000 x 128 bf16 over 119 rows 124 us + 13
//    us, floor 97; 19,456 x 128 9.7 + 3.9 us, where it waits for two rounds of tokens, one of rows and the barriers between.
//  - sorted: counting sorts of (token, row) by digits of up to 11 bits, then the sums over tiles of the sorted order, and a launch
//    that joins the runs that cross tiles and clears the rows that no token names.  40,961 x 259 fp32 over 50,021 rows 54 us: two
//    sorts of three launches 25, the sums 18, the rest 14; its floor is 18, and each of the eight launches waits on memory two or
//    three times.  Counts that a scatter adds up by itself instead of scan_kernel cost as much (66 us and 64).
#include "egnn_internal.h"
#include "egnn_rows.h"

namespace egnn {
namespace embed {

// A launch may have fewer than 2^32 threads: at most this many workgroups at a time
constexpr int64_t kMaxGrid = int64_t(1) << 20;

// Piece k of a row of VEC columns each; the last one ends with the row and overlaps the one before (same bits twice)
template <int VEC> __device__ __forceinline__ int first_column(int k, int C) {
  const int f = k * VEC;
  return f + VEC <= C || C < VEC ? f : C - VEC;
}
template <typename T, typename P, bool TAIL>
__device__ __forceinline__ void store_params(void* p, int f, int C, const float* v) {
  constexpr int N = Vec<T, TAIL>::N;
  P* q = (P*)p;
  if constexpr (std::is_same<T, P>::value) Vec<T, TAIL>::store(q, f, C, v);
  else if (!TAIL || C >= N) {
    Vec<P, false>::store(q, f, C, v);
    Vec<P, false>::store(q, f + N / 2, C, v + N / 2);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < C) q[i] = from_f32<P>(v[i]);
  }
}

// ---- forward ------------------------------------------------------------------------------
constexpr int NT = 256;
// Up to so many pieces a lane takes one: more workgroups come before more loads in flight
constexpr int64_t kFewPieces = 1024 * 1024;

struct FwdArgs {
  const void *tokens, *w;
  void* out;
  int64_t N, V, ldw;
  int32_t C, G, GT, R;                       // columns, pieces in a row, pieces in a tile of it, rows in a workgroup
  uint32_t magic;                            // l / GT = the high word of l magic (GT > 1)
  float scale;
};

template <typename T, typename P, typename I, bool TAIL, int U, bool PAST>
__global__ __launch_bounds__(NT) void fwd_kernel(FwdArgs a) {
  typedef Vec<T, TAIL> V;
  constexpr int VEC = V::N;
  int64_t n[U], t[U];
  int f[U];
  bool in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t l = u * NT + threadIdx.x;
    const uint32_t k = a.GT > 1 ? __umulhi(l, a.magic) : l;
    const int g = (int)(l - k * a.GT) + blockIdx.y * a.GT;
    n[u] = (int64_t)blockIdx.x * a.R + k;
    in[u] = (int)k < a.R && n[u] < a.N && g < a.G;
    f[u] = in[u] ? first_column<VEC>(g, a.C) : 0;
    t[u] = (int64_t)((const I*)a.tokens)[in[u] ? n[u] : 0];
  }
  float v[U][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool has = (uint64_t)t[u] < (uint64_t)a.V;
    load_params<T, P, TAIL>((const P*)a.w + (has ? t[u] : 0) * a.ldw, f[u], a.C, v[u]);
    const float s = a.scale;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[u][i] = has ? v[u][i] * s : 0.f;
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (in[u]) V::template store<PAST>((T*)a.out + n[u] * a.C, f[u], a.C, v[u]);
}

template <typename T, typename P, typename I, bool TAIL, int U, bool PAST>
static void launch_fwd(FwdArgs a, hipStream_t st) {
  a.G = (int32_t)cdiv(a.C, Vec<T>::N);
  const int tiles = (int)cdiv(a.G, NT * U);
  a.GT = (int32_t)cdiv(a.G, tiles);
  a.R = NT * U / a.GT;
  a.magic = a.GT > 1 ? (uint32_t)(((uint64_t(1) << 32) + a.GT - 1) / a.GT) : 0;
  const int64_t most = kMaxGrid / tiles * a.R, N = a.N;
  const FwdArgs all = a;
  for (int64_t n = 0; n < N; n += most) {
    a.tokens = (const I*)all.tokens + n;
    a.out = (T*)all.out + n * a.C;
    a.N = N - n < most ? N - n : most;
    fwd_kernel<T, P, I, TAIL, U, PAST><<<dim3((uint32_t)cdiv(a.N, a.R), (uint32_t)tiles), NT, 0, st>>>(a);
  }
}
template <typename T, typename P, typename I, bool TAIL>
static void launch_fwd(const FwdArgs& a, hipStream_t st) {
  if (a.N * cdiv(a.C, Vec<T>::N) < kFewPieces) launch_fwd<T, P, I, TAIL, 1, false>(a, st);
  else if (a.N * a.C * (int64_t)sizeof(T) < kPastStore) launch_fwd<T, P, I, TAIL, 4, false>(a, st);
  else launch_fwd<T, P, I, TAIL, 4, true>(a, st);
}

// ---- backward: sorting inside a workgroup --------------------------------------------------
constexpr int BT = 256, NW = BT / 64;        // threads and waves of a workgroup
constexpr int kBins = 2048;                  // values of a digit at most
constexpr int kChunk = 6144, kRange = 1024;  // local: tokens and table rows of a workgroup at most

// A stable counting sort of len values: bin_of(i) in [0, bins), or negative for none; put(i, bin, position).  cnt: NW * bins
// words, off: bins + 1 (off[b]: where bin b begins), memo: len halfwords.  The waves take consecutive parts, so a bin's values
// of a wave come after those of the waves before it; within 64 values the lanes of one bin find each other by votes on its
// bits.
template <typename Bin, typename Put>
__device__ __forceinline__ void sort_block(int len, int bins, uint32_t* cnt, uint32_t* off, uint16_t* memo, Bin bin_of, Put put) {
  __shared__ uint32_t wave_sum[NW];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int per = (len + BT - 1) / BT * 64, lo = w * per;
  for (int i = threadIdx.x; i < NW * bins; i += BT) cnt[i] = 0;
  __syncthreads();
  uint32_t* mine = cnt + w * bins;
  for (int r = 0; r < per; r += 256) {
    int b[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = lo + r + 64 * u + lane;
      b[u] = r + 64 * u < per && i < len ? bin_of(i) : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = lo + r + 64 * u + lane;
      if (r + 64 * u < per && i < len) memo[i] = (uint16_t)b[u];
      if (b[u] >= 0) atomicAdd(&mine[b[u]], 1u);
    }
  }
  __syncthreads();
  const int own = (bins + BT - 1) / BT, own0 = own * threadIdx.x, own1 = min(bins, own0 + own);   // a thread's bins
  uint32_t s = 0;
  for (int b = own0; b < own1; ++b)
#pragma unroll
    for (int k = 0; k < NW; ++k) s += cnt[k * bins + b];
  uint32_t inc = s;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t x = __shfl_up(inc, d, 64);
    if (lane >= d) inc += x;
  }
  if (lane == 63) wave_sum[w] = inc;
  __syncthreads();
  uint32_t base = inc - s;
  for (int k = 0; k < w; ++k) base += wave_sum[k];
  for (int b = own0; b < own1; ++b) {
    off[b] = base;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      const uint32_t c = cnt[k * bins + b];
      cnt[k * bins + b] = base;
      base += c;
    }
    if (b == bins - 1) off[bins] = base;
  }
  __syncthreads();
  const int bits = 32 - __clz(bins - 1);
  const uint64_t below = (uint64_t(1) << lane) - 1;
  for (int r = 0; r < per; r += 256) {
    int bin[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = lo + r + 64 * u + lane;
      bin[u] = r + 64 * u < per && i < len ? (int)(int16_t)memo[i] : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int b = bin[u];
      uint64_t same = __ballot(b >= 0);
      if (!same) continue;                   // (the whole wave)
      for (int k = 0; k < bits; ++k) {
        const bool one = b >> k & 1;
        const uint64_t v = __ballot(one);
        same &= one ? v : ~v;
      }
      uint32_t pos = 0;
      if (b >= 0) pos = mine[b] + (uint32_t)__popcll(same & below);
      wave_sync();
      if (b >= 0 && !(same & below)) mine[b] = pos + (uint32_t)__popcll(same);
      wave_sync();
      if (b >= 0) put(lo + r + 64 * u + lane, b, (int)pos);
    }
  }
  __syncthreads();
}

// ---- backward: sums over a tile of the sorted order -------------------------------------------
struct BwdArgs {
  const void *tokens, *g;
  void* gw;
  float* part;                               // local: partial tables [chunk][V][C]; sorted: the carries [tile][2][C]
  const uint64_t* sorted;
  int64_t N, V, ldg, padding;
  int32_t C, lpr, pieces;                    // columns, lanes of a row in a column tile, pieces of a row
  int32_t chunk, chunks, range;              // local: tokens and table rows of a workgroup
  int32_t span, tile;                        // sorted: positions of a group of lanes, and of a workgroup
  float scale;
};

// Positions [0, S) of a tile: key(p) and row(p) (a row of the gradient).  before / after: the first / last run goes on outside
// the tile.  A group of lpr lanes sums `span` positions; end(key, p): where the run of this key ends that holds position
// p - 1.  emit(key, kind, v) gets each run's sum: kind 0 the whole run, 1 its part if it began before the tile, 2 its part if it
// goes on behind it.
template <typename T, bool TAIL, bool PAST, typename Key, typename Row, typename End, typename Emit>
__device__ __forceinline__ void sum_tile(const BwdArgs& a, int S, int span, bool before, bool after, float* carry, Key key,
                                         Row row, End end, Emit emit) {
  typedef Vec<T, TAIL> V;
  constexpr int VEC = V::N, UR = 8;
  const int lpr = a.lpr, groups = BT / lpr, g = threadIdx.x / lpr, lane = threadIdx.x - g * lpr;
  const int k = blockIdx.y * lpr + lane;
  const bool lives = g < groups && k < a.pieces;
  const int f = lives ? first_column<VEC>(k, a.C) : 0;
  const int p0 = lives ? min(S, g * span) : S, p1 = min(S, p0 + span);
  float acc[VEC];
  auto slot = [&](int group, int which) { return carry + ((group * 2 + which) * lpr + lane) * VEC; };
  auto flush = [&](uint32_t cur) {
    const bool starts = p0 > 0 ? key(p0 - 1) == cur : before && key(0) == cur;   // before this span
    const bool goes_on = p1 < S ? key(p1) == cur : after && key(S - 1) == cur;
    if (!starts && !goes_on) { emit(cur, 0, f, acc); return; }
    float* out = slot(g, starts ? 0 : 1);
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = acc[i];
  };
  if (p0 < p1) {
    uint32_t cur = key(p0);
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
    for (int p = p0; p < p1; p += UR) {
      typename V::piece x[UR];
#pragma unroll
      for (int u = 0; u < UR; ++u) x[u] = V::template load<PAST>((const T*)a.g + row(min(p + u, p1 - 1)) * a.ldg, f, a.C);
      if (p + UR <= p1 && key(p + UR - 1) == cur) {   // one run: eight rows are added up by themselves first
        float e[UR][VEC];
#pragma unroll
        for (int u = 0; u < UR; ++u) V::floats(x[u], e[u]);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          acc[i] += ((e[0][i] + e[1][i]) + (e[2][i] + e[3][i])) + ((e[4][i] + e[5][i]) + (e[6][i] + e[7][i]));
      } else {
#pragma unroll
        for (int u = 0; u < UR; ++u) {
          if (p + u >= p1) break;
          const uint32_t q = key(p + u);
          if (q != cur) {
            flush(cur);
            cur = q;
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
          }
          float e[VEC];
          V::floats(x[u], e);
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[i] += e[i];
        }
      }
    }
    flush(cur);
  }
  __syncthreads();
  if (p0 >= p1) return;
  // the first group of a run that crosses spans joins it: its own part, then the heads of the groups behind
  const uint32_t last = key(p1 - 1), first = key(p0);
  const bool first_began = p0 > 0 ? key(p0 - 1) == first : before;
  auto join = [&](uint32_t cur, int which) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = slot(g, which)[i];
    const int h = (min(end(cur, p1), S) - 1) / span + 1;   // the groups up to that of its last position
#pragma unroll 4
    for (int q = g + 1; q < h; ++q)
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += slot(q, 0)[i];
    const bool ends = !after || key(S - 1) != cur;
    emit(cur, which == 0 ? 1 : ends ? 0 : 2, f, acc);
  };
  if (g == 0 && before) join(first, 0);      // began before the tile
  const bool last_began = last == first && first_began;
  const bool goes_on = p1 < S ? key(p1) == last : after;
  if (!last_began && goes_on) join(last, 1);
}

template <typename T, typename P, typename I, bool TAIL, bool PAST>
__global__ __launch_bounds__(BT) void local_kernel(BwdArgs a) {
  extern __shared__ __align__(16) uint32_t lds[];
  constexpr int VEC = Vec<T>::N;
  const uint32_t r = blockIdx.x / (uint32_t)a.chunks;
  const int64_t chunk = blockIdx.x - r * (uint32_t)a.chunks;
  const int64_t n0 = chunk * a.chunk, v0 = (int64_t)r * a.range;
  const int len = (int)(a.N - n0 < a.chunk ? a.N - n0 : a.chunk), bins = (int)(a.V - v0 < a.range ? a.V - v0 : a.range);
  uint32_t *ent = lds, *off = ent + a.chunk, *cnt = off + ((a.range + 4) & ~3);   // (cnt: at least the carries of sum_tile)
  uint16_t* memo = (uint16_t*)(cnt + max(NW * a.range, BT * 2 * VEC));
  const I* tokens = (const I*)a.tokens + n0;
  sort_block(len, bins, cnt, off, memo,
             [&](int i) {
               const uint64_t b = (uint64_t)((int64_t)tokens[i] - v0);
               return b < (uint64_t)bins ? (int)b : -1;
             },
             [&](int i, int b, int pos) { ent[pos] = (uint32_t)b << 16 | (uint32_t)i; });
  const int S = (int)off[bins], groups = BT / a.lpr;
  // (tokens outside the table or the range have no entry)
  auto write = [&](int64_t v, int f, const float* acc) {
    if (a.part) {
      store_params<T, float, TAIL>(a.part + (chunk * a.V + v) * a.C, f, a.C, acc);
    } else {
      float o[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = v == a.padding ? 0.f : acc[i] * a.scale;
      store_params<T, P, TAIL>((P*)a.gw + v * a.C, f, a.C, o);
    }
  };
  sum_tile<T, TAIL, PAST>(a, S, (S + groups - 1) / groups, false, false, (float*)cnt, [&](int p) { return ent[p] >> 16; },
                    [&](int p) { return n0 + (int64_t)(ent[p] & 0xffff); }, [&](uint32_t b, int) { return (int)off[b + 1]; },
                    [&](uint32_t b, int, int f, const float* acc) { write(v0 + b, f, acc); });
  const int g = threadIdx.x / a.lpr, k = blockIdx.y * a.lpr + threadIdx.x - g * a.lpr;
  if (g >= groups || k >= a.pieces) return;
  const float zero[VEC] = {};
  for (int b = g; b < bins; b += groups)
    if (off[b] == off[b + 1]) write(v0 + b, first_column<VEC>(k, a.C), zero);
}

// gW = the sum of the partial tables, M = V C values each: 16 pieces of 4 a workgroup, 64 groups joined in order
template <typename P>
__global__ __launch_bounds__(1024) void reduce_kernel(const float* part, int chunks, int64_t M, int64_t pad0, int64_t pad1,
                                                      float scale, P* gw) {
  __shared__ float red[64][16][5];
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
  const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
  for (int64_t f0 = (int64_t)blockIdx.x * 64; f0 < M; f0 += (int64_t)gridDim.x * 64) {
    const int64_t f = f0 + 4 * c;
    const int m = f + 4 <= M ? 4 : f < M ? (int)(M - f) : 0;
    double s[4] = {};                      // (many tokens: up to 5,462 tables one after the other)
#pragma unroll 4
    for (int b = k; b < chunks; b += 64) {
      const float* p = part + b * M + f;
      if (m == 4) {
        const type t = *(const type*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] += t[i];
      } else {
        for (int i = 0; i < m; ++i) s[i] += p[i];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) red[k][c][i] = (float)s[i];
    __syncthreads();
    for (int h = 32; h; h >>= 1) {
      if (k < h)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[k][c][i] += red[k + h][c][i];
      __syncthreads();
    }
    if (k == 0)
      for (int i = 0; i < m; ++i) gw[f + i] = from_f32<P>(f + i >= pad0 && f + i < pad1 ? 0.f : red[0][c][i] * scale);
  }
}

// ---- backward: the whole order sorted -------------------------------------------------------
constexpr int kSortTile = 4096;              // values of a workgroup in a pass at most

// A value is token << 32 | row; tokens outside the table get V and come last.
struct SortArgs {
  const void* tokens;                        // the first pass reads these
  const uint64_t* from;
  uint64_t* to;
  uint32_t *hist, *total;                    // [tile][digits], [digits]
  int64_t N, V;
  int32_t shift, digits, tile, tiles;
};
template <typename I, bool FIRST> __device__ __forceinline__ uint64_t sort_value(const SortArgs& a, int64_t n) {
  if (!FIRST) return a.from[n];
  const int64_t t = (int64_t)((const I*)a.tokens)[n];
  return ((uint64_t)t < (uint64_t)a.V ? (uint64_t)t : (uint64_t)a.V) << 32 | (uint64_t)n;
}
template <typename I, bool FIRST>
__global__ __launch_bounds__(BT) void hist_kernel(SortArgs a) {
  __shared__ uint32_t h[kBins];
  for (int d = threadIdx.x; d < a.digits; d += BT) h[d] = 0;
  __syncthreads();
  const int64_t n0 = (int64_t)blockIdx.x * a.tile, n1 = a.N - n0 < a.tile ? a.N : n0 + a.tile;
  for (int64_t n = n0 + threadIdx.x; n < n1; n += BT)
    atomicAdd(&h[(uint32_t)(sort_value<I, FIRST>(a, n) >> (32 + a.shift)) & (uint32_t)(a.digits - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < a.digits; d += BT) a.hist[(int64_t)blockIdx.x * a.digits + d] = h[d];
}
// hist[tile][d] becomes the sum of the tiles before; total[d]: of all.  16 digits a workgroup, 64 parts of the tiles.
__global__ __launch_bounds__(1024) void scan_kernel(SortArgs a) {
  __shared__ uint32_t part[64][17];
  const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
  const int d = blockIdx.x * 16 + c;
  const int per = (a.tiles + 63) / 64, b0 = min(a.tiles, k * per), b1 = min(a.tiles, b0 + per);
  uint32_t s = 0;
  if (d < a.digits) {
#pragma unroll 8
    for (int b = b0; b < b1; ++b) s += a.hist[(int64_t)b * a.digits + d];
  }
  part[k][c] = s;
  __syncthreads();
  uint32_t at = 0;
  for (int j = 0; j < k; ++j) at += part[j][c];
  if (d >= a.digits) return;
  for (int b = b0; b < b1; ++b) {
    const uint32_t x = a.hist[(int64_t)b * a.digits + d];
    a.hist[(int64_t)b * a.digits + d] = at;
    at += x;
  }
  if (k == 63) a.total[d] = at;
}
template <typename I, bool FIRST>
__global__ __launch_bounds__(BT) void scatter_kernel(SortArgs a) {
  extern __shared__ __align__(16) uint32_t lds[];
  __shared__ uint32_t sums[NW];
  uint32_t *base = lds, *off = base + a.digits, *cnt = off + a.digits + 4;
  uint16_t* memo = (uint16_t*)(cnt + NW * a.digits);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  // where a digit's values of this tile begin: all values of smaller digits, then those of the tiles before
  const int own = (a.digits + BT - 1) / BT, own0 = own * threadIdx.x, own1 = min(a.digits, own0 + own);   // a thread's digits
  uint32_t s = 0;
  for (int d = own0; d < own1; ++d) s += a.total[d];
  uint32_t inc = s;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t x = __shfl_up(inc, d, 64);
    if (lane >= d) inc += x;
  }
  if (lane == 63) sums[w] = inc;
  __syncthreads();
  uint32_t at = inc - s;
  for (int k = 0; k < w; ++k) at += sums[k];
  for (int d = own0; d < own1; ++d) {
    base[d] = at + a.hist[(int64_t)blockIdx.x * a.digits + d];
    at += a.total[d];
  }
  __syncthreads();
  const int64_t n0 = (int64_t)blockIdx.x * a.tile;
  const int len = (int)(a.N - n0 < a.tile ? a.N - n0 : a.tile);
  sort_block(len, a.digits, cnt, off, memo,
             [&](int i) { return (int)((uint32_t)(sort_value<I, FIRST>(a, n0 + i) >> (32 + a.shift)) & (uint32_t)(a.digits - 1)); },
             [&](int i, int d, int pos) { a.to[base[d] + (uint32_t)pos - off[d]] = sort_value<I, FIRST>(a, n0 + i); });
}

template <typename T, typename P, bool TAIL, bool PAST>
__global__ __launch_bounds__(BT) void sorted_kernel(BwdArgs a) {
  extern __shared__ __align__(16) uint32_t lds[];
  constexpr int VEC = Vec<T>::N;
  const int64_t b0 = (int64_t)blockIdx.x * a.tile;
  const int len = (int)(a.N - b0 < a.tile ? a.N - b0 : a.tile);
  uint32_t *key = lds, *row = key + ((a.tile + 2 + 3) & ~3);   // keys of the neighbours too: key[0] before, key[len + 1] behind
  float* carry = (float*)(row + ((a.tile + 3) & ~3));
  for (int p = threadIdx.x; p < len + 2; p += BT) {
    const int64_t q = b0 + p - 1;
    const uint64_t e = q >= 0 && q < a.N ? a.sorted[q] : ~uint64_t(0);
    key[p] = (uint32_t)(e >> 32);
    if (p > 0 && p <= len) row[p - 1] = (uint32_t)e;
  }
  __syncthreads();
  // the tokens outside the table come last, with key V: they have no sum
  int S = len;
  if (key[len] == (uint32_t)a.V) {           // (the first such position, by halving)
    int lo = 0, hi = len - 1;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (key[mid + 1] == (uint32_t)a.V) hi = mid;
      else lo = mid + 1;
    }
    S = lo;
  }
  const bool before = S > 0 && key[0] == key[1], after = S == len && key[len] == key[len + 1];
  auto end = [&](uint32_t v, int p) {
    for (int step = a.tile; step; step >>= 1)
      while (p + step <= S && key[p + step] == v) p += step;
    return p;
  };
  sum_tile<T, TAIL, PAST>(a, S, a.span, before, after, carry, [&](int p) { return key[p + 1]; },
                          [&](int p) { return (int64_t)row[p]; }, end,
                    [&](uint32_t v, int kind, int f, const float* acc) {
                      if (kind) {
                        store_params<T, float, TAIL>(a.part + ((int64_t)blockIdx.x * 2 + kind - 1) * a.C, f, a.C, acc);
                        return;
                      }
                      float o[VEC];
#pragma unroll
                      for (int i = 0; i < VEC; ++i) o[i] = v == a.padding ? 0.f : acc[i] * a.scale;
                      store_params<T, P, TAIL>((P*)a.gw + (int64_t)v * a.C, f, a.C, o);
                    });
}

// Table rows whose run crosses tiles, or that no token names
constexpr int FT = 256, kFixRows = 64, kLight = 16, kFew = 1024;
// The first position with a token of `want` or above, which is in [lo, lo + n], by a wave: 64 places of the rest at a time
__device__ __forceinline__ int64_t first_of(const uint64_t* sorted, int64_t lo, int64_t n, uint64_t want) {
  while (n > 0) {
    const int64_t step = (n + 63) / 64;
    const int64_t p = lo + lane_id() * step;
    const bool below = p < lo + n && sorted[p] >> 32 < want;
    const int k = (int)__popcll(__ballot(below));   // the places below it come first
    if (k == 0) return lo;
    const int64_t end = lo + n;
    lo += (k - 1) * step + 1;
    n = lo + step - 1 < end ? step - 1 : end - lo;
  }
  return lo;
}
// The last digit's totals say between which positions the tokens of 2^shift rows lie; a workgroup takes some of those rows.
template <typename T, typename P, bool TAIL>
__global__ __launch_bounds__(FT) void fix_kernel(BwdArgs a, const uint32_t* total, int shift, int rows) {
  constexpr int VEC = Vec<T>::N;
  __shared__ int32_t at[kFixRows + 1], t0[kFixRows], t1[kFixRows], ends[2], part_sum[FT / 64];
  __shared__ float join[FT * VEC];
  const int lpr = a.lpr, groups = FT / lpr, g = threadIdx.x / lpr, lane = threadIdx.x - g * lpr;
  const int k = blockIdx.y * lpr + lane;
  const bool lives = g < groups && k < a.pieces;
  const int f = lives ? first_column<VEC>(k, a.C) : 0;
  const int64_t blocks = (a.V + rows - 1) / rows;
  auto part = [&](int t, int which) { return a.part + ((int64_t)t * 2 + which) * a.C; };
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int64_t v0 = b * rows;             // (rows divides 2^shift, or shift is 0)
    const int nv = (int)(a.V - v0 < rows ? a.V - v0 : rows);
    auto write = [&](int i, const float* acc) {
      float o[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) o[j] = v0 + i == a.padding ? 0.f : acc[j] * a.scale;
      store_params<T, P, TAIL>((P*)a.gw + (v0 + i) * a.C, f, a.C, o);
    };
    // where the rows' tokens begin: behind those of all smaller last digits
    const int digit = (int)(v0 >> shift);
    uint32_t before = 0;
    for (int d = threadIdx.x; d < digit; d += FT) before += total[d];
#pragma unroll
    for (int m = 32; m; m >>= 1) before += __shfl_xor(before, m, 64);
    if (lane_id() == 0) part_sum[threadIdx.x / 64] = (int32_t)before;
    __syncthreads();
    int32_t s0 = part_sum[0] + part_sum[1] + part_sum[2] + part_sum[3], s1 = s0;
    if (shift) {
      s1 += (int32_t)total[digit];
      if (s1 - s0 > FT) {                    // among many: the part of these rows
        if (threadIdx.x < 128) {
          const int32_t p = (int32_t)first_of(a.sorted, s0, s1 - s0, (uint64_t)(v0 + (threadIdx.x < 64 ? 0 : nv)));
          if (lane_id() == 0) ends[threadIdx.x / 64] = p;
        }
        __syncthreads();
        s0 = ends[0];
        s1 = ends[1];
      }
    }
    if (!shift) {                            // a digit is a row
      if (threadIdx.x == 0) {
        at[0] = s0;
        for (int i = 0; i < nv; ++i) at[i + 1] = at[i] + (int32_t)total[v0 + i];
      }
    } else if (s1 - s0 <= kFew) {            // few tokens: each looks whether it begins the next rows
      for (int64_t p = s0 + (int64_t)threadIdx.x; p <= s1; p += FT) {   // (past s1 it may pass 2^31)
        // (tokens of the digit's rows before and behind these count as one row there)
        const int64_t v = p < s1 ? (int64_t)(a.sorted[p] >> 32) - v0 : nv;
        const int64_t u = p > s0 ? (int64_t)(a.sorted[p - 1] >> 32) - v0 + 1 : 0;
        for (int r = (int)(u > 0 ? u : 0); r <= (v < nv ? v : nv); ++r) at[r] = (int32_t)p;
      }
    } else if ((int)threadIdx.x <= nv) {     // many: by halving
      int32_t lo = s0, hi = s1;
      const uint64_t want = (uint64_t)(v0 + threadIdx.x);
      while (lo < hi) {
        const int32_t mid = lo + (hi - lo) / 2;
        if (a.sorted[mid] >> 32 >= want) hi = mid;
        else lo = mid + 1;
      }
      at[threadIdx.x] = lo;
    }
    __syncthreads();
    // the tiles of a run; t0 = t1: it is written already.  No run: one less.
    if ((int)threadIdx.x < nv) {
      const uint32_t s = at[threadIdx.x], e = at[threadIdx.x + 1];
      t0[threadIdx.x] = (int32_t)(s / (uint32_t)a.tile);
      t1[threadIdx.x] = s < e ? (int32_t)((e - 1) / (uint32_t)a.tile) : (int32_t)(s / (uint32_t)a.tile) - 1;
    }
    __syncthreads();
    for (int i = g; i < nv && lives; i += groups) {
      const int b0 = t0[i], b1 = t1[i];
      if (b0 == b1 || b1 - b0 > kLight) continue;
      float acc[VEC] = {};
      for (int t = b0; t <= b1; ++t) {
        float x[VEC];
        load_params<T, float, TAIL>(part(t, t == b0 ? 1 : 0), f, a.C, x);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += x[j];
      }
      write(i, acc);
    }
    // long runs: the groups take their tiles in turn, four at a time, and add them in 64 bits (one token of 2,000,000 over 1,024
    // columns of fp32 is 15,625 tiles of one group: in 32 bits equal rows were off by 3,899 x 2^-24, now by 2 x 2^-24; one by one,
    // 512 columns of bf16, 1,493 us and now 836)
    for (int i = 0; i < nv; ++i) {
      const int b0 = t0[i], b1 = t1[i];
      if (b1 - b0 <= kLight) continue;       // (the same for all threads)
      double acc[VEC] = {};
      if (lives) {
        for (int t = b0 + g; t <= b1; t += 4 * groups) {
          float x[4][VEC];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int q = min(t + u * groups, b1);
            load_params<T, float, TAIL>(part(q, q == b0 ? 1 : 0), f, a.C, x[u]);
          }
#pragma unroll
          for (int u = 1; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < VEC; ++j) x[u][j] = t + u * groups <= b1 ? x[u][j] : 0.f;
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += (x[0][j] + x[1][j]) + (x[2][j] + x[3][j]);
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < VEC; ++j) join[threadIdx.x * VEC + j] = (float)acc[j];
      __syncthreads();
      if (g == 0 && lives) {
        for (int h = 1; h < groups; ++h)
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += join[(h * lpr + lane) * VEC + j];
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = (float)acc[j];
        write(i, o);
      }
    }
    __syncthreads();
  }
}

// ---- backward: which form, and its launches ---------------------------------------------------
struct Plan {
  bool local;
  int lpr, pieces, tiles;                    // lanes of a row in a column tile, pieces of a row, column tiles
  int chunk, chunks, range, ranges;          // local
  int span, tile, blocks;                    // sorted: positions of a group, of a workgroup, workgroups
  int passes, bits, sort_tile, sort_tiles;
  size_t part, sorted, hist, bytes;          // offsets of sorted and hist behind part; bytes altogether
};
static Plan plan_of(const EgnnEmbedDims* d) {
  Plan p{};
  const int64_t N = d->N, V = d->V;
  p.pieces = (int)cdiv(d->C, d->dtype == EGNN_F32 ? 4 : 8);
  const int64_t least = N ? cdiv(N, kChunk) : 1;
  // local: few tokens, or few rows (40,961 x 259 fp32 over 2,000 rows by 7 ranges and 8 column tiles 81 us, sorted 40;
  // 500,000 x 64 bf16 over 500 rows 39, sorted 76)
  p.local = least == 1 || (V <= kRange && least * V <= N / 2);
  if (p.local) {
    // Partial tables: at most half as many rows as there are tokens, and none up to 4,096 tokens.  Chunks of 256 tokens or more,
    // of 512 among many (100,000 x 128 bf16 over 119 rows, 21.4 and 19.5 us; 19,456 x 128 with the forward 16.2 and 16.6), and
    // up to 1,024 of them, which costs the wide rows less than it gives the narrow ones (2,000,000 x 128 over 119 rows 133 us, with
    // 512 chunks 129; x 32 over 8 rows 46, and 51)
    int64_t K = N <= 4096 ? 1 : N / (2 * V);
    const int64_t least_chunk = N <= 65536 ? 256 : 512;
    if (K > cdiv(N, least_chunk)) K = cdiv(N, least_chunk);
    if (K > 1024) K = 1024;
    if (K < least) K = least;
    p.chunk = (int)cdiv(cdiv(N ? N : 1, K), 64) * 64;
    p.chunks = (int)cdiv(N ? N : 1, p.chunk);
    // too few of them: column tiles, down to 128 bytes of a row, then ranges of the table
    p.tiles = (int)cdiv(p.pieces, 64);
    while (p.chunks * p.tiles < 512 && cdiv(p.pieces, 2 * p.tiles) >= 8) p.tiles *= 2;
    p.lpr = (int)cdiv(p.pieces, p.tiles);
    int64_t R = cdiv(512, (int64_t)p.chunks * p.tiles);
    if (R > V) R = V;
    if (R < cdiv(V, kRange)) R = cdiv(V, kRange);
    p.range = (int)cdiv(V, R);
    p.ranges = (int)cdiv(V, p.range);
    p.bytes = p.chunks > 1 ? (size_t)p.chunks * V * d->C * 4 : 0;
    return p;
  }
  p.tiles = (int)cdiv(p.pieces, 64);
  p.lpr = (int)cdiv(p.pieces, p.tiles);
  int width = 0;                             // bits of a key: 0 .. V
  while (V >> width) ++width;
  p.passes = (int)cdiv(width, 11);
  p.bits = (int)cdiv(width, p.passes);
  p.sort_tile = (int)(N > 256 * (int64_t)kSortTile ? kSortTile : cdiv(N, 256 * 512) * 512);
  p.sort_tiles = (int)cdiv(N, p.sort_tile);
  const int groups = BT / p.lpr;
  int64_t span = N / ((int64_t)groups * 1024) / 8 * 8;
  span = span < 8 ? 8 : span > 32 ? 32 : span;
  while (span > 4 && span * groups > 2048) span /= 2;
  while (cdiv(N, span * groups) > kMaxGrid && span * groups <= 1024) span *= 2;
  p.span = (int)span;
  p.tile = (int)span * groups;
  p.blocks = (int)cdiv(N, p.tile);
  p.part = align_up((size_t)p.blocks * 2 * d->C * 4);
  p.sorted = align_up((size_t)N * 8);
  p.hist = align_up(((size_t)p.sort_tiles + 1) * 4 << p.bits);
  p.bytes = p.part + 2 * p.sorted + p.hist;
  return p;
}

template <typename T, typename P, typename I, bool TAIL, bool PAST>
static int launch_bwd(BwdArgs a, const Plan& p, void* ws, hipStream_t st) {
  constexpr int VEC = Vec<T>::N;
  const size_t carry = (size_t)BT * 2 * VEC * 4;
  a.lpr = p.lpr; a.pieces = p.pieces;
  if (p.local) {
    a.chunk = p.chunk; a.chunks = p.chunks; a.range = p.range;
    a.part = p.chunks > 1 ? (float*)ws : nullptr;
    const size_t cnt = (size_t)NW * p.range * 4;
    const size_t lds = ((size_t)p.chunk + ((p.range + 4) & ~3)) * 4 + (cnt > carry ? cnt : carry) + (size_t)p.chunk * 2;
    const dim3 grid((uint32_t)(p.chunks * (int64_t)p.ranges), (uint32_t)p.tiles);
    local_kernel<T, P, I, TAIL, PAST><<<grid, BT, lds, st>>>(a);
    if (p.chunks > 1) {
      const int64_t M = a.V * a.C, pad = a.padding * a.C;
      reduce_kernel<P><<<(uint32_t)(cdiv(M, 64) < kMaxGrid ? cdiv(M, 64) : kMaxGrid), 1024, 0, st>>>(a.part, p.chunks, M, a.padding < 0 ? 0 : pad,
                                                                a.padding < 0 ? 0 : pad + a.C, a.scale, (P*)a.gw);
    }
    return hipGetLastError() == hipSuccess ? EGNN_OK : EGNN_ERR_HIP;
  }
  char* at = (char*)ws;
  a.part = (float*)at;
  uint64_t *one = (uint64_t*)(at + p.part), *two = (uint64_t*)(at + p.part + p.sorted);
  SortArgs s{};
  s.tokens = a.tokens; s.N = a.N; s.V = a.V; s.digits = 1 << p.bits; s.tile = p.sort_tile; s.tiles = p.sort_tiles;
  s.total = (uint32_t*)(at + p.part + 2 * p.sorted);
  s.hist = s.total + s.digits;
  for (int k = 0; k < p.passes; ++k) {
    s.shift = k * p.bits;
    s.from = k & 1 ? one : two;
    s.to = k & 1 ? two : one;
    const size_t lds = ((size_t)(2 + NW) * s.digits + 4) * 4 + (size_t)s.tile * 2;
    if (!k) hist_kernel<I, true><<<(uint32_t)s.tiles, BT, 0, st>>>(s);
    else hist_kernel<I, false><<<(uint32_t)s.tiles, BT, 0, st>>>(s);
    scan_kernel<<<(uint32_t)cdiv(s.digits, 16), 1024, 0, st>>>(s);
    if (!k) scatter_kernel<I, true><<<(uint32_t)s.tiles, BT, lds, st>>>(s);
    else scatter_kernel<I, false><<<(uint32_t)s.tiles, BT, lds, st>>>(s);
  }
  a.sorted = s.to;
  a.span = p.span; a.tile = p.tile;
  const size_t lds = ((size_t)((p.tile + 5) & ~3) + ((p.tile + 3) & ~3)) * 4 + carry;
  const dim3 grid((uint32_t)p.blocks, (uint32_t)p.tiles);
  sorted_kernel<T, P, TAIL, PAST><<<grid, BT, lds, st>>>(a);
  const int tiles = (int)cdiv(p.pieces, FT);   // wider column tiles than those of the sums: every one looks for the rows again
  a.lpr = (int)cdiv(p.pieces, tiles);
  // about four rows a group of lanes (40,961 x 259 fp32 over 50,021 rows, three groups: 66, 59, 56 and 61 us at 64, 32, 16 and 8
  // rows; 1,000,000 x 32 over 131,072, 32 groups: 112, 112, 119 and 132), fewer where the table is short; a power of two
  int rows = 8;
  while (rows < kFixRows && rows < 4 * (FT / a.lpr)) rows *= 2;
  while (rows > 1 && ((s.shift && rows > 1 << s.shift) || cdiv(a.V, rows) < 512)) rows /= 2;
  const int64_t fix = cdiv(a.V, rows);
  const dim3 fgrid((uint32_t)(fix < kMaxGrid / tiles ? fix : kMaxGrid / tiles), (uint32_t)tiles);
  fix_kernel<T, P, TAIL><<<fgrid, FT, 0, st>>>(a, s.total, s.shift, rows);
  return hipGetLastError() == hipSuccess ? EGNN_OK : EGNN_ERR_HIP;
}

static bool dims_ok(const EgnnEmbedDims* d) {
  return d->N >= 0 && d->N <= INT32_MAX && d->V >= 1 && d->C >= 1 && d->C <= 1 << 20 && (int64_t)d->V * d->C < int64_t(1) << 40 &&
         (d->dtype == EGNN_F32 || d->dtype == EGNN_BF16) && (d->f32_table == 0 || d->f32_table == 1) &&
         (d->index64 == 0 || d->index64 == 1) && d->scale - d->scale == 0.f;
}
template <template <typename, typename, typename> class Go, typename... A>
static auto by_type(const EgnnEmbedDims* d, A... args) {
  if (d->dtype == EGNN_F32)
    return d->index64 ? Go<float, float, int64_t>::go(args...) : Go<float, float, int32_t>::go(args...);
  if (d->f32_table) return d->index64 ? Go<bf16, float, int64_t>::go(args...) : Go<bf16, float, int32_t>::go(args...);
  return d->index64 ? Go<bf16, bf16, int64_t>::go(args...) : Go<bf16, bf16, int32_t>::go(args...);
}
template <typename T, typename P, typename I> struct Fwd {
  static int go(const FwdArgs& a, hipStream_t st) {
    if (a.C % Vec<T>::N) launch_fwd<T, P, I, true>(a, st);
    else launch_fwd<T, P, I, false>(a, st);
    return hipGetLastError() == hipSuccess ? EGNN_OK : EGNN_ERR_HIP;
  }
};
template <typename T, typename P, typename I> struct Bwd {
  static int go(const BwdArgs& a, const Plan* p, void* ws, hipStream_t st) {
    if (a.N * a.C * (int64_t)sizeof(T) >= kPastLoad)
      return a.C % Vec<T>::N ? launch_bwd<T, P, I, true, true>(a, *p, ws, st) : launch_bwd<T, P, I, false, true>(a, *p, ws, st);
    return a.C % Vec<T>::N ? launch_bwd<T, P, I, true, false>(a, *p, ws, st) : launch_bwd<T, P, I, false, false>(a, *p, ws, st);
  }
};

}  // namespace embed
}  // namespace egnn

using namespace egnn::embed;

extern "C" {

int32_t egnn_embed_fwd(const EgnnEmbedDims* d, const void* tokens, const void* weight, int64_t ldw, void* out, void* stream) {
  if (!d) return EGNN_ERR_NULL;
  if (!dims_ok(d)) return EGNN_ERR_DIMS;
  if (d->N && (!tokens || !weight || !out)) return EGNN_ERR_NULL;
  if (ldw < 0) return EGNN_ERR_STRIDE;
  const uintptr_t e = d->dtype == EGNN_F32 ? 4 : 2, ep = d->f32_table ? 4 : e, ei = d->index64 ? 8 : 4;
  if ((uintptr_t)tokens % ei || (uintptr_t)weight % ep || (uintptr_t)out % e) return EGNN_ERR_ALIGN;
  if (!d->N) return EGNN_OK;
  FwdArgs a{};
  a.tokens = tokens; a.w = weight; a.out = out; a.N = d->N; a.V = d->V; a.ldw = ldw; a.C = d->C; a.scale = d->scale;
  return by_type<Fwd>(d, a, (hipStream_t)stream);
}

size_t egnn_embed_bwd_workspace_bytes(const EgnnEmbedDims* d) { return d && dims_ok(d) ? plan_of(d).bytes : 0; }

int32_t egnn_embed_bwd(const EgnnEmbedDims* d, int64_t padding, const void* grad_out, int64_t ldg, const void* tokens,
                       void* grad_weight, void* workspace, size_t workspace_bytes, void* stream) {
  if (!d) return EGNN_ERR_NULL;
  if (!dims_ok(d) || padding < -1 || padding >= d->V) return EGNN_ERR_DIMS;
  if (!grad_weight || (d->N && (!tokens || !grad_out))) return EGNN_ERR_NULL;
  if (ldg < 0) return EGNN_ERR_STRIDE;
  const uintptr_t e = d->dtype == EGNN_F32 ? 4 : 2, ep = d->f32_table ? 4 : e, ei = d->index64 ? 8 : 4;
  if ((uintptr_t)tokens % ei || (uintptr_t)grad_weight % ep || (uintptr_t)grad_out % e || (uintptr_t)workspace % 16)
    return EGNN_ERR_ALIGN;
  const Plan p = plan_of(d);
  if (p.bytes && (!workspace || workspace_bytes < p.bytes)) return EGNN_ERR_WORKSPACE;
  BwdArgs a{};
  a.tokens = tokens; a.g = grad_out; a.gw = grad_weight; a.N = d->N; a.V = d->V; a.ldg = ldg; a.padding = padding;
  a.C = d->C; a.scale = d->scale;
  return by_type<Bwd>(d, a, &p, workspace, (hipStream_t)stream);
}

}  // extern "C"
