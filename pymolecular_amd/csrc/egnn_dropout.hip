// Dropout of rows, with the residual sum behind it:  y = (residual +) keep ? up x : 0,  the mask of egnn_random.h.
// The backward is the same kernel on the gradient: gx = keep ? up gy : 0 (the residual's gradient is gy itself).
// A thread makes the 128 bits of eight columns and takes their values with them; in large calls four such groups at once, whose
// loads are on their way while the bits are made.  Bound by HBM: 2,000,000 x 128 bf16 168 us alone and 252 with a residual, 6.1 TB/s,
// with the vector units busy 0.62 and 0.51 of the time (the generator's products run at a quarter of their rate); 2,432 x 128
// fp32 2.7 us, a launch.
#include "egnn_internal.h"
#include "egnn_random.h"
#include "egnn_rows.h"

namespace egnn {
namespace dropout {

constexpr int NT = 256;

struct Args {
  const void *x, *r;
  void* y;
  int64_t N, row0, ldx, ldr;
  int32_t C, G, GT, R;                       // columns, groups in a row, groups in a tile of it, rows in a block
  uint32_t magic;                            // l / GT = the high word of l magic (GT > 1)
  DropArgs d;
};

template <typename T> struct Group {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  typedef T vals __attribute__((ext_vector_type(8)));
  template <bool PAST> static __device__ __forceinline__ vals load(const T* p, int n) {
    vals v;
    if (n >= 8) {
      if constexpr (PAST) v = __builtin_nontemporal_load(reinterpret_cast<const type*>(p));
      else v = *reinterpret_cast<const type*>(p);
    } else
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : (T)0.f;
    return v;
  }
  template <bool PAST> static __device__ __forceinline__ void store(T* p, int n, const float* v) {
    if (n >= 8) {
      type t;
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(v[i]);
      if constexpr (PAST) __builtin_nontemporal_store(t, reinterpret_cast<type*>(p));
      else *reinterpret_cast<type*>(p) = t;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = from_f32<T>(v[i]);
    }
  }
};

// U: groups of eight columns a thread; PAST: 1: the result is stored past the cache, 2: the operands are read past it too
template <typename T, bool RES, int U, int PAST>
__global__ __launch_bounds__(NT) void drop_kernel(Args a) {
  typedef Group<T> V;
  const Mask m = mask_of(a.d);
  typename V::vals x[U], r[U];
  int64_t n[U];
  int g[U];
  bool in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t l = u * NT + threadIdx.x;
    const uint32_t k = a.GT > 1 ? __umulhi(l, a.magic) : l;
    n[u] = (int64_t)blockIdx.x * a.R + k;
    g[u] = (int)(l - k * a.GT) + blockIdx.y * a.GT;
    in[u] = (int)k < a.R && n[u] < a.N && g[u] < a.G;
    if (in[u]) {
      x[u] = V::template load<PAST == 2>((const T*)a.x + n[u] * a.ldx + 8 * g[u], a.C - 8 * g[u]);
      if (RES) r[u] = V::template load<PAST == 2>((const T*)a.r + n[u] * a.ldr + 8 * g[u], a.C - 8 * g[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!in[u]) continue;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32((T)x[u][i]);
    drop<8, false>(m, (uint32_t)(a.row0 + n[u]), 8 * g[u], v);
    if (RES) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += to_f32((T)r[u][i]);
    }
    V::template store<(PAST > 0)>((T*)a.y + n[u] * a.C + 8 * g[u], a.C - 8 * g[u], v);
  }
}

// Up to so many groups a thread takes one: more workgroups come before more loads in flight (2,432 x 128 fp32: 3.5 us, and 4.1
// with four; 32,768 x 128 bf16: 4.2 and 5.1; at 1,048,576 groups the same)
constexpr int64_t kFewGroups = 1024 * 1024;
// A launch may have fewer than 2^32 threads: at most this many blocks at a time
constexpr int64_t kMaxGrid = int64_t(1) << 20;

template <typename T, int U, int PAST>
static void launch_parts(Args a, hipStream_t st) {
  a.G = (int32_t)cdiv(a.C, 8);
  const int tiles = (int)cdiv(a.G, NT * U);
  a.GT = (int32_t)cdiv(a.G, tiles);
  a.R = NT * U / a.GT;
  a.magic = a.GT > 1 ? (uint32_t)(((uint64_t(1) << 32) + a.GT - 1) / a.GT) : 0;
  const int64_t most = kMaxGrid / tiles * a.R, N = a.N;
  const Args all = a;
  for (int64_t n = 0; n < N; n += most) {
    a.x = (const T*)all.x + n * a.ldx;
    a.r = all.r ? (const T*)all.r + n * a.ldr : nullptr;
    a.y = (T*)all.y + n * a.C;
    a.row0 = n;
    a.N = N - n < most ? N - n : most;
    const dim3 grid((uint32_t)cdiv(a.N, a.R), (uint32_t)tiles);
    if (a.r) drop_kernel<T, true, U, PAST><<<grid, NT, 0, st>>>(a);
    else drop_kernel<T, false, U, PAST><<<grid, NT, 0, st>>>(a);
  }
}
// Past the cache: 600,000 x 128 bf16, with a residual, 84.4 us at 0 and 70.7 at 1; 2,000,000 x 128 271 at 0, 249 at 2.  A
// group of fp32 is two loads of half a line each, which are slower past the cache where it holds nothing anyway: 1,000,000 x
// 128, 271, 277 and 288 at 0, 1 and 2; 150,000 x 259, 96 and 89 at 0 and 1.
template <typename T>
static void launch(const Args& a, hipStream_t st) {
  const int64_t bytes = a.N * a.C * (int64_t)sizeof(T);
  if (a.N * cdiv(a.C, 8) < kFewGroups) launch_parts<T, 1, 0>(a, st);
  else if (bytes < kPastStore) launch_parts<T, 4, 0>(a, st);
  else if (bytes < kPastLoad) launch_parts<T, 4, 1>(a, st);
  else launch_parts<T, 4, sizeof(T) == 2 ? 2 : 0>(a, st);
}

}  // namespace dropout
}  // namespace egnn

extern "C" int32_t egnn_dropout(const EgnnDropout* drop, int32_t dtype, int64_t N, int32_t C, const void* x, int64_t ldx,
                                const void* residual, int64_t ldr, void* y, void* stream) {
  using namespace egnn;
  if (!drop) return EGNN_ERR_NULL;
  if (N < 0 || N > INT32_MAX || C < 1 || C > 1 << 20 || (dtype != EGNN_F32 && dtype != EGNN_BF16) || !drop_ok(drop))
    return EGNN_ERR_DIMS;
  if (!drop->rng || (N && (!x || !y))) return EGNN_ERR_NULL;
  if (ldx < 0 || (residual && ldr < 0)) return EGNN_ERR_STRIDE;
  const uintptr_t e = dtype == EGNN_F32 ? 4 : 2;
  if ((uintptr_t)x % e || (uintptr_t)residual % e || (uintptr_t)y % e || (uintptr_t)drop->rng % 8) return EGNN_ERR_ALIGN;
  if (!N) return EGNN_OK;
  dropout::Args a{};
  a.x = x; a.ldx = ldx; a.r = residual; a.ldr = ldr; a.y = y; a.N = N; a.C = C; a.d = drop_args(drop);
  if (dtype == EGNN_BF16) dropout::launch<bf16>(a, (hipStream_t)stream);
  else dropout::launch<float>(a, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? EGNN_OK : EGNN_ERR_HIP;
}
