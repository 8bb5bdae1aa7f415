// Orthogonalised updates by Newton-Schulz products, and the Muon step of a weight around them.
//
//   U = G, or for the optimiser  M <- mu M + (1 - mu) G,  U = (1 - mu) G + mu M  (Nesterov) or U = M
//   X = U / (|U|_F + eps), its short side first (m <= n);  `steps` times:  S = X X^T,  X <- a X + (b S + c S S) X
//   out = X, or  W <- (1 - lr decay) W - lr gain X
//
// Products run on the fp16 matrix instructions with fp32 accuracy: an operand is two fp16 pieces, x = hi + lo (22 bits and a
// sign, of values scaled so that nothing overflows), a product three matrix instructions, hi hi + hi lo + lo hi, summed in
// fp32; what is left out is 2^-24 of a term.  Operands lie in memory in the order of the instruction's registers: a tile of
// 16 rows x 32 inner values is 1 KB of hi pieces and 1 KB of lo pieces, lane l's 8 values (row l % 16, inner values
// 8 (l / 16) ..) at 16 l, so a wave loads one operand of one instruction as one contiguous 1 KB, and tiles that follow each
// other along the inner dimension lie next to each other.
#include <hip/hip_runtime.h>
#include <cmath>
#include <cstdint>

#include "kan_launch.h"
#include "kan_wave.h"

namespace pdekan {
namespace {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kItemsMax = kNsItemsMax;    // matrices (or stacks of equal ones) a launch
constexpr int kSumsMax = 256;             // partial sums of squares a matrix
constexpr int kTileHalves = 1024;         // a 16 x 32 tile: 512 hi pieces, 512 lo pieces

// One matrix, or a stack of `batch` equal ones, and its share of the workspace.
struct Item {
  const void* src;        // G; the optimiser's gradient
  float* mom;             // momentum, or nullptr
  void* out;              // X; the optimiser's weight
  char* ws;
  int64_t ws_stride;      // bytes a matrix
  int64_t size;           // rows * cols
  int rows, cols, m, n, mp, np, batch, tall;
  int nsum;               // partial sums of squares
  int chunks, kchunk;     // splits of the long axis in X X^T, inner tiles (of 32) a split
  float gain;
};
struct Items {
  Item it[kItemsMax];
  int first[kItemsMax + 1];               // first block of each item in this launch
  int n;
};

// workspace of a matrix: X [mp][np], X^T twice [np][mp], S and R [mp][mp] as two-piece tiles, then the splits' partial
// products and the partial sums of squares
__device__ __host__ inline int64_t plane_bytes(const Item& I) { return (int64_t)I.mp * I.np * 4; }
__device__ __host__ inline int64_t square_bytes(const Item& I) { return (int64_t)I.mp * I.mp * 4; }
__device__ __host__ inline int64_t off_xt(const Item& I, int k) { return plane_bytes(I) * (1 + k); }
__device__ __host__ inline int64_t off_s(const Item& I) { return plane_bytes(I) * 3; }
__device__ __host__ inline int64_t off_r(const Item& I) { return off_s(I) + square_bytes(I); }
__device__ __host__ inline int64_t off_part(const Item& I) { return off_r(I) + square_bytes(I); }
__device__ __host__ inline int tri_tiles(const Item& I) { const int t = (I.mp + 63) / 64; return t * (t + 1) / 2; }
__device__ __host__ inline int64_t off_sums(const Item& I) {
  if (I.m == 1) return 0;                 // a vector has nothing else
  return off_part(I) + (I.chunks > 1 ? (int64_t)I.chunks * tri_tiles(I) * 64 * 64 * 4 : 0);
}
__device__ __host__ inline int64_t item_bytes(const Item& I) {
  return (off_sums(I) + kSumsMax * (int64_t)sizeof(double) + 8 + 255) / 256 * 256;      // (8: the exponent, see x_scale)
}

struct Where { int item, local; };
__device__ __forceinline__ Where find_item(const Items& L) {
  int k = 0;
  while (k + 1 < L.n && (int)blockIdx.x >= L.first[k + 1]) ++k;
  return {k, (int)blockIdx.x - L.first[k]};
}

// (row, column) of the t-th tile of the upper triangle, columns first: (0,0) (0,1) (1,1) (0,2) ...
__device__ __forceinline__ void tri_tile(int t, int& bi, int& bj) {
  bj = (int)((__builtin_sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
  while (bj * (bj + 1) / 2 > t) --bj;
  while ((bj + 1) * (bj + 2) / 2 <= t) ++bj;
  bi = t - bj * (bj + 1) / 2;
}

// ---- exponents of the pieces --------------------------------------------------------------------------------------
// X has no singular value over the host's bound 2^kx, S none over 2^(2 kx), R none over 2^kr; entries are bounded alike, and
// pieces are scaled by powers of two to stay below 2^15.  Where eps dominates |U|_F, X starts as small as |U| / eps and its
// pieces are scaled up by 2^ex0 more, ex0 = the exponent of (|U| + eps) / |U|; a step multiplies X by at most 2^growth, so
// step k has 2^max(0, ex0 - growth k).
struct Scales { float x, s, r; int growth; };          // what the entries of X, S, R are multiplied by

__device__ __forceinline__ int* exponent_slot(const Item& I, char* ws) {
  return reinterpret_cast<int*>(ws + off_sums(I) + kSumsMax * (int64_t)sizeof(double));
}
__device__ __forceinline__ float x_scale(const Item& I, char* ws, const Scales& sc, int step) {
  const int ex = *exponent_slot(I, ws) - sc.growth * step;
  return ldexpf(sc.x, ex > 0 ? ex : 0);
}

// two pieces of four values
__device__ __forceinline__ void split4(const float (&v)[4], float scale, f16x4& hi, f16x4& lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y = v[i] * scale;
    hi[i] = (_Float16)y;
    lo[i] = (_Float16)(y - (float)hi[i]);
  }
}
// halves offset of (row, col) of a matrix with kt inner tiles a row of tiles; col % 4 == 0 addresses four values
__device__ __forceinline__ int64_t piece_at(int row, int col, int kt) {
  return ((int64_t)(row >> 4) * kt + (col >> 5)) * kTileHalves + ((row & 15) + 16 * ((col & 31) >> 3)) * 8 + (col & 7);
}
__device__ __forceinline__ void store_pieces(_Float16* base, int row, int col, int kt, const float (&v)[4], float scale) {
  f16x4 hi, lo;
  split4(v, scale, hi, lo);
  _Float16* p = base + piece_at(row, col, kt);
  *reinterpret_cast<f16x4*>(p) = hi;
  *reinterpret_cast<f16x4*>(p + 512) = lo;
}
__device__ __forceinline__ void load_pieces(const _Float16* base, int row, int col, int kt, float (&v)[4], float unscale) {
  const _Float16* p = base + piece_at(row, col, kt);
  const f16x4 hi = *reinterpret_cast<const f16x4*>(p), lo = *reinterpret_cast<const f16x4*>(p + 512);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = ((float)hi[i] + (float)lo[i]) * unscale;
}

// v[r] of lane t of a quad -> v[t] of lane r
__device__ __forceinline__ void quad_transpose(float (&v)[4]) {
  const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
  const float a = dpp_move<0xB1>(odd ? v[0] : v[1]), b = dpp_move<0xB1>(odd ? v[2] : v[3]);
  v[0] = odd ? a : v[0]; v[1] = odd ? v[1] : a;
  v[2] = odd ? b : v[2]; v[3] = odd ? v[3] : b;
  const float c = dpp_move<0x4E>(high ? v[0] : v[2]), d = dpp_move<0x4E>(high ? v[1] : v[3]);
  v[0] = high ? c : v[0]; v[2] = high ? v[2] : c;
  v[1] = high ? d : v[1]; v[3] = high ? v[3] : d;
}

// ---- U and its norm -------------------------------------------------------------------------------------------------

struct Momentum { float mu; int nesterov; };

template <typename T>
__device__ __forceinline__ float source_value(const Item& I, int64_t at, const Momentum& mo) {
  const float g = (float)static_cast<const T*>(I.src)[at];
  if (!I.mom) return g;
  const float m = I.mom[at];
  return mo.nesterov ? (1.0f - mo.mu) * g + mo.mu * m : m;
}

// Partial sums of squares of U in 64 bits (the squares of gradients as small as 1e-25 vanish in 32), one a block; the
// optimiser's momentum is updated on the way.
template <typename T>
__global__ void __launch_bounds__(kThreads) ns_norm_kernel(Items L, Momentum mo) {
  __shared__ double red[kThreads / 64];
  const Where w = find_item(L);
  const Item& I = L.it[w.item];
  const int b = w.local / I.nsum, part = w.local % I.nsum;
  const int64_t base = b * I.size;
  double s = 0.0;
  for (int64_t i = (int64_t)part * kThreads + threadIdx.x; i < I.size; i += (int64_t)I.nsum * kThreads) {
    if (I.mom) {
      const float g = (float)static_cast<const T*>(I.src)[base + i];
      I.mom[base + i] = fmaf(mo.mu, I.mom[base + i], (1.0f - mo.mu) * g);
    }
    const double u = source_value<T>(I, base + i, mo);
    s = fma(u, u, s);
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < kThreads / 64; ++k) s += red[k];
    reinterpret_cast<double*>(I.ws + b * I.ws_stride + off_sums(I))[part] = s;
  }
}

// |U|_F of a matrix from its partial sums, in every thread (one wave or more a block)
__device__ __forceinline__ double matrix_norm(const Item& I, int b) {
  const double* sums = reinterpret_cast<const double*>(I.ws + b * I.ws_stride + off_sums(I));
  double s = 0.0;
  for (int k = threadIdx.x & 63; k < I.nsum; k += 64) s += sums[k];
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
  return sqrt(s);
}

// X and X^T of a 64 x 64 tile as pieces.
template <typename T>
__global__ void __launch_bounds__(kThreads) ns_split_kernel(Items L, Momentum mo, float eps, Scales sc) {
  __shared__ float tile[64][65];
  const Where w = find_item(L);
  const Item& I = L.it[w.item];
  const int tm = (I.mp + 63) / 64, tn = (I.np + 63) / 64;
  const int b = w.local / (tm * tn), t = w.local % (tm * tn), bi = t % tm, bj = t / tm;
  const int64_t base = b * I.size;
  const double norm = matrix_norm(I, b);
  const float scale = (float)(1.0 / (norm + (double)eps));
  // at most 2^96: entries below 2^-96 |X| lose their low bits; (NaN and 0 norms: no shift)
  const double small = (norm + (double)eps) / norm;
  const int ex0 = small > 1.0 && norm > 0.0 ? (small < 7.9e28 ? ilogb(small) : 96) : 0;
  if (t == 0 && threadIdx.x == 0) *exponent_slot(I, I.ws + b * I.ws_stride) = ex0;
  const float scx = ldexpf(sc.x, ex0);
  for (int k = threadIdx.x; k < 64 * 64; k += kThreads) {
    // neighbouring threads on neighbouring addresses
    const int a = k / 64, c = k % 64;
    const int li = I.tall ? c : a, lj = I.tall ? a : c;
    const int i = bi * 64 + li, j = bj * 64 + lj;
    float v = 0.0f;
    if (i < I.m && j < I.n) v = source_value<T>(I, base + (I.tall ? (int64_t)j * I.m + i : (int64_t)i * I.n + j), mo) * scale;
    tile[li][lj] = v;
  }
  __syncthreads();
  char* ws = I.ws + b * I.ws_stride;
  _Float16 *x = reinterpret_cast<_Float16*>(ws), *xt = reinterpret_cast<_Float16*>(ws + off_xt(I, 0));
  const int ktx = I.np / 32, kt = I.mp / 32;
  for (int k = threadIdx.x; k < 64 * 16; k += kThreads) {
    const int r = k % 64, q = k / 64 * 4;
    const int i = bi * 64 + r, j = bj * 64 + q;
    if (i < I.mp && j < I.np) {
      const float v[4] = {tile[r][q], tile[r][q + 1], tile[r][q + 2], tile[r][q + 3]};
      store_pieces(x, i, j, ktx, v, scx);
    }
    const int i2 = bi * 64 + q, j2 = bj * 64 + r;
    if (i2 < I.mp && j2 < I.np) {
      const float v[4] = {tile[q][r], tile[q + 1][r], tile[q + 2][r], tile[q + 3][r]};
      store_pieces(xt, j2, i2, kt, v, scx);
    }
  }
}

// ---- products -------------------------------------------------------------------------------------------------------

// A wave's 32 x 32 share of a 64 x 64 block of P Q^T over inner tiles [k0, k1): acc[a][c] is the 16 x 16 block at rows
// 16 a of P and 16 c of Q; lane l holds Q's row l % 16 and P's rows 4 (l / 16) + r.
struct Acc { f32x4 v[2][2]; };
__device__ __forceinline__ void product(const _Float16* P, const _Float16* Q, int rp, int rq, int prows, int qrows, int kt,
                                        int k0, int k1, Acc& acc) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int c = 0; c < 2; ++c) acc.v[a][c] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  for (int k = k0; k < k1; ++k) {
    f16x8 ph[2], pl[2], qh[2], ql[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      // tiles past the padded matrix repeat its last one; what they give is never stored
      const int tp = min(rp / 16 + a, prows / 16 - 1), tq = min(rq / 16 + a, qrows / 16 - 1);
      const _Float16* p = P + ((int64_t)tp * kt + k) * kTileHalves + lane * 8;
      const _Float16* q = Q + ((int64_t)tq * kt + k) * kTileHalves + lane * 8;
      ph[a] = *reinterpret_cast<const f16x8*>(p);
      pl[a] = *reinterpret_cast<const f16x8*>(p + 512);
      qh[a] = *reinterpret_cast<const f16x8*>(q);
      ql[a] = *reinterpret_cast<const f16x8*>(q + 512);
    }
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        acc.v[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[a], qh[c], acc.v[a][c], 0, 0, 0);
        acc.v[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[a], ql[c], acc.v[a][c], 0, 0, 0);
        acc.v[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[a], qh[c], acc.v[a][c], 0, 0, 0);
      }
  }
}

// The symmetric m x m result of a wave: both triangles from one, blocks on the diagonal as they are.
__device__ __forceinline__ void store_symmetric(_Float16* S, int mp, int bi, int bj, int rp, int rq, const Acc& acc,
                                                float scale) {
  const int lane = threadIdx.x & 63, kt = mp / 32;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int p0 = rp + 16 * a, q0 = rq + 16 * c;
      if (p0 >= mp || q0 >= mp) continue;
      float v[4] = {acc.v[a][c][0], acc.v[a][c][1], acc.v[a][c][2], acc.v[a][c][3]};
      store_pieces(S, q0 + (lane & 15), p0 + 4 * (lane >> 4), kt, v, scale);
      if (bi != bj) {
        quad_transpose(v);
        store_pieces(S, p0 + 4 * (lane >> 4) + (lane & 3), q0 + (lane & 12), kt, v, scale);
      }
    }
}

// S = X X^T: block = (split of the long axis, tile of the upper triangle)
__global__ void __launch_bounds__(kThreads) ns_gram_kernel(Items L, Scales sc, int step) {
  const Where w = find_item(L);
  const Item& I = L.it[w.item];
  const int tiles = tri_tiles(I), per = tiles * I.chunks;
  const int b = w.local / per, rest = w.local % per, chunk = rest / tiles, t = rest % tiles;
  int bi, bj;
  tri_tile(t, bi, bj);
  char* ws = I.ws + b * I.ws_stride;
  const _Float16* x = reinterpret_cast<const _Float16*>(ws);
  const int wave = threadIdx.x >> 6, rp = bi * 64 + 32 * (wave & 1), rq = bj * 64 + 32 * (wave >> 1);
  const int kt = I.np / 32, k0 = chunk * I.kchunk, k1 = min(k0 + I.kchunk, kt);
  Acc acc;
  product(x, x, rp, rq, I.mp, I.mp, kt, k0, k1, acc);
  const float scx = x_scale(I, ws, sc, step), unscale = 1.0f / scx / scx;
  if (I.chunks == 1) {
    store_symmetric(reinterpret_cast<_Float16*>(ws + off_s(I)), I.mp, bi, bj, rp, rq, acc, unscale * sc.s);
    return;
  }
  f32x4* part = reinterpret_cast<f32x4*>(ws + off_part(I)) + ((int64_t)chunk * tiles + t) * 1024 + threadIdx.x;
#pragma unroll
  for (int a = 0; a < 4; ++a) part[a * kThreads] = acc.v[a >> 1][a & 1] * unscale;
}

// the sum of the splits, in their order
__global__ void __launch_bounds__(kThreads) ns_gram_sum_kernel(Items L, Scales sc) {
  const Where w = find_item(L);
  const Item& I = L.it[w.item];
  const int tiles = tri_tiles(I), b = w.local / tiles, t = w.local % tiles;
  int bi, bj;
  tri_tile(t, bi, bj);
  char* ws = I.ws + b * I.ws_stride;
  const f32x4* part = reinterpret_cast<const f32x4*>(ws + off_part(I)) + (int64_t)t * 1024 + threadIdx.x;
  Acc acc;
#pragma unroll
  for (int a = 0; a < 4; ++a) acc.v[a >> 1][a & 1] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  for (int k = 0; k < I.chunks; ++k)
#pragma unroll
    for (int a = 0; a < 4; ++a) acc.v[a >> 1][a & 1] += part[(int64_t)k * tiles * 1024 + a * kThreads];
  const int wave = threadIdx.x >> 6;
  store_symmetric(reinterpret_cast<_Float16*>(ws + off_s(I)), I.mp, bi, bj, bi * 64 + 32 * (wave & 1),
                  bj * 64 + 32 * (wave >> 1), acc, sc.s);
}

// R = b S + c S S
__global__ void __launch_bounds__(kThreads) ns_poly_kernel(Items L, Scales sc, float cb, float cc) {
  const Where w = find_item(L);
  const Item& I = L.it[w.item];
  const int tiles = tri_tiles(I), b = w.local / tiles, t = w.local % tiles;
  int bi, bj;
  tri_tile(t, bi, bj);
  char* ws = I.ws + b * I.ws_stride;
  const _Float16* s = reinterpret_cast<const _Float16*>(ws + off_s(I));
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, kt = I.mp / 32;
  const int rp = bi * 64 + 32 * (wave & 1), rq = bj * 64 + 32 * (wave >> 1);
  Acc acc;
  product(s, s, rp, rq, I.mp, I.mp, kt, 0, kt, acc);
  const float unscale = 1.0f / sc.s;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int p0 = rp + 16 * a, q0 = rq + 16 * c;
      if (p0 >= I.mp || q0 >= I.mp) continue;
      float v[4];
      load_pieces(s, q0 + (lane & 15), p0 + 4 * (lane >> 4), kt, v, unscale);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc.v[a][c][r] = fmaf(cc * unscale * unscale, acc.v[a][c][r], cb * v[r]);
    }
  store_symmetric(reinterpret_cast<_Float16*>(ws + off_r(I)), I.mp, bi, bj, rp, rq, acc, sc.r);
}

struct Finish { const float* lr_dev; float lr, decay; };

// what becomes of value x at element `at` of the matrix
template <typename T>
__device__ __forceinline__ void put(const Item& I, int64_t at, float x, float lr, const Finish& f) {
  T* out = static_cast<T*>(I.out);
  if (I.mom) out[at] = (T)fmaf((float)out[at], fmaf(-lr, f.decay, 1.0f), -(lr * I.gain) * x);
  else out[at] = (T)x;
}

// X <- a X + R X, computed as X^T <- a X^T + X^T R: block = 64 of the long axis x 64 of the short; the last step writes the
// result instead
template <typename T, bool LAST>
__global__ void __launch_bounds__(kThreads) ns_update_kernel(Items L, Scales sc, float ca, int step, Finish f) {
  const int from = step & 1;
  const Where w = find_item(L);
  const Item& I = L.it[w.item];
  const int tm = (I.mp + 63) / 64, tn = (I.np + 63) / 64;
  const int b = w.local / (tm * tn), t = w.local % (tm * tn), bi = t % tm, bj = t / tm;
  char* ws = I.ws + b * I.ws_stride;
  const _Float16* xt = reinterpret_cast<const _Float16*>(ws + off_xt(I, from));
  const _Float16* rm = reinterpret_cast<const _Float16*>(ws + off_r(I));
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, kt = I.mp / 32;
  const int rj = bj * 64 + 32 * (wave & 1), ri = bi * 64 + 32 * (wave >> 1);
  Acc acc;
  product(xt, rm, rj, ri, I.np, I.mp, kt, 0, kt, acc);
  const float scx = x_scale(I, ws, sc, step), next = x_scale(I, ws, sc, step + 1);
  const float unscale = 1.0f / scx / sc.r, own = ca / scx;
  const float lr = f.lr_dev ? *f.lr_dev : f.lr;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int j0 = rj + 16 * a, i0 = ri + 16 * c;
      if (j0 >= I.np || i0 >= I.mp) continue;
      // after the transpose lane l holds row j0 + 4 (l / 16) + l % 4 of X^T, columns i0 + (l & 12) ..
      float v[4], o[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = acc.v[a][c][r] * unscale;
      quad_transpose(v);
      const int j = j0 + 4 * (lane >> 4) + (lane & 3), i = i0 + (lane & 12);
      load_pieces(xt, j, i, kt, o, own);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += o[r];
      if constexpr (!LAST) {
        store_pieces(reinterpret_cast<_Float16*>(ws + off_xt(I, from ^ 1)), j, i, kt, v, next);
        quad_transpose(v);
        store_pieces(reinterpret_cast<_Float16*>(ws), i0 + (lane & 15), j0 + 4 * (lane >> 4), I.np / 32, v, next);
      } else if (I.tall) {
        if (j < I.n) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (i + r < I.m) put<T>(I, b * I.size + (int64_t)j * I.m + i + r, v[r], lr, f);
        }
      } else {
        quad_transpose(v);
        const int jj = j0 + 4 * (lane >> 4), ii = i0 + (lane & 15);
        if (ii < I.m) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (jj + r < I.n) put<T>(I, b * I.size + (int64_t)ii * I.n + jj + r, v[r], lr, f);
        }
      }
    }
}

// A matrix of one row (a vector): S is the number s = |X|^2 and X keeps its direction, so the whole iteration is one factor.
template <typename T>
__global__ void __launch_bounds__(kThreads) ns_vector_kernel(Items L, Momentum mo, float eps, NsCoefficients k, int steps,
                                                             Finish f) {
  const Where w = find_item(L);
  const Item& I = L.it[w.item];
  const int b = w.local / I.nsum, part = w.local % I.nsum;
  const double norm = matrix_norm(I, b);
  double factor = 1.0 / (norm + (double)eps), length = norm * factor;
  for (int i = 0; i < steps; ++i) {
    const double s = length * length, q = k.a + s * ((double)k.b + k.c * s);
    factor *= q;
    length *= q;
  }
  const float lr = f.lr_dev ? *f.lr_dev : f.lr;
  const int64_t base = b * I.size;
  for (int64_t i = (int64_t)part * kThreads + threadIdx.x; i < I.size; i += (int64_t)I.nsum * kThreads)
    put<T>(I, base + i, (float)((double)source_value<T>(I, base + i, mo) * factor), lr, f);
}

// ---- host -----------------------------------------------------------------------------------------------------------

int round_up(int64_t v, int a) { return (int)((v + a - 1) / a * a); }

Item make_item(const NsMatrix& M) {
  Item I{};
  I.src = M.src; I.mom = M.momentum; I.out = M.out; I.gain = M.gain;
  I.rows = (int)M.rows; I.cols = (int)M.cols; I.batch = (int)M.batch;
  I.tall = M.rows > M.cols;
  I.m = I.tall ? I.cols : I.rows;
  I.n = I.tall ? I.rows : I.cols;
  I.mp = round_up(I.m, 32);
  I.np = round_up(I.n, 32);
  I.size = M.rows * M.cols;
  const int64_t parts = (I.size + kThreads * 16 - 1) / (kThreads * 16);
  I.nsum = (int)(parts < kSumsMax ? parts : kSumsMax);
  // splits of the long axis: enough blocks for the card, at least four inner tiles each
  const int kt = I.np / 32, tiles = tri_tiles(I);
  int64_t chunks = (512 + (int64_t)tiles * I.batch - 1) / ((int64_t)tiles * I.batch);
  if (chunks > kt / 4) chunks = kt / 4;
  if (chunks < 1) chunks = 1;
  I.kchunk = (kt + (int)chunks - 1) / (int)chunks;
  I.chunks = (kt + I.kchunk - 1) / I.kchunk;
  I.ws_stride = I.m == 1 ? (int64_t)kSumsMax * (int64_t)sizeof(double) : item_bytes(I);
  return I;
}

int blocks_before(Items& L, int (*count)(const Item&)) {
  int total = 0;
  for (int i = 0; i < L.n; ++i) { L.first[i] = total; total += count(L.it[i]) * L.it[i].batch; }
  L.first[L.n] = total;
  return total;
}
int count_sums(const Item& I) { return I.nsum; }
int count_tiles(const Item& I) { return ((I.mp + 63) / 64) * ((I.np + 63) / 64); }
int count_tri(const Item& I) { return tri_tiles(I); }
int count_gram(const Item& I) { return tri_tiles(I) * I.chunks; }
int count_split(const Item& I) { return I.chunks > 1 ? tri_tiles(I) : 0; }

template <typename T>
void run_items(Items& L, const NsPlan& p, hipStream_t st) {
  const Momentum mo{p.momentum, p.nesterov};
  const Finish fin{p.lr_dev, p.lr, p.decay};
  const dim3 block(kThreads);
  auto launch_over = [&](int (*count)(const Item&), auto&& go) {
    const int blocks = blocks_before(L, count);
    if (blocks) go(dim3(blocks));
  };
  launch_over(count_sums, [&](dim3 g) { hipLaunchKernelGGL((ns_norm_kernel<T>), g, block, 0, st, L, mo); });
  Items V, M;                                          // vectors and matrices
  V.n = M.n = 0;
  for (int i = 0; i < L.n; ++i) {
    Items& to = L.it[i].m == 1 ? V : M;
    to.it[to.n++] = L.it[i];
  }
  if (V.n) {
    const int blocks = blocks_before(V, count_sums);
    hipLaunchKernelGGL((ns_vector_kernel<T>), dim3(blocks), block, 0, st, V, mo, p.eps, p.k, p.steps, fin);
  }
  if (!M.n) return;
  L = M;
  Scales sc{p.scale_x, p.scale_s, p.scale_r, p.growth};
  launch_over(count_tiles, [&](dim3 g) { hipLaunchKernelGGL((ns_split_kernel<T>), g, block, 0, st, L, mo, p.eps, sc); });
  for (int k = 0; k < p.steps; ++k) {
    launch_over(count_gram, [&](dim3 g) { hipLaunchKernelGGL(ns_gram_kernel, g, block, 0, st, L, sc, k); });
    Items S = L;                                       // the matrices whose long axis was split
    S.n = 0;
    for (int i = 0; i < L.n; ++i)
      if (L.it[i].chunks > 1) S.it[S.n++] = L.it[i];
    if (S.n) {
      const int blocks = blocks_before(S, count_split);
      hipLaunchKernelGGL(ns_gram_sum_kernel, dim3(blocks), block, 0, st, S, sc);
    }
    launch_over(count_tri, [&](dim3 g) { hipLaunchKernelGGL(ns_poly_kernel, g, block, 0, st, L, sc, p.k.b, p.k.c); });
    if (k + 1 < p.steps)
      launch_over(count_tiles, [&](dim3 g) {
        hipLaunchKernelGGL((ns_update_kernel<T, false>), g, block, 0, st, L, sc, p.k.a, k, fin);
      });
    else
      launch_over(count_tiles, [&](dim3 g) {
        hipLaunchKernelGGL((ns_update_kernel<T, true>), g, block, 0, st, L, sc, p.k.a, k, fin);
      });
  }
}

}  // namespace

const char* ns_refusal(const NsMatrix& M) {
  if (M.rows < 1 || M.cols < 1 || M.batch < 1) return "empty or negative sizes";
  const int64_t m = M.rows < M.cols ? M.rows : M.cols, n = M.rows < M.cols ? M.cols : M.rows;
  if (m > 32768 || n > (int64_t)1 << 30 || (m > 1 && n > (int64_t)1 << 24)) return "a side is too long (short side over 32768, or long side over 2^24, 2^30 for a vector)";
  // a launch holds fewer than 2^32 threads: 2^24 blocks of 256, over all the matrices that share it
  const int64_t tiles = ((m + 63) / 64) * ((n + 63) / 64);
  if (M.batch > ((int64_t)1 << 19) / (tiles > kSumsMax ? tiles : kSumsMax)) return "too many tiles in one stack";
  return nullptr;
}

bool ns_scales(const NsCoefficients& k, int steps, NsPlan* p) {
  // the largest |x (a + b x^2 + c x^4)| and |b s + c s^2| over the singular values a step can meet, by interval ends and
  // the inner extrema, step by step from [0, 1]
  for (const float v : {k.a, k.b, k.c})
    if (!(std::fabs(v) < 4096.0f)) return false;
  double top = 1.0, all = 1.0, rmax = 0.0, grow = 1.0;
  for (int i = 0; i < steps; ++i) {
    const double T = top;
    auto f = [&](double x) { return std::fabs(x * (k.a + x * x * (k.b + k.c * x * x))); };
    auto r = [&](double s) { return std::fabs(s * (k.b + k.c * s)); };
    double next = f(T);
    // inner extrema: a + 3 b s + 5 c s^2 = 0 with s = x^2
    if (k.c != 0.0f) {
      const double disc = 9.0 * k.b * k.b - 20.0 * (double)k.a * k.c;
      if (disc >= 0.0)
        for (const double sign : {-1.0, 1.0}) {
          const double s = (-3.0 * k.b + sign * std::sqrt(disc)) / (10.0 * k.c);
          if (s > 0.0 && s < T * T) next = std::fmax(next, f(std::sqrt(s)));
        }
    } else if (k.b != 0.0f) {
      const double s = -(double)k.a / (3.0 * k.b);
      if (s > 0.0 && s < T * T) next = std::fmax(next, f(std::sqrt(s)));
    }
    rmax = std::fmax(rmax, r(T * T));
    if (k.c != 0.0f) {
      const double s = -(double)k.b / (2.0 * k.c);
      if (s > 0.0 && s < T * T) rmax = std::fmax(rmax, r(s));
    }
    // |a + b s + c s^2| <= |a| + the bound on R: what a step multiplies any singular value by
    grow = std::fmax(grow, std::fabs(k.a) + rmax);
    top = next;
    all = std::fmax(all, top);
    if (!(all < 64.0) || !(rmax < 4096.0)) return false;
  }
  // 1.01: rounding can carry a singular value past the bound
  const int kx = (int)std::ceil(std::log2(all * 1.01)), kr = (int)std::ceil(std::log2(std::fmax(rmax, 1.0) * 1.01));
  p->scale_x = std::ldexp(1.0f, 15 - kx);
  p->scale_s = std::ldexp(1.0f, 15 - 2 * kx);
  p->scale_r = std::ldexp(1.0f, 15 - kr);
  p->growth = (int)std::ceil(std::log2(grow * 1.01));
  return true;
}

size_t ns_ws_bytes(const NsMatrix* mats, int count) {
  size_t sum = 0;
  for (int j = 0; j < count; ++j) {
    const Item I = make_item(mats[j]);
    sum += (size_t)I.ws_stride * I.batch;
  }
  return sum;
}

void launch_ns(int dtype, const NsMatrix* mats, int count, const NsPlan& p, void* ws, hipStream_t st) {
  Items L;
  L.n = 0;
  char* at = static_cast<char*>(ws);
  for (int j = 0; j < count && j < kItemsMax; ++j) {
    Item I = make_item(mats[j]);
    I.ws = at;
    at += I.ws_stride * I.batch;
    L.it[L.n++] = I;
  }
  switch (dtype) {
    case kNormF32: run_items<float>(L, p, st); break;
    case kNormBf16: run_items<__bf16>(L, p, st); break;
    default: run_items<_Float16>(L, p, st); break;
  }
}

}  // namespace pdekan
