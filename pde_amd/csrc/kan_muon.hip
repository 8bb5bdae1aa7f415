// Orthogonalised updates by Newton-Schulz products, and the Muon step of a weight around them.
//
//   U = G, or for the optimiser  M <- mu M + (1 - mu) G,  U = (1 - mu) G + mu M  (Nesterov) or U = M
//   X = U / (|U|_F + eps), its short side first (m <= n);  `steps` times:  S = X X^T,  X <- a X + (b S + c S S) X
//   out = X, or  W <- (1 - lr decay) W - lr gain X
//
// Products run on the fp16 matrix instructions with fp32 accuracy: an operand is two fp16 pieces, x = hi + lo (22 bits and a
// sign, of values scaled so that nothing overflows), a product three matrix instructions, hi hi + hi lo + lo hi, summed in
// fp32; what is left out is 2^-24 of a term (matrices of at most 32 rows take lo lo too).  Operands lie in memory in the order of the
// instruction's registers: a tile of 16 rows x 32 inner values is 1 KB of hi pieces and 1 KB of lo pieces, lane l's 8 values (row
// l % 16, inner values 8 (l / 16) ..) at 16 l, so a wave loads one operand of one instruction as one contiguous 1 KB, and tiles that
// follow each other along the inner dimension lie next to each other.
#include <hip/hip_runtime.h>
#include <climits>
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
constexpr int kSumsMax = 1024;            // partial sums of squares a matrix

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
  int bt, bts;            // rows and columns a block of the products takes, along the long axis and among squares: 64 or 128
  int chunks, kchunk;     // splits of the long axis in X X^T, inner tiles (of 32) a split
  int path;               // see enum Path
  int width, strips;      // columns of X a block of the small kernel takes, and how many such blocks there are
  float gain;
};
// kVector: one row, too long for one block;  kSingle: one block does everything (vectors too);  kStrips: one block a strip of
// columns, a launch a step;  kTiles: one launch a product
enum Path { kVector, kSingle, kStrips, kTiles };
struct Items {
  Item it[kItemsMax];
  int first[kItemsMax + 1];               // first block of each item in this launch, INT_MAX past the last
  int n;
};

// workspace of a matrix: X [mp][np], X^T twice [np][mp], five square matrices [mp][mp] as two-piece tiles, then the splits'
// partial products, the partial sums of squares and the numbers of struct Norm
__device__ __host__ inline int64_t plane_bytes(const Item& I) { return (int64_t)I.mp * I.np * 4; }
__device__ __host__ inline int64_t square_bytes(const Item& I) { return (int64_t)I.mp * I.mp * 4; }
__device__ __host__ inline int64_t off_xt(const Item& I, int k) { return plane_bytes(I) * (1 + k); }
enum Square { kS = 0, kQ = 1, kT = 2, kP0 = 3, kP1 = 4, kSquares = 5 };
__device__ __host__ inline int64_t off_sq(const Item& I, int k) { return plane_bytes(I) * 3 + square_bytes(I) * k; }
__device__ __host__ inline int64_t off_part(const Item& I) { return off_sq(I, kSquares); }
__device__ __host__ inline int tri_tiles(const Item& I) { const int t = (I.mp + I.bt - 1) / I.bt; return t * (t + 1) / 2; }
__device__ __host__ inline int tri_squares(const Item& I) { const int t = (I.mp + I.bts - 1) / I.bts; return t * (t + 1) / 2; }
__device__ __host__ inline int64_t off_sums(const Item& I) {
  if (I.path == kVector) return 0;        // a vector has nothing else
  return off_part(I) + (I.chunks > 1 ? (int64_t)I.chunks * tri_tiles(I) * I.bt * I.bt * 4 : 0);
}
// What the first kernels find out about a matrix.  X = factor U' with U' = U 2^-e: the composed form keeps U' itself, whose
// entries are those of U to the last bit, in the pieces, and applies the factor to the products; the other form has 1.
struct Norm { float factor; int ex; };
__device__ __host__ inline int64_t off_norm(const Item& I) { return off_sums(I) + I.nsum * (int64_t)sizeof(double); }
__device__ __host__ inline int64_t item_bytes(const Item& I) {
  return (off_norm(I) + (int64_t)sizeof(Norm) + 255) / 256 * 256;
}
template <typename H>
__device__ __forceinline__ H* at(char* ws, int64_t off) { return reinterpret_cast<H*>(ws + off); }

// The block's matrix, and its number among the blocks of it.  A lone matrix is read with the first kernel arguments, in a list
// with the second ones: each trip to them takes 0.7 us.
__device__ __forceinline__ int find_item(const Items& L, Item& I) {
  I = L.it[0];
  if (L.n == 1) return (int)blockIdx.x;
  int k = 0;
#pragma unroll
  for (int j = 1; j < kItemsMax; ++j) k += (int)blockIdx.x >= L.first[j];
  I = L.it[k];
  return (int)blockIdx.x - L.first[k];
}

// (row, column) of the t-th tile of the upper triangle, columns first: (0,0) (0,1) (1,1) (0,2) ...
__device__ __forceinline__ void tri_tile(int t, int& bi, int& bj) {
  bj = (int)((__builtin_sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
  while (bj * (bj + 1) / 2 > t) --bj;
  while ((bj + 1) * (bj + 2) / 2 <= t) ++bj;
  bi = t - bj * (bj + 1) / 2;
}

// ---- scales of the pieces -------------------------------------------------------------------------------------------
// X has no singular value over the host's bound 2^kx, S none over 2^(2 kx), and so on; entries are bounded alike, and pieces
// are scaled by powers of two to stay below 2^15.  Where eps dominates |U|_F, X starts as small as |U| / eps and its pieces
// are scaled up by 2^ex more, ex = the exponent of (|U| + eps) / |U|; a step multiplies X by at most 2^growth, so before step
// k it is 2^max(0, ex - growth k).
struct Scales { float x, s, q, t, p; int growth; };    // what the entries of X, S, Q (or R), T = Q S, P are multiplied by

__device__ __forceinline__ Norm* norm_slot(const Item& I, char* ws) {
  return at<Norm>(ws, off_norm(I));
}
__device__ __forceinline__ float x_scale(const Norm& n, const Scales& sc, int step) {
  const int ex = n.ex - sc.growth * step;
  return ldexpf(sc.x, ex > 0 ? ex : 0);
}

// halves offset of (row, col) of a matrix of PIECES pieces with kt inner tiles a row of tiles; col % 4 == 0 addresses four
// values
template <int PIECES>
__device__ __forceinline__ int64_t piece_at(int row, int col, int kt) {
  return ((int64_t)(row >> 4) * kt + (col >> 5)) * (512 * PIECES) + ((row & 15) + 16 * ((col & 31) >> 3)) * 8 + (col & 7);
}
__device__ __forceinline__ void store_pieces(_Float16* base, int row, int col, int kt, const float (&v)[4], float scale) {
  f16x4 hi, lo;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y = v[i] * scale;
    hi[i] = (_Float16)y;
    lo[i] = (_Float16)(y - (float)hi[i]);
  }
  _Float16* p = base + piece_at<2>(row, col, kt);
  *reinterpret_cast<f16x4*>(p) = hi;
  *reinterpret_cast<f16x4*>(p + 512) = lo;
}
// eight values of a row, col % 8 == 0
template <int PIECES>
__device__ __forceinline__ void store_pieces8(_Float16* base, int row, int col, int kt, const float (&v)[8], float scale) {
  f16x8 hi, lo;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = v[i] * scale;
    hi[i] = (_Float16)y;
    lo[i] = (_Float16)(y - (float)hi[i]);
  }
  _Float16* p = base + piece_at<PIECES>(row, col, kt);
  *reinterpret_cast<f16x8*>(p) = hi;
  if constexpr (PIECES == 2) *reinterpret_cast<f16x8*>(p + 512) = lo;
}
template <int PIECES>
__device__ __forceinline__ void load_pieces(const _Float16* base, int row, int col, int kt, float (&v)[4], float unscale) {
  const _Float16* p = base + piece_at<PIECES>(row, col, kt);
  const f16x4 hi = *reinterpret_cast<const f16x4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)hi[i];
  if constexpr (PIECES == 2) {
    const f16x4 lo = *reinterpret_cast<const f16x4*>(p + 512);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += (float)lo[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] *= unscale;
}

// the two pieces of four values, hi | lo << 16 each: what a quad of lanes can transpose and store twice
__device__ __forceinline__ void split_pieces(const float (&v)[4], float scale, float (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y = v[i] * scale;
    const _Float16 hi = (_Float16)y, lo = (_Float16)(y - (float)hi);
    p[i] = __uint_as_float((unsigned)__builtin_bit_cast(unsigned short, hi) |
                           (unsigned)__builtin_bit_cast(unsigned short, lo) << 16);
  }
}
__device__ __forceinline__ void store_packed(_Float16* base, int row, int col, int kt, const float (&p)[4]) {
  // hi halves of a pair: bytes 0, 1 of each; lo halves: bytes 2, 3
  const unsigned a = __float_as_uint(p[0]), b = __float_as_uint(p[1]), c = __float_as_uint(p[2]), d = __float_as_uint(p[3]);
  _Float16* to = base + piece_at<2>(row, col, kt);
  *reinterpret_cast<uint2*>(to) = make_uint2(__builtin_amdgcn_perm(b, a, 0x05040100u), __builtin_amdgcn_perm(d, c, 0x05040100u));
  *reinterpret_cast<uint2*>(to + 512) = make_uint2(__builtin_amdgcn_perm(b, a, 0x07060302u), __builtin_amdgcn_perm(d, c, 0x07060302u));
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

struct Momentum { float mu, rest; int nesterov; };           // rest: 1 - mu, rounded once (in 32 bits 1 - mu is 9.5e-7 off at 0.99)

template <typename T>
__device__ __forceinline__ float source_value(const Item& I, int64_t at, const Momentum& mo) {
  const float g = (float)static_cast<const T*>(I.src)[at];
  if (!I.mom) return g;
  const float m = I.mom[at];
  return mo.nesterov ? mo.rest * g + mo.mu * m : m;
}

// the momentum takes in g;  what U has there
__device__ __forceinline__ float moved(float g, float& m, const Momentum& mo) {
  m = fmaf(mo.mu, m, mo.rest * g);
  return mo.nesterov ? mo.rest * g + mo.mu * m : m;
}

// (Times here and below: mean of 20 calls under the profiler, the best in brackets.  2048 x 8192 bf16: 10.4 us (9.8), 3.2 TB/s; a step
// of KAN [2,256,256,256,1], 13 MB of gradients and momentum each: 10.8 (9.6).)
// Partial sums of squares of U in 64 bits (the squares of gradients as small as 1e-25 vanish in 32), one a block, a block's
// values contiguous, 16 bytes of G a thread; the optimiser's momentum is updated on the way.
template <typename T>
__global__ void __launch_bounds__(kThreads) ns_norm_kernel(Items L, Momentum mo) {
  constexpr int kVec = 16 / sizeof(T);
  typedef T Vec __attribute__((ext_vector_type(kVec)));
  __shared__ double red[kThreads / 64];
  Item I;
  const int here = find_item(L, I);
  const int b = here / I.nsum, part = here % I.nsum;
  const int64_t base = b * I.size, per = (I.size + I.nsum - 1) / I.nsum, span = (per + kThreads * kVec - 1) / (kThreads * kVec) * (kThreads * kVec);
  const int64_t lo = part * span, hi = lo + span < I.size ? lo + span : I.size;
  const T* src = static_cast<const T*>(I.src) + base;
  const bool wide = (((uintptr_t)src | (I.mom ? (uintptr_t)(I.mom + base) : 0)) & 15) == 0;
  double s = 0.0;
  if (wide) {
    constexpr int kTurns = 4;                            // a thread's loads on their way at once
    constexpr int64_t kTurn = kThreads * kVec;
    float* mom = I.mom ? I.mom + base : nullptr;
    for (int64_t at = lo + threadIdx.x * kVec; at + kVec <= hi; at += kTurns * kTurn) {
      Vec g[kTurns];
      float m[kTurns][kVec];
#pragma unroll
      for (int t = 0; t < kTurns; ++t) {
        const int64_t i = at + t * kTurn;
        if (i + kVec > hi) continue;
        g[t] = *reinterpret_cast<const Vec*>(src + i);
        if (mom) {
#pragma unroll
          for (int q = 0; q < kVec; q += 4) *reinterpret_cast<f32x4*>(m[t] + q) = *reinterpret_cast<const f32x4*>(mom + i + q);
        }
      }
#pragma unroll
      for (int t = 0; t < kTurns; ++t) {
        const int64_t i = at + t * kTurn;
        if (i + kVec > hi) continue;
        double u[kVec];
#pragma unroll
        for (int q = 0; q < kVec; ++q) {
          u[q] = (float)g[t][q];
          if (mom) u[q] = moved((float)g[t][q], m[t][q], mo);
          s = fma(u[q], u[q], s);
        }
        if (mom) {
#pragma unroll
          for (int q = 0; q < kVec; q += 4) *reinterpret_cast<f32x4*>(mom + i + q) = *reinterpret_cast<const f32x4*>(m[t] + q);
        }
      }
    }
    if (hi == I.size)
      for (int64_t i = hi - (hi - lo) % kVec + threadIdx.x; i < hi; i += kThreads) {
        const float g = (float)src[i];
        const double u = mom ? moved(g, mom[i], mo) : g;
        s = fma(u, u, s);
      }
  } else {
#pragma unroll 4
    for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) {
      const float g = (float)src[i];
      const double u = I.mom ? moved(g, I.mom[base + i], mo) : g;
      s = fma(u, u, s);
    }
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
#pragma unroll 4
  for (int k = threadIdx.x & 63; k < I.nsum; k += 64) s += sums[k];
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
  return sqrt(s);
}

struct Finish { const float* lr_dev; float lr, decay; };

// what becomes of value x at element `e` of the matrices (weights are fp32)
template <typename T>
__device__ __forceinline__ void put(const Item& I, int64_t e, float x, float lr, const Finish& f) {
  T* out = static_cast<T*>(I.out);
  if (sizeof(T) == 4 && I.mom) out[e] = (T)fmaf((float)out[e], fmaf(-lr, f.decay, 1.0f), -(lr * I.gain) * x);
  else out[e] = (T)x;
}

// what the steps multiply U by where it is a single row: S is the number |X|^2 and X keeps its direction
__device__ __forceinline__ double vector_factor(double norm, float eps, const NsCoefficients& k, int steps) {
  double factor = 1.0 / (norm + (double)eps), length = norm * factor;
  for (int i = 0; i < steps; ++i) {
    const double s = length * length, q = k.a + s * ((double)k.b + k.c * s);
    factor *= q;
    length *= q;
  }
  return factor;
}

// a block's share of a vector
template <typename T>
__device__ __forceinline__ void vector_share(const Item& I, int local, const Momentum& mo, float eps, const NsCoefficients& k, int steps,
                                             const Finish& f) {
  const int b = local / I.nsum, part = local % I.nsum;
  const double factor = vector_factor(matrix_norm(I, b), eps, k, steps);
  const float lr = f.lr_dev ? *f.lr_dev : f.lr;
  const int64_t base = b * I.size;
  for (int64_t i = (int64_t)part * kThreads + threadIdx.x; i < I.size; i += (int64_t)I.nsum * kThreads)
    put<T>(I, base + i, (float)((double)source_value<T>(I, base + i, mo) * factor), lr, f);
}
template <typename T>
__global__ void __launch_bounds__(kThreads) ns_vector_kernel(Items L, Momentum mo, float eps, NsCoefficients k, int steps,
                                                             Finish f) {
  Item I;
  const int here = find_item(L, I);
  vector_share<T>(I, here, mo, eps, k, steps, f);
}

// Bound by what it writes, two planes of pieces: 2048 x 8192 bf16, 33 MB in and 67 MB out, 28 us (27) = 3.6 TB/s; 256 x 5888 fp32, 6
// and 12 MB, 11.3 (9.1).
// X and X^T of a 64 x 64 tile as pieces, and the vectors of the list; COMPOSED: of U' in one piece (16-bit types: exact).
template <typename T, bool COMPOSED>
__global__ void __launch_bounds__(kThreads) ns_split_kernel(Items L, Momentum mo, float eps, Scales sc, NsCoefficients k, int steps,
                                                            Finish f) {
  constexpr int PX = COMPOSED ? 1 : 2;
  __shared__ float tile[64][65];
  Item I;
  const int here = find_item(L, I);
  if (I.path == kVector) {
    vector_share<T>(I, here, mo, eps, k, steps, f);
    return;
  }
  const int tm = (I.mp + 63) / 64, tn = (I.np + 63) / 64;
  const int b = here / (tm * tn), t = here % (tm * tn), bi = t % tm, bj = t / tm;
  const int64_t base = b * I.size;
  char* ws = I.ws + b * I.ws_stride;
  // all of a thread's values on their way before the norm is put together, four neighbours at once where all are whole fours
  typedef T Four __attribute__((ext_vector_type(4)));
  const T* src = static_cast<const T*>(I.src) + base;
  const int inner = I.tall ? I.m : I.n;
  const bool fours = inner % 4 == 0 && (uintptr_t)src % (4 * sizeof(T)) == 0 && !I.mom;
  float raw[16];
  // value u of the thread: row a of memory, value c of it
  auto place = [&](int u, int& a, int& c) {
    const int k = fours ? threadIdx.x * 4 + (u & 3) + (u >> 2) * (4 * kThreads) : threadIdx.x + u * kThreads;
    a = k / 64;
    c = k % 64;
  };
  auto element = [&](int a, int c, bool& in) {
    const int i = bi * 64 + (I.tall ? c : a), j = bj * 64 + (I.tall ? a : c);
    in = i < I.m && j < I.n;
    return I.tall ? (int64_t)j * I.m + i : (int64_t)i * I.n + j;
  };
  if (fours) {
#pragma unroll
    for (int u = 0; u < 16; u += 4) {
      int a, c;
      bool in;
      place(u, a, c);
      const int64_t e = element(a, c, in);
      Four v = {};
      if (in) v = *reinterpret_cast<const Four*>(src + e);
#pragma unroll
      for (int q = 0; q < 4; ++q) raw[u + q] = (float)v[q];
    }
  } else {
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      int a, c;
      bool in;
      place(u, a, c);
      const int64_t e = element(a, c, in);
      raw[u] = in ? source_value<T>(I, base + e, mo) : 0.0f;
    }
  }
  const double norm = matrix_norm(I, b), whole = norm + (double)eps, small = whole / norm;
  Norm nm;
  // at most 2^96: entries below 2^-96 |X| lose their low bits; (NaN and 0 norms: no shift)
  nm.ex = small > 1.0 && norm > 0.0 ? (small < 7.9e28 ? ilogb(small) : 96) : 0;
  // U 2^-e with 2^e >= |U| + eps: entries within [-1, 1], whatever their size; an infinite or NaN norm makes everything NaN
  const int e = whole < 1.0e300 ? ilogb(whole) + 1 : 0;
  const float factor = whole < 1.0e300 ? (float)ldexp(1.0 / whole, e) : __builtin_nanf("");
  nm.factor = COMPOSED ? factor : 1.0f;
  if (t == 0 && threadIdx.x == 0) *norm_slot(I, ws) = nm;
  const float scx = x_scale(nm, sc, 0);
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    int a, c;
    place(u, a, c);
    const float v = ldexpf(raw[u], -e);
    tile[I.tall ? c : a][I.tall ? a : c] = COMPOSED ? v : v * factor;
  }
  __syncthreads();
  _Float16 *x = at<_Float16>(ws, 0), *xt = at<_Float16>(ws, off_xt(I, 0));
  const int ktx = I.np / 32, kt = I.mp / 32;
  for (int k = threadIdx.x; k < 64 * 8; k += kThreads) {
    const int r = k % 64, q = k / 64 * 8;
    float v[8];
    const int i = bi * 64 + r, j = bj * 64 + q;
    if (i < I.mp && j < I.np) {
#pragma unroll
      for (int n = 0; n < 8; ++n) v[n] = tile[r][q + n];
      store_pieces8<PX>(x, i, j, ktx, v, scx);
    }
    const int i2 = bi * 64 + q, j2 = bj * 64 + r;
    if (i2 < I.mp && j2 < I.np) {
#pragma unroll
      for (int n = 0; n < 8; ++n) v[n] = tile[q + n][r];
      store_pieces8<PX>(xt, j2, i2, kt, v, scx);
    }
  }
}

// Sums of so few terms that a product takes lo lo too: see block_product.
__device__ __forceinline__ bool few_rows(const Item& I) { return I.mp == 32; }

// ---- products -------------------------------------------------------------------------------------------------------

// What bounds a product: the LDS where a block is 64 (a stage of 16 KB is read 32 KB for 192 cycles of matrix instructions a wave),
// the latency behind the L2 where it is 128, whose 80 KB hold two stages of two-piece operands.  Alone on the chip 2048 x 2048
// squares (three matrix instructions a product, the upper triangle) run at 0.60 PFLOP/s of matrix instructions in blocks of 64, 45 us
// (41); in blocks of 128, 57 us with four stages and one block a compute unit, more with two, the inner axis split over two to four
// blocks included.  128 blocks that fill the chip reach 1.06 PFLOP/s (X <- Q X, 2048 x 8192); a large library product 1.2.
// P Q^T of a BT x BT block over inner tiles [k0, k1), PP and PQ pieces an operand.  Four waves take a quarter each: acc[a][c]
// is the 16 x 16 block at rows 16 a of P and 16 c of Q; lane l holds Q's row l % 16 and P's rows 4 (l / 16) + r.
// Operand tiles go from memory to LDS without passing registers, kStages inner tiles of the whole block in a ring, and
// from LDS to registers as contiguous 1 KB reads.  `whole`: with lo lo, for matrices of few rows (see block_product).
template <int BT, int PP, int PQ>
struct Product {
  static constexpr int kW = BT / 32;                           // 16-row tiles a wave takes of either operand
  static constexpr int kFrags = BT / 16 * (PP + PQ);           // 1 KB pieces of tiles a stage
  static constexpr int kLoads = kFrags / 4;                    // a wave's
  // as many stages as leave room for three blocks of 64 or two of 128 a compute unit
  static constexpr int kRoom = BT == 64 ? 48 * 1024 : 80 * 1024;
  static constexpr int kStages = kRoom / (kFrags * 1024) < 4 ? kRoom / (kFrags * 1024) : 4;
  static constexpr int kLds = kFrags * 1024 * kStages;
  f32x4 v[kW][kW];

  __device__ __forceinline__ void run(const _Float16* P, const _Float16* Q, int bp, int bq, int prows, int qrows, int kt,
                                      int k0, int k1, char* lds, bool whole) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const _Float16* src[kLoads];
    int step[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      // tiles past the padded matrix repeat its last one; what they give is never stored
      const int f = wave * kLoads + u;
      const bool isp = f < BT / 16 * PP;
      const int g = isp ? f : f - BT / 16 * PP, pieces = isp ? PP : PQ;
      const int tile = min((isp ? bp : bq) * (BT / 16) + g / pieces, (isp ? prows : qrows) / 16 - 1);
      step[u] = 512 * pieces;
      src[u] = (isp ? P : Q) + ((int64_t)tile * kt + k0) * step[u] + (g % pieces) * 512 + lane * 8;
    }
    auto fetch = [&](int stage) {
      char* dst = lds + stage * (kFrags * 1024) + wave * (kLoads * 1024);
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src[u],
                                         (__attribute__((address_space(3))) void*)(dst + u * 1024), 16, 0, 0);
        src[u] += step[u];
      }
    };
#pragma unroll
    for (int a = 0; a < kW; ++a)
#pragma unroll
      for (int c = 0; c < kW; ++c) v[a][c] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    const int n = k1 - k0;
#pragma unroll
    for (int i = 0; i < kStages; ++i)
      if (i < n) fetch(i);
    // Step i multiplies what step i - 1 read from LDS, and reads the next inner tile meanwhile.  Its wait leaves the stages
    // after the next on their way; behind the barrier every wave has stage i in registers, so its place takes a new one.
    struct Regs { f16x8 p[kW][PP], q[kW][PQ]; };
    auto read = [&](Regs& r, int stage) {
      const char* base = lds + stage * (kFrags * 1024) + lane * 16;
#pragma unroll
      for (int a = 0; a < kW; ++a) {
#pragma unroll
        for (int h = 0; h < PP; ++h)
          r.p[a][h] = *reinterpret_cast<const f16x8*>(base + (((wave & 1) * kW + a) * PP + h) * 1024);
#pragma unroll
        for (int h = 0; h < PQ; ++h)
          r.q[a][h] = *reinterpret_cast<const f16x8*>(base + (BT / 16 * PP + ((wave >> 1) * kW + a) * PQ + h) * 1024);
      }
    };
    // one kind of product over all blocks, then the next: instructions on one accumulator stand kW^2 apart
    auto multiply = [&](const Regs& r) {
      if constexpr (BT == 64 && PP == 2 && PQ == 2) {
        if (whole)
#pragma unroll
          for (int a = 0; a < kW; ++a)
#pragma unroll
            for (int c = 0; c < kW; ++c) v[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(r.p[a][1], r.q[c][1], v[a][c], 0, 0, 0);
      }
#pragma unroll
      for (int kind = 0; kind < 3; ++kind) {
        const int hp = kind == 0, hq = kind == 1;
        if ((hp && PP == 1) || (hq && PQ == 1)) continue;
#pragma unroll
        for (int a = 0; a < kW; ++a)
#pragma unroll
          for (int c = 0; c < kW; ++c)
            v[a][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(r.p[a][hp ? PP - 1 : 0], r.q[c][hq ? PQ - 1 : 0], v[a][c], 0, 0, 0);
      }
    };
    auto landed = [&](bool more) {
      if (more) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kStages - 2) * kLoads) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    // the first stage: up to kStages - 1 younger ones
    if (n >= kStages) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kStages - 1) * kLoads) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    Regs ra, rb;
    read(ra, 0);
    int stage = 0;
    auto one = [&](int i, const Regs& now, Regs& next) {
      if (i + 1 < n) {
        landed(i + kStages <= n);
        if (i + kStages < n) fetch(stage);
        stage = stage + 1 == kStages ? 0 : stage + 1;
        read(next, stage);
      }
      multiply(now);
    };
    int i = 0;
    for (; i + 1 < n; i += 2) {
      one(i, ra, rb);
      one(i + 1, rb, ra);
    }
    if (i < n) multiply(ra);
  }
  // first rows of P and Q of this wave's part
  static __device__ __forceinline__ int row_p(int bp) { return bp * BT + (threadIdx.x >> 6 & 1) * (BT / 2); }
  static __device__ __forceinline__ int row_q(int bq) { return bq * BT + (threadIdx.x >> 7) * (BT / 2); }

  // f(16 x 16 block's first row of P, of Q, the lane's four values)
  template <typename F>
  __device__ __forceinline__ void each(int bp, int bq, int prows, int qrows, F&& f) {
#pragma unroll
    for (int a = 0; a < kW; ++a)
#pragma unroll
      for (int c = 0; c < kW; ++c) {
        const int p0 = row_p(bp) + 16 * a, q0 = row_q(bq) + 16 * c;
        if (p0 >= prows || q0 >= qrows) continue;
        float x[4] = {v[a][c][0], v[a][c][1], v[a][c][2], v[a][c][3]};
        f(p0, q0, x);
      }
  }
};

// A symmetric result: both triangles from one, blocks on the diagonal as they are.
__device__ __forceinline__ void store_symmetric(_Float16* S, int kt, bool diagonal, int p0, int q0, const float (&v)[4],
                                                float scale) {
  const int lane = threadIdx.x & 63;
  float p[4];
  split_pieces(v, scale, p);
  store_packed(S, q0 + (lane & 15), p0 + 4 * (lane >> 4), kt, p);
  if (!diagonal) {
    quad_transpose(p);
    store_packed(S, p0 + 4 * (lane >> 4) + (lane & 3), q0 + (lane & 12), kt, p);
  }
}

// Neighbouring blocks go to different XCDs, each with an L2 of its own: renumbered, an XCD's blocks are neighbours.
__device__ __forceinline__ int xcd_order(int local, int count) {
  const int per = count / 8;
  return local < per * 8 ? (local % 8) * per + local / 8 : local;
}

// 2048 x 8192 bf16 in 128 blocks of four splits: one piece 57 us (52), 0.64 PFLOP/s, two 127 (117), 0.86; 256 x 5888 fp32: 8.0 (5.6), 46
// splits of 10 tiles.
// S = X X^T: block = (split of the long axis, tile of the upper triangle)
template <int BT, int PX>
__global__ void __launch_bounds__(kThreads, BT == 64 ? 3 : 2) ns_gram_kernel(Items L, Scales sc, int step) {
  extern __shared__ char lds[];
  Item I;
  const int here = find_item(L, I);
  const int tiles = tri_tiles(I), per = tiles * I.chunks;
  const int local = xcd_order(here, per * I.batch), b = local / per, rest = local % per, chunk = rest / tiles, t = rest % tiles;
  int bi, bj;
  tri_tile(t, bi, bj);
  char* ws = I.ws + b * I.ws_stride;
  const _Float16* x = at<const _Float16>(ws, 0);
  const int kt = I.np / 32, k0 = chunk * I.kchunk, k1 = min(k0 + I.kchunk, kt);
  Product<BT, PX, PX> acc;
  acc.run(x, x, bi, bj, I.mp, I.mp, kt, k0, k1, lds, few_rows(I));
  const Norm nm = *norm_slot(I, ws);
  const float scx = x_scale(nm, sc, step), factor = step ? 1.0f : nm.factor, unscale = factor / scx * (factor / scx);
  if (I.chunks == 1) {
    acc.each(bi, bj, I.mp, I.mp, [&](int p0, int q0, float (&v)[4]) {
      store_symmetric(at<_Float16>(ws, off_sq(I, kS)), I.mp / 32, bi == bj, p0, q0, v, unscale * sc.s);
    });
    return;
  }
  constexpr int kAcc = BT * BT / 1024;                         // 16 x 16 blocks a wave
  f32x4* part = at<f32x4>(ws, off_part(I)) + ((int64_t)chunk * tiles + t) * (BT * BT / 4) + threadIdx.x;
#pragma unroll
  for (int a = 0; a < kAcc; ++a) part[a * kThreads] = acc.v[a / acc.kW][a % acc.kW] * unscale;
}

// the sum of the splits, in a fixed order: a block sums a quarter (BT = 128: a sixteenth) of a tile's 16 x 16 blocks, GROUPS
// groups of four waves every GROUPS-th split each
template <int BT, int GROUPS>
__global__ void __launch_bounds__(GROUPS * kThreads) ns_gram_sum_kernel(Items L, Scales sc) {
  constexpr int kAcc = BT * BT / 1024, kW = BT / 32;
  __shared__ f32x4 red[GROUPS][kThreads];
  Item I;
  const int here = find_item(L, I);
  const int tiles = tri_tiles(I), b = here / (tiles * kAcc), t = here / kAcc % tiles, a = here % kAcc;
  int bi, bj;
  tri_tile(t, bi, bj);
  char* ws = I.ws + b * I.ws_stride;
  const int tid = threadIdx.x % kThreads, group = threadIdx.x / kThreads;
  const f32x4* part = at<const f32x4>(ws, off_part(I)) + (int64_t)t * (BT * BT / 4) + a * kThreads + tid;
  f32x4 s = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int k = group; k < I.chunks; k += GROUPS) s += part[(int64_t)k * tiles * (BT * BT / 4)];
  if constexpr (GROUPS > 1) {
    red[group][tid] = s;
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) s += red[g][tid];
  }
  const int p0 = Product<BT, 2, 2>::row_p(bi) + 16 * (a / kW), q0 = Product<BT, 2, 2>::row_q(bj) + 16 * (a % kW);
  if (p0 >= I.mp || q0 >= I.mp) return;
  const float v[4] = {s[0], s[1], s[2], s[3]};
  store_symmetric(at<_Float16>(ws, off_sq(I, kS)), I.mp / 32, bi == bj, p0, q0, v, sc.s);
}

// 2048: 45 us (41), see Product; 256 (10 blocks): 6.4 (5.2), of which 1.3 until the arguments are there, 2.8 for 8 inner tiles and 1.4 to
// store.
// Q = a I + b S + c S S  (a = 0: R, the step less its multiple of one)
template <int BT>
__global__ void __launch_bounds__(kThreads, BT == 64 ? 3 : 2) ns_poly_kernel(Items L, Scales sc, NsCoefficients k, int out) {
  extern __shared__ char lds[];
  Item I;
  const int here = find_item(L, I);
  const int tiles = tri_squares(I), local = xcd_order(here, tiles * I.batch), b = local / tiles, t = local % tiles;
  int bi, bj;
  tri_tile(t, bi, bj);
  char* ws = I.ws + b * I.ws_stride;
  const _Float16* s = at<const _Float16>(ws, off_sq(I, kS));
  const int lane = threadIdx.x & 63, kt = I.mp / 32;
  Product<BT, 2, 2> acc;
  acc.run(s, s, bi, bj, I.mp, I.mp, kt, 0, kt, lds, few_rows(I));
  const float unscale = 1.0f / sc.s;
  acc.each(bi, bj, I.mp, I.mp, [&](int p0, int q0, float (&v)[4]) {
    const int q = q0 + (lane & 15), p = p0 + 4 * (lane >> 4);
    float o[4];
    load_pieces<2>(s, q, p, kt, o, unscale);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = fmaf(k.c * unscale * unscale, v[r], k.b * o[r]) + (p + r == q ? k.a : 0.0f);
    store_symmetric(at<_Float16>(ws, off_sq(I, out)), kt, bi == bj, p0, q0, v, sc.q);
  });
}

// Products of square matrices that commute (polynomials of one S), up to two in a launch: out = left right
struct SquareJob { int left, right, out; float scale; };       // scale: out's pieces over the product of the operands' pieces
struct SquareJobs { SquareJob j[2]; int n; };
template <int BT>
__global__ void __launch_bounds__(kThreads, BT == 64 ? 3 : 2) ns_square_kernel(Items L, SquareJobs jobs) {
  extern __shared__ char lds[];
  Item I;
  const int here = find_item(L, I);
  const int tiles = tri_squares(I), local = xcd_order(here, tiles * I.batch * jobs.n);
  const int b = local / (tiles * jobs.n), t = local % tiles;
  const SquareJob job = jobs.j[local / tiles % jobs.n];
  int bi, bj;
  tri_tile(t, bi, bj);
  char* ws = I.ws + b * I.ws_stride;
  const int kt = I.mp / 32;
  Product<BT, 2, 2> acc;
  acc.run(at<const _Float16>(ws, off_sq(I, job.left)), at<const _Float16>(ws, off_sq(I, job.right)), bi, bj, I.mp, I.mp, kt, 0,
          kt, lds, few_rows(I));
  acc.each(bi, bj, I.mp, I.mp, [&](int p0, int q0, float (&v)[4]) {
    store_symmetric(at<_Float16>(ws, off_sq(I, job.out)), kt, bi == bj, p0, q0, v, job.scale);
  });
}

// four values next to each other, all inside and aligned
template <typename T>
__device__ __forceinline__ void put4(const Item& I, int64_t e, const float (&x)[4], float lr, const Finish& f) {
  typedef T Four __attribute__((ext_vector_type(4)));
  Four* out = reinterpret_cast<Four*>(static_cast<T*>(I.out) + e);
  Four v;
  if (sizeof(T) == 4 && I.mom) {
    v = *out;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = (T)fmaf((float)v[r], fmaf(-lr, f.decay, 1.0f), -(lr * I.gain) * x[r]);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = (T)x[r];
  }
  *out = v;
}

// 2048 x 8192 bf16 in 128 blocks: of one piece (two matrix instructions a product) 149 us (139), 0.92 PFLOP/s, of two (three) 194 (184),
// 1.06; 256 x 5888 fp32: 11.4 (9.6), the latency of arguments, eight inner tiles and stores, with 368 blocks in less than two rounds.
// X <- a X + M X, computed as X^T <- a X^T + X^T M (M symmetric; a = 0: M holds all of the step): block = BT of the long axis x
// BT of the short; the last one writes the result instead.  PX pieces in, two out.
template <typename T, int BT, int PX, bool LAST>
__global__ void __launch_bounds__(kThreads, BT == 64 ? 3 : 2) ns_update_kernel(Items L, Scales sc, float ca, int square, float scale_m, int from,
                                                                int step, int next_step, Finish f) {
  extern __shared__ char lds[];
  Item I;
  const int here = find_item(L, I);
  const int tm = (I.mp + BT - 1) / BT, tn = (I.np + BT - 1) / BT;
  const int local = xcd_order(here, tm * tn * I.batch), b = local / (tm * tn), t = local % (tm * tn), bi = t % tm, bj = t / tm;
  char* ws = I.ws + b * I.ws_stride;
  const _Float16* xt = at<const _Float16>(ws, off_xt(I, from));
  const int lane = threadIdx.x & 63, kt = I.mp / 32;
  Product<BT, PX, 2> acc;
  acc.run(xt, at<const _Float16>(ws, off_sq(I, square)), bj, bi, I.np, I.mp, kt, 0, kt, lds, few_rows(I));
  const Norm nm = *norm_slot(I, ws);
  const float scx = x_scale(nm, sc, step), next = x_scale(nm, sc, next_step);
  const float factor = step ? 1.0f : nm.factor, unscale = factor / scx / scale_m, own = ca * factor / scx;
  const float lr = f.lr_dev ? *f.lr_dev : f.lr;
  const bool quads = (I.tall ? I.m : I.n) % 4 == 0 && (uintptr_t)I.out % (4 * sizeof(T)) == 0;
  acc.each(bj, bi, I.np, I.mp, [&](int j0, int i0, float (&v)[4]) {
    // after the transpose lane l holds row j0 + 4 (l / 16) + l % 4 of X^T, columns i0 + (l & 12) ..
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] *= unscale;
    quad_transpose(v);
    const int j = j0 + 4 * (lane >> 4) + (lane & 3), i = i0 + (lane & 12);
    if (ca != 0.0f) {
      float o[4];
      load_pieces<PX>(xt, j, i, kt, o, own);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += o[r];
    }
    if constexpr (!LAST) {
      float p[4];
      split_pieces(v, next, p);
      store_packed(at<_Float16>(ws, off_xt(I, from ^ 1)), j, i, kt, p);
      quad_transpose(p);
      store_packed(at<_Float16>(ws, 0), i0 + (lane & 15), j0 + 4 * (lane >> 4), I.np / 32, p);
    } else if (I.tall) {
      if (quads) {
        if (j < I.n && i < I.m) put4<T>(I, b * I.size + (int64_t)j * I.m + i, v, lr, f);
      } else if (j < I.n) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (i + r < I.m) put<T>(I, b * I.size + (int64_t)j * I.m + i + r, v[r], lr, f);
      }
    } else {
      quad_transpose(v);
      const int jj = j0 + 4 * (lane >> 4), ii = i0 + (lane & 15);
      if (quads) {
        if (ii < I.m && jj < I.n) put4<T>(I, b * I.size + (int64_t)ii * I.n + jj, v, lr, f);
      } else if (ii < I.m) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (jj + r < I.n) put<T>(I, b * I.size + (int64_t)ii * I.n + jj + r, v[r], lr, f);
      }
    }
  });
}

// ---- small matrices -------------------------------------------------------------------------------------------------

// A block of sixteen waves holds a strip of X's columns in LDS: X [mp][width] and X^T [width][mp] as two-piece tiles, and S or R
// [mp][mp], mp <= 128.  Where the strip is the whole matrix the block runs all steps on its own (kSingle); else each block
// leaves its part of X X^T in memory, and the launch of the next step lets every block of the matrix add up all parts - the
// sum, S S and R are formed once a block, which costs less than a launch of their own (kStrips).
constexpr int kSmallThreads = 1024, kSmallWaves = kSmallThreads / 64;
constexpr int kSmallRows = 128;                                // mp at most
constexpr int kTriMax = 36, kTriWave = (kTriMax + kSmallWaves - 1) / kSmallWaves;
constexpr int kUpdateWave = 4;                                 // 16 x 16 blocks of X a wave: width * mp / 256 / 16 at most
constexpr int kSmallLds = 150 * 1024;
constexpr int kPartsAhead = 16;                                // strips' parts a thread has on their way at once
constexpr float kFirst = 16384.0f;                             // what U 2^-e, |.| <= 1, is multiplied by before the first step

__device__ __host__ inline int tri16(int mp) { return mp / 16 * (mp / 16 + 1) / 2; }
__device__ __host__ inline int64_t strip_bytes(const Item& I) { return (int64_t)I.width * I.mp * 4; }
__device__ __host__ inline int64_t off_parts(const Item& I, int parity) {
  return strip_bytes(I) * I.strips + (int64_t)parity * I.strips * tri16(I.mp) * 1024;
}
__device__ __host__ inline int64_t off_squares_sum(const Item& I) { return off_parts(I, 2); }           // double [strips]
__device__ __host__ inline int64_t off_exponents(const Item& I) { return off_squares_sum(I) + I.strips * 8; }   // int [strips]
__device__ __host__ inline int64_t small_bytes(const Item& I) {
  return I.path == kSingle ? 256 : (off_exponents(I) + I.strips * 4 + 255) / 256 * 256;
}

// sum and maximum (not of NaNs) over the block, in every thread; red: a double and a float a wave
struct SumMax { double sum; float max; };
__device__ __forceinline__ SumMax block_sum_max(double s, float v, double* red, float* redf) {
  // over a row of 16 lanes as in wave_sum; the four rows through LDS with the waves
  s += dpp_move64<0xB1>(s);
  s += dpp_move64<0x4E>(s);
  s += dpp_move64<0x141>(s);
  s += dpp_move64<0x140>(s);
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  v = fmaxf(v, dpp_move<0x141>(v));
  v = fmaxf(v, dpp_move<0x140>(v));
  if ((threadIdx.x & 15) == 0) { red[threadIdx.x >> 4] = s; redf[threadIdx.x >> 4] = v; }
  __syncthreads();
  s = red[threadIdx.x & 63];
  v = redf[threadIdx.x & 63];
  s += dpp_move64<0xB1>(s);
  s += dpp_move64<0x4E>(s);
  s += dpp_move64<0x141>(s);
  s += dpp_move64<0x140>(s);
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  v = fmaxf(v, dpp_move<0x141>(v));
  v = fmaxf(v, dpp_move<0x140>(v));
  s += __shfl_xor(s, 16);
  s += __shfl_xor(s, 32);
  v = fmaxf(v, __shfl_xor(v, 16));
  v = fmaxf(v, __shfl_xor(v, 32));
  return {s, v};
}
// From the sum of squares, in 32 bits (`few` rows, whose errors are few: rounded once): everything over 2^e, so that nothing overflows.  first: 2^e / (|U| + eps);
// ex: the exponent of (|U| + eps) / |U|, see Scales
constexpr int kNoExponent = -1000;                             // of a strip of zeros
struct Start { float first; int ex; };
__device__ __forceinline__ Start start_of(double squares, float eps, int e, bool few) {
  const float norm = sqrtf((float)ldexp(squares, -2 * e)), eps_e = ldexpf(eps, -e);
  Start r;
  r.first = few ? (float)(1.0 / (sqrt(ldexp(squares, -2 * e)) + ldexp((double)eps, -e))) : 1.0f / (norm + eps_e);
  r.ex = 0;
  if (norm < eps_e && norm > 0.0f) {
    const float small = 1.0f + eps_e / norm;
    r.ex = small < 7.9e28f ? ilogbf(small) : 96;
  }
  return r;
}

// 16 x 16 block of P Q^T from tiles of two pieces in LDS: row of tiles `a` of P and `b` of Q, kt inner tiles a row.  `whole`: with
// lo lo, which is of one sign on the diagonal of S.  In sums of few terms its 2^-24 shows: errors of five steps at 5 x 64 are
// 1.2e-6 without it and with X apart from its pieces (see below), 0.9e-6 with both; fp32 products 0.7e-6.
__device__ __forceinline__ f32x4 block_product(const _Float16* P, const _Float16* Q, int a, int b, int kt, bool whole) {
  const int lane = threadIdx.x & 63;
  f32x4 lh = (f32x4){0.0f, 0.0f, 0.0f, 0.0f}, hl = lh, hh = lh;
  const _Float16 *p = P + a * kt * 1024 + lane * 8, *q = Q + b * kt * 1024 + lane * 8;
#pragma unroll 2
  for (int k = 0; k < kt; ++k) {
    const f16x8 ph = *reinterpret_cast<const f16x8*>(p + k * 1024), pl = *reinterpret_cast<const f16x8*>(p + k * 1024 + 512);
    const f16x8 qh = *reinterpret_cast<const f16x8*>(q + k * 1024), ql = *reinterpret_cast<const f16x8*>(q + k * 1024 + 512);
    if (whole) lh = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, ql, lh, 0, 0, 0);
    lh = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, qh, lh, 0, 0, 0);
    hl = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, ql, hl, 0, 0, 0);
    hh = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, qh, hh, 0, 0, 0);
  }
  return hh + (lh + hl);
}

// step < 0: the strips' U, their sums of squares and first parts;  step >= 0: that step of the strips;  SINGLE: everything
template <typename T, bool SINGLE>
__global__ void __launch_bounds__(kSmallThreads) ns_small_kernel(Items L, Momentum mo, float eps, NsCoefficients kc, int steps,
                                                                 int step, Scales sc, Finish f) {
  extern __shared__ char lds[];
  __shared__ double red[kSmallThreads / 16];
  __shared__ float redf[kSmallThreads / 16];
  Item I;
  const int here = find_item(L, I);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int b = here / I.strips, strip = here % I.strips;
  const int64_t base = b * I.size;
  const float lr = f.lr_dev ? *f.lr_dev : f.lr;
  if ((SINGLE || step < 0) && I.m == 1) {
    // X keeps the direction of the vector, S is the number |X|^2: the whole iteration is one factor
    constexpr int kTurns = 4;                            // a thread's loads on their way at once
    const T* src = static_cast<const T*>(I.src) + base;
    double s = 0.0;
    for (int at = tid; at < I.n; at += kTurns * kSmallThreads) {
      float g[kTurns], m[kTurns];
#pragma unroll
      for (int t = 0; t < kTurns; ++t) {
        const int i = min(at + t * kSmallThreads, I.n - 1);
        g[t] = (float)src[i];
        m[t] = I.mom ? I.mom[base + i] : 0.0f;
      }
#pragma unroll
      for (int t = 0; t < kTurns; ++t) {
        const int i = at + t * kSmallThreads;
        if (i >= I.n) break;
        const double u = I.mom ? moved(g[t], m[t], mo) : g[t];
        s = fma(u, u, s);
        if (I.mom) I.mom[base + i] = m[t];
      }
    }
    const double norm = sqrt(block_sum_max(s, 0.0f, red, redf).sum);
    const double factor = vector_factor(norm, eps, kc, steps);
    for (int at = tid; at < I.n; at += kTurns * kSmallThreads) {
      float u[kTurns];
#pragma unroll
      for (int t = 0; t < kTurns; ++t) u[t] = source_value<T>(I, base + min(at + t * kSmallThreads, I.n - 1), mo);
#pragma unroll
      for (int t = 0; t < kTurns; ++t) {
        const int i = at + t * kSmallThreads;
        if (i < I.n) put<T>(I, base + i, (float)((double)u[t] * factor), lr, f);
      }
    }
    return;
  }
  const int mp = I.mp, width = I.width, rb = mp / 16, mt = mp / 32, wb = width / 16, wt = width / 32, ntri = tri16(mp);
  const bool few = few_rows(I);
  _Float16* xt = reinterpret_cast<_Float16*>(lds);
  _Float16* x = xt + width * mp * 2;
  _Float16* sq = x + width * mp * 2;
  char* ws = I.ws + b * I.ws_stride;
  double* sums = at<double>(ws, off_squares_sum(I));
  int* exps = at<int>(ws, off_exponents(I));
  // the blocks of the upper triangle and of X that this wave computes, the same in every step
  int ta[kTriWave], tb[kTriWave], tj[kUpdateWave], ti[kUpdateWave];
#pragma unroll
  for (int q = 0; q < kTriWave; ++q) {
    const int t = wave + q * kSmallWaves;
    ta[q] = tb[q] = -1;
    if (t < ntri) tri_tile(t, ta[q], tb[q]);
  }
#pragma unroll
  for (int q = 0; q < kUpdateWave; ++q) {
    const int t = wave + q * kSmallWaves;
    ti[q] = t / wb;
    tj[q] = t - ti[q] * wb;
  }
  double squares = 0.0;
  int own_e = 0, all_e = 0;
  f32x4 parts[kTriWave];
#pragma unroll
  for (int q = 0; q < kTriWave; ++q) parts[q] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

  if (SINGLE || step < 0) {
    // U of the strip in fp32; a wave takes rows of memory, its lanes neighbouring values
    // (behind the square where there is room, so that X and X^T are made in one go)
    const int plane = width * mp * 2;                           // halves
    const bool apart = plane * 4 + mp * mp * 4 + width * (mp + 1) * 4 <= kSmallLds;
    float* u = apart ? reinterpret_cast<float*>(sq + mp * mp * 2) : reinterpret_cast<float*>(x);
    // [width][mp + 1]: lanes along either side hit other banks
    const int j0 = strip * width, rows = I.tall ? width : mp, across = I.tall ? mp : width;
    double s = 0.0;
    float big = 0.0f;
    for (int a = wave; a < rows; a += kSmallWaves) {
      for (int c = lane; c < across; c += 64) {
        const int i = I.tall ? c : a, j = I.tall ? a : c;
        float v = 0.0f;
        if (i < I.m && j0 + j < I.n) {
          const int64_t e = base + (I.tall ? (int64_t)(j0 + j) * I.m + i : (int64_t)i * I.n + j0 + j);
          if (I.mom) I.mom[e] = fmaf(mo.mu, I.mom[e], mo.rest * (float)static_cast<const T*>(I.src)[e]);
          v = source_value<T>(I, e, mo);
          s = fma((double)v, (double)v, s);
          big = fmaxf(big, fabsf(v));
        }
        u[j * (mp + 1) + i] = v;
      }
    }
    const SumMax all = block_sum_max(s, big, red, redf);
    s = all.sum;
    big = all.max;
    const int e = big > 0.0f ? (big < INFINITY ? ilogbf(big) + 1 : 0) : kNoExponent;
    const int per = mp / 4, across4 = 64 / per, jl = lane / per, il = (lane - jl * per) * 4;       // lanes a column of X, columns a wave
    if (jl < across4) {
      for (int j = wave * across4 + jl; j < width; j += kSmallWaves * across4) {
        const float* t = u + j * (mp + 1) + il;
        const float v[4] = {ldexpf(t[0], -e), ldexpf(t[1], -e), ldexpf(t[2], -e), ldexpf(t[3], -e)};
        store_pieces(xt, j, il, mt, v, kFirst);
      }
    }
    if (!apart) __syncthreads();
    for (int jb = wave; jb < width / 4; jb += kSmallWaves) {
      for (int i = lane; i < mp; i += 64) {
        if (apart) {
          const float* t = u + jb * 4 * (mp + 1) + i;
          const float v[4] = {ldexpf(t[0], -e), ldexpf(t[mp + 1], -e), ldexpf(t[2 * (mp + 1)], -e), ldexpf(t[3 * (mp + 1)], -e)};
          store_pieces(x, i, jb * 4, wt, v, kFirst);
        } else {
          _Float16* to = x + piece_at<2>(i, jb * 4, wt);
          const _Float16* from = xt + piece_at<2>(jb * 4, i, mt);        // rows of X^T lie 8 halves apart
          f16x4 hi, lo;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            hi[r] = from[8 * r];
            lo[r] = from[8 * r + 512];
          }
          *reinterpret_cast<f16x4*>(to) = hi;
          *reinterpret_cast<f16x4*>(to + 512) = lo;
        }
      }
    }
    own_e = e;
    squares = s;
    if constexpr (!SINGLE) {
      __syncthreads();
      if (tid == 0) { sums[strip] = s; exps[strip] = e; }
      // X^T's pieces to memory
      const f32x4* from = reinterpret_cast<const f32x4*>(xt);
      f32x4* to = at<f32x4>(ws, strip_bytes(I) * strip);
      for (int k = tid; k < width * mp / 4; k += kSmallThreads) to[k] = from[k];
    }
  } else {
    // X^T's pieces on their way to LDS, 1 KB a wave and turn, while the sums and the parts below are read
    const char* from = ws + strip_bytes(I) * strip + lane * 16;
    for (int k = wave * 1024; k < width * mp * 4; k += kSmallWaves * 1024)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + k),
                                       (__attribute__((address_space(3))) void*)(lds + k), 16, 0, 0);
    if (step > 0) {
      // the strips' parts of S; the first step's have a factor each, see below
#pragma unroll
      for (int q = 0; q < kTriWave; ++q) {
        if (ta[q] < 0) continue;
        const f32x4* part = at<const f32x4>(ws, off_parts(I, step & 1)) + (wave + q * kSmallWaves) * 64 + lane;
        for (int p0 = 0; p0 < I.strips; p0 += kPartsAhead) {
          f32x4 v[kPartsAhead];
#pragma unroll
          for (int p = 0; p < kPartsAhead; ++p) v[p] = part[(int64_t)min(p0 + p, I.strips - 1) * ntri * 64];
#pragma unroll
          for (int p = 0; p < kPartsAhead; ++p)
            if (p0 + p < I.strips) parts[q] += v[p];
        }
      }
    }
    double s = 0.0;
    int most = kNoExponent;
    for (int k = lane; k < I.strips; k += 64) {
      s += sums[k];
      most = max(most, exps[k]);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      s += __shfl_xor(s, d);
      most = max(most, __shfl_xor(most, d));
    }
    squares = s;
    own_e = exps[strip];
    all_e = most;
  }
  const Start start = start_of(squares, eps, own_e, few);
  Norm nm;
  nm.factor = 1.0f;
  nm.ex = SINGLE ? start.ex : start_of(squares, eps, all_e, few).ex;        // the same in all strips
  const float inv_s = 1.0f / sc.s, inv_q = 1.0f / sc.q;
  if (SINGLE || step < 0) __syncthreads();

  // this wave's blocks of X in fp32: lane l holds row 16 ti + l % 16, columns 16 tj + 4 (l / 16) ..
  float xv[kUpdateWave][4];

  for (int k = SINGLE ? 0 : step; k >= 0 && k < steps; ++k) {
    // X over its pieces; U 2^-e holds the first step's
    const float inv_x = k == 0 ? start.first * (1.0f / kFirst) : 1.0f / x_scale(nm, sc, k);
    // S
#pragma unroll
    for (int q = 0; q < kTriWave; ++q) {
      if (ta[q] < 0) continue;
      f32x4 r = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (SINGLE) {
        r = block_product(x, x, ta[q], tb[q], wt, few) * (inv_x * inv_x);
      } else {
        if (k == 0) {
          // a strip's factor by a lane of its own
          const f32x4* part = at<const f32x4>(ws, off_parts(I, 0)) + (wave + q * kSmallWaves) * 64 + lane;
          for (int p0 = 0; p0 < I.strips; p0 += 64) {
            const float own = p0 + lane < I.strips ? start_of(squares, eps, exps[p0 + lane], few).first * (1.0f / kFirst) : 0.0f;
            const int n = min(64, I.strips - p0);
            for (int p1 = 0; p1 < n; p1 += kPartsAhead) {
              f32x4 v[kPartsAhead];
#pragma unroll
              for (int p = 0; p < kPartsAhead; ++p) v[p] = part[(int64_t)(p0 + min(p1 + p, n - 1)) * ntri * 64];
#pragma unroll
              for (int p = 0; p < kPartsAhead; ++p) {
                if (p1 + p >= n) continue;
                const float f1 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(own), p1 + p));
                r += v[p] * (f1 * f1);
              }
            }
          }
        } else {
          r = parts[q] * (inv_x * inv_x);
        }
      }
      float v[4] = {r[0], r[1], r[2], r[3]};
      store_symmetric(sq, mt, ta[q] == tb[q], ta[q] * 16, tb[q] * 16, v, sc.s);
    }
    if constexpr (!SINGLE) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // X^T has landed
    __syncthreads();
    // R = b S + c S S, in the place of S once every wave has read it
    float rv[kTriWave][4];
#pragma unroll
    for (int q = 0; q < kTriWave; ++q) {
      if (ta[q] < 0) continue;
      const f32x4 r = block_product(sq, sq, ta[q], tb[q], mt, few);
      float o[4];
      load_pieces<2>(sq, tb[q] * 16 + (lane & 15), ta[q] * 16 + 4 * (lane >> 4), mt, o, inv_s);
#pragma unroll
      for (int i = 0; i < 4; ++i) rv[q][i] = fmaf(kc.c * inv_s * inv_s, r[i], kc.b * o[i]);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kTriWave; ++q)
      if (ta[q] >= 0) store_symmetric(sq, mt, ta[q] == tb[q], ta[q] * 16, tb[q] * 16, rv[q], sc.q);
    __syncthreads();
    // X <- a X + R X, likewise
    const bool last = k + 1 == steps;
    const float next = x_scale(nm, sc, k + 1), unscale = inv_x * inv_q;
    // (with few rows X is what its pieces hold in every step: R follows from those, and a X + R X of another X is off by |a + R|
    // times their rounding where the step itself forgets it.  With more the copy in fp32 saves LDS reads)
    if (!SINGLE || k == 0 || few) {
#pragma unroll
      for (int q = 0; q < kUpdateWave; ++q) {
        if (ti[q] >= rb) continue;
        load_pieces<2>(xt, tj[q] * 16 + 4 * (lane >> 4) + (lane & 3), ti[q] * 16 + (lane & 12), mt, xv[q], inv_x);
        quad_transpose(xv[q]);
      }
    }
#pragma unroll
    for (int q = 0; q < kUpdateWave; ++q) {
      if (ti[q] >= rb) continue;
      const f32x4 r = block_product(xt, sq, tj[q], ti[q], mt, few);
#pragma unroll
      for (int i = 0; i < 4; ++i) xv[q][i] = fmaf(kc.a, xv[q][i], r[i] * unscale);
    }
    if (last) {
#pragma unroll 1
      for (int q = 0; q < kUpdateWave; ++q) {
        if (ti[0] >= rb) break;
        const int j = tj[0] * 16 + 4 * (lane >> 4) + (lane & 3), i = ti[0] * 16 + (lane & 12);
        const int j4 = tj[0] * 16 + 4 * (lane >> 4), i1 = ti[0] * 16 + (lane & 15);
        if (I.tall) {
          quad_transpose(xv[0]);
          const int jj = strip * width + j;
          if (jj < I.n) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (i + r < I.m) put<T>(I, base + (int64_t)jj * I.m + i + r, xv[0][r], lr, f);
          }
        } else {
          const int jj = strip * width + j4;
          if (i1 < I.m) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (jj + r < I.n) put<T>(I, base + (int64_t)i1 * I.n + jj + r, xv[0][r], lr, f);
          }
        }
        // the next block moves up, so that this code is there once
#pragma unroll
        for (int n = 0; n + 1 < kUpdateWave; ++n) {
          ti[n] = ti[n + 1];
          tj[n] = tj[n + 1];
#pragma unroll
          for (int r = 0; r < 4; ++r) xv[n][r] = xv[n + 1][r];
        }
        ti[kUpdateWave - 1] = rb;
      }
      return;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kUpdateWave; ++q) {
      if (ti[q] >= rb) continue;
      float v[4];
      split_pieces(xv[q], next, v);
      store_packed(x, ti[q] * 16 + (lane & 15), tj[q] * 16 + 4 * (lane >> 4), wt, v);
      quad_transpose(v);
      store_packed(SINGLE ? xt : at<_Float16>(ws, strip_bytes(I) * strip), tj[q] * 16 + 4 * (lane >> 4) + (lane & 3),
                   ti[q] * 16 + (lane & 12), mt, v);
    }
    __syncthreads();
    if constexpr (!SINGLE) break;
  }
  if constexpr (!SINGLE) {
    // this strip's part of the next S, as the pieces multiply
    f32x4* part = at<f32x4>(ws, off_parts(I, (step + 1) & 1)) + (int64_t)strip * ntri * 64;
#pragma unroll
    for (int q = 0; q < kTriWave; ++q)
      if (ta[q] >= 0) part[(wave + q * kSmallWaves) * 64 + lane] = block_product(x, x, ta[q], tb[q], wt, few);
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------

int round_up(int64_t v, int a) { return (int)((v + a - 1) / a * a); }

void choose_path(Item& I, Path least);

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
  // a block of the norm takes at least 4096 values; all matrices together about eight blocks a compute unit
  const int64_t parts = (I.size + kThreads * 16 - 1) / (kThreads * 16), most = kSumsMax / (I.batch < 4 ? I.batch : 4);
  I.nsum = (int)(parts < most ? parts : most);
  // Blocks of 128 x 128 read half as much for a product as blocks of 64 x 64, but need more inner tiles to get going and more
  // blocks to fill the chip.  Where rows times blocks reach 2^19, us in blocks of 64 and of 128: 2048 x 8192 bf16 1417 and 1120, fp32
  // 2533 and 1859; 2048 x 2048 fp32 794 and 753; 1024 x 8192 bf16 364 and 357; 512 x 32768 fp32 727 and 721; and below it: 1500 x
  // 3000 bf16 473 and 486; 1024 x 4096 bf16 287 and 302; 512 x 16384 fp32 419 and 429; 4 x 1000 x 771 fp16 294 and 311.
  constexpr int64_t kBigBlocks = 1 << 19;
  const int64_t big = (int64_t)((I.mp + 127) / 128) * ((I.np + 127) / 128) * I.batch;
  I.bt = I.m > 64 && I.mp * big >= kBigBlocks ? 128 : 64;
  // Among squares only the upper triangle's blocks are computed: 128 x 128 ones where rows times those reach 600000 and a matrix has four
  // rows of them, of which the diagonal's are half wasted.  In blocks of 64 and of 128: 2600 x 2600 bf16 1457 and 1243 us, 4096 x 4096
  // 5540 and 4286, 3 x 2048 x 2048 1841 and 1601, 40 x 1000 x 1000 3555 and 3041, 64 x 700 x 700 fp32 2315 and 2297; and otherwise:
  // 2300 x 2300 bf16 985 and 1032, 2 x 2048 x 2048 1310 and 1367, 8 x 1024 x 1024 742 and 812, 32 x 700 x 700 fp32 1223 and 1279, 2000 x
  // 129 x 129 2918 and 3118.
  constexpr int64_t kBigSquares = 600000;
  const int64_t t128 = (I.mp + 127) / 128, tri = t128 * (t128 + 1) / 2 * I.batch;
  I.bts = t128 >= 4 && I.mp * tri >= kBigSquares ? 128 : 64;
  // splits of the long axis: two blocks a compute unit, at least four inner tiles each
  const int kt = I.np / 32, tiles = tri_tiles(I);
  int64_t chunks = (512 + (int64_t)tiles * I.batch - 1) / ((int64_t)tiles * I.batch);
  if (chunks > kt / 4) chunks = kt / 4;
  if (chunks < 1) chunks = 1;
  I.kchunk = (kt + (int)chunks - 1) / (int)chunks;
  I.chunks = (kt + I.kchunk - 1) / I.kchunk;
  choose_path(I, kSingle);
  return I;
}

// The small kernels' path of a matrix, or a slower-starting one: `least` is kSingle, kStrips or kTiles.
void choose_path(Item& I, Path least) {
  // the widest strip whose X, X^T and square fit the LDS and the waves' registers
  const int room = I.mp <= kSmallRows ? (kSmallLds - I.mp * I.mp * 4) / (I.mp * 8) / 32 * 32 : 0;
  const int hold = kUpdateWave * kSmallWaves * 256 / I.mp, widest = room < hold ? room : hold;
  I.strips = 1;
  I.width = I.np;
  I.path = kTiles;
  if (I.m == 1) {
    I.path = I.n <= 65536 && least < kTiles ? kSingle : kVector;
  } else if (I.mp <= kSmallRows && least < kTiles) {
    if (I.np <= widest && least == kSingle) {
      I.path = kSingle;
    } else {
      // strips of 64 columns, of 128 where there would be many: a block of the next step reads a part of tri16 KB of each, which
      // has to stay below what the launches that it saves cost
      int width = 64, strips = (I.np + 63) / 64;
      if (I.mp <= 64 && strips * tri16(I.mp) > 512) { width = 128; strips = (I.np + 127) / 128; }
      if ((int64_t)strips * tri16(I.mp) <= 1024) { I.path = kStrips; I.width = width; I.strips = strips; }
    }
  }
  I.ws_stride = I.path == kVector ? (I.nsum * (int64_t)sizeof(double) + 255) / 256 * 256 : I.path == kTiles ? item_bytes(I) : small_bytes(I);
}

// The matrices of one list.  Those that could go alone in fewer launches join the launches of the others that take more of
// them, and vectors beside tiles take part in the launches of the norms and of the pieces: beside those they cost next to
// nothing, on their own their whole time.  Matrices that one block does alone join only where all of them are at most kSinglesJoin:
// more take longer than a launch of their own, and far more workspace.  Beside 60 x 1000, us with them and apart: 128 of 64 x 64 63
// and 78, 256 108 and 78, 4096 851 and 390; beside 300 x 300: 128 of 4 x 6 128 and 133, 256 134 and 132, 4096 398 and 327, 128
// of 64 x 64 142 and 141.  Strips beside tiles gain in any number (256 of 40 x 900: 349 and 900), vectors too (4096 of 50: 128 and 146).
constexpr int64_t kSinglesJoin = 128;
void make_items(const NsMatrix* mats, int count, Items& L) {
  L.n = 0;
  Path most = kSingle;
  int64_t singles = 0;
  for (int j = 0; j < count && j < kItemsMax; ++j) {
    const Item& I = L.it[L.n++] = make_item(mats[j]);
    if (I.m > 1 && I.path > most) most = (Path)I.path;
    if (I.m > 1 && I.path == kSingle) singles += I.batch;
  }
  for (int j = 0; j < L.n; ++j) {
    Item& I = L.it[j];
    if (I.m == 1 ? most == kTiles : I.path < most && (I.path != kSingle || singles <= kSinglesJoin)) choose_path(I, most);
  }
}

int blocks_before(Items& L, int (*count)(const Item&), int times = 1) {
  int total = 0;
  for (int i = 0; i < L.n; ++i) { L.first[i] = total; total += count(L.it[i]) * L.it[i].batch * times; }
  for (int i = L.n; i <= kItemsMax; ++i) L.first[i] = INT_MAX;
  return total;
}
int count_sums(const Item& I) { return I.nsum; }
int count_strips(const Item& I) { return I.strips; }
int count_split(const Item& I) { return I.path == kVector ? I.nsum : ((I.mp + 63) / 64) * ((I.np + 63) / 64); }
int count_tiles(const Item& I) { return ((I.mp + I.bt - 1) / I.bt) * ((I.np + I.bt - 1) / I.bt); }
int count_squares(const Item& I) { return tri_squares(I); }
int count_gram(const Item& I) { return tri_tiles(I) * I.chunks; }
int count_parts(const Item& I) { return I.chunks > 1 ? tri_tiles(I) * (I.bt * I.bt / 1024) : 0; }

template <int THREADS = kThreads, typename K, typename... A>
void launch(K kernel, int blocks, size_t lds, hipStream_t st, const A&... args) {
  if (!blocks) return;
  ensure_dynamic_lds((const void*)kernel, lds);
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(THREADS), lds, st, args...);
}

// the products of all matrices of one block size
template <typename T, int BT>
struct Steps {
  Items& L;
  const NsPlan& p;
  const Scales sc;
  const Finish fin;
  hipStream_t st;

  template <int PX>
  void gram(int step) {
    launch(ns_gram_kernel<BT, PX>, blocks_before(L, count_gram), Product<BT, PX, PX>::kLds, st, L, sc, step);
    Items S = L;                                       // the matrices whose long axis was split
    S.n = 0;
    for (int i = 0; i < L.n; ++i)
      if (L.it[i].chunks > 1) S.it[S.n++] = L.it[i];
    // With many splits four groups of waves share them: fp32 matrices by one group and by four, 8 splits (256 x 1024) 110 and 114 us, 16
    // 118 and 122, 32 137 and 139, 40 151 and 156; 46 164 and 161, 156 (150 x 20000) 195 and 189.
    int most = 0;
    for (int i = 0; i < S.n; ++i) most = S.it[i].chunks > most ? S.it[i].chunks : most;
    const int sums = blocks_before(S, count_parts);
    if (most >= 44) launch<4 * kThreads>(ns_gram_sum_kernel<BT, 4>, sums, 0, st, S, sc);
    else launch(ns_gram_sum_kernel<BT, 1>, sums, 0, st, S, sc);
  }
  // go(the matrices whose squares go in blocks of `bts`, their number of blocks), for each block size there is
  template <int BTS, typename Go>
  void squares_of(int jobs, Go&& go) {
    Items S = L;
    S.n = 0;
    for (int i = 0; i < L.n; ++i)
      if (L.it[i].bts == BTS) S.it[S.n++] = L.it[i];
    const int blocks = blocks_before(S, count_squares, jobs);
    if (blocks) go(S, blocks);
  }
  template <int BTS>
  void poly_in(const NsCoefficients& k, int out) {
    squares_of<BTS>(1, [&](const Items& S, int blocks) {
      launch(ns_poly_kernel<BTS>, blocks, Product<BTS, 2, 2>::kLds, st, S, sc, k, out);
    });
  }
  void poly(float a, int out) {
    poly_in<64>({a, p.k.b, p.k.c}, out);
    poly_in<128>({a, p.k.b, p.k.c}, out);
  }
  template <int BTS>
  void squares_in(const SquareJobs& jobs) {
    squares_of<BTS>(jobs.n, [&](const Items& S, int blocks) {
      launch(ns_square_kernel<BTS>, blocks, Product<BTS, 2, 2>::kLds, st, S, jobs);
    });
  }
  void squares(const SquareJobs& jobs) {
    squares_in<64>(jobs);
    squares_in<128>(jobs);
  }
  template <int PX>
  void update(float a, int square, float scale_m, int from, int step, int next) {
    const int blocks = blocks_before(L, count_tiles);
    constexpr int kLds = Product<BT, PX, 2>::kLds;
    if (next < p.steps) launch(ns_update_kernel<T, BT, PX, false>, blocks, kLds, st, L, sc, a, square, scale_m, from, step, next, fin);
    else launch(ns_update_kernel<T, BT, PX, true>, blocks, kLds, st, L, sc, a, square, scale_m, from, step, next, fin);
  }

  // step by step: S = X X^T, R = b S + c S S, X <- a X + R X
  void plain() {
    for (int k = 0; k < p.steps; ++k) {
      gram<2>(k);
      poly(0.0f, kQ);
      update<2>(p.k.a, kQ, sc.q, k & 1, k, k + 1);
    }
  }

  // Up to three steps composed in the square matrices, then one product with X: with Q = a I + b S + c S S the step takes X to
  // Q X and S to Q S Q, and all of these commute.  Three products along the long axis for five steps instead of ten.
  // Rounding errors of S in the small singular directions grow by a^2 a step, and Q and its products carry their multiple of one
  // through the sums of the matrix instructions: X is 4e-6 (4 x 1000 x 771) to 6e-6 (2048 x 8192) off before it is rounded, against
  // the 2^-9 or 2^-12 of a 16-bit result, and a new S is formed after three steps.  X keeps two pieces between the segments: one
  // (2^-12 of each value) would move one bf16 result in twenty to its neighbour.  2048 x 8192 bf16: 1096 us, 1007 with one.
  void composed() {
    for (int k = 0, part = 0; k < p.steps; ++part) {
      const int start = k, n = p.steps - k < 3 ? p.steps - k : 3;
      if (part == 0) gram<1>(0);
      else gram<2>(start);
      int cur = kP0;                                     // the composed steps so far; the first one is its own Q
      float scale = sc.q;
      for (int i = 0; i < n; ++i, ++k) {
        const int q = i == 0 ? kP0 : kQ;
        poly(p.k.a, q);
        SquareJobs jobs{};
        if (i > 0) {
          const int out = cur == kP0 ? kP1 : kP0;
          jobs.j[jobs.n++] = {kQ, cur, out, sc.p / (sc.q * scale)};
          cur = out;
          scale = sc.p;
        }
        if (i + 1 < n) jobs.j[jobs.n++] = {q, kS, kT, sc.t / (sc.q * sc.s)};
        if (jobs.n) squares(jobs);
        if (i + 1 < n) {
          SquareJobs next{};
          next.j[next.n++] = {kT, q, kS, sc.s / (sc.t * sc.q)};
          squares(next);
        }
      }
      if (part == 0) update<1>(0.0f, cur, scale, 0, 0, k);
      else update<2>(0.0f, cur, scale, part & 1, start, k);
    }
  }
};

template <typename T, int BT>
void run_products(Items& L, const NsPlan& p, const Scales& sc, const Finish& fin, hipStream_t st) {
  if (!L.n) return;
  Steps<T, BT> s{L, p, sc, fin, st};
  if constexpr (sizeof(T) == 4) s.plain();
  else s.composed();
}

template <typename T>
void run_items(const Items& L, const NsPlan& p, hipStream_t st) {
  const Momentum mo{p.momentum, p.momentum_rest, p.nesterov};
  const Finish fin{p.lr_dev, p.lr, p.decay};
  Items V, O, S, M, B, N;         // vectors, single blocks, strips, products in blocks of 64 and of 128; whose norm goes first
  V.n = O.n = S.n = M.n = B.n = N.n = 0;
  size_t lds = 0;
  for (int i = 0; i < L.n; ++i) {
    const Item& I = L.it[i];
    Items& to = I.path == kVector ? V : I.path == kSingle ? O : I.path == kStrips ? S : I.bt == 128 ? B : M;
    to.it[to.n++] = I;
    if (I.path == kVector || I.path == kTiles) N.it[N.n++] = I;
    else if (I.m > 1) {
      size_t need = (size_t)I.width * I.mp * 8 + (size_t)I.mp * I.mp * 4;
      const size_t apart = need + (size_t)I.width * (I.mp + 1) * 4;
      if (apart <= kSmallLds) need = apart;
      if (need > lds) lds = need;
    }
  }
  // vectors take part in the first launch of strips, or the second of tiles (see make_items)
  Items F = S;
  if (S.n) {
    O.n = 0;
    for (int i = 0; i < L.n; ++i)
      if (L.it[i].path == kSingle) (L.it[i].m == 1 ? F.it[F.n++] : O.it[O.n++]) = L.it[i];
  }
  // the small kernels form R, the composed products Q
  const Scales small{p.scale_x, p.scale_s, p.scale_r, p.scale_t, p.scale_p, p.growth};
  launch<kSmallThreads>(ns_small_kernel<T, true>, blocks_before(O, count_strips), lds, st, O, mo, p.eps, p.k, p.steps, 0, small,
                        fin);
  if (S.n)
    for (int k = -1; k < p.steps; ++k)
      launch<kSmallThreads>(ns_small_kernel<T, false>, blocks_before(k < 0 ? F : S, count_strips), lds, st, k < 0 ? F : S, mo, p.eps, p.k,
                            p.steps, k, small, fin);
  launch(ns_norm_kernel<T>, blocks_before(N, count_sums), 0, st, N, mo);
  const Scales sc{p.scale_x, p.scale_s, sizeof(T) == 4 ? p.scale_r : p.scale_q, p.scale_t, p.scale_p, p.growth};
  if (!M.n && !B.n) launch(ns_vector_kernel<T>, blocks_before(V, count_sums), 0, st, V, mo, p.eps, p.k, p.steps, fin);
  for (Items* X : {&M, &B}) {
    if (!X->n) continue;
    Items W = *X;
    for (int i = 0; i < V.n; ++i) W.it[W.n++] = V.it[i];
    V.n = 0;
    launch(ns_split_kernel<T, sizeof(T) == 2>, blocks_before(W, count_split), 0, st, W, mo, p.eps, sc, p.k, p.steps, fin);
  }
  run_products<T, 64>(M, p, sc, fin, st);
  run_products<T, 128>(B, p, sc, fin, st);
}

}  // namespace

const char* ns_refusal(const NsMatrix& M) {
  if (M.rows < 1 || M.cols < 1 || M.batch < 1) return "empty or negative sizes";
  const int64_t m = M.rows < M.cols ? M.rows : M.cols, n = M.rows < M.cols ? M.cols : M.rows;
  if (m > 32768 || n > (int64_t)1 << 30 || (m > 1 && n > (int64_t)1 << 24)) return "a side is too long (short side over 32768, or long side over 2^24, 2^30 for a vector)";
  // a launch holds fewer than 2^32 threads, over the 16 entries that may share it in blocks of up to 1024
  const int64_t tiles = ((m + 63) / 64) * ((n + 63) / 64), values = (m * n + 4095) / 4096;
  const int64_t sums = values < kSumsMax ? values : kSumsMax, most = m > 1 && tiles > sums ? tiles : sums;
  if (most > (int64_t)1 << 18 || M.batch > (most < 1 << 17 ? ((int64_t)1 << 17) / most : 1)) return "too many tiles in one stack";
  return nullptr;
}

bool ns_scales(const NsCoefficients& k, int steps, NsPlan* p) {
  // the largest |x (a + b x^2 + c x^4)|, |b s + c s^2| and |a + b s + c s^2| over the singular values a step can meet, by interval ends and
  // the inner extrema, step by step from [0, 1]
  for (const float v : {k.a, k.b, k.c})
    if (!(std::fabs(v) < 4096.0f)) return false;
  double top = 1.0, all = 1.0, rmax = 0.0, qmax = 1.0;
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
    auto q = [&](double s) { return std::fabs(k.a + s * (k.b + k.c * s)); };
    qmax = std::fmax(qmax, std::fmax(q(0.0), q(T * T)));
    if (k.c != 0.0f) {
      const double s = -(double)k.b / (2.0 * k.c);
      if (s > 0.0 && s < T * T) qmax = std::fmax(qmax, q(s));
    }
    top = next;
    all = std::fmax(all, top);
    if (!(all < 64.0) || !(rmax < 4096.0) || !(qmax < 4096.0)) return false;
  }
  // 1.01: rounding can carry a singular value past the bound
  const int kx = (int)std::ceil(std::log2(all * 1.01)), kr = (int)std::ceil(std::log2(std::fmax(rmax, 1.0) * 1.01));
  p->scale_x = std::ldexp(1.0f, 15 - kx);
  p->scale_s = std::ldexp(1.0f, 15 - 2 * kx);
  p->scale_r = std::ldexp(1.0f, 15 - kr);
  const int kq = (int)std::ceil(std::log2(qmax * 1.01)), kp = (int)std::ceil(3.0 * std::log2(qmax * 1.01));
  p->growth = kq;
  p->scale_q = std::ldexp(1.0f, 15 - kq);
  p->scale_t = std::ldexp(1.0f, 15 - kq - 2 * kx);
  p->scale_p = std::ldexp(1.0f, 15 - kp);
  return true;
}

size_t ns_ws_bytes(const NsMatrix* mats, int count) {
  Items L;
  make_items(mats, count, L);
  size_t sum = 0;
  for (int j = 0; j < L.n; ++j) sum += (size_t)L.it[j].ws_stride * L.it[j].batch;
  return sum;
}

void launch_ns(int dtype, const NsMatrix* mats, int count, const NsPlan& p, void* ws, hipStream_t st) {
  Items L;
  make_items(mats, count, L);
  char* at = static_cast<char*>(ws);
  for (int j = 0; j < L.n; ++j) {
    L.it[j].ws = at;
    at += L.it[j].ws_stride * L.it[j].batch;
  }
  switch (dtype) {
    case kNormF32: run_items<float>(L, p, st); break;
    case kNormBf16: run_items<__bf16>(L, p, st); break;
    default: run_items<_Float16>(L, p, st); break;
  }
}

}  // namespace pdekan
