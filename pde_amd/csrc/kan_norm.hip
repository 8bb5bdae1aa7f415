// Group norm followed by an activation, channels last: on plain values [n][s][C] in fp32, bf16 or fp16 (statistics of a
// group run over the s positions and the C / groups channels of a sample) and on derivative jets [n][C][J] in fp32
// (statistics per point).  Sums, statistics and every intermediate are fp32, sums over a sample's positions 64-bit beyond 32 rows (the
// statistics' throughout); a 16-bit tensor is rounded once, at the store.
//
//   z = (x - mean) r,  r = (var + eps)^-1/2,  y = f(w z + b)
//   backward: p = gy f',  gb = sum p,  gw = sum p z,  q = w p,  gx = r (q - mean(q) - z mean(q z))
//
// Two families of kernels:
//   rows (norm_rows_*, norm_jet_*): one point at a time, a group of a point = L adjacent lanes, K vectors a lane.  The
//     data of a group stays in registers between the statistics and the result: x is read once, y written once.
//   grids (norm_grid_*): samples of many positions.  Launch 1 leaves partial statistics per chunk of positions, launch 2
//     merges them (Chan's formula) and applies; the second reading of x comes mostly from the caches.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cstdint>

#include "kan_launch.h"
#include "kan_wave.h"

namespace pdekan {
namespace {

constexpr int kThreads = 256;

template <typename T, int N> struct VecOf { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T> struct VecOf<T, 1> { typedef T type; };

template <typename T, int N>
__device__ __forceinline__ void widen(const typename VecOf<T, N>::type& r, float (&v)[N]) {
  if constexpr (N == 1) v[0] = (float)r;
  else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)r[i];
  }
}
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[N]) {
  widen<T, N>(*reinterpret_cast<const typename VecOf<T, N>::type*>(p), v);
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[N]) {
  typename VecOf<T, N>::type r;
  if constexpr (N == 1) r = (T)v[0];
  else {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = (T)v[i];
  }
  *reinterpret_cast<typename VecOf<T, N>::type*>(p) = r;
}

// sum over the L adjacent lanes of a group (L a power of two, groups aligned to L), in every lane of the group
template <int L>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (L >= 2) v += dpp_move<0xB1>(v);
  if constexpr (L >= 4) v += dpp_move<0x4E>(v);
  if constexpr (L >= 8) v += dpp_move<0x141>(v);
  if constexpr (L >= 16) v += dpp_move<0x140>(v);
  if constexpr (L >= 32) v = sum_xor16(v);
  if constexpr (L >= 64) v = sum_xor32(v);
  return v;
}

// exp(S u), S = -1 or 2: 2^p with p = S u log2(e) rounded, for FULL (fp32 tensors) times what the rounding left out: |p| steps of
// 2^-24, which results of 16 bits do not show (8 x 4096 x 320 bf16 SiLU, all four launches 70 us with and 64 without)
template <int S, bool FULL>
__device__ __forceinline__ float exp_times(float u) {
  constexpr float kHi = S * 1.44269502162933349609375f, kLo = S * 1.9259629911266e-8f;      // log2(e) in two parts
  if constexpr (!FULL) return __builtin_amdgcn_exp2f(u * kHi);
  const float p = u * kHi, rest = fmaf(u, kLo, fmaf(u, kHi, -p));
  const float e = __builtin_amdgcn_exp2f(p);
  return fabsf(p) < 127.0f ? fmaf(e, rest * 0.6931471805599453f, e) : e;      // (0, infinity and NaN as they are)
}

// f and its first ORDER derivatives at u.
//   tanh: 1 - q with q = 2 / (exp(2|u|) + 1), slope q (2 - q), which keeps its bits where tanh is nearly 1; below 0.625, where 1 - q
//   loses some, u + u^3 p(u^2) with p a polynomial fitted for the least relative error: of degree 4 (5e-9), or for tensors of 16 bits,
//   which take the slope as 1 - t^2 too, of degree 3 (1.4e-7)
//   silu: u s, s = 1 / (1 + exp(-u)); 1 - s = exp(-u) s where s is nearly 1
template <int ACT, int ORDER, bool FULL>
__device__ __forceinline__ void activation(float u, float (&f)[ORDER + 1]) {
  if constexpr (ACT == kNormActTanh) {
    const float u2 = u * u, a = fabsf(u);
    const float poly = FULL ? fmaf(u2, fmaf(u2, fmaf(u2, fmaf(u2, -0.00571705587f, 0.0206505991f), -0.0537435003f), 0.133314908f), -0.333332837f)
                            : fmaf(u2, fmaf(u2, fmaf(u2, 0.0152269052f, -0.0519716218f), 0.133087143f), -0.333323747f);
    const float inner = fmaf(u * u2, poly, u);
    const bool near = a < 0.625f;
    float t, slope;
    if constexpr (FULL) {
      // (43: finite; a NaN stays one.  The value alone loses at most half a step without the exponential's rest, the slope more)
      const float d = exp_times<2, (ORDER > 0)>(a > 43.0f ? 43.0f : a) + 1.0f;
      float q = __builtin_amdgcn_rcpf(d);
      q = 2.0f * fmaf(fmaf(-d, q, 1.0f), q, q);
      t = near ? inner : copysignf(1.0f - q, u);
      slope = near ? fmaf(-t, t, 1.0f) : q * (2.0f - q);
    } else {
      t = near ? inner : fmaf(-2.0f, __builtin_amdgcn_rcpf(exp_times<2, false>(u) + 1.0f), 1.0f);
      slope = fmaf(-t, t, 1.0f);
    }
    f[0] = t;
    if constexpr (ORDER >= 1) f[1] = slope;
    if constexpr (ORDER >= 2) f[2] = -2.0f * t * f[1];
    if constexpr (ORDER >= 3) f[3] = f[1] * (6.0f * t * t - 2.0f);
  } else if constexpr (ACT == kNormActSilu) {
    const float e = exp_times<-1, FULL>(u), s = __builtin_amdgcn_rcpf(1.0f + e);
    f[0] = u * s;
    if constexpr (ORDER >= 1) {
      const float d = s * (!FULL || u < 0.0f ? 1.0f - s : e * s), h = 1.0f - 2.0f * s;
      f[1] = fmaf(u, d, s);
      if constexpr (ORDER >= 2) f[2] = d * fmaf(u, h, 2.0f);
      if constexpr (ORDER >= 3) f[3] = d * (3.0f * h + u * (1.0f - 6.0f * d));
    }
  } else {
    f[0] = u;
    if constexpr (ORDER >= 1) f[1] = 1.0f;
    if constexpr (ORDER >= 2) f[2] = 0.0f;
    if constexpr (ORDER >= 3) f[3] = 0.0f;
  }
}

// body(IntC<kind>) for the activation `act`, which is the same in the whole grid: one branch a kernel, not one a value
template <int V> struct IntC { static constexpr int value = V; };
template <typename F>
__device__ __forceinline__ void by_activation(int act, F&& body) {
  if (act == kNormActTanh) body(IntC<kNormActTanh>{});
  else if (act == kNormActSilu) body(IntC<kNormActSilu>{});
  else body(IntC<kNormActIdentity>{});
}

// Which (sample, group) a lane group of a rows kernel takes.  A block holds 256 / L lane groups: `gpb` groups of `ppb`
// samples; blocks that share a range of groups walk the samples with stride npb * ppb, so a lane keeps its channels
// (their weights and the sums of their gradients stay in registers).  A sample has s positions (jets: one).
struct RowMap { int64_t n; int s, C, G, cpg, gpb, ppb, gchunks, npb; };

struct RowPlace { int g, pi; int64_t p, step; bool on; };
template <int L>
__device__ __forceinline__ RowPlace row_place(const RowMap& m) {
  const int slot = threadIdx.x / L;
  const int gi = slot % m.gpb, pi = slot / m.gpb;
  const int gc = blockIdx.x % m.gchunks, pb = blockIdx.x / m.gchunks;
  RowPlace r;
  r.g = gc * m.gpb + gi;
  r.pi = pi;
  r.on = pi < m.ppb && r.g < m.G;
  r.p = (int64_t)pb * m.ppb + pi;
  r.step = (int64_t)m.npb * m.ppb;
  return r;
}

// The block's sums of gw / gb over its samples, in a fixed order, into a row of part [npb * s][2][C] for each position
// (npb * s = 1: gw and gb themselves).  Lane groups of the same group of channels sit gpb slots apart.
template <int N, int L>
__device__ __forceinline__ void row_grad_out(const RowMap& m, const RowPlace& r, const float (&gw)[N], const float (&gb)[N],
                                             int c0, bool valid, float* part_w, float* part_b, float (*red)[N + 1]) {
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) red[threadIdx.x][i] = which ? gb[i] : gw[i];
    __syncthreads();
    float* part = which ? part_b : part_w;
    if (part && r.on && r.pi == 0 && valid) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float s = red[threadIdx.x][i];
        for (int k = 1; k < m.ppb; ++k) s += red[threadIdx.x + k * m.gpb * L][i];
        part[c0 + i] = s;
      }
    }
  }
}

// Points (and samples of up to 512 values a group): a group in the registers of L lanes, so x (and gy) is read once and y (gx)
// written once, with 16-byte accesses where the tensors allow them.  HBM bounds it.  2^19 x 256 fp32, groups of 32, tanh:
// forward 212 us (best of 20: 193; 1.07 GB, 5.1 TB/s), backward 368 (360; 1.61 GB, 4.4 TB/s); bf16 135 and 199 (4.0 TB/s); a large copy
// reaches 5.0 TB/s.  10000 x 64: 5.1 us of launch and latency.
template <typename T, int VEC, int L, int K, bool BWD>
__global__ void __launch_bounds__(kThreads) norm_rows_kernel(RowMap m, const T* __restrict__ x, const T* __restrict__ gy,
                                                             const float* __restrict__ w, const float* __restrict__ b,
                                                             float eps, int act, T* __restrict__ out,
                                                             float* part_w, float* part_b, int part_stride) {
  __shared__ float red[BWD ? kThreads : 1][VEC + 1];
  const RowPlace r = row_place<L>(m);
  const int lane = threadIdx.x % L;
  const float inv = 1.0f / (float)(m.cpg * m.s);
  const int nvg = m.cpg / VEC, nv = nvg * m.s;
  bool valid[K];
  int off[K], pos[K];
  float wv[K][VEC], bv[K][VEC], gwv[K][VEC], gbv[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int v = lane + L * k;
    valid[k] = r.on && v < nv;
    pos[k] = m.s == 1 ? 0 : v / nvg;
    const int c0 = r.g * m.cpg + (v - pos[k] * nvg) * VEC;
    off[k] = pos[k] * m.C + c0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      wv[k][i] = valid[k] && w ? w[c0 + i] : 1.0f;
      bv[k][i] = valid[k] && b ? b[c0 + i] : 0.0f;
      gwv[k][i] = gbv[k][i] = 0.0f;
    }
  }
  by_activation(act, [&](auto kind) {
    constexpr int ACT = decltype(kind)::value;
    if (!r.on) return;
    for (int64_t p = r.p; p < m.n; p += r.step) {
      const int64_t at = p * m.s * m.C;
      float e[K][VEC], q[K][VEC];
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[k][i] = q[k][i] = 0.0f;
        if (valid[k]) {
          load_vec<T, VEC>(x + at + off[k], e[k]);
          if constexpr (BWD) load_vec<T, VEC>(gy + at + off[k], q[k]);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) s += e[k][i];
      }
      const float mean = group_sum<L>(s) * inv;
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          e[k][i] = valid[k] ? e[k][i] - mean : 0.0f;
          v = fmaf(e[k][i], e[k][i], v);
        }
      const float rs = rsqrtf(fmaf(group_sum<L>(v), inv, eps));
      if constexpr (!BWD) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            float f[1];
            activation<ACT, 0, sizeof(T) == 4>(fmaf(e[k][i] * rs, wv[k][i], bv[k][i]), f);
            e[k][i] = f[0];
          }
          if (valid[k]) store_vec<T, VEC>(out + at + off[k], e[k]);
        }
      } else {
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float z = e[k][i] * rs;
            float f[2];
            activation<ACT, 1, sizeof(T) == 4>(fmaf(z, wv[k][i], bv[k][i]), f);
            const float pv = q[k][i] * f[1];
            gbv[k][i] += pv;
            gwv[k][i] = fmaf(pv, z, gwv[k][i]);
            q[k][i] = pv * wv[k][i];
            s1 += q[k][i];
            s2 = fmaf(q[k][i], z, s2);
            e[k][i] = z;
          }
        s1 = group_sum<L>(s1) * inv;
        s2 = group_sum<L>(s2) * inv;
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) e[k][i] = rs * (q[k][i] - s1 - e[k][i] * s2);
          if (valid[k]) store_vec<T, VEC>(out + at + off[k], e[k]);
        }
      }
    }
  });
  if constexpr (BWD) {
    if (part_w || part_b) {
      const int64_t row = (int64_t)(blockIdx.x / m.gchunks) * m.s;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int64_t at = (row + pos[k]) * part_stride;
        row_grad_out<VEC, L>(m, r, gwv[k], gbv[k], off[k] - pos[k] * m.C, valid[k], part_w ? part_w + at : nullptr,
                             part_b ? part_b + at : nullptr, red);
      }
    }
  }
}

// Jets.  Slots of a channel: value x, first derivatives x'_d (d < ND), second derivatives x''_d (d < NS), along each
// direction d the chain rule of the norm and of the activation.  With e, f, s the slots less their means over the group,
// V = mean(e^2) + eps, A = mean(e f), B = mean(f^2 + e s):
//   r = V^-1/2,  r' = -r^3 A,  r'' = -r^3 B + 3 r^5 A^2
//   z = e r,  z' = f r + e r',  z'' = s r + 2 f r' + e r'',  u = w z + b, u' = w z', u'' = w z''
//   y = F(u),  y' = F1 u',  y'' = F2 u'^2 + F1 u''
// Backward (h = cotangent times w, on z, z', z''):
//   gu'' = F1 gy'', gu' = F1 gy' + 2 F2 u' gy'', gu = F1 gy + sum_d F2 u' gy' + (F3 u'^2 + F2 u'') gy''
//   gr = sum e h + sum_d (f h' + s h''),  gr' = sum (e h' + 2 f h''),  gr'' = sum e h''
//   gV = -r^3 gr / 2 + sum_d 3/2 r^5 A gr' + (3/2 r^5 B - 15/2 r^7 A^2) gr'',  gA = -r^3 gr' + 6 r^5 A gr'', gB = -r^3 gr''
//   ge = r h + 2 e gV / M + sum_d (r' h' + r'' h'' + (f gA + s gB) / M),  gf = r h' + 2 r' h'' + (e gA + 2 f gB) / M,
//   gs = r h'' + e gB / M, each less its mean over the group (the means of e, f, s vanish: only h's remain)
// A lane holds a channel's whole jet (J = 4 or 12 floats, 16-byte accesses), a group sits in L lanes: the five sums of the
// forward and the backward's cross the lanes in registers.  HBM bounds it: 2^19 x 64 x 4, forward 208 us (best of 20: 193;
// 1.07 GB, 5.2 TB/s), backward 369 (361; 1.61 GB, 4.4 TB/s); 12 slots: 30011 x 128 x 12, 81 us (77; 369 MB, 4.6 TB/s) and 125 (113;
// 553 MB, 4.4 TB/s).
template <int ND, int NS, int L, int K, bool BWD>
__global__ void __launch_bounds__(kThreads) norm_jet_kernel(RowMap m, const float* __restrict__ x,
                                                            const float* __restrict__ gy, const float* __restrict__ w,
                                                            const float* __restrict__ b, float eps, int act,
                                                            float* __restrict__ out, float* part_w, float* part_b,
                                                            int part_stride) {
  constexpr int J = 1 + ND + NS;
  const RowPlace r = row_place<L>(m);
  const int lane = threadIdx.x % L;
  const float inv = 1.0f / (float)m.cpg;
  bool valid[K];
  float wv[K], bv[K], gwv[K], gbv[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    valid[k] = r.on && lane + L * k < m.cpg;
    const int c = r.g * m.cpg + lane + L * k;
    wv[k] = valid[k] && w ? w[c] : 1.0f;
    bv[k] = valid[k] && b ? b[c] : 0.0f;
    gwv[k] = gbv[k] = 0.0f;
  }
  by_activation(act, [&](auto kind) {
    constexpr int ACT = decltype(kind)::value;
    if (!r.on) return;
    for (int64_t p = r.p; p < m.n; p += r.step) {
      const int64_t at = (p * m.C + (int64_t)r.g * m.cpg + lane) * J;
      float e[K][J], h[K][J];
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int j = 0; j < J; ++j) e[k][j] = h[k][j] = 0.0f;
        if (valid[k]) {
          if constexpr (J % 4 == 0) {
#pragma unroll
            for (int j = 0; j < J; j += 4) {
              float t[4];
              load_vec<float, 4>(x + at + (int64_t)L * k * J + j, t);
#pragma unroll
              for (int i = 0; i < 4; ++i) e[k][j + i] = t[i];
              if constexpr (BWD) {
                load_vec<float, 4>(gy + at + (int64_t)L * k * J + j, t);
#pragma unroll
                for (int i = 0; i < 4; ++i) h[k][j + i] = t[i];
              }
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) s += e[k][j];
        s = group_sum<L>(s) * inv;
#pragma unroll
        for (int k = 0; k < K; ++k) e[k][j] = valid[k] ? e[k][j] - s : 0.0f;
      }
      float V = 0.0f, A[ND], B[NS];
#pragma unroll
      for (int k = 0; k < K; ++k) V = fmaf(e[k][0], e[k][0], V);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        A[d] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) A[d] = fmaf(e[k][0], e[k][1 + d], A[d]);
        A[d] = group_sum<L>(A[d]) * inv;
      }
#pragma unroll
      for (int d = 0; d < NS; ++d) {
        B[d] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k)
          B[d] = fmaf(e[k][1 + d], e[k][1 + d], fmaf(e[k][0], e[k][1 + ND + d], B[d]));
        B[d] = group_sum<L>(B[d]) * inv;
      }
      const float rs = rsqrtf(fmaf(group_sum<L>(V), inv, eps));
      const float r3 = rs * rs * rs, r5 = r3 * rs * rs;
      float r1[ND], r2[NS];
#pragma unroll
      for (int d = 0; d < ND; ++d) r1[d] = -r3 * A[d];
#pragma unroll
      for (int d = 0; d < NS; ++d) r2[d] = fmaf(3.0f * r5 * A[d], A[d], -r3 * B[d]);
      if constexpr (!BWD) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          float f[3], y[J];
          activation<ACT, 2, true>(fmaf(e[k][0] * rs, wv[k], bv[k]), f);
          y[0] = f[0];
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const float u1 = wv[k] * fmaf(e[k][0], r1[d], e[k][1 + d] * rs);
            y[1 + d] = f[1] * u1;
            if (d < NS) {
              const float u2 = wv[k] * fmaf(e[k][0], r2[d], fmaf(2.0f * e[k][1 + d], r1[d], e[k][1 + ND + d] * rs));
              y[1 + ND + d] = fmaf(f[2] * u1, u1, f[1] * u2);
            }
          }
          if (valid[k]) {
#pragma unroll
            for (int j = 0; j < J; j += 4) {
              const float t[4] = {y[j], y[j + 1], y[j + 2], y[j + 3]};
              store_vec<float, 4>(out + at + (int64_t)L * k * J + j, t);
            }
          }
        }
      } else {
        float gr = 0.0f, gr1[ND], gr2[NS], hm[J];
#pragma unroll
        for (int d = 0; d < ND; ++d) gr1[d] = 0.0f;
#pragma unroll
        for (int d = 0; d < NS; ++d) gr2[d] = 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j) hm[j] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const float z = e[k][0] * rs;
          float f[4];
          activation<ACT, 3, true>(fmaf(z, wv[k], bv[k]), f);
          float gu = f[1] * h[k][0], gw = 0.0f;
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const float z1 = fmaf(e[k][0], r1[d], e[k][1 + d] * rs), u1 = wv[k] * z1;
            float gu1 = f[1] * h[k][1 + d];
            gu = fmaf(f[2] * u1, h[k][1 + d], gu);
            if (d < NS) {
              const float z2 = fmaf(e[k][0], r2[d], fmaf(2.0f * e[k][1 + d], r1[d], e[k][1 + ND + d] * rs));
              const float u2 = wv[k] * z2, g2 = h[k][1 + ND + d];
              gu = fmaf(fmaf(f[3] * u1, u1, f[2] * u2), g2, gu);
              gu1 = fmaf(2.0f * f[2] * u1, g2, gu1);
              const float gu2 = f[1] * g2;
              gw = fmaf(gu2, z2, gw);
              h[k][1 + ND + d] = wv[k] * gu2;
              gr2[d] = fmaf(e[k][0], h[k][1 + ND + d], gr2[d]);
              gr1[d] = fmaf(2.0f * e[k][1 + d], h[k][1 + ND + d], gr1[d]);
              gr = fmaf(e[k][1 + ND + d], h[k][1 + ND + d], gr);
            }
            gw = fmaf(gu1, z1, gw);
            h[k][1 + d] = wv[k] * gu1;
            gr1[d] = fmaf(e[k][0], h[k][1 + d], gr1[d]);
            gr = fmaf(e[k][1 + d], h[k][1 + d], gr);
          }
          gbv[k] += gu;
          gwv[k] += fmaf(gu, z, gw);
          h[k][0] = wv[k] * gu;
          gr = fmaf(e[k][0], h[k][0], gr);
#pragma unroll
          for (int j = 0; j < J; ++j) hm[j] += h[k][j];
        }
        gr = group_sum<L>(gr);
#pragma unroll
        for (int d = 0; d < ND; ++d) gr1[d] = group_sum<L>(gr1[d]);
#pragma unroll
        for (int d = 0; d < NS; ++d) gr2[d] = group_sum<L>(gr2[d]);
#pragma unroll
        for (int j = 0; j < J; ++j) hm[j] = group_sum<L>(hm[j]) * inv;
        // gA, gB and gV, each already divided by the number of channels
        float gA[ND], gB[NS], gV = -0.5f * r3 * gr;
        const float r7 = r5 * rs * rs;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          gA[d] = -r3 * gr1[d];
          gV = fmaf(1.5f * r5 * A[d], gr1[d], gV);
          if (d < NS) {
            gA[d] = fmaf(6.0f * r5 * A[d], gr2[d], gA[d]);
            gB[d] = -r3 * gr2[d] * inv;
            gV = fmaf(fmaf(1.5f * r5, B[d], -7.5f * r7 * A[d] * A[d]), gr2[d], gV);
          }
          gA[d] *= inv;
        }
        gV *= 2.0f * inv;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          float g[J];
          g[0] = fmaf(rs, h[k][0] - hm[0], e[k][0] * gV);
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            g[0] = fmaf(r1[d], h[k][1 + d] - hm[1 + d], fmaf(e[k][1 + d], gA[d], g[0]));
            g[1 + d] = fmaf(rs, h[k][1 + d] - hm[1 + d], e[k][0] * gA[d]);
            if (d < NS) {
              const float h2 = h[k][1 + ND + d] - hm[1 + ND + d];
              g[0] = fmaf(r2[d], h2, fmaf(e[k][1 + ND + d], gB[d], g[0]));
              g[1 + d] = fmaf(2.0f * r1[d], h2, fmaf(2.0f * e[k][1 + d], gB[d], g[1 + d]));
              g[1 + ND + d] = fmaf(rs, h2, e[k][0] * gB[d]);
            }
          }
          if (valid[k]) {
#pragma unroll
            for (int j = 0; j < J; j += 4) {
              const float t[4] = {g[j], g[j + 1], g[j + 2], g[j + 3]};
              store_vec<float, 4>(out + at + (int64_t)L * k * J + j, t);
            }
          }
        }
      }
    }
  });
  if constexpr (BWD) {
    __shared__ float red[kThreads][2];
    if (part_w || part_b) {
      const int64_t row = (int64_t)(blockIdx.x / m.gchunks) * part_stride;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float gw1[1] = {gwv[k]}, gb1[1] = {gbv[k]};
        row_grad_out<1, L>(m, r, gw1, gb1, r.g * m.cpg + lane + L * k, valid[k], part_w ? part_w + row : nullptr,
                           part_b ? part_b + row : nullptr, red);
      }
    }
  }
}

// out_w[c], out_b[c] = sums over the rows of part [rows][2][C], in a fixed order: a block takes COLS columns, THREADS / COLS
// threads a column, eight loads of a thread in flight.  In 64 bits: a thread's chain is rows / (THREADS / COLS) long, up to
// 2^18 where there are millions of samples, and the additions hide behind the loads.
template <int COLS, int THREADS>
__device__ __forceinline__ void finish_columns(int col_block, const float* __restrict__ part, int64_t rows, int C,
                                               float* out_w, float* out_b) {
  constexpr int kSlices = THREADS / COLS;
  __shared__ double red[kSlices][COLS + 1];
  const int cl = threadIdx.x % COLS, sl = threadIdx.x / COLS;
  const int col = col_block * COLS + cl;
  double s = 0.0;
  if (col < 2 * C) {
#pragma unroll 8
    for (int64_t i = sl; i < rows; i += kSlices) s += (double)part[i * 2 * C + col];
  }
  red[sl][cl] = s;
  __syncthreads();
  if (sl == 0 && col < 2 * C) {
#pragma unroll
    for (int i = 1; i < kSlices; ++i) s += red[i][cl];
    float* out = col < C ? out_w : out_b;
    if (out) out[col < C ? col : col - C] = (float)s;
  }
}
constexpr int kFinishCols = 32, kGridFinishCols = 8;
__global__ void __launch_bounds__(1024) norm_finish_kernel(const float* __restrict__ part, int64_t rows, int C,
                                                           float* out_w, float* out_b) {
  finish_columns<kFinishCols, 1024>(blockIdx.x, part, rows, C, out_w, out_b);
}

// ---- samples of many positions ------------------------------------------------------------------------------------

// Four launches for forward and backward; each reads its rows with VEC channels a thread, 8 x 4096 x 320 bf16 (21 MB a tensor): statistics
// 11.5 us, apply 15, sums 20, gradient 19.  A third of that is the arithmetic (SiLU and its slope: about 25 vector instructions a
// value), the rest latency: chunks are short, and every block first reduces or merges.
constexpr int kAhead = 4;              // rows a thread of the second launches loads before the sums are merged

// A block takes one chunk of positions of one sample and all its channels: thread = (vector of channels, row slot).
struct GridMap {
  int64_t n, s, rows;                  // rows: positions a chunk (the last may have fewer)
  int64_t sums;                        // blocks of the backward's sums, of `per` samples each (the last may have fewer)
  int C, G, cpg, chunks, per;          // per: 1 where a sample has more than one chunk, a block takes one of those
};

template <int VEC>
struct GridThread {
  int nv, txn, tyn, tx, ty;
  int64_t sample, row0, row1;
  int chunk;
  __device__ __forceinline__ GridThread(const GridMap& m, int64_t block) {
    nv = m.C / VEC;
    txn = nv < kThreads ? nv : kThreads;
    tyn = kThreads / txn;
    tx = threadIdx.x % txn;
    ty = threadIdx.x / txn;
    sample = block / m.chunks;
    chunk = (int)(block % m.chunks);
    row0 = chunk * m.rows;
    row1 = row0 + m.rows < m.s ? row0 + m.rows : m.s;
  }
};

// body(raw x[N], raw y[N], N) for a thread's rows from `row`, N at a time, whose loads are on their way at once, then half as many and
// so on down to one; TWO: y too.  (Loads with a condition each would wait for one another.)
template <typename T, int VEC, int N, bool TWO, typename F>
__device__ __forceinline__ void for_rows(const GridMap& m, const GridThread<VEC>& t, int64_t row, const T* __restrict__ x, const T* __restrict__ y,
                                         F&& body) {
  typedef typename VecOf<T, VEC>::type Raw;
  Raw rx[N], ry[N];
  for (; row + (N - 1) * t.tyn < t.row1; row += N * t.tyn) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      rx[j] = *reinterpret_cast<const Raw*>(x + (row + j * t.tyn) * m.C);
      if constexpr (TWO) ry[j] = *reinterpret_cast<const Raw*>(y + (row + j * t.tyn) * m.C);
    }
    body(rx, ry, IntC<N>{});
  }
  if constexpr (N > 1) for_rows<T, VEC, N / 2, TWO>(m, t, row, x, y, body);
}

// bytes of LDS ahead of the per-channel numbers: two sums and a number a thread and channel where a channel's rows are spread
// over several threads
template <int VEC>
__device__ __host__ constexpr int red_bytes(int C) { return C / VEC > kThreads / 2 ? 0 : kThreads * VEC * 20; }

// own(c, sum of s1, sum of s2, k) once for each channel c of the tile: over the threads of its row slots, through red [2][threads x
// VEC], where there are several (all channels are one tile then).  With more than eight slots every thread adds up a part first.
template <int VEC, typename Own>
__device__ __forceinline__ void channel_sums(const GridThread<VEC>& t, int tile, bool on, const double (&s1)[VEC], const double (&s2)[VEC],
                                             const float (&k)[VEC], double* red, Own own) {
  const int slots = t.row1 - t.row0 < t.tyn ? (int)(t.row1 - t.row0) : t.tyn;
  if (slots == 1) {
    if (on && t.ty == 0) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) own((tile + t.tx) * VEC + i, s1[i], s2[i], k[i]);
    }
    return;
  }
  const int cols = t.txn * VEC;
  double* red2 = red + kThreads * VEC;
  float* redk = reinterpret_cast<float*>(red2 + kThreads * VEC);
  __syncthreads();
  if (on && t.ty < slots) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      red[t.ty * cols + i * t.txn + t.tx] = s1[i];
      red2[t.ty * cols + i * t.txn + t.tx] = s2[i];
      if (t.ty == 0) redk[i * t.txn + t.tx] = k[i];
    }
  }
  __syncthreads();
  int parts = slots;
  if (slots > 8) {
    parts = kThreads / (2 * cols) > 1 ? kThreads / (2 * cols) : 1;
    if (parts > slots) parts = slots;
    // (a thread's sum takes the place of its first term)
    for (int job = threadIdx.x; job < 2 * cols * parts; job += kThreads) {
      const int part = job / (2 * cols), col = job - part * 2 * cols;
      double* at = col < cols ? red + col : red2 + col - cols;
      double s = at[part * cols];
      for (int y = part + parts; y < slots; y += parts) s += at[y * cols];
      at[part * cols] = s;
    }
    __syncthreads();
  }
  for (int col = threadIdx.x; col < cols; col += kThreads) {
    double a = red[col], b = red2[col];
    for (int y = 1; y < parts; ++y) {
      a += red[y * cols + col];
      b += red2[y * cols + col];
    }
    const int i = col / t.txn;
    own((col - i * t.txn) * VEC + i, a, b, redk[col]);
  }
}
// not below zero; a NaN stays one
__device__ __forceinline__ double not_negative(double v) { return v < 0.0 ? 0.0 : v; }

// Partial statistics of a chunk: per channel the sums of x - k and (x - k)^2 with k the chunk's first value of that channel,
// in 64 bits.  k may stand apart from the rest (the boundary value of a field): the sum of squares then loses up to n (k -
// mean)^2 / M2 <= n, the chunk's positions, to the square of the sum, 24 bits of 53 at most.  In 32 bits the sums of 2^18 positions
// near 10^4 behind a first one of 0 were 13 % off.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, VEC == 8 ? 3 : VEC >= 2 ? 4 : 6) norm_grid_stats_kernel(GridMap m, const T* __restrict__ x,
                                                                   double2* __restrict__ part) {
  extern __shared__ double lds64[];                   // see red_bytes;  [2][C]: mean and sum of squared deviations of each channel
  double* chan64 = lds64 + red_bytes<VEC>(m.C) / 8;
  const GridThread<VEC> t(m, blockIdx.x);
  const T* base = x + t.sample * m.s * m.C;
  const double cnt = (double)(t.row1 - t.row0), inv = 1.0 / cnt, inv_cpg = 1.0 / m.cpg;
  for (int tile = 0; tile < t.nv; tile += t.txn) {
    const int vec = tile + t.tx;
    const bool on = t.ty < t.tyn && vec < t.nv;
    float k[VEC];
    double s1[VEC], s2[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) k[i] = s1[i] = s2[i] = 0.0f;
    if (on) {
      load_vec<T, VEC>(base + t.row0 * m.C + vec * VEC, k);
      for_rows<T, VEC, VEC >= 4 ? 4 : 8, false>(m, t, t.row0 + t.ty, base + vec * VEC, nullptr, [&](const auto& rx, const auto&, auto rows) {
#pragma unroll
        for (int j = 0; j < decltype(rows)::value; ++j) {
          float v[VEC];
          widen<T, VEC>(rx[j], v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const double d = (double)v[i] - (double)k[i];
            s1[i] += d;
            s2[i] = fma(d, d, s2[i]);
          }
        }
      });
    }
    channel_sums<VEC>(t, tile, on, s1, s2, k, lds64, [&](int c, double a, double b, float first) {
      const double d = a * inv;
      chan64[c] = (double)first + d;
      chan64[m.C + c] = not_negative(fma(-d, a, b));
    });
  }
  __syncthreads();
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  for (int g = wave; g < m.G; g += kThreads / 64) {
    double s = 0.0, q = 0.0;
    for (int c = lane; c < m.cpg; c += 64) s += chan64[g * m.cpg + c];
    const double mean = wave_sum64(s) * inv_cpg;
    for (int c = lane; c < m.cpg; c += 64) {
      const double d = chan64[g * m.cpg + c] - mean;
      q += fma(cnt * d, d, chan64[m.C + g * m.cpg + c]);
    }
    q = wave_sum64(q);
    if (lane == 0) part[(int64_t)blockIdx.x * m.G + g] = make_double2(mean, q);
  }
}

__device__ __forceinline__ double chunk_rows(const GridMap& m, int chunk) {
  const int64_t left = m.s - chunk * m.rows;
  return (double)(left < m.rows ? left : m.rows);
}

// Sums over a sample's chunks of two numbers a (chunk, group), part [chunks][G], each group's by 256 / G threads (loads of
// all chunks in flight at once, neighbouring threads on neighbouring groups): term(chunk, value, first chunk's value)
// adds to s.  take(g, s, first) gets the totals, one thread a group.  Pair: double2 or float2; added up in 64 bits.
template <typename Pair, typename Term, typename Take>
__device__ __forceinline__ void merge_chunks(const GridMap& m, const Pair* __restrict__ part, double2 (*red), Term term, Take take) {
  if (m.chunks == 1) {
    for (int g = threadIdx.x; g < m.G; g += kThreads) {
      const Pair v = part[g];
      double2 s = make_double2(0.0, 0.0);
      term(0, v, v, s);
      take(g, s, v);
    }
    return;
  }
  constexpr int kBatch = 8;                           // loads of a thread on their way at once
  const int gw = m.G < kThreads ? m.G : kThreads, per = kThreads / gw;
  const int gl = threadIdx.x % gw, sub = threadIdx.x / gw;
  for (int g0 = 0; g0 < m.G; g0 += gw) {
    const int g = g0 + gl;
    double2 s = make_double2(0.0, 0.0);
    Pair first;
    first.x = first.y = 0;
    if (g < m.G && sub < per) {
      first = part[g];
      for (int k0 = sub; k0 < m.chunks; k0 += kBatch * per) {
        Pair v[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) v[j] = part[(int64_t)min(k0 + j * per, m.chunks - 1) * m.G + g];
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
          if (k0 + j * per < m.chunks) term(k0 + j * per, v[j], first, s);
      }
    }
    __syncthreads();
    red[threadIdx.x] = s;
    __syncthreads();
    if (g < m.G && sub == 0) {
      for (int i = 1; i < per; ++i) {
        const double2 o = red[gl + i * gw];
        s.x += o.x;
        s.y += o.y;
      }
      take(g, s, first);
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) norm_grid_apply_kernel(GridMap m, const T* __restrict__ x,
                                                                   const float* __restrict__ w,
                                                                   const float* __restrict__ b, float eps, int act,
                                                                   const double2* __restrict__ part, T* __restrict__ y,
                                                                   float2* stats) {
  extern __shared__ float chan[];                     // [2][G]
  __shared__ double2 red[kThreads];
  float *mu = chan, *rs = chan + m.G;
  const GridThread<VEC> t(m, blockIdx.x);
  const int64_t base = t.sample * m.s * m.C;
  // a thread's first rows are on their way while the statistics are merged
  typedef typename VecOf<T, VEC>::type Raw;
  Raw ahead[kAhead];
  const bool first_on = t.ty < t.tyn && t.tx < t.nv;
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    const int64_t row = t.row0 + t.ty + j * t.tyn;
    if (first_on && row < t.row1) ahead[j] = *reinterpret_cast<const Raw*>(x + base + row * m.C + t.tx * VEC);
  }
  // mean and r of the sample's groups, about the first chunk's mean (one of the means: see the stats kernel)
  const double width = (double)m.cpg, inv_s = 1.0 / (double)m.s, inv_all = inv_s / width;
  merge_chunks(m, part + t.sample * m.chunks * m.G, red,
               [&](int k, double2 v, double2 first, double2& s) {
                 const double cnt = chunk_rows(m, k), d = v.x - first.x;
                 s.x = fma(cnt, d, s.x);
                 s.y += fma(cnt * width * d, d, v.y);
               },
               [&](int g, double2 s, double2 first) {
                 const double d = s.x * inv_s, var = not_negative(fma(-d * width, s.x, s.y)) * inv_all;
                 mu[g] = (float)(first.x + d);
                 rs[g] = rsqrtf((float)(var + (double)eps));
                 if (t.chunk == 0 && stats) stats[t.sample * m.G + g] = make_float2(mu[g], rs[g]);
               });
  __syncthreads();
  for (int tile = 0; tile < t.nv; tile += t.txn) {
    const int vec = tile + t.tx;
    if (t.ty >= t.tyn || vec >= t.nv) continue;
    float wr[VEC], bv[VEC], mean[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = vec * VEC + i, g = c / m.cpg;
      wr[i] = (w ? w[c] : 1.0f) * rs[g];
      bv[i] = b ? b[c] : 0.0f;
      mean[i] = mu[g];
    }
    by_activation(act, [&](auto kind) {
      constexpr int ACT = decltype(kind)::value;
      auto one = [&](int64_t row, const Raw& raw) {
        float v[VEC];
        widen<T, VEC>(raw, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float f[1];
          activation<ACT, 0, sizeof(T) == 4>(fmaf(v[i] - mean[i], wr[i], bv[i]), f);
          v[i] = f[0];
        }
        store_vec<T, VEC>(y + base + row * m.C + vec * VEC, v);
      };
      int64_t row = t.row0 + t.ty;
      if (tile == 0) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j, row += t.tyn)
          if (row < t.row1) one(row, ahead[j]);
      }
#pragma unroll 4
      for (; row < t.row1; row += t.tyn) one(row, *reinterpret_cast<const Raw*>(x + base + row * m.C + vec * VEC));
    });
  }
}

// Backward, launch 1: per chunk and group the sums of w p and w p z with p = gy f' (part_g [n * chunks][G]), and per block and
// channel those of p z and p (part_c [sums][2][C], not wanted: nullptr).  A thread adds 32 rows in fp32, and what they come to
// in 64 bits: a chunk may have any number of rows.  A block adds up to 64 samples in its row of part_c, which stays in the L2: a
// row a sample would be 8 bytes a value where samples are single wide points.
constexpr int kChain = 32;
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, VEC == 8 ? 2 : 4) norm_grid_sums_kernel(GridMap m, const T* __restrict__ x,
                                                                  const T* __restrict__ gy, const float* __restrict__ w,
                                                                  const float* __restrict__ b, int act,
                                                                  const float2* __restrict__ stats,
                                                                  float* __restrict__ part_c, float2* __restrict__ part_g) {
  extern __shared__ double lds64[];                   // see red_bytes;  [2][C]: sums of w p z, w p
  float* chan = reinterpret_cast<float*>(lds64 + red_bytes<VEC>(m.C) / 8);
  float* mine = part_c ? part_c + (int64_t)blockIdx.x * 2 * m.C : nullptr;
  const int64_t first = (int64_t)blockIdx.x * m.per, all = m.n * m.chunks, end = first + m.per < all ? first + m.per : all;
  for (int64_t item = first; item < end; ++item) {
    const GridThread<VEC> t(m, item);
    const int64_t base = t.sample * m.s * m.C;
    for (int tile = 0; tile < t.nv; tile += t.txn) {
      const int vec = tile + t.tx;
      const bool on = t.ty < t.tyn && vec < t.nv;
      double s1[VEC], s2[VEC];
      float wv[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) s1[i] = s2[i] = wv[i] = 0.0f;
      if (on) {
        float bv[VEC], mean[VEC], rs[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int c = vec * VEC + i;
          const float2 st = stats[t.sample * m.G + c / m.cpg];
          wv[i] = w ? w[c] : 1.0f;
          bv[i] = b ? b[c] : 0.0f;
          mean[i] = st.x;
          rs[i] = st.y;
        }
        by_activation(act, [&](auto kind) {
          constexpr int ACT = decltype(kind)::value;
          float c1[VEC], c2[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) c1[i] = c2[i] = 0.0f;
          int terms = 0;
          auto fold = [&]() {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              s1[i] += c1[i];
              s2[i] += c2[i];
              c1[i] = c2[i] = 0.0f;
            }
            terms = 0;
          };
          for_rows<T, VEC, VEC >= 4 ? 2 : 4, true>(m, t, t.row0 + t.ty, x + base + vec * VEC, gy + base + vec * VEC, [&](const auto& rx, const auto& ry, auto rows) {
#pragma unroll
            for (int j = 0; j < decltype(rows)::value; ++j) {
              float v[VEC], g[VEC];
              widen<T, VEC>(rx[j], v);
              widen<T, VEC>(ry[j], g);
#pragma unroll
              for (int i = 0; i < VEC; ++i) {
                const float z = (v[i] - mean[i]) * rs[i];
                float f[2];
                activation<ACT, 1, sizeof(T) == 4>(fmaf(z, wv[i], bv[i]), f);
                const float p = g[i] * f[1];
                c1[i] += p;
                c2[i] = fmaf(p, z, c2[i]);
              }
            }
            terms += decltype(rows)::value;
            if (terms > kChain - 4) fold();
          });
          fold();
        });
      }
      channel_sums<VEC>(t, tile, on, s1, s2, wv, lds64, [&](int c, double a, double q, float wc) {
        if (mine) {
          mine[c] = (item > first ? mine[c] : 0.0f) + (float)q;
          mine[m.C + c] = (item > first ? mine[m.C + c] : 0.0f) + (float)a;
        }
        chan[c] = wc * (float)q;
        chan[m.C + c] = wc * (float)a;
      });
    }
    __syncthreads();
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    for (int g = wave; g < m.G; g += kThreads / 64) {
      double a = 0.0, q = 0.0;
      for (int c = lane; c < m.cpg; c += 64) {
        q += chan[g * m.cpg + c];
        a += chan[m.C + g * m.cpg + c];
      }
      a = wave_sum64(a);
      q = wave_sum64(q);
      if (lane == 0) part_g[item * m.G + g] = make_float2((float)a, (float)q);
    }
    __syncthreads();                                   // (the next sample's sums take chan's place)
  }
}

// Backward, launch 2: gx from the merged sums of the sample; the first blocks sum gw and gb over all chunks instead
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) norm_grid_grad_kernel(GridMap m, const T* __restrict__ x,
                                                                  const T* __restrict__ gy, const float* __restrict__ w,
                                                                  const float* __restrict__ b, int act,
                                                                  const float2* __restrict__ stats,
                                                                  const float* __restrict__ part_c,
                                                                  const float2* __restrict__ part_g, T* __restrict__ gx,
                                                                  float* gw, float* gb, int finish_blocks) {
  extern __shared__ float chan[];                     // [2][G]
  __shared__ double2 red[kThreads];
  if ((int)blockIdx.x < finish_blocks) {
    finish_columns<kGridFinishCols, kThreads>(blockIdx.x, part_c, m.sums, m.C, gw, gb);
    return;
  }
  const GridThread<VEC> t(m, blockIdx.x - finish_blocks);
  const int64_t base = t.sample * m.s * m.C;
  typedef typename VecOf<T, VEC>::type Raw;
  Raw ahead_x[kAhead], ahead_g[kAhead];
  const bool first_on = t.ty < t.tyn && t.tx < t.nv;
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    const int64_t row = t.row0 + t.ty + j * t.tyn;
    if (first_on && row < t.row1) {
      ahead_x[j] = *reinterpret_cast<const Raw*>(x + base + row * m.C + t.tx * VEC);
      ahead_g[j] = *reinterpret_cast<const Raw*>(gy + base + row * m.C + t.tx * VEC);
    }
  }
  const float inv = 1.0f / ((float)m.s * (float)m.cpg);
  merge_chunks(m, part_g + t.sample * m.chunks * m.G, red,
               [&](int, float2 v, float2, double2& s) { s.x += v.x; s.y += v.y; },
               [&](int g, double2 s, float2) { chan[g] = (float)s.x * inv; chan[m.G + g] = (float)s.y * inv; });
  __syncthreads();
  for (int tile = 0; tile < t.nv; tile += t.txn) {
    const int vec = tile + t.tx;
    if (t.ty >= t.tyn || vec >= t.nv) continue;
    float wv[VEC], bv[VEC], mean[VEC], rs[VEC], a[VEC], q[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = vec * VEC + i, g = c / m.cpg;
      const float2 st = stats[t.sample * m.G + g];
      wv[i] = w ? w[c] : 1.0f;
      bv[i] = b ? b[c] : 0.0f;
      mean[i] = st.x;
      rs[i] = st.y;
      a[i] = chan[g];
      q[i] = chan[m.G + g];
    }
    by_activation(act, [&](auto kind) {
      constexpr int ACT = decltype(kind)::value;
      auto one = [&](int64_t row, const Raw& rx, const Raw& rg) {
        float v[VEC], g[VEC];
        widen<T, VEC>(rx, v);
        widen<T, VEC>(rg, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float z = (v[i] - mean[i]) * rs[i];
          float f[2];
          activation<ACT, 1, sizeof(T) == 4>(fmaf(z, wv[i], bv[i]), f);
          v[i] = rs[i] * (g[i] * f[1] * wv[i] - a[i] - z * q[i]);
        }
        store_vec<T, VEC>(gx + base + row * m.C + vec * VEC, v);
      };
      int64_t row = t.row0 + t.ty;
      if (tile == 0) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j, row += t.tyn)
          if (row < t.row1) one(row, ahead_x[j], ahead_g[j]);
      }
#pragma unroll 2
      for (; row < t.row1; row += t.tyn)
        one(row, *reinterpret_cast<const Raw*>(x + base + row * m.C + vec * VEC),
            *reinterpret_cast<const Raw*>(gy + base + row * m.C + vec * VEC));
    });
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------

constexpr int kRowBlocks = 2048;       // 8 blocks of 4 waves a compute unit: all that fit, so that a block's channels stay with it
// Two blocks a compute unit: each merges all chunks of its sample, which more blocks have more of, and fewer leave it idle.
// All four launches of 8 x 4096 x 320 bf16 with 256, 384, 512, 768, 1024 blocks: 65, 69, 64, 78, 88 us, of 32 x 1024 x 640 102, 100, 91,
// 103, 109; of 2 x 16384 x 512 with at most 64, 128, 256 chunks a sample: 128, 84, 83 us.
constexpr int kGridBlocks = 512, kChunksMax = 256, kSamplesMax = 64;
constexpr size_t kStaticLds = 8 * 1024, kLds = 160 * 1024;     // at least what the grid kernels declare themselves; all there is

int pow2_at_least(int v) { int p = 1; while (p < v) p *= 2; return p; }

RowMap row_map(int64_t n, int s, int C, int G, int L) {
  RowMap m;
  m.n = n; m.s = s; m.C = C; m.G = G; m.cpg = C / G;
  const int rpb = kThreads / L;
  if (G <= rpb) { m.gpb = G; m.ppb = rpb / G; m.gchunks = 1; }
  else { m.gpb = rpb; m.ppb = 1; m.gchunks = (G + rpb - 1) / rpb; }
  if (m.ppb > n) m.ppb = (int)n;
  // with several positions the partial gradients take a row each: fewer blocks, but one a compute unit at least
  const int blocks = s == 1 ? kRowBlocks : kRowBlocks / s > 256 ? kRowBlocks / s : 256;
  const int64_t need = (n + m.ppb - 1) / m.ppb, most = blocks / m.gchunks > 0 ? blocks / m.gchunks : 1;
  m.npb = (int)(need < most ? need : most);
  return m;
}

// lanes and vectors a lane of a group of `values` values
struct RowShape { int vec, L, K; };
RowShape row_shape(int values, int vec) {
  const int nv = values / vec;
  int L = pow2_at_least(nv);
  if (L < 4) L = 4;
  if (L > 64) L = 64;
  const int K = pow2_at_least((nv + L - 1) / L);
  return {vec, L, K};
}

int elem_size(int dtype) { return dtype == kNormF32 ? 4 : 2; }

// the widest vector that divides the rows' addresses: 16 bytes, 4 bytes (16-bit types) or one element
int vec_width(int dtype, int unit, const void* a, const void* b, const void* c) {
  const int es = elem_size(dtype);
  const uintptr_t low = (uintptr_t)a | (uintptr_t)b | (uintptr_t)c;
  for (const int bytes : {16, 4}) {
    const int v = bytes / es;
    if (v > 1 && unit % v == 0 && low % bytes == 0) return v;
  }
  return 1;
}

// A launch may ask for 64 KB of LDS with what the kernel declares itself; beyond, the limit of its dynamic part is raised first, up
// to what is left of all there is.
void ensure_lds(const void* kernel, size_t dynamic) {
  if (dynamic + kStaticLds > 64 * 1024) ensure_dynamic_lds(kernel, std::min(dynamic + kStaticLds, kLds - kStaticLds));
}

GridMap grid_map(int64_t n, int64_t s, int C, int G) {
  GridMap m;
  m.n = n; m.s = s; m.C = C; m.G = G; m.cpg = C / G;
  int64_t chunks = (kGridBlocks + n - 1) / n;
  // a chunk of at least 4096 values: shorter ones cost more in their partial results than they spread
  const int64_t least = (4096 + C - 1) / C;
  if (chunks > s / least) chunks = s / least;
  if (chunks > kChunksMax) chunks = kChunksMax;
  if (chunks < 1) chunks = 1;
  m.rows = (s + chunks - 1) / chunks;
  m.chunks = (int)((s + m.rows - 1) / m.rows);
  // blocks of the backward's sums: as many as the chip holds, more where that would be more than 64 samples each
  const int64_t per = m.chunks > 1 ? 1 : (n + kRowBlocks - 1) / kRowBlocks;
  m.per = (int)(per < kSamplesMax ? per : kSamplesMax);
  m.sums = (n * m.chunks + m.per - 1) / m.per;
  return m;
}

// 512 values a group: with one element a vector (the least aligned tensors) the 64 lanes of a wave still hold it
bool rows_kernel_takes(int64_t s, int cpg) { return s <= 32 && s * cpg <= 512; }

template <typename T, int VEC, bool BWD>
void run_rows(const RowShape& sh, const RowMap& m, const T* x, const T* gy, const float* w, const float* b, float eps,
              int act, T* out, float* pw, float* pb, int stride, hipStream_t st) {
  const dim3 grid(m.npb * m.gchunks), block(kThreads);
#define PDEKAN_ROWS(LL, KK)                                                                                         \
  if (sh.L == LL && sh.K == KK) {                                                                                   \
    hipLaunchKernelGGL((norm_rows_kernel<T, VEC, LL, KK, BWD>), grid, block, 0, st, m, x, gy, w, b, eps, act, out, \
                       pw, pb, stride);                                                                             \
    return;                                                                                                         \
  }
  PDEKAN_ROWS(4, 1) PDEKAN_ROWS(8, 1) PDEKAN_ROWS(16, 1) PDEKAN_ROWS(32, 1) PDEKAN_ROWS(64, 1)
  if constexpr (VEC <= 4) { PDEKAN_ROWS(64, 2) }
  if constexpr (VEC <= 2) { PDEKAN_ROWS(64, 4) }
  if constexpr (VEC <= 1) { PDEKAN_ROWS(64, 8) }
#undef PDEKAN_ROWS
}

template <typename T, bool BWD>
void run_rows_vec(int vec, const RowShape& sh, const RowMap& m, const void* x, const void* gy, const float* w,
                  const float* b, float eps, int act, void* out, float* pw, float* pb, int stride, hipStream_t st) {
  constexpr int kWide = 16 / sizeof(T);
  const T *xt = static_cast<const T*>(x), *gt = static_cast<const T*>(gy);
  T* ot = static_cast<T*>(out);
  if (vec == kWide) run_rows<T, kWide, BWD>(sh, m, xt, gt, w, b, eps, act, ot, pw, pb, stride, st);
  else if (sizeof(T) == 2 && vec == 2) run_rows<T, 2, BWD>(sh, m, xt, gt, w, b, eps, act, ot, pw, pb, stride, st);
  else run_rows<T, 1, BWD>(sh, m, xt, gt, w, b, eps, act, ot, pw, pb, stride, st);
}

template <bool BWD>
void rows_any(int dtype, const NormShape& p, const void* x, const void* gy, const float* w, const float* b, float eps,
              int act, void* out, float* gw, float* gb, float* part, hipStream_t st) {
  const int vec = vec_width(dtype, p.C / p.G, x, gy, out);
  const RowShape sh = row_shape(p.C / p.G * (int)p.s, vec);
  const RowMap m = row_map(p.n, (int)p.s, p.C, p.G, sh.L);
  float *pw = nullptr, *pb = nullptr;
  const bool direct = m.npb * m.s == 1;
  if (BWD && (gw || gb)) { pw = direct ? gw : part; pb = direct ? gb : part + p.C; }
  const int stride = 2 * p.C;
  switch (dtype) {
    case kNormF32: run_rows_vec<float, BWD>(vec, sh, m, x, gy, w, b, eps, act, out, pw, pb, stride, st); break;
    case kNormBf16: run_rows_vec<__bf16, BWD>(vec, sh, m, x, gy, w, b, eps, act, out, pw, pb, stride, st); break;
    default: run_rows_vec<_Float16, BWD>(vec, sh, m, x, gy, w, b, eps, act, out, pw, pb, stride, st); break;
  }
  if (BWD && (gw || gb) && !direct)
    hipLaunchKernelGGL(norm_finish_kernel, dim3((2 * p.C + kFinishCols - 1) / kFinishCols), dim3(1024), 0, st, part,
                       (int64_t)m.npb * m.s, p.C, gw, gb);
}

template <int ND, int NS, bool BWD>
void run_jet(const RowShape& sh, const RowMap& m, const float* x, const float* gy, const float* w, const float* b,
             float eps, int act, float* out, float* pw, float* pb, int stride, hipStream_t st) {
  const dim3 grid(m.npb * m.gchunks), block(kThreads);
#define PDEKAN_JETS(LL, KK)                                                                                          \
  if (sh.L == LL && sh.K == KK) {                                                                                    \
    hipLaunchKernelGGL((norm_jet_kernel<ND, NS, LL, KK, BWD>), grid, block, 0, st, m, x, gy, w, b, eps, act, out, pw, \
                       pb, stride);                                                                                  \
    return;                                                                                                          \
  }
  PDEKAN_JETS(4, 1) PDEKAN_JETS(8, 1) PDEKAN_JETS(16, 1) PDEKAN_JETS(32, 1) PDEKAN_JETS(64, 1) PDEKAN_JETS(64, 2)
  PDEKAN_JETS(64, 4) PDEKAN_JETS(64, 8)
#undef PDEKAN_JETS
}

template <bool BWD>
void jet_any(const NormShape& p, int n_dir, const float* x, const float* gy, const float* w, const float* b, float eps,
             int act, float* out, float* gw, float* gb, float* part, hipStream_t st) {
  const RowShape sh = row_shape(p.C / p.G, 1);
  const RowMap m = row_map(p.n, 1, p.C, p.G, sh.L);
  float *pw = nullptr, *pb = nullptr;
  const bool direct = m.npb == 1;
  if (BWD && (gw || gb)) { pw = direct ? gw : part; pb = direct ? gb : part + p.C; }
  const int stride = 2 * p.C;
  if (n_dir == 2) run_jet<2, 1, BWD>(sh, m, x, gy, w, b, eps, act, out, pw, pb, stride, st);
  else run_jet<6, 5, BWD>(sh, m, x, gy, w, b, eps, act, out, pw, pb, stride, st);
  if (BWD && (gw || gb) && !direct)
    hipLaunchKernelGGL(norm_finish_kernel, dim3((2 * p.C + kFinishCols - 1) / kFinishCols), dim3(1024), 0, st, part,
                       (int64_t)m.npb, p.C, gw, gb);
}

template <typename T, int VEC>
void grid_forward(const GridMap& m, const T* x, const float* w, const float* b, float eps, int act, T* y, float2* stats,
                  double2* part, hipStream_t st) {
  const unsigned blocks = (unsigned)(m.n * m.chunks);
  const size_t lds = red_bytes<VEC>(m.C) + 2 * (size_t)m.C * sizeof(double), lds_g = 2 * (size_t)m.G * sizeof(float);
  ensure_lds((const void*)norm_grid_stats_kernel<T, VEC>, lds);
  ensure_lds((const void*)norm_grid_apply_kernel<T, VEC>, lds_g);
  hipLaunchKernelGGL((norm_grid_stats_kernel<T, VEC>), dim3(blocks), dim3(kThreads), lds, st, m, x, part);
  hipLaunchKernelGGL((norm_grid_apply_kernel<T, VEC>), dim3(blocks), dim3(kThreads), lds_g, st, m, x, w, b, eps, act,
                     part, y, stats);
}
template <typename T, int VEC>
void grid_backward(const GridMap& m, const T* x, const T* gy, const float* w, const float* b, int act,
                   const float2* stats, T* gx, float* gw, float* gb, float* part_c, float2* part_g, hipStream_t st) {
  const unsigned blocks = (unsigned)(m.n * m.chunks);
  const size_t lds = red_bytes<VEC>(m.C) + 2 * (size_t)m.C * sizeof(float), lds_g = 2 * (size_t)m.G * sizeof(float);
  ensure_lds((const void*)norm_grid_sums_kernel<T, VEC>, lds);
  ensure_lds((const void*)norm_grid_grad_kernel<T, VEC>, lds_g);
  hipLaunchKernelGGL((norm_grid_sums_kernel<T, VEC>), dim3((unsigned)m.sums), dim3(kThreads), lds, st, m, x, gy, w, b, act,
                     stats, gw || gb ? part_c : nullptr, part_g);
  const unsigned extra = gw || gb ? (2 * m.C + kGridFinishCols - 1) / kGridFinishCols : 0;
  hipLaunchKernelGGL((norm_grid_grad_kernel<T, VEC>), dim3(blocks + extra), dim3(kThreads), lds_g, st, m, x, gy, w, b,
                     act, stats, part_c, part_g, gx, gw, gb, (int)extra);
}

}  // namespace

const char* norm_refusal(const NormShape& p, int n_dir, int n_second) {
  if (p.n < 1 || p.s < 1 || p.C < 1 || p.G < 1) return "empty or negative sizes";
  if (p.C % p.G) return "the channels do not divide into the groups";
  if (p.C > kNormChannelsMax) return "more than 8192 channels";
  if (p.n > (int64_t)1 << 40 || p.s > (int64_t)1 << 24 || p.n * p.s > ((int64_t)1 << 46) / p.C) return "too many values";
  const bool jets = n_dir || n_second;
  if (jets && !((n_dir == 2 && n_second == 1) || (n_dir == 6 && n_second == 5))) return "jets of (2, 1) or (6, 5) derivatives only";
  if (jets && (p.s != 1 || p.C / p.G > 512)) return "jets take one position and at most 512 channels a group";
  // one block of 256 threads a sample at least, and a launch holds fewer than 2^32 threads
  if (!rows_kernel_takes(p.s, p.C / p.G) && p.n > (int64_t)1 << 23) return "more than 2^23 samples of many positions";
  return nullptr;
}

size_t norm_ws_bytes(const NormShape& p, bool backward) {
  if (rows_kernel_takes(p.s, p.C / p.G)) {
    if (!backward) return 0;
    // lane groups differ with the tensors' alignment: the widest spread of blocks over points any of them gives
    size_t most = 0;
    for (int L = 4; L <= 64; L *= 2) {
      const RowMap m = row_map(p.n, (int)p.s, p.C, p.G, L);
      if (m.npb * m.s > 1 && (size_t)m.npb * m.s > most) most = (size_t)m.npb * m.s;
    }
    return most * 2 * p.C * sizeof(float);
  }
  const GridMap m = grid_map(p.n, p.s, p.C, p.G);
  const size_t blocks = (size_t)m.n * m.chunks;
  return backward ? blocks * m.G * sizeof(float2) + (size_t)m.sums * 2 * m.C * sizeof(float) : blocks * m.G * sizeof(double2);
}

bool norm_wants_stats(const NormShape& p) { return !rows_kernel_takes(p.s, p.C / p.G); }

#define PDEKAN_GRID(call)                                                                                      \
  do {                                                                                                         \
    switch (dtype) {                                                                                           \
      case kNormF32: { using T = float; if (vec == 4) { constexpr int V = 4; call; } else { constexpr int V = 1; call; } break; } \
      case kNormBf16: { using T = __bf16; if (vec == 8) { constexpr int V = 8; call; } else if (vec == 2) { constexpr int V = 2; call; } else { constexpr int V = 1; call; } break; } \
      default: { using T = _Float16; if (vec == 8) { constexpr int V = 8; call; } else if (vec == 2) { constexpr int V = 2; call; } else { constexpr int V = 1; call; } break; } \
    }                                                                                                          \
  } while (0)

void launch_norm_forward(int dtype, const NormShape& p, const void* x, const float* w, const float* b, float eps, int act,
                         void* y, float* stats, void* ws, hipStream_t st) {
  if (rows_kernel_takes(p.s, p.C / p.G)) {
    rows_any<false>(dtype, p, x, nullptr, w, b, eps, act, y, nullptr, nullptr, nullptr, st);
    return;
  }
  const GridMap m = grid_map(p.n, p.s, p.C, p.G);
  const int vec = vec_width(dtype, p.C, x, y, nullptr);
  double2* part = static_cast<double2*>(ws);
  float2* s2 = reinterpret_cast<float2*>(stats);
  PDEKAN_GRID((grid_forward<T, V>(m, (const T*)x, w, b, eps, act, (T*)y, s2, part, st)));
}

void launch_norm_backward(int dtype, const NormShape& p, const void* x, const void* gy, const float* w, const float* b,
                          float eps, int act, const float* stats, void* gx, float* gw, float* gb, void* ws,
                          hipStream_t st) {
  if (rows_kernel_takes(p.s, p.C / p.G)) {
    rows_any<true>(dtype, p, x, gy, w, b, eps, act, gx, gw, gb, static_cast<float*>(ws), st);
    return;
  }
  const GridMap m = grid_map(p.n, p.s, p.C, p.G);
  const int vec = vec_width(dtype, p.C, x, gy, gx);
  float2* part_g = static_cast<float2*>(ws);
  float* part_c = reinterpret_cast<float*>(part_g + (size_t)m.n * m.chunks * m.G);
  const float2* s2 = reinterpret_cast<const float2*>(stats);
  PDEKAN_GRID((grid_backward<T, V>(m, (const T*)x, (const T*)gy, w, b, act, s2, (T*)gx, gw, gb, part_c, part_g, st)));
}

void launch_norm_jet_forward(const NormShape& p, int n_dir, const float* x, const float* w, const float* b, float eps,
                             int act, float* y, hipStream_t st) {
  jet_any<false>(p, n_dir, x, nullptr, w, b, eps, act, y, nullptr, nullptr, nullptr, st);
}

void launch_norm_jet_backward(const NormShape& p, int n_dir, const float* x, const float* gy, const float* w,
                              const float* b, float eps, int act, float* gx, float* gw, float* gb, void* ws,
                              hipStream_t st) {
  jet_any<true>(p, n_dir, x, gy, w, b, eps, act, gx, gw, gb, static_cast<float*>(ws), st);
}

}  // namespace pdekan
