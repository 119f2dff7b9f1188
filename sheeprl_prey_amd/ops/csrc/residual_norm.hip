// Norms before and after a block, fused with the block's gate and residual scale (gfx950), over rows of D:
//
//   n = norm(h) * pw + pb,   y = x + scale * act(gate) * n,   u = norm(y) * rw + rb
//
// norm divides by the root of the mean square + eps, after taking the mean off for LayerNorm.  Backward, with
// B(d; z, r) = r (d - z mean(d z) [- mean(d)]) the norm's own backward (z its output, r = 1 / root):
//   g = dy + B(du rw; norm(y), r_y) = dx,   dgate = g scale n act',   dh = B(g scale act pw; norm(h), r_h),
//   dscale = sum g act n,  dpw = sum g scale act norm(h),  dpb = sum g scale act,  drw = sum du norm(y),  drb = sum du
// with the sums over the rows.
//
// Bound by memory: 3 reads and 2 writes an element forward, 5 and 3 backward.  A row is read once and stays in
// registers: L lanes of a row hold V elements each (V / 4 reads of 16 bytes in fp32), so every statistic is taken of registers.
// The parameter sums stay in registers too over the rows that a group of lanes walks; each workgroup leaves one
// partial sum of every column and residual_norm_sum_kernel adds them in a fixed order, so results repeat bit by bit.
#include "delta.h"
#include "residual_norm.h"

namespace srl {
namespace rnorm {

using delta::bf16;
using delta::ld1;
using delta::st1;

// Sum over the L lanes of a row (L <= 64: aligned lanes of a wave; more: whole workgroup of L threads).
template <int L>
__device__ __forceinline__ float2 row_sum2(float2 v, float* red) {
  if constexpr (L <= 64) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) {
      v.x += __shfl_xor(v.x, o, 64);
      v.y += __shfl_xor(v.y, o, 64);
    }
    return v;
  } else {
    constexpr int NW = L / 64;
    v.x = wave_sum(v.x);
    v.y = wave_sum(v.y);
    const int w = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[2 * w] = v.x, red[2 * w + 1] = v.y;
    __syncthreads();
    float2 s = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NW; ++i) s.x += red[2 * i], s.y += red[2 * i + 1];
    return s;
  }
}

// Element e of lane i of a row: G = 4 neighbours at a time, i.e. column (e / 4) * 4 L + 4 i + e % 4.
template <typename T, int L, int V>
__device__ __forceinline__ void load_row(const T* p, int i, int D, bool vec, float* o) {
#pragma unroll
  for (int e = 0; e < V; e += 4) {
    const int c = (e / 4) * 4 * L + 4 * i;
    if (vec) {
      if (c < D) delta::ldv<4>(p + c, o + e);
      else {
#pragma unroll
        for (int j = 0; j < 4; ++j) o[e + j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[e + j] = c + j < D ? ld1(p + c + j) : 0.f;
    }
  }
}
__device__ __forceinline__ void st4(float* p, const float* v) { *reinterpret_cast<delta::f4*>(p) = delta::f4{v[0], v[1], v[2], v[3]}; }
__device__ __forceinline__ void st4(bf16* p, const float* v) {
  uint2 w;
  w.x = (uint32_t)delta::f2bf(v[0]) | ((uint32_t)delta::f2bf(v[1]) << 16);
  w.y = (uint32_t)delta::f2bf(v[2]) | ((uint32_t)delta::f2bf(v[3]) << 16);
  *reinterpret_cast<uint2*>(p) = w;
}
template <typename T, int L, int V>
__device__ __forceinline__ void store_row(T* p, int i, int D, bool vec, const float* v) {
#pragma unroll
  for (int e = 0; e < V; e += 4) {
    const int c = (e / 4) * 4 * L + 4 * i;
    if (vec) {
      if (c < D) st4(p + c, v + e);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < D) st1(p + c + j, v[e + j]);
    }
  }
}
template <int L, int V>
__device__ __forceinline__ void load_par(const float* p, int i, int D, float other, float* o) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = (e / 4) * 4 * L + 4 * i + e % 4;
    o[e] = p && c < D ? p[c] : other;
  }
}

// z <- norm(z), and the factor; columns past D stay zero.  The mean goes first: a sum of squares about it loses nothing.
template <int L, int V>
__device__ __forceinline__ float normalise(float* z, int i, const Args& a, float* red) {
  if (a.layer) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) s += z[e];
    const float mean = row_sum2<L>(float2{s, 0.f}, red).x * a.inv_d;
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = (e / 4) * 4 * L + 4 * i + e % 4 < a.D ? z[e] - mean : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) q = fmaf(z[e], z[e], q);
  const float r = 1.f / sqrtf(row_sum2<L>(float2{q, 0.f}, red).x * a.inv_d + a.eps);
#pragma unroll
  for (int e = 0; e < V; ++e) z[e] *= r;
  return r;
}

__device__ __forceinline__ float sig(float x) { return 1.f / (1.f + expf(-x)); }
// act(z) and its slope
__device__ __forceinline__ float gate_act(float z, int act, float& slope) {
  if (act == ACT_NONE) {
    slope = 1.f;
    return z;
  }
  const float s = sig(z), d = s * (1.f - s);
  if (act == SIGMOID) {
    slope = d;
    return s;
  }
  slope = fmaf(z, d, s);
  return z * s;
}

template <typename T, int L, int V>
__global__ void __launch_bounds__(L <= 64 ? 256 : L) residual_norm_fwd_kernel(Args a, int vec) {
  __shared__ float red[2 * (L <= 64 ? 1 : L / 64)];
  constexpr int RPB = L <= 64 ? 256 / L : 1;
  const int i = threadIdx.x % L;
  const long row = (long)blockIdx.x * RPB + threadIdx.x / L;
  if (L <= 64 && row >= a.rows) return;
  float x[V], n[V], w[V];
  load_row<T, L, V>(reinterpret_cast<const T*>(a.h) + row * a.hs, i, a.D, vec, n);
  load_row<T, L, V>(reinterpret_cast<const T*>(a.x) + row * a.xs, i, a.D, vec, x);
  if (a.gate) load_row<T, L, V>(reinterpret_cast<const T*>(a.gate) + row * a.gs, i, a.D, vec, w);
  normalise<L, V>(n, i, a, red);
  float p[V];
  load_par<L, V>(a.pw, i, a.D, 1.f, p);
#pragma unroll
  for (int e = 0; e < V; ++e) n[e] *= p[e];
  load_par<L, V>(a.pb, i, a.D, 0.f, p);
#pragma unroll
  for (int e = 0; e < V; ++e) n[e] += p[e];
  load_par<L, V>(a.scale, i, a.D, a.s1, p);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float s;
    x[e] = fmaf(p[e] * (a.gate ? gate_act(w[e], a.act, s) : 1.f), n[e], x[e]);
    if ((e / 4) * 4 * L + 4 * i + e % 4 >= a.D) x[e] = 0.f;
  }
  store_row<T, L, V>(reinterpret_cast<T*>(a.y) + row * a.D, i, a.D, vec, x);
  normalise<L, V>(x, i, a, red);
  load_par<L, V>(a.rw, i, a.D, 1.f, p);
  load_par<L, V>(a.rb, i, a.D, 0.f, w);
#pragma unroll
  for (int e = 0; e < V; ++e) x[e] = fmaf(x[e], p[e], w[e]);
  store_row<T, L, V>(reinterpret_cast<T*>(a.u) + row * a.D, i, a.D, vec, x);
}

// d <- B(d; z, r)
template <int L, int V>
__device__ __forceinline__ void norm_back(float* d, const float* z, float r, int i, const Args& a, float* red) {
  float2 s = {0.f, 0.f};
#pragma unroll
  for (int e = 0; e < V; ++e) {
    s.x = fmaf(d[e], z[e], s.x);
    s.y += d[e];
  }
  s = row_sum2<L>(s, red);
  const float m = s.x * a.inv_d, c = a.layer ? s.y * a.inv_d : 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) d[e] = r * (d[e] - z[e] * m - c);
}

template <typename T, int L, int V>
__global__ void __launch_bounds__(L <= 64 ? 256 : L) residual_norm_bwd_kernel(Args a, BwdArgs o, int vec) {
  __shared__ float red[2 * (L <= 64 ? 1 : L / 64)];
  __shared__ float acc[L <= 64 ? 256 * V : 1];
  constexpr int RPB = L <= 64 ? 256 / L : 1;
  const int i = threadIdx.x % L, grp = threadIdx.x / L;
  float gS[V], gP[V], gPb[V], gR[V], gRb[V];
#pragma unroll
  for (int e = 0; e < V; ++e) gS[e] = gP[e] = gPb[e] = gR[e] = gRb[e] = 0.f;
  for (long row = (long)blockIdx.x * RPB + grp; row < a.rows; row += (long)gridDim.x * RPB) {
    float x[V], hn[V], gt[V], d[V], t[V], p[V];
    load_row<T, L, V>(reinterpret_cast<const T*>(a.h) + row * a.hs, i, a.D, vec, hn);
    load_row<T, L, V>(reinterpret_cast<const T*>(a.x) + row * a.xs, i, a.D, vec, x);
    if (a.gate) load_row<T, L, V>(reinterpret_cast<const T*>(a.gate) + row * a.gs, i, a.D, vec, gt);
    if (o.du) load_row<T, L, V>(reinterpret_cast<const T*>(o.du) + row * o.dus, i, a.D, vec, d);
    if (o.dy) load_row<T, L, V>(reinterpret_cast<const T*>(o.dy) + row * o.dys, i, a.D, vec, t);
    const float rh = normalise<L, V>(hn, i, a, red);
    // n = hn pw + pb; gt becomes act, and y goes into x
    float n[V], sl[V];
    load_par<L, V>(a.pw, i, a.D, 1.f, n);
    load_par<L, V>(a.pb, i, a.D, 0.f, p);
#pragma unroll
    for (int e = 0; e < V; ++e) n[e] = fmaf(hn[e], n[e], p[e]);
    load_par<L, V>(a.scale, i, a.D, a.s1, p);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (a.gate) gt[e] = gate_act(gt[e], a.act, sl[e]);
      else gt[e] = 1.f;
      x[e] = fmaf(p[e] * gt[e], n[e], x[e]);
      if ((e / 4) * 4 * L + 4 * i + e % 4 >= a.D) x[e] = 0.f;
    }
    const float ry = normalise<L, V>(x, i, a, red);
    if (o.du) {
      float w[V];
      load_par<L, V>(a.rw, i, a.D, 1.f, w);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        gR[e] = fmaf(d[e], x[e], gR[e]);
        gRb[e] += d[e];
        d[e] *= w[e];
      }
      norm_back<L, V>(d, x, ry, i, a, red);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = 0.f;
    }
    if (o.dy) {
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] += t[e];
    }
    store_row<T, L, V>(reinterpret_cast<T*>(o.dx) + row * a.D, i, a.D, vec, d);
    if (o.dgate) {
#pragma unroll
      for (int e = 0; e < V; ++e) t[e] = d[e] * p[e] * n[e] * sl[e];
      store_row<T, L, V>(reinterpret_cast<T*>(o.dgate) + row * a.D, i, a.D, vec, t);
    }
    load_par<L, V>(a.pw, i, a.D, 1.f, t);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      gS[e] = fmaf(d[e] * gt[e], n[e], gS[e]);
      d[e] *= p[e] * gt[e];
      if ((e / 4) * 4 * L + 4 * i + e % 4 >= a.D) d[e] = 0.f;
      gP[e] = fmaf(d[e], hn[e], gP[e]);
      gPb[e] += d[e];
      d[e] *= t[e];
    }
    norm_back<L, V>(d, hn, rh, i, a, red);
    store_row<T, L, V>(reinterpret_cast<T*>(o.dh) + row * a.D, i, a.D, vec, d);
  }
  float* g[5] = {gS, gP, gPb, gR, gRb};
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    float* out = o.part + ((long)blockIdx.x * 5 + k) * a.D;
    if constexpr (L <= 64) {  // the workgroup's row groups, in order
      __syncthreads();
#pragma unroll
      for (int e = 0; e < V; ++e) acc[grp * L * V + (e / 4) * 4 * L + 4 * i + e % 4] = g[k][e];
      __syncthreads();
      for (int c = threadIdx.x; c < a.D; c += 256) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < RPB; ++r) s += acc[r * L * V + c];
        out[c] = s;
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = (e / 4) * 4 * L + 4 * i + e % 4;
        if (c < a.D) out[c] = g[k][e];
      }
    }
  }
}

// out[k][c] = sum of part[w][k][c] over the workgroups: 16 rows of partials at a time, joined in a fixed order.
__global__ void __launch_bounds__(256) residual_norm_sum_kernel(const float* part, float* out, int W, int n) {
  __shared__ float s[16][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  float v = 0.f;
  if (col < n)
    for (int w = r; w < W; w += 16) v += part[(long)w * n + col];
  s[r][c] = v;
  __syncthreads();
  if (r == 0 && col < n) {
    v = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) v += s[k][c];
    out[col] = v;
  }
}

template <typename T, int L, int V>
static void run(const Args& a, const BwdArgs* o, bool vec, int W, hipStream_t st) {
  constexpr int RPB = L <= 64 ? 256 / L : 1, TH = L <= 64 ? 256 : L;
  if (o) residual_norm_bwd_kernel<T, L, V><<<W, TH, 0, st>>>(a, *o, vec);
  else residual_norm_fwd_kernel<T, L, V><<<(a.rows + RPB - 1) / RPB, TH, 0, st>>>(a, vec);
}

template <typename T>
static void pick(const Args& a, const BwdArgs* o, bool vec, int W, hipStream_t st) {
  if (a.D <= 64) run<T, 16, 4>(a, o, vec, W, st);
  else if (a.D <= 256) run<T, 64, 4>(a, o, vec, W, st);
  else if (a.D <= 512) run<T, 64, 8>(a, o, vec, W, st);
  else if (a.D <= 1024) run<T, 256, 4>(a, o, vec, W, st);
  else if (a.D <= 2048) run<T, 256, 8>(a, o, vec, W, st);
  else if (a.D <= 4096) run<T, 512, 8>(a, o, vec, W, st);
  else run<T, 1024, 8>(a, o, vec, W, st);
}

int residual_norm_groups(int rows, int D) {
  const int rpb = D <= 64 ? 16 : D <= 512 ? 4 : 1;
  const int need = (rows + rpb - 1) / rpb;
  return need < 1024 ? need : 1024;
}

void launch_residual_norm_fwd(const Args& a, bool is_bf16, bool vec, hipStream_t st) {
  if (is_bf16) pick<bf16>(a, nullptr, vec, 0, st);
  else pick<float>(a, nullptr, vec, 0, st);
}

void launch_residual_norm_bwd(const Args& a, const BwdArgs& o, float* sums, bool is_bf16, bool vec, hipStream_t st) {
  const int W = residual_norm_groups(a.rows, a.D), n = 5 * a.D;
  if (is_bf16) pick<bf16>(a, &o, vec, W, st);
  else pick<float>(a, &o, vec, W, st);
  residual_norm_sum_kernel<<<(n + 15) / 16, 256, 0, st>>>(o.part, sums, W, n);
}

}  // namespace rnorm
}  // namespace srl
