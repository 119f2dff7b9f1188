// Norms before and after a block, fused with the block's gate and residual scale (gfx950), over rows of D:
//
//   n = norm(h) * pw + pb,   y = x + scale * act(gate) * n,   u = norm(y) * rw + rb
//
// norm divides by the root of the mean square + eps, after taking the mean off for LayerNorm.  Backward, with
// B(d; z, r) = r (d - z mean(d z) [- mean(d)]) the norm's own backward (z its output, r = 1 / root):
//   g = dy + B(du rw; norm(y), r_y) = dx,   dgate = g scale n act',   dh = B(g scale act pw; norm(h), r_h),
// and, summed over the rows,
//   A = sum g act norm(h),  Z = sum g act:   dscale = pw A + pb Z,  dpw = scale A,  dpb = scale Z,
//   drw = sum du norm(y),  drb = sum du.
//
// Bound by memory: 3 reads and 2 writes an element forward, 5 and 3 backward.  A row is read once and stays in
// registers: L lanes hold V elements each, so every statistic is taken of registers.  A workgroup walks many rows and keeps the
// weights in registers too (fp32 weights read again for each row would be more than the row itself in bf16), and the next row
// is on its way while this one is worked on.  The parameter sums stay in registers over the rows that a group of lanes
// walks; each workgroup leaves one partial sum of every column and residual_norm_sum_kernel adds them in a fixed order,
// so results repeat bit by bit.
//
// Measured, in a kernel trace: forward, bf16, 8191 x 2048 29 us (5.8 TB/s), 8192 x 4096 61 us (5.5 TB/s; a copy of that size 5.2); backward
// 8192 x 4096 129 us (4.2 TB/s: two workgroups of 512 a CU, for the partial sums' sake) and 13 us for the sums; fp32, 16384
// x 256 16 and 26 us and 6 us.  bf16 rows of 1001 go by elements: 5003 of them 19 and 39 us.  Outputs are stored through the
// caches: past them the kernel is up to 12 % faster by itself, but what reads y and u next loses more (98 -> 109 us together).
#include "delta.h"
#include "residual_norm.h"

namespace srl {
namespace rnorm {

using delta::bf16;
using delta::ld1;
using delta::st1;

// Column of element e of lane i.  VEC: 16 bytes of neighbours a lane (8 where V is less); else (rows that are not
// aligned) one element a lane, so that a wave still reads neighbours.
template <typename T, int L, int V, bool VEC>
__device__ __forceinline__ int column(int e, int i) {
  constexpr int G = V < 16 / (int)sizeof(T) ? V : 16 / (int)sizeof(T);
  return VEC ? (e / G) * G * L + G * i + e % G : e * L + i;
}

// One row's elements of a lane as they lie in memory, so that a row on its way costs few registers.
template <typename T, int L, int V, bool VEC>
struct Row {
  static constexpr int G = V < 16 / (int)sizeof(T) ? V : 16 / (int)sizeof(T), NB = V * (int)sizeof(T) / 4;
  uint32_t w[VEC ? NB : 1];
  T e_[VEC ? 1 : V];
  __device__ __forceinline__ void load(const T* p, int i, int D) {
#pragma unroll
    for (int e = 0; e < V; e += VEC ? G : 1) {
      const int c = column<T, L, V, VEC>(e, i);
      if constexpr (VEC) {
        constexpr int W = G * (int)sizeof(T) / 4;
        uint32_t* o = w + e * (int)sizeof(T) / 4;
        if (c < D) {
          if constexpr (W == 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(p + c);
            o[0] = x.x, o[1] = x.y, o[2] = x.z, o[3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(p + c);
            o[0] = x.x, o[1] = x.y;
          }
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j) o[j] = 0;
        }
      } else {
        if (c < D) e_[e] = p[c];
        else e_[e] = T{};
      }
    }
  }
  __device__ __forceinline__ void get(float* o) const {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if constexpr (!VEC) o[e] = ld1(&e_[e]);
      else if constexpr (sizeof(T) == 4) o[e] = __builtin_bit_cast(float, w[e]);
      else o[e] = __builtin_bit_cast(float, e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
  }
};
template <typename T, int L, int V, bool VEC>
__device__ __forceinline__ void store_row(T* p, int i, int D, const float* v) {
  constexpr int G = Row<T, L, V, VEC>::G;
#pragma unroll
  for (int e = 0; e < V; e += VEC ? G : 1) {
    const int c = column<T, L, V, VEC>(e, i);
    if (c >= D) continue;
    if constexpr (!VEC) {
      st1(p + c, v[e]);
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<delta::f4*>(p + c) = delta::f4{v[e], v[e + 1], v[e + 2], v[e + 3]};
    } else {
      uint32_t w[G / 2];
#pragma unroll
      for (int j = 0; j < G / 2; ++j) w[j] = delta::f2bf2(v[e + 2 * j], v[e + 2 * j + 1]);
      if constexpr (G == 8) *reinterpret_cast<uint4*>(p + c) = uint4{w[0], w[1], w[2], w[3]};
      else *reinterpret_cast<uint2*>(p + c) = uint2{w[0], w[1]};
    }
  }
}
// Weights of a lane's columns; those past D read the last one's, and no result takes them.  VEC: 16 bytes at a time, for each
// element by itself reads every cache line eight times.
template <typename T, int L, int V, bool VEC>
__device__ __forceinline__ void load_par(const float* p, int i, int D, float other, float* o) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = other;
  } else if constexpr (VEC) {
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      const delta::f4 x = *reinterpret_cast<const delta::f4*>(p + min(column<T, L, V, VEC>(e, i), D - 4));
#pragma unroll
      for (int j = 0; j < 4; ++j) o[e + j] = x[j];
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = p[min(column<T, L, V, VEC>(e, i), D - 1)];
  }
}

// Sum over the L lanes of a row: 16 lanes or a wave in registers, more through LDS.  The two buffers take turns, so one barrier
// a sum is enough: a wave that writes a buffer again has passed the barrier of the sum between.
template <int L>
struct Sum {
  float* red;  // [2][2 * L / 64]
  int turn = 0;
  __device__ __forceinline__ float2 operator()(float2 v) {
    if constexpr (L == 16) {
      return float2{row16_sum(v.x), row16_sum(v.y)};
    } else {
      v.x = wave_sum_dpp(v.x);
      v.y = wave_sum_dpp(v.y);
      if constexpr (L > 64) {
        constexpr int NW = L / 64;
        float* r = red + turn * 2 * NW;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) *reinterpret_cast<float2*>(r + 2 * (threadIdx.x >> 6)) = v;
        __syncthreads();
        v = float2{0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NW; ++i) v.x += r[2 * i], v.y += r[2 * i + 1];
      }
      return v;
    }
  }
};

// z <- norm(z), and the factor; columns past D stay zero.  The mean goes first: a sum of squares about it loses nothing.
template <typename T, int L, int V, bool VEC>
__device__ __forceinline__ float normalise(float* z, int i, const Args& a, Sum<L>& sum) {
  if (a.layer) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) s += z[e];
    const float mean = sum(float2{s, 0.f}).x * a.inv_d;
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = column<T, L, V, VEC>(e, i) < a.D ? z[e] - mean : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) q = fmaf(z[e], z[e], q);
  const float r = 1.f / sqrtf(sum(float2{q, 0.f}).x * a.inv_d + a.eps);
#pragma unroll
  for (int e = 0; e < V; ++e) z[e] *= r;
  return r;
}

// by the hardware's exponential and reciprocal: each is off by one unit in the last place and the exponential by |x| 2^-24 more,
// against 2.5 times the instructions of expf and a division, which bound the kernel in bf16
__device__ __forceinline__ float sig(float x) { return __builtin_amdgcn_rcpf(1.f + __expf(-x)); }
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

template <int L>
constexpr int threads() { return L <= 64 ? 256 : L; }
template <int L>
constexpr int rows_at_once() { return L <= 64 ? 256 / L : 1; }

template <typename T, int L, int V, bool VEC>
__global__ void __launch_bounds__(threads<L>()) residual_norm_fwd_kernel(Args a) {
  __shared__ __align__(16) float red[4 * (L <= 64 ? 1 : L / 64)];
  constexpr int RPB = rows_at_once<L>();
  const int i = threadIdx.x % L;
  Sum<L> sum{red};
  long row = (long)blockIdx.x * RPB + threadIdx.x / L;
  if (row >= a.rows) return;  // whole workgroups where the lanes of a row are more than a wave
  float sp[V], sb[V], rw[V], rb[V];
  Row<T, L, V, VEC> rx, rh, rg;
  const T *xp = reinterpret_cast<const T*>(a.x), *hp = reinterpret_cast<const T*>(a.h), *gp = reinterpret_cast<const T*>(a.gate);
  rh.load(hp + row * a.hs, i, a.D);
  rx.load(xp + row * a.xs, i, a.D);
  if (gp) rg.load(gp + row * a.gs, i, a.D);
  load_par<T, L, V, VEC>(a.scale, i, a.D, a.s1, rw);
  load_par<T, L, V, VEC>(a.pw, i, a.D, 1.f, sp);
  load_par<T, L, V, VEC>(a.pb, i, a.D, 0.f, sb);
#pragma unroll
  for (int e = 0; e < V; ++e) sp[e] *= rw[e], sb[e] *= rw[e];
  load_par<T, L, V, VEC>(a.rw, i, a.D, 1.f, rw);
  load_par<T, L, V, VEC>(a.rb, i, a.D, 0.f, rb);
  const long step = (long)gridDim.x * RPB;
  while (true) {
    float x[V], n[V], g[V];
    rh.get(n);
    rx.get(x);
    if (gp) rg.get(g);
    const long next = row + step;
    if (next < a.rows) {
      rh.load(hp + next * a.hs, i, a.D);
      rx.load(xp + next * a.xs, i, a.D);
      if (gp) rg.load(gp + next * a.gs, i, a.D);
    }
    normalise<T, L, V, VEC>(n, i, a, sum);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float s;
      const float act = gp ? gate_act(g[e], a.act, s) : 1.f;
      x[e] = column<T, L, V, VEC>(e, i) < a.D ? fmaf(act, fmaf(n[e], sp[e], sb[e]), x[e]) : 0.f;
    }
    store_row<T, L, V, VEC>(reinterpret_cast<T*>(a.y) + row * a.D, i, a.D, x);
    normalise<T, L, V, VEC>(x, i, a, sum);
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = fmaf(x[e], rw[e], rb[e]);
    store_row<T, L, V, VEC>(reinterpret_cast<T*>(a.u) + row * a.D, i, a.D, x);
    if (next >= a.rows) break;
    row = next;
  }
}

// d <- B(d; z, r)
template <int L, int V>
__device__ __forceinline__ void norm_back(float* d, const float* z, float r, const Args& a, Sum<L>& sum) {
  float2 s = {0.f, 0.f};
#pragma unroll
  for (int e = 0; e < V; ++e) {
    s.x = fmaf(d[e], z[e], s.x);
    s.y += d[e];
  }
  s = sum(s);
  const float m = s.x * a.inv_d, c = a.layer ? s.y * a.inv_d : 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) d[e] = r * (d[e] - z[e] * m - c);
}

template <typename T, int L, int V, bool VEC>
__global__ void __launch_bounds__(threads<L>()) residual_norm_bwd_kernel(Args a, BwdArgs o) {
  __shared__ __align__(16) float red[4 * (L <= 64 ? 1 : L / 64)];
  __shared__ float acc[L <= 64 ? 256 * V : 1];
  constexpr int RPB = rows_at_once<L>();
  const int i = threadIdx.x % L, grp = threadIdx.x / L;
  Sum<L> sum{red};
  float gA[V], gZ[V], gR[V], gRb[V], pw[V], pb[V], sc[V], rw[V];
#pragma unroll
  for (int e = 0; e < V; ++e) gA[e] = gZ[e] = gR[e] = gRb[e] = 0.f;
  load_par<T, L, V, VEC>(a.scale, i, a.D, a.s1, sc);
  load_par<T, L, V, VEC>(a.pw, i, a.D, 1.f, pw);
  load_par<T, L, V, VEC>(a.pb, i, a.D, 0.f, pb);
  load_par<T, L, V, VEC>(a.rw, i, a.D, 1.f, rw);
  const T *xp = reinterpret_cast<const T*>(a.x), *hp = reinterpret_cast<const T*>(a.h), *gp = reinterpret_cast<const T*>(a.gate);
  const T *yp = reinterpret_cast<const T*>(o.dy), *up = reinterpret_cast<const T*>(o.du);
  const long step = (long)gridDim.x * RPB;
  long row = (long)blockIdx.x * RPB + grp;
  Row<T, L, V, VEC> rx, rh, rg, ry, ru;
  auto fetch = [&](long r) {
    rh.load(hp + r * a.hs, i, a.D);
    rx.load(xp + r * a.xs, i, a.D);
    if (gp) rg.load(gp + r * a.gs, i, a.D);
    if (up) ru.load(up + r * o.dus, i, a.D);
    if (yp) ry.load(yp + r * o.dys, i, a.D);
  };
  if (row < a.rows) fetch(row);
  for (; row < a.rows; row += step) {
    float x[V], hn[V], act[V], sl[V], d[V], t[V];
    rh.get(hn);
    rx.get(x);
#pragma unroll
    for (int e = 0; e < V; ++e) act[e] = 1.f, sl[e] = 0.f, d[e] = 0.f, t[e] = 0.f;
    if (gp) {
      rg.get(act);
#pragma unroll
      for (int e = 0; e < V; ++e) act[e] = gate_act(act[e], a.act, sl[e]);
    }
    if (up) ru.get(d);
    if (yp) ry.get(t);
    if (row + step < a.rows) fetch(row + step);
    const float fh = normalise<T, L, V, VEC>(hn, i, a, sum);
#pragma unroll
    for (int e = 0; e < V; ++e)
      x[e] = column<T, L, V, VEC>(e, i) < a.D ? fmaf(sc[e] * act[e], fmaf(hn[e], pw[e], pb[e]), x[e]) : 0.f;
    const float fy = normalise<T, L, V, VEC>(x, i, a, sum);
    if (up) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        gR[e] = fmaf(d[e], x[e], gR[e]);
        gRb[e] += d[e];
        d[e] *= rw[e];
      }
      norm_back<L, V>(d, x, fy, a, sum);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) d[e] += t[e];
    store_row<T, L, V, VEC>(reinterpret_cast<T*>(o.dx) + row * a.D, i, a.D, d);
    if (o.dgate) {
#pragma unroll
      for (int e = 0; e < V; ++e) t[e] = d[e] * sc[e] * fmaf(hn[e], pw[e], pb[e]) * sl[e];
      store_row<T, L, V, VEC>(reinterpret_cast<T*>(o.dgate) + row * a.D, i, a.D, t);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      d[e] = column<T, L, V, VEC>(e, i) < a.D ? d[e] * act[e] : 0.f;
      gA[e] = fmaf(d[e], hn[e], gA[e]);
      gZ[e] += d[e];
      d[e] *= sc[e] * pw[e];
    }
    norm_back<L, V>(d, hn, fh, a, sum);
    store_row<T, L, V, VEC>(reinterpret_cast<T*>(o.dh) + row * a.D, i, a.D, d);
  }
  auto leave = [&](const float* g, int k) {
    float* out = o.part + ((long)blockIdx.x * 4 + k) * a.D;
    if constexpr (L <= 64) {  // the workgroup's row groups, in order
      __syncthreads();
#pragma unroll
      for (int e = 0; e < V; ++e) acc[grp * L * V + column<T, L, V, VEC>(e, i)] = g[e];
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
        const int c = column<T, L, V, VEC>(e, i);
        if (c < a.D) out[c] = g[e];
      }
    }
  };
  leave(gA, 0);
  leave(gZ, 1);
  leave(gR, 2);
  leave(gRb, 3);
}

// The four sums of 16 columns over the workgroups' partials, 16 waves a row of partials each at a time, joined in a
// fixed order; then the five gradients, out [5, D]: scale, post weight and bias, pre weight and bias.  (4 columns a workgroup,
// for four times the workgroups, read every cache line on eight chiplets: 19 us instead of 11 at 1024 partials of 1001 columns.)
__global__ void __launch_bounds__(1024) residual_norm_sum_kernel(const float* part, float* out, int W, Args a) {
  __shared__ float s[16][64];
  const int lane = threadIdx.x & 63, r = threadIdx.x >> 6, k = lane >> 4, c = blockIdx.x * 16 + (lane & 15);
  float v = 0.f;
  if (c < a.D) {
    const float* p = part + (long)k * a.D + c;
#pragma unroll 16
    for (int w = r; w < W; w += 16) v += p[(long)w * 4 * a.D];
  }
  s[r][lane] = v;
  __syncthreads();
  if (r != 0) return;
  v = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) v += s[j][lane];
  const float A = __shfl(v, lane & 15, 64), Z = __shfl(v, 16 + (lane & 15), 64);
  if (c >= a.D) return;
  if (k == 0) {
    const float pw = a.pw ? a.pw[c] : 1.f, pb = a.pb ? a.pb[c] : 0.f, sc = a.scale ? a.scale[c] : a.s1;
    out[c] = fmaf(pw, A, pb * Z);
    out[a.D + c] = sc * A;
    out[2 * (long)a.D + c] = sc * Z;
  } else if (k >= 2) {
    out[(long)(k + 1) * a.D + c] = v;
  }
}

template <typename T, int L, int V, bool VEC>
static void run(const Args& a, const BwdArgs* o, int W, hipStream_t st) {
  constexpr int RPB = rows_at_once<L>(), TH = threads<L>();
  if (o) {
    residual_norm_bwd_kernel<T, L, V, VEC><<<W, TH, 0, st>>>(a, *o);
  } else {
    const int need = (a.rows + RPB - 1) / RPB, most = 256 * (2048 / TH);
    residual_norm_fwd_kernel<T, L, V, VEC><<<need < most ? need : most, TH, 0, st>>>(a);
  }
}

template <typename T, bool VEC>
static void pick(const Args& a, const BwdArgs* o, int W, hipStream_t st) {
  // as few lanes a row as leave a lane at most 8 elements of each operand: with more of them the weights and the parameter
  // sums of the backward pass do not fit the registers
  if (a.D <= 64) run<T, 16, 4, VEC>(a, o, W, st);
  else if (a.D <= 256) run<T, 64, 4, VEC>(a, o, W, st);
  else if (a.D <= 512) run<T, 64, 8, VEC>(a, o, W, st);
  else if (a.D <= 1024) run<T, 256, 4, VEC>(a, o, W, st);
  else if (a.D <= 2048) run<T, 256, 8, VEC>(a, o, W, st);
  else if (a.D <= 4096) run<T, 512, 8, VEC>(a, o, W, st);
  else run<T, 1024, 8, VEC>(a, o, W, st);
}

int residual_norm_groups(int rows, int D) {
  const int rpb = D <= 64 ? 16 : D <= 512 ? 4 : 1;
  const int need = (rows + rpb - 1) / rpb, most = D <= 4096 ? 512 : 256;
  return need < most ? need : most;
}

static void start(const Args& a, const BwdArgs* o, int W, bool is_bf16, bool vec, hipStream_t st) {
  if (is_bf16) {
    if (vec) pick<bf16, true>(a, o, W, st);
    else pick<bf16, false>(a, o, W, st);
  } else {
    if (vec) pick<float, true>(a, o, W, st);
    else pick<float, false>(a, o, W, st);
  }
}

void launch_residual_norm_fwd(const Args& a, bool is_bf16, bool vec, hipStream_t st) { start(a, nullptr, 0, is_bf16, vec, st); }

void launch_residual_norm_bwd(const Args& a, const BwdArgs& o, float* sums, bool is_bf16, bool vec, hipStream_t st) {
  const int W = residual_norm_groups(a.rows, a.D);
  start(a, &o, W, is_bf16, vec, st);
  residual_norm_sum_kernel<<<(a.D + 15) / 16, 1024, 0, st>>>(o.part, sums, W, a);
}

}  // namespace rnorm
}  // namespace srl
