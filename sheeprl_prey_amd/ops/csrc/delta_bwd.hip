// The gated delta rule, chunked form, backward (the mathematics and the layout: delta.h).
//
// With dS the gradient of a chunk's last state, dO that of its outputs, and T = (I + A)^-1:
//   dU = P^T dO + diag(e) K dS,   dR = T^T dU,   dV = diag(beta) dR,
//   dS0 = gam_C dS + scale Q^T diag(gam) dO - K^T diag(beta gam) dR:
// again nothing mixes the value columns, so delta_bwd_walk_kernel walks the chunks backwards with one wave a strip of 16
// of them, dS in registers, split into segments over a long axis as the forward walk is (the map of dS over a segment
// is the transpose of Pseg).  What sums over the value columns is left to delta_grads_kernel, one workgroup a chunk
// and no order among them:
//   W1 = M o tril(dO U^T),  W2 = -diag(beta) M o tril(dR U^T, -1),  GO = dO S0^T, GR = dR S0^T, GU = U dS^T,
//   dQ = scale (diag(gam) GO + W1 K),
//   dK = -diag(beta gam) GR + diag(e) GU + scale W1^T Q + (W2 + W2^T) K,
//   dbeta_i = dR_i . v_i - gam_i k_i . GR_i + sum_j (W2 / beta o K K^T)_ij,
//   dG_i = scale gam_i q_i . GO_i - beta_i gam_i k_i . GR_i + (row_i - column_i)(scale W1 o Q K^T + W2 o K K^T) - F_i,
// F_i = e_i k_i . GU_i, dG of the chunk's last step takes sum F + gam_C <S0, dS> too, and the gradient of g_i is the
// sum of dG over the steps from i to the end of its segment.
//
// Measured at 4096 steps x 2 x 16 heads of 128 in bf16, us in a kernel trace: maps 99, joins 24, walk 111 (bound as the forward
// walk is), gradients of q and k 273.  The last reads the states and their gradients at every chunk, 192 KB a chunk and head of which
// a third of its time is, and has one workgroup on a CU; the rest is products on operands cut into three parts, whose reads
// from LDS take as long as the matrix instructions.
#include "delta.h"

namespace srl {
namespace delta {

template <typename T, int DKT>
__global__ void __launch_bounds__(512) delta_bwd_short_kernel(Args a, BwdArgs o) {
  constexpr int C = 16, LD = 16 * DKT + 4, DKp = 16 * DKT;
  extern __shared__ __align__(16) unsigned char lds[];
  Gates<C>& s = *reinterpret_cast<Gates<C>*>(lds);
  float* K = reinterpret_cast<float*>(lds + sizeof(Gates<C>));
  float* Q = K + C * LD;
  float* A = Q + C * LD;
  float* P = A + C * LT;
  float* Td = P + C * LT;

  const int lane = threadIdx.x & 63, l16 = lane & 15, kq = lane >> 4, wave = wave_id(), nw = blockDim.x >> 6;
  const int BH = a.B * a.Hv, bh = blockIdx.x, b = bh / a.Hv, h = bh % a.Hv, hk = h / (a.Hv / a.Hk);
  const int Dvp = pitch(a.Dv), dv = 16 * wave + l16;
  const int len = a.lengths ? max(0, min(a.T, a.lengths[b])) : a.T;
  const T* qp = reinterpret_cast<const T*>(a.q) + (long)b * a.qb + (long)hk * a.qh;
  const T* kp = reinterpret_cast<const T*>(a.k) + (long)b * a.kb + (long)hk * a.kh;
  const T* gp = o.dout ? reinterpret_cast<const T*>(o.dout) + (long)b * o.ob + (long)h * o.oh : nullptr;

  Column<T, 1> dc;
  if (gp) dc.fetch(gp + min(dv, a.Dv - 1), o.ot, 0, max(len, 1), kq);
  load_rows<T, DKT, C, 4>(K, s.rk, kp, a.kt, a.Dk, 0, len, a.veck, a.normalize, a.eps);
  load_rows<T, DKT, C, 4>(Q, s.rq, qp, a.qt, a.Dk, 0, len, a.vecq, a.normalize, a.eps);
  if (wave == 0) chunk_gates<C>(a, s, b, h, 0, len, lane);
  f4 S[DKT];  // the gradient of the state
#pragma unroll
  for (int m = 0; m < DKT; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * m + 4 * kq + r;
      S[m][r] = (o.dlast && d < a.Dk && dv < a.Dv) ? o.dlast[((long)bh * a.Dk + d) * a.Dv + dv] : 0.f;
      o.dSc[((long)bh * DKp + d) * Dvp + dv] = S[m][r];
    }
  lds_barrier();
  const f4 dy = dc.get(0, 0, len, kq, gp && dv < a.Dv);
  pair_tiles<DKT>(K, Q, A, P, s, a.scale, wave, nw);
  f4 u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < DKT; ++m) u = mm16(row4(K + l16 * LD + 16 * m + 4 * kq), S[m], u);
  lds_barrier();
  if (wave == 0) diag_inverse(A, Td);
  lds_barrier();
  const f4 be = row4(s.beta + 4 * kq), ga = row4(s.gam + 4 * kq);
  u = mm16(col4(P + 4 * kq * LT + l16, LT), dy, u * row4(s.e + 4 * kq));
  u = mm16(col4(Td + 4 * kq * LT + l16, LT), u, f4{0.f, 0.f, 0.f, 0.f});
  T* vp = reinterpret_cast<T*>(o.dv) + (long)bh * a.Dv + dv;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int t = 4 * kq + r;
    o.dR[((long)bh * C + t) * Dvp + dv] = u[r];
    if (t < a.T && dv < a.Dv) st1(vp + (long)t * BH * a.Dv, t < len ? be[r] * u[r] : 0.f);
  }
  if (!o.dstate) return;
  const float gc = s.gam[C - 1];
  const f4 w = dy * (a.scale * ga), z = -(u * ga * be);
#pragma unroll
  for (int m = 0; m < DKT; ++m) {
    S[m] = mm16(col4(Q + 4 * kq * LD + 16 * m + l16, LD), w, S[m] * gc);
    S[m] = mm16(col4(K + 4 * kq * LD + 16 * m + l16, LD), z, S[m]);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * m + 4 * kq + r;
      if (d < a.Dk && dv < a.Dv) o.dstate[((long)bh * a.Dk + d) * a.Dv + dv] = S[m][r];
    }
  }
}

template <typename T, int DKT, int NWT, bool MAP>
__global__ void __launch_bounds__(64 * NWT) delta_bwd_walk_kernel(Args a, BwdArgs o) {
  using St = Stage<T, DKT, NWT, 2>;
  constexpr bool SP = St::SP;
  constexpr int C = 64, NT = 4, DKp = 16 * DKT, Dvp = NWT == 4 ? 64 : 128;
  extern __shared__ __align__(16) unsigned char lds[];
  St st(lds);

  const int lane = threadIdx.x & 63, l16 = lane & 15, kq = lane >> 4, wave = wave_id();
  const int BH = a.B * a.Hv, bh = blockIdx.x % BH, seg = blockIdx.x / BH;
  const int b = bh / a.Hv, h = bh % a.Hv, hk = h / (a.Hv / a.Hk);
  const int nvs = (a.Dv + 15) >> 4, dv = 16 * wave + l16;
  const bool works = wave < nvs;
  const int len = a.lengths ? max(0, min(a.T, a.lengths[b])) : a.T;
  const T* qp = reinterpret_cast<const T*>(a.q) + (long)b * a.qb + (long)hk * a.qh;
  const T* kp = reinterpret_cast<const T*>(a.k) + (long)b * a.kb + (long)hk * a.kh;
  const T* gp = o.dout ? reinterpret_cast<const T*>(o.dout) + (long)b * o.ob + (long)h * o.oh : nullptr;
  const float* pairs = o.pairs + (long)bh * a.N * PAIR_FLOATS;

  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  f4 S[DKT];          // the gradient of the state
  Column<T, NT> dn;   // the next chunk's of the outputs
  const T* gcol = gp + min(dv, a.Dv - 1);
#pragma unroll
  for (int m = 0; m < DKT; ++m) S[m] = zero;
  if (!MAP && works) {
    if (a.nseg > 1) {
      const float* p = o.dSseg + ((((long)bh * a.nseg + seg) * nvs + wave) * DKT * 64 + lane) * 4;
#pragma unroll
      for (int m = 0; m < DKT; ++m) S[m] = row4(p + m * 256);
    } else if (o.dlast) {
#pragma unroll
      for (int m = 0; m < DKT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int d = 16 * m + 4 * kq + r;
          if (d < a.Dk && dv < a.Dv) S[m][r] = o.dlast[((long)bh * a.Dk + d) * a.Dv + dv];
        }
    }
  }
  const int n0 = seg * a.cps, n1 = min(a.N, n0 + a.cps), live = min(n1, (len + C - 1) / C);
  if (n0 < live) {
    st.fetch(a, qp, kp, pairs + (long)(live - 1) * PAIR_FLOATS, (live - 1) * C, len);
    if (gp) dn.fetch(gcol, o.ot, (live - 1) * C, len, kq);
  }
  for (int n = live - 1; n >= n0; --n) {
    const int t0 = n * C;
    if (!MAP && works) {
      float* p = o.dSc + ((long)bh * a.N + n) * DKp * Dvp + 4 * kq * Dvp + dv;
#pragma unroll
      for (int m = 0; m < DKT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[(16 * m + r) * Dvp] = S[m][r];
    }
    lds_barrier();
    st.turn();
    st.commit(t0, len, a.Dk);
    lds_barrier();
    f4 dy[NT], u[NT];
#pragma unroll
    for (int ti = 0; ti < NT; ++ti) dy[ti] = dn.get(ti, t0, len, kq, gp && dv < a.Dv), u[ti] = zero;
    // the next chunk on its way, a part at a time: see Stage
    auto ahead = [&](auto part) {
      if (n > n0) st.fetch(part, a, qp, kp, pairs + (long)(n - 1) * PAIR_FLOATS, t0 - C, len);
    };
    if (!works) {
      each<0, 3>(ahead);
      continue;
    }
    if (n > n0 && gp) dn.fetch(gcol, o.ot, t0 - C, len, kq);
    part_ends();
    each<0, DKT / 2>([&](auto M) {
      constexpr int m2 = M;
      const Op16<SP> s0 = cut<SP>(S[2 * m2]), s1 = cut<SP>(S[2 * m2 + 1]);
#pragma unroll
      for (int ti = 0; ti < NT; ++ti) u[ti] = mm32(st.k(ti, m2), s0, s1, u[ti]);
      part_ends();
      if constexpr (m2 < 2) ahead(M);
    });
    if constexpr (DKT == 2) ahead(std::integral_constant<int, 1>{});
    part_ends();
    // dR: backward substitution by blocks of 16 steps
    Op16<SP> ub[NT], db[NT];
    each<0, NT>([&](auto I) {
      constexpr int ti = NT - 1 - I;
      db[ti] = cut<SP>(dy[ti]);
      f4 r = u[ti] * st.e(ti) * st.rk4(ti);
      r = mm_tiles<ti, NT>([&](int x) { return st.P(x, ti); }, [&](auto x) { return db[decltype(x)::value]; }, r);
      r = mm_tiles<ti + 1, NT>([&](int x) { return st.A(x, ti); }, [&](auto x) { return ub[decltype(x)::value]; }, r);
      u[ti] = mm16o(st.Ti(ti), cut<SP>(r), zero);
      ub[ti] = cut<SP>(u[ti]);
      if constexpr (ti == NT - 1) ahead(std::integral_constant<int, 2>{});
    });
    if (!MAP) {
      const long vstep = afresh((long)BH * a.Dv);
      float* p = o.dR + ((long)bh * a.N + n) * C * Dvp + 4 * kq * Dvp + dv;
      T* vp = reinterpret_cast<T*>(o.dv) + (long)bh * a.Dv + dv + (t0 + 4 * kq) * vstep;
#pragma unroll
      for (int ti = 0; ti < NT; ++ti) {
        const f4 g = u[ti] * st.beta(ti);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int t = t0 + 16 * ti + 4 * kq + r;
          p[(16 * ti + r) * Dvp] = u[ti][r];
          if (t < a.T && dv < a.Dv) st1(vp + (16 * ti + r) * vstep, t < len ? g[r] : 0.f);
        }
      }
    }
    part_ends();
    const float gc = st.gam_last();
#pragma unroll
    for (int m = 0; m < DKT; ++m) S[m] *= gc;
#pragma unroll
    for (int t2 = 0; t2 < NT / 2; ++t2) {
      Op16<SP> w[2], z[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int ti = 2 * t2 + x;
        const f4 ga = st.gam(ti);
        w[x] = cut<SP>(dy[ti] * (a.scale * ga * st.rq4(ti)));
        z[x] = cut<SP>(-(u[ti] * ga * st.beta(ti) * st.rk4(ti)));
      }
#pragma unroll
      for (int m = 0; m < DKT; ++m) {
        S[m] = mm32(st.qt(m, t2), w[0], w[1], S[m]);
        S[m] = mm32(st.kt(m, t2), z[0], z[1], S[m]);
      }
    }
  }
  if (!works) return;
  if (MAP) {
    float* p = o.Xseg + ((((long)bh * a.nseg + seg) * nvs + wave) * DKT * 64 + lane) * 4;
#pragma unroll
    for (int m = 0; m < DKT; ++m) *reinterpret_cast<f4*>(p + m * 256) = S[m];
    return;
  }
  if (dv >= a.Dv) return;
  T* vp = reinterpret_cast<T*>(o.dv) + (long)bh * a.Dv + dv;  // behind the sequence's end: zeros
  for (int t = max(n0, live) * C + kq; t < min(a.T, n1 * C); t += 4) st1(vp + (long)t * BH * a.Dv, 0.f);
  if (seg == 0 && o.dstate) {
#pragma unroll
    for (int m = 0; m < DKT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * m + 4 * kq + r;
        if (d < a.Dk) o.dstate[((long)bh * a.Dk + d) * a.Dv + dv] = S[m][r];
      }
  }
}

constexpr int DVB = 32;  // value columns staged at once

// One wave, lane i the chunk's step i: the sum of dG over the steps from i to the end of its segment, as suffix sums less
// that of the next segment's first step.
template <int C>
__device__ __forceinline__ float segment_suffix(const Gates<C>& s, double dG, int i) {
  double suf = dG;
#pragma unroll
  for (int x = 1; x < C; x <<= 1) {
    const double y = __shfl_down(suf, x, 64);
    if (i + x < C) suf += y;
  }
  const unsigned long long starts = __ballot(i < C && i > 0 && s.seg[i < C ? i : 0] != s.seg[i > 0 && i < C ? i - 1 : 0]);
  const unsigned long long later = i < 63 ? starts >> (i + 1) : 0ull;
  const int nx = later ? i + __ffsll((long long)later) : i;
  const double beyond = __shfl(suf, nx, 64);
  return (float)(suf - (later ? beyond : 0.0));
}

// A chunk of 16 (a whole sequence): what sums over the value columns, one wave per 16 key columns.
template <int DKT>
struct PairLds {
  static constexpr int LD = 16 * DKT + 4, LV = DVB + 4, stage = 3 * 16 * LV, w = 2 * 16 * LT, big = stage > w ? stage : w;
  float K[16 * LD], Q[16 * LD], big_[big];
  Gates<16> s;
  float rows[2][16], cols[2][16], rowb[16], dots[5][DKT][16], dRv[16], sd[DKT];
};

template <typename T, int DKT>
__global__ void __launch_bounds__(64 * DKT) delta_bwd_pair_kernel(Args a, BwdArgs o, int per_value_head) {
  using L = PairLds<DKT>;
  constexpr int C = 16, LD = L::LD, LV = L::LV, DKp = 16 * DKT, NW = DKT;
  constexpr int RPT = (C * (DVB / 4) + 64 * NW - 1) / (64 * NW);
  extern __shared__ __align__(16) unsigned char lds[];
  L& l = *reinterpret_cast<L*>(lds);
  Gates<C>& s = l.s;
  float *sO = l.big_, *sR = sO + C * LV, *sU = sR + C * LV, *W1 = l.big_, *W2 = W1 + C * LT;

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, kq = lane >> 4, wave = wave_id();
  const int BH = a.B * a.Hv, bh = blockIdx.x;
  const int b = bh / a.Hv, h = bh % a.Hv, hk = h / (a.Hv / a.Hk);
  const int Dvp = pitch(a.Dv), Dve = 16 * ((a.Dv + 15) >> 4);
  const int len = a.lengths ? max(0, min(a.T, a.lengths[b])) : a.T;
  const int Ho = per_value_head ? a.Hv : a.Hk, ho = per_value_head ? h : hk;
  const bool same = per_value_head == 0;  // the outputs have the inputs' type

  auto put = [&](void* base, int t, int d, float v) {
    const long at = (((long)t * a.B + b) * Ho + ho) * a.Dk + d;
    if (same) st1(reinterpret_cast<T*>(base) + at, v);
    else reinterpret_cast<float*>(base)[at] = v;
  };

  if (len == 0) {
    for (int x = tid; x < a.T * a.Dk; x += 64 * NW) {
      put(o.dq, x / a.Dk, x % a.Dk, 0.f);
      put(o.dk, x / a.Dk, x % a.Dk, 0.f);
    }
    if (tid < a.T) {
      o.dg[(long)tid * BH + bh] = 0.f;
      o.db[(long)tid * BH + bh] = 0.f;
    }
    return;
  }

  constexpr int RL = C * 16 / (64 * NW) > 0 ? C * 16 / (64 * NW) : 1;
  load_rows<T, DKT, C, RL>(l.K, s.rk, reinterpret_cast<const T*>(a.k) + (long)b * a.kb + (long)hk * a.kh, a.kt, a.Dk, 0, len, a.veck,
                       a.normalize, a.eps);
  load_rows<T, DKT, C, RL>(l.Q, s.rq, reinterpret_cast<const T*>(a.q) + (long)b * a.qb + (long)hk * a.qh, a.qt, a.Dk, 0, len, a.vecq,
                       a.normalize, a.eps);
  if (wave == 0) chunk_gates<C>(a, s, b, h, 0, len, lane);

  const T* vp = reinterpret_cast<const T*>(a.v) + (long)b * a.vb + (long)h * a.vh;
  const T* gp = o.dout ? reinterpret_cast<const T*>(o.dout) + (long)b * o.ob + (long)h * o.oh : nullptr;
  const float* up = o.U + (long)bh * C * Dvp;
  const float* rp = o.dR + (long)bh * C * Dvp;
  const float* s0 = o.Sc + ((long)bh * DKp + 16 * wave + l16) * Dvp;
  const float* ds = o.dSc + ((long)bh * DKp + 16 * wave + l16) * Dvp;

  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  f4 GO = zero, GR = zero, GU = zero, D = zero;
  float dRv[RPT], sdot = 0.f;
#pragma unroll
  for (int x = 0; x < RPT; ++x) dRv[x] = 0.f;

  for (int c0 = 0; c0 < Dve; c0 += DVB) {
#pragma unroll
    for (int x = 0; x < RPT; ++x) {
      const int at = tid + x * 64 * NW, i = at / (DVB / 4), c = c0 + 4 * (at % (DVB / 4));
      if (i < C) {
        f4 g = zero, r = zero, u = zero;
        if (c < Dve) {
          r = row4(rp + i * Dvp + c);
          u = row4(up + i * Dvp + c);
          if (i < len) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (c + j < a.Dv) {
                if (gp) g[j] = ld1(gp + (long)i * o.ot + c + j);
                dRv[x] = fmaf(r[j], ld1(vp + (long)i * a.vt + c + j), dRv[x]);
              }
          }
        }
        const int w = i * LV + c - c0;
        *reinterpret_cast<f4*>(sO + w) = g;
        *reinterpret_cast<f4*>(sR + w) = r;
        *reinterpret_cast<f4*>(sU + w) = u;
      }
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < DVB / 16; ++m) {
      const int c = c0 + 16 * m;
      if (c < Dve) {
        const f4 x = row4(s0 + c + 4 * kq), y = row4(ds + c + 4 * kq);
#pragma unroll
        for (int j = 0; j < 4; ++j) sdot = fmaf(x[j], y[j], sdot);
        const int w = l16 * LV + 16 * m + 4 * kq;
        GO = mm16(x, row4(sO + w), GO);
        GR = mm16(x, row4(sR + w), GR);
        GU = mm16(y, row4(sU + w), GU);
        if (wave < 2) D = mm16(row4(sU + w), row4((wave == 0 ? sO : sR) + w), D);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int x = 0; x < RPT; ++x) {
    const int i = (tid + x * 64 * NW) / (DVB / 4);
    const float v = seg_sum(dRv[x], DVB / 4);
    if (i < C && (tid & (DVB / 4 - 1)) == 0) l.dRv[i] = v;
  }
  sdot = wave_sum(sdot);
  if (lane == 0) l.sd[wave] = sdot;

  // W1 (wave 0) and W2 (wave 1), over the staging area, and the row and column sums of what the decays see of them
  if (wave < 2) {
    const bool first = wave == 0;
    const float* kj = l.K + l16 * LD + 4 * kq;
    const float* xi = (first ? l.Q : l.K) + l16 * LD + 4 * kq;
    f4 d = zero;
#pragma unroll
    for (int m = 0; m < DKT; ++m) d = mm16(row4(kj + 16 * m), row4(xi + 16 * m), d);
    const int i = l16, j0 = 4 * kq;
    const double Gi = s.G[i];
    const int segi = s.seg[i];
    const float be = s.beta[i];
    f4 w;
    float rs = 0.f, rb = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float m = pair_decay<C>(s, i, j0 + r, Gi, segi);
      float e;
      if (first) {
        w[r] = m * D[r];
        e = a.scale * w[r] * d[r];
      } else {
        const float z = j0 + r < i ? -m * D[r] : 0.f;
        w[r] = be * z;
        rb = fmaf(z, d[r], rb);
        e = w[r] * d[r];
      }
      rs += e;
      const float cs = row16_sum(e);
      if (l16 == 0) l.cols[wave][4 * kq + r] = cs;
    }
    *reinterpret_cast<f4*>((first ? W1 : W2) + i * LT + j0) = w;
    rs += __shfl_xor(rs, 16, 64);
    rs += __shfl_xor(rs, 32, 64);
    rb += __shfl_xor(rb, 16, 64);
    rb += __shfl_xor(rb, 32, 64);
    if (kq == 0) {
      l.rows[wave][l16] = rs;
      if (!first) l.rowb[l16] = rb;
    }
  }
  __syncthreads();

  // this wave's 16 key columns of dQ^T and dK^T
  const int kc = 16 * wave, i = l16;
  const f4 q = row4(l.Q + i * LD + kc + 4 * kq), k = row4(l.K + i * LD + kc + 4 * kq);
  float dd[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    dd[0] = fmaf(q[r], GO[r], dd[0]);
    dd[1] = fmaf(k[r], GR[r], dd[1]);
    dd[2] = fmaf(k[r], GU[r], dd[2]);
  }
  const float ga = s.gam[i], be = s.beta[i], e = s.e[i];
  const f4 kcol = col4(l.K + 4 * kq * LD + kc + l16, LD), qcol = col4(l.Q + 4 * kq * LD + kc + l16, LD);
  f4 dQ = mm16(kcol, row4(W1 + i * LT + 4 * kq), ga * GO);
  f4 w = mm16(kcol, row4(W2 + i * LT + 4 * kq), zero);
  const f4 z = mm16(qcol, col4(W1 + 4 * kq * LT + i, LT), zero);
  w = mm16(kcol, col4(W2 + 4 * kq * LT + i, LT), w);
  dQ *= a.scale;
  f4 dK = w + a.scale * z - (be * ga) * GR + e * GU;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    dd[3] = fmaf(q[r], dQ[r], dd[3]);
    dd[4] = fmaf(k[r], dK[r], dd[4]);
  }
#pragma unroll
  for (int x = 0; x < 5; ++x) {
    dd[x] += __shfl_xor(dd[x], 16, 64);
    dd[x] += __shfl_xor(dd[x], 32, 64);
    if (kq == 0) l.dots[x][wave][i] = dd[x];
  }
  __syncthreads();
  if (a.normalize) {
    float dq = 0.f, dk = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      dq += l.dots[3][x][i];
      dk += l.dots[4][x][i];
    }
    dQ = s.rq[i] * (dQ - dq * q);
    dK = s.rk[i] * (dK - dk * k);
  }
  if (i < a.T) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = kc + 4 * kq + r;
      if (d < a.Dk) {
        put(o.dq, i, d, i < len ? dQ[r] : 0.f);
        put(o.dk, i, d, i < len ? dK[r] : 0.f);
      }
    }
  }
  if (wave == 0) {
    double dG = 0.0;
    float F = 0.f, db = 0.f;
    if (lane < C) {
      float go = 0.f, gr = 0.f, gu = 0.f;
#pragma unroll
      for (int x = 0; x < NW; ++x) {
        go += l.dots[0][x][i];
        gr += l.dots[1][x][i];
        gu += l.dots[2][x][i];
      }
      F = e * gu;
      db = l.dRv[i] - ga * gr;
      dG = (double)(a.scale * ga * go) - (double)(be * ga * gr) - (double)F;
      dG += (double)l.rows[0][i];
      dG -= (double)l.cols[0][i];
      dG += (double)l.rows[1][i];
      db += l.rowb[i];
      dG -= (double)l.cols[1][i];
    }
    const float sumF = wave_sum(F);
    if (lane == C - 1) {
      float sd = 0.f;
#pragma unroll
      for (int x = 0; x < NW; ++x) sd += l.sd[x];
      dG += (double)(sumF + ga * sd);
    }
    const float g = segment_suffix<C>(s, dG, lane);
    if (lane < a.T) {
      o.dg[(long)lane * BH + bh] = s.rst[lane] ? 0.f : g;
      o.db[(long)lane * BH + bh] = lane < len ? db : 0.f;
    }
  }
}

// Value columns of U, dR and dO on their way to LDS, DVB at a time: [64][DVB], for operands over all of them at once.
template <typename T, int TH>
struct Values;

template <int TH>
struct Values<float, TH> {
  static constexpr int LV = DVB + 4, BYTES = 3 * 64 * LV * 4;
  float *O, *R, *U;
  __device__ __forceinline__ explicit Values(void* lds) : O((float*)lds), R(O + 64 * LV), U(R + 64 * LV) {}
  __device__ __forceinline__ void put(int i, int c, f4 g, f4 r, f4 u) {
    *reinterpret_cast<f4*>(O + i * LV + c) = g;
    *reinterpret_cast<f4*>(R + i * LV + c) = r;
    *reinterpret_cast<f4*>(U + i * LV + c) = u;
  }
  struct Cut {
    Op16<false> a, b;
  };
  static __device__ __forceinline__ Cut at(const float* M, int t, int l16, int kq) {
    const float* p = M + (16 * t + l16) * LV + 4 * kq;
    return {{row4(p)}, {row4(p + 16)}};
  }
  __device__ __forceinline__ Cut r(int t, int l16, int kq) const { return at(R, t, l16, kq); }
  __device__ __forceinline__ Cut u(int t, int l16, int kq) const { return at(U, t, l16, kq); }
  __device__ __forceinline__ Exact32<false> o(int t, int l16, int kq) const {
    const float* p = O + (16 * t + l16) * LV + 4 * kq;
    return {row4(p), row4(p + 16)};
  }
};

template <int TH>
struct Values<bf16, TH> {
  static constexpr int LV = DVB + 8, PL = 64 * LV, BYTES = 7 * PL * 2;
  uint16_t *O, *R, *U;  // R and U in three parts
  __device__ __forceinline__ explicit Values(void* lds) : O((uint16_t*)lds), R(O + PL), U(R + 3 * PL) {}
  __device__ __forceinline__ void put(int i, int c, f4 g, f4 r, f4 u) {
    const int w = i * LV + place(c);
    *reinterpret_cast<u2*>(O + w) = part(g);
    const Op16<true> x = cut3(r), y = cut3(u);
    *reinterpret_cast<u2*>(R + w) = x.p0;
    *reinterpret_cast<u2*>(R + PL + w) = x.p1;
    *reinterpret_cast<u2*>(R + 2 * PL + w) = x.p2;
    *reinterpret_cast<u2*>(U + w) = y.p0;
    *reinterpret_cast<u2*>(U + PL + w) = y.p1;
    *reinterpret_cast<u2*>(U + 2 * PL + w) = y.p2;
  }
  struct Cut {
    Op16<true> a, b;
  };
  static __device__ __forceinline__ Cut at(const uint16_t* M, int t, int l16, int kq) {
    const uint16_t* p = M + (16 * t + l16) * LV + 8 * kq;
    const u4 x = *reinterpret_cast<const u4*>(p), y = *reinterpret_cast<const u4*>(p + PL), z = *reinterpret_cast<const u4*>(p + 2 * PL);
    return {{x.xy, y.xy, z.xy}, {x.zw, y.zw, z.zw}};
  }
  __device__ __forceinline__ Cut r(int t, int l16, int kq) const { return at(R, t, l16, kq); }
  __device__ __forceinline__ Cut u(int t, int l16, int kq) const { return at(U, t, l16, kq); }
  __device__ __forceinline__ Exact32<true> o(int t, int l16, int kq) const {
    return {*reinterpret_cast<const u4*>(O + (16 * t + l16) * LV + 8 * kq)};
  }
};

// four neighbours of a row of D that is read in whole fours (vec) or by its elements
__device__ __forceinline__ f4 four(const float* p, int c, int D, bool vec) {
  if (vec) return row4(p + min(c, D - 4));
  return f4{p[min(c, D - 1)], p[min(c + 1, D - 1)], p[min(c + 2, D - 1)], p[min(c + 3, D - 1)]};
}
__device__ __forceinline__ f4 four(const bf16* p, int c, int D, bool vec) {
  if (vec) {
    const u2 w = *reinterpret_cast<const u2*>(p + min(c, D - 4));
    return f4{__builtin_bit_cast(float, w.x << 16), __builtin_bit_cast(float, w.x & 0xffff0000u), __builtin_bit_cast(float, w.y << 16),
              __builtin_bit_cast(float, w.y & 0xffff0000u)};
  }
  return f4{ld1(p + min(c, D - 1)), ld1(p + min(c + 1, D - 1)), ld1(p + min(c + 2, D - 1)), ld1(p + min(c + 3, D - 1))};
}

// PRE: W1, W1^T and W2 + W2^T wait in LDS as the operands that all waves read, cut once, not by each of eight waves (half of
// the vector instructions of the kernel); narrower heads keep the LDS for a second workgroup on the CU.
template <typename T, int DKT>
struct GradsLds {
  static constexpr bool PRE = Stage<T, DKT, DKT, 3>::SP && DKT == 8;
  static constexpr int NTL = 10, W = 2 * NTL * TS * 4, V = Values<T, 64 * DKT>::BYTES, P = W + (PRE ? 36 * 1536 : 0), BIG = P > V ? P : V;
  Gates<64> s;
  float rows[NTL][16], cols[NTL][16], rowb[NTL][16], dots[5][DKT][64], dRv[64], sd[DKT];
  __align__(16) unsigned char big[BIG], stage[Stage<T, DKT, DKT, 3>::BYTES];
};

// Chunks of 64: what sums over the value columns (the head of this file), one wave per 16 key columns.  ONE: a value head a
// workgroup, and delta_head_sum_kernel adds those that share a key head.  Else a workgroup takes the G value heads of a key
// head one after the other and leaves the sum of their dq and dk, which is for heads wider than 64 alone, of which a CU holds
// one workgroup in any case: of narrower ones it holds two, and 1024 steps x 32 x 8 heads of 64 took 281 us so and 363 us in
// turn.
template <typename T, int DKT, bool ONE>
__global__ void __launch_bounds__(64 * DKT, ONE && DKT > 2 ? 2 : 1) delta_grads_kernel(Args a, BwdArgs o, int G_) {
  const int G = ONE ? 1 : G_;
  using L = GradsLds<T, DKT>;
  using St = Stage<T, DKT, DKT, 3>;
  constexpr bool SP = St::SP;
  constexpr int C = 64, NT = 4, NTL = 10, DKp = 16 * DKT, NW = DKT, TH = 64 * NW;
  constexpr int TPW = (NTL + NW - 1) / NW, RPT = C * (DVB / 4) / TH;
  extern __shared__ __align__(16) unsigned char lds[];
  L& l = *reinterpret_cast<L*>(lds);
  Gates<C>& s = l.s;
  St st(l.stage);
  Values<T, TH> val(l.big);
  float *W1 = reinterpret_cast<float*>(l.big), *W2 = W1 + NTL * TS;
  u2* ops = reinterpret_cast<u2*>(W2 + NTL * TS);  // PRE: [36][part][lane]: 10 of W1, 10 of W1^T, 16 of W2 + W2^T

  int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, kq = lane >> 4;
  const int wave = wave_id();
  // the lane's place afresh in each turn over the heads: see afresh()
  auto turn = [&]() {
    st.turn();
    tid = st.tid, lane = tid & 63, l16 = st.l16, kq = st.kq;
  };
  const int BH = a.B * a.Hv, rep = a.Hv / a.Hk, BG = BH / G, bg = blockIdx.x % BG, n = blockIdx.x / BG, t0 = n * C;
  const int b = bg / (a.Hv / G), h0 = (bg % (a.Hv / G)) * G, hk = h0 / rep;
  const int Dvp = pitch(a.Dv), Dve = 16 * ((a.Dv + 15) >> 4);
  const int len = a.lengths ? max(0, min(a.T, a.lengths[b])) : a.T;
  const bool same = G == rep;  // dq and dk are whole: in the inputs' type, else fp32 for each value head
  const int Ho = same ? a.Hk : a.Hv, ho = same ? hk : h0;

  auto put = [&](void* base, int i, int d, f4 v) {
    const long at = (((long)(t0 + i) * a.B + b) * Ho + ho) * a.Dk + d;
    if (a.Dk % 4 == 0) {
      if (!same || sizeof(T) == 4) *reinterpret_cast<f4*>(reinterpret_cast<float*>(base) + at) = v;
      else *reinterpret_cast<u2*>(reinterpret_cast<T*>(base) + at) = part(v);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (d + r >= a.Dk) break;
        if (same) st1(reinterpret_cast<T*>(base) + at + r, v[r]);
        else reinterpret_cast<float*>(base)[at + r] = v[r];
      }
    }
  };
  const f4 zero = {0.f, 0.f, 0.f, 0.f};

  if (t0 >= len) {
    const int m = min(C, a.T - t0), q4 = (a.Dk + 3) / 4;
    for (int x = tid; x < m * q4; x += TH) {
      put(o.dq, x / q4, 4 * (x % q4), zero);
      put(o.dk, x / q4, 4 * (x % q4), zero);
    }
    for (int x = tid; x < m * G; x += TH) {
      const long at = (long)(t0 + x / G) * BH + b * a.Hv + h0 + x % G;
      o.dg[at] = 0.f;
      o.db[at] = 0.f;
    }
    return;
  }

  const T* vp = reinterpret_cast<const T*>(a.v) + (long)b * a.vb;
  const T* gp = o.dout ? reinterpret_cast<const T*>(o.dout) + (long)b * o.ob : vp;  // without dO: read and left out
  const long gt = o.dout ? o.ot : a.vt, gh = o.dout ? o.oh : a.vh;
  const long c_at = (long)b * a.Hv * a.N + n;  // the chunk of head h: c_at + h N

  // the next DVB value columns on their way, in four parts: issued all at once the reads of all waves queue up, and the waves
  // with them, for as long as the products of a step take; between the products they cost a fraction of that
  f4 g_[RPT], r_[RPT], u_[RPT], v_[RPT], x_[2], y_[2];
  auto fetch = [&](auto part, int h, int c0) {
    constexpr int P = decltype(part)::value;
    const long ch = c_at + (long)h * a.N;
    if constexpr (P < 3) {
#pragma unroll
      for (int x = 0; x < RPT; ++x) {
        const int at = tid + x * TH, i = at / (DVB / 4), c = c0 + 4 * (at % (DVB / 4)), ce = min(c, Dve - 4);
        const int t = min(t0 + i, len - 1);
        if constexpr (P == 0) r_[x] = row4(o.dR + ch * C * Dvp + i * Dvp + ce);
        if constexpr (P == 1) u_[x] = row4(o.U + ch * C * Dvp + i * Dvp + ce);
        if constexpr (P == 2) {
          g_[x] = four(gp + t * gt + h * gh, c, a.Dv, o.vecg);
          v_[x] = four(vp + t * a.vt + h * a.vh, c, a.Dv, o.vecv);
        }
      }
    } else {
      const float* s0 = o.Sc + (ch * DKp + 16 * wave + l16) * Dvp + 4 * kq;
      const float* ds = o.dSc + (ch * DKp + 16 * wave + l16) * Dvp + 4 * kq;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int c = min(c0 + 16 * m, Dve - 16);
        x_[m] = row4(s0 + c);
        y_[m] = row4(ds + c);
      }
    }
  };

  st.fetch(a, reinterpret_cast<const T*>(a.q) + (long)b * a.qb + (long)hk * a.qh, reinterpret_cast<const T*>(a.k) + (long)b * a.kb + (long)hk * a.kh,
           o.pairs + (c_at + (long)h0 * a.N) * PAIR_FLOATS, t0, len);
  each<0, 4>([&](auto part) { fetch(part, h0, 0); });
  f4 dQ[NT], dK[NT];
#pragma unroll
  for (int ti = 0; ti < NT; ++ti) dQ[ti] = dK[ti] = zero;
  st.commit(t0, len, a.Dk);

  const int kc = 16 * wave;  // this wave's key columns
  int h = h0;
  do {
  const long bh = (long)b * a.Hv + h;
  const float* pair = o.pairs + (c_at + (long)h * a.N) * PAIR_FLOATS;
  if (h > h0) lds_barrier();  // the head before is done with LDS
  turn();
  if (wave == NW - 1) chunk_gates<C>(a, s, b, h, t0, len, lane);
  f4 GO[NT], GR[NT], GU[NT], D1[TPW], D2[TPW], pw[TPW];
  float dRv[RPT], sdot = 0.f;
#pragma unroll
  for (int ti = 0; ti < NT; ++ti) GO[ti] = GR[ti] = GU[ti] = zero;
#pragma unroll
  for (int x = 0; x < TPW; ++x) {
    D1[x] = D2[x] = zero;
    pw[x] = row4(pair + (PAIR_P + min(wave + x * NW, NTL - 1)) * 256 + l16 * 16 + 4 * kq);
  }
#pragma unroll
  for (int x = 0; x < RPT; ++x) dRv[x] = 0.f;

  for (int c0 = 0; c0 < Dve; c0 += DVB) {
    if (c0) lds_barrier();  // the columns before are done with LDS
#pragma unroll
    for (int x = 0; x < RPT; ++x) {
      const int at = tid + x * TH, i = at / (DVB / 4), c = c0 + 4 * (at % (DVB / 4));
      const bool live = t0 + i < len;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = c + j < a.Dv;
        r_[x][j] = in ? r_[x][j] : 0.f;
        u_[x][j] = in ? u_[x][j] : 0.f;
        g_[x][j] = in && live && o.dout ? g_[x][j] : 0.f;
        dRv[x] = fmaf(r_[x][j], in && live ? v_[x][j] : 0.f, dRv[x]);
      }
      val.put(i, c - c0, g_[x], r_[x], u_[x]);
    }
    const f4 x0 = x_[0], x1 = c0 + 16 < Dve ? x_[1] : zero, y0 = y_[0], y1 = c0 + 16 < Dve ? y_[1] : zero;
    lds_barrier();
    const bool on = c0 + DVB < Dve, more = on || (!ONE && h + 1 < h0 + G);
    const int hn = on ? h : h + 1, cn = on ? c0 + DVB : 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) sdot = fmaf(x0[j], y0[j], fmaf(x1[j], y1[j], sdot));
    part_ends();
    const Op16<SP> a0 = cut<SP>(x0), a1 = cut<SP>(x1), b0 = cut<SP>(y0), b1 = cut<SP>(y1);
    each<0, NT>([&](auto ti) {
      if (more) fetch(ti, hn, cn);
      GO[ti] = mm32r(a0, a1, val.o(ti, l16, kq), GO[ti]);
      const auto r = val.r(ti, l16, kq);
      GR[ti] = mm32(a0, a1, r.a, r.b, GR[ti]);
      const auto u = val.u(ti, l16, kq);
      GU[ti] = mm32(b0, b1, u.a, u.b, GU[ti]);
      part_ends();
    });
#pragma unroll
    for (int x = 0; x < TPW; ++x) {
      const int t = wave + x * NW;
      if (t < NTL) {
        int ti, tj;
        lower_tile(t, ti, tj);
        const auto u = val.u(tj, l16, kq);
        D1[x] = mm32r(u.a, u.b, val.o(ti, l16, kq), D1[x]);
        const auto r = val.r(ti, l16, kq);
        D2[x] = mm32(u.a, u.b, r.a, r.b, D2[x]);
      }
    }
  }
#pragma unroll
  for (int x = 0; x < RPT; ++x) {
    const float v = seg_sum(dRv[x], DVB / 4);
    if ((tid & (DVB / 4 - 1)) == 0) l.dRv[(tid + x * TH) / (DVB / 4)] = v;
  }
  sdot = wave_sum(sdot);
  if (lane == 0) l.sd[wave] = sdot;
  lds_barrier();  // the values are done with
  turn();
  part_ends();

  auto put_op = [&](int x, f4 v) {
    if constexpr (L::PRE) {
      const Op16<true> c = cut3(v);
      u2* p = ops + x * 192 + lane;
      p[0] = c.p0, p[64] = c.p1, p[128] = c.p2;
    }
  };
  auto get_op = [&](int x) -> Op16<SP> {
    if constexpr (L::PRE) {
      const u2* p = ops + x * 192 + lane;
      return {p[0], p[64], p[128]};
    } else {
      return {};
    }
  };
  // W1, W2 in their place, and the row and column sums of what the decays see of them
#pragma unroll
  for (int x = 0; x < TPW; ++x) {
    const int t = wave + x * NW;
    if (t < NTL) {
      int ti, tj;
      lower_tile(t, ti, tj);
      const int i = 16 * ti + l16, j0 = 16 * tj + 4 * kq;
      const f4 p = pw[x];
      f4 kk = zero;
#pragma unroll
      for (int m2 = 0; m2 < DKT / 2; ++m2) kk = mm32x(st.k(tj, m2), st.k(ti, m2), kk);
      if (SP) kk *= st.rk4(tj) * st.gates[256 + i];
      const double Gi = s.G[i];
      const int segi = s.seg[i];
      const float be = s.beta[i];
      f4 w1, w2;
      float rs = 0.f, rb = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float m = pair_decay<C>(s, i, j0 + r, Gi, segi);
        w1[r] = m * D1[x][r];
        const float z = j0 + r < i ? -m * D2[x][r] : 0.f;
        w2[r] = be * z;
        rb = fmaf(z, kk[r], rb);
        const float e = fmaf(D1[x][r], p[r], w2[r] * kk[r]);
        rs += e;
        const float cs = row16_sum(e);
        if (l16 == 0) l.cols[t][4 * kq + r] = cs;
      }
      if constexpr (L::PRE) put_op(t, w1 * st.rk4(tj));
      *reinterpret_cast<f4*>(W1 + t * TS + l16 * TL + 4 * kq) = w1;
      *reinterpret_cast<f4*>(W2 + t * TS + l16 * TL + 4 * kq) = w2;
      rs += __shfl_xor(rs, 16, 64);
      rs += __shfl_xor(rs, 32, 64);
      rb += __shfl_xor(rb, 16, 64);
      rb += __shfl_xor(rb, 32, 64);
      if (kq == 0) {
        l.rows[t][l16] = rs;
        l.rowb[t][l16] = rb;
      }
    }
  }
  lds_barrier();
  turn();
  part_ends();
  auto row_of = [&](const float* W, int ti, int tj) { return row4(W + (ti * (ti + 1) / 2 + tj) * TS + l16 * TL + 4 * kq); };
  auto col_of = [&](const float* W, int ti, int tj) { return col4(W + (ti * (ti + 1) / 2 + tj) * TS + 4 * kq * TL + l16, TL); };
  // operands against steps of tile tk: rows of W1 and of W2 + W2^T, and of W1^T
  auto w1_op = [&](int ti, int tk) -> Op16<SP> {
    if constexpr (L::PRE) return tk <= ti ? get_op(ti * (ti + 1) / 2 + tk) : cut<SP>(zero);
    else return cut<SP>(tk <= ti ? row_of(W1, ti, tk) * st.rk4(tk) : zero);
  };
  auto w1t_op = [&](int ti, int tk) -> Op16<SP> {
    if constexpr (L::PRE) return tk >= ti ? get_op(NTL + tk * (tk + 1) / 2 + ti) : cut<SP>(zero);
    else return cut<SP>(tk >= ti ? col_of(W1, tk, ti) * st.rq4(tk) : zero);
  };
  auto w2_sum = [&](int ti, int tk) {
    f4 w = zero;
    if (tk <= ti) w += row_of(W2, ti, tk);
    if (tk >= ti) w += col_of(W2, tk, ti);
    return w * st.rk4(tk);
  };
  auto w2_op = [&](int ti, int tk) -> Op16<SP> {
    if constexpr (L::PRE) return get_op(2 * NTL + NT * ti + tk);
    else return cut<SP>(w2_sum(ti, tk));
  };
  if constexpr (L::PRE) {
    const int w0 = (int)afresh(wave);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int t = w0 + x * NW;
      if (t < NT * NT) put_op(2 * NTL + t, w2_sum(t / NT, t % NT));
      else if (t < NT * NT + NTL) {
        int ti, tj;
        lower_tile(t - NT * NT, ti, tj);
        put_op(NTL + t - NT * NT, col_of(W1, ti, tj) * st.rq4(ti));
      }
    }
    lds_barrier();
    part_ends();
  }
  // this wave's key columns of dQ^T and dK^T
#pragma unroll
  for (int ti = 0; ti < NT; ++ti) {
    const int i = 16 * ti + l16;
    const float ga = s.gam[i], be = s.beta[i], e = s.e[i];
    const f4 q = st.q_of(i, kc + 4 * kq), k = st.k_of(i, kc + 4 * kq);
    float d0 = 0.f, d1 = 0.f, d2 = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      d0 = fmaf(q[r], GO[ti][r], d0);
      d1 = fmaf(k[r], GR[ti][r], d1);
      d2 = fmaf(k[r], GU[ti][r], d2);
    }
    part_ends();
    f4 x = ga * GO[ti], w = zero, z = zero;
#pragma unroll
    for (int t2 = 0; t2 < 2; ++t2) {
      const int ta = 2 * t2, tb = 2 * t2 + 1;
      const Exact32<SP> kt = st.kt(wave, t2);
      if (ta <= ti) x = mm32(kt, w1_op(ti, ta), w1_op(ti, tb), x);
      if (L::PRE) part_ends();
      if (tb >= ti) z = mm32(st.qt(wave, t2), w1t_op(ti, ta), w1t_op(ti, tb), z);
      if (L::PRE) part_ends();
      w = mm32(kt, w2_op(ti, ta), w2_op(ti, tb), w);
      if (L::PRE) part_ends();
    }
    dQ[ti] += a.scale * x;
    dK[ti] += w + a.scale * z - (be * ga) * GR[ti] + e * GU[ti];
    float dd[3] = {d0, d1, d2};
#pragma unroll
    for (int y = 0; y < 3; ++y) {
      dd[y] += __shfl_xor(dd[y], 16, 64);
      dd[y] += __shfl_xor(dd[y], 32, 64);
      if (kq == 0) l.dots[y][wave][i] = dd[y];
    }
  }
  lds_barrier();
  if (wave == 0) {
    const int i = lane;
    float go = 0.f, gr = 0.f, gu = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      go += l.dots[0][w][i];
      gr += l.dots[1][w][i];
      gu += l.dots[2][w][i];
    }
    const float ga = s.gam[i], be = s.beta[i], F = s.e[i] * gu;
    float db = l.dRv[i] - ga * gr;
    double dG = (double)(a.scale * ga * go) - (double)(be * ga * gr) - (double)F;
#pragma unroll
    for (int t = 0; t < NTL; ++t) {
      int ti, tj;
      lower_tile(t, ti, tj);
      if (ti == i >> 4) {
        dG += (double)l.rows[t][i & 15];
        db += l.rowb[t][i & 15];
      }
      if (tj == i >> 4) dG -= (double)l.cols[t][i & 15];
    }
    const float sumF = wave_sum(F);
    if (i == C - 1) {
      float sd = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) sd += l.sd[w];
      dG += (double)(sumF + ga * sd);
    }
    const float g = segment_suffix<C>(s, dG, i);
    if (t0 + i < a.T) {
      o.dg[(long)(t0 + i) * BH + bh] = s.rst[i] ? 0.f : g;
      o.db[(long)(t0 + i) * BH + bh] = t0 + i < len ? db : 0.f;
    }
  }
  } while (!ONE && ++h < h0 + G);

  turn();
  // through the scaling to unit length
  if (a.normalize) {
#pragma unroll
    for (int ti = 0; ti < NT; ++ti) {
      const int i = 16 * ti + l16;
      const f4 q = st.q_of(i, kc + 4 * kq), k = st.k_of(i, kc + 4 * kq);
      float dd[2] = {0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        dd[0] = fmaf(q[r], dQ[ti][r], dd[0]);
        dd[1] = fmaf(k[r], dK[ti][r], dd[1]);
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        dd[y] += __shfl_xor(dd[y], 16, 64);
        dd[y] += __shfl_xor(dd[y], 32, 64);
        if (kq == 0) l.dots[3 + y][wave][i] = dd[y];
      }
    }
  }
  lds_barrier();
#pragma unroll
  for (int ti = 0; ti < NT; ++ti) {
    const int i = 16 * ti + l16;
    if (a.normalize) {
      float dq = 0.f, dk = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        dq += l.dots[3][w][i];
        dk += l.dots[4][w][i];
      }
      dQ[ti] = st.gates[192 + i] * (dQ[ti] - dq * st.q_of(i, kc + 4 * kq));
      dK[ti] = st.gates[256 + i] * (dK[ti] - dk * st.k_of(i, kc + 4 * kq));
    }
    if (t0 + i < a.T && kc + 4 * kq < a.Dk) {
      const bool live = t0 + i < len;
      put(o.dq, i, kc + 4 * kq, live ? dQ[ti] : zero);
      put(o.dk, i, kc + 4 * kq, live ? dK[ti] : zero);
    }
  }
}

// Per-value-head dq and dk in fp32 -> the sums over the value heads that share a key head, rounded once.  Bound by memory: V
// neighbours a thread (4 where Dk allows).
template <typename T, int V>
__global__ void delta_head_sum_kernel(const float* xq, const float* xk, T* yq, T* yk, long n, int rep, int Dk) {
  const long i = ((long)blockIdx.x * blockDim.x + threadIdx.x) * V;
  if (i >= n) return;
  const float* x = blockIdx.y ? xk : xq;
  T* y = (blockIdx.y ? yk : yq) + i;
  const long row = i / Dk, d = i % Dk;
  x += row * rep * Dk + d;
  if constexpr (V == 4) {
    f4 v = {0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r < rep; ++r) v += row4(x + (long)r * Dk);
    if constexpr (sizeof(T) == 4) *reinterpret_cast<f4*>(y) = v;
    else *reinterpret_cast<u2*>(y) = part(v);
  } else {
    float v = 0.f;
    for (int r = 0; r < rep; ++r) v += x[(long)r * Dk];
    st1(y, v);
  }
}

template <typename T, int DKT, int NWT, bool MAP>
static void launch_walk(const Args& a, const BwdArgs& o, hipStream_t st) {
  const int lds = Stage<T, DKT, NWT, 2>::BYTES;
  allow_lds<delta_bwd_walk_kernel<T, DKT, NWT, MAP>>(lds);
  delta_bwd_walk_kernel<T, DKT, NWT, MAP><<<a.B * a.Hv * a.nseg, 64 * NWT, lds, st>>>(a, o);
}

template <typename T, int DKT, int C>
static void launch_c(const Args& a, const BwdArgs& o, bool per_value_head, hipStream_t st) {
  const int nvs = (a.Dv + 15) / 16, BH = a.B * a.Hv;
  if constexpr (C == 16) {
    delta_bwd_short_kernel<T, DKT><<<BH, 64 * nvs, strip_lds<DKT>(), st>>>(a, o);
    const int lds = (int)sizeof(PairLds<DKT>);
    allow_lds<delta_bwd_pair_kernel<T, DKT>>(lds);
    delta_bwd_pair_kernel<T, DKT><<<BH, 64 * DKT, lds, st>>>(a, o, per_value_head ? 1 : 0);
  } else {
    if (a.nseg > 1) {
      if (nvs <= 4) launch_walk<T, DKT, 4, true>(a, o, st);
      else launch_walk<T, DKT, 8, true>(a, o, st);
      launch_delta_scan(a, o.dlast, o.Ptr, o.Xseg, o.dSseg, true, st);
    }
    if (nvs <= 4) launch_walk<T, DKT, 4, false>(a, o, st);
    else launch_walk<T, DKT, 8, false>(a, o, st);
    const int lds = (int)sizeof(GradsLds<T, DKT>);
    if constexpr (DKT == 8) {
      if (const int G = a.Hv / a.Hk; G > 1 && !per_value_head) {
        allow_lds<delta_grads_kernel<T, DKT, false>>(lds);
        delta_grads_kernel<T, DKT, false><<<BH / G * a.N, 64 * DKT, lds, st>>>(a, o, G);
        return;
      }
    }
    allow_lds<delta_grads_kernel<T, DKT, true>>(lds);
    delta_grads_kernel<T, DKT, true><<<BH * a.N, 64 * DKT, lds, st>>>(a, o, 1);
  }
}

template <typename T>
static void launch_t(const Args& a, const BwdArgs& o, int C, bool pv, hipStream_t st) {
  if (C == 16) {
    if (a.Dk <= 32) launch_c<T, 2, 16>(a, o, pv, st);
    else if (a.Dk <= 64) launch_c<T, 4, 16>(a, o, pv, st);
    else launch_c<T, 8, 16>(a, o, pv, st);
  } else {
    if (a.Dk <= 32) launch_c<T, 2, 64>(a, o, pv, st);
    else if (a.Dk <= 64) launch_c<T, 4, 64>(a, o, pv, st);
    else launch_c<T, 8, 64>(a, o, pv, st);
  }
}

void launch_delta_bwd(const Args& a, const BwdArgs& o, int C, bool is_bf16, bool per_value_head, hipStream_t st) {
  if (is_bf16) launch_t<bf16>(a, o, C, per_value_head, st);
  else launch_t<float>(a, o, C, per_value_head, st);
}

void launch_delta_head_sum(const float* xq, const float* xk, void* yq, void* yk, long rows, int rep, int Dk, bool is_bf16, hipStream_t st) {
  const long n = rows * Dk;
  const int V = Dk % 4 == 0 ? 4 : 1;
  const dim3 g((unsigned)((n / V + 255) / 256), 2);
  auto launch = [&](auto* q, auto* k) {
    using T = std::remove_pointer_t<decltype(q)>;
    if (V == 4) delta_head_sum_kernel<T, 4><<<g, 256, 0, st>>>(xq, xk, q, k, n, rep, Dk);
    else delta_head_sum_kernel<T, 1><<<g, 256, 0, st>>>(xq, xk, q, k, n, rep, Dk);
  };
  if (is_bf16) launch(reinterpret_cast<bf16*>(yq), reinterpret_cast<bf16*>(yk));
  else launch(reinterpret_cast<float*>(yq), reinterpret_cast<float*>(yk));
}

}  // namespace delta
}  // namespace srl
