// The gated delta rule, chunked form, forward (the mathematics and the layout: delta.h).
//
// Chunks of 64 steps: delta_pairs_kernel finds A, P, the inverses of the diagonal blocks of I + A and the gates of every
// chunk, all chunks at once, for the forward and the backward walk.  delta_walk_kernel<MAP = false> walks the chunks of
// one segment of one (sequence, value head), one wave per 16 value columns, the next chunk's operands on their way while it
// works on this one.  With few heads the chip would wait for the walk, so a long axis is split into segments: the walk is
// affine in its first state, S_last = Pseg S_first + Rseg, and <MAP = true> finds both for every segment at once, Rseg as the
// walk from zero and Pseg as the walk of the identity's columns with v = 0; delta_scan_kernel joins the segments; then
// every segment walks again from its first state and writes the outputs.
//
// Sequences of at most 16 steps are one chunk of 16: delta_short_kernel does all of it at once (8 steps x 128 x 2 heads of 32
// in 9 us: latency, of its reads, the substitution and the joins of the waves).
//
// Measured at 4096 steps x 2 x 16 heads of 128 in bf16 (8 segments a head), us in a kernel trace: pairs 38, maps 110, joins
// 18, walk 112.  The bytes would take 20 us and the products 13: a walk is bound by the chain of one chunk (23500 cycles by the
// clock, 21500 with 8 heads: operands and the other waves 6000 and 4500, their way into LDS 2000, K S and Q S 4300, the
// substitution, each block of which waits for the one before, 3900, the outputs 3400 to 3700, the state 1700), with two waves a
// SIMD to hide its waits.  Q S and the outputs wait for no later chunk and are in the chain all the same.
#include "delta.h"

namespace srl {
namespace delta {

template <typename T, int DKT>
__global__ void __launch_bounds__(512) delta_short_kernel(Args a, FwdOut o) {
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
  const T* vp = reinterpret_cast<const T*>(a.v) + (long)b * a.vb + (long)h * a.vh;

  // a sequence of no steps reads its first one, which is there, and counts none of it
  Column<T, 1> vc;
  vc.fetch(vp + min(dv, a.Dv - 1), a.vt, 0, max(len, 1), kq);
  load_rows<T, DKT, C, 4>(K, s.rk, kp, a.kt, a.Dk, 0, len, a.veck, a.normalize, a.eps);
  load_rows<T, DKT, C, 4>(Q, s.rq, qp, a.qt, a.Dk, 0, len, a.vecq, a.normalize, a.eps);
  if (wave == 0) chunk_gates<C>(a, s, b, h, 0, len, lane);
  const float* s0 = state_before(a, b, len);
  f4 S[DKT];
#pragma unroll
  for (int m = 0; m < DKT; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * m + 4 * kq + r;
      S[m][r] = (s0 && d < a.Dk && dv < a.Dv) ? s0[((long)bh * a.Dk + d) * a.Dv + dv] : 0.f;
      if (o.Sc) o.Sc[((long)bh * DKp + d) * Dvp + dv] = S[m][r];
    }
  lds_barrier();
  const f4 v = vc.get(0, 0, len, kq, dv < a.Dv);
  pair_tiles<DKT>(K, Q, A, P, s, a.scale, wave, nw);
  f4 u = {0.f, 0.f, 0.f, 0.f}, y = u;
#pragma unroll
  for (int m = 0; m < DKT; ++m) {
    u = mm16(row4(K + l16 * LD + 16 * m + 4 * kq), S[m], u);
    y = mm16(row4(Q + l16 * LD + 16 * m + 4 * kq), S[m], y);
  }
  lds_barrier();
  if (wave == 0) diag_inverse(A, Td);
  lds_barrier();
  const f4 ga = row4(s.gam + 4 * kq);
  u = mm16(row4(Td + l16 * LT + 4 * kq), row4(s.beta + 4 * kq) * (v - ga * u), f4{0.f, 0.f, 0.f, 0.f});
  y = mm16(row4(P + l16 * LT + 4 * kq), u, y * (a.scale * ga));
  T* op = reinterpret_cast<T*>(o.out) + (long)bh * a.Dv + dv;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int t = 4 * kq + r;
    if (o.U) o.U[((long)bh * C + t) * Dvp + dv] = u[r];
    if (t < a.T && dv < a.Dv) st1(op + (long)t * BH * a.Dv, t < len ? y[r] : 0.f);
  }
  const float gc = s.gam[C - 1];
  const f4 w = u * row4(s.e + 4 * kq);
#pragma unroll
  for (int m = 0; m < DKT; ++m) {
    S[m] = mm16(col4(K + 4 * kq * LD + 16 * m + l16, LD), w, S[m] * gc);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * m + 4 * kq + r;
      if (d < a.Dk && dv < a.Dv) o.last[((long)bh * a.Dk + d) * a.Dv + dv] = S[m][r];
    }
  }
}

// One workgroup a chunk and G value heads that share a key head: the products k_j . k_i and q_i . k_j serve them all.  Bound by
// the writes of 25 KB a chunk and head and by the inverses' substitution: 2048 chunks of 128 columns in 38 us (1.4 TB/s).
template <typename T, int DKT>
struct PairsLds {
  static constexpr bool SP = sizeof(T) == 2;
  static constexpr int LD = SP ? 16 * DKT + 8 : 16 * DKT + 4;  // bf16 rows raw, in the order of place(); fp32 rows of unit length
  typename std::conditional<SP, uint16_t, float>::type K[64 * LD], Q[64 * LD];
  Gates<64> s;
  float A[4 * TS];  // the four diagonal tiles
};

template <typename T, int DKT>
__global__ void __launch_bounds__(256) delta_pairs_kernel(Args a, float* pairs, int G) {
  using L = PairsLds<T, DKT>;
  constexpr bool SP = L::SP;
  constexpr int C = 64, LD = L::LD, NE = DKT;
  extern __shared__ __align__(16) unsigned char lds[];
  L& l = *reinterpret_cast<L*>(lds);
  Gates<C>& s = l.s;

  const int lane = threadIdx.x & 63, l16 = lane & 15, kq = lane >> 4, wave = wave_id();
  const int Hg = a.Hv / G, bg = blockIdx.x % (a.B * Hg), n = blockIdx.x / (a.B * Hg), t0 = n * C;
  const int b = bg / Hg, h0 = (bg % Hg) * G, hk = h0 / (a.Hv / a.Hk);
  const int len = a.lengths ? max(0, min(a.T, a.lengths[b])) : a.T;
  if (t0 >= len) return;
  const T* kp = reinterpret_cast<const T*>(a.k) + (long)b * a.kb + (long)hk * a.kh;
  const T* qp = reinterpret_cast<const T*>(a.q) + (long)b * a.qb + (long)hk * a.qh;
  if constexpr (!SP) {
    load_rows<T, DKT, C, 4>(l.K, s.rk, kp, a.kt, a.Dk, t0, len, a.veck, a.normalize, a.eps);
    load_rows<T, DKT, C, 4>(l.Q, s.rq, qp, a.qt, a.Dk, t0, len, a.vecq, a.normalize, a.eps);
  } else {
    const int sub = threadIdx.x & 15, c0 = sub * NE, D = a.Dk;
    auto rows = [&](uint16_t* M, float* rn, const T* src, long st, bool vec) {
      T x[4][NE];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const T* p = src + (long)max(0, min(t0 + (int)(threadIdx.x >> 4) + 16 * r, len - 1)) * st;
        if (vec) {
#pragma unroll
          for (int j = 0; j < NE; j += 2)
            *reinterpret_cast<uint32_t*>(&x[r][j]) = *reinterpret_cast<const uint32_t*>(p + min(c0 + j, D - 2));
        } else {
#pragma unroll
          for (int j = 0; j < NE; ++j) x[r][j] = p[min(c0 + j, D - 1)];
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = (threadIdx.x >> 4) + 16 * r;
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < NE; ++j) {
          if (t0 + i >= len || c0 + j >= D) x[r][j].x = 0;
          const float f = ld1(&x[r][j]);
          ss = fmaf(f, f, ss);
          M[i * LD + place(c0 + j)] = x[r][j].x;
        }
        const float nn = unit_factor(row16_sum(ss), t0 + i < len, a.normalize, a.eps);
        if (sub == 0) rn[i] = nn;
      }
    };
    rows(l.K, s.rk, kp, a.kt, a.veck);
    rows(l.Q, s.rq, qp, a.qt, a.vecq);
  }
  if (wave == 3) chunk_gates<C>(a, s, b, h0, t0, len, lane);
  lds_barrier();

  // This wave's tiles x = wave, wave + 4, wave + 8, the diagonal ones first: their inverses follow while the others wait.
  auto tile_of = [](int x, int& ti, int& tj) {
    ti = x < 4 ? x : x < 7 ? x - 3 : x < 9 ? x - 5 : 3;
    tj = x < 4 ? x : x < 7 ? x - 4 : x < 9 ? x - 7 : 0;
  };
  f4 kk[3], qk[3];
#pragma unroll
  for (int y = 0; y < 3; ++y) {
    kk[y] = qk[y] = f4{0.f, 0.f, 0.f, 0.f};
    const int x = wave + 4 * y;
    if (x >= 10) continue;
    int ti, tj;
    tile_of(x, ti, tj);
    if constexpr (SP) {
      const int at = 8 * kq, kj = (16 * tj + l16) * LD + at, xi = (16 * ti + l16) * LD + at;
#pragma unroll
      for (int m2 = 0; m2 < DKT / 2; ++m2) {
        const b8 k = *reinterpret_cast<const b8*>(l.K + kj + 32 * m2);
        kk[y] = mfma32(k, *reinterpret_cast<const b8*>(l.K + xi + 32 * m2), kk[y]);
        qk[y] = mfma32(k, *reinterpret_cast<const b8*>(l.Q + xi + 32 * m2), qk[y]);
      }
      const f4 rj = row4(s.rk + 16 * tj + 4 * kq);
      kk[y] *= rj * s.rk[16 * ti + l16];
      qk[y] *= rj * s.rq[16 * ti + l16];
    } else {
      const int kj = (16 * tj + l16) * LD + 4 * kq, xi = (16 * ti + l16) * LD + 4 * kq;
#pragma unroll
      for (int m = 0; m < DKT; ++m) {
        const f4 k = row4(l.K + kj + 16 * m), ki = row4(l.K + xi + 16 * m), qi = row4(l.Q + xi + 16 * m);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          kk[y] = mfma4(k[j], ki[j], kk[y]);
          qk[y] = mfma4(k[j], qi[j], qk[y]);
        }
      }
    }
    qk[y] *= a.scale;
  }
  for (int g = 0; g < G; ++g) {
    if (g > 0) {
      lds_barrier();
      if (wave == 3) chunk_gates<C>(a, s, b, h0 + g, t0, len, lane);
      lds_barrier();
    }
    float* out = pairs + (((long)b * a.Hv + h0 + g) * a.N + n) * PAIR_FLOATS;
#pragma unroll
    for (int y = 0; y < 3; ++y) {
      const int x = wave + 4 * y;
      if (x >= 10) continue;
      int ti, tj;
      tile_of(x, ti, tj);
      const int i = 16 * ti + l16, j0 = 16 * tj + 4 * kq, t = ti * (ti + 1) / 2 + tj;
      const double Gi = s.G[i];
      const int segi = s.seg[i];
      const float be = s.beta[i];
      f4 dk, dq;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float m = pair_decay<C>(s, i, j0 + r, Gi, segi);
        dk[r] = j0 + r < i ? be * m * kk[y][r] : 0.f;
        dq[r] = m * qk[y][r];
      }
      *reinterpret_cast<f4*>(out + (PAIR_A + t) * 256 + l16 * 16 + 4 * kq) = dk;
      *reinterpret_cast<f4*>(out + (PAIR_P + t) * 256 + l16 * 16 + 4 * kq) = dq;
      if (y == 0) {  // diagonal: this wave's own tile, no barrier between its writes and its reads
        float* d = l.A + ti * TS;
        *reinterpret_cast<f4*>(d + l16 * TL + 4 * kq) = dk;
        __builtin_amdgcn_wave_barrier();
        float c[16];
#pragma unroll
        for (int i2 = 0; i2 < 16; ++i2) {
          float v = i2 == l16 ? 1.f : 0.f;
#pragma unroll
          for (int m4 = 0; m4 < i2; m4 += 4) {
            const f4 r = row4(d + i2 * TL + m4);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (m4 + j < i2) v = fmaf(-r[j], c[m4 + j], v);
          }
          c[i2] = v;
        }
#pragma unroll
        for (int i2 = 0; i2 < 16; ++i2)
          if ((i2 >> 2) == kq) out[(PAIR_T + ti) * 256 + i2 * 16 + l16] = c[i2];
      }
    }
    float* gt = out + PAIR_TILES * 256;
    gt[threadIdx.x] = wave == 0 ? s.beta[lane] : wave == 1 ? s.gam[lane] : wave == 2 ? s.e[lane] : s.rq[lane];
    if (wave == 0) gt[256 + lane] = s.rk[lane];
  }
}

template <typename T, int DKT, int NWT, bool MAP>
__global__ void __launch_bounds__(64 * NWT) delta_walk_kernel(Args a, FwdOut o) {
  using St = Stage<T, DKT, NWT, MAP ? 1 : 0>;
  constexpr bool SP = St::SP;
  constexpr int C = 64, NT = 4, DKp = 16 * DKT, Dvp = NWT == 4 ? 64 : 128;
  extern __shared__ __align__(16) unsigned char lds[];
  St st(lds);

  const int lane = threadIdx.x & 63, l16 = lane & 15, kq = lane >> 4, wave = wave_id();
  const int BH = a.B * a.Hv, bh = blockIdx.x % BH, seg = blockIdx.x / BH;
  const int b = bh / a.Hv, h = bh % a.Hv, hk = h / (a.Hv / a.Hk);
  const int nvs = (a.Dv + 15) >> 4;
  const int len = a.lengths ? max(0, min(a.T, a.lengths[b])) : a.T;
  const bool vstrip = wave < nvs, works = wave < nvs + (MAP ? DKT : 0);  // the other waves only move operands
  const int dv = 16 * (vstrip ? wave : wave - nvs) + l16;
  const T* qp = reinterpret_cast<const T*>(a.q) + (long)b * a.qb + (long)hk * a.qh;
  const T* kp = reinterpret_cast<const T*>(a.k) + (long)b * a.kb + (long)hk * a.kh;
  const T* vp = reinterpret_cast<const T*>(a.v) + (long)b * a.vb + (long)h * a.vh;
  const float* pairs = o.pairs + (long)bh * a.N * PAIR_FLOATS;

  f4 S[DKT];
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < DKT; ++m) S[m] = zero;
  if (MAP) {
    if (!vstrip) {
#pragma unroll
      for (int m = 0; m < DKT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[m][r] = 16 * m + 4 * kq + r == dv ? 1.f : 0.f;
    }
  } else if (works && a.nseg > 1) {
    const float* p = o.Sseg + ((((long)bh * a.nseg + seg) * nvs + wave) * DKT * 64 + lane) * 4;
#pragma unroll
    for (int m = 0; m < DKT; ++m) S[m] = row4(p + m * 256);
  } else if (const float* s0 = state_before(a, b, len); works && s0) {
#pragma unroll
    for (int m = 0; m < DKT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * m + 4 * kq + r;
        if (d < a.Dk && dv < a.Dv) S[m][r] = s0[((long)bh * a.Dk + d) * a.Dv + dv];
      }
  }
  Column<T, NT> v;
  const T* vcol = vp + min(dv, a.Dv - 1);
  const int n0 = seg * a.cps, n1 = min(a.N, n0 + a.cps), live = min(n1, (len + C - 1) / C);
  if (n0 < live) {
    st.fetch(a, qp, kp, pairs + (long)n0 * PAIR_FLOATS, n0 * C, len);
    if (vstrip) v.fetch(vcol, a.vt, n0 * C, len, kq);
  }
  for (int n = n0; n < live; ++n) {
    const int t0 = n * C;
    if (!MAP && o.Sc && works) {
      float* p = o.Sc + ((long)bh * a.N + n) * DKp * Dvp + 4 * kq * Dvp + dv;
#pragma unroll
      for (int m = 0; m < DKT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[(16 * m + r) * Dvp] = S[m][r];
    }
    lds_barrier();  // the chunk before is done with LDS
    st.turn();
    st.commit(t0, len, a.Dk);
    lds_barrier();
    f4 u[NT];
#pragma unroll
    for (int ti = 0; ti < NT; ++ti) u[ti] = st.beta(ti) * v.get(ti, t0, len, kq, vstrip && dv < a.Dv);
    // the next chunk on its way, a part at a time: see Stage
    auto ahead = [&](auto part) {
      if (n + 1 < live) st.fetch(part, a, qp, kp, pairs + (long)(n + 1) * PAIR_FLOATS, t0 + C, len);
    };
    if (!works) {
      each<0, 3>(ahead);
      continue;
    }
    if (n + 1 < live && vstrip) v.fetch(vcol, a.vt, t0 + C, len, kq);
    part_ends();
    // K S0 and Q S0
    f4 ks[NT], y[NT];
#pragma unroll
    for (int ti = 0; ti < NT; ++ti) ks[ti] = y[ti] = zero;
    each<0, DKT / 2>([&](auto M) {
      constexpr int m2 = M;
      const Op16<SP> s0 = cut<SP>(S[2 * m2]), s1 = cut<SP>(S[2 * m2 + 1]);
#pragma unroll
      for (int ti = 0; ti < NT; ++ti) {
        ks[ti] = mm32(st.k(ti, m2), s0, s1, ks[ti]);
        if constexpr (!MAP) y[ti] = mm32(st.q(ti, m2), s0, s1, y[ti]);
      }
      part_ends();
      if constexpr (m2 < 2) ahead(M);
    });
    if constexpr (DKT == 2) ahead(std::integral_constant<int, 1>{});
    part_ends();
    // U: forward substitution by blocks of 16 steps
    Op16<SP> ub[NT];
    each<0, NT>([&](auto I) {
      constexpr int ti = I;
      f4 r = u[ti] - st.beta(ti) * st.gam(ti) * st.rk4(ti) * ks[ti];
      r = mm_tiles<0, ti>([&](int x) { return st.A(ti, x); }, [&](auto x) { return ub[decltype(x)::value]; }, r);
      u[ti] = mm16o(st.Ti(ti), cut<SP>(r), zero);
      ub[ti] = cut<SP>(u[ti]);
      if constexpr (ti == 0) ahead(std::integral_constant<int, 2>{});
    });
    part_ends();
    if constexpr (!MAP) {
      if (o.U) {
        float* p = o.U + ((long)bh * a.N + n) * C * Dvp + 4 * kq * Dvp + dv;
#pragma unroll
        for (int ti = 0; ti < NT; ++ti)
#pragma unroll
          for (int r = 0; r < 4; ++r) p[(16 * ti + r) * Dvp] = u[ti][r];
      }
      const long ostep = afresh((long)BH * a.Dv);
      T* op = reinterpret_cast<T*>(o.out) + (long)bh * a.Dv + dv + (t0 + 4 * kq) * ostep;
      each<0, NT>([&](auto I) {
        constexpr int ti = I;
        const f4 w = mm_tiles<0, ti + 1>([&](int x) { return st.P(ti, x); }, [&](auto x) { return ub[decltype(x)::value]; },
                                         y[ti] * (a.scale * st.gam(ti) * st.rq4(ti)));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int t = t0 + 16 * ti + 4 * kq + r;
          if (t < a.T && dv < a.Dv) st1(op + (16 * ti + r) * ostep, t < len ? w[r] : 0.f);
        }
      });
    }
    part_ends();
    // S' = gam_C S + K^T diag(e) U
    const float gc = st.gam_last();
#pragma unroll
    for (int m = 0; m < DKT; ++m) S[m] *= gc;
#pragma unroll
    for (int t2 = 0; t2 < NT / 2; ++t2) {
      const Op16<SP> w0 = cut<SP>(u[2 * t2] * st.e(2 * t2) * st.rk4(2 * t2)), w1 = cut<SP>(u[2 * t2 + 1] * st.e(2 * t2 + 1) * st.rk4(2 * t2 + 1));
#pragma unroll
      for (int m = 0; m < DKT; ++m) S[m] = mm32(st.kt(m, t2), w0, w1, S[m]);
    }
  }
  if (!works) return;
  if (MAP) {
    if (vstrip) {
      float* p = o.Rseg + ((((long)bh * a.nseg + seg) * nvs + wave) * DKT * 64 + lane) * 4;
#pragma unroll
      for (int m = 0; m < DKT; ++m) *reinterpret_cast<f4*>(p + m * 256) = S[m];
    } else {
      const int col = wave - nvs;  // the tile column
      float* p = o.Pseg + ((long)bh * a.nseg + seg) * DKp * DKp + col * 256 + ((l16 >> 2) * 16 + 4 * kq) * 4 + (l16 & 3);
#pragma unroll
      for (int m = 0; m < DKT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[m * DKT * 256 + 4 * r] = S[m][r];
      if (o.Ptr) {
        float* t = o.Ptr + ((long)bh * a.nseg + seg) * DKp * DKp + col * DKT * 256 + lane * 4;
#pragma unroll
        for (int m = 0; m < DKT; ++m) *reinterpret_cast<f4*>(t + m * 256) = S[m];
      }
    }
    return;
  }
  if (dv >= a.Dv) return;
  T* op = reinterpret_cast<T*>(o.out) + (long)bh * a.Dv + dv;  // behind the sequence's end: zeros
  for (int t = max(n0, live) * C + kq; t < min(a.T, n1 * C); t += 4) st1(op + (long)t * BH * a.Dv, 0.f);
  if (seg == a.nseg - 1) {
#pragma unroll
    for (int m = 0; m < DKT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * m + 4 * kq + r;
        if (d < a.Dk) o.last[((long)bh * a.Dk + d) * a.Dv + dv] = S[m][r];
      }
  }
}

// Joins the segments: S_{s+1} = Pseg_s S_s + Rseg_s, or backwards (REV) dS_s = Pseg_s^T dS_{s+1} + Xseg_s with the maps
// transposed.  One workgroup per 16 columns, one wave per 16 rows; the state goes through LDS in three bf16 parts, and the
// next two maps are on their way meanwhile.  Every strip of a head reads the head's maps, 64 KB each: 32 heads of 128 in 8
// segments take 18 us (7.5 TB/s out of the L2s), 8 heads in 32 segments 48 us, 1.5 us a join, which is bound by the join's chain.
template <int DKT, bool REV>
__global__ void __launch_bounds__(64 * DKT) delta_scan_kernel(Args a, const float* dlast, const float* P, const float* R, float* out) {
  constexpr int DKp = 16 * DKT, LD = DKp + 8;
  __shared__ __align__(16) uint16_t S[2][3][16 * LD];
  const int lane = threadIdx.x & 63, m = wave_id(), l16 = lane & 15, kq = lane >> 4;
  // the strips of a head BH workgroups apart: on one chiplet, whose L2 then has the head's maps, where 8 divides BH
  const int Dk = a.Dk, Dv = a.Dv, nseg = a.nseg, nvs = (Dv + 15) >> 4, BH = gridDim.x / nvs, bh = blockIdx.x % BH, strip = blockIdx.x / BH, dv = 16 * strip + l16;
  const int len = a.lengths ? max(0, min(a.T, a.lengths[bh / a.Hv])) : a.T;
  const float* first = REV ? dlast : state_before(a, bh / a.Hv, len);
  f4 s, r[3], x[3][DKT];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = 16 * m + 4 * kq + j;
    s[j] = (first && d < Dk && dv < Dv) ? first[((long)bh * Dk + d) * Dv + dv] : 0.f;
  }
  auto at = [&](int i) { return (long)bh * nseg + (REV ? nseg - 1 - i : i); };
  auto native = [&](long g) { return ((g * nvs + strip) * DKT + m) * 256 + lane * 4; };
  auto fetch = [&](int i, f4* xs, f4& rs) {
    const float* p = P + at(i) * DKp * DKp + m * DKT * 256 + lane * 4;
#pragma unroll
    for (int k = 0; k < DKT; ++k) xs[k] = row4(p + k * 256);
    rs = row4(R + native(at(i)));
  };
  auto step = [&](int i, const f4* xs, const f4& rs, uint16_t (*l)[16 * LD]) {
    *reinterpret_cast<f4*>(out + native(at(i))) = s;
    const Op16<true> c = cut3(s);
    const int w = l16 * LD + place(16 * m + 4 * kq);
    *reinterpret_cast<u2*>(l[0] + w) = c.p0;
    *reinterpret_cast<u2*>(l[1] + w) = c.p1;
    *reinterpret_cast<u2*>(l[2] + w) = c.p2;
    lds_barrier();  // two buffers: the one before is free once every wave is here
    f4 n[2] = {rs, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int k = 0; k < DKT; k += 2) {
      const int a = l16 * LD + 16 * k + 8 * kq;
      const u4 p0 = *reinterpret_cast<const u4*>(l[0] + a), p1 = *reinterpret_cast<const u4*>(l[1] + a), p2 = *reinterpret_cast<const u4*>(l[2] + a);
      const Op16<true> b0 = {p0.xy, p1.xy, p2.xy}, b1 = {p0.zw, p1.zw, p2.zw};
      n[(k >> 1) & 1] = mm32(cut3(xs[k]), cut3(xs[k + 1]), b0, b1, n[(k >> 1) & 1]);
    }
    s = n[0] + n[1];
  };
  const int last = nseg - 1;  // the last segment's first state is the end of it
  fetch(0, x[0], r[0]);
  fetch(min(1, last), x[1], r[1]);
  for (int i = 0; i < last; i += 3) {
    fetch(min(i + 2, last), x[2], r[2]);
    step(i, x[0], r[0], S[i & 1]);
    if (i + 1 >= last) break;
    fetch(min(i + 3, last), x[0], r[0]);
    step(i + 1, x[1], r[1], S[(i + 1) & 1]);
    if (i + 2 >= last) break;
    fetch(min(i + 4, last), x[1], r[1]);
    step(i + 2, x[2], r[2], S[i & 1]);
  }
  *reinterpret_cast<f4*>(out + native(at(last))) = s;
}

template <typename T, int DKT, int NWT, bool MAP>
static void launch_walk(const Args& a, const FwdOut& o, hipStream_t st) {
  const int lds = Stage<T, DKT, NWT, MAP ? 1 : 0>::BYTES;
  allow_lds<delta_walk_kernel<T, DKT, NWT, MAP>>(lds);
  delta_walk_kernel<T, DKT, NWT, MAP><<<a.B * a.Hv * a.nseg, 64 * NWT, lds, st>>>(a, o);
}

template <typename T, int DKT>
static void launch_dk(const Args& a, const FwdOut& o, int C, hipStream_t st) {
  const int nvs = (a.Dv + 15) / 16, BH = a.B * a.Hv;
  if (C == 16) {
    const int lds = (int)strip_lds<DKT>();
    delta_short_kernel<T, DKT><<<BH, 64 * nvs, lds, st>>>(a, o);
    return;
  }
  const int lds = (int)sizeof(PairsLds<T, DKT>);
  allow_lds<delta_pairs_kernel<T, DKT>>(lds);
  const int G = a.B * a.Hk * a.N >= 512 ? a.Hv / a.Hk : 1;  // fewer workgroups than that leave CUs idle
  delta_pairs_kernel<T, DKT><<<BH / G * a.N, 256, lds, st>>>(a, o.pairs, G);
  if (a.nseg > 1) {
    if (nvs + DKT <= 8) launch_walk<T, DKT, 8, true>(a, o, st);
    else launch_walk<T, DKT, 16, true>(a, o, st);
    launch_delta_scan(a, nullptr, o.Pseg, o.Rseg, o.Sseg, false, st);
  }
  if (nvs <= 4) launch_walk<T, DKT, 4, false>(a, o, st);
  else launch_walk<T, DKT, 8, false>(a, o, st);
}

template <typename T>
static void launch_t(const Args& a, const FwdOut& o, int C, hipStream_t st) {
  if (a.Dk <= 32) launch_dk<T, 2>(a, o, C, st);
  else if (a.Dk <= 64) launch_dk<T, 4>(a, o, C, st);
  else launch_dk<T, 8>(a, o, C, st);
}

void launch_delta_fwd(const Args& a, const FwdOut& o, int C, bool is_bf16, hipStream_t st) {
  if (is_bf16) launch_t<bf16>(a, o, C, st);
  else launch_t<float>(a, o, C, st);
}

template <int DKT>
static void launch_scan(const Args& a, const float* dlast, const float* P, const float* X, float* S, bool rev, hipStream_t st) {
  const int g = a.B * a.Hv * ((a.Dv + 15) / 16);
  if (rev) delta_scan_kernel<DKT, true><<<g, 64 * DKT, 0, st>>>(a, dlast, P, X, S);
  else delta_scan_kernel<DKT, false><<<g, 64 * DKT, 0, st>>>(a, dlast, P, X, S);
}

void launch_delta_scan(const Args& a, const float* dlast, const float* P, const float* X, float* S, bool rev, hipStream_t st) {
  if (a.Dk <= 32) launch_scan<2>(a, dlast, P, X, S, rev, st);
  else if (a.Dk <= 64) launch_scan<4>(a, dlast, P, X, S, rev, st);
  else launch_scan<8>(a, dlast, P, X, S, rev, st);
}

}  // namespace delta
}  // namespace srl
