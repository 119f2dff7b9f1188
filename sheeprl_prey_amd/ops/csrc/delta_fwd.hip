// The gated delta rule, chunked form, forward (the mathematics and the layout: delta.h).
//
// delta_fwd_kernel<MAP = false>: one workgroup walks the chunks of one segment of one (sequence, value head), one wave
// per 16 value columns.  With few heads the chip would wait for the walk, so a long axis is split into segments: the
// walk is affine in its first state, S_last = Pseg S_first + Rseg, and <MAP = true> finds both for every segment at
// once, Rseg as the walk from zero and Pseg as the walk of the identity's columns with v = 0; delta_scan_kernel joins
// the segments; then every segment walks again from its first state and writes the outputs.
#include "delta.h"

namespace srl {
namespace delta {

template <typename T, int DKT, int C, bool MAP>
__global__ void __launch_bounds__(MAP ? 1024 : 512) delta_fwd_kernel(Args a, FwdOut o) {
  constexpr int LD = 16 * DKT + 4, LC = C + 4, NT = C / 16, DKp = 16 * DKT;
  extern __shared__ __align__(16) unsigned char lds[];
  Gates<C>& s = *reinterpret_cast<Gates<C>*>(lds);
  float* K = reinterpret_cast<float*>(lds + sizeof(Gates<C>));
  float* Q = K + (MAP ? 0 : C * LD);
  float* A = Q + C * LD;
  float* P = A + (MAP ? 0 : C * LC);
  float* Td = P + C * LC;

  const int lane = threadIdx.x & 63, l16 = lane & 15, kq = lane >> 4, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const int BH = a.B * a.Hv, bh = blockIdx.x % BH, seg = blockIdx.x / BH;
  const int b = bh / a.Hv, h = bh % a.Hv, hk = h / (a.Hv / a.Hk);
  const int nvs = (a.Dv + 15) >> 4, Dvp = 16 * nvs;
  const int len = a.lengths ? max(0, min(a.T, a.lengths[b])) : a.T;
  const bool vstrip = !MAP || wave < nvs;
  const int dv = 16 * (vstrip ? wave : wave - nvs) + l16;
  const T* qp = reinterpret_cast<const T*>(a.q) + (long)b * a.qb + (long)hk * a.qh;
  const T* kp = reinterpret_cast<const T*>(a.k) + (long)b * a.kb + (long)hk * a.kh;
  const T* vp = reinterpret_cast<const T*>(a.v) + (long)b * a.vb + (long)h * a.vh;

  f4 S[DKT];
  if (MAP) {
#pragma unroll
    for (int m = 0; m < DKT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[m][r] = (!vstrip && 16 * m + 4 * kq + r == dv) ? 1.f : 0.f;
  } else if (a.nseg > 1) {
    const float* p = o.Sseg + ((long)bh * a.nseg + seg) * DKp * Dvp + dv;
#pragma unroll
    for (int m = 0; m < DKT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[m][r] = p[(16 * m + 4 * kq + r) * Dvp];
  } else {
#pragma unroll
    for (int m = 0; m < DKT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * m + 4 * kq + r;
        S[m][r] = (a.state && d < a.Dk && dv < a.Dv) ? a.state[((long)bh * a.Dk + d) * a.Dv + dv] : 0.f;
      }
  }

  const int n1 = min(a.N, (seg + 1) * a.cps);
  for (int n = seg * a.cps; n < n1; ++n) {
    const int t0 = n * C;
    if (!MAP && o.Sc) {
      float* p = o.Sc + ((long)bh * a.N + n) * DKp * Dvp + dv;
#pragma unroll
      for (int m = 0; m < DKT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[(16 * m + 4 * kq + r) * Dvp] = S[m][r];
    }
    if (t0 >= len) {  // behind the sequence's end: the state stays, the outputs are zero
      if (!MAP && dv < a.Dv) {
        T* op = reinterpret_cast<T*>(o.out) + (long)bh * a.Dv + dv;
        for (int i = kq; i < C && t0 + i < a.T; i += 4) st1(op + (long)(t0 + i) * BH * a.Dv, 0.f);
      }
      continue;
    }
    __syncthreads();  // the chunk before is done with LDS
    load_rows<T, DKT, C>(K, s.rk, kp, a.kt, a.Dk, t0, len, a.veck, a.normalize, a.eps);
    if (!MAP) load_rows<T, DKT, C>(Q, s.rq, qp, a.qt, a.Dk, t0, len, a.vecq, a.normalize, a.eps);
    if (wave == 0) chunk_gates<C>(a, s, b, h, t0, len, lane);
    f4 v[NT];
#pragma unroll
    for (int ti = 0; ti < NT; ++ti)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = t0 + 16 * ti + 4 * kq + r;
        v[ti][r] = (vstrip && t < len && dv < a.Dv) ? ld1(vp + (long)t * a.vt + dv) : 0.f;
      }
    __syncthreads();
    pair_tiles<DKT, C>(K, MAP ? nullptr : Q, A, P, s, a.scale, wave, nw);
    // K S0 while the other waves finish their tiles
    f4 u[NT];
#pragma unroll
    for (int ti = 0; ti < NT; ++ti) u[ti] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < DKT; ++m) {
      f4 x[NT];
#pragma unroll
      for (int ti = 0; ti < NT; ++ti) x[ti] = row4(K + (16 * ti + l16) * LD + 16 * m + 4 * kq);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int ti = 0; ti < NT; ++ti) u[ti] = mfma4(x[ti][j], S[m][j], u[ti]);
    }
    __syncthreads();
    if (wave == 0) diag_inverse<C>(A, Td);
    __syncthreads();
    // U: forward substitution by blocks of 16 steps
#pragma unroll
    for (int ti = 0; ti < NT; ++ti) {
      const f4 be = row4(s.beta + 16 * ti + 4 * kq), ga = row4(s.gam + 16 * ti + 4 * kq);
      f4 r = be * (v[ti] - ga * u[ti]);
#pragma unroll
      for (int tc = 0; tc < ti; ++tc) r = mm16(-row4(A + (16 * ti + l16) * LC + 16 * tc + 4 * kq), u[tc], r);
      u[ti] = mm16(row4(Td + (16 * ti + l16) * LT + 4 * kq), r, f4{0.f, 0.f, 0.f, 0.f});
    }
    if (!MAP) {
      if (o.U) {
        float* p = o.U + ((long)bh * a.N + n) * C * Dvp + dv;
#pragma unroll
        for (int ti = 0; ti < NT; ++ti)
#pragma unroll
          for (int r = 0; r < 4; ++r) p[(16 * ti + 4 * kq + r) * Dvp] = u[ti][r];
      }
      f4 y[NT];
#pragma unroll
      for (int ti = 0; ti < NT; ++ti) y[ti] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < DKT; ++m) {
        f4 x[NT];
#pragma unroll
        for (int ti = 0; ti < NT; ++ti) x[ti] = row4(Q + (16 * ti + l16) * LD + 16 * m + 4 * kq);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int ti = 0; ti < NT; ++ti) y[ti] = mfma4(x[ti][j], S[m][j], y[ti]);
      }
      T* op = reinterpret_cast<T*>(o.out) + (long)bh * a.Dv + dv;
#pragma unroll
      for (int ti = 0; ti < NT; ++ti) {
        f4 w = y[ti] * (a.scale * row4(s.gam + 16 * ti + 4 * kq));
#pragma unroll
        for (int tj = 0; tj <= ti; ++tj) w = mm16(row4(P + (16 * ti + l16) * LC + 16 * tj + 4 * kq), u[tj], w);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int t = t0 + 16 * ti + 4 * kq + r;
          if (t < a.T && dv < a.Dv) st1(op + (long)t * BH * a.Dv, t < len ? w[r] : 0.f);
        }
      }
    }
    // S' = gam_C S + K^T diag(e) U
    const float gc = s.gam[C - 1];
#pragma unroll
    for (int m = 0; m < DKT; ++m) S[m] *= gc;
#pragma unroll
    for (int ti = 0; ti < NT; ++ti) {
      const f4 w = u[ti] * row4(s.e + 16 * ti + 4 * kq);
      f4 x[DKT];
#pragma unroll
      for (int m = 0; m < DKT; ++m) x[m] = col4(K + (16 * ti + 4 * kq) * LD + 16 * m + l16, LD);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int m = 0; m < DKT; ++m) S[m] = mfma4(x[m][j], w[j], S[m]);
    }
  }
  if (MAP) {
    const int ld = vstrip ? Dvp : DKp;
    float* p = (vstrip ? o.Rseg : o.Pseg) + ((long)bh * a.nseg + seg) * DKp * ld + dv;
#pragma unroll
    for (int m = 0; m < DKT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) p[(16 * m + 4 * kq + r) * ld] = S[m][r];
  } else if (seg == a.nseg - 1 && dv < a.Dv) {
#pragma unroll
    for (int m = 0; m < DKT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * m + 4 * kq + r;
        if (d < a.Dk) o.last[((long)bh * a.Dk + d) * a.Dv + dv] = S[m][r];
      }
  }
}

// Joins the segments: S_{s+1} = Pseg_s S_s + Rseg_s (REV: dS_s = Pseg_s^T dS_{s+1} + Xseg_s), one wave per 16 columns.
template <int DKT, bool REV>
__global__ void __launch_bounds__(64) delta_scan_kernel(const float* first, const float* P, const float* R, float* out, int nseg,
                                                        int Dk, int Dv) {
  constexpr int DKp = 16 * DKT;
  const int lane = threadIdx.x, l16 = lane & 15, kq = lane >> 4;
  const int nvs = (Dv + 15) >> 4, Dvp = 16 * nvs, bh = blockIdx.x / nvs, dv = 16 * (blockIdx.x % nvs) + l16;
  f4 S[DKT];
#pragma unroll
  for (int m = 0; m < DKT; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * m + 4 * kq + r;
      S[m][r] = (first && d < Dk && dv < Dv) ? first[((long)bh * Dk + d) * Dv + dv] : 0.f;
    }
  for (int i = 0; i < nseg; ++i) {
    const int s = REV ? nseg - 1 - i : i;
    const long at = ((long)bh * nseg + s) * DKp;
    f4 n[DKT];
#pragma unroll
    for (int m = 0; m < DKT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) out[(at + 16 * m + 4 * kq + r) * Dvp + dv] = S[m][r];
    if (i == nseg - 1) break;
#pragma unroll
    for (int m = 0; m < DKT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) n[m][r] = R[(at + 16 * m + 4 * kq + r) * Dvp + dv];
    const float* p = P + at * DKp;
#pragma unroll
    for (int mk = 0; mk < DKT; ++mk) {
      f4 x[DKT];
#pragma unroll
      for (int m = 0; m < DKT; ++m)
        x[m] = REV ? col4(p + (16 * mk + 4 * kq) * DKp + 16 * m + l16, DKp) : row4(p + (16 * m + l16) * DKp + 16 * mk + 4 * kq);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int m = 0; m < DKT; ++m) n[m] = mfma4(x[m][j], S[mk][j], n[m]);
    }
#pragma unroll
    for (int m = 0; m < DKT; ++m) S[m] = n[m];
  }
}

template <typename T, int DKT, int C, bool MAP>
static void launch_one(const Args& a, const FwdOut& o, hipStream_t st) {
  const size_t lds = strip_lds<DKT, C>(!MAP);
  allow_lds<delta_fwd_kernel<T, DKT, C, MAP>>((int)lds);
  const int nvs = (a.Dv + 15) / 16;
  delta_fwd_kernel<T, DKT, C, MAP><<<a.B * a.Hv * a.nseg, 64 * (nvs + (MAP ? DKT : 0)), lds, st>>>(a, o);
}

template <typename T, int DKT>
static void launch_dk(const Args& a, const FwdOut& o, int C, hipStream_t st) {
  if (C == 16) {
    launch_one<T, DKT, 16, false>(a, o, st);
    return;
  }
  if (a.nseg > 1) {
    launch_one<T, DKT, 64, true>(a, o, st);
    delta_scan_kernel<DKT, false><<<a.B * a.Hv * ((a.Dv + 15) / 16), 64, 0, st>>>(a.state, o.Pseg, o.Rseg, o.Sseg, a.nseg, a.Dk, a.Dv);
  }
  launch_one<T, DKT, 64, false>(a, o, st);
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

void launch_delta_scan_rev(const float* dlast, const float* P, const float* X, float* dS, int BH, int nseg, int Dk, int Dv,
                           hipStream_t st) {
  const int g = BH * ((Dv + 15) / 16);
  if (Dk <= 32) delta_scan_kernel<2, true><<<g, 64, 0, st>>>(dlast, P, X, dS, nseg, Dk, Dv);
  else if (Dk <= 64) delta_scan_kernel<4, true><<<g, 64, 0, st>>>(dlast, P, X, dS, nseg, Dk, Dv);
  else delta_scan_kernel<8, true><<<g, 64, 0, st>>>(dlast, P, X, dS, nseg, Dk, Dv);
}

}  // namespace delta
}  // namespace srl
