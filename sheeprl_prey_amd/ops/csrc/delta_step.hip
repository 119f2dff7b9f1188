// The gated delta rule, recurrent form (the mathematics: delta.h): single steps, and short sequences that need no gradient.
//
// A step must read and write the whole state, 8 bytes for every 7 operations: it is bound by memory, and by latency where the
// states are few.  One wave owns 32 value columns of one (sequence, head): 8 lanes of 16 bytes cover a row's 128 bytes,
// 8 rows at once, the state in registers over all steps.  Both read-outs are taken from the state BEFORE the update,
//   o = scale (exp(g) S^T q + (q . k) u),
// so a step has one round of reductions over the key rows instead of two that wait for each other.
//
// The state goes past the caches (non-temporal): between two steps a program's weights and activations would drive it out.
// 256 sequences x 16 heads of 128 x 128, bf16, states other than the last step's: 110 us, 4.9 TB/s of state (a copy of that
// size 5.2), 133 us through the caches; 512 MiB of states 207 and 232 us.  Of the very state of the step before, with nothing
// in between, 128 to 256 MiB take 5 to 8 % longer so, less than that no longer.  16 sequences x 2 heads of 32 x 32: 6.1 us,
// the launch.
#include "delta.h"

namespace srl {
namespace delta {

template <typename T, int NP, bool VEC>
__global__ void __launch_bounds__(256) delta_step_kernel(Args a, T* out, float* S2, long sb, long sh) {
  const int lane = threadIdx.x & 63, c4 = lane & 7, rg = lane >> 3;
  const int ncb = (a.Dv + 31) >> 5;
  const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (long)a.B * a.Hv * ncb) return;
  const int cb = (int)(item % ncb), bh = (int)(item / ncb), b = bh / a.Hv, h = bh % a.Hv, hk = h / (a.Hv / a.Hk);
  const int dv = 32 * cb + 4 * c4;
  const int len = a.lengths ? max(0, min(a.T, a.lengths[b])) : a.T;
  const bool live = dv < a.Dv;
  const long so = (long)b * sb + (long)h * sh + dv;

  f4 S[NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int d = 8 * p + rg;
    S[p] = f4{0.f, 0.f, 0.f, 0.f};
    if (a.state && d < a.Dk && live) {
      const float* x = a.state + so + (long)d * a.Dv;
      if (VEC) S[p] = __builtin_nontemporal_load(reinterpret_cast<const f4*>(x));
      else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (dv + j < a.Dv) S[p][j] = x[j];
      }
    }
  }
  const T* qp = reinterpret_cast<const T*>(a.q) + (long)b * a.qb + (long)hk * a.qh;
  const T* kp = reinterpret_cast<const T*>(a.k) + (long)b * a.kb + (long)hk * a.kh;
  const T* vp = reinterpret_cast<const T*>(a.v) + (long)b * a.vb + (long)h * a.vh + dv;
  const long BH = (long)a.B * a.Hv;
  T* op = out + (long)bh * a.Dv + dv;

  for (int t = 0; t < len; ++t) {
    float q[NP], k[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int d = 8 * p + rg;
      k[p] = d < a.Dk ? ld1(kp + (long)t * a.kt + d) : 0.f;
      q[p] = d < a.Dk ? ld1(qp + (long)t * a.qt + d) : 0.f;
    }
    const float g = a.g[(long)t * a.gt + (long)b * a.gb + (long)h * a.gh];
    const float be = a.beta[(long)t * a.bt + (long)b * a.bb + (long)h * a.bh_];
    const bool rst = a.first && a.first[(long)t * a.ft + (long)b * a.fb];
    f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (dv + j < a.Dv) v[j] = ld1(vp + (long)t * a.vt + j);
    const float keep = rst ? 0.f : expf(g);
    if (keep == 0.f) {  // also where S is not finite
#pragma unroll
      for (int p = 0; p < NP; ++p) S[p] = f4{0.f, 0.f, 0.f, 0.f};
    }
    float kk = 0.f, qq = 0.f, qk = 0.f;
    f4 ks = {0.f, 0.f, 0.f, 0.f}, qs = ks;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      kk = fmaf(k[p], k[p], kk);
      qq = fmaf(q[p], q[p], qq);
      qk = fmaf(q[p], k[p], qk);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ks[j] = fmaf(k[p], S[p][j], ks[j]);
        qs[j] = fmaf(q[p], S[p][j], qs[j]);
      }
    }
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) {
      kk += __shfl_xor(kk, o, 64);
      qq += __shfl_xor(qq, o, 64);
      qk += __shfl_xor(qk, o, 64);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ks[j] += __shfl_xor(ks[j], o, 64);
        qs[j] += __shfl_xor(qs[j], o, 64);
      }
    }
    const float rk = a.normalize ? 1.f / sqrtf(kk + a.eps) : 1.f, rq = a.normalize ? 1.f / sqrtf(qq + a.eps) : 1.f;
    const f4 u = be * (v - (keep * rk) * ks);
    const f4 y = (a.scale * rq) * (keep * qs + (qk * rk) * u);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const float kn = k[p] * rk;
#pragma unroll
      for (int j = 0; j < 4; ++j) S[p][j] = fmaf(kn, u[j], keep * S[p][j]);
    }
    if (rg == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (dv + j < a.Dv) st1(op + (long)t * BH * a.Dv + j, y[j]);
    }
  }
  if (rg == 0)
    for (int t = len; t < a.T; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (dv + j < a.Dv) st1(op + (long)t * BH * a.Dv + j, 0.f);
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int d = 8 * p + rg;
    if (d < a.Dk && live) {
      float* x = S2 + so + (long)d * a.Dv;
      if (VEC) __builtin_nontemporal_store(S[p], reinterpret_cast<f4*>(x));
      else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (dv + j < a.Dv) x[j] = S[p][j];
      }
    }
  }
}

template <typename T, bool VEC>
static void launch_v(const Args& a, void* out, float* S2, long sb, long sh, hipStream_t st) {
  const long items = (long)a.B * a.Hv * ((a.Dv + 31) / 32);
  const dim3 g((unsigned)((items + 3) / 4));
  T* o = reinterpret_cast<T*>(out);
  if (a.Dk <= 32) delta_step_kernel<T, 4, VEC><<<g, 256, 0, st>>>(a, o, S2, sb, sh);
  else if (a.Dk <= 64) delta_step_kernel<T, 8, VEC><<<g, 256, 0, st>>>(a, o, S2, sb, sh);
  else delta_step_kernel<T, 16, VEC><<<g, 256, 0, st>>>(a, o, S2, sb, sh);
}

void launch_delta_steps(const Args& a, void* out, float* S2, long sb, long sh, bool is_bf16, hipStream_t st) {
  const bool vec = a.Dv % 4 == 0 && sb % 4 == 0 && sh % 4 == 0 && reinterpret_cast<uintptr_t>(S2) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(a.state) % 16 == 0;
  if (is_bf16) {
    if (vec) launch_v<bf16, true>(a, out, S2, sb, sh, st);
    else launch_v<bf16, false>(a, out, S2, sb, sh, st);
  } else {
    if (vec) launch_v<float, true>(a, out, S2, sb, sh, st);
    else launch_v<float, false>(a, out, S2, sb, sh, st);
  }
}

}  // namespace delta
}  // namespace srl
