// The gated delta rule (gfx950): shared definitions of delta_step.hip, delta_fwd.hip and delta_bwd.hip.
//
// Per sequence b and value head h, with S [Dk, Dv] (S = 0 where first) and unit-length q, k:
//   S <- exp(g_t) S;  u_t = beta_t (v_t - S^T k_t);  S <- S + k_t u_t^T;  o_t = scale S^T q_t.
//
// The chunked form takes C steps at once.  With G_i the sum of g since the chunk's start, M_ij = exp(G_i - G_j)
// for j <= i with no reset between them (else 0), gam_i = what is left of the chunk's first state S0 at step i,
// e_j = M_{C-1,j}, A = tril(diag(beta) (M o K K^T), -1), P = scale M o Q K^T:
//   (I + A) U = diag(beta) (V - diag(gam) K S0),  O = scale diag(gam) Q S0 + P U,  S' = gam_C S0 + K^T diag(e) U.
// The columns of V, U, O and S never mix, so ONE WAVE OWNS 16 OF THEM: its strip of S, U and O stays in registers
// through the whole sequence, in the accumulator layout of v_mfma_f32_16x16x4_f32 (register r of lane l: row
// 4 (l/16) + r, column l%16).  That layout is also a B operand of the same instruction if the contraction index is
// taken in the order k = 16 m + 4 (l/16) + j, j = 0..3, for which the A operand is one 16-byte read of a row:
// products chain from registers to registers, and only K, Q, A and P, which all strips share, go through LDS.
#pragma once
#include <type_traits>

#include "common.h"
#include "delta_args.h"

namespace srl {
namespace delta {

typedef float f4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float bf2f(uint16_t h) { return __builtin_bit_cast(float, (uint32_t)h << 16); }
// round to nearest, ties to even (v_cvt_pk_bf16_f32)
typedef float f2_ __attribute__((ext_vector_type(2)));
typedef __bf16 b2_ __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t f2bf2(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_{lo, hi}), b2_));
}
__device__ __forceinline__ uint16_t f2bf(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
struct bf16 { uint16_t x; };
// the wave's number in its workgroup, in a scalar register: branches and addresses that go by it cost no vector registers
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const bf16* p) { return bf2f(p->x); }
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(bf16* p, float v) { p->x = f2bf(v); }

// N elements at a 16-byte (or N * size, if less) aligned address
template <int N>
__device__ __forceinline__ void ldv(const float* p, float* o) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f4 x = *reinterpret_cast<const f4*>(p + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i + j] = x[j];
    }
  } else {
    const float2 x = *reinterpret_cast<const float2*>(p);
    o[0] = x.x;
    o[1] = x.y;
  }
}
template <int N>
__device__ __forceinline__ void ldv(const bf16* p, float* o) {
  uint32_t w[N / 2];
  if constexpr (N == 8) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else if constexpr (N == 4) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x, w[1] = x.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    o[2 * i] = __builtin_bit_cast(float, w[i] << 16);
    o[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ f4 mfma4(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
// c += A B over 16 contraction indexes: a = A[row][4 (l/16) ..+3], b = the B operand's four registers
__device__ __forceinline__ f4 mm16(f4 a, f4 b, f4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = mfma4(a[j], b[j], c);
  return c;
}
__device__ __forceinline__ f4 row4(const float* p) { return *reinterpret_cast<const f4*>(p); }
// four rows of one column: the transposed operand
__device__ __forceinline__ f4 col4(const float* p, int ld) { return f4{p[0], p[ld], p[2 * ld], p[3 * ld]}; }

// What every step of a chunk has: cumulated decay, segment number, beta, gam, e; and 1 / |q|, 1 / |k|.
template <int C>
struct Gates {
  double G[C];
  int seg[C];
  float beta[C], gam[C], e[C], rq[C], rk[C];
  int rst[C];
};

// Lanes 0..C-1 of one wave: the chunk's gates.  A step that resets, or whose decay rounds to zero, starts a new
// segment and leaves its own g out of G: pairs of one segment only ever use differences of G, which are taken in
// 64 bits because a sum over the chunk may be large beside the difference.
template <int C>
__device__ __forceinline__ void chunk_gates(const Args& a, Gates<C>& s, int b, int h, int t0, int len, int lane) {
  const int i = lane, t = t0 + i;
  const bool ok = i < C && t < len;
  float g = 0.f, be = 0.f;
  bool rst = false;
  if (ok) {
    g = a.g[(long)t * a.gt + (long)b * a.gb + (long)h * a.gh];
    be = a.beta[(long)t * a.bt + (long)b * a.bb + (long)h * a.bh_];
    rst = (a.first && a.first[(long)t * a.ft + (long)b * a.fb]) || g <= GONE;
  }
  const unsigned long long m = __ballot(rst);
  double G = rst ? 0.0 : (double)g;
#pragma unroll
  for (int o = 1; o < C; o <<= 1) {
    const double x = __shfl_up(G, o, 64);
    if (lane >= o) G += x;
  }
  const int seg = __popcll(m & (~0ull >> (63 - lane)));
  const double Gl = __shfl(G, C - 1, 64);
  const int segl = __shfl(seg, C - 1, 64);
  if (i < C) {
    s.G[i] = G;
    s.seg[i] = seg;
    s.beta[i] = be;
    s.gam[i] = seg == 0 ? expf((float)G) : 0.f;
    s.e[i] = seg == segl ? expf((float)(Gl - G)) : 0.f;
    s.rst[i] = rst || !ok;
  }
}

// The state before the first step, which a reset there leaves unread, whatever it holds (gates of zero would not stop a NaN).
__device__ __forceinline__ const float* state_before(const Args& a, int b, int len) {
  return len > 0 && a.first && a.first[(long)b * a.fb] ? nullptr : a.state;
}

// A uniform value that the compiler does not carry over from one turn of a loop to the next: addresses that it would work out
// once and hold in registers through the whole walk (32 of 64 bits each, to no end but spills) are worked out again instead.
__device__ __forceinline__ long afresh(long x) {
  asm volatile("" : "+s"(x));
  return x;
}

// Reads that a wave has on their way must not hide behind branches or selects of their results (each would be waited for by
// itself): rows behind the end and columns past the width are read from the nearest that is there, and zeroed afterwards.
// There is a first step in any case.

// What scales a row of sum of squares ss to unit length.  Zero for rows behind the end, which are read as zeros: with eps = 0 their
// factor would be infinite, and a NaN in a row that does not count spoils the sums over the chunk.
__device__ __forceinline__ float unit_factor(float ss, bool live, bool normalize, float eps) {
  return !live ? 0.f : normalize ? 1.f / sqrtf(ss + eps) : 1.f;
}

// Rows t0.. of one head into LDS as fp32 [C][16 DKT + 4], scaled to unit length; 16 lanes a row, R rows a thread.
template <typename T, int DKT, int C, int R>
__device__ __forceinline__ void load_rows(float* dst, float* rn, const T* src, long st, int D, int t0, int len, bool vec,
                                          bool normalize, float eps) {
  constexpr int LD = 16 * DKT + 4, NE = DKT;
  const int sub = threadIdx.x & 15, c0 = sub * NE;
  float x[R][NE];
  const T* p[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = (threadIdx.x >> 4) + r * (blockDim.x >> 4);
    p[r] = src + (long)max(0, min(t0 + i, len - 1)) * st;
  }
  if (vec) {
#pragma unroll
    for (int r = 0; r < R; ++r) ldv<NE>(p[r] + min(c0, D - NE), x[r]);
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < NE; ++j) x[r][j] = ld1(p[r] + min(c0 + j, D - 1));
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = (threadIdx.x >> 4) + r * (blockDim.x >> 4);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      x[r][j] = (t0 + i < len && c0 + j < D) ? x[r][j] : 0.f;
      ss = fmaf(x[r][j], x[r][j], ss);
    }
    const float n = unit_factor(row16_sum(ss), t0 + i < len, normalize, eps);
    if (i < C) {
      float* d = dst + i * LD + c0;
#pragma unroll
      for (int j = 0; j < NE; ++j) d[j] = x[r][j] * n;
      if (sub == 0) rn[i] = n;
    }
  }
}

// A strip's values at the 64 (NT = 4) or 16 steps from t0 on: as they lie in memory, and as numbers
template <typename T, int NT>
struct Column {
  T raw[NT][4];
  __device__ __forceinline__ void fetch(const T* p, long st, int t0, int len, int kq) {
#pragma unroll
    for (int ti = 0; ti < NT; ++ti)
#pragma unroll
      for (int r = 0; r < 4; ++r) raw[ti][r] = p[(long)min(t0 + 16 * ti + 4 * kq + r, len - 1) * st];
  }
  __device__ __forceinline__ f4 get(int ti, int t0, int len, int kq, bool on) const {
    f4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = (on && t0 + 16 * ti + 4 * kq + r < len) ? ld1(&raw[ti][r]) : 0.f;
    return v;
  }
};

template <int C>
__device__ __forceinline__ float pair_decay(const Gates<C>& s, int i, int j, double Gi, int segi) {
  return (j <= i && s.seg[j] == segi) ? expf((float)(Gi - s.G[j])) : 0.f;
}

// tile t of the lower triangle of an NT x NT grid of 16 x 16 tiles, by rows
__device__ __forceinline__ void lower_tile(int t, int& ti, int& tj) {
  ti = t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0;
  tj = t - ti * (ti + 1) / 2;
}

// A chunk of 16: A = tril(diag(beta) (M o K K^T), -1) and P = scale M o Q K^T, a wave each where there are two.
constexpr int LT = 20;  // a row of a 16 x 16 tile in LDS
template <int DKT>
__device__ __forceinline__ void pair_tiles(const float* K, const float* Q, float* A, float* P, const Gates<16>& s, float scale,
                                           int wave, int nw) {
  constexpr int LD = 16 * DKT + 4;
  const int l16 = threadIdx.x & 15, kq = (threadIdx.x >> 4) & 3;
  for (int task = wave; task < 2; task += nw) {
    const float* kj = K + l16 * LD + 4 * kq;
    const float* xi = (task == 0 ? K : Q) + l16 * LD + 4 * kq;
    f4 d = {0.f, 0.f, 0.f, 0.f}, d2 = d;
#pragma unroll
    for (int m = 0; m < DKT; m += 2) {
      d = mm16(row4(kj + 16 * m), row4(xi + 16 * m), d);
      d2 = mm16(row4(kj + 16 * m + 16), row4(xi + 16 * m + 16), d2);
    }
    d += d2;
    const int i = l16, j0 = 4 * kq;
    const double Gi = s.G[i];
    const int segi = s.seg[i];
    const float be = s.beta[i];
    f4 o;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float m = pair_decay<16>(s, i, j0 + r, Gi, segi);
      o[r] = task == 0 ? (j0 + r < i ? be * m * d[r] : 0.f) : scale * m * d[r];
    }
    *reinterpret_cast<f4*>((task == 0 ? A : P) + i * LT + j0) = o;
  }
}

// One wave: the inverse of I + A for a chunk of 16, a column a lane, by forward substitution.
__device__ __forceinline__ void diag_inverse(const float* A, float* Td) {
  const int c = threadIdx.x & 63;
  if (c >= 16) return;
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float s = i == c ? 1.f : 0.f;
#pragma unroll
    for (int m4 = 0; m4 < i; m4 += 4) {
      const f4 r = row4(A + i * LT + m4);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (m4 + j < i) s = fmaf(-r[j], x[m4 + j], s);
    }
    x[i] = s;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) Td[i * LT + c] = x[i];
}

// A barrier for what goes through LDS: __syncthreads() would also wait for every store to memory on its way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ---------------------------------------------------------------- products of the strip kernels
// fp32 operands (K, Q, dO in fp32) take v_mfma_f32_16x16x4_f32: 64 operations a cycle and SIMD.  Where K, Q and dO are
// bf16 they are exact operands of v_mfma_f32_16x16x32_bf16 (1024 a cycle), and everything else is cut into three bf16 parts,
// x = p0 + p1 + p2 (8 bits each, so all 24 of x): an exact operand takes three products, two cut operands the six whose
// parts are not below 2^-24 of the largest.  fp32 sums throughout, so both forms round alike; two parts would be 2^-17 off.
typedef short s4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));  // not HIP's uint2: its union keeps operands out of registers
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

template <bool SP>
struct Op16;  // an operand over 16 contraction indexes, 4 a lane
template <>
struct Op16<false> {
  f4 x;
};
template <>
struct Op16<true> {
  u2 p0, p1, p2;
};
__device__ __forceinline__ u2 part(f4 x) { return u2{f2bf2(x[0], x[1]), f2bf2(x[2], x[3])}; }
__device__ __forceinline__ f4 rest(f4 x, u2 p) {
  return f4{x[0] - __builtin_bit_cast(float, p.x << 16), x[1] - __builtin_bit_cast(float, p.x & 0xffff0000u),
            x[2] - __builtin_bit_cast(float, p.y << 16), x[3] - __builtin_bit_cast(float, p.y & 0xffff0000u)};
}
__device__ __forceinline__ Op16<true> cut3(f4 x) {
  const u2 p0 = part(x);
  const f4 r = rest(x, p0);
  const u2 p1 = part(r);
  return {p0, p1, part(rest(r, p1))};
}
template <bool SP>
__device__ __forceinline__ Op16<SP> cut(f4 x) {
  if constexpr (SP) return cut3(x);
  else return Op16<false>{x};
}
template <bool SP>
struct Exact32;  // a K, Q or dO operand over 32 contraction indexes, 8 a lane
template <>
struct Exact32<false> {
  f4 a, b;
};
template <>
struct Exact32<true> {
  u4 x;
};
__device__ __forceinline__ b8 join(u2 a, u2 b) { return __builtin_bit_cast(b8, __builtin_shufflevector(a, b, 0, 1, 2, 3)); }
__device__ __forceinline__ f4 mfma32(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mm32(const Exact32<false>& a, const Op16<false>& b0, const Op16<false>& b1, f4 c) {
  return mm16(a.b, b1.x, mm16(a.a, b0.x, c));
}
__device__ __forceinline__ f4 mm32(const Exact32<true>& a, const Op16<true>& b0, const Op16<true>& b1, f4 c) {
  const b8 x = __builtin_bit_cast(b8, a.x);
  c = mfma32(x, join(b0.p2, b1.p2), c);
  c = mfma32(x, join(b0.p1, b1.p1), c);
  c = mfma32(x, join(b0.p0, b1.p0), c);
  return c;
}
// the exact operand on the right
__device__ __forceinline__ f4 mm32r(const Op16<false>& a0, const Op16<false>& a1, const Exact32<false>& b, f4 c) {
  return mm16(a1.x, b.b, mm16(a0.x, b.a, c));
}
__device__ __forceinline__ f4 mm32r(const Op16<true>& a0, const Op16<true>& a1, const Exact32<true>& b, f4 c) {
  const b8 x = __builtin_bit_cast(b8, b.x);
  c = mfma32(join(a0.p2, a1.p2), x, c);
  c = mfma32(join(a0.p1, a1.p1), x, c);
  c = mfma32(join(a0.p0, a1.p0), x, c);
  return c;
}
__device__ __forceinline__ f4 mm32x(const Exact32<false>& a, const Exact32<false>& b, f4 c) { return mm16(a.b, b.b, mm16(a.a, b.a, c)); }
__device__ __forceinline__ f4 mm32x(const Exact32<true>& a, const Exact32<true>& b, f4 c) {
  return mfma32(__builtin_bit_cast(b8, a.x), __builtin_bit_cast(b8, b.x), c);
}
// two cut operands over 32 indexes, and over 16
__device__ __forceinline__ f4 mm32(const Op16<false>& a0, const Op16<false>& a1, const Op16<false>& b0, const Op16<false>& b1, f4 c) {
  return mm16(a1.x, b1.x, mm16(a0.x, b0.x, c));
}
__device__ __forceinline__ f4 mm32(const Op16<true>& a0, const Op16<true>& a1, const Op16<true>& b0, const Op16<true>& b1, f4 c) {
  const b8 x0 = join(a0.p0, a1.p0), x1 = join(a0.p1, a1.p1), y0 = join(b0.p0, b1.p0), y1 = join(b0.p1, b1.p1);
  c = mfma32(join(a0.p2, a1.p2), y0, c);
  c = mfma32(x1, y1, c);
  c = mfma32(x0, join(b0.p2, b1.p2), c);
  c = mfma32(x1, y0, c);
  c = mfma32(x0, y1, c);
  c = mfma32(x0, y0, c);
  return c;
}
// c + a b over 16 indexes.  Cut operands are summed from zero and added to c by plain additions: the 16 x 16 x 16 product must
// not take over an accumulator that a 16 x 16 x 32 product has just written (the wait that this needs is not put in by the
// compiler, and the first two rows of each four came out wrong).
__device__ __forceinline__ f4 mm16o(const Op16<false>& a, const Op16<false>& b, f4 c) { return mm16(a.x, b.x, c); }
__device__ __forceinline__ f4 mm16o(const Op16<true>& a, const Op16<true>& b, f4 c) {
  const s4 x0 = __builtin_bit_cast(s4, a.p0), x1 = __builtin_bit_cast(s4, a.p1), y0 = __builtin_bit_cast(s4, b.p0), y1 = __builtin_bit_cast(s4, b.p1);
  f4 d = {0.f, 0.f, 0.f, 0.f};
  d = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, a.p2), y0, d, 0, 0, 0);
  d = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(x1, y1, d, 0, 0, 0);
  d = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(x0, __builtin_bit_cast(s4, b.p2), d, 0, 0, 0);
  d = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(x1, y0, d, 0, 0, 0);
  d = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(x0, y1, d, 0, 0, 0);
  d = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(x0, y0, d, 0, 0, 0);
  return c + d;
}

// f(0), ..., f(N - 1) with compile-time indexes: arrays of operands stay in registers
template <int I, int N, typename F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<I + 1, N>(f);
  }
}

// A chunk of 64 steps on its way from memory to LDS for the strip kernels: K (and Q) as they lie in memory, the pair tiles,
// the gates.  fetch() starts the reads for the next chunk, commit() writes what has arrived to LDS: the reads have the whole
// walk over the present chunk to arrive in, and are issued in three parts (K; Q; tiles and gates) between its products: all at
// once they queue up, and the waves with them, for 2000 to 5000 of a chunk's 17000 to 24000 cycles.  MODE: 0 forward,
// 1 forward without Q and P (maps), 2 backward, 3 without the tiles (gradients of q and k).
// What the kernels read: k(ti, m2), q(ti, m2): rows of steps against 32 key columns; kt(m, t2), qt(m, t2): rows of key columns
// against 32 steps; A (negated), P, Ti: tiles, transposed in the backward mode; rk4, rq4: factors that are not in k and q yet.
constexpr int TS = 320, TL = 20;  // a fp32 tile in LDS: 16 rows of 20: reads of rows and of columns are free of bank conflicts
template <typename T, int DKT, int NWT, int MODE>
struct Stage;

template <int MODE>
struct TileIndex {
  static constexpr int N = MODE == 3 ? 0 : MODE == 1 ? 14 : 24;
  static __device__ __forceinline__ int A(int ti, int tj) { return ti * (ti + 1) / 2 + tj; }
  static __device__ __forceinline__ int P(int ti, int tj) { return 10 + ti * (ti + 1) / 2 + tj; }
  static __device__ __forceinline__ int Ti(int ti) { return (MODE == 1 ? 10 : 20) + ti; }
  static __device__ __forceinline__ int source(int x) { return MODE == 1 && x >= 10 ? x + 10 : x; }  // in the pair data
};

template <int DKT, int NWT, int MODE>
struct Stage<float, DKT, NWT, MODE> {
  using TI = TileIndex<MODE>;
  static constexpr bool SP = false, HQ = MODE != 1;
  static constexpr int LD = 16 * DKT + 4, NE = DKT, RR = 16 / NWT, TH = 64 * NWT, NT4 = (TI::N * 64 + TH - 1) / TH;
  static constexpr int BYTES = 4 * ((HQ ? 2 : 1) * 64 * LD + TI::N * TS + 5 * 64);
  float *K, *Q, *tile, *gates;  // gates: beta, gam, e, rq, rk
  float rk_[RR][NE], rq_[HQ ? RR : 1][NE];
  float nk[RR], nq[RR];
  f4 tl[NT4 > 0 ? NT4 : 1], ga;
  int tid, l16, kq;

  __device__ __forceinline__ explicit Stage(void* lds)
      : K((float*)lds), Q(K + 64 * LD), tile(K + (HQ ? 2 : 1) * 64 * LD), gates(tile + TI::N * TS), tid(threadIdx.x), l16(threadIdx.x & 15),
        kq((threadIdx.x >> 4) & 3) {}
  // The lane's place, worked out afresh in each turn of a walk: see afresh().
  __device__ __forceinline__ void turn() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    tid = t, l16 = t & 15, kq = (t >> 4) & 3;
  }
  // all of a chunk at once
  template <typename T>
  __device__ __forceinline__ void fetch(const Args& a, const T* qp, const T* kp, const float* pair, int t0, int len) {
    each<0, 3>([&](auto part) { fetch(part, a, qp, kp, pair, t0, len); });
  }
  __device__ __forceinline__ Exact32<false> rows(const float* M, int ti, int m2) const {
    const float* p = M + (16 * ti + l16) * LD + 32 * m2 + 4 * kq;
    return {row4(p), row4(p + 16)};
  }
  __device__ __forceinline__ Exact32<false> cols(const float* M, int m, int t2) const {
    const float* p = M + (32 * t2 + 4 * kq) * LD + 16 * m + l16;
    return {col4(p, LD), col4(p + 16 * LD, LD)};
  }
  __device__ __forceinline__ Exact32<false> k(int ti, int m2) const { return rows(K, ti, m2); }
  __device__ __forceinline__ Exact32<false> q(int ti, int m2) const { return rows(Q, ti, m2); }
  __device__ __forceinline__ Exact32<false> kt(int m, int t2) const { return cols(K, m, t2); }
  __device__ __forceinline__ Exact32<false> qt(int m, int t2) const { return cols(Q, m, t2); }
  __device__ __forceinline__ Op16<false> tl_(int x) const {
    const float* p = tile + x * TS;
    return {MODE == 2 ? col4(p + 4 * kq * TL + l16, TL) : row4(p + l16 * TL + 4 * kq)};
  }
  __device__ __forceinline__ Op16<false> A(int ti, int tj) const { return tl_(TI::A(ti, tj)); }
  __device__ __forceinline__ Op16<false> P(int ti, int tj) const { return tl_(TI::P(ti, tj)); }
  __device__ __forceinline__ Op16<false> Ti(int ti) const { return tl_(TI::Ti(ti)); }
  __device__ __forceinline__ f4 beta(int ti) const { return row4(gates + 16 * ti + 4 * kq); }
  __device__ __forceinline__ f4 gam(int ti) const { return row4(gates + 64 + 16 * ti + 4 * kq); }
  __device__ __forceinline__ f4 e(int ti) const { return row4(gates + 128 + 16 * ti + 4 * kq); }
  __device__ __forceinline__ float gam_last() const { return gates[127]; }
  __device__ __forceinline__ f4 rk4(int) const { return f4{1.f, 1.f, 1.f, 1.f}; }
  __device__ __forceinline__ f4 rq4(int) const { return f4{1.f, 1.f, 1.f, 1.f}; }

  // four key columns from c on of step i, scaled to unit length
  __device__ __forceinline__ f4 k_of(int i, int c) const { return row4(K + i * LD + c); }
  __device__ __forceinline__ f4 q_of(int i, int c) const { return row4(Q + i * LD + c); }
  __device__ __forceinline__ void rows_(float (*w)[NE], const float* src, long st, int D, int t0, int len, bool vec) {
    const int c0 = (tid & 15) * NE;
    const float* p[RR];
#pragma unroll
    for (int r = 0; r < RR; ++r) p[r] = src + (long)min(t0 + (tid >> 4) + r * 4 * NWT, len - 1) * st;
    if (vec) {
#pragma unroll
      for (int r = 0; r < RR; ++r) ldv<NE>(p[r] + min(c0, D - NE), w[r]);
    } else {
#pragma unroll
      for (int r = 0; r < RR; ++r)
#pragma unroll
        for (int j = 0; j < NE; ++j) w[r][j] = p[r][min(c0 + j, D - 1)];
    }
  }
  template <int P>
  __device__ __forceinline__ void fetch(std::integral_constant<int, P>, const Args& a, const float* qp, const float* kp, const float* pair,
                                        int t0, int len) {
    if constexpr (P == 0) rows_(rk_, kp, a.kt, a.Dk, t0, len, a.veck);
    if constexpr (P == 1 && HQ) rows_(rq_, qp, a.qt, a.Dk, t0, len, a.vecq);
    if constexpr (P != 2) return;
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      const float* n = pair + PAIR_TILES * 256 + (tid >> 4) + r * 4 * NWT;
      nk[r] = n[256];
      if constexpr (HQ) nq[r] = n[192];
    }
#pragma unroll
    for (int x = 0; x < NT4; ++x) {
      const int at = min(tid + x * TH, TI::N * 64 - 1);  // 16 bytes each
      tl[x] = row4(pair + 256 * TI::source(at >> 6) + 4 * (at & 63));
    }
    ga = row4(pair + PAIR_TILES * 256 + 4 * min(tid, 79));
  }
  __device__ __forceinline__ void commit(int t0, int len, int D) {
    const int c0 = (tid & 15) * NE;
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      const int i = (tid >> 4) + r * 4 * NWT;
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        const bool in = t0 + i < len && c0 + j < D;
        K[i * LD + c0 + j] = in ? rk_[r][j] * nk[r] : 0.f;
        if constexpr (HQ) Q[i * LD + c0 + j] = in ? rq_[r][j] * nq[r] : 0.f;
      }
    }
#pragma unroll
    for (int x = 0; x < NT4; ++x) {
      const int at = tid + x * TH;
      if (at < TI::N * 64) *reinterpret_cast<f4*>(tile + (at >> 6) * TS + ((at >> 2) & 15) * TL + 4 * (at & 3)) = (at >> 6) < 10 ? -tl[x] : tl[x];
    }
    if (tid < 80) *reinterpret_cast<f4*>(gates + 4 * tid) = ga;
  }
};

// The place of contraction index c among a row's: the 8 that a lane takes of 32 lie together (16 m + 4 (l/16) + j, two m).
__device__ __forceinline__ int place(int c) { return (c & ~31) | ((c & 12) << 1) | ((c & 16) >> 2) | (c & 3); }

template <int DKT, int NWT, int MODE>
struct Stage<bf16, DKT, NWT, MODE> {
  using TI = TileIndex<MODE>;
  static constexpr bool SP = true, HQ = MODE != 1, QT = MODE >= 2;
  static constexpr int LR = 16 * DKT + 8, LC = 64 + 8, TH = 64 * NWT, NT4 = (TI::N * 64 + TH - 1) / TH;
  static constexpr int CP = 8 * DKT, RG = TH / CP < 16 ? TH / CP : 16, NG = 16 / RG;  // pairs of columns, groups of four rows at once, of a thread
  static constexpr int ROWS = 64 * LR, COLS = 16 * DKT * LC;
  static constexpr int BYTES = 2 * (ROWS + COLS + (HQ ? (QT ? COLS : ROWS) : 0)) + TI::N * 1536 + 5 * 64 * 4;
  uint16_t *Kr, *Kc, *Qx;
  u2* tile;   // [tile][part][lane]
  float* gates;  // beta, gam, e, rq, rk
  uint32_t rk_[NG][4], rq_[HQ ? NG : 1][4];
  f4 tl[NT4 > 0 ? NT4 : 1], ga;
  int tid, l16, kq;

  __device__ __forceinline__ explicit Stage(void* lds)
      : Kr((uint16_t*)lds), Kc(Kr + ROWS), Qx(Kc + COLS), tile((u2*)(Qx + (HQ ? (QT ? COLS : ROWS) : 0))),
        gates((float*)(tile + TI::N * 192)), tid(threadIdx.x), l16(threadIdx.x & 15), kq((threadIdx.x >> 4) & 3) {}
  // The lane's place, worked out afresh in each turn of a walk: see afresh().
  __device__ __forceinline__ void turn() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    tid = t, l16 = t & 15, kq = (t >> 4) & 3;
  }
  // all of a chunk at once
  template <typename T>
  __device__ __forceinline__ void fetch(const Args& a, const T* qp, const T* kp, const float* pair, int t0, int len) {
    each<0, 3>([&](auto part) { fetch(part, a, qp, kp, pair, t0, len); });
  }
  __device__ __forceinline__ Exact32<true> rows(const uint16_t* M, int ti, int m2) const {
    return {*reinterpret_cast<const u4*>(M + (16 * ti + l16) * LR + 32 * m2 + 8 * kq)};
  }
  __device__ __forceinline__ Exact32<true> cols(const uint16_t* M, int m, int t2) const {
    return {*reinterpret_cast<const u4*>(M + (16 * m + l16) * LC + 32 * t2 + 8 * kq)};
  }
  __device__ __forceinline__ Exact32<true> k(int ti, int m2) const { return rows(Kr, ti, m2); }
  __device__ __forceinline__ Exact32<true> q(int ti, int m2) const { return rows(Qx, ti, m2); }
  __device__ __forceinline__ Exact32<true> kt(int m, int t2) const { return cols(Kc, m, t2); }
  __device__ __forceinline__ Exact32<true> qt(int m, int t2) const { return cols(Qx, m, t2); }
  __device__ __forceinline__ Op16<true> tl_(int x) const {
    const u2* p = tile + x * 192 + 16 * kq + l16;
    return {p[0], p[64], p[128]};
  }
  __device__ __forceinline__ Op16<true> A(int ti, int tj) const { return tl_(TI::A(ti, tj)); }
  __device__ __forceinline__ Op16<true> P(int ti, int tj) const { return tl_(TI::P(ti, tj)); }
  __device__ __forceinline__ Op16<true> Ti(int ti) const { return tl_(TI::Ti(ti)); }
  __device__ __forceinline__ f4 beta(int ti) const { return row4(gates + 16 * ti + 4 * kq); }
  __device__ __forceinline__ f4 gam(int ti) const { return row4(gates + 64 + 16 * ti + 4 * kq); }
  __device__ __forceinline__ f4 e(int ti) const { return row4(gates + 128 + 16 * ti + 4 * kq); }
  __device__ __forceinline__ float gam_last() const { return gates[127]; }
  __device__ __forceinline__ f4 rq4(int ti) const { return row4(gates + 192 + 16 * ti + 4 * kq); }
  __device__ __forceinline__ f4 rk4(int ti) const { return row4(gates + 256 + 16 * ti + 4 * kq); }

  __device__ __forceinline__ f4 k_of(int i, int c) const {
    const u2 w = *reinterpret_cast<const u2*>(Kr + i * LR + place(c));
    const float n = gates[256 + i];
    return f4{n * __builtin_bit_cast(float, w.x << 16), n * __builtin_bit_cast(float, w.x & 0xffff0000u), n * __builtin_bit_cast(float, w.y << 16),
              n * __builtin_bit_cast(float, w.y & 0xffff0000u)};
  }
  __device__ __forceinline__ f4 q_of(int i, int c) const {  // Qx holds columns
    const uint16_t* p = Qx + c * LC + place(i);
    const float n = gates[192 + i];
    return f4{n * bf2f(p[0]), n * bf2f(p[LC]), n * bf2f(p[2 * LC]), n * bf2f(p[3 * LC])};
  }
  __device__ __forceinline__ void rows4(uint32_t (*w)[4], const bf16* src, long st, int D, int t0, int len, bool vec) {
    const int c = 2 * (tid % CP), i0 = 4 * (tid / CP < 16 ? tid / CP : 0);
    const bf16* p[NG][4];
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) p[g][r] = src + (long)min(t0 + i0 + 4 * g * RG + r, len - 1) * st;
    if (vec) {
      const int x = min(c, D - 2);
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) w[g][r] = *reinterpret_cast<const uint32_t*>(p[g][r] + x);
    } else {
      const int x = min(c, D - 1), y = min(c + 1, D - 1);
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) w[g][r] = (uint32_t)p[g][r][x].x | (uint32_t)p[g][r][y].x << 16;
    }
  }
  template <int P>
  __device__ __forceinline__ void fetch(std::integral_constant<int, P>, const Args& a, const bf16* qp, const bf16* kp, const float* pair,
                                        int t0, int len) {
    if constexpr (P == 0) rows4(rk_, kp, a.kt, a.Dk, t0, len, a.veck);
    if constexpr (P == 1 && HQ) rows4(rq_, qp, a.qt, a.Dk, t0, len, a.vecq);
    if constexpr (P != 2) return;
#pragma unroll
    for (int x = 0; x < NT4; ++x) {
      const int at = min(tid + x * TH, TI::N * 64 - 64 + (tid & 63));  // 64 divides TH: at & 63 is the lane
      const float* p = pair + 256 * TI::source(at >> 6);
      tl[x] = MODE == 2 ? col4(p + 4 * kq * 16 + l16, 16) : row4(p + 16 * l16 + 4 * kq);
    }
    ga = row4(pair + PAIR_TILES * 256 + 4 * min(tid, 79));
  }
  __device__ __forceinline__ void put_rows(uint16_t* M, const uint32_t* w, int i) {
    const int c = place(2 * (tid % CP));
#pragma unroll
    for (int r = 0; r < 4; ++r) *reinterpret_cast<uint32_t*>(M + (i + r) * LR + c) = w[r];
  }
  __device__ __forceinline__ void put_cols(uint16_t* M, const uint32_t* w, int i) {
    uint16_t* p = M + 2 * (tid % CP) * LC + place(i);
    *reinterpret_cast<u2*>(p) = u2{(w[0] & 0xffffu) | (w[1] << 16), (w[2] & 0xffffu) | (w[3] << 16)};
    *reinterpret_cast<u2*>(p + LC) = u2{(w[0] >> 16) | (w[1] & 0xffff0000u), (w[2] >> 16) | (w[3] & 0xffff0000u)};
  }
  __device__ __forceinline__ void commit(int t0, int len, int D) {
    const int g0 = tid / CP, c = 2 * (tid % CP);
    const uint32_t cm = c + 1 < D ? ~0u : c < D ? 0xffffu : 0u;
    if (g0 < 16) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int i = 4 * (g0 + g * RG);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t m = t0 + i + r < len ? cm : 0u;
          rk_[g][r] &= m;
          if constexpr (HQ) rq_[g][r] &= m;
        }
        put_rows(Kr, rk_[g], i);
        put_cols(Kc, rk_[g], i);
        if constexpr (HQ) {
          if constexpr (QT) put_cols(Qx, rq_[g], i);
          else put_rows(Qx, rq_[g], i);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < NT4; ++x) {
      const int at = tid + x * TH;
      if (at < TI::N * 64) {
        const Op16<true> o = cut3((at >> 6) < 10 ? -tl[x] : tl[x]);
        u2* p = tile + (at >> 6) * 192 + (at & 63);
        p[0] = o.p0, p[64] = o.p1, p[128] = o.p2;
      }
    }
    if (tid < 80) *reinterpret_cast<f4*>(gates + 4 * tid) = ga;
  }
};

// Between two parts of a walk: operands of the second are not read from LDS before the first is done, which would cost spills, and
// a reload from memory waits for everything that is on its way.
__device__ __forceinline__ void part_ends() { __builtin_amdgcn_sched_barrier(0); }

// c + sum over x = X..N-1 of tile(x) operand(x): pairs of tiles where there are two
template <int X, int N, typename FA, typename FB>
__device__ __forceinline__ f4 mm_tiles(FA&& tile, FB&& operand, f4 c) {
  if constexpr (X + 1 < N) {
    c = mm32(tile(X), tile(X + 1), operand(std::integral_constant<int, X>{}), operand(std::integral_constant<int, X + 1>{}), c);
    return mm_tiles<X + 2, N>(tile, operand, c);
  } else if constexpr (X < N) {
    return mm16o(tile(X), operand(std::integral_constant<int, X>{}), c);
  } else {
    return c;
  }
}

// See AskedLds.
template <auto F>
static void allow_lds(int bytes) {
  static AskedLds asked;
  asked.allow(reinterpret_cast<const void*>(F), bytes);
}

// LDS bytes of the kernels of a chunk of 16: the gates; K and Q; A, P and the inverse
template <int DKT>
constexpr size_t strip_lds() {
  return sizeof(Gates<16>) + sizeof(float) * (2 * 16 * (16 * DKT + 4) + 3 * 16 * LT);
}

}  // namespace delta
}  // namespace srl
