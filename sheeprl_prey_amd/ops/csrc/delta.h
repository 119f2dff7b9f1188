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
#include <atomic>

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

// Rows t0.. of one head into LDS as fp32 [C][16 DKT + 4], scaled to unit length; 16 lanes a row.
template <typename T, int DKT, int C>
__device__ __forceinline__ void load_rows(float* dst, float* rn, const T* src, long st, int D, int t0, int len, bool vec,
                                          bool normalize, float eps) {
  constexpr int LD = 16 * DKT + 4, NE = DKT;
  const int sub = threadIdx.x & 15, c0 = sub * NE;
  for (int i = threadIdx.x >> 4; i < C; i += blockDim.x >> 4) {
    const bool ok = t0 + i < len;
    float x[NE];
#pragma unroll
    for (int j = 0; j < NE; ++j) x[j] = 0.f;
    if (ok) {
      const T* p = src + (long)(t0 + i) * st + c0;
      if (vec) {
        if (c0 < D) ldv<NE>(p, x);
      } else {
#pragma unroll
        for (int j = 0; j < NE; ++j)
          if (c0 + j < D) x[j] = ld1(p + j);
      }
    }
    float r = 1.f;
    if (normalize) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < NE; ++j) ss = fmaf(x[j], x[j], ss);
      r = 1.f / sqrtf(row16_sum(ss) + eps);
    }
    float* d = dst + i * LD + c0;
#pragma unroll
    for (int j = 0; j < NE; ++j) d[j] = x[j] * r;
    if (sub == 0) rn[i] = r;
  }
}

template <int C>
__device__ __forceinline__ float pair_decay(const Gates<C>& s, int i, int j, double Gi, int segi) {
  return (j <= i && s.seg[j] == segi) ? expf((float)(Gi - s.G[j])) : 0.f;
}

// tile t of the lower triangle of an NT x NT grid of 16 x 16 tiles, by rows
__device__ __forceinline__ void lower_tile(int t, int& ti, int& tj) {
  ti = t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0;
  tj = t - ti * (ti + 1) / 2;
}

// A = tril(diag(beta) (M o K K^T), -1) and, with Q, P = scale M o Q K^T, lower tiles only, one tile a wave at a time.
template <int DKT, int C>
__device__ __forceinline__ void pair_tiles(const float* K, const float* Q, float* A, float* P, const Gates<C>& s, float scale,
                                           int wave, int nw) {
  constexpr int LD = 16 * DKT + 4, LC = C + 4, NT = C / 16, NTL = NT * (NT + 1) / 2;
  const int l16 = threadIdx.x & 15, kq = (threadIdx.x >> 4) & 3;
  const int n = Q ? 2 * NTL : NTL;
  for (int task = wave; task < n; task += nw) {
    int ti, tj;
    lower_tile(task < NTL ? task : task - NTL, ti, tj);
    const float* kj = K + (16 * tj + l16) * LD + 4 * kq;
    const float* xi = (task < NTL ? K : Q) + (16 * ti + l16) * LD + 4 * kq;
    f4 d = {0.f, 0.f, 0.f, 0.f}, d2 = d;
#pragma unroll
    for (int m = 0; m < DKT; m += 2) {
      d = mm16(row4(kj + 16 * m), row4(xi + 16 * m), d);
      d2 = mm16(row4(kj + 16 * m + 16), row4(xi + 16 * m + 16), d2);
    }
    d += d2;
    const int i = 16 * ti + l16, j0 = 16 * tj + 4 * kq;
    const double Gi = s.G[i];
    const int segi = s.seg[i];
    const float be = s.beta[i];
    f4 o;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float m = pair_decay<C>(s, i, j0 + r, Gi, segi);
      o[r] = task < NTL ? (j0 + r < i ? be * m * d[r] : 0.f) : scale * m * d[r];
    }
    *reinterpret_cast<f4*>((task < NTL ? A : P) + i * LC + j0) = o;
  }
}

// One wave: the inverses of the 16 x 16 diagonal blocks of I + A, a column a lane, by forward substitution.
constexpr int LT = 20;
template <int C>
__device__ __forceinline__ void diag_inverse(const float* A, float* Td) {
  constexpr int LC = C + 4, NT = C / 16;
  const int c = threadIdx.x & 15, q = (threadIdx.x >> 4) & 3;
  if (q >= NT) return;
  const float* a = A + 16 * q * (LC + 1);
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float s = i == c ? 1.f : 0.f;
#pragma unroll
    for (int m4 = 0; m4 < i; m4 += 4) {
      const f4 r = row4(a + i * LC + m4);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (m4 + j < i) s = fmaf(-r[j], x[m4 + j], s);
    }
    x[i] = s;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) Td[(16 * q + i) * LT + c] = x[i];
}

// A barrier for what goes through LDS: __syncthreads() would also wait for every store to memory on its way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A chunk of 64 steps on its way from memory to LDS for the strip kernels: K (and Q) as they lie in memory, the pair tiles,
// the gates.  fetch() starts the reads for the next chunk, commit() writes what has arrived to LDS: the reads have the whole
// walk over the present chunk to arrive in.
constexpr int TS = 320, TL = 20;  // a tile in LDS: 16 rows of 20: reads of rows and of columns are free of bank conflicts
template <typename T, int DKT, int NWT, bool QP>
struct Stage {
  static constexpr int LD = 16 * DKT + 4, NE = DKT, RR = 16 / NWT, TH = 64 * NWT;
  static constexpr int NB = NE * (int)sizeof(T) / 4, TILES = QP ? PAIR_TILES : 14, NT4 = (TILES * 64 + TH - 1) / TH;
  static constexpr int FLOATS = (QP ? 2 : 1) * 64 * LD + TILES * TS + 3 * 64;
  float *K, *Q, *tile, *gates;  // gates: beta, gam, e
  uint32_t rk_[RR][NB], rq_[QP ? RR : 1][NB];
  float nk[RR], nq[RR];
  f4 tl[NT4], ga;

  __device__ __forceinline__ explicit Stage(float* lds) : K(lds), Q(lds + 64 * LD), tile(lds + (QP ? 2 : 1) * 64 * LD), gates(tile + TILES * TS) {}
  // tile x of A (x = 0..9 by rows), P and T
  __device__ __forceinline__ const float* A(int ti, int tj) const { return tile + (ti * (ti + 1) / 2 + tj) * TS; }
  __device__ __forceinline__ const float* P(int ti, int tj) const { return tile + (10 + ti * (ti + 1) / 2 + tj) * TS; }
  __device__ __forceinline__ const float* Ti(int ti) const { return tile + ((QP ? 20 : 10) + ti) * TS; }

  __device__ __forceinline__ void row(uint32_t* w, const T* p, int D, bool ok, bool vec) {
    const int c0 = (threadIdx.x & 15) * NE;
#pragma unroll
    for (int j = 0; j < NB; ++j) w[j] = 0;
    if (!ok || c0 >= D) return;
    if (vec) {
      if constexpr (NB >= 4) {
#pragma unroll
        for (int j = 0; j < NB; j += 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p + c0) + j);
          w[j] = x.x, w[j + 1] = x.y, w[j + 2] = x.z, w[j + 3] = x.w;
        }
      } else if constexpr (NB == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(p + c0);
        w[0] = x.x, w[1] = x.y;
      } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p + c0);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NE; ++j)
        if (c0 + j < D) {
          if constexpr (sizeof(T) == 4) w[j] = __builtin_bit_cast(uint32_t, p[c0 + j]);
          else w[j / 2] |= (uint32_t)p[c0 + j].x << (16 * (j & 1));
        }
    }
  }
  __device__ __forceinline__ void fetch(const Args& a, const T* qp, const T* kp, const float* pair, int t0, int len) {
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      const int i = (threadIdx.x >> 4) + r * 4 * NWT;
      row(rk_[r], kp + (long)(t0 + i) * a.kt, a.Dk, t0 + i < len, a.veck);
      nk[r] = pair[PAIR_TILES * 256 + 256 + i];
      if constexpr (QP) {
        row(rq_[r], qp + (long)(t0 + i) * a.qt, a.Dk, t0 + i < len, a.vecq);
        nq[r] = pair[PAIR_TILES * 256 + 192 + i];
      }
    }
#pragma unroll
    for (int x = 0; x < NT4; ++x) {
      const int at = threadIdx.x + x * TH;  // 16 bytes each
      if (at < TILES * 64) tl[x] = row4(pair + 4 * (QP || at < 640 ? at : at + 640));
    }
    if (threadIdx.x < 48) ga = row4(pair + PAIR_TILES * 256 + 4 * threadIdx.x);
  }
  __device__ __forceinline__ void put(float* d, const uint32_t* w, float n) {
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      float x;
      if constexpr (sizeof(T) == 4) x = __builtin_bit_cast(float, w[j]);
      else x = __builtin_bit_cast(float, j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
      d[j] = x * n;
    }
  }
  __device__ __forceinline__ void commit() {
    const int c0 = (threadIdx.x & 15) * NE;
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      const int i = (threadIdx.x >> 4) + r * 4 * NWT;
      put(K + i * LD + c0, rk_[r], nk[r]);
      if constexpr (QP) put(Q + i * LD + c0, rq_[r], nq[r]);
    }
#pragma unroll
    for (int x = 0; x < NT4; ++x) {
      const int at = threadIdx.x + x * TH;
      if (at < TILES * 64) *reinterpret_cast<f4*>(tile + (at >> 6) * TS + ((at >> 2) & 15) * TL + 4 * (at & 3)) = tl[x];
    }
    if (threadIdx.x < 48) *reinterpret_cast<f4*>(gates + 4 * threadIdx.x) = ga;
  }
};

// More than 64 KB of LDS has to be asked for, once for each kernel and device.
template <auto F>
static void allow_lds(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  (void)hipGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return;
  (void)hipFuncSetAttribute(reinterpret_cast<const void*>(F), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  done.fetch_or(bit, std::memory_order_relaxed);
}

// LDS bytes of the strip kernels
template <int DKT, int C>
constexpr size_t strip_lds(bool q) {
  return sizeof(float) * ((q ? 2 : 1) * C * (16 * DKT + 4) + (q ? 2 : 1) * C * (C + 4) + C * LT) + sizeof(Gates<C>);
}

}  // namespace delta
}  // namespace srl
