// Arguments and launchers of the gated delta rule (host side; the kernels: delta.h).
#pragma once
#include <hip/hip_runtime_api.h>
#include <stdint.h>

#include <atomic>

namespace srl {
namespace delta {

constexpr int MAXD = 128;        // head dimensions
inline __host__ __device__ int pitch(int Dv) { return Dv <= 64 ? 64 : 128; }  // of a row of value columns in the workspaces: Dvp below
constexpr float GONE = -104.0f;  // exp(g) rounds to zero in fp32 below this: the step forgets all that was before it

// More than 64 KB of LDS has to be asked for, once for each kernel and device.  A request that fails is made again by the next
// call; the launch after it reports the error.
struct AskedLds {
  std::atomic<uint64_t> done{0};
  void allow(const void* kernel, int bytes) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  }
};

struct Args {
  const void *q, *k, *v;
  const float *g, *beta;
  const uint8_t* first;   // [T, B] or null
  const int* lengths;     // [B] or null
  const float* state;     // [B, Hv, Dk, Dv] contiguous, or null (zeros)
  long qt, qb, qh, kt, kb, kh, vt, vb, vh, gt, gb, gh, bt, bb, bh_, ft, fb;  // element strides of t, b, head
  int T, B, Hk, Hv, Dk, Dv;
  int normalize, vecq, veck;
  float scale, eps;
  // plan: N chunks of C steps, in nseg segments of cps chunks
  int N, nseg, cps;
};

// What all value columns of a chunk of 64 steps share, from delta_pairs_kernel: the lower 16 x 16 tiles of A and P (10
// each, by rows) and the inverses of the diagonal blocks of I + A (4), row-major; then beta, gam, e, 1 / |q| and 1 / |k|.
constexpr int PAIR_TILES = 24, PAIR_A = 0, PAIR_P = 10, PAIR_T = 20, PAIR_FLOATS = PAIR_TILES * 256 + 5 * 64;

struct FwdOut {
  float* pairs;     // [BH, N, PAIR_FLOATS] (chunks of 64)
  void* out;        // [T, B, Hv, Dv] contiguous
  float* last;      // [B, Hv, Dk, Dv]
  float* Sc;        // [BH, N, DKp, Dvp] each chunk's first state, or null
  float* U;         // [BH, N, C, Dvp], or null
  float* Sseg;      // [BH, nseg, ceil(Dv / 16), DKp / 16, 64, 4] each segment's first state (nseg > 1), as the registers hold it
  float* Rseg;      // the same: a segment's last state from a zero first state
  // the map from a segment's first to its last state, tile by tile as the products that join segments read it (a wave's
  // read is 1 KB in a row): Pseg by rows, and transposed for the backward pass (or null)
  float *Pseg, *Ptr;  // [BH, nseg, DKp / 16, DKp / 16, 64, 4]
};

struct BwdArgs {
  const void* dout;  // [T, B, Hv, Dv] by strides, or null
  long ot, ob, oh;
  int vecv, vecg;  // v and dout can be read four at a time
  const float* dlast;  // [B, Hv, Dk, Dv] contiguous, or null
  const float *Sc, *U, *pairs, *Ptr;
  float* dSc;   // [BH, N, DKp, Dvp] gradient of each chunk's last state
  float* dR;    // [BH, N, C, Dvp]
  float* Xseg;   // as Rseg: the gradient of a segment's first state where that of its last is zero
  float* dSseg;  // as Sseg: the gradient of each segment's last state
  void *dq, *dk;  // contiguous: [T, B, Hk, Dk] in the inputs' type, or [T, B, Hv, Dk] in fp32, to be summed
  void* dv;
  float *dg, *db, *dstate;
};

void launch_delta_fwd(const Args& a, const FwdOut& o, int C, bool is_bf16, hipStream_t st);
void launch_delta_bwd(const Args& a, const BwdArgs& o, int C, bool is_bf16, bool per_value_head, hipStream_t st);
// S (or, rev, dS) at the segments' ends from that before the first step (or dlast), the maps P and X
void launch_delta_scan(const Args& a, const float* dlast, const float* P, const float* X, float* S, bool rev, hipStream_t st);
void launch_delta_head_sum(const float* xq, const float* xk, void* yq, void* yk, long rows, int rep, int Dk, bool is_bf16, hipStream_t st);
// delta_step.hip: the recurrent form; S2 (the state after it) may be a.state itself
void launch_delta_steps(const Args& a, void* out, float* S2, long sb, long sh, bool is_bf16, hipStream_t st);

}  // namespace delta
}  // namespace srl
