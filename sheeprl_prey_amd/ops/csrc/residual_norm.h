// Arguments and launchers of the gated residual norms (host side; the kernels: residual_norm.hip).
#pragma once
#include <hip/hip_runtime_api.h>

namespace srl {
namespace rnorm {

constexpr int MAXD = 8192;  // row width

struct Args {
  const void *x, *h, *gate;  // rows of D, element strides between rows
  long xs, hs, gs;
  const float *scale, *pw, *pb, *rw, *rb;  // [D] or null (s1 for scale, 1 for pw and rw, 0 for pb and rb)
  void *y, *u;                             // [rows, D] contiguous
  int rows, D, layer, act;                 // act: ACT_NONE / ACT_SILU / 5 = sigmoid; gate null: 1
  float eps, inv_d, s1;  // s1: the scale where `scale` is null
};

struct BwdArgs {
  const void *dy, *du;  // rows of D by strides; either may be null
  long dys, dus;
  void *dx, *dh, *dgate;  // [rows, D] contiguous; dgate null without a gate
  float* part;            // [workgroups, 4, D]: sums of g act norm(h), g act, du norm(y), du
};

constexpr int SIGMOID = 5;

int residual_norm_groups(int rows, int D);
void launch_residual_norm_fwd(const Args& a, bool is_bf16, bool vec, hipStream_t st);
void launch_residual_norm_bwd(const Args& a, const BwdArgs& o, float* sums, bool is_bf16, bool vec, hipStream_t st);

}  // namespace rnorm
}  // namespace srl
