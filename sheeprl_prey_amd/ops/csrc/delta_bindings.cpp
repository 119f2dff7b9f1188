// Torch bindings of the gated delta rule (delta_*.hip) and the gated residual norms (residual_norm.hip).  Every
// operand's device, type, shape and strides are checked here against what the kernels index with; launches go to the current
// stream of the operands' device.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "delta_args.h"
#include "residual_norm.h"

namespace {

using torch::Tensor;
using OptT = c10::optional<Tensor>;

hipStream_t cur() { return c10::hip::getCurrentHIPStream().stream(); }
void launched(const char* name) {
  const hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, name, ": launch failed: ", hipGetErrorString(e));
}
bool has(const OptT& t) { return t.has_value() && t->defined(); }

void on(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, ": must be on ", like.device(), ", is on ", t.device());
}
void shape(const Tensor& t, c10::IntArrayRef s, const char* name) {
  TORCH_CHECK(t.sizes() == s, name, ": shape ", t.sizes(), ", expected ", s);
}

// q, k, v [T, B, H, D] with unit last stride, decay, beta [T, B, Hv] fp32, first [T, B] bytes, lengths [B] int32
srl::delta::Args delta_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay, const Tensor& beta,
                            const OptT& state, const OptT& first, const OptT& lengths, double scale, bool normalize, double eps) {
  using namespace srl::delta;
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "gated_delta: q, k, v [T, B, H, D]");
  TORCH_CHECK(q.scalar_type() == torch::kFloat32 || q.scalar_type() == torch::kBFloat16, "gated_delta: fp32 or bf16");
  const int64_t T = v.size(0), B = v.size(1), Hv = v.size(2), Dv = v.size(3), Hk = q.size(2), Dk = q.size(3);
  TORCH_CHECK(T >= 1 && B >= 1 && Hk >= 1 && Hv >= Hk && Hv % Hk == 0, "gated_delta: T, B >= 1 and Hv a multiple of Hk");
  TORCH_CHECK(Dk >= 1 && Dk <= MAXD && Dv >= 1 && Dv <= MAXD, "gated_delta: head dimensions 1..", MAXD);
  TORCH_CHECK(T < (1 << 24) && B * Hv < (1 << 20), "gated_delta: too many steps or heads");
  shape(q, {T, B, Hk, Dk}, "gated_delta q");
  shape(k, {T, B, Hk, Dk}, "gated_delta k");
  shape(decay, {T, B, Hv}, "gated_delta decay");
  shape(beta, {T, B, Hv}, "gated_delta beta");
  for (auto* t : {&q, &k, &v}) {
    on(*t, q, "gated_delta q, k, v");
    TORCH_CHECK(t->scalar_type() == q.scalar_type(), "gated_delta: q, k, v of one type");
    TORCH_CHECK(t->stride(3) == 1 || t->size(3) == 1, "gated_delta: unit last stride");
  }
  for (auto* t : {&decay, &beta}) {
    on(*t, q, "gated_delta decay, beta");
    TORCH_CHECK(t->scalar_type() == torch::kFloat32, "gated_delta: decay, beta fp32");
  }
  Args a{};
  a.q = q.data_ptr(), a.k = k.data_ptr(), a.v = v.data_ptr();
  a.g = decay.data_ptr<float>(), a.beta = beta.data_ptr<float>();
  a.qt = q.stride(0), a.qb = q.stride(1), a.qh = q.stride(2);
  a.kt = k.stride(0), a.kb = k.stride(1), a.kh = k.stride(2);
  a.vt = v.stride(0), a.vb = v.stride(1), a.vh = v.stride(2);
  a.gt = decay.stride(0), a.gb = decay.stride(1), a.gh = decay.stride(2);
  a.bt = beta.stride(0), a.bb = beta.stride(1), a.bh_ = beta.stride(2);
  if (has(first)) {
    on(*first, q, "gated_delta is_first");
    shape(*first, {T, B}, "gated_delta is_first");
    TORCH_CHECK(first->element_size() == 1, "gated_delta: is_first bool or uint8");
    a.first = reinterpret_cast<const uint8_t*>(first->data_ptr());
    a.ft = first->stride(0), a.fb = first->stride(1);
  }
  if (has(lengths)) {
    on(*lengths, q, "gated_delta lengths");
    shape(*lengths, {B}, "gated_delta lengths");
    TORCH_CHECK(lengths->scalar_type() == torch::kInt32 && lengths->is_contiguous(), "gated_delta: lengths int32, contiguous");
    a.lengths = lengths->data_ptr<int>();
  }
  if (has(state)) {
    on(*state, q, "gated_delta state");
    shape(*state, {B, Hv, Dk, Dv}, "gated_delta state");
    TORCH_CHECK(state->scalar_type() == torch::kFloat32, "gated_delta: state fp32");
    a.state = state->data_ptr<float>();
  }
  a.T = (int)T, a.B = (int)B, a.Hk = (int)Hk, a.Hv = (int)Hv, a.Dk = (int)Dk, a.Dv = (int)Dv;
  a.normalize = normalize, a.scale = (float)scale, a.eps = (float)eps;
  // wide reads of a row: 16 lanes take a sixteenth of the padded width each
  const int ne = Dk <= 32 ? 2 : Dk <= 64 ? 4 : 8, bytes = std::min<int>(16, ne * (int)q.element_size());
  auto wide = [&](const Tensor& t) {
    bool ok = Dk % ne == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0;
    for (int i = 0; i < 3; ++i) ok = ok && t.stride(i) * t.element_size() % bytes == 0;
    return ok;
  };
  a.vecq = wide(q), a.veck = wide(k);
  return a;
}

int dkp(int Dk) { return Dk <= 32 ? 32 : Dk <= 64 ? 64 : 128; }

// Chunks of 64 steps (16 where the whole sequence fits); a long axis is split into segments while the heads alone leave
// the 256 CUs idle.  Returns C.
int delta_plan(srl::delta::Args& a) {
  const int C = a.T <= 16 ? 16 : 64, BH = a.B * a.Hv;
  a.N = (a.T + C - 1) / C;
  a.nseg = 1;
  a.cps = a.N;
  if (a.N >= 8 && BH <= 128) {
    const int want = std::min(a.N / 2, std::max(2, 256 / BH));
    a.cps = (a.N + want - 1) / want;
    a.nseg = (a.N + a.cps - 1) / a.cps;
  }
  return C;
}

// -> {out, last, Sc, U, Pseg}; the last three (what the backward pass needs) are empty unless `save`
std::vector<Tensor> gated_delta_fwd(Tensor q, Tensor k, Tensor v, Tensor decay, Tensor beta, OptT state, OptT first, OptT lengths,
                                    double scale, bool normalize, double eps, bool save) {
  auto a = delta_args(q, k, v, decay, beta, state, first, lengths, scale, normalize, eps);
  if (a.state) TORCH_CHECK(state->is_contiguous(), "gated_delta: contiguous state");
  const c10::DeviceGuard guard(q.device());
  const int C = delta_plan(a), BH = a.B * a.Hv, DKp = dkp(a.Dk), Dvp = (a.Dv + 15) / 16 * 16;
  auto f = decay.options();
  auto out = torch::empty({a.T, a.B, a.Hv, a.Dv}, v.options());
  auto last = torch::empty({a.B, a.Hv, a.Dk, a.Dv}, f);
  Tensor Sc = torch::empty({0}, f), U = Sc, Ps = Sc, Ss, Rs;
  srl::delta::FwdOut o{};
  o.out = out.data_ptr(), o.last = last.data_ptr<float>();
  if (save) {
    Sc = torch::empty({BH, a.N, DKp, Dvp}, f);
    U = torch::empty({BH, a.N, C, Dvp}, f);
    o.Sc = Sc.data_ptr<float>(), o.U = U.data_ptr<float>();
  }
  if (a.nseg > 1) {
    Ss = torch::empty({BH, a.nseg, DKp, Dvp}, f);
    Rs = torch::empty({BH, a.nseg, DKp, Dvp}, f);
    Ps = torch::empty({BH, a.nseg, DKp, DKp}, f);
    o.Sseg = Ss.data_ptr<float>(), o.Rseg = Rs.data_ptr<float>(), o.Pseg = Ps.data_ptr<float>();
  }
  srl::delta::launch_delta_fwd(a, o, C, q.scalar_type() == torch::kBFloat16, cur());
  launched("gated_delta_fwd");
  return {out, last, Sc, U, Ps};
}

// -> {dq, dk, dv, ddecay, dbeta, dstate}
std::vector<Tensor> gated_delta_bwd(Tensor q, Tensor k, Tensor v, Tensor decay, Tensor beta, OptT state, OptT first, OptT lengths,
                                    double scale, bool normalize, double eps, Tensor Sc, Tensor U, Tensor Pseg, OptT dout,
                                    OptT dlast) {
  auto a = delta_args(q, k, v, decay, beta, state, first, lengths, scale, normalize, eps);
  const c10::DeviceGuard guard(q.device());
  const int C = delta_plan(a), BH = a.B * a.Hv, DKp = dkp(a.Dk), Dvp = (a.Dv + 15) / 16 * 16;
  shape(Sc, {BH, a.N, DKp, Dvp}, "gated_delta_bwd states");
  shape(U, {BH, a.N, C, Dvp}, "gated_delta_bwd updates");
  auto f = decay.options();
  srl::delta::BwdArgs o{};
  if (has(dout)) {
    on(*dout, q, "gated_delta_bwd dout");
    shape(*dout, {a.T, a.B, a.Hv, a.Dv}, "gated_delta_bwd dout");
    TORCH_CHECK(dout->scalar_type() == q.scalar_type() && (dout->stride(3) == 1 || a.Dv == 1), "gated_delta_bwd: dout's type, unit last stride");
    o.dout = dout->data_ptr();
    o.ot = dout->stride(0), o.ob = dout->stride(1), o.oh = dout->stride(2);
  }
  if (has(dlast)) {
    on(*dlast, q, "gated_delta_bwd dlast");
    shape(*dlast, {a.B, a.Hv, a.Dk, a.Dv}, "gated_delta_bwd dlast");
    TORCH_CHECK(dlast->scalar_type() == torch::kFloat32 && dlast->is_contiguous(), "gated_delta_bwd: dlast fp32, contiguous");
    o.dlast = dlast->data_ptr<float>();
  }
  auto dSc = torch::empty({BH, a.N, DKp, Dvp}, f), dR = torch::empty({BH, a.N, C, Dvp}, f);
  Tensor X, dSs;
  if (a.nseg > 1) {
    shape(Pseg, {BH, a.nseg, DKp, DKp}, "gated_delta_bwd maps");
    X = torch::empty({BH, a.nseg, DKp, Dvp}, f);
    dSs = torch::empty({BH, a.nseg, DKp, Dvp}, f);
    o.Pseg = Pseg.data_ptr<float>(), o.Xseg = X.data_ptr<float>(), o.dSseg = dSs.data_ptr<float>();
  }
  const bool shared = a.Hk != a.Hv, bf = q.scalar_type() == torch::kBFloat16;
  auto dq = torch::empty({a.T, a.B, a.Hk, a.Dk}, q.options()), dk = torch::empty_like(dq);
  auto dv = torch::empty({a.T, a.B, a.Hv, a.Dv}, q.options());
  auto dg = torch::empty({a.T, a.B, a.Hv}, f), db = torch::empty({a.T, a.B, a.Hv}, f);
  auto ds = torch::empty({a.B, a.Hv, a.Dk, a.Dv}, f);
  Tensor dqh, dkh;
  if (shared) {
    dqh = torch::empty({a.T, a.B, a.Hv, a.Dk}, f);
    dkh = torch::empty({a.T, a.B, a.Hv, a.Dk}, f);
  }
  o.Sc = Sc.data_ptr<float>(), o.U = U.data_ptr<float>();
  o.dSc = dSc.data_ptr<float>(), o.dR = dR.data_ptr<float>();
  o.dq = shared ? dqh.data_ptr() : dq.data_ptr();
  o.dk = shared ? dkh.data_ptr() : dk.data_ptr();
  o.dv = dv.data_ptr(), o.dg = dg.data_ptr<float>(), o.db = db.data_ptr<float>(), o.dstate = ds.data_ptr<float>();
  srl::delta::launch_delta_bwd(a, o, C, bf, shared, cur());
  if (shared) {
    const long rows = (long)a.T * a.B * a.Hk;
    srl::delta::launch_delta_head_sum(dqh.data_ptr<float>(), dq.data_ptr(), rows, a.Hv / a.Hk, a.Dk, bf, cur());
    srl::delta::launch_delta_head_sum(dkh.data_ptr<float>(), dk.data_ptr(), rows, a.Hv / a.Hk, a.Dk, bf, cur());
  }
  launched("gated_delta_bwd");
  return {dq, dk, dv, dg, db, ds};
}

// The recurrent form over all T steps: out [T, B, Hv, Dv]; the state after them goes to state_out (which may be state)
Tensor gated_delta_steps(Tensor q, Tensor k, Tensor v, Tensor decay, Tensor beta, OptT state, OptT first, OptT lengths, double scale,
                         bool normalize, double eps, Tensor state_out) {
  auto a = delta_args(q, k, v, decay, beta, state, first, lengths, scale, normalize, eps);
  const c10::DeviceGuard guard(q.device());
  on(state_out, q, "gated_delta state");
  shape(state_out, {a.B, a.Hv, a.Dk, a.Dv}, "gated_delta state");
  TORCH_CHECK(state_out.scalar_type() == torch::kFloat32, "gated_delta: state fp32");
  TORCH_CHECK((state_out.stride(3) == 1 || a.Dv == 1) && (state_out.stride(2) == a.Dv || a.Dk == 1), "gated_delta: state [B, Hv, Dk, Dv] with contiguous [Dk, Dv]");
  if (a.state) TORCH_CHECK(state->strides() == state_out.strides(), "gated_delta: the states before and after have the same strides");
  auto out = torch::empty({a.T, a.B, a.Hv, a.Dv}, v.options());
  srl::delta::launch_delta_steps(a, out.data_ptr(), state_out.data_ptr<float>(), state_out.stride(0), state_out.stride(1),
                                 q.scalar_type() == torch::kBFloat16, cur());
  launched("gated_delta_steps");
  return out;
}

// ------------------------------------------------------------------ gated residual norms
const float* par(const OptT& t, const Tensor& x, const char* name) {
  if (!has(t)) return nullptr;
  on(*t, x, name);
  TORCH_CHECK(t->scalar_type() == torch::kFloat32 && t->is_contiguous() && t->dim() == 1 && t->size(0) == x.size(1), name,
              ": fp32 [", x.size(1), "], contiguous");
  return t->data_ptr<float>();
}

// rows [R, D] with unit last stride; clears `vec` if 16 bytes at a time cannot be read
void rows_of(const Tensor& t, const Tensor& x, const char* name, const void** p, long* stride, bool* vec) {
  on(t, x, name);
  TORCH_CHECK(t.scalar_type() == x.scalar_type() && t.sizes() == x.sizes() && (t.stride(1) == 1 || t.size(1) == 1), name,
              ": rows like x with unit last stride");
  const int n = 16 / (int)t.element_size();
  *p = t.data_ptr();
  *stride = t.stride(0);
  *vec = *vec && x.size(1) % n == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && t.stride(0) % n == 0;
}

srl::rnorm::Args norm_args(const Tensor& x, const Tensor& h, const OptT& gate, const OptT& scale, const OptT& pw, const OptT& pb,
                           const OptT& rw, const OptT& rb, bool layer, int64_t act, double eps, double s1, bool* vec) {
  TORCH_CHECK(x.dim() == 2 && (x.scalar_type() == torch::kFloat32 || x.scalar_type() == torch::kBFloat16),
              "gated_residual_norm: rows [R, D] in fp32 or bf16");
  TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= srl::rnorm::MAXD, "gated_residual_norm: 1..", srl::rnorm::MAXD, " columns");
  TORCH_CHECK(x.size(0) >= 1 && x.size(0) < (1ll << 31) - 64, "gated_residual_norm: 1..2^31 rows");
  srl::rnorm::Args a{};
  *vec = true;
  rows_of(x, x, "gated_residual_norm x", &a.x, &a.xs, vec);
  rows_of(h, x, "gated_residual_norm h", &a.h, &a.hs, vec);
  if (has(gate)) rows_of(*gate, x, "gated_residual_norm gate", &a.gate, &a.gs, vec);
  a.scale = par(scale, x, "gated_residual_norm scale");
  a.pw = par(pw, x, "gated_residual_norm post_weight"), a.pb = par(pb, x, "gated_residual_norm post_bias");
  a.rw = par(rw, x, "gated_residual_norm pre_weight"), a.rb = par(rb, x, "gated_residual_norm pre_bias");
  a.rows = (int)x.size(0), a.D = (int)x.size(1), a.layer = layer, a.act = (int)act;
  a.eps = (float)eps, a.inv_d = 1.f / (float)x.size(1), a.s1 = (float)s1;
  return a;
}

std::vector<Tensor> residual_norm_fwd(Tensor x, Tensor h, OptT gate, OptT scale, OptT pw, OptT pb, OptT rw, OptT rb, bool layer,
                                      int64_t act, double eps, double s1) {
  bool vec;
  auto a = norm_args(x, h, gate, scale, pw, pb, rw, rb, layer, act, eps, s1, &vec);
  const c10::DeviceGuard guard(x.device());
  auto y = torch::empty({x.size(0), x.size(1)}, x.options()), u = torch::empty_like(y);
  a.y = y.data_ptr(), a.u = u.data_ptr();
  srl::rnorm::launch_residual_norm_fwd(a, x.scalar_type() == torch::kBFloat16, vec, cur());
  launched("residual_norm_fwd");
  return {y, u};
}

// -> {dx, dh, dgate (empty without a gate), sums [5, D]: dscale, dpost_weight, dpost_bias, dpre_weight, dpre_bias}
std::vector<Tensor> residual_norm_bwd(Tensor x, Tensor h, OptT gate, OptT scale, OptT pw, OptT pb, OptT rw, OptT rb, bool layer,
                                      int64_t act, double eps, double s1, OptT dy, OptT du) {
  bool vec;
  auto a = norm_args(x, h, gate, scale, pw, pb, rw, rb, layer, act, eps, s1, &vec);
  const c10::DeviceGuard guard(x.device());
  srl::rnorm::BwdArgs o{};
  if (has(dy)) rows_of(*dy, x, "gated_residual_norm dy", &o.dy, &o.dys, &vec);
  if (has(du)) rows_of(*du, x, "gated_residual_norm du", &o.du, &o.dus, &vec);
  auto dx = torch::empty({x.size(0), x.size(1)}, x.options()), dh = torch::empty_like(dx);
  auto dg = has(gate) ? torch::empty_like(dx) : torch::empty({0}, x.options());
  auto f = x.options().dtype(torch::kFloat32);
  auto sums = torch::empty({5, x.size(1)}, f);
  auto part = torch::empty({srl::rnorm::residual_norm_groups(a.rows, a.D), 4, x.size(1)}, f);
  o.dx = dx.data_ptr(), o.dh = dh.data_ptr(), o.dgate = has(gate) ? dg.data_ptr() : nullptr, o.part = part.data_ptr<float>();
  srl::rnorm::launch_residual_norm_bwd(a, o, sums.data_ptr<float>(), x.scalar_type() == torch::kBFloat16, vec, cur());
  launched("residual_norm_bwd");
  return {dx, dh, dg, sums};
}

}  // namespace

void register_delta(pybind11::module& m) {
  m.def("gated_delta_fwd", &gated_delta_fwd);
  m.def("gated_delta_bwd", &gated_delta_bwd);
  m.def("gated_delta_steps", &gated_delta_steps);
  m.def("residual_norm_fwd", &residual_norm_fwd);
  m.def("residual_norm_bwd", &residual_norm_bwd);
}
