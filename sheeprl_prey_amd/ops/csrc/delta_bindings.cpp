// Torch bindings of the gated delta rule (delta_*.hip) and the gated residual norms (residual_norm.hip).  Every
// operand's device, type, shape and strides are checked here against what the kernels index with; launches go to the current
// stream of the operands' device.
#include <torch/extension.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <torch/csrc/autograd/functions/basic_ops.h>

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

void on(const Tensor& t, const Tensor& like) {
  TORCH_CHECK_VALUE(t.device() == like.device(), "every operand must be on ", like.device(), ", got ", t.device());
}
void shape(const Tensor& t, c10::IntArrayRef s, const char* name) {
  TORCH_CHECK_VALUE(t.sizes() == s, name, " must be ", s, ", got ", t.sizes());
}
bool two_types(const Tensor& t) { return t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16; }
Tensor unit_last(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
Tensor f32(const Tensor& t) { return t.scalar_type() == torch::kFloat32 ? t : t.to(torch::kFloat32); }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
OptT opt_of(const Tensor& t) { return t.defined() ? OptT(t) : OptT(); }
Tensor val(const OptT& t) { return has(t) ? *t : Tensor(); }
const float* fp(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

// The gradients of an operator that is differentiable once: a second differentiation raises an error.
void once(torch::autograd::variable_list& g, const char* name) {
  if (!at::GradMode::is_enabled()) return;
  torch::autograd::variable_list in;
  std::vector<size_t> at;
  for (size_t i = 0; i < g.size(); ++i)
    if (g[i].defined()) {
      in.push_back(g[i].detach().requires_grad_());
      at.push_back(i);
    }
  auto err = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " is differentiable once", (int64_t)in.size());
  auto out = (*err)(std::move(in));
  for (size_t j = 0; j < at.size(); ++j) g[at[j]] = out[j];
}

// A captured backward pass would have to wait for the default stream if an eager autograd graph that ran there still holds a
// leaf of it; a capture does not allow that, and the error ends the process from the engine's thread.  It is refused here,
// where the operands themselves are the leaves.
void capturable(std::initializer_list<const Tensor*> operands, const char* name) {
  for (const Tensor* t : operands) {
    if (!wants(*t) || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!node || !node->stream().has_value() || node->stream()->id() != 0) continue;
    TORCH_CHECK(c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None, name,
                ": a leaf of this captured pass belongs to an autograd graph of the default stream that is still alive: drop that graph first");
  }
}

// ------------------------------------------------------------------ gated delta rule
// What every entry takes, checked: q, k [T, B, Hk, Dk], v [T, B, Hv, Dv] (a single step comes as T = 1) of one type,
// decay, beta [T, B, Hv], state [B, Hv, Dk, Dv] fp32, first [T, B], lengths [B].
void delta_check(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay, const Tensor& beta, const Tensor& state,
                 int lead) {
  const char* where = lead == 2 ? "[T, B, heads, dim]" : "[B, heads, dim]";
  TORCH_CHECK_VALUE(q.dim() == lead + 2 && k.dim() == lead + 2 && v.dim() == lead + 2, "q, k, v must be ", where, ", got ", q.sizes(), ", ",
                    k.sizes(), ", ", v.sizes());
  TORCH_CHECK_VALUE(q.sizes() == k.sizes() && q.sizes().slice(0, lead) == v.sizes().slice(0, lead),
                    "q and k must have one shape and v their leading sizes: ", q.sizes(), ", ", k.sizes(), ", ", v.sizes());
  const int64_t Hk = q.size(lead), Dk = q.size(lead + 1), Hv = v.size(lead), Dv = v.size(lead + 1), B = v.size(lead - 1);
  TORCH_CHECK_VALUE(Hk >= 1 && Hv >= Hk && Hv % Hk == 0, "the value heads (", Hv, ") must be a multiple of the key heads (", Hk, ")");
  TORCH_CHECK_VALUE(Dk >= 1 && Dk <= srl::delta::MAXD && Dv >= 1 && Dv <= srl::delta::MAXD, "head dimensions must be 1..",
                    srl::delta::MAXD, ", got ", Dk, " and ", Dv);
  TORCH_CHECK_VALUE((lead == 1 || v.size(0) <= (1 << 24)) && B * Hv <= (1 << 20), "at most 2^24 steps and 2^20 states, got ", v.sizes());
  TORCH_CHECK_VALUE(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), "q, k, v must have one type, got ",
                    q.scalar_type(), ", ", k.scalar_type(), ", ", v.scalar_type());
  TORCH_CHECK_VALUE(two_types(v), "q, k, v must be float32 or bfloat16, got ", v.scalar_type());
  shape(decay, v.sizes().slice(0, lead + 1), "decay and beta");
  shape(beta, v.sizes().slice(0, lead + 1), "decay and beta");
  TORCH_CHECK_VALUE(decay.is_floating_point() && beta.is_floating_point(), "decay and beta must be floating point");
  for (auto* t : {&q, &k, &decay, &beta}) on(*t, v);
  if (state.defined()) {
    shape(state, {B, Hv, Dk, Dv}, "state");
    TORCH_CHECK_VALUE(state.scalar_type() == torch::kFloat32, "state must be float32, got ", state.scalar_type());
    on(state, v);
  }
}

Tensor delta_first(const OptT& x, c10::IntArrayRef s, const Tensor& like) {
  if (!has(x)) return Tensor();
  Tensor f = x->dim() == (int64_t)s.size() + 1 && x->size(-1) == 1 ? x->squeeze(-1) : *x;
  shape(f, s, "is_first");
  on(f, like);
  return f.scalar_type() == torch::kBool || f.scalar_type() == torch::kUInt8 ? f : f.ne(0);
}

Tensor delta_lengths(const OptT& x, int64_t B, int64_t T, const Tensor& like) {
  if (!has(x)) return Tensor();
  TORCH_CHECK_VALUE(x->dim() == 1 && x->size(0) == B && (x->scalar_type() == torch::kInt32 || x->scalar_type() == torch::kInt64),
                    "lengths must be int32 or int64 [", B, "], got ", x->scalar_type(), " ", x->sizes());
  on(*x, like);
  // the kernels clamp to 0..T; 64 bits are clamped before they are cut to 32, which would turn a length of 2^31 into a negative one
  return x->scalar_type() == torch::kInt32 ? x->contiguous() : x->clamp(0, T).to(torch::kInt32).contiguous();
}

struct DeltaOpts {
  double scale, eps;
  bool normalize;
};

// operands as delta_check and the conversions above leave them, each with a unit last stride; single steps (lead = 1) come
// without the time axis
srl::delta::Args delta_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay, const Tensor& beta,
                            const Tensor& first, const Tensor& lengths, const DeltaOpts& o, int lead = 2) {
  using namespace srl::delta;
  Args a{};
  a.q = q.data_ptr(), a.k = k.data_ptr(), a.v = v.data_ptr();
  a.g = decay.data_ptr<float>(), a.beta = beta.data_ptr<float>();
  const int i = lead - 1;  // the batch axis
  a.qb = q.stride(i), a.qh = q.stride(i + 1), a.kb = k.stride(i), a.kh = k.stride(i + 1), a.vb = v.stride(i), a.vh = v.stride(i + 1);
  a.gb = decay.stride(i), a.gh = decay.stride(i + 1), a.bb = beta.stride(i), a.bh_ = beta.stride(i + 1);
  if (lead == 2) a.qt = q.stride(0), a.kt = k.stride(0), a.vt = v.stride(0), a.gt = decay.stride(0), a.bt = beta.stride(0);
  if (first.defined()) {
    a.first = reinterpret_cast<const uint8_t*>(first.data_ptr());
    a.fb = first.stride(i);
    if (lead == 2) a.ft = first.stride(0);
  }
  if (lengths.defined()) a.lengths = lengths.data_ptr<int>();
  a.T = lead == 2 ? (int)v.size(0) : 1, a.B = (int)v.size(i), a.Hk = (int)q.size(i + 1), a.Hv = (int)v.size(i + 1), a.Dk = (int)q.size(i + 2),
  a.Dv = (int)v.size(i + 2);
  a.normalize = o.normalize, a.scale = (float)o.scale, a.eps = (float)o.eps;
  // wide reads of a row: 16 lanes take a sixteenth of the padded width each
  const int Dk = a.Dk, ne = Dk <= 32 ? 2 : Dk <= 64 ? 4 : 8, bytes = std::min<int>(16, ne * (int)q.element_size());
  auto wide = [&](const Tensor& t) {
    bool ok = Dk % ne == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0;
    for (int d = 0; d <= lead; ++d) ok = ok && t.stride(d) * t.element_size() % bytes == 0;
    return ok;
  };
  a.vecq = wide(q), a.veck = wide(k);
  return a;
}

int dkp(int Dk) { return Dk <= 32 ? 32 : Dk <= 64 ? 64 : 128; }

// Chunks of 64 steps, or one of 16 where the whole sequence fits (16 steps x 128 x 2 heads of 32, forward and backward: 30 us
// and 58 us as a chunk of 64; x 16 x 16 of 128: 73 and 89).  An axis of 8 chunks or more is split into segments while the
// heads alone leave two thirds of the 256 CUs idle; the segments' maps cost as much as the walk itself.  Forward over 1024
// steps with and without segments: 48 heads of 128 133 and 177 us, 64 heads 157 and 181, 80 heads 189 and 190, 96 heads (two
// segments) 216 and 191; 64 heads of 64 105 and 158.  512 steps of 8 heads: 70 and 93; 256 steps of 16 heads of 64: 50 and 48.
// Returns C.
int delta_plan(srl::delta::Args& a) {
  const int C = a.T <= 16 ? 16 : 64, BH = a.B * a.Hv;
  a.N = (a.T + C - 1) / C;
  a.nseg = 1;
  a.cps = a.N;
  if (a.N >= 8 && 256 / BH >= 3) {
    const int want = std::min(a.N / 2, 256 / BH);
    a.cps = (a.N + want - 1) / want;
    a.nseg = (a.N + a.cps - 1) / a.cps;
  }
  return C;
}

// One allocation for several fp32 workspaces, each on a 256-byte boundary
struct Workspace {
  int64_t n = 0;
  int64_t add(int64_t count) {
    const int64_t at = n;
    n += (count + 63) / 64 * 64;
    return at;
  }
  Tensor make(const Tensor& like) const { return torch::empty({n}, like.options().dtype(torch::kFloat32)); }
};

// the maps of all segments
int64_t map_floats(const srl::delta::Args& a) { return (int64_t)a.B * a.Hv * a.nseg * dkp(a.Dk) * dkp(a.Dk); }

// What a forward pass leaves for the backward pass, in one workspace: Sc, U, the transposed maps, pairs
struct DeltaSaved {
  int64_t Sc, U, P, pairs, n;
  DeltaSaved(const srl::delta::Args& a, int C) {
    const int64_t BH = (int64_t)a.B * a.Hv, DKp = dkp(a.Dk), Dvp = srl::delta::pitch(a.Dv);
    Workspace w;
    Sc = w.add(BH * a.N * DKp * Dvp);
    U = w.add(BH * a.N * C * Dvp);
    P = w.add(a.nseg > 1 ? map_floats(a) : 0);
    pairs = w.add(C == 64 ? BH * a.N * srl::delta::PAIR_FLOATS : 0);
    n = w.n;
  }
};

// -> {out, last} and, in `saved` if it is not null, what the backward pass needs
std::pair<Tensor, Tensor> delta_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay, const Tensor& beta,
                                        const Tensor& state, const Tensor& first, const Tensor& lengths, const DeltaOpts& opt,
                                        Tensor* saved) {
  auto a = delta_args(q, k, v, decay, beta, first, lengths, opt);
  a.state = fp(state);
  const c10::DeviceGuard guard(q.device());
  const int C = delta_plan(a);
  const int64_t BH = (int64_t)a.B * a.Hv, DKp = dkp(a.Dk), Dvp = srl::delta::pitch(a.Dv);
  auto out = torch::empty({a.T, a.B, a.Hv, a.Dv}, v.options());
  auto last = torch::empty({a.B, a.Hv, a.Dk, a.Dv}, decay.options());
  srl::delta::FwdOut o{};
  o.out = out.data_ptr(), o.last = last.data_ptr<float>();
  const DeltaSaved at(a, C);
  if (saved) {
    *saved = torch::empty({at.n}, decay.options());
    float* p = saved->data_ptr<float>();
    o.Sc = p + at.Sc, o.U = p + at.U, o.pairs = p + at.pairs;
    if (a.nseg > 1) o.Ptr = p + at.P;
  }
  Tensor ws;
  if (a.nseg > 1 || !saved) {
    Workspace w;
    const int64_t segs = a.nseg > 1 ? BH * a.nseg * DKp : 0, s = w.add(segs * Dvp), r = w.add(segs * Dvp);
    const int64_t m = w.add(segs ? map_floats(a) : 0), pr = w.add(!saved && C == 64 ? BH * a.N * srl::delta::PAIR_FLOATS : 0);
    ws = w.make(q);
    float* p = ws.data_ptr<float>();
    o.Sseg = p + s, o.Rseg = p + r, o.Pseg = p + m;
    if (!saved) o.pairs = p + pr;
  }
  srl::delta::launch_delta_fwd(a, o, C, q.scalar_type() == torch::kBFloat16, cur());
  launched("gated_delta");
  return {out, last};
}

struct GatedDeltaFn : public torch::autograd::Function<GatedDeltaFn> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, Tensor q, Tensor k, Tensor v, Tensor decay, Tensor beta,
                                                OptT state, OptT first_, OptT lengths_, double scale, bool normalize, double eps,
                                                bool want_state) {
    Tensor saved;
    const Tensor first = val(first_), lengths = val(lengths_);
    auto r = delta_forward(q, k, v, decay, beta, val(state), first, lengths, DeltaOpts{scale, eps, normalize}, &saved);
    ctx->save_for_backward({q, k, v, decay, beta, first, lengths, saved});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["normalize"] = normalize;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["want_state"] = want_state;
    ctx->set_materialize_grads(false);
    return {r.first, r.second};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list g(12);
    Tensor dout = grads[0], dlast = grads[1];
    if (!dout.defined() && !dlast.defined()) return g;
    const auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2], &decay = s[3], &beta = s[4];
    auto a = delta_args(q, k, v, decay, beta, s[5], s[6],
                        DeltaOpts{ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["normalize"].toBool()});
    const c10::DeviceGuard guard(q.device());
    const int C = delta_plan(a);
    const int64_t BH = (int64_t)a.B * a.Hv, DKp = dkp(a.Dk), Dvp = srl::delta::pitch(a.Dv);
    srl::delta::BwdArgs o{};
    if (dout.defined()) {
      dout = unit_last(dout);
      o.dout = dout.data_ptr();
      o.ot = dout.stride(0), o.ob = dout.stride(1), o.oh = dout.stride(2);
    }
    if (dlast.defined()) {
      dlast = dlast.contiguous();
      o.dlast = dlast.data_ptr<float>();
    }
    auto fours = [&](const Tensor& t) {
      const int64_t e = t.element_size(), m = 4 * e;
      bool ok = a.Dv % 4 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % m == 0;
      for (int i = 0; i < 3; ++i) ok = ok && t.stride(i) * e % m == 0;
      return ok;
    };
    o.vecv = fours(v);
    o.vecg = dout.defined() ? fours(dout) : o.vecv;
    const DeltaSaved at(a, C);
    TORCH_CHECK(s[7].numel() == at.n, "gated_delta: the plan changed between the passes");
    const float* sp = s[7].data_ptr<float>();
    o.Sc = sp + at.Sc, o.U = sp + at.U, o.pairs = sp + at.pairs, o.Ptr = sp + at.P;
    // dq and dk of shared key heads: one workgroup a key head where heads are wide (delta_grads_kernel) and fill the 256 CUs
    // twice so (4096 steps x 2 x 8: the separate sums cost 54 us more), else one a value head and a sum
    const bool shared = a.Hk != a.Hv && (C == 16 || a.Dk <= 64 || (int64_t)a.B * a.Hk * a.N < 512), bf = q.scalar_type() == torch::kBFloat16;
    Workspace w;
    const int64_t segs = a.nseg > 1 ? BH * a.nseg * DKp * Dvp : 0, heads = shared ? (int64_t)a.T * BH * a.Dk : 0;
    const int64_t ds = w.add(BH * a.N * DKp * Dvp), dr = w.add(BH * a.N * C * Dvp), x = w.add(segs), dss = w.add(segs), hq = w.add(heads),
                  hk = w.add(heads);
    const Tensor ws = w.make(q);
    float* p = ws.data_ptr<float>();
    o.dSc = p + ds, o.dR = p + dr, o.Xseg = p + x, o.dSseg = p + dss;
    auto dq = torch::empty({a.T, a.B, a.Hk, a.Dk}, q.options()), dk = torch::empty({a.T, a.B, a.Hk, a.Dk}, q.options());
    auto dv = torch::empty({a.T, a.B, a.Hv, a.Dv}, q.options());
    auto dg = torch::empty({a.T, a.B, a.Hv}, decay.options()), db = torch::empty({a.T, a.B, a.Hv}, decay.options());
    o.dq = shared ? (void*)(p + hq) : dq.data_ptr();
    o.dk = shared ? (void*)(p + hk) : dk.data_ptr();
    o.dv = dv.data_ptr(), o.dg = dg.data_ptr<float>(), o.db = db.data_ptr<float>();
    if (ctx->saved_data["want_state"].toBool()) {
      g[5] = torch::empty({a.B, a.Hv, a.Dk, a.Dv}, decay.options());
      o.dstate = g[5].data_ptr<float>();
    }
    srl::delta::launch_delta_bwd(a, o, C, bf, shared, cur());
    if (shared) {
      const long rows = (long)a.T * a.B * a.Hk;
      srl::delta::launch_delta_head_sum(p + hq, p + hk, dq.data_ptr(), dk.data_ptr(), rows, a.Hv / a.Hk, a.Dk, bf, cur());
    }
    launched("gated_delta backward");
    g[0] = dq, g[1] = dk, g[2] = dv, g[3] = dg, g[4] = db;
    once(g, "gated_delta");
    return g;
  }
};

// The recurrent form over all steps; the state after them goes to `after` (which may be `state`)
Tensor delta_steps(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay, const Tensor& beta, const Tensor& state,
                   const Tensor& first, const Tensor& lengths, const DeltaOpts& opt, const Tensor& after, int lead) {
  auto a = delta_args(q, k, v, decay, beta, first, lengths, opt, lead);
  a.state = fp(state);
  const c10::DeviceGuard guard(q.device());
  auto out = torch::empty(v.sizes(), v.options());
  srl::delta::launch_delta_steps(a, out.data_ptr(), after.data_ptr<float>(), after.stride(0), after.stride(1),
                                 q.scalar_type() == torch::kBFloat16, cur());
  launched("gated_delta");
  return out;
}

// Up to this many steps without a gradient the recurrent kernel is taken, whose time goes with the steps.  Against a chunk of 16,
// in a graph over four states in turn: 64 x 16 heads of 128 in fp32 4 steps 39 and 46 us, 6 steps 47 and 47, 8 steps 55 and 47,
// in bf16 2 steps 39 and 46, 3 steps 48 and 46, 4 steps 59 and 46; 64 x 8 heads of 64 in fp32 3 steps 12.4 and 13.3, 4 steps
// 14.1 and 13.4; 256 x 2 heads of 32 in fp32 4 steps 8.7 and 9.7, 6 steps 11.1 and 9.7.  The forms cross at 4 to 6 steps in fp32
// and at 3 in bf16.
constexpr int RECURRENT_MAX_STEPS = 4;

std::pair<Tensor, Tensor> gated_delta(Tensor q, Tensor k, Tensor v, Tensor decay, Tensor beta, OptT state_, OptT first_, OptT lengths_,
                                      c10::optional<double> scale, bool normalize, double eps) {
  Tensor state = val(state_);
  delta_check(q, k, v, decay, beta, state, 2);
  const int64_t T = v.size(0), B = v.size(1);
  const Tensor first = delta_first(first_, {T, B}, v), lengths = delta_lengths(lengths_, B, T, v);
  const DeltaOpts opt{scale.has_value() ? *scale : 1.0 / std::sqrt((double)q.size(3)), eps, normalize};
  q = unit_last(q), k = unit_last(k), v = unit_last(v), decay = f32(decay), beta = f32(beta);
  if (state.defined()) state = state.contiguous();
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v) || wants(decay) || wants(beta) || wants(state))) {
    capturable({&q, &k, &v, &decay, &beta, &state}, "gated_delta");
    auto r = GatedDeltaFn::apply(q, k, v, decay, beta, opt_of(state), opt_of(first), opt_of(lengths), opt.scale, normalize, eps, wants(state));
    return {r[0], r[1]};
  }
  if (T <= RECURRENT_MAX_STEPS) {
    auto last = torch::empty({B, v.size(2), q.size(3), v.size(3)}, decay.options());
    auto out = delta_steps(q, k, v, decay, beta, state, first, lengths, opt, last, 2);
    return {out, last};
  }
  return delta_forward(q, k, v, decay, beta, state, first, lengths, opt, nullptr);
}

// Whether an operand shares memory with one of the states, outer and inner their leading axes by stride.  Where either has gaps
// (a slice of a larger store), every run of the operand is looked up among the states, which lie one behind the other.
bool lies_in(const Tensor& t, const Tensor& state, int64_t outer, int64_t inner) {
  const auto o = at::get_overlap_status(state, t);
  if (o != at::MemOverlapStatus::TooHard) return o != at::MemOverlapStatus::No;
  if (!t.is_alias_of(state)) return false;
  const int64_t e = state.element_size(), n1 = state.size(outer), n2 = state.size(inner), s1 = state.stride(outer) * e, s2 = state.stride(inner) * e,
                one = state.size(2) * state.size(3) * e;
  const char* base = static_cast<const char*>(state.const_data_ptr());
  auto hit = [&](const char* p, int64_t n) {  // the last state that begins before the end of the n bytes: does it reach into them?
    const int64_t r = p - base, z = r + n - 1;
    if (z < 0) return false;
    const int64_t i = n1 > 1 ? std::min(z / s1, n1 - 1) : 0, rest = z - i * (n1 > 1 ? s1 : 0), j = n2 > 1 ? std::min(rest / s2, n2 - 1) : 0;
    return i * (n1 > 1 ? s1 : 0) + j * (n2 > 1 ? s2 : 0) + one > r;
  };
  const int64_t te = t.element_size(), nd = t.dim(), last = t.size(-1);
  const bool runs = last == 1 || t.stride(-1) == 1;
  std::vector<int64_t> at(nd, 0);
  const char* p = static_cast<const char*>(t.const_data_ptr());
  while (true) {
    if (hit(p, runs ? last * te : te)) return true;
    int64_t d = runs ? nd - 2 : nd - 1;  // the next run, or element
    for (; d >= 0; --d) {
      p += t.stride(d) * te;
      if (++at[d] < t.size(d)) break;
      p -= at[d] * t.stride(d) * te;
      at[d] = 0;
    }
    if (d < 0) return false;
  }
}

Tensor gated_delta_step(Tensor q, Tensor k, Tensor v, Tensor decay, Tensor beta, Tensor state, OptT first_, c10::optional<double> scale,
                        bool normalize, double eps) {
  delta_check(q, k, v, decay, beta, state, 1);
  TORCH_CHECK(!at::GradMode::is_enabled() ||
                  !(wants(q) || wants(k) || wants(v) || wants(decay) || wants(beta) || wants(state)),
              "gated_delta_step updates the state in place and has no gradient: use gated_delta, or torch.no_grad()");
  const int64_t B = state.size(0), Hv = state.size(1), Dk = state.size(2), Dv = state.size(3);
  const Tensor first = delta_first(first_, {B}, v);
  TORCH_CHECK_VALUE((Dv == 1 || state.stride(3) == 1) && (Dk == 1 || state.stride(2) == Dv),
                    "each [Dk, Dv] of the state must be contiguous, got strides ", state.strides());
  int64_t d0 = 0, d1 = 1;
  if (B > 1 && Hv > 1 && state.stride(0) < state.stride(1)) std::swap(d0, d1);
  // d1 the inner of the two leading axes
  if (B == 1) std::swap(d0, d1);
  int64_t least = Dk * Dv;
  for (int64_t d : {d1, d0}) {
    if (state.size(d) <= 1) continue;
    TORCH_CHECK_VALUE(state.stride(d) >= least, "the states must not overlap, got strides ", state.strides());
    least = state.stride(d) * state.size(d);
  }
  for (const Tensor* t : std::initializer_list<const Tensor*>{&q, &k, &v, &decay, &beta, &first})
    TORCH_CHECK_VALUE(!t->defined() || !lies_in(*t, state, d0, d1), "no operand may lie in the state that is updated");
  const DeltaOpts opt{scale.has_value() ? *scale : 1.0 / std::sqrt((double)Dk), eps, normalize};
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return delta_steps(unit_last(q), unit_last(k), unit_last(v), f32(decay), f32(beta), state, first, Tensor(), opt, state, 1);
}

// ------------------------------------------------------------------ gated residual norms
// rows of the last axis with unit stride, by a view where there is one
Tensor rows2d(const Tensor& t) {
  const int64_t D = t.size(-1);
  if (t.dim() == 2) return unit_last(t);
  if (t.is_contiguous()) return t.view({-1, D});
  return unit_last(t.reshape({-1, D}));
}

// clears `vec` if 16 bytes at a time cannot be read
void rows_of(const Tensor& t, const void** p, long* stride, bool* vec) {
  const int n = 16 / (int)t.element_size();
  *p = t.data_ptr();
  *stride = t.stride(0);
  *vec = *vec && t.size(1) % n == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && t.stride(0) % n == 0;
}

struct NormOpts {
  bool layer;
  int64_t act;
  double eps, s1;
};

// x, h, gate as rows; the weights fp32 [D], contiguous, or undefined
srl::rnorm::Args norm_args(const Tensor& x, const Tensor& h, const Tensor& gate, const Tensor& scale, const Tensor& pw, const Tensor& pb,
                           const Tensor& rw, const Tensor& rb, const NormOpts& o, bool* vec) {
  srl::rnorm::Args a{};
  *vec = true;
  rows_of(x, &a.x, &a.xs, vec);
  rows_of(h, &a.h, &a.hs, vec);
  if (gate.defined()) rows_of(gate, &a.gate, &a.gs, vec);
  a.scale = fp(scale), a.pw = fp(pw), a.pb = fp(pb), a.rw = fp(rw), a.rb = fp(rb);
  a.rows = (int)x.size(0), a.D = (int)x.size(1), a.layer = o.layer, a.act = (int)o.act;
  a.eps = (float)o.eps, a.inv_d = 1.f / (float)x.size(1), a.s1 = (float)o.s1;
  return a;
}

std::pair<Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& h, const Tensor& gate, const Tensor& scale, const Tensor& pw,
                                       const Tensor& pb, const Tensor& rw, const Tensor& rb, const NormOpts& o) {
  bool vec;
  const Tensor x2 = rows2d(x), h2 = rows2d(h), g2 = gate.defined() ? rows2d(gate) : gate;
  auto a = norm_args(x2, h2, g2, scale, pw, pb, rw, rb, o, &vec);
  const c10::DeviceGuard guard(x.device());
  auto y = torch::empty(x.sizes(), x.options()), u = torch::empty(x.sizes(), x.options());
  a.y = y.data_ptr(), a.u = u.data_ptr();
  srl::rnorm::launch_residual_norm_fwd(a, x.scalar_type() == torch::kBFloat16, vec, cur());
  launched("gated_residual_norm");
  return {y, u};
}

struct ResidualNormFn : public torch::autograd::Function<ResidualNormFn> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, Tensor x, Tensor h, OptT gate_, OptT scale_, OptT pw_,
                                                OptT pb_, OptT rw_, OptT rb_, bool layer, int64_t act, double eps, double s1,
                                                int64_t want) {
    const Tensor gate = val(gate_), scale = val(scale_), pw = val(pw_), pb = val(pb_), rw = val(rw_), rb = val(rb_);
    auto r = norm_forward(x, h, gate, scale, pw, pb, rw, rb, NormOpts{layer, act, eps, s1});
    ctx->save_for_backward({x, h, gate, scale, pw, pb, rw, rb});
    ctx->saved_data["layer"] = layer;
    ctx->saved_data["act"] = act;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["s1"] = s1;
    ctx->saved_data["want"] = want;
    ctx->set_materialize_grads(false);
    return {r.first, r.second};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list g(13);
    if (!grads[0].defined() && !grads[1].defined()) return g;
    const int64_t want = ctx->saved_data["want"].toInt();
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &gate = s[2];
    bool vec;
    const Tensor x2 = rows2d(x), h2 = rows2d(s[1]), g2 = gate.defined() ? rows2d(gate) : gate;
    auto a = norm_args(x2, h2, g2, s[3], s[4], s[5], s[6], s[7],
                       NormOpts{ctx->saved_data["layer"].toBool(), ctx->saved_data["act"].toInt(), ctx->saved_data["eps"].toDouble(),
                                ctx->saved_data["s1"].toDouble()},
                       &vec);
    const c10::DeviceGuard guard(x.device());
    srl::rnorm::BwdArgs o{};
    Tensor dy, du;
    if (grads[0].defined()) {
      dy = rows2d(grads[0]);
      rows_of(dy, &o.dy, &o.dys, &vec);
    }
    if (grads[1].defined()) {
      du = rows2d(grads[1]);
      rows_of(du, &o.du, &o.dus, &vec);
    }
    g[0] = torch::empty(x.sizes(), x.options());
    g[1] = torch::empty(x.sizes(), x.options());
    if (want & 1) g[2] = torch::empty(x.sizes(), x.options());
    const auto f = x.options().dtype(torch::kFloat32);
    const Tensor sums = torch::empty({5, a.D}, f), part = torch::empty({srl::rnorm::residual_norm_groups(a.rows, a.D), 4, a.D}, f);
    o.dx = g[0].data_ptr(), o.dh = g[1].data_ptr(), o.dgate = g[2].defined() ? g[2].data_ptr() : nullptr, o.part = part.data_ptr<float>();
    srl::rnorm::launch_residual_norm_bwd(a, o, sums.data_ptr<float>(), x.scalar_type() == torch::kBFloat16, vec, cur());
    launched("gated_residual_norm backward");
    for (int i = 0; i < 5; ++i)
      if (want >> (i + 1) & 1) g[3 + i] = sums.select(0, i);
    once(g, "gated_residual_norm");
    return g;
  }
};

std::pair<Tensor, Tensor> gated_residual_norm(Tensor x, Tensor h, OptT gate_, OptT scale_, OptT pw_, OptT pb_, OptT rw_, OptT rb_, bool layer,
                                              int64_t act, double eps, double s1) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && h.sizes() == x.sizes(), "x and h must have one shape, got ", x.sizes(), " and ", h.sizes());
  const int64_t D = x.size(-1);
  TORCH_CHECK_VALUE(D >= 1 && D <= srl::rnorm::MAXD, "the last axis must be 1..", srl::rnorm::MAXD, " wide, got ", D);
  TORCH_CHECK_VALUE(two_types(x), "x must be float32 or bfloat16, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.numel() / D < (1ll << 31) - 64, "fewer than 2^31 - 64 rows, got ", x.sizes());
  auto operand = [&](const Tensor& t) {
    TORCH_CHECK_VALUE(t.device() == x.device() && t.is_floating_point(), "every operand must be floating point on ", x.device(), ", got ",
                      t.scalar_type(), " on ", t.device());
  };
  operand(h);
  if (h.scalar_type() != x.scalar_type()) h = h.to(x.scalar_type());
  Tensor gate = val(gate_);
  if (gate.defined()) {
    operand(gate);
    if (gate.scalar_type() != x.scalar_type()) gate = gate.to(x.scalar_type());
    if (gate.sizes() != x.sizes()) gate = gate.expand(x.sizes());
  }
  const char* names[5] = {"scale", "post_weight", "post_bias", "pre_weight", "pre_bias"};
  Tensor w[5] = {val(scale_), val(pw_), val(pb_), val(rw_), val(rb_)};
  bool any = wants(x) || wants(h) || wants(gate);
  int64_t want = wants(gate);  // and a bit for each weight: the gradients that are made
  for (int i = 0; i < 5; ++i) {
    if (!w[i].defined()) continue;
    if (i == 0 && w[0].dim() == 0) w[0] = w[0].expand({D});
    shape(w[i], {D}, names[i]);
    operand(w[i]);
    w[i] = f32(w[i]).contiguous();
    if (reinterpret_cast<uintptr_t>(w[i].data_ptr()) % 16) w[i] = w[i].clone();  // the kernels read four at a time
    any = any || wants(w[i]);
    want |= (int64_t)wants(w[i]) << (i + 1);
  }
  if (at::GradMode::is_enabled() && any) {
    capturable({&x, &h, &gate, &w[0], &w[1], &w[2], &w[3], &w[4]}, "gated_residual_norm");
    auto r = ResidualNormFn::apply(x, h, opt_of(gate), opt_of(w[0]), opt_of(w[1]), opt_of(w[2]), opt_of(w[3]), opt_of(w[4]), layer, act, eps, s1, want);
    return {r[0], r[1]};
  }
  return norm_forward(x, h, gate, w[0], w[1], w[2], w[3], w[4], NormOpts{layer, act, eps, s1});
}

}  // namespace

void register_delta(pybind11::module& m) {
  m.def("gated_delta", &gated_delta);
  m.def("gated_delta_step", &gated_delta_step);
  m.def("gated_residual_norm", &gated_residual_norm);
}
