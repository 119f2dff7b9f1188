"""The gated delta rule and the gated residual norms off the GPU: the definitions in 64 bits, differences, refusals."""
import pytest
import torch

from sheeprl_prey_amd import ops


def delta_oracle(q, k, v, decay, beta, state=None, is_first=None, lengths=None, scale=None, normalize=True, eps=1e-6):
    """The rule sequence by sequence, head by head, step by step, in fp64; differentiable."""
    T, B, Hv, Dv = v.shape
    Hk, Dk = q.shape[2:]
    scale = Dk**-0.5 if scale is None else scale
    outs, lasts = [], []
    for b in range(B):
        n = T if lengths is None else max(0, min(T, int(lengths[b])))
        for h in range(Hv):
            S = torch.zeros(Dk, Dv, dtype=torch.float64) if state is None else state[b, h].double()
            o = []
            for t in range(n):
                qt, kt, vt = q[t, b, h // (Hv // Hk)].double(), k[t, b, h // (Hv // Hk)].double(), v[t, b, h].double()
                if normalize:
                    qt, kt = qt / (qt @ qt + eps).sqrt(), kt / (kt @ kt + eps).sqrt()
                if is_first is not None and bool(is_first[t, b]):
                    S = torch.zeros_like(S)
                else:
                    S = decay[t, b, h].double().exp() * S
                u = beta[t, b, h].double() * (vt - kt @ S)
                S = S + torch.outer(kt, u)
                o.append(scale * (qt @ S))
            o += [torch.zeros(Dv, dtype=torch.float64)] * (T - n)
            outs.append(torch.stack(o))
            lasts.append(S)
    return torch.stack(outs, 1).view(T, B, Hv, Dv), torch.stack(lasts).view(B, Hv, Dk, Dv)


def norm_oracle(x, h, gate, scale, pw, pb, rw, rb, norm, act, eps):
    def nrm(z, w, b):
        m = z.mean(-1, keepdim=True) if norm == "layer" else 0.0
        z = (z - m) / (((z - m) ** 2).mean(-1, keepdim=True) + eps).sqrt()
        return (z if w is None else z * w.double()) + (0.0 if b is None else b.double())

    a = 1.0 if scale is None else scale.double() if isinstance(scale, torch.Tensor) else scale
    if gate is not None:
        g = gate.double()
        a = a * {"silu": g * torch.sigmoid(g), "sigmoid": torch.sigmoid(g), "none": g}[act]
    y = x.double() + a * nrm(h.double(), pw, pb)
    return y, nrm(y, rw, rb)


def delta_inputs(T, B, Hk, Hv, Dk, Dv, dtype=torch.float32, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    d = dict(q=n(T, B, Hk, Dk).to(dtype), k=n(T, B, Hk, Dk).to(dtype), v=n(T, B, Hv, Dv).to(dtype),
             decay=-torch.nn.functional.softplus(n(T, B, Hv) - 1), beta=torch.sigmoid(n(T, B, Hv)), state=n(B, Hv, Dk, Dv) * 0.5)
    return {k: t.to(device) for k, t in d.items()}


@pytest.mark.parametrize("T,B,Hk,Hv,Dk,Dv", [(1, 1, 1, 1, 1, 1), (7, 3, 2, 4, 5, 6), (20, 2, 1, 3, 16, 9)])
def test_delta_reference_matches_oracle(T, B, Hk, Hv, Dk, Dv):
    x = delta_inputs(T, B, Hk, Hv, Dk, Dv)
    first = torch.rand(T, B) < 0.2
    lengths = torch.randint(0, T + 1, (B,))
    for kw in ({}, {"is_first": first}, {"lengths": lengths}, {"is_first": first, "lengths": lengths, "scale": 0.7, "normalize": False}):
        args = dict(x) if kw.get("normalize", True) else {**x, "k": 0.3 * x["k"]}
        out, last = ops.gated_delta(**args, **kw)
        eo, el = delta_oracle(**args, **kw)
        # fp32 along T steps of Dk-term sums: (T + Dk) roundings, terms at most 8 times the result
        tol = (T + Dk) * 8 * 2.0**-24
        torch.testing.assert_close(out.double(), eo, rtol=tol, atol=tol)
        torch.testing.assert_close(last.double(), el, rtol=tol, atol=tol * 8)


def test_delta_reference_gradients_by_differences():
    x = {k: t.double().requires_grad_() for k, t in delta_inputs(6, 2, 1, 2, 3, 4).items()}
    first = torch.tensor([[1, 0], [0, 0], [0, 1], [0, 0], [1, 0], [0, 0]], dtype=torch.bool)
    lengths = torch.tensor([6, 4])
    names = list(x)

    def f(*t):
        return ops.gated_delta(**dict(zip(names, t)), is_first=first, lengths=lengths)

    assert torch.autograd.gradcheck(f, tuple(x.values()), atol=1e-6)


def test_delta_step_is_one_step_and_updates_in_place():
    x = delta_inputs(1, 3, 2, 4, 8, 6)
    out, last = ops.gated_delta(**x)
    store = torch.zeros(5, 3, 4, 8, 6)
    store[2] = x["state"]
    got = ops.gated_delta_step(*(x[n][0] for n in ("q", "k", "v", "decay", "beta")), store[2])
    assert torch.equal(got, out[0]) and torch.equal(store[2], last)
    assert torch.equal(store[0], torch.zeros_like(store[0]))


def test_delta_no_steps_and_no_sequences():
    x = delta_inputs(0, 2, 1, 1, 4, 4)
    out, last = ops.gated_delta(**x)
    assert out.shape == (0, 2, 1, 4) and torch.equal(last, x["state"]) and last is not x["state"]
    x = delta_inputs(3, 0, 1, 1, 4, 4)
    out, last = ops.gated_delta(**x)
    assert out.shape == (3, 0, 1, 4) and last.shape == (0, 1, 4, 4)


@pytest.mark.parametrize("change,match", [
    (dict(k=torch.zeros(4, 2, 1, 7)), "one shape"),
    (dict(v=torch.zeros(4, 2, 3, 8)), "multiple of the key heads"),
    (dict(q=torch.zeros(4, 2, 2, 129), k=torch.zeros(4, 2, 2, 129)), "1..128"),
    (dict(v=torch.zeros(4, 2, 2, 8, dtype=torch.bfloat16)), "one type"),
    (dict(decay=torch.zeros(4, 2)), "decay and beta"),
    (dict(beta=torch.zeros(4, 2, 2, dtype=torch.int64)), "floating point"),
    (dict(state=torch.zeros(2, 2, 8, 7)), "state must be"),
    (dict(state=torch.zeros(2, 2, 8, 8, dtype=torch.bfloat16)), "state must be"),
    (dict(is_first=torch.zeros(2, 4, dtype=torch.bool)), "is_first must be"),
    (dict(lengths=torch.zeros(2)), "lengths must be"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths must be"),
    (dict(q=torch.zeros(4, 2, 8)), "heads, dim"),
])
def test_delta_refusals(change, match):
    x = delta_inputs(4, 2, 2, 2, 8, 8)
    with pytest.raises(ValueError, match=match):
        ops.gated_delta(**{**x, **change})


def test_delta_other_types_refused():
    x = delta_inputs(4, 2, 2, 2, 8, 8, torch.float16)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        ops.gated_delta(**x)


def test_delta_step_refusals():
    x = {k: t if k == "state" else t[0] for k, t in delta_inputs(1, 2, 1, 2, 8, 8).items()}
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.gated_delta_step(**{**x, "q": x["q"].clone().requires_grad_()})
    with pytest.raises(ValueError, match="contiguous"):
        ops.gated_delta_step(**{**x, "state": x["state"].transpose(2, 3)})
    with pytest.raises(ValueError, match="overlap"):
        ops.gated_delta_step(**{**x, "state": x["state"][:1].expand(2, 2, 8, 8)})
    with pytest.raises(ValueError, match="heads, dim"):
        ops.gated_delta_step(**{**x, "q": x["q"][None]})


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("act", ["silu", "sigmoid", "none"])
def test_norm_reference_matches_oracle_and_differences(norm, act):
    g = torch.Generator().manual_seed(1)
    n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()  # noqa: E731
    args = (n(2, 3, 5), n(2, 3, 5), n(2, 3, 5), n(5), n(5), n(5), n(5), n(5))
    y, u = ops.gated_residual_norm(*args, norm=norm, act=act, eps=1e-3)
    ey, eu = norm_oracle(*args, norm, act, 1e-3)
    torch.testing.assert_close(y, ey)
    torch.testing.assert_close(u, eu)
    assert torch.autograd.gradcheck(lambda *t: ops.gated_residual_norm(*t, norm=norm, act=act, eps=1e-3), args, atol=1e-6)


def test_norm_defaults_and_broadcast_gate():
    x, h = torch.randn(4, 6), torch.randn(4, 6)
    y, u = ops.gated_residual_norm(x, h)
    torch.testing.assert_close(y, x + torch.nn.functional.layer_norm(h, (6,)))
    torch.testing.assert_close(u, torch.nn.functional.layer_norm(y, (6,)))
    gate = torch.randn(4, 1, requires_grad=True)
    y, u = ops.gated_residual_norm(x, h, gate, 0.5)
    y.sum().backward()
    torch.testing.assert_close(y, x + 0.5 * torch.nn.functional.silu(gate) * torch.nn.functional.layer_norm(h, (6,)))
    assert gate.grad.shape == (4, 1)


@pytest.mark.parametrize("kw,match", [
    (dict(norm="batch"), "norm must be"), (dict(act="relu"), "act must be"), (dict(h=torch.zeros(4, 5)), "one shape"),
    (dict(scale=torch.zeros(5)), "scale must be"), (dict(pre_bias=torch.zeros(4, 6)), "pre_bias must be"),
    (dict(x=torch.zeros(1, 8193), h=torch.zeros(1, 8193)), "1..8192"), (dict(x=torch.zeros(4, 6).half()), "float32 or bfloat16"),
    (dict(post_weight=torch.zeros(6, dtype=torch.int32)), "floating point"),
])
def test_norm_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        ops.gated_residual_norm(**{**dict(x=torch.zeros(4, 6), h=torch.zeros(4, 6)), **kw})


# ------------------------------------------------------------------ the recurrent policy's blocks
def _blocks(num_blocks=2, **kw):
    from sheeprl_prey_amd.models import GatedDeltaBlocks

    torch.manual_seed(0)
    m = GatedDeltaBlocks(7, 12, num_blocks, **{**dict(key_heads=1, value_heads=2, key_dim=5, value_dim=6), **kw})
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.1 * torch.randn_like(p))
    return m


def test_the_policys_step_leaves_the_callers_states():
    from sheeprl_prey_amd.algos.ppo_recurrent.agent import build_recurrent_model
    from sheeprl_prey_amd.utils.utils import dotdict

    mlp = dotdict({"apply": False})
    m, _ = build_recurrent_model(7, dotdict(cell="gated_delta", pre_rnn_mlp=mlp, post_rnn_mlp=mlp, gated_delta=dict(
        hidden_size=12, num_blocks=2, key_heads=1, value_heads=2, key_dim=5, value_dim=6)))
    x, states = torch.randn(1, 3, 7), m.initial_states(3)
    with torch.no_grad():
        out, after = m.step(x, states)
        assert not states[0].any()
        want, last = m(x, states)
    torch.testing.assert_close(out, want)
    torch.testing.assert_close(after[0], last[0])


def test_blocks_step_by_step_are_the_sequence():
    m = _blocks()
    x, state = torch.randn(5, 3, 7), m.initial_state(3)
    out, last = m(x, state)
    assert out.shape == (5, 3, 12) and last.shape == (1, 3, m.state_size) and not state.any()
    with torch.no_grad():
        steps = torch.cat([m.step(x[t:t + 1], state) for t in range(5)])
    torch.testing.assert_close(out, steps)
    torch.testing.assert_close(last, state)


def test_blocks_lengths_are_the_sequences_alone():
    m = _blocks()
    x, state = torch.randn(6, 2, 7), torch.randn(1, 2, m.state_size)
    out, last = m(x, state, lengths=torch.tensor([4, 6]))
    a, la = m(x[:4, :1], state[:, :1])
    torch.testing.assert_close(out[:4, :1], a)
    torch.testing.assert_close(last[:, :1], la)
    first = torch.zeros(6, 2, 1)
    first[3] = 1
    out, last = m(x, state, is_first=first)
    b, lb = m(x[3:], torch.zeros_like(state))
    torch.testing.assert_close(out[3:], b)
    torch.testing.assert_close(last, lb)


def test_blocks_gradients_reach_every_parameter_and_agree_with_differences():
    m = _blocks().double()
    x = torch.randn(4, 2, 7, dtype=torch.float64)
    w = torch.randn(4, 2, 12, dtype=torch.float64)

    def loss():
        # the stream is fp32 by design: this test follows the same operations in fp64
        s, u = m.input(x), None
        u = torch.nn.functional.layer_norm(s, (12,), m.norm_weight[0], m.norm_bias[0], m.eps)
        states = m._states(torch.zeros(1, 2, m.state_size, dtype=torch.float64))
        for i in range(m.num_blocks):
            (q, k, v, _, _), gate = m._project(u, i)
            a, b = m.proj[i](u).split(m._sizes, -1)[3:5]
            decay = -torch.nn.functional.softplus(a) * m.rate[i].exp()
            o, _ = ops.gated_delta(q, k, v, decay, torch.sigmoid(b), states[:, i])
            s, u = m._close(s, o, gate, i)
        return (u * w).sum()

    loss().backward()
    g = torch.Generator().manual_seed(3)
    for n, p in m.named_parameters():
        assert p.grad is not None and p.grad.abs().max() > 0, n
        d = torch.randn(p.shape, generator=g, dtype=torch.float64)
        with torch.no_grad():
            p.add_(1e-5 * d)
            up = loss()
            p.sub_(2e-5 * d)
            down = loss()
            p.add_(1e-5 * d)
        # central differences: h^2 = 1e-10 of the third derivative, and 2^-52 / h of the loss
        assert abs((up - down) / 2e-5 - (p.grad * d).sum()) <= 1e-6 * (1 + p.grad.norm() * d.norm()), n


@pytest.mark.parametrize("kw,match", [(dict(num_blocks=0), "num_blocks"), (dict(key_heads=2, value_heads=3), "multiple of")])
def test_blocks_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        _blocks(**kw)


def test_recurrent_ppo_refuses_another_cell():
    from sheeprl_prey_amd.algos.ppo_recurrent.agent import build_recurrent_model
    from sheeprl_prey_amd.utils.utils import dotdict

    with pytest.raises(ValueError, match="algo.rnn.cell"):
        build_recurrent_model(4, dotdict({"cell": "gru"}))


@pytest.mark.parametrize("T", [5, 70])
def test_rows_behind_a_length_need_no_eps(T):
    x = {n: t.requires_grad_() for n, t in delta_inputs(T, 2, 1, 2, 8, 6).items()}
    lengths = torch.tensor([T, T // 2])
    out, last = ops.gated_delta(**x, lengths=lengths, eps=0.0)
    eo, el = delta_oracle(**x, lengths=lengths, eps=0.0)
    tol = (T + 8) * 8 * 2.0**-24  # as above
    torch.testing.assert_close(out.double(), eo, rtol=tol, atol=tol)
    torch.testing.assert_close(last.double(), el, rtol=tol, atol=tol * 8)
    for g in torch.autograd.grad(out.sum() + last.sum(), list(x.values())):
        assert torch.isfinite(g).all()


@pytest.mark.parametrize("cell", ["lstm", "gated_delta"])
@pytest.mark.parametrize("apply", [True, False])
def test_the_policys_heads_are_as_wide_as_the_recurrent_models_output(cell, apply):
    from sheeprl_prey_amd.algos.ppo_recurrent.agent import RecurrentPPOAgent
    from sheeprl_prey_amd.config.compose import compose
    from sheeprl_prey_amd.envs import spaces
    from sheeprl_prey_amd.utils.utils import dotdict

    cfg = dotdict(compose(["exp=ppo_recurrent", "env=gym", f"algo.rnn.cell={cell}", "algo.rnn.lstm.hidden_size=24", "algo.rnn.gated_delta.hidden_size=16",
                           f"algo.rnn.post_rnn_mlp.apply={apply}", "algo.rnn.post_rnn_mlp.dense_units=20"]))
    obs_space = spaces.Dict({"state": spaces.Box(-1, 1, (5,), "float32")})
    agent = RecurrentPPOAgent([3], obs_space, cfg.algo.encoder, cfg.algo.rnn, cfg.algo.actor, cfg.algo.critic, [], ["state"], False,
                              cfg.distribution, 2)
    assert agent.rnn.output_dim == (20 if apply else agent.rnn_hidden_size) and agent.rnn_hidden_size == (24 if cell == "lstm" else 16)
    actions, logp, _, values, states = agent({"state": torch.randn(4, 2, 5)}, torch.zeros(4, 2, 3), agent.initial_states)
    assert actions[0].shape == (4, 2, 3) and logp.shape == values.shape == (4, 2, 1) and len(states) == len(agent.rnn.state_keys)
    (values.sum() + logp.sum()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in agent.parameters())


LONG_LENGTHS = [2**31, 2**63 - 1, 2**32 + 2, -(2**32) + 2, -1, 3]  # in 32 bits: negative, -1, 2, 2, -1, 3


@pytest.mark.parametrize("T", [5])
def test_lengths_past_32_bits_are_clamped(T):
    x = delta_inputs(T, len(LONG_LENGTHS), 1, 2, 4, 4)
    out, last = ops.gated_delta(**x, lengths=torch.tensor(LONG_LENGTHS))
    want, el = ops.gated_delta(**x, lengths=torch.tensor([T, T, T, 0, 0, 3], dtype=torch.int32))
    assert torch.equal(out, want) and torch.equal(last, el)


def test_what_lies_behind_a_length_is_not_read():
    x = delta_inputs(7, 2, 1, 2, 8, 6)
    lengths = torch.tensor([4, 7])
    d_out, d_last = torch.randn_like(x["v"]), torch.randn_like(x["state"])

    def run():
        leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
        out = ops.gated_delta(**leaves, lengths=lengths)
        return (*out, *torch.autograd.grad(out, list(leaves.values()), (d_out, d_last)))

    want = run()
    for t in (d_out, *(x[n] for n in ("q", "k", "v", "decay", "beta"))):
        t[4:, 0] = float("nan")
    for a, b in zip(run(), want):
        assert torch.equal(a, b)


def test_a_reset_reads_neither_the_state_nor_the_decay():
    x = delta_inputs(6, 2, 1, 2, 8, 6)
    first = torch.zeros(6, 2, dtype=torch.bool)
    first[0, 0] = first[3, 1] = True

    def run():
        leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
        out = ops.gated_delta(**leaves, is_first=first)
        return (*out, *torch.autograd.grad(out, list(leaves.values()), [torch.ones_like(t) for t in out]))

    want = run()
    x["state"][0] = float("nan")
    x["decay"][0, 0] = x["decay"][3, 1] = float("nan")
    for a, b in zip(run(), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_sums_stay_in_fp32_under_autocast(dtype):
    x = delta_inputs(9, 2, 1, 2, 8, 6, dtype)
    one = [x[n][0] for n in ("q", "k", "v", "decay", "beta")]

    def run():
        leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
        out = ops.gated_delta(**leaves)
        res = [*out, *torch.autograd.grad(out, list(leaves.values()), [torch.ones_like(t) for t in out])]
        S = x["state"].clone()
        return [*res, ops.gated_delta_step(*one, S), S, *ops.gated_residual_norm(x["v"], x["v"] + 1, x["v"] - 1)]

    want = run()
    with torch.autocast("cpu", torch.bfloat16):
        got = run()
    # two fp32 forms, each (T + Dk) roundings of terms at most 8 times the result, then half a step of the type each
    tol = 2 * (9 + 8) * 8 * 2.0**-24
    for a, b in zip(got, want):
        step = 2.0**-7 if b.dtype == torch.bfloat16 else 0.0
        assert a.dtype == b.dtype
        torch.testing.assert_close(a.double(), b.double(), rtol=tol + step, atol=tol * 8)


def test_a_failed_request_for_lds_is_made_again(tmp_path):
    """The host code that asks for a kernel's LDS, with the two runtime calls that it makes replaced: the first request fails."""
    import os
    import shutil
    import subprocess

    cxx = shutil.which("g++")
    rocm = os.environ.get("ROCM_HOME", "/opt/rocm")
    if not cxx or not os.path.isdir(os.path.join(rocm, "include", "hip")):
        pytest.skip("needs g++ and the HIP headers")
    src = tmp_path / "lds.cpp"
    src.write_text("""
#include "delta_args.h"
static int device = 0, asked = 0;
static hipError_t answer = hipErrorInvalidValue;
extern "C" hipError_t hipGetDevice(int* d) { *d = device; return hipSuccess; }
extern "C" hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { ++asked; return answer; }
int main() {
  srl::delta::AskedLds l;
  l.allow(nullptr, 1 << 16);
  answer = hipSuccess;
  l.allow(nullptr, 1 << 16);
  if (asked != 2) return 1;
  l.allow(nullptr, 1 << 16);
  if (asked != 2) return 2;
  device = 3;
  l.allow(nullptr, 1 << 16);
  return asked == 3 ? 0 : 3;
}
""")
    csrc = os.path.join(os.path.dirname(ops.__file__), "csrc")
    exe = str(tmp_path / "lds")
    subprocess.check_call([cxx, "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I", csrc, "-I", os.path.join(rocm, "include"), str(src), "-o", exe])
    assert subprocess.call([exe]) == 0
