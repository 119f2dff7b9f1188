"""The gated delta rule's kernels (``delta_*.hip``) against the rule in 64 bits: every variant that the plan chooses (recurrent,
chunks of 16 and of 64 steps, segments of a long axis), odd sizes, resets, lengths, strides, shared key heads, extreme
decays, streams, graphs."""
import pytest
import torch

from sheeprl_prey_amd import ops
from tests.test_delta_cpu import delta_inputs, delta_oracle

pytestmark = pytest.mark.gpu
NAMES = ("q", "k", "v", "decay", "beta", "state")

# A result passes through at most 128 (key dimensions) + 64 (substitution) + 64 (steps of a chunk) dependent fp32 roundings of
# 2^-24; terms are taken to be at most 8 times the result's root mean square: 256 * 8 * 2^-24 = 2^-13 of it.
SUMS = 2.0**-13


def close(got, want, name="", terms=0.0):
    """Half a step of the type relative to the value, and the sums' roundings relative to the root mean square of the result, or of
    the `terms` it is a difference of."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), name
    half = 2.0**-8 if name.endswith("bf16") else 2.0**-24
    allowed = half * want.abs() + SUMS * (want.square().mean().sqrt() + terms).clamp_min(1e-30)
    worst = ((got - want).abs() / allowed).max().item() if want.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} times the allowed difference"


def tag(name, t):
    return f"{name} {'bf16' if t.dtype == torch.bfloat16 else 'fp32'}"


def run_train(x, d_out, d_last, **kw):
    leaves = {n: t.detach().clone().requires_grad_() for n, t in x.items() if t is not None}
    out, last = ops.gated_delta(**leaves, **kw)
    grads = torch.autograd.grad((out, last), list(leaves.values()), (d_out, d_last))
    return out, last, dict(zip(leaves, grads))


def oracle_train(x, d_out, d_last, **kw):
    leaves = {n: t.detach().double().cpu().requires_grad_() for n, t in x.items() if t is not None}
    kw = {n: t.cpu() if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
    out, last = delta_oracle(**leaves, **kw)
    grads = torch.autograd.grad((out, last), list(leaves.values()), (d_out.double().cpu(), d_last.double().cpu()), allow_unused=True)
    return out, last, {n: torch.zeros_like(t) if g is None else g for (n, t), g in zip(leaves.items(), grads)}


def projected(x, d_out, d_last, **kw):
    """The gradient of a key is r (d - k^ (k^ . d)), with r = 1 / |k|, k^ = r k and d the gradient of k^: the difference of two
    vectors, the longer of length r |d|, that carry the roundings of their own sums.  Where k^ (k^ . d) is nearly all of d (in one
    dimension all but eps r^2 of it) the result is as much smaller than they are as it likes.  So the roundings allowed in d_q and
    d_k count relative to the root mean square of r d too, which this gives, from the rule with unit vectors as its leaves."""
    y = {n: t.detach().double().cpu() for n, t in x.items() if t is not None}
    r = {n: (y[n].square().sum(-1, keepdim=True) + 1e-6).rsqrt() for n in "qk"}
    for n in "qk":
        y[n] = (y[n] * r[n]).requires_grad_()
    kw = {n: t.cpu() if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
    d = torch.autograd.grad(delta_oracle(**y, **kw, normalize=False), [y["q"], y["k"]], (d_out.double().cpu(), d_last.double().cpu()), allow_unused=True)
    return {n: 0.0 if g is None else (r[n] * g).square().mean().sqrt() for n, g in zip("qk", d)}


def check_train(x, **kw):
    T, B, Hv, Dv = x["v"].shape
    g = torch.Generator().manual_seed(T)
    d_out = torch.randn(T, B, Hv, Dv, generator=g).to(x["v"].dtype).cuda()
    d_last = torch.randn(B, Hv, x["q"].shape[-1], Dv, generator=g).cuda()
    got, want = run_train(x, d_out, d_last, **kw), oracle_train(x, d_out, d_last, **kw)
    close(got[0], want[0], tag("out", got[0]))
    close(got[1], want[1], "last fp32")
    terms = projected(x, d_out, d_last, **kw)
    for n in want[2]:
        close(got[2][n], want[2][n], tag("d_" + n, got[2][n]), terms.get(n, 0.0))
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T,B,Hk,Hv,Dk,Dv", [
    (1, 2, 1, 1, 16, 16), (8, 5, 2, 2, 32, 32), (15, 1, 1, 3, 33, 17), (16, 2, 2, 2, 64, 128), (17, 3, 1, 1, 32, 48),
    (63, 1, 1, 2, 64, 64), (64, 2, 2, 2, 128, 128), (65, 1, 1, 1, 128, 16), (100, 2, 1, 2, 1, 1), (130, 1, 2, 2, 48, 80),
    (200, 2, 1, 1, 65, 100),
])
def test_training_matches_the_rule(T, B, Hk, Hv, Dk, Dv, dtype):
    check_train(delta_inputs(T, B, Hk, Hv, Dk, Dv, dtype, T, "cuda"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T,B,Hk,Hv,Dk,Dv", [(513, 1, 1, 1, 32, 32), (640, 1, 1, 2, 128, 128), (700, 2, 1, 1, 40, 24)])
def test_training_over_segments(T, B, Hk, Hv, Dk, Dv, dtype):
    check_train(delta_inputs(T, B, Hk, Hv, Dk, Dv, dtype, T, "cuda"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T,n,Hk,Hv,Dk,Dv", [(500, 32, 1, 2, 72, 20), (260, 26, 2, 6, 128, 16)])
def test_training_with_many_chunks_of_shared_key_heads(T, n, Hk, Hv, Dk, Dv, dtype):
    """A workgroup takes the value heads of a key head in turn: two sequences, n times over."""
    x = delta_inputs(T, 2, Hk, Hv, Dk, Dv, dtype, T, "cuda")
    g = torch.Generator().manual_seed(T)
    d_out, d_last = torch.randn(T, 2, Hv, Dv, generator=g).to(dtype).cuda(), torch.randn(2, Hv, Dk, Dv, generator=g).cuda()
    lengths = torch.tensor([T - 7, T // 3], dtype=torch.int32).cuda()
    want, terms = oracle_train(x, d_out, d_last, lengths=lengths), projected(x, d_out, d_last, lengths=lengths)

    def over(t, batch):
        return torch.cat([t] * n, batch)

    out, last, grads = run_train({k: over(t, int(k != "state")) for k, t in x.items()}, over(d_out, 1), over(d_last, 0), lengths=over(lengths, 0))
    close(out, over(want[0], 1), tag("out", out))
    close(last, over(want[1], 0), "last fp32")
    for k in NAMES:
        close(grads[k], over(want[2][k], int(k != "state")), tag("d_" + k, grads[k]), terms.get(k, 0.0))


@pytest.mark.parametrize("T", [5, 70, 530])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_resets_and_lengths(T, dtype):
    x = delta_inputs(T, 4, 1, 2, 24, 40, dtype, T, "cuda")
    g = torch.Generator().manual_seed(T)
    first = (torch.rand(T, 4, generator=g) < 0.1).cuda()
    first[0, 0] = True
    first[T - 1, 1] = True
    lengths = torch.tensor([T, T, max(1, T // 3), 0], dtype=torch.int32).cuda()
    out, last, grads = check_train(x, is_first=first, lengths=lengths)
    assert torch.equal(last[3], x["state"][3]) and not out[:, 3].any() and not out[max(1, T // 3):, 2].any()
    assert not grads["q"][:, 3].any() and not grads["v"][:, 3].any()
    with torch.no_grad():
        o2, l2 = ops.gated_delta(**x, is_first=first.float().unsqueeze(-1), lengths=lengths.long())
    close(o2, out, tag("out", out))
    close(l2, last, "last fp32")


@pytest.mark.parametrize("T", [3, 40, 520])
def test_what_lies_behind_a_length_is_not_read(T):
    x = delta_inputs(T, 2, 1, 2, 32, 32, torch.float32, 1, "cuda")
    lengths = torch.tensor([T - 2, T], dtype=torch.int32).cuda()
    d_out, d_last = torch.randn_like(x["v"]), torch.randn_like(x["state"])
    a = run_train(x, d_out, d_last, lengths=lengths)
    for n in ("q", "k", "v", "decay", "beta"):
        x[n][T - 2:, 0] = float("nan")
    d_out = d_out.clone()
    d_out[T - 2:, 0] = float("nan")
    b = run_train(x, d_out, d_last, lengths=lengths)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for n in NAMES:
        assert torch.equal(a[2][n], b[2][n]), n
    with torch.no_grad():
        o, l = ops.gated_delta(**x, lengths=lengths)
    assert torch.isfinite(o).all() and torch.isfinite(l).all()


@pytest.mark.parametrize("T", [6, 80])
def test_a_value_that_is_not_finite_stays_in_its_sequence(T):
    x = delta_inputs(T, 3, 2, 2, 16, 16, torch.float32, 2, "cuda")
    with torch.no_grad():
        a, la = ops.gated_delta(**x)
        x["k"][2, 1, 0] = float("inf")
        b, lb = ops.gated_delta(**x)
    keep = torch.ones(3, 2, dtype=torch.bool)
    keep[1, 0] = False
    assert torch.equal(a[:, keep], b[:, keep]) and torch.equal(la[keep], lb[keep])


@pytest.mark.parametrize("T", [12, 64, 300])
def test_extreme_decays_and_rates(T):
    x = delta_inputs(T, 2, 1, 2, 32, 16, torch.float32, 3, "cuda")
    x["decay"][T // 2, 0, 0] = float("-inf")
    x["decay"][T // 3, 0, 1] = -1e30
    x["decay"][T // 4, 1, 0] = -110.0
    x["decay"][T // 5, 1, 0] = -90.0
    x["decay"][:, 1, 1] = 0.0
    x["beta"][T // 2:, 1, 0] = 0.0
    x["beta"][: T // 2, 1, 1] = 1.0
    y = {n: t.clone() for n, t in x.items()}
    y["decay"] = y["decay"].clamp_min(-800.0)  # exp() is zero in 64 bits too
    d_out, d_last = torch.randn_like(x["v"]), torch.randn_like(x["state"])
    got, want = run_train(x, d_out, d_last), oracle_train(y, d_out, d_last)
    close(got[0], want[0], "out fp32")
    close(got[1], want[1], "last fp32")
    for n in NAMES:
        close(got[2][n], want[2][n], f"d_{n} fp32")
    with torch.no_grad():
        out, last = ops.gated_delta(**x)
    close(out, want[0], "out fp32")
    close(last, want[1], "last fp32")


@pytest.mark.parametrize("T", [4, 16, 70, 530])
def test_a_reset_forgets_a_state_that_is_not_finite(T):
    x = delta_inputs(T, 1, 1, 1, 16, 16, torch.float32, 4, "cuda")
    bad = {**x, "state": torch.full_like(x["state"], float("nan"))}
    first = torch.zeros(T, 1, dtype=torch.bool, device="cuda")
    first[0] = True
    with torch.no_grad():
        a, b = ops.gated_delta(**x, is_first=first), ops.gated_delta(**bad, is_first=first)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        S = bad["state"].clone()
        out = ops.gated_delta_step(*(x[n][0] for n in NAMES[:5]), S, is_first=first[0])
    close(out, a[0][0], "out fp32")
    assert torch.isfinite(S).all()
    w, z = torch.randn_like(x["v"]), torch.randn_like(x["state"])
    c, d = run_train(x, w, z, is_first=first), run_train(bad, w, z, is_first=first)
    assert torch.equal(c[0], d[0]) and torch.equal(c[1], d[1]) and all(torch.equal(c[2][n], d[2][n]) for n in NAMES)
    assert not d[2]["state"].any()


@pytest.mark.parametrize("T", [9, 70])
def test_strides_and_broadcast_operands(T):
    B, H, D = 3, 2, 32
    x = delta_inputs(T, B, H, H, D, D, torch.float32, 5, "cuda")
    d_out, d_last = torch.randn_like(x["v"]), torch.randn_like(x["state"])
    a = run_train(x, d_out, d_last)
    # batch first, heads first, a slice of a wider projection, a last stride of 2
    y = dict(x)
    y["q"] = x["q"].transpose(0, 1).contiguous().transpose(0, 1)
    y["k"] = x["k"].permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    wide = torch.randn(T, B, H, D + 3, device="cuda")
    wide[..., 1:D + 1] = x["v"]
    y["v"] = wide[..., 1:D + 1]
    pairs = torch.randn(T, B, H, D, 2, device="cuda")
    pairs[..., 0] = x["q"]
    for q in (y["q"], pairs[..., 0]):
        with torch.no_grad():
            out, last = ops.gated_delta(q, *(y[n] for n in NAMES[1:]))
        close(out, a[0], "out fp32")
        close(last, a[1], "last fp32")
    # one decay and one beta for every head; a gradient that is an expanded tensor
    decay, beta = x["decay"][..., :1].clone().requires_grad_(), x["beta"][:1].clone().requires_grad_()
    out, _ = ops.gated_delta(x["q"], x["k"], x["v"], decay.expand(T, B, H), beta.expand(T, B, H), x["state"])
    gd, gb = torch.autograd.grad(out.sum(), (decay, beta))
    d64, b64 = decay.detach().double().cpu().requires_grad_(), beta.detach().double().cpu().requires_grad_()
    xc = {n: x[n].double().cpu() for n in NAMES}
    eo, _ = delta_oracle(xc["q"], xc["k"], xc["v"], d64.expand(T, B, H), b64.expand(T, B, H), xc["state"])
    ed, eb = torch.autograd.grad(eo.sum(), (d64, b64))
    close(gd, ed, "d_decay fp32")
    close(gb, eb, "d_beta fp32")


def test_only_some_gradients_and_only_some_outputs():
    x = delta_inputs(40, 2, 1, 2, 32, 32, torch.float32, 6, "cuda")
    q = x["q"].clone().requires_grad_()
    out, last = ops.gated_delta(**{**x, "q": q, "state": None})
    w = torch.randn_like(last)
    (g,) = torch.autograd.grad((last * w).sum(), q, retain_graph=True)
    assert not g.any()  # the state does not see the queries
    (g,) = torch.autograd.grad(out.square().sum(), q)
    x64 = {n: x[n].double().cpu() for n in NAMES[1:5]}
    q64 = x["q"].double().cpu().requires_grad_()
    eo, _ = delta_oracle(q64, *(x64[n] for n in NAMES[1:5]))
    (eg,) = torch.autograd.grad(eo.square().sum(), q64)
    close(g, eg, "d_q fp32")


def test_gradient_by_differences():
    x = delta_inputs(70, 1, 1, 1, 16, 16, torch.float32, 7, "cuda")
    w, z = torch.randn_like(x["v"]), torch.randn_like(x["state"])
    got = run_train(x, w, z)[2]
    x64 = {n: t.double().cpu() for n, t in x.items()}

    def f(**y):
        out, last = delta_oracle(**{**x64, **y})
        return ((out * w.double().cpu()).sum() + (last * z.double().cpu()).sum()).item()

    g = torch.Generator().manual_seed(7)
    for n in NAMES:
        d = torch.randn(x64[n].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        diff = (f(**{n: x64[n] + h * d}) - f(**{n: x64[n] - h * d})) / (2 * h)
        along = (got[n].double().cpu() * d).sum().item()
        # the gradient's own roundings, and h^2 of the difference
        assert abs(along - diff) <= SUMS * got[n].double().cpu().norm().item() * 4 + 1e-7 * abs(diff), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("B,Hk,Hv,Dk,Dv", [(1, 1, 1, 1, 1), (16, 2, 2, 32, 32), (3, 2, 6, 48, 80), (5, 1, 2, 128, 128), (2, 1, 1, 65, 33)])
def test_steps_follow_the_rule(B, Hk, Hv, Dk, Dv, dtype):
    T = 6
    x = delta_inputs(T, B, Hk, Hv, Dk, Dv, dtype, 8, "cuda")
    first = (torch.rand(T, B, generator=torch.Generator().manual_seed(1)) < 0.3).cuda()
    store = torch.full((B, 2, Hv, Dk, Dv), 7.0, device="cuda")
    S = store[:, 1]
    S.copy_(x["state"])
    outs = [ops.gated_delta_step(*(x[n][t] for n in NAMES[:5]), S, is_first=first[t]) for t in range(T)]
    want, last = delta_oracle(**{n: t.cpu() for n, t in x.items()}, is_first=first.cpu())
    close(torch.stack(outs), want, tag("out", outs[0]))
    close(S, last, "state fp32")
    assert (store[:, 0] == 7.0).all()
    with torch.no_grad():
        out, l2 = ops.gated_delta(**x, is_first=first)
        few, _ = ops.gated_delta(**{n: t if n == "state" else t[:4] for n, t in x.items()}, is_first=first[:4])
    close(out, want, tag("out", out))
    close(l2, last, "last fp32")
    assert torch.equal(few, torch.stack(outs[:4]))  # the same kernel


def test_results_repeat_bit_by_bit():
    for T, B in ((40, 9), (600, 1)):
        x = delta_inputs(T, B, 1, 2, 64, 64, torch.float32, 9, "cuda")
        d_out, d_last = torch.randn_like(x["v"]), torch.randn_like(x["state"])
        a, b = run_train(x, d_out, d_last), run_train(x, d_out, d_last)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(a[2][n], b[2][n]) for n in NAMES)


def test_on_a_side_stream_two_at_once():
    xs = [delta_inputs(530, 1, 1, 1, 64, 64, torch.float32, s, "cuda") for s in (1, 2)]
    with torch.no_grad():
        want = [ops.gated_delta(**x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for st, x in zip(streams, xs):
        with torch.cuda.stream(st), torch.no_grad():
            got.append(ops.gated_delta(**x))
    torch.cuda.synchronize()
    for (a, la), (b, lb) in zip(want, got):
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_captured_training_replays_beside_eager_work():
    """Forward and backward in one graph, replayed on new inputs with eager passes of other leaves in between."""
    x = delta_inputs(530, 1, 1, 2, 32, 32, torch.float32, 10, "cuda")
    d_out, d_last = torch.randn_like(x["v"]), torch.randn_like(x["state"])
    static = {n: t.clone().requires_grad_() for n, t in x.items()}

    def step():
        out, last = ops.gated_delta(**static)
        return (out.detach(), last.detach(), *torch.autograd.grad((out, last), list(static.values()), (d_out, d_last)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for seed in (11, 12, 13):
        y = delta_inputs(530, 1, 1, 2, 32, 32, torch.float32, seed, "cuda")
        with torch.no_grad():
            for n in NAMES:
                static[n].copy_(y[n])
        graph.replay()
        got = [t.clone() for t in res]
        want = run_train(y, d_out, d_last)
        torch.cuda.synchronize()
        for a, b in zip(got, (want[0], want[1], *(want[2][n] for n in NAMES))):
            assert torch.equal(a, b)


def test_captured_steps_carry_the_state():
    x = delta_inputs(4, 4, 1, 2, 32, 32, torch.float32, 14, "cuda")
    S = x["state"].clone()
    cur = {n: x[n][0].clone() for n in NAMES[:5]}
    graph = torch.cuda.CUDAGraph()
    scratch = S.clone()
    ops.gated_delta_step(*cur.values(), scratch)
    with torch.cuda.graph(graph):
        out = ops.gated_delta_step(*cur.values(), S)
    S.copy_(x["state"])
    with torch.no_grad():
        want, last = ops.gated_delta(**x)
    for t in range(4):
        for n in NAMES[:5]:
            cur[n].copy_(x[n][t])
        graph.replay()
        assert torch.equal(out, want[t])
    assert torch.equal(S, last)


def test_a_capture_beside_a_living_graph_of_the_same_leaves_is_refused():
    x = {n: t.requires_grad_() for n, t in delta_inputs(20, 2, 1, 1, 16, 16, torch.float32, 16, "cuda").items()}
    out, _ = ops.gated_delta(**x)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="still alive"):
            ops.gated_delta(**x)
        (torch.ones(1, device="cuda") + 1).detach()
    torch.autograd.grad(out.sum(), list(x.values()), allow_unused=True)


def test_offsets_past_32_bits():
    """Operands of more than 2^31 elements: the last sequences come out as they do by themselves."""
    B, T, Dk, Dv = 262200, 64, 16, 128
    x = delta_inputs(T, 4, 1, 1, Dk, Dv, torch.bfloat16, 17, "cuda")
    big = {n: t.new_zeros(*t.shape[:1 if n != "state" else 0], B, *t.shape[2 if n != "state" else 1:]) for n, t in x.items()}
    for n, t in x.items():
        (big[n] if n == "state" else big[n].transpose(0, 1))[-4:] = t if n == "state" else t.transpose(0, 1)
    assert big["v"].numel() > 2**31
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    want = ops.gated_delta(**leaves)
    d_out = torch.randn_like(want[0])
    grads = torch.autograd.grad(want[0], list(leaves.values()), d_out)
    big = {n: t.requires_grad_() for n, t in big.items()}
    got = ops.gated_delta(**big)
    assert torch.equal(got[0][:, -4:], want[0]) and torch.equal(got[1][-4:], want[1])
    w = torch.zeros_like(got[0])
    w[:, -4:] = d_out
    for n, a, b in zip(x, torch.autograd.grad(got[0], list(big.values()), w), grads):
        assert torch.equal(a[-4:] if n == "state" else a[:, -4:], b), n
        assert not (a[:100] if n == "state" else a[:, :100]).any() or n in ("decay", "beta"), n


def test_a_store_of_states_past_32_bits():
    B, D = 140000, 128
    x = delta_inputs(1, 3, 1, 1, D, D, torch.float32, 18, "cuda")
    S = torch.zeros(B, 1, D, D, device="cuda")
    assert S.numel() > 2**31
    S[-3:] = x["state"]
    a = [torch.zeros(B, *x[n].shape[2:], device="cuda") for n in NAMES[:5]]
    for t, n in zip(a, NAMES):
        t[-3:] = x[n][0]
    out = ops.gated_delta_step(*a, S)
    want = ops.gated_delta_step(*(x[n][0] for n in NAMES[:5]), x["state"])
    assert torch.equal(out[-3:], want) and torch.equal(S[-3:], x["state"]) and not S[:-3].any()


def test_an_operand_in_the_state_is_refused():
    S = torch.zeros(2, 1, 8, 8, device="cuda")
    q = torch.zeros(2, 1, 8, device="cuda")
    with pytest.raises(ValueError, match="in the state"):
        ops.gated_delta_step(q, q, S.view(-1)[:16].view(2, 1, 8), torch.zeros(2, 1, device="cuda"), torch.zeros(2, 1, device="cuda"), S)


def test_eager_form_on_the_gpu_when_fusion_is_off():
    x = delta_inputs(20, 2, 1, 2, 32, 32, torch.float32, 15, "cuda")
    with torch.no_grad():
        a = ops.gated_delta(**x)
        ops.set_fused(False)
        try:
            b = ops.gated_delta(**x)
        finally:
            ops.set_fused(True)
    close(a[0], b[0], "out fp32")
    close(a[1], b[1], "last fp32")


def test_operands_on_two_devices_are_refused():
    x = delta_inputs(4, 2, 1, 1, 8, 8, device="cuda")
    with pytest.raises(ValueError, match="every operand must be on"):
        ops.gated_delta(**{**x, "beta": x["beta"].cpu()})


@pytest.mark.parametrize("change,match", [
    (dict(k=torch.zeros(4, 2, 1, 7)), "one shape"),
    (dict(v=torch.zeros(4, 2, 3, 8)), "multiple of the key heads"),
    (dict(q=torch.zeros(4, 2, 2, 129), k=torch.zeros(4, 2, 2, 129)), "1..128"),
    (dict(v=torch.zeros(4, 2, 2, 8, dtype=torch.bfloat16)), "one type"),
    (dict(q=torch.zeros(4, 2, 2, 8).half(), k=torch.zeros(4, 2, 2, 8).half(), v=torch.zeros(4, 2, 2, 8).half()), "float32 or bfloat16"),
    (dict(decay=torch.zeros(4, 2)), "decay and beta"),
    (dict(beta=torch.zeros(4, 2, 2, dtype=torch.int64)), "floating point"),
    (dict(state=torch.zeros(2, 2, 8, 7)), "state must be"),
    (dict(state=torch.zeros(2, 2, 8, 8, dtype=torch.bfloat16)), "state must be"),
    (dict(is_first=torch.zeros(2, 4, dtype=torch.bool)), "is_first must be"),
    (dict(lengths=torch.zeros(2)), "lengths must be"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths must be"),
    (dict(q=torch.zeros(4, 2, 8)), "heads, dim"),
])
def test_refusals(change, match):
    x = delta_inputs(4, 2, 2, 2, 8, 8, device="cuda")
    with pytest.raises(ValueError, match=match):
        ops.gated_delta(**{**x, **{n: t.cuda() for n, t in change.items()}})


def test_step_refusals():
    x = {k: t if k == "state" else t[0] for k, t in delta_inputs(1, 2, 1, 2, 8, 8, device="cuda").items()}
    before = x["state"].clone()
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.gated_delta_step(**{**x, "q": x["q"].clone().requires_grad_()})
    with pytest.raises(ValueError, match="contiguous"):
        ops.gated_delta_step(**{**x, "state": x["state"].transpose(2, 3)})
    for bad in (x["state"][:1].expand(2, 2, 8, 8), x["state"][:, :1].expand(2, 2, 8, 8), x["state"].as_strided((2, 2, 8, 8), (128, 60, 8, 1))):
        with pytest.raises(ValueError, match="overlap"):
            ops.gated_delta_step(**{**x, "state": bad})
    with pytest.raises(ValueError, match="heads, dim"):
        ops.gated_delta_step(**{**x, "q": x["q"][None]})
    assert torch.equal(before, x["state"])
    heads_first = x["state"].transpose(0, 1).contiguous().transpose(0, 1)
    a, b = ops.gated_delta_step(**x), ops.gated_delta_step(**{**x, "state": heads_first})
    assert torch.equal(a, b) and torch.equal(x["state"], heads_first)


def test_a_second_differentiation_is_refused():
    x = {n: t.requires_grad_() for n, t in delta_inputs(20, 1, 1, 1, 16, 16, device="cuda").items()}
    out, _ = ops.gated_delta(**x)
    (g,) = torch.autograd.grad(out.square().sum(), x["v"], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
