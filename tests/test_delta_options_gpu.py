"""The options of the gated delta rule through the kernels, against the rule in 64 bits: ``eps``, ``scale``, ``normalize``, gradients
of one output alone, strides in bf16."""
import pytest
import torch

from sheeprl_prey_amd import ops
from tests.test_delta_cpu import LONG_LENGTHS, delta_inputs, delta_oracle
from tests.test_delta_gpu import NAMES, close, oracle_train, run_train, tag

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])


def projected(x, d_out, d_last, eps, **kw):
    """Root mean square of r d, with d the gradient of the unit vectors and r their factor: d_q and d_k are differences of vectors of
    that length, whose roundings they carry, where q and k are scaled to unit length."""
    y = {n: t.detach().double().cpu() for n, t in x.items()}
    r = {n: (y[n].square().sum(-1, keepdim=True) + eps).rsqrt() for n in "qk"}
    for n in "qk":
        y[n] = (y[n] * r[n]).requires_grad_()
    kw = {n: t.cpu() if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
    d = torch.autograd.grad(delta_oracle(**y, **kw, normalize=False), [y["q"], y["k"]], (d_out.double().cpu(), d_last.double().cpu()))
    return {n: (r[n] * g).square().mean().sqrt() for n, g in zip("qk", d)}


def gradients_of(x, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(x["v"].shape, generator=g).to(x["v"].dtype).cuda(), torch.randn(x["state"].shape, generator=g).cuda())


def check_train(x, **kw):
    d_out, d_last = gradients_of(x)
    got, want = run_train(x, d_out, d_last, **kw), oracle_train(x, d_out, d_last, **kw)
    terms = {} if not kw.get("normalize", True) else projected(x, d_out, d_last, **{"eps": 1e-6, **kw})
    close(got[0], want[0], tag("out", got[0]))
    close(got[1], want[1], "last fp32")
    for n in NAMES:
        close(got[2][n], want[2][n], tag("d_" + n, got[2][n]), terms.get(n, 0.0))


@TYPES
@pytest.mark.parametrize("T", [3, 5, 16, 70, 530])
def test_no_eps_with_chunks_that_are_not_full(T, dtype):
    x = delta_inputs(T, 3, 1, 2, 24, 40, dtype, T, "cuda")
    check_train(x, eps=0.0)
    lengths = torch.tensor([T, T // 2 + 1, 0], dtype=torch.int32).cuda()
    check_train(x, eps=0.0, lengths=lengths)
    with torch.no_grad():
        out, last = ops.gated_delta(**x, eps=0.0, lengths=lengths)
    want, el = delta_oracle(**{n: t.cpu() for n, t in x.items()}, eps=0.0, lengths=lengths.cpu())
    close(out, want, tag("out", out))
    close(last, el, "last fp32")


@pytest.mark.parametrize("T", [4, 5, 70, 530])
def test_lengths_past_32_bits_are_clamped(T):
    x = delta_inputs(T, len(LONG_LENGTHS), 1, 2, 32, 32, torch.float32, T, "cuda")
    long, short = (torch.tensor(n).cuda() for n in (LONG_LENGTHS, [T, T, T, 0, 0, 3]))
    w, z = gradients_of(x)
    a, b = run_train(x, w, z, lengths=long), run_train(x, w, z, lengths=short.int())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(a[2][n], b[2][n]) for n in NAMES)
    with torch.no_grad():
        a, b = ops.gated_delta(**x, lengths=long), ops.gated_delta(**x, lengths=short.int())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("T", [4, 16, 70, 530])
def test_a_reset_reads_neither_the_state_nor_the_decay(T):
    x = delta_inputs(T, 2, 1, 2, 32, 24, torch.float32, T, "cuda")
    first = torch.zeros(T, 2, dtype=torch.bool, device="cuda")
    first[0, 0] = first[T - 2, 1] = True
    w, z = gradients_of(x)
    a = run_train(x, w, z, is_first=first)
    with torch.no_grad():
        few = ops.gated_delta(**x, is_first=first)
    x["state"][0] = float("nan")
    x["decay"][0, 0] = x["decay"][T - 2, 1] = float("nan")
    b = run_train(x, w, z, is_first=first)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(a[2][n], b[2][n]) for n in NAMES)
    with torch.no_grad():
        assert all(torch.equal(p, q) for p, q in zip(few, ops.gated_delta(**x, is_first=first)))


@pytest.mark.parametrize("T", [2, 5, 20])
def test_as_many_states_as_are_allowed(T):
    """2^20 states: the last ones come out as they do by themselves; one more is refused."""
    B = 2**20
    x = delta_inputs(T, 3, 1, 1, 2, 3, torch.float32, T, "cuda")
    big = {n: t.new_zeros(*t.shape[:int(n != "state")], B, *t.shape[1 + int(n != "state"):]) for n, t in x.items()}
    for n, t in x.items():
        (big[n] if n == "state" else big[n].transpose(0, 1))[-3:] = t if n == "state" else t.transpose(0, 1)
    with torch.no_grad():
        (a, la), (b, lb) = ops.gated_delta(**big), ops.gated_delta(**x)
        assert torch.equal(a[:, -3:], b) and torch.equal(la[-3:], lb) and not a[:, :-3].any() and not la[:-3].any()
        with pytest.raises(ValueError, match="2\\^20 states"):
            ops.gated_delta(**{n: torch.cat((t, t[:1] if n == "state" else t[:, :1]), int(n != "state")) for n, t in big.items()})
    w, z = gradients_of(x)
    want = run_train(x, w, z)[2]
    bw, bz = torch.zeros_like(big["v"]), torch.zeros_like(big["state"])
    bw[:, -3:], bz[-3:] = w, z
    got = run_train(big, bw, bz)[2]
    for n in NAMES:
        assert torch.equal(got[n][-3:] if n == "state" else got[n][:, -3:], want[n]), n


def test_as_many_steps_as_are_allowed():
    """2^24 steps of one head as they are in two halves; one more is refused."""
    T = 2**24
    x = delta_inputs(1, 1, 1, 1, 4, 4, torch.float32, 1, "cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(T, 1, 1, 4, generator=g, device="cuda") for _ in range(3))
    decay = -torch.rand(T, 1, 1, generator=g, device="cuda")
    beta = torch.rand(T, 1, 1, generator=g, device="cuda")
    with torch.no_grad():
        out, last = ops.gated_delta(q, k, v, decay, beta, x["state"])
        h = T // 2
        a, mid = ops.gated_delta(*(t[:h] for t in (q, k, v, decay, beta)), x["state"])
        b, end = ops.gated_delta(*(t[h:] for t in (q, k, v, decay, beta)), mid)
        close(out[:h], a, "out fp32")
        close(out[h:], b, "out fp32")
        close(last, end, "last fp32")
        with pytest.raises(ValueError, match="2\\^24 steps"):
            ops.gated_delta(*(torch.cat((t, t[:1])) for t in (q, k, v, decay, beta)), x["state"])


def unscaled(x):
    """Keys and queries of a length near one, taken as they are: the rule without the scaling is stable below a length of sqrt(2)."""
    D = x["k"].shape[-1]
    return {**x, "q": (x["q"].float() * D**-0.5).to(x["q"].dtype), "k": (0.7 * x["k"].float() * D**-0.5).to(x["k"].dtype)}


OPTIONS = pytest.mark.parametrize("kw", [dict(normalize=False), dict(scale=0.7), dict(eps=0.3), dict(normalize=False, scale=-1.3)],
                                  ids=["unscaled", "scale", "eps", "unscaled-scale"])
SIZES = pytest.mark.parametrize("T,Hk,Hv,Dk,Dv", [(3, 1, 2, 32, 24), (8, 1, 2, 40, 24), (70, 2, 2, 72, 40), (530, 1, 2, 24, 20)])


@TYPES
@OPTIONS
@SIZES
def test_options_in_training(T, Hk, Hv, Dk, Dv, kw, dtype):
    x = delta_inputs(T, 2, Hk, Hv, Dk, Dv, dtype, T, "cuda")
    check_train(unscaled(x) if "normalize" in kw else x, **kw)


@TYPES
@OPTIONS
@SIZES
def test_options_without_a_gradient(T, Hk, Hv, Dk, Dv, kw, dtype):
    x = delta_inputs(T, 2, Hk, Hv, Dk, Dv, dtype, T, "cuda")
    x = unscaled(x) if "normalize" in kw else x
    with torch.no_grad():
        out, last = ops.gated_delta(**x, **kw)
        S = x["state"].clone()
        steps = torch.stack([ops.gated_delta_step(*(x[n][t] for n in NAMES[:5]), S, **kw) for t in range(min(T, 8))])
    want, el = delta_oracle(**{n: t.cpu() for n, t in x.items()}, **kw)
    close(out, want, tag("out", out))
    close(last, el, "last fp32")
    close(steps, want[:8], tag("out", steps))
    if T <= 8:
        close(S, el, "state fp32")


@TYPES
@pytest.mark.parametrize("kw", [dict(normalize=False, scale=0.7), dict(eps=0.3)], ids=["unscaled", "eps"])
def test_options_with_shared_key_heads_in_turn(kw, dtype):
    """Wide heads and enough chunks that one workgroup takes the value heads of a key head in turn: two sequences, 32 times over."""
    T, n = 500, 32
    x = delta_inputs(T, 2, 1, 2, 72, 20, dtype, T, "cuda")
    x = unscaled(x) if "normalize" in kw else x
    w, z = gradients_of(x)
    want = oracle_train(x, w, z, **kw)
    terms = {} if "normalize" in kw else projected(x, w, z, **kw)

    def over(t, batch):
        return torch.cat([t] * n, batch)

    out, last, grads = run_train({k: over(t, int(k != "state")) for k, t in x.items()}, over(w, 1), over(z, 0), **kw)
    close(out, over(want[0], 1), tag("out", out))
    close(last, over(want[1], 0), "last fp32")
    for k in NAMES:
        close(grads[k], over(want[2][k], int(k != "state")), tag("d_" + k, grads[k]), terms.get(k, 0.0))


@TYPES
@pytest.mark.parametrize("which", [0, 1], ids=["out", "last"])
@pytest.mark.parametrize("T", [9, 70, 530])
def test_the_gradient_of_one_output_alone(T, which, dtype):
    x = delta_inputs(T, 2, 1, 2, 32, 24, dtype, T, "cuda")
    d = gradients_of(x)
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    got = torch.autograd.grad(ops.gated_delta(**leaves)[which], list(leaves.values()), d[which], allow_unused=True)
    exact = {n: t.double().cpu().requires_grad_() for n, t in x.items()}
    want = torch.autograd.grad(delta_oracle(**exact)[which], list(exact.values()), d[which].double().cpu(), allow_unused=True)
    zero = [torch.zeros_like(t) for t in d]
    terms = projected(x, *(d[i] if i == which else zero[i] for i in range(2)), 1e-6)
    for n, a, b in zip(NAMES, got, want):
        if b is None:  # the last state does not see the queries
            assert not a.any(), n
        else:
            close(a, b, tag("d_" + n, a), terms.get(n, 0.0))


@TYPES
@pytest.mark.parametrize("T", [3, 9, 70, 530])
def test_strides(T, dtype):
    """Batch first, heads first, a slice of a wider projection, a last stride of 2, one decay for all heads."""
    B, H, D = 2, 2, 32
    x = delta_inputs(T, B, H, H, D, D, dtype, T, "cuda")
    w, z = gradients_of(x)
    wide = torch.zeros(T, B, H, D + 3, device="cuda", dtype=dtype)
    wide[..., 1:D + 1] = x["v"]
    pairs = torch.zeros(T, B, H, D, 2, device="cuda", dtype=dtype)
    pairs[..., 0] = x["k"]
    x["decay"] = x["decay"][..., :1].contiguous().expand(T, B, H)
    y = {"q": x["q"].transpose(0, 1).contiguous().transpose(0, 1), "k": pairs[..., 0], "v": wide[..., 1:D + 1],
         "decay": x["decay"], "beta": x["beta"].permute(2, 0, 1).contiguous().permute(1, 2, 0),
         "state": x["state"].transpose(0, 1).contiguous().transpose(0, 1)}
    dw = torch.zeros(T, B, H, D + 1, device="cuda", dtype=dtype)
    dw[..., 1:] = w
    want = oracle_train(x, w, z)
    terms = projected(x, w, z, 1e-6)
    leaves = {n: t.requires_grad_() for n, t in y.items()}
    out, last = ops.gated_delta(**leaves)
    grads = torch.autograd.grad((out, last), list(leaves.values()), (dw[..., 1:], z.transpose(0, 1).contiguous().transpose(0, 1)))
    close(out, want[0], tag("out", out))
    close(last, want[1], "last fp32")
    for n, g in zip(NAMES, grads):
        close(g, want[2][n], tag("d_" + n, g), terms.get(n, 0.0))
    with torch.no_grad():
        out, last = ops.gated_delta(**y)
    close(out, want[0], tag("out", out))
    close(last, want[1], "last fp32")


@TYPES
@pytest.mark.parametrize("name", ["q", "k", "v", "decay", "beta", "state"])
@pytest.mark.parametrize("T", [3, 9, 70, 530])
def test_a_value_that_is_not_finite_stays_in_its_sequence_and_key_head(T, name, dtype):
    x = delta_inputs(T, 2, 2, 4, 16, 16, dtype, T, "cuda")
    w, z = gradients_of(x)
    a = run_train(x, w, z)
    with torch.no_grad():
        c = ops.gated_delta(**x)
    if name == "state":
        x["state"][1, 1, 3, 3] = float("nan")
    else:
        x[name][T // 2, 1, 0] = float("nan")
    b = run_train(x, w, z)
    with torch.no_grad():
        d = ops.gated_delta(**x)

    def equal(s, t, axis):  # heads of key head 1, and all of sequence 0
        half = s.shape[axis + 1] // 2
        for u in range(2):
            p, q = s.select(axis, u), t.select(axis, u)
            if u == 1:
                p, q = p.narrow(axis, half, p.shape[axis] - half), q.narrow(axis, half, q.shape[axis] - half)
            if not torch.equal(p, q):
                return False
        return True

    assert equal(a[0], b[0], 1) and equal(a[1], b[1], 0) and equal(c[0], d[0], 1) and equal(c[1], d[1], 0)
    for n in NAMES:
        assert equal(a[2][n], b[2][n], int(n != "state")), n


def test_an_operand_in_a_slice_of_a_store_of_states_is_refused():
    """States with gaps between them: what lies in the gaps is an operand like any other, what lies in a state is refused."""
    B, Hv, D = 4, 2, 8
    row = Hv * D * D
    flat = torch.randn(B, row + 5 * Hv * D, device="cuda")
    S, gap = flat[:, :row].view(B, Hv, D, D), flat[:, row:].view(B, 5, Hv, D)
    gates = torch.rand(2, B, Hv, device="cuda")
    q, k, v = (gap[:, i] for i in range(3))
    copies, T = [t.clone() for t in (q, k, v, -gates[0], gates[1])], S.clone()
    want = ops.gated_delta_step(*copies, T)
    rest = flat[:, row:].clone()
    assert torch.equal(ops.gated_delta_step(q, k, v, -gates[0], gates[1], S), want) and torch.equal(S, T) and torch.equal(flat[:, row:], rest)
    before = flat.clone()
    decay, beta = -gates[0], gates[1]
    flags = flat.view(torch.uint8)
    for bad in (dict(q=S[:, :, 0]), dict(k=S[:, :, :, 3]), dict(v=flat[:, row - 1:row - 1 + Hv * D].view(B, Hv, D)),
                dict(beta=S[:, :, D - 1, D - 1]), dict(decay=flat[3:, row - 1:row + Hv - 1].expand(B, Hv)), dict(is_first=flags[:, 7])):
        with pytest.raises(ValueError, match="in the state"):
            ops.gated_delta_step(**{**dict(q=q, k=k, v=v, decay=decay, beta=beta, state=S), **bad})
    heads = flat[:, :row].view(B, Hv, D, D)[:, :1]  # the other head's state is free
    one = dict(q=q[:, :1], k=k[:, :1], v=S[:, 1:, 0], decay=decay[:, :1], beta=beta[:, :1], state=heads)
    T = heads.clone()
    want = ops.gated_delta_step(**{**one, "v": one["v"].clone(), "state": T})
    with pytest.raises(ValueError, match="in the state"):
        ops.gated_delta_step(**{**one, "v": S[:, :1, 0]})
    assert torch.equal(flat, before)
    assert torch.equal(ops.gated_delta_step(**one), want) and torch.equal(heads, T)
