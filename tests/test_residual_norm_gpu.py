"""The gated residual norms' kernels (``residual_norm.hip``) against the definition in 64 bits, forward and backward."""
import pytest
import torch

from sheeprl_prey_amd import ops
from tests.test_delta_cpu import norm_oracle

pytestmark = pytest.mark.gpu
NAMES = ("x", "h", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")


def inputs(rows, D, dtype, seed=0, bias=True, gate=True):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = dict(x=(2 * n(rows, D)).to(dtype), h=n(rows, D).to(dtype), gate=n(rows, D).to(dtype) if gate else None, scale=0.5 + 0.1 * n(D),
             post_weight=1 + 0.1 * n(D), post_bias=0.1 * n(D) if bias else None, pre_weight=1 + 0.1 * n(D), pre_bias=0.1 * n(D) if bias else None)
    return {k: None if t is None else t.cuda() for k, t in x.items()}


def close(got, want, terms, bf16):
    """Half a step of the type, and `terms` fp32 roundings of a sum whose terms are at most 8 times the result's rms."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all()
    allowed = (2.0**-8 if bf16 else 2.0**-24) * want.abs() + terms * 8 * 2.0**-24 * want.square().mean().sqrt().clamp_min(1e-30)
    assert ((got - want).abs() <= allowed).all(), ((got - want).abs() / allowed).max()


def check(a, dy, du, norm, act, eps=1e-5):
    leaves = {n: t.detach().clone().requires_grad_() for n, t in a.items() if t is not None}
    exact = {n: t.detach().double().cpu().requires_grad_() for n, t in leaves.items()}
    outs = ops.gated_residual_norm(**leaves, norm=norm, act=act, eps=eps)
    eouts = norm_oracle(*(exact.get(n) for n in NAMES), norm, act, eps)
    rows, D = a["x"].shape
    bf = a["x"].dtype == torch.bfloat16
    # a statistic is a tree of at most 16 + 10 additions; it enters both norms and their backward passes: 8 of them
    row_terms = 8 * 32
    for o, e in zip(outs, eouts):
        close(o, e, row_terms, bf)
    use = [i for i, d in enumerate((dy, du)) if d is not None]
    ds = [(dy, du)[i] for i in use]
    got = torch.autograd.grad([outs[i] for i in use], list(leaves.values()), ds, allow_unused=True)
    want = torch.autograd.grad([eouts[i] for i in use], list(exact.values()), [d.double().cpu() for d in ds], allow_unused=True)
    for n, g, w in zip(leaves, got, want):
        w = torch.zeros_like(exact[n]) if w is None else w
        # a column's sum runs over at most rows / 1024 + 1024 / 16 + 32 additions in a row
        close(g, w, row_terms + (0 if n in NAMES[:3] else rows // 1024 + 96), bf and n in NAMES[:3])
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 17), (16, 64), (37, 65), (130, 256), (9, 300), (70, 512), (33, 1001), (5, 1536), (17, 2048), (6, 4095),
                                    (4, 4096), (3, 6001), (2, 8192), (3000, 24)])
def test_forward_and_backward(rows, D, dtype):
    for norm, act, bias in (("layer", "silu", True), ("rms", "sigmoid", False)):
        a = inputs(rows, D, dtype, rows + D, bias)
        # the norm of a single value is 0 / sqrt(0 + eps) under "layer": a larger eps keeps its gradient in range
        check(a, torch.randn_like(a["x"]), torch.randn_like(a["x"]), norm, act, 1e-1 if D == 1 else 1e-5)


@pytest.mark.parametrize("which", ["dy", "du"])
def test_one_output_alone(which):
    a = inputs(50, 96, torch.float32)
    d = torch.randn_like(a["x"])
    check(a, d if which == "dy" else None, d if which == "du" else None, "layer", "none")


def test_without_gate_weights_or_scale():
    a = {n: t if n in ("x", "h") else None for n, t in inputs(40, 128, torch.float32).items()}
    check(a, torch.randn_like(a["x"]), torch.randn_like(a["x"]), "layer", "silu")
    y, u = ops.gated_residual_norm(a["x"], a["h"], scale=0.25)
    ey, eu = norm_oracle(a["x"].cpu(), a["h"].cpu(), None, 0.25, None, None, None, None, "layer", "silu", 1e-5)
    close(y, ey, 256, False)
    close(u, eu, 256, False)


def test_strides_leading_axes_and_broadcast_gate():
    a = inputs(60, 68, torch.float32)
    wide = torch.randn(60, 70, device="cuda")
    wide[:, 1:69] = a["x"]
    want = ops.gated_residual_norm(**a)
    for x in (wide[:, 1:69], a["x"].t().contiguous().t()):
        for g, w in zip(ops.gated_residual_norm(**{**a, "x": x}), want):
            close(g, w, 256, False)
    y, u = ops.gated_residual_norm(**{**a, "x": a["x"].view(5, 12, 68), "h": a["h"].view(5, 12, 68), "gate": a["gate"].view(5, 12, 68)})
    assert torch.equal(y.view(60, 68), want[0]) and torch.equal(u.view(60, 68), want[1])
    gate = torch.randn(60, 1, device="cuda", requires_grad=True)
    y, _ = ops.gated_residual_norm(**{**a, "gate": gate})
    (g,) = torch.autograd.grad(y.sum(), gate)
    g64 = gate.detach().double().cpu().requires_grad_()
    ey, _ = norm_oracle(a["x"].cpu(), a["h"].cpu(), g64.expand(60, 68), *(a[n].cpu() for n in NAMES[3:]), "layer", "silu", 1e-5)
    (eg,) = torch.autograd.grad(ey.sum(), g64)
    close(g, eg, 256 + 68, False)


def test_repeats_bit_by_bit_and_rows_are_apart():
    a = inputs(5000, 200, torch.bfloat16)
    dy, du = torch.randn_like(a["x"]), torch.randn_like(a["x"])
    g1, g2 = (check(a, dy, du, "layer", "silu") for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(g1, g2))
    y, u = ops.gated_residual_norm(**a)
    a["h"][7] = float("nan")
    y2, u2 = ops.gated_residual_norm(**a)
    keep = torch.arange(5000, device="cuda") != 7
    assert torch.equal(y[keep], y2[keep]) and torch.equal(u[keep], u2[keep]) and y2[7].isnan().all()


def test_weights_that_begin_anywhere():
    rows, D = 5, 96
    g = torch.Generator(device="cuda").manual_seed(4)
    x, h, gate = (torch.randn(rows, D, generator=g, device="cuda") for _ in range(3))
    w = [torch.randn(D, generator=g, device="cuda") for _ in range(5)]
    flat = torch.zeros(5, D + 1, device="cuda")
    for a, b in zip(flat, w):
        a[1:] = b

    def run(ws):
        leaves = [t.clone().requires_grad_() for t in (x, h, gate)]
        y, u = ops.gated_residual_norm(*leaves, *ws)
        return [y.detach(), u.detach(), *torch.autograd.grad(y.sum() + (u * x).sum(), leaves + ws)]

    odd = [t[1:].requires_grad_() for t in flat]
    assert any(t.data_ptr() % 16 for t in odd)
    for a, b in zip(run(odd), run([t.requires_grad_() for t in w])):
        assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """Operands of more than 2^31 elements: the last rows come out as they do by themselves."""
    rows, D = 2**20 + 8, 2048
    g = torch.Generator(device="cuda").manual_seed(1)
    x, h, gate, dy, du = ((torch.randn(8, D, generator=g, device="cuda")).bfloat16() for _ in range(5))
    big = []
    for t in (x, h, gate, dy, du):
        b = torch.zeros(rows, D, device="cuda", dtype=torch.bfloat16)
        b[-8:] = t
        big.append(b)
    assert big[0].numel() > 2**31

    def run(x, h, gate, dy, du):
        leaves = [t.requires_grad_() for t in (x, h, gate)]
        y, u = ops.gated_residual_norm(*leaves, 0.5, norm="rms")
        return [y.detach(), u.detach(), *torch.autograd.grad((y, u), leaves, (dy, du))]

    for a, b in zip(run(*big), run(x, h, gate, dy, du)):
        assert torch.equal(a[-8:], b)
        assert not a[:100].any()


def test_no_rows():
    y, u = ops.gated_residual_norm(torch.zeros(0, 16, device="cuda"), torch.zeros(0, 16, device="cuda"))
    assert y.shape == u.shape == (0, 16)


def test_captured_training_replays():
    a = {n: t.requires_grad_() for n, t in inputs(300, 128, torch.float32).items()}
    dy, du = torch.randn_like(a["x"]), torch.randn_like(a["x"])

    def step():
        y, u = ops.gated_residual_norm(**a)
        return (y.detach(), u.detach(), *torch.autograd.grad((y, u), list(a.values()), (dy, du)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for seed in (1, 2, 3):
        new = inputs(300, 128, torch.float32, seed)
        with torch.no_grad():
            for n in a:
                a[n].copy_(new[n])
        graph.replay()
        got = [t.clone() for t in res]
        b = {n: t.requires_grad_() for n, t in new.items()}
        y, u = ops.gated_residual_norm(**b)
        want = (y, u, *torch.autograd.grad((y, u), list(b.values()), (dy, du)))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("kw,match", [
    (dict(norm="batch"), "norm must be"), (dict(act="relu"), "act must be"), (dict(h=torch.zeros(4, 5)), "one shape"),
    (dict(scale=torch.zeros(5)), "scale must be"), (dict(pre_bias=torch.zeros(4, 6)), "pre_bias must be"),
    (dict(x=torch.zeros(1, 8193), h=torch.zeros(1, 8193)), "1..8192"), (dict(x=torch.zeros(4, 6).half()), "float32 or bfloat16"),
    (dict(post_weight=torch.zeros(6, dtype=torch.int32)), "floating point"),
])
def test_refusals(kw, match):
    args = {**dict(x=torch.zeros(4, 6), h=torch.zeros(4, 6)), **kw}
    with pytest.raises(ValueError, match=match):
        ops.gated_residual_norm(**{n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in args.items()})
    with pytest.raises(ValueError, match="floating point on"):
        ops.gated_residual_norm(torch.zeros(4, 6, device="cuda"), torch.zeros(4, 6, device="cuda"), torch.zeros(4, 6))


def test_mixed_types_and_a_second_differentiation():
    a = inputs(8, 32, torch.bfloat16)
    want = ops.gated_residual_norm(**a)
    got = ops.gated_residual_norm(**{**a, "h": a["h"].float(), "gate": a["gate"].float(), "scale": a["scale"].double()})
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    x = a["x"].float().requires_grad_()
    y, _ = ops.gated_residual_norm(x, a["h"])
    (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
