"""The gated delta rule and the gated residual norms together, as recurrent PPO runs them: the blocks on the kernels against the
same blocks in eager form, one captured training step, the single steps of the player, and the command line."""
import copy

import pytest
import torch

from sheeprl_prey_amd import ops
from sheeprl_prey_amd.models import GatedDeltaBlocks
from tests.test_algos import PPO_KEYS, STD, _check_ckpt
from tests.test_algos_gpu import _run

pytestmark = pytest.mark.gpu


def blocks(num_blocks=2, hidden=64, **kw):
    torch.manual_seed(0)
    m = GatedDeltaBlocks(24, hidden, num_blocks, **kw)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.1 * torch.randn_like(p))
    return m.cuda()


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-30)).item()


@pytest.mark.parametrize("T,N,kw", [(8, 16, {}), (70, 5, dict(key_heads=1, value_heads=3, key_dim=16, value_dim=24)), (600, 1, {})])
def test_blocks_agree_with_their_eager_form(T, N, kw):
    m = blocks(**kw)
    x, w = torch.randn(T, N, 24, device="cuda"), torch.randn(T, N, 64, device="cuda")
    lengths = torch.randint(1, T + 1, (N,), device="cuda")
    first = torch.rand(T, N, 1, device="cuda") < 0.05

    def run():
        state = 0.3 * torch.ones(1, N, m.state_size, device="cuda", requires_grad=True)
        out, last = m(x, state, lengths=lengths, is_first=first)
        return (out, last, *torch.autograd.grad((out * w).sum() + last.sum(), [state, *m.parameters()]))

    got = run()
    ops.set_fused(False)
    try:
        want = run()
    finally:
        ops.set_fused(True)
    # both forms round in fp32 along two blocks of at most 256 dependent roundings each, and a parameter's gradient sums
    # T N rows whose parts are taken to be 8 times their sum: 2 * 256 * 8 * 2^-24, both ways
    for a, b in zip(got, want):
        assert rel(a, b) <= 2 * 2 * 256 * 8 * 2.0**-24, rel(a, b)


def test_blocks_under_autocast_stay_near_fp32():
    m = blocks(1)
    x, state = torch.randn(40, 6, 24, device="cuda"), m.initial_state(6, "cuda")
    want, _ = m(x, state)
    with torch.autocast("cuda", torch.bfloat16):
        got, last = m(x, state)
        got.float().square().mean().backward()
    assert last.dtype == torch.float32 and all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    # six matrix products and the delta rule on operands of 8 bits, each at most 2^-8 of its size off
    assert rel(got, want) <= 8 * 2.0**-8


def test_player_steps_follow_the_sequence_and_replay():
    m = blocks()
    x, state = torch.randn(6, 16, 24, device="cuda"), m.initial_state(16, "cuda")
    want, last = m(x, state)
    with torch.no_grad():
        eager = torch.cat([m.step(x[t:t + 1], state) for t in range(6)])
        assert rel(eager, want) <= 2 * 2 * 256 * 8 * 2.0**-24 and rel(state, last) <= 2 * 2 * 256 * 8 * 2.0**-24
        cur, S = x[:1].clone(), m.initial_state(16, "cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m.step(cur, S.clone())
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m.step(cur, S)
        S.zero_()
        for t in range(6):
            cur.copy_(x[t:t + 1])
            graph.replay()
            assert torch.equal(out, eager[t:t + 1])
        assert torch.equal(S, state)


def test_captured_training_step_of_the_blocks():
    m = blocks()
    x, w, state = torch.randn(80, 4, 24, device="cuda"), torch.randn(80, 4, 64, device="cuda"), m.initial_state(4, "cuda")
    params = list(m.parameters())

    def grads(mod, inp):
        out, _ = mod(inp, state)
        return torch.autograd.grad((out * w).sum(), list(mod.parameters()))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(m, x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = grads(m, x)
    twin = copy.deepcopy(m)
    for seed in (1, 2, 3):
        torch.manual_seed(seed)
        x.copy_(torch.randn_like(x))
        with torch.no_grad():
            for p, q in zip(params, twin.parameters()):
                p.mul_(1.01)
                q.copy_(p)
        graph.replay()
        got = [g.clone() for g in res]
        want = grads(twin, x.clone())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert rel(a, b) <= 2 * 256 * 8 * 2.0**-24


@pytest.mark.parametrize("env_id", ["CartPole-v1", "Pendulum-v1"])
def test_recurrent_ppo_with_gated_delta_blocks(env_id):
    _run(STD + ["exp=ppo_recurrent", "algo.rnn.cell=gated_delta", f"env.id={env_id}", "env.mask_velocities=False", "mlp_keys.encoder=[state]", "algo.rollout_steps=8",
                "per_rank_sequence_length=4", "per_rank_num_batches=2", "algo.update_epochs=2", "root_dir=ppo_rec_delta",
                f"run_name={env_id}"])
    _check_ckpt("ppo_rec_delta", env_id, PPO_KEYS, False)
