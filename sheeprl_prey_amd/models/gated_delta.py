"""A recurrent core of gated-delta-rule blocks: the alternative to the LSTM in recurrent policies.

Each block reads the normed residual stream, projects it to queries, keys, values, a forgetting rate and a writing
strength per head and an output gate, runs the gated delta rule (``ops.gated_delta``: a matrix state per head, chunked over
whole sequences) and hands its output to ``ops.gated_residual_norm``, which closes the block (norm, gate, residual scale,
residual) and norms what the next block reads, in one pass."""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from sheeprl_prey_amd import ops
from sheeprl_prey_amd.models.models import Linear


class GatedDeltaBlocks(nn.Module):
    """``[T, N, input_size] -> [T, N, hidden_size]`` with a state ``[1, N, state_size]`` (fp32, zeros at an episode's start)."""

    def __init__(self, input_size: int, hidden_size: int, num_blocks: int = 1, key_heads: int = 2, value_heads: int = 2,
                 key_dim: int = 32, value_dim: int = 32, eps: float = 1e-5) -> None:
        super().__init__()
        if num_blocks < 1:
            raise ValueError(f"num_blocks must be at least 1, got {num_blocks}")
        if key_heads < 1 or value_heads % key_heads:
            raise ValueError(f"value_heads ({value_heads}) must be a multiple of key_heads ({key_heads})")
        self.hidden_size, self.num_blocks, self.eps = hidden_size, num_blocks, eps
        self.heads = (key_heads, value_heads, key_dim, value_dim)
        self.state_size = num_blocks * value_heads * key_dim * value_dim
        self._sizes = [key_heads * key_dim, key_heads * key_dim, value_heads * value_dim, value_heads, value_heads, hidden_size]
        self.input = Linear(input_size, hidden_size)
        self.proj = nn.ModuleList(Linear(hidden_size, sum(self._sizes)) for _ in range(num_blocks))
        self.out = nn.ModuleList(Linear(value_heads * value_dim, hidden_size) for _ in range(num_blocks))

        def each(n, value):
            return nn.ParameterList(nn.Parameter(torch.full((hidden_size,), value)) for _ in range(n))

        self.norm_weight, self.norm_bias = each(num_blocks + 1, 1.0), each(num_blocks + 1, 0.0)
        self.post_weight, self.post_bias, self.scale = each(num_blocks, 1.0), each(num_blocks, 0.0), each(num_blocks, 1.0)
        # softplus(0) exp(rate) = 0.5 ... 0.01 a step over the heads: memories of a few steps to some hundred
        rates = torch.linspace(math.log(0.5), math.log(0.01), value_heads) if value_heads > 1 else torch.tensor([math.log(0.1)])
        self.rate = nn.ParameterList(nn.Parameter(rates - math.log(math.log(2.0))) for _ in range(num_blocks))

    def initial_state(self, n: int, device=None) -> Tensor:
        return torch.zeros(1, n, self.state_size, device=device)

    def _project(self, u: Tensor, block: int):
        Hk, Hv, Dk, Dv = self.heads
        q, k, v, a, b, gate = self.proj[block](u).split(self._sizes, -1)
        lead = u.shape[:-1]
        decay = -F.softplus(a.float()) * self.rate[block].exp()
        return (q.view(*lead, Hk, Dk), k.view(*lead, Hk, Dk), v.view(*lead, Hv, Dv), decay, torch.sigmoid(b.float())), gate

    def _start(self, x: Tensor) -> Tuple[Tensor, Tensor]:
        x = self.input(x).float()  # the residual stream stays fp32 under autocast
        return x, ops.ln_act(x, self.norm_weight[0], self.norm_bias[0], self.eps)

    def _close(self, x: Tensor, o: Tensor, gate: Tensor, block: int) -> Tuple[Tensor, Tensor]:
        return ops.gated_residual_norm(
            x, self.out[block](o.flatten(-2)), gate, self.scale[block], self.post_weight[block], self.post_bias[block],
            self.norm_weight[block + 1], self.norm_bias[block + 1], norm="layer", act="silu", eps=self.eps)

    def _states(self, state: Tensor) -> Tensor:
        Hk, Hv, Dk, Dv = self.heads
        return state.view(-1, self.num_blocks, Hv, Dk, Dv)

    def forward(self, x: Tensor, state: Tensor, lengths: Optional[Tensor] = None, is_first: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
        """Whole sequences: outputs and the state after them.  ``lengths [N]``: steps behind a sequence's end leave its state;
        ``is_first [T, N(, 1)]``: steps that start from a zero state."""
        x, u = self._start(x)
        states, after = self._states(state), []
        for i in range(self.num_blocks):
            qkv, gate = self._project(u, i)
            o, last = ops.gated_delta(*qkv, states[:, i], lengths=lengths, is_first=is_first)
            after.append(last)
            x, u = self._close(x, o, gate, i)
        return u, (after[0] if self.num_blocks == 1 else torch.stack(after, 1)).reshape(1, -1, self.state_size)

    def step(self, x: Tensor, state: Tensor) -> Tensor:
        """One step ``[1, N, input_size]`` without a gradient, ``state`` updated in place."""
        x, u = self._start(x[0])
        states = self._states(state)
        for i in range(self.num_blocks):
            qkv, gate = self._project(u, i)
            o = ops.gated_delta_step(*qkv, states[:, i])
            x, u = self._close(x, o, gate, i)
        return u[None]
