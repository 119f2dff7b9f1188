"""Norms before and after a block, fused with the block's gate and residual scale (``csrc/residual_norm.hip``)."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor

import sheeprl_prey_amd.ops as ops
from sheeprl_prey_amd.ops import reference as ref

MAX_WIDTH = 8192
GATE_ACTS = {"none": 0, "silu": 1, "sigmoid": 5}


def gated_residual_norm(
    x: Tensor, h: Tensor, gate: Optional[Tensor] = None, scale: Union[Tensor, float, None] = None,
    post_weight: Optional[Tensor] = None, post_bias: Optional[Tensor] = None, pre_weight: Optional[Tensor] = None,
    pre_bias: Optional[Tensor] = None, *, norm: str = "layer", act: str = "silu", eps: float = 1e-5,
) -> Tuple[Tensor, Tensor]:
    """The end of one residual block and the start of the next, over the last axis (up to 8192 wide)::

        y = x + scale * act(gate) * (norm(h) * post_weight + post_bias);   u = norm(y) * pre_weight + pre_bias

    ``x`` is the residual stream, ``h`` the block's output (the same shape), ``gate`` broadcasts to it; ``y`` continues the
    stream and ``u`` is what the next block reads.  ``norm`` is ``"layer"`` or ``"rms"``; ``act`` ``"silu"``,
    ``"sigmoid"`` or ``"none"``; a gate of None counts as 1.  ``scale`` is a number or ``[D]``; weights of None
    count as 1, biases of None as 0.  ``x`` is float32 or bfloat16, ``h`` and ``gate`` are taken in its type, the weights in
    float32; statistics and sums are float32 and ``u`` is taken from ``y`` before its rounding.  Differentiable (once) in every
    tensor; the weights' gradients are summed in a fixed order."""
    if norm not in ("layer", "rms"):
        raise ValueError(f"norm must be 'layer' or 'rms', got {norm!r}")
    if act not in GATE_ACTS:
        raise ValueError(f"act must be one of {sorted(GATE_ACTS)}, got {act!r}")
    s1 = 1.0
    if scale is not None and not isinstance(scale, Tensor):
        s1, scale = float(scale), None
    if x.is_cuda and ops._FUSED and x.numel():
        return ops._ext().gated_residual_norm(x, h, gate, scale, post_weight, post_bias, pre_weight, pre_bias, norm == "layer",
                                              GATE_ACTS[act], eps, s1)
    if x.dim() < 1 or h.shape != x.shape:
        raise ValueError(f"x and h must have one shape, got {tuple(x.shape)} and {tuple(h.shape)}")
    D = x.shape[-1]
    if not 1 <= D <= MAX_WIDTH:
        raise ValueError(f"the last axis must be 1..{MAX_WIDTH} wide, got {D}")
    allowed = (torch.float32, torch.bfloat16) if x.is_cuda else (torch.float32, torch.bfloat16, torch.float64)
    if x.dtype not in allowed:
        raise ValueError(f"x must be float32 or bfloat16, got {x.dtype}")
    if scale is not None and scale.dim() == 0:
        scale = scale.expand(D)
    for name, t in (("scale", scale), ("post_weight", post_weight), ("post_bias", post_bias), ("pre_weight", pre_weight), ("pre_bias", pre_bias)):
        if t is not None and tuple(t.shape) != (D,):
            raise ValueError(f"{name} must be [{D}], got {tuple(t.shape)}")
    for t in (h, gate, scale, post_weight, post_bias, pre_weight, pre_bias):
        if t is not None and (t.device != x.device or not t.is_floating_point()):
            raise ValueError(f"every operand must be floating point on {x.device}, got {t.dtype} on {t.device}")
    if gate is not None:
        gate = gate.to(x.dtype).expand(x.shape)
    h = h.to(x.dtype)
    return ref.gated_residual_norm(x, h, gate, s1 if scale is None else scale, post_weight, post_bias, pre_weight, pre_bias, norm, act, eps)
