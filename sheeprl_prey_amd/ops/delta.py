"""The gated delta rule (``csrc/delta_*.hip``): a linear recurrence with a matrix state, for sequences and single steps.

Per sequence and value head, with a state ``S [Dk, Dv]`` in fp32 (``S = 0`` at a step that ``is_first`` marks)::

    S <- exp(decay_t) S;   u_t = beta_t (v_t - S^T k_t);   S <- S + k_t u_t^T;   out_t = scale S^T q_t

``q`` and ``k`` are scaled to unit length first (``normalize``).  Value head ``h`` reads query / key head ``h // (Hv // Hk)``.
Layouts follow the framework: time first, ``[T, B, heads, dim]``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

import sheeprl_prey_amd.ops as ops
from sheeprl_prey_amd.ops import reference as ref

MAX_HEAD_DIM = 128


def _check(q: Tensor, k: Tensor, v: Tensor, decay: Tensor, beta: Tensor, state: Optional[Tensor], lead: Tuple[str, ...]) -> None:
    n = len(lead)
    where = "[" + ", ".join(lead) + ", heads, dim]"
    if q.dim() != n + 2 or k.dim() != n + 2 or v.dim() != n + 2:
        raise ValueError(f"q, k, v must be {where}, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if q.shape != k.shape or q.shape[:n] != v.shape[:n]:
        raise ValueError(f"q and k must have one shape and v their leading sizes: {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    Hk, Dk, Hv, Dv = q.shape[-2], q.shape[-1], v.shape[-2], v.shape[-1]
    if Hk < 1 or Hv < Hk or Hv % Hk:
        raise ValueError(f"the value heads ({Hv}) must be a multiple of the key heads ({Hk})")
    if not (1 <= Dk <= MAX_HEAD_DIM and 1 <= Dv <= MAX_HEAD_DIM):
        raise ValueError(f"head dimensions must be 1..{MAX_HEAD_DIM}, got {Dk} and {Dv}")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError(f"q, k, v must have one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    allowed = (torch.float32, torch.bfloat16) if v.is_cuda else (torch.float32, torch.bfloat16, torch.float64)
    if v.dtype not in allowed:
        raise ValueError(f"q, k, v must be float32 or bfloat16, got {v.dtype}")
    if decay.shape != v.shape[:-1] or beta.shape != v.shape[:-1]:
        raise ValueError(f"decay and beta must be {tuple(v.shape[:-1])}, got {tuple(decay.shape)} and {tuple(beta.shape)}")
    if not (decay.is_floating_point() and beta.is_floating_point()):
        raise ValueError("decay and beta must be floating point")
    if state is not None:
        if state.shape != (v.shape[n - 1], Hv, Dk, Dv):
            raise ValueError(f"state must be {(v.shape[n - 1], Hv, Dk, Dv)}, got {tuple(state.shape)}")
        want = torch.float64 if v.dtype == torch.float64 else torch.float32
        if state.dtype != want:
            raise ValueError(f"state must be {want}, got {state.dtype}")
    for t in (q, k, decay, beta, state):
        if t is not None and t.device != v.device:
            raise ValueError(f"every operand must be on {v.device}, got {t.device}")


def _flags(x: Optional[Tensor], shape, name: str, device) -> Optional[Tensor]:
    if x is None:
        return None
    if x.dim() == len(shape) + 1 and x.shape[-1] == 1:
        x = x[..., 0]
    if tuple(x.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{name} must be on {device}, got {x.device}")
    return x if x.dtype in (torch.bool, torch.uint8) else x != 0


def _lengths(x: Optional[Tensor], B: int, T: int, device) -> Optional[Tensor]:
    if x is None:
        return None
    if tuple(x.shape) != (B,) or x.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"lengths must be int32 or int64 [{B}], got {x.dtype} {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"lengths must be on {device}, got {x.device}")
    return x.clamp(0, T)


def _fused(t: Tensor) -> bool:
    """The kernels take fp32 and bf16 as they come, so autocast regions use them too.  They check their operands as
    ``_check`` and its neighbours do here for the eager form."""
    return t.is_cuda and ops._FUSED


def gated_delta(
    q: Tensor, k: Tensor, v: Tensor, decay: Tensor, beta: Tensor, state: Optional[Tensor] = None, *,
    is_first: Optional[Tensor] = None, lengths: Optional[Tensor] = None, scale: Optional[float] = None,
    normalize: bool = True, eps: float = 1e-6,
) -> Tuple[Tensor, Tensor]:
    """``(out [T, B, Hv, Dv], last state [B, Hv, Dk, Dv])`` of the gated delta rule over ``T`` steps.

    ``q``, ``k`` ``[T, B, Hk, Dk]`` and ``v`` ``[T, B, Hv, Dv]`` in float32 or bfloat16, head dimensions up to 128, any
    strides (a copy is made only where the last one is not 1); ``decay`` (the logarithm of what a step keeps, <= 0) and
    ``beta`` ``[T, B, Hv]``; ``state`` fp32, zeros if None.  ``is_first [T, B(, 1)]`` marks steps that start from a
    zero state; there ``decay`` has no effect.  ``lengths [B]`` (clamped to 0..T): steps at or after a sequence's length change nothing,
    give zero outputs and get zero gradients, and are not read.  ``scale`` defaults to ``Dk ** -0.5``; ``eps`` is added to the sum of
    squares and may be zero where no row that counts is.  A value that is
    not finite in a step that counts spoils the results of its own sequence and key head, before it and after it, and
    nothing else; one in ``state`` those of its sequence and head, unless ``is_first`` marks the first step.

    Differentiable in ``q``, ``k``, ``v``, ``decay``, ``beta`` and ``state`` (once).  The sums, decays and states are fp32;
    outputs and gradients are rounded once to the operand's type, those of shared key heads after their sum.  A pass with its
    backward can be captured into a graph as long as no eager autograd graph of the same leaves is alive on the default
    stream (refused where ``q`` ... ``state`` are the leaves)."""
    if _fused(v) and v.numel() and q.numel():
        return ops._ext().gated_delta(q, k, v, decay, beta, state, is_first, lengths, scale, normalize, eps)
    _check(q, k, v, decay, beta, state, ("T", "B"))
    T, B = v.shape[:2]
    first = _flags(is_first, (T, B), "is_first", v.device)
    lens = _lengths(lengths, B, T, v.device)
    scale = float(q.shape[-1]) ** -0.5 if scale is None else float(scale)
    return ref.gated_delta(q, k, v, decay, beta, state, first, lens, scale, normalize, eps)


def gated_delta_step(
    q: Tensor, k: Tensor, v: Tensor, decay: Tensor, beta: Tensor, state: Tensor, *, is_first: Optional[Tensor] = None,
    scale: Optional[float] = None, normalize: bool = True, eps: float = 1e-6,
) -> Tensor:
    """One step for every sequence, ``state`` updated IN PLACE: ``out [B, Hv, Dv]``.

    ``q``, ``k`` ``[B, Hk, Dk]``, ``v [B, Hv, Dv]``, ``decay``, ``beta`` ``[B, Hv]``, ``is_first [B(, 1)]`` as in
    :func:`gated_delta`; ``state`` fp32 ``[B, Hv, Dk, Dv]``, each ``[Dk, Dv]`` contiguous and none overlapping (a slice of a larger
    store of states is fine) and without another operand in it.  No gradient; a captured graph replays it on the same state."""
    if _fused(v) and v.numel() and q.numel():
        return ops._ext().gated_delta_step(q, k, v, decay, beta, state, is_first, scale, normalize, eps)
    _check(q, k, v, decay, beta, state, ("B",))
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, decay, beta, state)):
        raise RuntimeError("gated_delta_step updates the state in place and has no gradient: use gated_delta, or torch.no_grad()")
    B, Hv, Dk, Dv = state.shape
    first = _flags(is_first, (B,), "is_first", v.device)
    scale = float(Dk) ** -0.5 if scale is None else float(scale)
    if not ((Dv == 1 or state.stride(3) == 1) and (Dk == 1 or state.stride(2) == Dv)):
        raise ValueError(f"each [Dk, Dv] of the state must be contiguous, got strides {state.stride()}")
    least = Dk * Dv
    for stride, n in sorted((state.stride(d), state.shape[d]) for d in (0, 1) if state.shape[d] > 1):
        if stride < least:
            raise ValueError(f"the states must not overlap, got strides {state.stride()}")
        least = stride * n
    if B == 0:
        return torch.empty_like(v)
    out, last = ref.gated_delta(*(t[None] for t in (q, k, v, decay, beta)), state, None if first is None else first[None], None, scale,
                                normalize, eps)
    state.copy_(last)
    return out[0]
