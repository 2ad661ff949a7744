"""Linear attention with a decay for each head: whole histories, their
gradients, and one new position at a time.

For the valid positions of one (batch, head), with ``l = exp(log_decay[h])``::

    S_t = l * S_{t-1} + k_t v_t^T          out_t = scale * q_t^T S_t

``padding_mask`` is the framework's [B, L] bool mask, True = valid.  A masked
position takes no part, wherever it stands: it neither decays nor writes the
state, its output and its gradients are zero, and what its rows of q, k, v hold
is not read.  A left-padded, a right-padded and an unpadded batch of the same
histories therefore give the same states.

An infinity or a NaN at a valid position, or in a state, stays with its (batch,
head): the outputs and states that depend on it are not finite, NaN where the
formula gives an infinity too (the kernels split operands into sums, where it
becomes inf - inf), and so may the outputs of up to 63 positions before it be
(they share a product with it, with a weight of zero).

The state [B, H, Dk, Dv] (float32) is all that a history leaves behind:
``linear_attention(..., return_state=True)`` gives it, ``initial_state``
continues from it, and :func:`linear_attention_step` adds one position to it in
time that does not depend on the history's length.

What the kernels hold in fewer than 32 bits: with bfloat16 inputs the weights of
the position pairs within 64 positions, rounded once to bfloat16 (2^-8 of each
term), and the state's part of an output, taken as two bfloat16 numbers (2^-17;
three in the decay's gradient).  States, their updates and every sum are float32,
and float16 and float32 inputs meet float32 products alone.

CPU path: explicit torch math (the numerics reference).  GPU path: the gfx950
kernels of ``hip/linear_attention.hip``; falls back loudly per
replay_amd.ops.require_hip_on_gpu.
"""

from __future__ import annotations

import functools
import math
from typing import Optional, Tuple, Union

import torch
from torch._C import _is_tracing  # torch.jit.is_tracing() without its 0.4 us
from torch.autograd.function import once_differentiable

from replay_amd.ops import hip_ext, require_hip_on_gpu

#: head sizes that the kernels hold in registers
MAX_HEAD_DIM = 128
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _scale(q: torch.Tensor, scale: Optional[float]) -> float:
    if scale is None:
        return 1.0 / math.sqrt(max(q.shape[-1], 1)) if q.dim() else 1.0
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    return float(scale)


def _check(q, k, v, log_decay, mask, state, scale, dims: int, mask_name: str, state_name: str) -> None:
    where = "[B, H, L, D]" if dims == 4 else "[B, H, D]"
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != dims:
            raise ValueError(f"{name} must be {where}, got {tuple(t.shape)}")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError("q, k and v must share dtype and device")
        if t.shape[:-1] != q.shape[:-1]:
            raise ValueError(f"q and {name} must agree up to the head size: {tuple(q.shape)}, {tuple(t.shape)}")
    if k.shape != q.shape:
        raise ValueError(f"q and k must have the same head size: {q.shape[-1]}, {k.shape[-1]}")
    allowed = _DTYPES if q.is_cuda else (*_DTYPES, torch.float64)
    if q.dtype not in allowed:
        raise ValueError(f"unsupported dtype {q.dtype}")
    for t in (q, v):
        if not 1 <= t.shape[-1] <= MAX_HEAD_DIM:
            raise ValueError(f"head sizes must be from 1 to {MAX_HEAD_DIM}, got {t.shape[-1]}")
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    if log_decay.shape != (q.shape[1],) or log_decay.dtype != wide or log_decay.device != q.device:
        raise ValueError(f"log_decay must be {wide} of shape ({q.shape[1]},) on q's device")
    if mask is not None:
        shape = (q.shape[0], q.shape[2]) if dims == 4 else (q.shape[0],)
        if mask.dtype != torch.bool or tuple(mask.shape) != shape or mask.device != q.device:
            raise ValueError(f"{mask_name} must be bool of shape {shape} on q's device")
    if state is not None:
        shape = (q.shape[0], q.shape[1], q.shape[-1], v.shape[-1])
        if state.dtype != wide or tuple(state.shape) != shape or state.device != q.device:
            raise ValueError(f"{state_name} must be {wide} of shape {shape} on q's device")


def _power(log_decay: torch.Tensor, n: torch.Tensor) -> torch.Tensor:
    """l^n with l^0 = 1 also for a decay of zero (log_decay -inf)."""
    return torch.where(n > 0, torch.exp(log_decay * n.clamp(min=1)), torch.ones_like(n))


def _without_autocast(function):
    """Autocast would take the float32 products and sums to 16 bits."""

    @functools.wraps(function)
    def call(q, *args, **kwargs):
        with torch.autocast(q.device.type, enabled=False):
            return function(q, *args, **kwargs)

    return call


@_without_autocast
def eager_linear_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    padding_mask: Optional[torch.Tensor],
    initial_state: Optional[torch.Tensor],
    scale: float,
    chunk: int = 64,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Chunk by chunk in plain torch (32 bits, 64 for float64 inputs)."""
    B, H, L, Dk = q.shape
    dtype, wide = q.dtype, log_decay.dtype
    valid = q.new_ones(B, L, dtype=torch.bool) if padding_mask is None else padding_mask
    zero = torch.zeros((), dtype=wide, device=q.device)
    q, k, v = (torch.where(valid[:, None, :, None], t.to(wide), zero) for t in (q, k, v))
    ld = log_decay.view(1, H, 1)
    state = initial_state if initial_state is not None else q.new_zeros(B, H, Dk, v.shape[-1])
    if not L:  # a copy where no position changes it: the state after is never the one before
        state = state.clone()
    outs = []
    for s in range(0, L, chunk):
        qc, kc, vc = (t[:, :, s : s + chunk] for t in (q, k, v))
        n = valid[:, None, s : s + chunk].to(wide).cumsum(-1)
        last = n[..., -1:]
        gap = n[..., :, None] - n[..., None, :]
        weight = torch.where(gap >= 0, _power(ld[..., None], gap), zero).tril()
        inter = (qc @ state) * _power(ld, n)[..., None]
        outs.append(inter + ((qc @ kc.transpose(-1, -2)) * weight) @ vc)
        added = (kc * _power(ld, last - n)[..., None]).transpose(-1, -2) @ vc
        state = _power(ld, last)[..., None] * state + added
    out = torch.cat(outs, 2) * scale if outs else torch.zeros_like(v)
    return out.to(dtype), state


class LinearAttentionFunction(torch.autograd.Function):
    """Saves its inputs and, where the history was cut into segments, their
    start states; the pair weights are recomputed in the backward pass."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, padding_mask, initial_state, scale, return_state):
        out, state, seg = hip_ext().linear_attention_fwd(
            q, k, v, log_decay, padding_mask, initial_state, scale, return_state
        )
        ctx.save_for_backward(q, k, v, log_decay, padding_mask, initial_state, seg)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, state

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dstate):
        q, k, v, log_decay, padding_mask, initial_state, seg = ctx.saved_tensors
        if dout is None:
            if dstate is None:
                return (None,) * 8
            dout = torch.zeros_like(v)
        need_decay = ctx.needs_input_grad[3]
        need_state = initial_state is not None and ctx.needs_input_grad[5]
        dq, dk, dv, ddecay, ds0 = hip_ext().linear_attention_bwd(
            q, k, v, log_decay, padding_mask, initial_state, dout, dstate, seg, ctx.scale, need_decay, need_state
        )
        return dq, dk, dv, ddecay if need_decay else None, None, ds0 if need_state else None, None, None


def linear_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    padding_mask: Optional[torch.Tensor] = None,
    initial_state: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    return_state: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Causal linear attention over whole histories.

    :param q, k: [B, H, L, Dk], bfloat16, float16 or float32, any strides.
    :param v: [B, H, L, Dv].
    :param log_decay: [H] float32, the natural logarithm of each head's decay;
        at most 0 (-inf keeps nothing of the past).
    :param padding_mask: [B, L] bool, True = valid.
    :param initial_state: [B, H, Dk, Dv] float32, zeros if not given.
    :param scale: 1 / sqrt(Dk) if not given.
    :param return_state: return the state after the last position as well.
    :return: [B, H, L, Dv] in q's dtype (its memory is laid out [B, L, H, Dv]),
        and the state if asked for.

    Differentiable once in q, k, v, log_decay and initial_state; on the GPU in
    reverse mode alone (a dual tensor is refused there).
    """
    scale = _scale(q, scale)
    args = (q, k, v, log_decay, padding_mask, initial_state, scale)
    if not require_hip_on_gpu(q):
        _check(*args, 4, "padding_mask", "initial_state")
        out, state = eager_linear_attention(*args)
        return (out, state) if return_state else out
    try:
        # a trace records the autograd function, but not the extension's call
        if _is_tracing() or torch.is_grad_enabled() and (
            q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad
            or (initial_state is not None and initial_state.requires_grad)
        ):
            out, state = LinearAttentionFunction.apply(*args, return_state)
        else:
            out, state, _ = hip_ext().linear_attention_fwd(*args, return_state)
    except RuntimeError:
        # the extension refuses what _check does, without the cost of asking twice
        _check(*args, 4, "padding_mask", "initial_state")
        raise
    return (out, state) if return_state else out


def linear_attention_step(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    state: torch.Tensor,
    active: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """One new position for each row, for serving (not differentiable, and on
    the GPU not traceable).

    :param q, k: [B, H, Dk]; v: [B, H, Dv].
    :param state: [B, H, Dk, Dv] float32, UPDATED IN PLACE; each head's
        [Dk, Dv] block must be contiguous, and no two blocks may overlap.  A
        backward pass that still needs it (as ``initial_state``) then raises.
    :param active: [B] bool; a row that is False keeps its state and gets a
        zero output.
    :return: [B, H, Dv] in q's dtype.
    """
    scale = _scale(q, scale)
    if torch.is_grad_enabled() and (
        q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad or state.requires_grad
    ):
        raise RuntimeError(
            "linear_attention_step updates the state in place and is not differentiable: "
            "call it under torch.no_grad(), or use linear_attention"
        )
    if not require_hip_on_gpu(q):
        _check(q, k, v, log_decay, active, state, scale, 3, "active", "state")
        _check_blocks(state)
        return _eager_step(q, k, v, log_decay, state, active, scale)
    if _is_tracing():
        raise RuntimeError("linear_attention_step cannot be traced on the GPU: the trace would leave it out")
    try:
        return hip_ext().linear_attention_step(q, k, v, log_decay, state, active, scale)
    except RuntimeError:
        # the extension refuses what these do, without the cost of asking twice
        _check(q, k, v, log_decay, active, state, scale, 3, "active", "state")
        _check_blocks(state)
        raise


def _check_blocks(state: torch.Tensor) -> None:
    B, H, Dk, Dv = state.shape
    if not state.numel():
        return
    if (Dv > 1 and state.stride(3) != 1) or (Dk > 1 and state.stride(2) != Dv):
        raise ValueError("each head's [Dk, Dv] block of the state must be contiguous")
    # rows and heads in the order of their strides, each past the one before
    reach = Dk * Dv
    for stride, size in sorted((state.stride(i), state.shape[i]) for i in (0, 1) if state.shape[i] > 1):
        if stride < reach:
            raise ValueError("blocks of the state overlap in memory")
        reach += stride * (size - 1)


@_without_autocast
def _eager_step(q, k, v, log_decay, state, active, scale: float) -> torch.Tensor:
    wide = log_decay.dtype
    qw, kw, vw = q.to(wide), k.to(wide), v.to(wide)
    new = torch.exp(log_decay).view(1, -1, 1, 1) * state + kw[..., :, None] * vw[..., None, :]
    out = (qw[..., :, None] * new).sum(-2) * scale
    if active is not None:
        new = torch.where(active.view(-1, 1, 1, 1), new, state)
        out = torch.where(active.view(-1, 1, 1), out, torch.zeros_like(out))
    state.copy_(new)
    return out.to(q.dtype)
