"""Linear layer with bias, activation and residual in its epilogue.

    y = act(x W^T + bias) + residual

One product instead of a product and up to three passes over its output, and
a backward pass whose products are the framework's own kernels too
(``hip/fused_linear.hip``).  CPU path: explicit torch math; GPU path: falls
back loudly per replay_amd.ops.require_hip_on_gpu.

Products and sums are float32 with one rounding of the result.  Two more in the
backward pass of an activation, both to the inputs' type: the slope is taken at
``x W^T + bias`` as kept from the forward pass, and dy times the slope is what the
products for dx and dW read (the bias gradient sums it before that rounding).

Beside :class:`replay_amd.ops.fast_linear.ChunkedWgradLinear` this is the form
for layers whose activation or residual follows at once
(:class:`replay_amd.nn.ffn.PointWiseFeedForward` with ``fused=True``).
"""

from __future__ import annotations

from typing import Optional

import torch
from torch._C import _is_tracing  # torch.jit.is_tracing() without its 0.4 us
from torch.autograd.function import once_differentiable

from replay_amd.ops import hip_ext, require_hip_on_gpu

#: the names, and their codes in the extension
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def eager_fused_linear(x, weight, bias, activation: str, residual) -> torch.Tensor:
    z = torch.nn.functional.linear(x, weight, bias)
    if activation == "relu":
        z = torch.relu(z)
    elif activation == "gelu":
        z = torch.nn.functional.gelu(z)
    elif activation == "silu":
        z = torch.nn.functional.silu(z)
    return z if residual is None else z + residual


class FusedLinearFunction(torch.autograd.Function):
    """Saves x, the weight, and what the activation's slope is taken at: the
    product before the activation, or for relu without a residual the output."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        grads = any(ctx.needs_input_grad[:3])
        from_y = act == ACTIVATIONS["relu"] and residual is None
        y, z = hip_ext().fused_linear_fwd(x, weight, bias, residual, act, grads and act != 0 and not from_y)
        if grads:
            ctx.save_for_backward(x, weight, y if from_y else z)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            x, weight, z = ctx.saved_tensors
            dx, dw, db = hip_ext().fused_linear_bwd(dy, x, weight, z, ctx.act, need_x, need_w, need_b)
        return (
            dx if need_x else None,
            dw if need_w else None,
            db if need_b else None,
            dy if need_r else None,
            None,
        )


def _autocast(dtype: torch.dtype, *given: Optional[torch.Tensor]):
    """What autocast makes of a linear layer's tensors: float64 and integers stay."""
    return (
        t.to(dtype) if t is not None and t.is_floating_point() and t.dtype != torch.float64 else t for t in given
    )


def _check(x, weight, bias, residual) -> None:
    given = [t for t in (x, weight, bias, residual) if t is not None]
    if any(t.device != x.device for t in given):
        raise ValueError("x, weight, bias and residual must be on one device")
    if any(t.dtype != x.dtype for t in given):
        raise ValueError("x, weight, bias and residual must share one dtype")
    if x.dtype not in (_DTYPES if x.is_cuda else (*_DTYPES, torch.float64)):
        raise ValueError(f"unsupported dtype {x.dtype}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x [..., K] and weight [N, K] do not fit: {tuple(x.shape)}, {tuple(weight.shape)}")
    N = weight.shape[0]
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"bias must be ({N},), got {tuple(bias.shape)}")
    shape = (*x.shape[:-1], N)
    if residual is not None and residual.shape != shape:
        raise ValueError(f"residual must be {shape}, got {tuple(residual.shape)}")


def fused_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    activation: str = "none",
    residual: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``.

    :param x: [..., K]; bfloat16, float16 or float32.
    :param weight: [N, K], as ``torch.nn.Linear`` keeps it; bias: [N].
    :param activation: "none", "relu", "gelu" (by erf) or "silu".
    :param residual: [..., N], of x's leading dimensions; never broadcast.
    :return: [..., N] in the inputs' dtype, accumulated in float32.

    All tensors share dtype and device; under autocast they are cast to its
    dtype first, as ``torch.nn.Linear``'s are (which leaves float64 as it is).
    Differentiable once, on the GPU in reverse mode alone (a dual tensor is
    refused there).
    """
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    kind = "cuda" if x.is_cuda else "cpu"
    if torch.is_autocast_enabled(kind):
        x, weight, bias, residual = _autocast(torch.get_autocast_dtype(kind), x, weight, bias, residual)
    if not require_hip_on_gpu(x):
        _check(x, weight, bias, residual)
        return eager_fused_linear(x, weight, bias, activation, residual)
    try:
        # a trace records the autograd function, but not the extension's call
        if _is_tracing() or torch.is_grad_enabled() and (
            x.requires_grad or weight.requires_grad
            or (bias is not None and bias.requires_grad)
            or (residual is not None and residual.requires_grad)
        ):
            return FusedLinearFunction.apply(x, weight, bias, residual, act)
        return hip_ext().fused_linear_fwd(x, weight, bias, residual, act, False)[0]
    except RuntimeError:
        # the extension refuses what _check does, without the cost of asking twice
        _check(x, weight, bias, residual)
        raise


def fused_linear_residual(
    x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], residual: torch.Tensor
) -> torch.Tensor:
    """``x @ weight.T + bias + residual`` for a residual stream: in one product
    where the residual has the product's type.  A wider one (float32 under
    autocast) is added in its own type instead, so that a stream of blocks is
    not rounded to 16 bits by each."""
    kind = "cuda" if x.is_cuda else "cpu"
    dt = torch.get_autocast_dtype(kind) if torch.is_autocast_enabled(kind) else x.dtype
    if torch.promote_types(dt, residual.dtype) != dt:
        return fused_linear(x, weight, bias) + residual
    return fused_linear(x, weight, bias, residual=residual)
