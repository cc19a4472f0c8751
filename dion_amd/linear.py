"""The product a weight matrix stands for, with its bias, activation and residual in one kernel, and its gradients: what the
matrices that the optimizers update compute, and where their gradients come from.
"""
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import ops


def _rows(t: Optional[Tensor]) -> Optional[Tensor]:
    return t if t is None or t.dim() == 2 else t.reshape(-1, t.shape[-1])


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, residual):
        need = ctx.needs_input_grad
        y, slope = ops.linear_forward(_rows(x), weight, bias, activation, _rows(residual), need[0] or need[1] or need[2])
        ctx.save_for_backward(x if need[1] else None, weight, slope)
        ctx.activation, ctx.lead = activation, x.shape[:-1]
        ctx.bias_dtype = bias.dtype if bias is not None and need[2] else None
        return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, slope = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[1] or ctx.bias_dtype is not None:
            dx, dw, db = ops.linear_backward(_rows(dy), slope, ctx.activation, _rows(x), weight, need[0], need[1],
                                             ctx.bias_dtype)
            if dx is not None and len(ctx.lead) != 1:
                dx = dx.view(*ctx.lead, weight.shape[1])
        return dx, dw, db, None, dy if need[4] else None


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: Optional[str] = None,
           residual: Optional[Tensor] = None) -> Tensor:
    """``act(x W^T + b) + residual``: ``x [..., fan_in]``, ``weight [fan_out, fan_in]``, ``residual [..., fan_out]`` bfloat16,
    ``bias [fan_out]`` bfloat16 or float32; returns bfloat16 ``[..., fan_out]``.  ``activation``: None, "relu", "relu_squared",
    "gelu" (by the error function), "gelu_tanh" or "silu".  Sums are float32, and the result is rounded once.

    Differentiable once with respect to every tensor.  For the backward pass it keeps ``x``, the weight and, with an
    activation, its slopes in 16 bits an element; the gradient that reaches ``z = x W^T + b`` is rounded to bfloat16 for the two
    products, not for the bias.  Any sizes and strides; rows that are not whole 16-byte chunks (feature counts that are not
    multiples of 8) are copied first."""
    ops.check_linear(x, weight, bias, activation, residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, activation, residual)
    y, _slope = ops.linear_forward(_rows(x), weight, bias, activation, _rows(residual), False)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.shape[0])
