"""The product a weight matrix stands for, with its bias, activation and residual in one kernel, and both projections of a gated
feed-forward block with their product in one, and their gradients: what the matrices that the optimizers update compute, and where
their gradients come from.
"""
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, residual):
        need = ctx.needs_input_grad
        y, slope = ops.linear_forward(x, weight, bias, activation, residual, need[0] or need[1] or need[2])
        ctx.save_for_backward(x if need[1] else None, weight if need[0] else None, slope)
        ctx.activation = activation
        ctx.bias_dtype = bias.dtype if bias is not None and need[2] else None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, slope = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[1] or ctx.bias_dtype is not None:
            dx, dw, db = ops.linear_backward(dy, slope, ctx.activation, x, weight, need[0], need[1], ctx.bias_dtype)
        return dx, dw, db, None, dy if need[4] else None


# A leaf's accumulation node runs on the stream on which it was made and lives as long as a graph that holds it.  Recorded by a
# capture, a backward pass that meets a node of another stream makes that stream wait inside the capture, and torch then ends the
# process.  torch does not say which stream that is, so a node keeps the stream of the first product that it is seen in: as a
# leaf among the operands, or below a weight or bias that is a cast or view of one.  A capture looks at every node below its result and
# is refused before its backward pass where one has another stream.
_ACCUMULATE = type(torch.autograd.graph.get_gradient_edge(torch.zeros((), requires_grad=True)).node)
_STREAM, _EAGER, _CAPTURED = ("dion_amd.linear: " + key for key in ("stream", "leaves noted on", "leaves captured on"))


def _below(node) -> list:
    return [below for below, _index in node.next_functions]


def _check_leaves(nodes: list, device: torch.device, stream: int, capturing: bool, op: str = "linear") -> None:
    """Looks at every leaf below ``nodes``; a node that an earlier call has looked below is passed by."""
    done, seen = _CAPTURED if capturing else _EAGER, set()
    while nodes:
        node = nodes.pop()
        if node is None or node in seen:
            continue
        if not isinstance(node, _ACCUMULATE):
            if node.metadata.get(done) != stream:
                seen.add(node)
                nodes.extend(_below(node))
        elif node.variable.device == device and node.metadata.setdefault(_STREAM, stream) != stream and capturing:
            raise RuntimeError(f"{op}: captured while a result of an earlier call with the same leaf, on another stream, still "
                               "has its graph; delete or detach that result first")
    for node in seen:  # (only here: none of them stays marked where one was refused)
        node.metadata[done] = stream


def _check_capture(y: Tensor, *weights: Optional[Tensor], op: str = "linear") -> None:
    stream = ops._stream_handle(y.device)
    with ops._device_of(y):
        capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        nodes = [y.grad_fn]
    else:
        nodes = [node for node in _below(y.grad_fn) if isinstance(node, _ACCUMULATE)]
        nodes += [t.grad_fn for t in weights if t is not None and t.grad_fn is not None]
    _check_leaves(nodes, y.device, stream, capturing, op)


# The kernels have no tangents, and a tensor can have one without requires_grad.
def _refuse_tangents(*operands: Optional[Tensor], op: str = "linear") -> None:
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in operands):
        raise NotImplementedError(f"{op}: forward-mode derivatives are not supported")


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: Optional[str] = None,
           residual: Optional[Tensor] = None) -> Tensor:
    """``act(x W^T + b) + residual``: ``x [..., fan_in]``, ``weight [fan_out, fan_in]``, ``residual [..., fan_out]`` bfloat16,
    ``bias [fan_out]`` bfloat16 or float32; returns bfloat16 ``[..., fan_out]``.  ``activation``: None, "relu", "relu_squared",
    "gelu" (by the error function), "gelu_tanh" or "silu".  Sums are float32, and the result is rounded once.

    Differentiable once with respect to every tensor, in reverse mode (a forward-mode tangent is refused: NotImplementedError).  For
    the backward pass it keeps ``x`` where the weight needs a gradient, the weight where ``x`` does and, with an activation, its
    slopes in 16 bits an element; what it keeps must not change between the two passes (autograd raises).  The gradient that
    reaches ``z = x W^T + b`` is rounded to bfloat16 for the two products, not for the bias.  Any sizes and strides, up to
    2^21 - 8 features and 2^30 tokens; rows that are not whole 16-byte chunks (feature counts that are not multiples of 8) are
    copied first.

    Both passes can be captured into a graph, together, while no result of an earlier call on the same leaves on another
    stream has its autograd graph: that is refused (RuntimeError), for leaves among the operands and below a weight or bias that is
    a cast or a view.  A leaf that another operation has used on another stream, and whose result still has its graph, is not
    noticed: torch ends the process in the backward pass of such a capture, as it does without this product."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, weight, bias, residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        y = _Linear.apply(x, weight, bias, activation, residual)
        _check_capture(y, weight, bias)
        return y
    return ops.linear_forward(x, weight, bias, activation, residual, False)[0]


def _once(backward):
    """``once_differentiable`` where the pass is recorded for another derivative; otherwise the function itself, which then costs less."""
    recorded = once_differentiable(backward)
    return lambda ctx, dy: (recorded if torch.is_grad_enabled() else backward)(ctx, dy)


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight_gate, weight_up, bias_gate, bias_up, activation):
        need = ctx.needs_input_grad
        biases = ((bias_gate, need[3]), (bias_up, need[4]))
        ctx.bias_dtypes = [b.dtype if b is not None and n else None for b, n in biases]
        # (sums that are stored as float32 are worth it; whether one is asked for does not change the other gradients)
        ctx.keep = 32 if any(b is not None and b.dtype == torch.float32 for b, _ in biases) else 24
        h, kept = ops.gated_forward(x, weight_gate, weight_up, bias_gate, bias_up, activation, ctx.keep)
        weights = (weight_gate, weight_up) if need[0] else (None, None)
        ctx.save_for_backward(x if need[1] or need[2] else None, *weights, kept)
        return h

    @staticmethod
    @_once
    def backward(ctx, dh):
        need = ctx.needs_input_grad
        x, weight_gate, weight_up, kept = ctx.saved_tensors
        return (*ops.gated_backward(dh, kept, ctx.keep, x, weight_gate, weight_up, *need[:3], *ctx.bias_dtypes), None)


def gated_linear(x: Tensor, weight_gate: Tensor, weight_up: Tensor, bias_gate: Optional[Tensor] = None,
                 bias_up: Optional[Tensor] = None, activation: Optional[str] = "silu") -> Tensor:
    """Both projections of a gated feed-forward block, ``act(x Wg^T + bg) * (x Wu^T + bu)``: ``x [..., fan_in]``, the weights
    ``[fan_out, fan_in]`` bfloat16 (the two halves of one tensor, or any two), the biases ``[fan_out]`` bfloat16 or float32;
    returns bfloat16 ``[..., fan_out]``.  ``activation``: as for ``linear``; None for the product of the projections alone.  Sums are
    float32, and the result is rounded once.

    Differentiable once with respect to every tensor, in reverse mode (a forward-mode tangent is refused: NotImplementedError).  For
    the backward pass it keeps ``x`` where a weight needs a gradient, the weights where ``x`` does, and ``act(g)`` and ``act'(g) u`` in
    24 bits each (32 beside a float32 bias); the gradients that reach the two projections are rounded to bfloat16 for the products, not for the biases.  The gradients of the two
    weights, where both are asked for, share an allocation.  Sizes, strides and captures as for ``linear``, up to 2^20 - 8
    columns of the result."""
    operands = (x, weight_gate, weight_up, bias_gate, bias_up)
    if forward_ad._current_level >= 0:
        _refuse_tangents(*operands, op="gated_linear")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands):
        h = _GatedLinear.apply(*operands, activation)
        _check_capture(h, *operands[1:], op="gated_linear")
        return h
    return ops.gated_forward(*operands, activation, 0)[0]
