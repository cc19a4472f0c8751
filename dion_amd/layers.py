"""What stands before and between the products of weights, with its gradients: rows of a table of embeddings, and layer norm.  Their
parameters are those that the optimizers' AdamW and Lion groups hold.
"""
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import ops
from .linear import _check_capture, _once, _refuse_tangents


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, dtype):
        y, stats = ops.layer_norm_forward(x, weight, bias, eps, dtype, True)
        need = ctx.needs_input_grad
        ctx.save_for_backward(x if need[0] or need[1] else None, weight if need[0] else None, stats)
        ctx.dtypes = bias.dtype if bias is not None and need[2] else None, weight.dtype if weight is not None else None
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*ops.layer_norm_backward(dy, x, weight, stats, need[0], need[1], *ctx.dtypes), None, None)


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5,
               dtype: Optional[torch.dtype] = None) -> Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension: ``x [..., width]``, ``weight`` and ``bias``
    ``[width]``, bfloat16 or float32 each; the result is of ``dtype`` (None: that of ``x``).  ``var`` is the mean square of the centred
    values; arithmetic and sums are float32, and the result is rounded once.  A row whose squared distances from its mean add up past float32
    (values past about 1.8e19 / sqrt(width)) comes out as the bias, with a gradient of zero; one whose values do (past 3.4e38 / width, of
    one sign) as NaN.

    Differentiable once with respect to every tensor, in reverse mode (a forward-mode tangent is refused: NotImplementedError).  For
    the backward pass it keeps two float32 values a row, ``x`` where it or the weight needs a gradient, and the weight where ``x`` does.  Gradients are of their tensor's type, sums of
    the weight's and the bias's float32 until they are rounded, and repeat bit for bit.  Any strides (a last dimension that is not
    contiguous is copied), up to 2^30 rows and 2^24 columns.  Captures as for ``linear``."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, weight, bias, op="layer_norm")
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        y = _LayerNorm.apply(x, weight, bias, eps, dtype)
        _check_capture(y, weight, bias, op="layer_norm")
        return y
    return ops.layer_norm_forward(x, weight, bias, eps, dtype, False)[0]


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx, dtype):
        ctx.save_for_backward(ids)
        ctx.table = weight.shape[0], scale, padding_idx, weight.dtype
        return ops.embedding_forward(ids, weight, scale, dtype)

    @staticmethod
    @_once
    def backward(ctx, dy):
        ids = ctx.saved_tensors[0]
        return None, ops.embedding_backward(dy, ids, *ctx.table), None, None, None


def embedding(ids: Tensor, weight: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None,
              dtype: Optional[torch.dtype] = None) -> Tensor:
    """``scale * weight[ids]``: ``ids`` int64 or int32 of any shape, ``weight [vocab, width]`` bfloat16 or float32; the result
    ``[..., width]`` is of ``dtype`` (None: that of the weight) and rounded once.  An id outside the table gives a row of NaN and no
    gradient.

    Differentiable once with respect to the weight, in reverse mode (a forward-mode tangent is refused: NotImplementedError).  Its
    gradient is dense, of the weight's type: every row is ``scale`` times the float32 sum of the gradients of its tokens, added in their
    order, so that it repeats bit for bit; that of row ``padding_idx`` (negative: from the end) is zero.  For the backward
    pass it keeps ``ids``.  At most 2^24 rows and 2^30 tokens.  Captures as for ``linear``."""
    if padding_idx is not None:
        rows = weight.shape[0] if weight.dim() else 0
        if not -rows <= padding_idx < rows:
            raise ValueError(f"embedding: padding_idx {padding_idx} is outside a table of {rows} rows")
        padding_idx %= rows
    if forward_ad._current_level >= 0:
        _refuse_tangents(weight, op="embedding")
    if torch.is_grad_enabled() and weight.requires_grad:
        y = _Embedding.apply(ids, weight, scale, padding_idx, dtype)
        _check_capture(y, weight, op="embedding")
        return y
    return ops.embedding_forward(ids, weight, scale, dtype)
