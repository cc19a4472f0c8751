"""What layer norm keeps for its backward pass."""
import itertools

import pytest
import torch

from dion_amd import layer_norm, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float32


def tensors(rows, d, x, p, y):
    gen = torch.Generator(device=DEV).manual_seed(rows + d)
    rnd = lambda *s: torch.empty(*s, device=DEV).normal_(0, 1, generator=gen)  # noqa: E731
    return [rnd(rows, d).to(x), rnd(d).to(p), rnd(d).to(p)], rnd(rows, d).to(y)


# few rows, many, rows that are read again; whole pieces, pairs, single elements
@pytest.mark.parametrize("rows,d", [(30, 72), (30, 77), (1500, 770), (1500, 1001), (1100, 2048), (40, 20001), (7, 12290)])
@pytest.mark.parametrize("x,p,y", [(BF, FP, BF), (FP, BF, BF), (BF, BF, FP)])
def test_only_what_a_gradient_reads_is_kept(rows, d, x, p, y):
    """x may be changed between the passes where only the bias needs a gradient, the weight where x needs none; autograd refuses the rest."""
    operands, dy = tensors(rows, d, x, p, y)
    every = [t.clone().requires_grad_() for t in operands]
    all_grads = torch.autograd.grad(layer_norm(*every, dtype=y), every, dy)
    for needs in itertools.product((False, True), repeat=3):
        if not any(needs):
            continue
        for which in (0, 1):
            leaves = [t.clone().requires_grad_(need) for t, need in zip(operands, needs)]
            out = layer_norm(*leaves, dtype=y)
            with torch.no_grad():
                leaves[which].fill_(float("nan"))
            grads = lambda: torch.autograd.grad(out, [t for t in leaves if t.requires_grad], dy)  # noqa: E731
            if needs[0] or which == 0 and needs[1]:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    grads()
            else:
                assert all(torch.equal(g, w) for g, w in zip(grads(), [w for w, need in zip(all_grads, needs) if need])), needs


def test_operator_call_without_x_or_the_weight():
    (x, w, b), dy = tensors(20, 40, BF, FP, FP)
    _y, stats = ops.layer_norm_forward(x, w, b, 1e-5, FP, True)
    _dx, dw, db = ops.layer_norm_backward(dy, x, w, stats, True, True, BF)
    got = ops.layer_norm_backward(dy, x, None, stats, False, True, BF, FP)
    assert got[0] is None and torch.equal(got[1], dw) and torch.equal(got[2], db)
    got = ops.layer_norm_backward(dy, None, None, stats, False, False, BF)
    assert got[:2] == (None, None) and torch.equal(got[2], db)
    good = dict(dy=dy, x=x, weight=w, stats=stats, need_dx=True, need_dw=True, bias_dtype=BF)
    for bad in ({"x": None}, {"x": None, "need_dx": False}, {"weight": None}, {"x": None, "need_dx": False, "need_dw": False, "dy": dy[:5]}):
        with pytest.raises(ValueError, match="layer_norm"):
            ops.layer_norm_backward(**{**good, **bad})
    with pytest.raises(TypeError, match="layer_norm"):
        ops.layer_norm_backward(**{**good, "weight_dtype": torch.float16})
    with pytest.raises(TypeError, match="layer_norm"):
        ops.layer_norm_backward(**{**good, "x": None, "need_dx": False, "need_dw": False, "dy": dy.half()})
