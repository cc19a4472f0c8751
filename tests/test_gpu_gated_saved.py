"""What gated projections keep for their backward pass."""
import pytest
import torch

from dion_amd import gated_linear, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def tensors(t, k, n):
    gen = torch.Generator(device=DEV).manual_seed(2)
    rnd = lambda *s: torch.empty(*s, device=DEV).normal_(0, 1, generator=gen).bfloat16()  # noqa: E731
    return [rnd(t, k), rnd(n, k), rnd(n, k), rnd(n), rnd(n).float()], rnd(t, n)


@pytest.mark.parametrize("t,k,n", [(24, 40, 56), (33, 77, 130)])
def test_the_weights_are_kept_for_the_gradient_of_x_alone(t, k, n):
    """Without it they may be changed between the two passes; with it autograd refuses the change."""
    operands, dh = tensors(t, k, n)
    every = [p.clone().requires_grad_() for p in operands]
    all_grads = torch.autograd.grad(gated_linear(*every), every, dh)
    for needs in ((0, 1, 1, 1, 1), (0, 1, 0, 0, 0), (0, 0, 1, 1, 0), (0, 0, 0, 1, 0), (0, 0, 0, 1, 1)):
        for change in (False, True):
            leaves = [p.clone().requires_grad_(bool(need)) for p, need in zip(operands, needs)]
            h = gated_linear(*leaves)
            if change:
                with torch.no_grad():
                    leaves[1].mul_(3.0)
                    leaves[2].mul_(3.0)
            grads = torch.autograd.grad(h, [p for p, need in zip(leaves, needs) if need], dh)
            want = [g for g, need in zip(all_grads, needs) if need]
            assert all(torch.equal(p, q) for p, q in zip(grads, want)), needs  # (few tokens: no reduction is split)
    for needs in ((1, 1, 1, 1, 1), (1, 0, 0, 0, 0)):
        for which in (1, 2):
            leaves = [p.clone().requires_grad_(bool(need)) for p, need in zip(operands, needs)]
            h = gated_linear(*leaves)
            with torch.no_grad():
                leaves[which].mul_(3.0)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(h, leaves[0], dh)


def test_operator_call_without_weights():
    (x, wg, wu, _bg, _bu), dh = tensors(12, 40, 24)
    _h, kept = ops.gated_forward(x, wg, wu, None, None, "silu", 24)
    full = ops.gated_backward(dh, kept, 24, x, wg, wu, True, True, True, torch.float32, torch.float32)
    got = ops.gated_backward(dh, kept, 24, x, None, None, False, True, True, torch.float32, torch.float32)
    assert got[0] is None and all(torch.equal(p, q) for p, q in zip(full[1:], got[1:]))
    got = ops.gated_backward(dh, kept, 24, None, None, None, False, False, False, torch.float32, torch.float32)
    assert got[:3] == (None, None, None) and all(torch.equal(p, q) for p, q in zip(full[3:], got[3:]))
    good = dict(dh=dh, kept=kept, keep=24, x=x, weight_gate=wg, weight_up=wu, need_dx=False, need_dgate=True, need_dup=True,
                bias_gate_dtype=None, bias_up_dtype=None)
    for bad in ({"weight_gate": None}, {"weight_up": None}, {"weight_gate": None, "weight_up": None, "need_dx": True}, {"x": None},
                {"weight_gate": None, "weight_up": None, "x": x[:8]}, {"weight_gate": None, "weight_up": None, "x": x[:5], "dh": dh[:5]}):
        with pytest.raises(ValueError, match="gated_linear"):
            ops.gated_backward(**{**good, **bad})
    with pytest.raises(TypeError, match="gated_linear"):
        ops.gated_backward(**{**good, "weight_gate": None, "weight_up": None, "dh": dh.float()})


def test_either_weights_gradient_may_be_changed_in_place():
    """... while a graph keeps the other one, though both lie in one allocation."""
    (x, wg, wu, _bg, _bu), dh = tensors(24, 40, 56)
    wg.requires_grad_(), wu.requires_grad_()
    scale = torch.ones(56, 40, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    for kept in (0, 1):
        grads = torch.autograd.grad(gated_linear(x, wg, wu), [wg, wu], dh)
        want = grads[kept].clone()
        penalty = (grads[kept] * scale).sum()
        grads[1 - kept].zero_()
        assert torch.equal(torch.autograd.grad(penalty, scale)[0], want)
