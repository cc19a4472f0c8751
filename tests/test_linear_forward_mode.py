"""Forward-mode derivatives of the product of a weight: refused, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from dion_amd import linear


def operands(device="cpu"):
    bf = lambda *s: torch.ones(*s, dtype=torch.bfloat16, device=device)  # noqa: E731
    return [bf(4, 8), bf(16, 8), bf(16), bf(4, 16)]


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_is_refused(which, grad):
    ts = operands()
    if grad:
        ts[1].requires_grad_()
    with fwd.dual_level():
        ts[which] = fwd.make_dual(ts[which], torch.ones_like(ts[which]))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                linear(ts[0], ts[1], ts[2], activation="silu", residual=ts[3])


@pytest.mark.gpu
def test_operands_without_a_tangent_in_a_dual_level():
    x, w, b, r = operands("cuda")
    want = linear(x, w, b, activation="gelu", residual=r)
    w.requires_grad_()
    with fwd.dual_level():
        y = linear(x, w, b, activation="gelu", residual=r)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            linear(fwd.make_dual(x, x), w)
    assert torch.equal(y, want) and torch.autograd.grad(y.sum(), w)[0].shape == w.shape
