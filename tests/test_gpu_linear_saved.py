"""What the product of a weight keeps for its backward pass."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("t,k,n", [(24, 40, 56), (33, 77, 130)])
def test_the_weight_is_kept_for_the_gradient_of_x_alone(act, t, k, n):
    """Without it the weight may be changed, or go, between the two passes; with it autograd refuses the change."""
    from dion_amd import linear

    gen = torch.Generator(device=DEV).manual_seed(2)
    rnd = lambda *s: torch.empty(*s, device=DEV).normal_(0, 1, generator=gen).bfloat16()  # noqa: E731
    x, w, b, dy = rnd(t, k), rnd(n, k), rnd(n), rnd(t, n)
    for needs in ((False, True, True), (False, False, True), (False, True, False)):
        got = []
        for change in (False, True):
            leaves = [p.clone().requires_grad_(need) for p, need in zip((x, w, b), needs)]
            y = linear(*leaves, activation=act)
            if change:
                with torch.no_grad():
                    leaves[1].mul_(3.0)
            got.append(torch.autograd.grad(y, [p for p, need in zip(leaves, needs) if need], dy))
        assert all(torch.equal(p, q) for p, q in zip(*got)), needs
    for act_needs in ((True, True, True), (True, False, False)):
        leaves = [p.clone().requires_grad_(need) for p, need in zip((x, w, b), act_needs)]
        y = linear(*leaves, activation=act)
        with torch.no_grad():
            leaves[1].mul_(3.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, leaves[0], dy)


def test_operator_call_without_a_weight():
    from dion_amd import ops

    gen = torch.Generator(device=DEV).manual_seed(4)
    rnd = lambda *s: torch.empty(*s, device=DEV).normal_(0, 1, generator=gen).bfloat16()  # noqa: E731
    x, w, dy = rnd(12, 40), rnd(24, 40), rnd(12, 24)
    _dx, dw, db = ops.linear_backward(dy, None, None, x, w, True, True, torch.float32)
    none, dw2, db2 = ops.linear_backward(dy, None, None, x, None, False, True, torch.float32)
    assert none is None and torch.equal(dw, dw2) and torch.equal(db, db2)
    none, none2, db3 = ops.linear_backward(dy, None, None, None, None, False, False, torch.float32)
    assert none is None and none2 is None and torch.equal(db, db3)
    with pytest.raises(ValueError, match="linear"):
        ops.linear_backward(dy, None, None, x, None, True, True, torch.float32)
    with pytest.raises(ValueError, match="linear"):
        ops.linear_backward(dy, None, None, x[:8], None, False, True, torch.float32)
    with pytest.raises(TypeError):
        ops.linear_backward(dy.float(), None, None, x, None, False, True, torch.float32)
    with pytest.raises(ValueError, match="unknown activation"):
        ops.linear_backward(dy, None, "swish", x, None, False, True, torch.float32)
