"""Results changed in place, as a residual addition or a dropout does, whatever the input's number of dimensions."""
import pytest
import torch

from dion_amd import embedding, gated_linear, layer_norm, linear

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("lead", [(), (6,), (2, 3), (1, 2, 3), (0, 3)])
@pytest.mark.parametrize("name", ["linear", "linear_silu", "gated_linear", "layer_norm", "embedding"])
def test_a_result_changed_in_place(name, lead):
    gen = torch.Generator(device=DEV).manual_seed(5)
    rnd = lambda *s: torch.empty(*s, device=DEV).normal_(0, 1, generator=gen).bfloat16()  # noqa: E731
    x, w, u, res, dy = rnd(*lead, 24), rnd(24, 24), rnd(24, 24), rnd(*lead, 24), rnd(*lead, 24)
    ids = torch.arange(res[..., 0].numel(), device=DEV).view(lead) % 5
    got = []
    for in_place in (False, True):
        leaves = [t.clone().requires_grad_() for t in (x, w, u, res)]
        call = {"linear": lambda: linear(leaves[0], leaves[1]), "linear_silu": lambda: linear(leaves[0], leaves[1], activation="silu"),
                "gated_linear": lambda: gated_linear(*leaves[:3]), "layer_norm": lambda: layer_norm(leaves[0], leaves[1][0]),
                "embedding": lambda: embedding(ids, leaves[1])}[name]
        y = call()
        assert not y._is_view()
        if in_place:
            y += leaves[3]
            y.mul_(2.0)
        else:
            y = (y + leaves[3]) * 2.0
        got.append((y, *torch.autograd.grad(y, leaves, dy, allow_unused=True)))
    for p, q in zip(*got):
        assert (p is None and q is None) or torch.equal(p, q)
