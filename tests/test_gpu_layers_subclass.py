"""Operands of a class of one's own that holds its data as any tensor does."""
import pytest
import torch

from dion_amd import embedding, gated_linear, layer_norm, linear

pytestmark = pytest.mark.gpu


class Named(torch.Tensor):
    pass


CALLS = {"linear": (lambda a, b, c: linear(a, b, c[0], activation="silu"), 3), "gated_linear": (lambda a, b, c: gated_linear(a, b, c), 3),
         "layer_norm": (lambda a, b, c: layer_norm(a, b[0], c[0]), 3),
         "embedding": (lambda a, b, c: embedding(torch.arange(6, device="cuda").as_subclass(type(c)), a), 1)}


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("name", CALLS)
def test_a_class_of_ones_own(name, which):
    gen = torch.Generator(device="cuda").manual_seed(1)
    operands = [torch.empty(16, 16, device="cuda").normal_(0, 1, generator=gen).bfloat16() for _ in range(3)]
    call, used = CALLS[name]
    got = []
    for kind in (torch.Tensor, Named):
        leaves = [(t.clone().as_subclass(kind) if i == which else t.clone()).requires_grad_() for i, t in enumerate(operands)]
        y = call(*leaves)
        got.append((y, *torch.autograd.grad(y, leaves[:used], torch.ones_like(y))))
    assert all(torch.equal(p, q) for p, q in zip(*got))
