"""Activations of a weight's product and their slopes at finite values whose squares or doubles pass fp32."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("act", [None, "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("tokens", [16, 300])
def test_huge_values(act, tokens):
    """Past 100 every one of these activations is z or 0 to fp32's last bit, and its slope 1 or 0 (in float64 too: the tails are
    below e^-100 z)."""
    from dion_amd import linear

    size = torch.tensor([1e2, 1e3, 1e6, 1e12, 1e18, 2e19, 1e22, 1e30, 1e37, 1.6e38, 2e38, 3e38], device=DEV)
    z = torch.cat([size, -size]).repeat(13)[:tokens].bfloat16()
    x = torch.zeros(tokens, 8, device=DEV, dtype=torch.bfloat16)
    x[:, 0] = z
    w = torch.zeros(16, 8, device=DEV, dtype=torch.bfloat16)
    w[:, 0] = 1
    xl = x.requires_grad_()
    y = linear(xl, w, activation=act)
    want = z.clamp_min(0) if act else z
    # (silu's and gelu's tails at -100 are below 1e-40, which bf16 of fp32's flushed results may give as zero)
    assert bool(((y - want[:, None]).abs() <= 1e-38).all()), (act, y[:, 0], z)
    dy = torch.zeros_like(y)
    dy[:, 3] = 1.0
    (dx,) = torch.autograd.grad(y, xl, dy)
    assert torch.equal(dx[:, 0], (z > 0).to(dx.dtype) if act else torch.ones_like(z)), (act, dx[:, 0], z)
