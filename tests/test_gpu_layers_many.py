"""More rows than one launch has threads for: what a launch counts modulo 2^32 would leave the rest of a result unwritten."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float32


def pieces(n, step=1 << 24):
    return ((a, min(a + step, n)) for a in range(0, n, step))


# (a wavefront a token, and two)
@pytest.mark.parametrize("tokens,width", [(2 ** 26 - 3, 8), (2 ** 26 + 77, 8), (2 ** 25 + 3, 257)])
def test_rows_of_a_table(tokens, width):
    from dion_amd import embedding

    ids = (torch.arange(tokens, device=DEV, dtype=torch.int32) * 7).remainder_(5)
    w = torch.randn(5, width, device=DEV).to(BF)
    y = torch.full((tokens, width), 7.0, device=DEV, dtype=BF)  # (what the result's memory may hold)
    del y
    y = embedding(ids, w)
    for a, b in pieces(tokens):
        assert torch.equal(y[a:b], w[ids[a:b].long()]), a


def test_their_gradient():
    from dion_amd import embedding

    tokens = 2 ** 26 + 77
    ids = (torch.arange(tokens, device=DEV, dtype=torch.int32) * 7).remainder_(5)
    w = torch.randn(5, 8, device=DEV).requires_grad_()
    y = embedding(ids, w, dtype=BF)
    (g,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert torch.equal(g, torch.bincount(ids, minlength=5)[:, None].float().expand(5, 8))  # (whole numbers below 2^24)
