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


@pytest.mark.parametrize("rows", [2 ** 26 - 3, 2 ** 26 + 77])
def test_layer_norm(rows):
    """A wavefront a row; every row is one of five, and its results those of a call on few of them."""
    from dion_amd import layer_norm

    few = torch.randn(1000, 8, device=DEV).to(BF)
    few = few[:5].repeat(200, 1)
    dfew = torch.randn(5, 8, device=DEV).to(BF).repeat(200, 1)
    w = (1 + 0.3 * torch.randn(8, device=DEV)).requires_grad_()
    x = few[:5].repeat(rows // 5 + 1, 1)[:rows].requires_grad_()
    dy = dfew[:5].repeat(rows // 5 + 1, 1)[:rows]
    z = torch.full((rows, 8), 7.0, device=DEV, dtype=BF)
    del z
    y, want = layer_norm(x, w), layer_norm(few, w)
    (dx,) = torch.autograd.grad(y, x, dy, retain_graph=True)
    leaf = few.detach().requires_grad_()
    (dwant,) = torch.autograd.grad(layer_norm(leaf, w), leaf, dfew)
    for got, five in ((y.detach(), want[:5].detach()), (dx, dwant[:5])):
        for a, b in pieces(rows, 5 << 22):
            assert torch.equal(got[a:b], five.repeat((b - a) // 5 + 1, 1)[:b - a]), a
    # The sums: rows / 4096 additions in a group of wavefronts, 4 where a workgroup's meet, 256 parts.  xh: 8 additions and a product for the
    # mean and for the variance, whose error counts half, and five roundings: 16 of the value and of what the mean adds to it.
    (dw,) = torch.autograd.grad(y, w, dy)
    times = torch.bincount(torch.arange(rows, device=DEV) % 5).double()[:, None]
    five = few[:5].double()
    c = five - five.mean(1, keepdim=True)
    r = 1 / ((c * c).mean(1, keepdim=True) + 1e-5).sqrt()
    xh, d = c * r, dfew[:5].double()
    off = 16 * 2.0 ** -24 * (d.abs() * (xh.abs() + five.abs().mean(1, keepdim=True) * r) * times).sum(0)
    off += (rows / 4096 + 4 + 256) * 2.0 ** -24 * ((d * xh).abs() * times).sum(0)
    assert bool(((dw.double() - (d * xh * times).sum(0)).abs() <= off).all())
