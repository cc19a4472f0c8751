"""A captured pass whose weight is a cast of an fp32 leaf."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_a_captured_pass_of_a_cast_weight():
    from dion_amd import linear

    gen = torch.Generator(device=DEV).manual_seed(6)
    rnd = lambda *s: torch.empty(*s, device=DEV).normal_(0, 1, generator=gen)  # noqa: E731
    w, b = rnd(136, 72).requires_grad_(), rnd(136).requires_grad_()
    x, dy = rnd(50, 72).bfloat16(), rnd(50, 136).bfloat16()

    def both():
        y = linear(linear(x, w.bfloat16(), b, activation="silu"), w.t().bfloat16()[:, :136])
        return (y.detach(), *torch.autograd.grad(y, (w, b), dy[:, :72]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.synchronize()
    alive = linear(x, w.bfloat16())
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="still has its graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            linear(x, w.bfloat16())
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(4):
        x.copy_(rnd(50, 72))
        eager = [t.clone() for t in both()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager)), k
