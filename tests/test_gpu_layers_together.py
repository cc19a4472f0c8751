"""The layers as a model uses them: rows of a table, layer norm, gated projections, the product back into the stream, a head of its own,
trained with Muon on the matrices and AdamW on the rest."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def parameters():
    gen = torch.Generator(device=DEV).manual_seed(5)
    rnd = lambda *s, std: torch.nn.Parameter(torch.empty(*s, device=DEV).normal_(0, std, generator=gen))  # noqa: E731
    p = {"table": rnd(50, 96, std=1.0), "gate": rnd(200, 96, std=0.1), "up": rnd(200, 96, std=0.1), "down": rnd(96, 200, std=0.07)}
    p.update(norm=torch.nn.Parameter(torch.ones(96, device=DEV)), shift=torch.nn.Parameter(torch.zeros(96, device=DEV)))
    return p


def forward(p, ids):
    from dion_amd import embedding, gated_linear, layer_norm, linear

    h = embedding(ids, p["table"], scale=0.5, padding_idx=49, dtype=torch.bfloat16)
    n = layer_norm(h, p["norm"], p["shift"])
    return linear(gated_linear(n, p["gate"].bfloat16(), p["up"].bfloat16()), p["down"].bfloat16(), residual=h)


def exact(p, ids):
    """In float64, with no rounding; row 49 of the table has no gradient."""
    table = p["table"]
    h = 0.5 * torch.where((ids == 49)[..., None], table.detach()[ids], table[ids])
    c = h - h.mean(-1, keepdim=True)
    n = c / ((c * c).mean(-1, keepdim=True) + 1e-5).sqrt() * p["norm"] + p["shift"]
    g = n @ p["gate"].t()
    return (g * torch.sigmoid(g) * (n @ p["up"].t())) @ p["down"].t() + h


def test_a_block_is_trained():
    from dion import Muon

    p = parameters()
    gen = torch.Generator(device=DEV).manual_seed(6)
    ids = torch.randint(0, 50, (4, 33), device=DEV, generator=gen)
    ids[:, 25:] = 49
    target = torch.empty(4, 33, 96, device=DEV).normal_(0, 1, generator=gen)
    opt = Muon([{"params": [p["gate"], p["up"], p["down"]]},
                {"params": [p["table"], p["norm"], p["shift"]], "algorithm": "adamw", "lr": 1e-3, "state_bits": 8}], lr=0.02)
    for k in range(4):
        opt.zero_grad()
        (forward(p, ids).float() - target).square().mean().backward()
        if k == 0:
            q = {n: t.detach().double().requires_grad_() for n, t in p.items()}
            (exact(q, ids) - target.double()).square().mean().backward()
            for n in p:
                # on the way to a gradient at most eight tensors are rounded to bf16 (2^-8 each, at random): the weights, the
                # embedding, the norm, g u, the output, dy and what comes back through the products
                assert float((p[n].grad.double() - q[n].grad).norm() / q[n].grad.norm()) < 8 * 2.0 ** -8, n
        before = {n: t.detach().clone() for n, t in p.items()}
        opt.step()
        assert all(bool(t.isfinite().all()) and not torch.equal(t, before[n]) for n, t in p.items())


def test_the_whole_pass_is_captured():
    p = parameters()
    ids = torch.randint(0, 50, (3, 40), device=DEV)
    dy = torch.randn(3, 40, 96, device=DEV).bfloat16()
    leaves = list(p.values())

    def both():
        y = forward(p, ids)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(4):
        ids.copy_(torch.randint(0, 50, ids.shape, device=DEV))
        dy.copy_(torch.randn(dy.shape, device=DEV))
        with torch.no_grad():
            p["gate"].mul_(0.9)
        eager = [t.clone() for t in both()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), k
