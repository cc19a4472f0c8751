"""AdamW with moments in 8 bits where gradients are exactly zero beside live ones, as the rows of tokens that do not
occur have them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def fresh(x):
    n = x.numel()
    blocks = -(-n // 128)
    return (torch.zeros(n, dtype=torch.int8, device=DEV), torch.zeros(blocks, device=DEV),
            torch.zeros(n, dtype=torch.uint8, device=DEV), torch.zeros(blocks, device=DEV))


def update(x, g, state, step, lr=1e-3, wd=0.0, cautious=False, seed=0, eps=1e-8):
    from dion_amd import ops

    m, ms, v, vs = state
    ops.adamw8_step([x], [g], [m], [ms], [v], [vs], [step], torch.tensor(lr, device=DEV), 0.9, 0.95, wd, eps, cautious, seed=seed)


@pytest.mark.parametrize("xdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width,cautious", [(3, False), (1001, True)])
def test_elements_without_a_gradient_stand_still(xdt, gdt, width, cautious):
    """Every other run of ``width`` elements has no gradient, in blocks that the others keep alive: its codes stay zero and its
    parameters the same bits, whatever the random numbers are (10^7 of them without a gradient, five steps)."""
    gen = torch.Generator(device=DEV).manual_seed(width)
    n = 20_000_003
    x = torch.empty(n, device=DEV).normal_(0, 0.1, generator=gen).to(xdt)
    still = torch.arange(n, device=DEV) // width % 2 == 0
    held, state, step = x[still], fresh(x), torch.zeros((), device=DEV)
    for _ in range(5):
        g = torch.empty(n, device=DEV).normal_(0, 1e-4, generator=gen).masked_fill_(still, 0.0).to(gdt)
        update(x, g, state, step, cautious=cautious, seed=12)
        assert not bool(state[0][still].any()) and not bool(state[2][still].any())
        assert torch.equal(x[still], held)
    assert bool((state[0][~still] != 0).any()) and int(state[2][~still].min()) >= 1


def test_elements_without_a_gradient_only_decay():
    n = 6_000_000
    x, still = torch.ones(n, device=DEV), torch.arange(n, device=DEV) % 2 == 0
    g = torch.full((n,), 1e-3, device=DEV).masked_fill_(still, 0.0)
    state, step, want = fresh(x), torch.zeros((), device=DEV), torch.ones((), device=DEV)
    keep = 1 - torch.tensor(0.01, device=DEV) * torch.tensor(0.1, device=DEV)
    for _ in range(3):
        update(x, g, state, step, lr=0.01, wd=0.1)
        want = want * keep
    # three products, and the rounding of 1 - lr wd in each: 2^-24 of one, twice, a step
    assert float((x[still] - want).abs().max()) <= 6 * 2.0 ** -24 and torch.equal(x[still], x[0].expand(n // 2))


def test_a_first_moment_is_not_kept_beside_a_second_one_of_zero():
    """Gradients whose squares vanish in fp32 (1e-23) in blocks of larger ones (1e-17): the next step would divide by epsilon alone."""
    n = 1 << 22
    x, tiny = torch.zeros(n, device=DEV), torch.arange(n, device=DEV) % 4 != 0
    g = torch.full((n,), 1e-17, device=DEV).masked_fill_(tiny, 1e-23)
    state, step = fresh(x), torch.zeros((), device=DEV)
    for _ in range(3):
        update(x, g, state, step)
        assert not bool(state[2][tiny].any()) and not bool(state[0][tiny].any())
        # (the largest of a block over its scale may be 127 or 255 but for the quotient's rounding)
        assert int(state[0][~tiny].min()) >= 126 and int(state[2][~tiny].min()) >= 254


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_embedding_through_step(dtype):
    """Rows of an odd width of which a few have a gradient each step: the others keep their bits, and their state stays zero."""
    from dion import Muon

    gen = torch.Generator(device=DEV).manual_seed(1)
    emb = torch.nn.Parameter(torch.empty(20000, 333, device=DEV).normal_(0, 0.1, generator=gen).to(dtype))
    opt = Muon([{"params": [emb], "algorithm": "adamw", "lr": 1e-3, "state_bits": 8, "weight_decay": 0.0}], lr=0.02)
    first, unseen = emb.detach().clone(), torch.ones(20000, dtype=torch.bool, device=DEV)
    for _ in range(6):
        rows = torch.randint(0, 20000, (6000,), device=DEV, generator=gen)
        unseen[rows] = False
        opt.zero_grad()
        (emb[rows].float() * 1e-3).square().sum().backward()
        opt.step()
        assert torch.equal(emb.detach()[unseen], first[unseen])
        state = opt.state[emb]
        assert not bool(state["momentum"][unseen].any()) and not bool(state["variance"][unseen].any())
    assert bool(unseen.any()) and not torch.equal(emb.detach(), first)
