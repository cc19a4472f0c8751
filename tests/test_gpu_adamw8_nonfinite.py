"""AdamW with moments in 8 bits where one block of a tensor is not finite."""
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


@pytest.mark.parametrize("xdt,gdt", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("rounds", [2049, 9 * 2048 + 1])
def test_a_block_that_is_not_finite_keeps_to_itself(xdt, gdt, rounds):
    """The block one round of a workgroup (2048 elements) before a short last block, and every other block: only its own
    scale becomes NaN."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    n = 2048 * rounds + 5
    x0 = torch.empty(n, device=DEV).normal_(0, 0.1, generator=gen).to(xdt)
    g = torch.empty(n, device=DEV).normal_(0, 1e-2, generator=gen).to(gdt)
    bad = g.clone()
    bad[2048 * (rounds - 1) + 3] = float("nan")
    bad[77] = float("inf")
    runs = []
    for grad in (g, bad):
        x, state, step = x0.clone(), fresh(x0), torch.zeros((), device=DEV)
        for _ in range(2):
            update(x, grad, state, step)
        runs.append((x, *state))
    (x, m, ms, v, vs), (xb, mb, msb, vb, vsb) = runs
    lost = torch.zeros(ms.numel(), dtype=torch.bool, device=DEV)
    lost[16 * (rounds - 1)] = lost[0] = True
    assert torch.equal(msb.isnan(), lost) and torch.equal(vsb.isnan(), lost)
    rest = ~lost.repeat_interleave(128)[:n]
    assert torch.equal(msb[~lost], ms[~lost]) and torch.equal(vsb[~lost], vs[~lost])
    for a, b in ((x, xb), (m, mb), (v, vb)):
        assert torch.equal(a[rest], b[rest])
