"""Layer norm of rows whose sums come near the end of float32, and leave it."""
import pytest
import torch

from test_gpu_layer_norm import BF, FP, make, run_and_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d", [16, 77, 4096, 12290, 40003])
def test_rows_whose_sums_fit(d, dtype):
    """Squares that add up to a tenth of the largest float32 against the formulas."""
    x, w, b, _dy = make(6, d, FP, seed=7)
    x = x / x.std(1, keepdim=True) * (3.4e37 / d) ** 0.5
    run_and_check(x.to(dtype), w, b, torch.randn(6, d, device="cuda").to(dtype))


@pytest.mark.parametrize("d", [16, 77, 4096, 12290, 40003])
def test_rows_whose_sums_do_not_fit(d):
    """Squares ten times past it: the bias, and no gradient.  Values whose own sum is: NaN.  The rows beside them are as without."""
    from dion_amd import layer_norm

    x, w, b, dy = make(6, d, FP, seed=8)
    gen = torch.Generator(device="cuda").manual_seed(1)
    sign = torch.where(torch.rand(d, device="cuda", generator=gen) < 0.5, -1.0, 1.0)
    sign[0], sign[1] = 1.0, -1.0
    bad = x.clone()
    bad[2] = sign * (3.4e39 / d) ** 0.5
    bad[4] = 3.4e38 / d * 4
    outs = []
    for v in (x, bad):
        leaf = v.clone().requires_grad_()
        y = layer_norm(leaf, w, b)
        outs.append((y.detach(), torch.autograd.grad(y, leaf, dy)[0]))
    (y0, g0), (y, g) = outs
    rest = [0, 1, 3, 5]
    assert torch.equal(y[rest], y0[rest]) and torch.equal(g[rest], g0[rest])
    assert torch.equal(y[2], b) and not bool(g[2].any())
    assert bool(y[4].isnan().all()) and bool(g[4].isnan().all())
