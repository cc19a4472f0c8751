"""What the backward passes of gated projections, layer norm and embedding find of what the forward passes kept: moved away and back by hooks,
changed in place, read twice; and gradients of two weights that are neighbours in memory by chance."""
import pytest
import torch

from dion_amd import embedding, gated_linear, layer_norm, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def calls():
    gen = torch.Generator(device=DEV).manual_seed(3)
    rnd = lambda *s: torch.empty(*s, device=DEV).normal_(0, 1, generator=gen).bfloat16().requires_grad_()  # noqa: E731
    x, wg, wu, w, b, table = rnd(30, 72), rnd(41, 72), rnd(41, 72), rnd(72), rnd(72), rnd(50, 72)
    ids = torch.arange(30, device=DEV) % 7
    return {"gated_linear": (lambda: gated_linear(x, wg, wu), [x, wg, wu]), "layer_norm": (lambda: layer_norm(x, w, b), [x, w, b]),
            "embedding": (lambda: embedding(ids, table), [table])}, ids


@pytest.mark.parametrize("name", ["gated_linear", "layer_norm", "embedding"])
def test_hooks_on_what_is_saved(name):
    call, leaves = calls()[0][name]
    y = call()
    dy = torch.ones_like(y)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(want, torch.autograd.grad(y, leaves, dy)))  # (read twice)
    with torch.autograd.graph.save_on_cpu():
        y = call()
    assert all(torch.equal(p, q) for p, q in zip(want, torch.autograd.grad(y, leaves, dy)))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t):
        y = call()
    with pytest.raises((RuntimeError, ValueError), match=name):
        torch.autograd.grad(y, leaves, dy)


@pytest.mark.parametrize("name", ["gated_linear", "layer_norm", "embedding"])
def test_what_is_saved_must_not_change(name):
    some, ids = calls()
    call, leaves = some[name]
    y = call()
    with torch.no_grad():
        (ids if name == "embedding" else leaves[0]).add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaves, torch.ones_like(y))


def test_weights_gradients_that_are_neighbours_by_chance():
    """Seven rows that belong to somebody else lie between the two gradients, as far apart as one product would want them."""
    from dion_amd import _lib

    t, k, n = 20, 64, 41
    gen = torch.Generator(device=DEV).manual_seed(4)
    x, wg, wu, dh = (torch.empty(s, device=DEV).normal_(0, 1, generator=gen).bfloat16() for s in ((t, k), (n, k), (n, k), (t, n)))
    _h, kept = ops.gated_forward(x, wg, wu, None, None, "silu", 24)
    want = ops.gated_backward(dh, kept, 24, x, wg, wu, False, True, True, None, None)
    lib = _lib.load()
    nbytes = lib.dion_gated_workspace_bytes(t, k, n, 1, 15)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    for behind in (0, 1):
        all_ = torch.full((48 + n, k), 7.0, device=DEV, dtype=torch.bfloat16)
        rc = lib.dion_gated_backward(dh.data_ptr(), n, kept.data_ptr(), 24, x.data_ptr(), k, None, 0, None, 0, None, all_.data_ptr(),
                                     all_[48:].data_ptr(), behind, None, 0, None, 0, t, k, n, ws.data_ptr(), nbytes,
                                     torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        assert torch.equal(all_[:n], want[1]) and torch.equal(all_[48:], want[2])
        assert bool((all_[n:48] == (0.0 if behind else 7.0)).all())
