"""Hooks on what the forward passes save that give back another tensor on the same GPU: it is looked at before its address is used."""
import pytest
import torch

from dion_amd import embedding, gated_linear, layer_norm, linear

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Wrapper(torch.Tensor):
    """A tensor without data of its own."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    def __tensor_flatten__(self):
        return ["inner"], None

    @staticmethod
    def __tensor_unflatten__(inner_tensors, meta, outer_size, outer_stride):
        return Wrapper(inner_tensors["inner"])

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        assert func is torch.ops.aten.detach.default  # (autograd's own, of what a hook gives back)
        return Wrapper(args[0].inner)


FORMS = {"shorter": lambda t: t[:-1], "other_type": lambda t: t.to({torch.uint8: torch.int8, torch.int64: torch.int16}.get(t.dtype, torch.float16)),
         "flat": lambda t: t.reshape(-1)[:1], "apart": lambda t: t.repeat_interleave(2, -1)[..., ::2], "wrapper": Wrapper}


def calls():
    gen = torch.Generator(device=DEV).manual_seed(3)
    rnd = lambda *s: torch.empty(*s, device=DEV).normal_(0, 1, generator=gen).bfloat16().requires_grad_()  # noqa: E731
    x, wg, wu, w, b, table = rnd(30, 72), rnd(41, 72), rnd(41, 72), rnd(72), rnd(72), rnd(50, 72)
    ids = torch.arange(30, device=DEV) % 7
    return {"gated_linear": (lambda: gated_linear(x, wg, wu), [x, wg, wu], 4), "layer_norm": (lambda: layer_norm(x, w, b), [x, w, b], 3),
            "embedding": (lambda: embedding(ids, table), [table], 1), "linear": (lambda: linear(x, wg, activation="silu"), [x, wg], 3)}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("name", ["gated_linear", "layer_norm", "embedding", "linear"])
def test_hooks_that_give_back_another_tensor(name, form):
    call, leaves, saved = calls()[name]
    y = call()
    dy = torch.ones_like(y)
    want = torch.autograd.grad(y, leaves, dy)
    for which in range(saved):
        count = []

        def pack(t):
            count.append(t)
            return len(count) - 1, t.detach()

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda p: FORMS[form](p[1]) if p[0] == which else p[1]):
            y = call()
        assert len(count) == saved
        print(name, form, which, count[which].dtype, tuple(count[which].shape), flush=True)
        raw = count[which].dtype in (torch.uint8, torch.int16, torch.float32)  # (what a call keeps for itself)
        if form == "apart" and not raw:
            assert all(torch.equal(p, q) for p, q in zip(want, torch.autograd.grad(y, leaves, dy)))
        else:
            with pytest.raises((ValueError, TypeError), match=f"{name}|wrapper subclass"):
                torch.autograd.grad(y, leaves, dy)
