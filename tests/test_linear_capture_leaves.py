"""Which leaves of a product's graph are looked at before a capture goes on, on the host: the products are stood in for by torch's own."""
import contextlib
import sys

import pytest
import torch

from dion_amd import linear, ops

EAGER, CAPTURE = 11, 22  # streams


@pytest.fixture
def product(monkeypatch):
    """``linear`` on CPU tensors, as if on the given stream, captured or not."""
    where = {"stream": EAGER, "capturing": False}
    monkeypatch.setattr(ops, "linear_forward", lambda x, w, b, act, r, keep: (x @ w.t() if b is None else x @ w.t() + b, None))
    monkeypatch.setattr(ops, "_stream_handle", lambda device: where["stream"])
    monkeypatch.setattr(ops, "_device_of", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: where["capturing"])

    def call(*args, captured=False, **kw):
        where.update(stream=CAPTURE if captured else EAGER, capturing=captured)
        return linear(*args, **kw)

    return call


def leaf(*shape):
    return torch.ones(*shape, dtype=torch.bfloat16).requires_grad_()


FORMS = {
    "direct": (lambda: leaf(16, 8), lambda w: w),
    "cast": (lambda: torch.ones(16, 8).requires_grad_(), lambda w: w.bfloat16()),
    "slice": (lambda: leaf(48, 8), lambda w: w[16:32]),
    "transposed": (lambda: leaf(8, 16), lambda w: w.t()),
    "cast of a slice": (lambda: torch.ones(48, 8).requires_grad_(), lambda w: w[:16].bfloat16()),
}


@pytest.mark.parametrize("form", FORMS)
def test_a_weight_of_a_living_eager_result_is_refused(product, form):
    make, view = FORMS[form]
    w, x = make(), torch.ones(4, 8, dtype=torch.bfloat16)
    alive = product(x, view(w))
    for _ in range(2):  # (refused again, not only the first time)
        with pytest.raises(RuntimeError, match="still has its graph"):
            product(x, view(w), captured=True)
    del alive
    kept = product(x, view(w), captured=True)
    again = product(x, view(w), captured=True)
    assert kept.requires_grad and again.requires_grad
    product(x, view(w))  # an eager call beside it is no capture


def test_a_bias_and_a_weight_behind_other_products(product):
    """The leaf of an earlier product of the captured pass, and a bias that is a view of a leaf."""
    w1, w2, b, x = leaf(8, 8), leaf(16, 8), leaf(3, 16), torch.ones(4, 8, dtype=torch.bfloat16)
    alive = product(x, w2, b[1])
    with pytest.raises(RuntimeError, match="still has its graph"):
        product(x, leaf(16, 8), b[2], captured=True)
    del alive
    product(x, leaf(16, 8), b[2], captured=True)
    alive = product(x, w1)
    hidden = x @ w1.t()  # (the leaf is reached through x alone)
    with pytest.raises(RuntimeError, match="still has its graph"):
        product(hidden.relu(), w2, captured=True)
    del alive, hidden
    y = x
    for _ in range(200):  # every node of a deep graph is looked at once, not once for every product behind it
        y = product(y, w1, captured=True)
    assert y.requires_grad


def test_a_graph_that_was_made_eagerly_and_is_used_in_a_capture(product):
    """A cast weight that was made, and used, before the capture."""
    w, x = torch.ones(16, 8).requires_grad_(), torch.ones(4, 8, dtype=torch.bfloat16)
    half = w.bfloat16()
    product(x, half)
    with pytest.raises(RuntimeError, match="still has its graph"):
        product(x, half, captured=True)


@pytest.mark.parametrize("captured", [False, True])
def test_a_node_is_looked_at_once(product, monkeypatch, captured):
    """Weights that one deep graph makes, and products along a residual stream: what a call looks at is what is new in it."""
    module, looked = sys.modules["dion_amd.linear"], []
    below = module._below
    monkeypatch.setattr(module, "_below", lambda node: looked.append(1) or below(node))
    made = torch.ones(16, 16).requires_grad_()
    for _ in range(300):
        made = made * 1.0
    h = torch.ones(4, 16, dtype=torch.bfloat16)
    for _ in range(40):
        h = h + product(h.relu(), made.bfloat16(), captured=captured)
    assert h.requires_grad and 300 <= len(looked) <= 300 + 40 * 8
