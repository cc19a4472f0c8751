"""What gated projections, layer norm and embedding refuse on the host, without a GPU."""
import os

import pytest
import torch
import torch.autograd.forward_ad as fwd

from dion_amd import _lib, embedding, gated_linear, layer_norm

NEEDS_LIB = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libdion_hip.so not built in this checkout")
P = 4096  # an address that is never read: every call below ends on the host


def gated_forward(lib, x=P, ldx=64, wg=P, ldg=64, wu=P, ldu=64, bg=None, bgt=0, bu=None, but=0, act=5, h=P, kept=None, bits=24, t=8, k=64,
                  n=32, ws=None, nbytes=0):
    return lib.dion_gated_forward(x, ldx, wg, ldg, wu, ldu, bg, bgt, bu, but, act, h, kept, bits, t, k, n, ws, nbytes, None)


def gated_backward(lib, dh=P, ld=32, kept=P, bits=32, x=P, ldx=64, wg=P, ldg=64, wu=P, ldu=64, dx=P, dg=P, du=P, behind=0, dbg=None, dbgt=0,
                   dbu=None, dbut=0, t=8, k=64, n=32, ws=None, nbytes=0):
    return lib.dion_gated_backward(dh, ld, kept, bits, x, ldx, wg, ldg, wu, ldu, dx, dg, du, behind, dbg, dbgt, dbu, dbut, t, k, n, ws, nbytes, None)


def norm_forward(lib, x=P, ldx=64, xt=0, w=P, wt=1, b=P, bt=1, y=P, yt=0, mean=None, rstd=None, rows=8, width=64, eps=1e-5):
    return lib.dion_layer_norm_forward(x, ldx, xt, w, wt, b, bt, y, yt, mean, rstd, rows, width, eps, None)


def norm_backward(lib, dy=P, ld=64, yt=0, x=P, ldx=64, xt=0, w=P, wt=1, mean=P, rstd=P, dx=P, dw=P, db=P, bt=1, rows=8, width=64,
                  ws=P, nbytes=1 << 30):
    return lib.dion_layer_norm_backward(dy, ld, yt, x, ldx, xt, w, wt, mean, rstd, dx, dw, db, bt, rows, width, ws, nbytes, None)


def rows_forward(lib, ids=P, bits=64, t=8, w=P, ldw=64, wt=1, v=100, d=64, y=P, yt=0):
    return lib.dion_embedding_forward(ids, bits, t, w, ldw, wt, v, d, 1.0, y, yt, None)


def rows_backward(lib, ids=P, bits=64, t=8, dy=P, ld=64, yt=0, v=100, d=64, pad=-1, dw=P, wt=1, ws=P, nbytes=1 << 30):
    return lib.dion_embedding_backward(ids, bits, t, dy, ld, yt, v, d, 1.0, pad, dw, wt, ws, nbytes, None)


CASES = {
    gated_forward: ({"t": -1}, {"k": 0}, {"n": 0}, {"n": 1 << 20}, {"k": 1 << 21}, {"t": (1 << 30) + 1}, {"act": 6}, {"act": -1},
                    {"x": None}, {"wg": None}, {"wu": None}, {"h": None}, {"h": P + 1}, {"x": P + 1}, {"ldx": 63}, {"ldg": 63},
                    {"ldu": 63}, {"bg": P, "bgt": 2}, {"bu": P, "but": -1}, {"bg": P + 2, "bgt": 1}, {"bu": P + 1}, {"kept": P + 8}, {"kept": P, "bits": 16}),
    gated_backward: ({"t": -1}, {"dh": None}, {"ld": 31}, {"kept": None}, {"kept": P + 2}, {"bits": 16}, {"x": None}, {"wg": None}, {"wu": None},
                     {"ldx": 8}, {"ldg": 8}, {"ldu": 8}, {"dbg": P, "dbgt": 3}, {"dbu": P, "dbut": 3}, {"n": 1 << 20}, {"dx": P + 1},
                     {"dg": P + 1}, {"du": P + 1}, {"dbu": P + 2, "dbut": 1}, {"behind": 1}, {"behind": 1, "du": None},
                     {"behind": 1, "n": 30, "ld": 30, "du": P + 30 * 64 * 2}),
    norm_forward: ({"rows": -1}, {"width": 0}, {"width": (1 << 24) + 1}, {"x": None}, {"y": None}, {"ldx": 63}, {"xt": 2}, {"yt": -1},
                   {"wt": 2}, {"bt": 2}, {"x": P + 1}, {"w": P + 2}, {"mean": P}, {"rstd": P}, {"mean": P + 2, "rstd": P},
                   {"eps": -1.0}, {"eps": float("nan")}),
    norm_backward: ({"rows": -1}, {"width": 0}, {"dy": None}, {"x": None}, {"ld": 63}, {"ldx": 63}, {"mean": None}, {"rstd": None},
                    {"xt": 2}, {"yt": 2}, {"wt": 2}, {"bt": 2}, {"dx": P + 1}, {"dw": P + 2}, {"db": P + 2},
                    {"rstd": P + 2}),
    rows_forward: ({"bits": 16}, {"t": -1}, {"v": 0}, {"d": 0}, {"v": (1 << 24) + 1}, {"t": (1 << 30) + 1}, {"ids": None}, {"ids": P + 4},
                   {"w": None}, {"y": None}, {"ldw": 63}, {"wt": 2}, {"yt": 2}, {"w": P + 2}),
    rows_backward: ({"bits": 8}, {"t": -1}, {"v": 0}, {"ids": None}, {"dy": None}, {"dw": None}, {"ld": 63}, {"yt": 2}, {"wt": 2},
                    {"pad": 100}, {"dw": P + 2}),
}


@NEEDS_LIB
@pytest.mark.parametrize("call", CASES, ids=lambda c: c.__name__)
def test_c_entry_points_refuse(call):
    lib = _lib.load()
    for kw in CASES[call]:
        assert call(lib, **kw) == -1, kw
        assert "dion_" in lib.dion_last_error().decode()


@NEEDS_LIB
def test_workspaces_are_checked():
    lib = _lib.load()
    for kw in ({}, {"ws": P, "nbytes": 100}, {"ws": P + 8, "nbytes": 1 << 20}):
        assert gated_forward(lib, k=63, ldx=63, ldg=63, ldu=63, **kw) == -2 and "workspace" in lib.dion_last_error().decode()
        assert gated_backward(lib, **kw) == -2
        assert norm_backward(lib, **{"ws": None, "nbytes": 0, "rows": 2000, **kw}) == -2
        assert rows_backward(lib, **{"ws": None, "nbytes": 0, **kw}) == -2
    assert gated_forward(lib, t=0, x=None, h=None) == 0 and norm_forward(lib, rows=0, x=None, y=None) == 0
    assert rows_forward(lib, t=0, ids=None, y=None) == 0
    bytes_of = lib.dion_gated_workspace_bytes
    assert bytes_of(8, 64, 32, 0, 0) == 0 and bytes_of(-1, 64, 32, 0, 0) == 0 and bytes_of(0, 64, 32, 1, 15) >= 0
    for t, k, n in ((1, 8, 8), (777, 1000, 2730), (65, 4096, 300), (16384, 4096, 14336)):
        for backward in (0, 1):
            one = [bytes_of(t, k, n, backward, 1 << b) for b in range(4)]
            assert bytes_of(t, k, n, backward, 15) >= max(one) and all(b % 256 == 0 for b in one)
    assert lib.dion_gated_kept_bytes(3, 33, 24) == 3 * 64 * 6 and lib.dion_gated_kept_bytes(3, 32, 32) == 3 * 32 * 8
    assert lib.dion_gated_kept_bytes(-1, 8, 24) == 0 and lib.dion_gated_kept_bytes(3, 32, 16) == 0
    assert lib.dion_layer_norm_workspace_bytes(0, 8) == 0 and lib.dion_layer_norm_workspace_bytes(1024, 8) == 0
    assert lib.dion_layer_norm_workspace_bytes(1025, 8) >= 2 * 8 * 4 and lib.dion_layer_norm_workspace_bytes(1, 20000) >= 2 * 20000 * 4
    assert lib.dion_embedding_workspace_bytes(0, 8, 8) >= 9 * 4 + 8 * 4 and lib.dion_embedding_workspace_bytes(1, 0, 8) == 0


def bf(*s, device="cpu"):
    return torch.zeros(*s, dtype=torch.bfloat16, device=device)


def test_wrong_tensors_are_refused():
    x, w = bf(4, 8), bf(16, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        gated_linear(x, w, w)
    with pytest.raises(ValueError, match="unknown activation"):
        gated_linear(x, w, w, activation="swish")
    for bad in ((bf(4, 9), w, w), (x, bf(2, 16, 8), w), (torch.zeros((), dtype=torch.bfloat16), w, w)):
        with pytest.raises(ValueError, match="does not fit"):
            gated_linear(*bad)
    with pytest.raises(ValueError, match="empty weights"):
        gated_linear(bf(4, 0), bf(16, 0), bf(16, 0))
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer_norm(x)
    for bad in (torch.zeros(()), torch.zeros(4, 0)):
        with pytest.raises(ValueError, match="no last dimension"):
            layer_norm(bad)
    ids = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        embedding(ids, w)
    for bad in (torch.zeros(8), torch.zeros(0, 8), torch.zeros(8, 0), torch.zeros(2, 3, 4)):
        with pytest.raises(ValueError, match="expected a table"):
            embedding(ids, bad)
    for bad in (16, -17):
        with pytest.raises(ValueError, match="outside a table"):
            embedding(ids, w, padding_idx=bad)


@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_is_refused(grad):
    w = torch.ones(16, 8, requires_grad=grad)
    with fwd.dual_level():
        for call in (lambda d: gated_linear(d(bf(4, 8)), w.bfloat16(), w.bfloat16()), lambda d: gated_linear(bf(4, 8), w, d(w.detach())),
                     lambda d: layer_norm(bf(4, 8), w[0], d(w[1].detach())), lambda d: layer_norm(d(bf(4, 8))),
                     lambda d: embedding(torch.zeros(3, dtype=torch.int64), d(w.detach()))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(lambda t: fwd.make_dual(t, torch.ones_like(t)))


@pytest.mark.gpu
def test_wrong_gpu_tensors_are_refused():
    x, w, f = bf(4, 8, device="cuda"), bf(16, 8, device="cuda"), torch.zeros(16, device="cuda")
    good = {"x": x, "weight_gate": w, "weight_up": w}
    for bad in ({"x": x.float()}, {"weight_gate": w.half()}, {"weight_up": w.float()}, {"bias_gate": f.double()}, {"bias_up": f.half()}):
        with pytest.raises(TypeError, match="gated_linear"):
            gated_linear(**{**good, **bad})
    for bad in ({"weight_up": w[:8]}, {"bias_gate": f[:8]}, {"bias_up": f[None]}, {"weight_up": w.t()}):
        with pytest.raises(ValueError, match="gated_linear"):
            gated_linear(**{**good, **bad})
    with pytest.raises(RuntimeError, match="no CPU path"):
        gated_linear(x, w, w.cpu())
    for bad in ({"x": x.half()}, {"weight": f[:8].double()}, {"bias": f[:8].half()}, {"dtype": torch.float16}):
        with pytest.raises(TypeError, match="layer_norm"):
            layer_norm(**{"x": x, **bad})
    for bad in ({"weight": f}, {"bias": f[:8, None]}, {"eps": -1e-5}, {"eps": float("nan")}):
        with pytest.raises(ValueError, match="layer_norm"):
            layer_norm(**{"x": x, **bad})
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad in ({"ids": ids.float()}, {"ids": ids.to(torch.int16)}, {"weight": w.half()}, {"dtype": torch.float64}):
        with pytest.raises(TypeError, match="embedding"):
            embedding(**{"ids": ids, "weight": w, **bad})
    with pytest.raises(RuntimeError, match="no CPU path"):
        embedding(ids.cpu(), w)
