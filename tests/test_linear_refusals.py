"""What the product of a weight refuses on the host, without a GPU."""
import ctypes
import os

import pytest
import torch

from dion_amd import _lib, linear

NEEDS_LIB = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libdion_hip.so not built in this checkout")
P = 4096  # an address that is never read: every call below ends on the host


def forward(lib, x=P, ldx=64, w=P, ldw=64, bias=None, bdt=0, act=0, r=None, ldr=0, y=P, slope=None, t=8, k=64, n=32, ws=None,
            nbytes=0):
    return lib.dion_linear_forward(x, ldx, w, ldw, bias, bdt, act, r, ldr, y, slope, t, k, n, ws, nbytes, None)


def backward(lib, dy=P, lddy=32, slope=None, act=0, x=P, ldx=64, w=P, ldw=64, dx=P, dw=P, db=None, dbt=0, t=8, k=64, n=32, ws=None,
             nbytes=0):
    return lib.dion_linear_backward(dy, lddy, slope, act, x, ldx, w, ldw, dx, dw, db, dbt, t, k, n, ws, nbytes, None)


@NEEDS_LIB
def test_c_entry_points_refuse():
    lib = _lib.load()
    for call, cases in ((forward, ({"t": -1}, {"k": 0}, {"n": 0}, {"n": 1 << 21}, {"k": 1 << 21}, {"t": (1 << 30) + 1}, {"act": 6}, {"act": -1},
                                   {"x": None}, {"w": None}, {"y": None}, {"x": P + 1}, {"ldx": 63}, {"ldw": 63},
                                   {"bias": P, "bdt": 2}, {"r": P, "ldr": 31}, {"slope": P})),
                        (backward, ({"t": -1}, {"dy": None}, {"lddy": 31}, {"x": None}, {"w": None}, {"ldx": 8}, {"act": 1}, {"slope": P},
                                    {"db": P, "dbt": 3}, {"dy": P + 1}))):
        for kw in cases:
            assert call(lib, **kw) == -1, (call.__name__, kw)
            assert "dion_linear" in lib.dion_last_error().decode()
    # a workspace that is missing, short or off its line, where one is needed: rows that are not whole chunks
    for kw in ({}, {"ws": P, "nbytes": 100}, {"ws": P + 8, "nbytes": 1 << 20}):
        assert forward(lib, k=63, ldx=63, ldw=63, **kw) == -2 and "workspace" in lib.dion_last_error().decode()
    assert backward(lib, db=P) == -2
    assert forward(lib, t=0, x=None, y=None) == 0


@NEEDS_LIB
def test_workspace_bytes():
    bytes_of = _lib.load().dion_linear_workspace_bytes
    assert bytes_of(8, 64, 32, 0, 0, 0) == 0 and bytes_of(-1, 64, 32, 0, 0, 0) == 0 and bytes_of(0, 64, 32, 1, 3, 7) >= 0
    assert bytes_of(8, 63, 32, 0, 0, 3) == 8 * 64 * 2 + 32 * 64 * 2
    for t, k, n in ((1, 8, 8), (777, 1000, 2730), (65, 4096, 300), (16384, 4096, 14336)):
        for backward_ in (0, 1):
            one = [bytes_of(t, k, n, backward_, 1, 1 << b) for b in range(3)]
            assert bytes_of(t, k, n, backward_, 1, 7) >= max(one) and all(b % 256 == 0 for b in one)


def test_wrong_tensors_are_refused():
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(RuntimeError, match="no CPU path"):
        linear(bf(4, 8), bf(16, 8))
    with pytest.raises(ValueError, match="unknown activation"):
        linear(bf(4, 8), bf(16, 8), activation="swish")
    with pytest.raises(ValueError, match="does not fit"):
        linear(bf(4, 9), bf(16, 8))
    with pytest.raises(ValueError, match="does not fit"):
        linear(bf(4, 8), bf(2, 16, 8))
    with pytest.raises(ValueError, match="does not fit"):
        linear(torch.zeros((), dtype=torch.bfloat16), bf(16, 8))
    with pytest.raises(ValueError, match="empty weight"):
        linear(bf(4, 0), bf(16, 0))
    assert ctypes.sizeof(ctypes.c_size_t) == 8


@pytest.mark.gpu
def test_wrong_gpu_tensors_are_refused():
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    x, w = bf(4, 8), bf(16, 8)
    for bad in ({"x": x.float()}, {"weight": w.half()}, {"bias": bf(16).double()}, {"residual": bf(4, 16).float()}):
        with pytest.raises(TypeError):
            linear(**{"x": x, "weight": w, **bad})
    for bad in ({"bias": bf(8)}, {"residual": bf(1, 16)}, {"residual": bf(4, 8)}):
        with pytest.raises(ValueError):
            linear(**{"x": x, "weight": w, **bad})
    with pytest.raises(RuntimeError, match="no CPU path"):
        linear(x, w, bias=torch.zeros(16, dtype=torch.bfloat16))
