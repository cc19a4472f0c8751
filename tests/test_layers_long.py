"""Rows and columns past what the C entries' int holds are refused, not counted modulo 2^32."""
import os

import pytest
import torch

from dion_amd import _lib, embedding, gated_linear, layer_norm, linear, ops

BF = torch.bfloat16
LONG = 2 ** 32 + 5  # five, to an int


@pytest.mark.parametrize("shape", [(LONG, 1), (1, LONG), (2 ** 31, 1), (2 ** 16, 2 ** 16 + 1, 1), (3, 2, LONG)])
def test_rows_that_an_int_does_not_count(shape):
    with pytest.raises(ValueError, match="passes the kernels'"):
        ops._rows(torch.empty(shape, dtype=BF, device="meta"))


@pytest.mark.parametrize("shape,rows", [((2 ** 31 - 1, 1), 2 ** 31 - 1), ((2 ** 16, 2 ** 14, 8), 2 ** 30), ((7,), 1)])
def test_rows_that_an_int_counts(shape, rows):
    t, _address, ld, _copy = ops._rows(torch.empty(shape, dtype=BF, device="meta"))
    assert t.shape == (rows, shape[-1]) and ld == shape[-1]


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libdion_hip.so not built in this checkout")
def test_c_entries_refuse_more_rows_than_layer_norm_takes():
    from test_layers_refusals import norm_backward, norm_forward

    lib = _lib.load()
    for call in (norm_forward, norm_backward):
        assert call(lib, rows=2 ** 30 + 1) == -1 and "2^30 rows" in lib.dion_last_error().decode()
    assert lib.dion_layer_norm_workspace_bytes(2 ** 30 + 1, 8) == 0 and lib.dion_layer_norm_workspace_bytes(2 ** 30, 8) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [LONG, 2 ** 31 + 9])
def test_calls_refuse_them(rows):
    one = torch.ones(1, 1, device="cuda", dtype=BF)
    long, ids = one.expand(rows, 1), torch.zeros(1, device="cuda", dtype=torch.int32)
    for call in (lambda: layer_norm(long), lambda: linear(long, one), lambda: gated_linear(long, one, one),
                 lambda: embedding(ids.expand(rows), one), lambda: embedding(ids, long), lambda: linear(one, long),
                 lambda: gated_linear(one, long, long), lambda: layer_norm(one.expand(1, rows)), lambda: layer_norm(long.view(rows, 1, 1)),
                 lambda: linear(long, one, residual=long)):
        with pytest.raises(ValueError, match="passes the kernels'"):
            call()
    with pytest.raises(ValueError, match="passes the kernels'"):
        ops.embedding_backward(one, ids, rows, 1.0, None, BF)


@pytest.mark.gpu
def test_more_rows_than_layer_norm_takes():
    x = torch.ones(2 ** 30 + 1, 1, device="cuda", dtype=BF)
    with pytest.raises(ValueError, match="more than 2\\^30 rows"):
        layer_norm(x)
