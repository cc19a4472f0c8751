"""Results of layer norm over its operands, at the C entries: dx over x or dy, which other workgroups read for the sums over the rows,
is refused; y may be x."""
import os

import pytest
import torch

from dion_amd import _lib
from test_layers_refusals import norm_backward

NEEDS_LIB = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libdion_hip.so not built in this checkout")
X, DY, FAR = 1 << 20, 2 << 20, 3 << 20  # addresses that are never read: a call that is not refused is not made


@NEEDS_LIB
@pytest.mark.parametrize("dw,db", [(FAR, FAR), (None, None)])
def test_dx_over_an_operand_is_refused(dw, db):
    lib = _lib.load()
    row, rows, pitch = 64 * 2, 8, 80 * 2
    for dx in (X, X + 2, X - 2, X - rows * row + 2, X + 7 * pitch + row - 2, X + 70 * 2, DY, DY + 3 * row, DY + rows * row - 2, DY - rows * row + 2):
        assert norm_backward(lib, dy=DY, ld=64, x=X, ldx=80, dx=dx, dw=dw, db=db, mean=FAR, rstd=FAR) == -1, dx
        assert "overlaps" in lib.dion_last_error().decode()
    assert norm_backward(lib, dy=DY, x=X, dx=X, rows=1, ldx=0, ld=0, mean=FAR, rstd=FAR, dw=dw, db=db) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,d", [(40, 96), (9, 1001), (300, 4096), (7, 5000), (5, 16000), (3, 30000), (3, 40003)])
def test_y_may_be_x(rows, d, dtype):
    from dion_amd import layer_norm

    x = torch.randn(rows, d, device="cuda").to(dtype)
    w, b = torch.randn(d, device="cuda"), torch.randn(d, device="cuda")
    want = layer_norm(x, w, b)
    code = int(dtype == torch.float32)
    rc = _lib.load().dion_layer_norm_forward(x.data_ptr(), d, code, w.data_ptr(), 1, b.data_ptr(), 1, x.data_ptr(), code, None, None, rows, d,
                                             1e-5, torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(x, want)


@pytest.mark.gpu
def test_dx_beside_its_operands():
    """One buffer, no byte shared: the rows of dx right behind those of x, and dy behind them."""
    from dion_amd import ops

    rows, d = 20, 40
    buf = torch.randn(3, rows, d, device="cuda").bfloat16()
    x, dx, dy = buf
    w = torch.randn(d, device="cuda")
    _y, stats = ops.layer_norm_forward(x, w, None, 1e-5, None, True)
    want, dw, db = ops.layer_norm_backward(dy, x, w, stats, True, True, torch.float32)
    sums = torch.empty(2, d, device="cuda")
    at = stats.data_ptr()
    rc = _lib.load().dion_layer_norm_backward(dy.data_ptr(), d, 0, x.data_ptr(), d, 0, w.data_ptr(), 1, at, at + 4 * rows, dx.data_ptr(),
                                              sums[0].data_ptr(), sums[1].data_ptr(), 1, rows, d, None, 0,
                                              torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(dx, want) and torch.equal(sums[0], dw) and torch.equal(sums[1], db)
