"""Rows past the 2^32 threads of a launch, a workgroup each."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [2 ** 24 - 1, 2 ** 24 + 9])
def test_scale_rows(rows, dtype):
    from dion_amd import ops

    u = torch.randn(rows, 3, device="cuda").bfloat16()
    scale = torch.rand(rows, device="cuda")
    got = ops.scale_rows(u, scale, dtype)
    assert torch.equal(got, (u.float() * scale[:, None]).to(dtype))
