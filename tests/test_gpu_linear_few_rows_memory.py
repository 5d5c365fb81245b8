"""The dense linear's forward of up to 16 rows has a kernel that takes no workspace: none is asked for and none is allocated."""

import pytest
import torch


def test_sizes():
    from primus_amd import _lib

    lib = _lib.load()
    for n, k in ((14336, 4096), (4096, 4096), (32, 32), (256, 14336)):
        for m in (0, 1, 16):
            assert lib.mxl_linear_bf16_forward_workspace_bytes(m, n, k) == 0
        for m in (17, 64, 333, 2051):
            assert lib.mxl_linear_bf16_forward_workspace_bytes(m, n, k) == lib.mxl_linear_bf16_workspace_bytes(m, n, k)
    assert lib.mxl_linear_bf16_workspace_bytes(17, 4096, 4096) > 0
    assert lib.mxl_linear_bf16_forward_workspace_bytes(-1, 32, 32) == lib.mxl_linear_bf16_forward_workspace_bytes(1, 33, 32) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 16])
def test_the_forward_allocates_its_output_alone(gpu, m):
    from primus_amd.pytorch import ops

    a, b = torch.randn(m, 4096, device=gpu).bfloat16(), torch.randn(14336, 4096, device=gpu).bfloat16()
    want = torch.nn.functional.silu(a.double() @ b.double().t())
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    y = ops.gemm_bias_act(a, b, activation="silu")
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before + 1
    # fp32 sums of 4096 products, through a slope of at most 1.13, and one rounding
    err = 1.13 * (4096 + 64) * 2.0 ** -23 * (a.double().abs() @ b.double().abs().t()) + 2.0 ** -17 * want.abs()
    assert bool(((y.double() - want).abs() <= err + 2.0 ** -8 * (want.abs() + err)).all())
