"""``ops.permute_tokens`` / ``ops.unpermute_tokens`` of a batch without tokens, whose buffer still has padding rows: forward, every gradient
and the C entries."""

import ctypes

import pytest
import torch


def test_the_entry_takes_empty_outputs():
    """No tokens: nothing to write, whatever the rows' probabilities are (an empty output has no address)."""
    from primus_amd import _lib

    p = ctypes.cast(ctypes.create_string_buffer(1 << 12), ctypes.c_void_p)
    call = _lib.load().mxl_combine_rows
    assert call(p, 224, 16, _lib.DT_BF16, None, 0, 2, None, p, None, _lib.DT_F32, None, None) == 0
    assert call(p, 224, 16, _lib.DT_BF16, None, 0, 2, None, None, None, _lib.DT_F32, None, None) == 0
    assert call(p, 224, 16, _lib.DT_BF16, None, 0, 33, None, p, None, _lib.DT_F32, None, None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("align", [1, 16, 32])
@pytest.mark.parametrize("experts", [1, 8])
@pytest.mark.parametrize("probs_dtype", [None, torch.float32, torch.bfloat16])
def test_gradients_without_tokens(gpu, align, experts, probs_dtype):
    from primus_amd.pytorch import ops

    x = torch.zeros(0, 48, dtype=torch.bfloat16, device=gpu, requires_grad=True)
    idx = torch.zeros(0, 2, dtype=torch.int64, device=gpu)
    p = None if probs_dtype is None else torch.zeros(0, 2, dtype=probs_dtype, device=gpu, requires_grad=True)
    rows, row_probs, lens, perm = ops.permute_tokens(x, idx, experts, probs=p, align=align)
    n = experts * (align - 1) // align * align
    assert rows.shape == (n, 48) and lens.tolist() == [0] * (experts - 1) + [n] and not bool(rows.any())
    if p is None:
        (dx,) = torch.autograd.grad(rows, x, torch.ones_like(rows))
    else:
        assert row_probs.shape == (n,) and not bool(row_probs.any())
        dx, dp = torch.autograd.grad([rows, row_probs], [x, p], [torch.ones_like(rows), torch.ones_like(row_probs)], retain_graph=True)
        assert dp.shape == (0, 2) and dp.dtype == probs_dtype
        (dp,) = torch.autograd.grad(row_probs, p, torch.ones_like(row_probs))
        assert dp.shape == (0, 2) and dp.dtype == probs_dtype
    assert dx.shape == (0, 48)
    out = torch.ones(n, 48, dtype=torch.bfloat16, device=gpu, requires_grad=True)
    y = ops.unpermute_tokens(out, perm, probs=p)
    assert y.shape == (0, 48)
    grads = torch.autograd.grad(y, [out] if p is None else [out, p], torch.zeros_like(y))
    assert grads[0].shape == (n, 48) and not bool(grads[0].any()) and (p is None or grads[1].shape == (0, 2))
