"""The dense linear's backward refuses a kept activation input or a gradient buffer that is on another device than the other operands before
a kernel is handed its address."""

import pytest
import torch

from primus_amd import _lib
from primus_amd.pytorch import kernels as K


def _bf(*shape, device="cpu"):
    return torch.zeros(*shape, dtype=torch.bfloat16, device=device)


@pytest.mark.parametrize("name,call", [
    ("accum_into", lambda: K.linear_bf16_bwd_impl(_bf(4, 64), _bf(4, 32), _bf(64, 32), None, None, accum_into=torch.zeros(64, 32, device="meta"))),
    ("z", lambda: K.linear_bf16_bwd_impl(_bf(4, 64), _bf(4, 32), _bf(64, 32), _bf(4, 64, device="meta"), "gelu")),
    ("a", lambda: K.linear_bf16_bwd_impl(_bf(4, 64), _bf(4, 32, device="meta"), _bf(64, 32), None, None)),
    ("z", lambda: K.linear_bf16_dz_impl(_bf(4, 64), _bf(4, 64, device="meta"), "gelu")),
])
def test_refused(monkeypatch, name, call):
    monkeypatch.setattr(K, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(K, "_on", lambda device: pytest.fail("nothing may be launched"))
    monkeypatch.setattr(_lib, "load", lambda: pytest.fail("nothing may be launched"))
    with pytest.raises(ValueError, match=f"^{name} must live on the device"):
        call()
