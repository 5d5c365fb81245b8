"""``ops.permute_tokens``: the probabilities' gradient where the rows need none, by the framework's own kernel, bit for bit."""

import ctypes

import pytest
import torch


def test_the_entry_moves_probabilities_alone():
    """Malformed calls are -1, well-formed ones -3 on a machine without a GPU."""
    if torch.cuda.device_count() > 0:
        pytest.skip("a GPU is present: the well-formed calls would be real launches")
    from primus_amd import _lib

    p = ctypes.cast(ctypes.create_string_buffer(1 << 12), ctypes.c_void_p)
    call = lambda **k: _lib.load().mxl_combine_rows(*[{**dict(x=None, rows=8, h=1, dt=0, ro=p, t=4, k=2, pr=None, rp=p, po=p, pd=0, y=None, st=None), **k}[n]  # noqa: E731
                                                      for n in ("x", "rows", "h", "dt", "ro", "t", "k", "pr", "rp", "po", "pd", "y", "st")])
    assert call() == -3 and call(t=0, ro=None, po=None) == 0
    for bad in (dict(rp=None), dict(po=None), dict(rp=None, po=None), dict(ro=None), dict(k=0), dict(k=33), dict(pd=3), dict(t=-1), dict(y=p)):
        assert call(**bad) == -1, bad


def test_refusals():
    from primus_amd.pytorch import kernels as K

    for rp, ro in ((torch.zeros(4, 2), torch.zeros(2, 2, dtype=torch.int64)), (torch.zeros(4), torch.zeros(2, 2)), (torch.zeros(4), torch.zeros(2, 33, dtype=torch.int64)),
                   (torch.zeros(4).double(), torch.zeros(2, 2, dtype=torch.int64)), (torch.zeros(4), torch.zeros(2, 2, dtype=torch.int64))):
        with pytest.raises(ValueError):
            K.entry_probs_impl(rp, ro)


@pytest.mark.gpu
@pytest.mark.parametrize("t,k,experts,align", [(1, 1, 1, 1), (7, 3, 5, 16), (333, 6, 32, 1), (3001, 8, 256, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradient_without_the_rows(gpu, monkeypatch, t, k, experts, align, dtype):
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(t + k)
    idx = torch.randint(-1, experts, (t, k), generator=gen)
    x = torch.randn(t, 24, generator=gen).to(gpu)
    p = torch.rand(t, k, generator=gen).to(dtype).to(gpu).requires_grad_()
    _, row_probs, _, perm = ops.permute_tokens(x, idx.to(gpu), experts, probs=p, align=align)
    d = torch.randn(2 * row_probs.numel(), generator=gen).to(dtype).to(gpu)[::2]       # (strided)
    want = torch.where(perm.row_of >= 0, d[perm.row_of.clamp(min=0)], 0.0)
    monkeypatch.setattr(torch, "where", lambda *a, **k: pytest.fail("the library's indexing in place of the kernel"))
    (got,) = torch.autograd.grad(row_probs, p, d)
    assert got.dtype == dtype and torch.equal(got, want)
