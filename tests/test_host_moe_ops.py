"""Refusals of the operators around the expert MLP: every one before a launch, so they are checked without a GPU.  Tensors of a GPU
are stood in for by a subclass that says it is one; the last check needs none."""

import ctypes

import pytest
import torch

from primus_amd import _lib
from primus_amd.pytorch import kernels as K
from primus_amd.pytorch import ops


@pytest.fixture()
def on_gpu(monkeypatch):
    """The checks as for tensors on the GPU."""
    monkeypatch.setattr(K, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(_lib, "load", lambda: pytest.fail("nothing may be launched"))


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 8)
    for call in (lambda: ops.gemm_bias_act(_bf(4, 32), _bf(32, 32)), lambda: ops.topk_routing(x, 2), lambda: ops.permute_tokens(x, torch.zeros(4, 2, dtype=torch.int64), 3),
                 lambda: ops.unpermute_tokens(x, ops.TokenPermutation(torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, dtype=torch.int32)))):
        with pytest.raises(ValueError, match="GPU only"):
            call()


@pytest.mark.parametrize("why,call", [
    ("2-D tensor", lambda: ops.topk_routing(torch.randn(2, 3, 4), 2)),
    ("float32, bfloat16 or float16", lambda: ops.topk_routing(torch.randn(2, 4).double(), 2)),
    ("topk", lambda: ops.topk_routing(torch.randn(2, 4), 5)),
    ("topk", lambda: ops.topk_routing(torch.randn(2, 64), 33)),
    ("topk", lambda: ops.topk_routing(torch.randn(2, 4), 0)),
    ("number of experts", lambda: ops.topk_routing(torch.randn(2, 1025), 2)),
    ("number of experts", lambda: ops.topk_routing(torch.randn(2, 0), 1)),
    ("score_function", lambda: ops.topk_routing(torch.randn(2, 4), 2, score_function="relu")),
    ("group_topk needs num_groups", lambda: ops.topk_routing(torch.randn(2, 4), 2, group_topk=1)),
    ("num_groups needs group_topk", lambda: ops.topk_routing(torch.randn(2, 4), 2, num_groups=2)),
    ("num_groups must divide", lambda: ops.topk_routing(torch.randn(2, 4), 2, num_groups=3, group_topk=1)),
    ("num_groups must divide", lambda: ops.topk_routing(torch.randn(2, 130), 2, num_groups=65, group_topk=1)),
    ("group_topk must be in", lambda: ops.topk_routing(torch.randn(2, 4), 2, num_groups=2, group_topk=3)),
    ("hold topk experts", lambda: ops.topk_routing(torch.randn(2, 8), 3, num_groups=4, group_topk=1)),
    ("expert_bias", lambda: ops.topk_routing(torch.randn(2, 4), 2, expert_bias=torch.zeros(3))),
    ("expert_bias", lambda: ops.topk_routing(torch.randn(2, 4), 2, expert_bias=torch.zeros(4).double())),
    ("token_mask", lambda: ops.topk_routing(torch.randn(2, 4), 2, token_mask=torch.ones(3, dtype=torch.bool))),
    ("token_mask", lambda: ops.topk_routing(torch.randn(2, 4), 2, token_mask=torch.ones(2))),
    ("indices", lambda: ops.permute_tokens(torch.randn(4, 8), torch.zeros(3, 2, dtype=torch.int64), 3)),
    ("integers", lambda: ops.permute_tokens(torch.randn(4, 8), torch.zeros(4, 2), 3)),
    ("integers", lambda: ops.permute_tokens(torch.randn(4, 8), torch.zeros(4, 2, dtype=torch.bool), 3)),
    ("x must be float32", lambda: ops.permute_tokens(torch.randn(4, 8).double(), torch.zeros(4, 2, dtype=torch.int64), 3)),
    ("2.21", lambda: ops.gemm_bias_act(_bf(1, 1).expand(1, 32), _bf(1, 1).expand((1 << 21) + 32, 32))),
    ("x must be", lambda: ops.permute_tokens(torch.randn(4), torch.zeros(4, 2, dtype=torch.int64), 3)),
    ("number of experts", lambda: ops.permute_tokens(torch.randn(4, 8), torch.zeros(4, 2, dtype=torch.int64), 0)),
    ("number of experts", lambda: ops.permute_tokens(torch.randn(4, 8), torch.zeros(4, 2, dtype=torch.int64), 1025)),
    ("align", lambda: ops.permute_tokens(torch.randn(4, 8), torch.zeros(4, 2, dtype=torch.int64), 3, align=0)),
    ("topk must be", lambda: ops.permute_tokens(torch.randn(4, 8), torch.zeros(4, 33, dtype=torch.int64), 3)),
    ("shape of indices", lambda: ops.permute_tokens(torch.randn(4, 8), torch.zeros(4, 2, dtype=torch.int64), 3, probs=torch.zeros(4, 3))),
    ("probs must be", lambda: ops.permute_tokens(torch.randn(4, 8), torch.zeros(4, 2, dtype=torch.int64), 3, probs=torch.zeros(4, 2).double())),
    ("row_of", lambda: ops.unpermute_tokens(torch.randn(4, 8), ops.TokenPermutation(torch.zeros(4, 2), torch.zeros(4, dtype=torch.int32)))),
    ("entry_of", lambda: ops.unpermute_tokens(torch.randn(4, 8), ops.TokenPermutation(torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4)))),
    ("made for", lambda: ops.unpermute_tokens(torch.randn(4, 8), ops.TokenPermutation(torch.zeros(4, 2, dtype=torch.int64), torch.zeros(5, dtype=torch.int32)))),
    ("probs must be", lambda: ops.unpermute_tokens(torch.randn(4, 8), ops.TokenPermutation(torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, dtype=torch.int32)),
                                                   probs=torch.zeros(4, 3))),
    ("a must be", lambda: ops.gemm_bias_act(_bf(32), _bf(32, 32))),
    ("a must be", lambda: ops.gemm_bias_act(_bf(4, 32), _bf(1, 32, 32))),
    ("2-D bfloat16", lambda: ops.gemm_bias_act(torch.randn(4, 32), _bf(32, 32))),
    ("2-D bfloat16", lambda: ops.gemm_bias_act(_bf(4, 32), torch.randn(32, 32))),
    ("contraction lengths", lambda: ops.gemm_bias_act(_bf(4, 64), _bf(32, 32))),
    ("multiples of 32", lambda: ops.gemm_bias_act(_bf(4, 48), _bf(32, 48))),
    ("multiples of 32", lambda: ops.gemm_bias_act(_bf(4, 32), _bf(40, 32))),
    ("activation must be", lambda: ops.gemm_bias_act(_bf(4, 32), _bf(32, 32), activation="tanh")),
    ("bias must be", lambda: ops.gemm_bias_act(_bf(4, 32), _bf(32, 32), bias=_bf(31))),
    ("bias must be", lambda: ops.gemm_bias_act(_bf(4, 32), _bf(32, 32), bias=_bf(32).half())),
    ("residual must have", lambda: ops.gemm_bias_act(_bf(4, 32), _bf(32, 32), residual=_bf(5, 32))),
    ("residual must be", lambda: ops.gemm_bias_act(_bf(4, 32), _bf(32, 32), residual=torch.randn(4, 32))),
    ("fuse_bgrad_accum_pattern", lambda: ops.gemm_bias_act(_bf(4, 32), _bf(32, 32), fuse_bgrad_accum_pattern="other")),
    ("main_grad", lambda: ops.gemm_bias_act(_bf(4, 32), _bf(32, 32), fuse_bgrad_accum_pattern="megatron")),
    ("4 GiB", lambda: ops.gemm_bias_act(_bf(1, 1).expand(1, 1 << 17), _bf(1, 1).expand(1 << 15, 1 << 17))),
    ("not empty", lambda: ops.unpermute_tokens(torch.randn(4, 0), ops.TokenPermutation(torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, dtype=torch.int32)))),
])
def test_refusals(on_gpu, why, call):
    with pytest.raises(ValueError, match=why):
        call()


def test_c_entries_check_before_they_touch_the_device():
    """Malformed calls are MXL_EINVAL (-1), well-formed ones MXL_ENODEV (-3) on a machine without a GPU."""
    if torch.cuda.device_count() > 0:
        pytest.skip("a GPU is present: the well-formed calls would be real launches")
    lib = _lib.load()
    buf = ctypes.create_string_buffer(1 << 16)
    p = ctypes.cast(buf, ctypes.c_void_p)
    f = ctypes.c_float(1.0)
    ws = lib.mxl_topk_routing_workspace_bytes(40, 8)
    route = lambda **k: lib.mxl_topk_routing(*[{**dict(l=p, dt=0, t=40, e=8, k=2, s=0, b=None, g=1, gk=1, r=1, sc=f, m=None, pr=p, i=p, c=p, w=p, wb=ws, st=None), **k}[n]  # noqa: E731
                                               for n in ("l", "dt", "t", "e", "k", "s", "b", "g", "gk", "r", "sc", "m", "pr", "i", "c", "w", "wb", "st")])
    assert ws > 0 and route() == -3 and lib.mxl_topk_routing_workspace_bytes(16, 8) == 0 and route(t=16, w=None, wb=0) == -3
    for bad in (dict(l=None), dict(dt=3), dict(t=-1), dict(e=0), dict(e=1025), dict(k=0), dict(k=9), dict(s=2), dict(g=3), dict(g=2, gk=3), dict(g=8, gk=1),
                dict(pr=None), dict(i=None), dict(c=None), dict(w=None), dict(wb=ws - 1)):
        assert route(**bad) == -1, bad
    assert lib.mxl_topk_routing_workspace_bytes(-1, 8) == -1 and lib.mxl_topk_routing_workspace_bytes(1, 0) == -1
    bwd = lambda **k: lib.mxl_topk_routing_bwd(*[{**dict(d=p, l=p, dt=0, i=p, t=4, e=8, k=2, s=0, r=1, sc=f, o=p, st=None), **k}[n] for n in ("d", "l", "dt", "i", "t", "e", "k", "s", "r", "sc", "o", "st")])  # noqa: E731
    assert bwd() == -3 and bwd(t=0) == 0
    for bad in (dict(d=None), dict(o=None), dict(dt=-1), dict(k=33), dict(e=2000)):
        assert bwd(**bad) == -1, bad
    pw = lib.mxl_permute_plan_workspace_bytes(5000, 4)
    plan = lambda **k: lib.mxl_permute_plan(*[{**dict(i=p, n=5000, e=4, a=1, r=5000, ro=p, eo=p, gl=p, pr=None, pb=0, rp=None, w=p, wb=pw, st=None), **k}[n]  # noqa: E731
                                              for n in ("i", "n", "e", "a", "r", "ro", "eo", "gl", "pr", "pb", "rp", "w", "wb", "st")])
    assert pw > 0 and plan() == -3 and lib.mxl_permute_plan_workspace_bytes(8, 4) == 0 and plan(n=8, w=None, wb=0) == -3
    for bad in (dict(i=None), dict(n=-1), dict(e=0), dict(e=1025), dict(a=0), dict(r=4999), dict(ro=None), dict(eo=None), dict(gl=None), dict(pr=p, pb=3, rp=p), dict(pb=4, rp=p),
                dict(w=None), dict(wb=pw - 1), dict(a=32, r=5000)):
        assert plan(**bad) == -1, bad
    both = lambda **k: lib.mxl_permute_tokens(*[{**dict(x=p, t=2500, rb=16, i=p, k=2, e=4, a=1, r=5000, ro=p, eo=p, gl=p, pr=None, pb=0, rp=None, o=p, w=p, wb=pw, st=None), **k}[n]  # noqa: E731
                                                for n in ("x", "t", "rb", "i", "k", "e", "a", "r", "ro", "eo", "gl", "pr", "pb", "rp", "o", "w", "wb", "st")])
    assert both() == -3
    for bad in (dict(x=None), dict(t=-1), dict(rb=0), dict(rb=(1 << 24) + 1), dict(i=None), dict(k=0), dict(k=33), dict(e=0), dict(a=0), dict(r=4999), dict(ro=None), dict(eo=None), dict(gl=None),
                dict(pr=p, pb=3, rp=p), dict(o=None), dict(w=None), dict(wb=pw - 1)):
        assert both(**bad) == -1, bad
    assert lib.mxl_permute_rows(p, 4, 16, p, 2, p, 8, p, None) == -3
    assert lib.mxl_permute_rows(p, 4, 0, p, 2, p, 8, p, None) == -1 and lib.mxl_permute_rows(p, 4, 16, p, 33, p, 8, p, None) == -1
    assert lib.mxl_permute_rows(p, 4, 16, p, 2, None, 8, p, None) == -1 and lib.mxl_permute_rows(None, 4, 16, p, 2, p, 8, p, None) == -1
    assert lib.mxl_combine_rows(p, 8, 16, 1, p, 4, 2, p, None, None, 0, p, None) == -3
    assert lib.mxl_combine_rows(p, 8, 16, 1, p, 4, 2, None, p, None, 0, p, None) == -1 and lib.mxl_combine_rows(p, 8, 0, 1, p, 4, 2, p, None, None, 0, p, None) == -1
    assert lib.mxl_combine_rows(p, 8, 16, 3, p, 4, 2, p, None, None, 0, p, None) == -1 and lib.mxl_combine_rows(p, 8, 16, 1, p, 4, 2, p, None, None, 5, p, None) == -1
    assert lib.mxl_combine_rows_bwd(p, p, 8, 16, 1, p, p, 4, 2, p, 0, p, p, None) == -3
    assert lib.mxl_combine_rows_bwd(None, p, 8, 16, 1, p, p, 4, 2, p, 0, p, p, None) == -1 and lib.mxl_combine_rows_bwd(p, p, 8, 16, 1, p, p, 4, 2, None, 0, p, p, None) == -1
    assert lib.mxl_combine_rows_bwd(p, p, 8, 16, 1, p, None, 4, 2, p, 0, p, p, None) == -1
    lin = lambda **k: lib.mxl_linear_bf16(*[{**dict(a=p, b=p, bias=p, bd=1, act=3, r=p, m=4, n=32, k=32, y=p, z=None, w=None, wb=0, st=None), **k}[n]  # noqa: E731
                                            for n in ("a", "b", "bias", "bd", "act", "r", "m", "n", "k", "y", "z", "w", "wb", "st")])
    odd = ctypes.c_void_p(p.value + 8)
    assert p.value % 16 == 0 and lin() == -3 and lin(m=0) == 0
    for bad in (dict(a=None), dict(b=None), dict(y=None), dict(bd=2), dict(act=4), dict(act=-1), dict(m=-1), dict(n=48), dict(k=8), dict(n=0), dict(n=1 << 16, k=1 << 16),
                dict(a=odd), dict(b=odd), dict(bias=odd), dict(r=odd), dict(y=odd), dict(z=odd), dict(m=128, n=128, k=4096), dict(m=128, n=128, k=4096, w=p, wb=64)):
        assert lin(**bad) == -1, bad
    need = lib.mxl_linear_bf16_workspace_bytes(128, 128, 4096)
    assert need > 0 and lin(m=128, n=128, k=4096, w=p, wb=need) == -3 and lib.mxl_linear_bf16_workspace_bytes(4096, 4096, 4096) == 0
    assert lib.mxl_linear_bf16_workspace_bytes(1, 1, 1) == -1
    dgrad = lambda a, b, m, n, k, w=None, wb=0: lib.mxl_linear_bf16_dgrad(a, b, m, n, k, p, w, wb, None)  # noqa: E731
    assert dgrad(p, p, 4, 32, 32) == -3 and dgrad(p, p, 4, 32, 33) == -1 and dgrad(None, p, 4, 32, 32) == -1 and dgrad(p, p, 0, 32, 32) == 0
    assert dgrad(p, p, 128, 4096, 128) == -1 and dgrad(p, p, 128, 4096, 128, p, need) == -3
    ws = lib.mxl_linear_bf16_dz_workspace_bytes(80, 32)
    dz = lambda **k: lib.mxl_linear_bf16_dz(*[{**dict(dy=p, z=p, act=1, m=80, n=32, dz=p, db=p, dbd=0, w=p, wb=ws, st=None), **k}[n] for n in ("dy", "z", "act", "m", "n", "dz", "db", "dbd", "w", "wb", "st")])  # noqa: E731
    assert ws == 10 * 32 * 4 and lib.mxl_linear_bf16_dz_workspace_bytes(64, 32) == 0 and dz(m=64, w=None, wb=0) == -3 and dz() == -3 and dz(act=3, db=None) == 0
    for bad in (dict(dy=None), dict(z=None), dict(dz=None), dict(act=9), dict(n=31), dict(w=None), dict(wb=ws - 1), dict(dbd=2), dict(dy=odd)):
        assert dz(**bad) == -1, bad
    need = lib.mxl_linear_bf16_bwd_workspace_bytes(100, 64, 32, 1, 1, 1, 0, 1)
    assert need > 0 and lib.mxl_linear_bf16_bwd_workspace_bytes(100, 64, 32, 3, 0, 0, 0, 0) == 0 and lib.mxl_linear_bf16_bwd_workspace_bytes(1, 1, 1, 3, 0, 0, 0, 0) == -1
    bwd = lambda **k: lib.mxl_linear_bf16_bwd(*[{**dict(dy=p, a=p, b=p, z=p, act=1, m=100, n=64, k=32, da=p, db=p, f=0, dbias=p, dbd=0, w=p, wb=need, st=None), **k}[n]  # noqa: E731
                                                for n in ("dy", "a", "b", "z", "act", "m", "n", "k", "da", "db", "f", "dbias", "dbd", "w", "wb", "st")])
    assert bwd() == -3 and bwd(act=3, da=None, db=None, dbias=None, w=None, wb=0) == 0
    for bad in (dict(dy=None), dict(b=None), dict(z=None), dict(act=7), dict(n=33), dict(f=1), dict(dbd=2), dict(w=None), dict(wb=need - 1)):
        assert bwd(**bad) == -1, bad
    need = lib.mxl_linear_bf16_wgrad_workspace_bytes(4096, 64, 64, 0)
    wgrad = lambda dz, a, m, n, k, db, f=0, w=None, wb=0: lib.mxl_linear_bf16_wgrad(dz, a, m, n, k, db, f, w, wb, None)  # noqa: E731
    assert need > 0 and wgrad(p, p, 4096, 64, 64, p, 0, p, need) == -3 and wgrad(p, p, 7, 32, 32, p) == -3 and wgrad(p, p, 7, 32, 32, p, 2, p, 4096) == -3
    for bad in ((None, p, 7, 32, 32, p), (p, None, 7, 32, 32, p), (p, p, 7, 32, 32, None), (p, p, 7, 33, 32, p), (p, p, 7, 32, 32, p, 1), (p, p, 7, 32, 32, p, 2), (p, p, 7, 32, 32, p, 2, p, 4095), (p, p, 4096, 64, 64, p),
                (p, p, 4096, 64, 64, p, 0, p, need - 1), (p, p, 1 << 20, 4096, 4096, p), (odd, p, 7, 32, 32, p)):
        assert wgrad(*bad) == -1, bad
