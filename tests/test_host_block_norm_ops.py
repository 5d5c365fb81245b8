"""Refusals of the norms where blocks meet, the gradient norm and clipping, before a launch, and which gate a row has: checked without a GPU."""

import ctypes
import math

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


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    x, w = _t(4, 8), _t(8)
    for call in (lambda: ops.add_rmsnorm(x, x, w), lambda: ops.rmsnorm_add(x, x, w), lambda: ops.grad_norm([x]), lambda: ops.clip_grads([x], 1.0),
                 lambda: ops.clip_grads([x], 1.0, norm=torch.ones(()))):
        with pytest.raises(ValueError, match="GPU only"):
            call()


@pytest.mark.parametrize("why,call", [
    ("x must be float32", lambda: ops.add_rmsnorm(_t(4, 8).double(), _t(4, 8).double(), _t(8).double())),
    ("one shape", lambda: ops.add_rmsnorm(_t(4, 8), _t(8, 4), _t(8))),
    ("one shape", lambda: ops.add_rmsnorm(_t(4, 8), _t(8), _t(8))),
    ("one shape", lambda: ops.add_rmsnorm(_t(()), _t(()), _t(1))),
    ("type of x or be float32", lambda: ops.add_rmsnorm(_t(4, 8), _t(4, 8).half(), _t(8))),
    ("type of x or be float32", lambda: ops.add_rmsnorm(_t(4, 8).float(), _t(4, 8), _t(8).float())),
    ("normalised dim", lambda: ops.add_rmsnorm(_t(1, 16385), _t(1, 16385), _t(16385))),
    ("normalised dim", lambda: ops.add_rmsnorm(_t(4, 0), _t(4, 0), _t(0))),
    ("weight must be", lambda: ops.add_rmsnorm(_t(4, 8), _t(4, 8), _t(7))),
    ("weight must be", lambda: ops.add_rmsnorm(_t(4, 8), _t(4, 8), _t(1, 8))),
    ("weight must be", lambda: ops.add_rmsnorm(_t(4, 8), _t(4, 8), _t(8).float())),
    ("post_weight must be", lambda: ops.add_rmsnorm(_t(4, 8), _t(4, 8), _t(8), post_weight=_t(8).half())),
    ("weight must be", lambda: ops.rmsnorm_add(_t(4, 8), _t(4, 8), _t(9))),
    ("gate must have the type", lambda: ops.add_rmsnorm(_t(4, 8), _t(4, 8), _t(8), gate=_t(8).float())),
    ("must broadcast", lambda: ops.add_rmsnorm(_t(4, 8), _t(4, 8), _t(8), gate=_t(4))),
    ("must broadcast", lambda: ops.add_rmsnorm(_t(4, 8), _t(4, 8), _t(8), gate=_t(3, 8))),
    ("must broadcast", lambda: ops.add_rmsnorm(_t(4, 8), _t(4, 8), _t(8), gate=_t(1, 4, 8))),
    ("must broadcast", lambda: ops.add_rmsnorm(_t(2, 3, 4, 8), _t(2, 3, 4, 8), _t(8), gate=_t(2, 1, 4, 8))),
])
def test_norms_refuse(on_gpu, why, call):
    with pytest.raises(ValueError, match=why):
        call()


def test_norms_refuse_negative_eps(on_gpu, monkeypatch):
    monkeypatch.setattr(K, "_block_norm_args", lambda *a: (4, 8, 1, 1, (1, 1, 0)))
    for call in (lambda: ops.add_rmsnorm(_t(4, 8), _t(4, 8), _t(8), -1e-6), lambda: ops.add_rmsnorm(_t(4, 8), _t(4, 8), _t(8), math.nan),
                 lambda: ops.add_rmsnorm(_t(4, 8), _t(4, 8), _t(8), post_weight=_t(8), post_eps=-1.0), lambda: ops.rmsnorm_add(_t(4, 8), _t(4, 8), _t(8), -1.0)):
        with pytest.raises(ValueError, match="eps"):
            call()


@pytest.mark.parametrize("shape,gate,want", [
    ((4, 8), (8,), (4, 1, 8)), ((4, 8), (1,), (4, 1, 1)), ((4, 8), (), (4, 1, 1)), ((4, 8), (4, 8), (1, 4, 8)), ((4, 8), (4, 1), (1, 4, 1)),
    ((2, 3, 8), (2, 1, 8), (3, 2, 8)), ((2, 3, 8), (1, 3, 8), (1, 3, 8)), ((2, 3, 8), (3, 1), (1, 3, 1)), ((2, 3, 5, 8), (2, 3, 1, 8), (5, 6, 8)),
    ((2, 3, 5, 8), (3, 1, 8), (5, 3, 8)), ((2, 1, 5, 8), (2, 1, 5, 8), (1, 10, 8)), ((8,), (8,), (1, 1, 8)), ((8,), (), (1, 1, 1)), ((1, 8), (1, 8), (1, 1, 8)),
])
def test_gate_rows(shape, gate, want):
    """Row r of x has gate row r // div % mod: the one that broadcasting gives it."""
    div, mod, cols = K._gate_rows(torch.Size(shape), torch.Size(gate))
    assert (div, mod, cols) == want
    numbers = torch.arange(math.prod(gate)).reshape(gate).expand(shape).reshape(-1, shape[-1])
    flat = torch.arange(math.prod(gate)).reshape(mod, cols)
    for r in range(numbers.shape[0]):
        assert torch.equal(numbers[r], flat[r // div % mod].expand(shape[-1]))


@pytest.mark.parametrize("why,call", [
    ("dense tensors", lambda: ops.grad_norm([None])),
    ("dense tensors", lambda: ops.grad_norm([torch.zeros(3).to_sparse()])),
    ("must be float32", lambda: ops.grad_norm([torch.zeros(3).double()])),
    ("must be float32", lambda: ops.grad_norm([torch.zeros(3), torch.zeros(3, dtype=torch.int64)])),
    ("norm_type", lambda: ops.grad_norm([torch.zeros(3)], 1.0)),
    ("norm_type", lambda: ops.grad_norm([], 3)),
    ("max_norm", lambda: ops.clip_grads([torch.zeros(3)], -1.0)),
    ("max_norm", lambda: ops.clip_grads([torch.zeros(3)], math.nan)),
    ("same shape", lambda: ops.clip_grads([torch.zeros(3)], 1.0, out=[])),
    ("same shape", lambda: ops.clip_grads([torch.zeros(3)], 1.0, out=[torch.zeros(4)])),
    ("overlap", lambda: ops.clip_grads([torch.zeros(1, 3).expand(2, 3)], 1.0)),
])
def test_gradient_lists_refuse(on_gpu, why, call):
    with pytest.raises(ValueError, match=why):
        call()


def _arrays(spans):
    n = len(spans)
    return ((ctypes.c_uint64 * n)(*[s[0] for s in spans]), (ctypes.c_int64 * n)(*[s[1] for s in spans]), (ctypes.c_int32 * n)(*[s[2] for s in spans]))


def test_c_entries_refuse():
    """The C ABI's own checks: -1 before anything is launched, -3 (no device) here for a call that is right."""
    if torch.cuda.device_count() > 0:
        pytest.skip("a GPU is present: these calls would be real launches")
    lib = _lib.load()
    buf = ctypes.create_string_buffer(1 << 16)
    p = ctypes.addressof(buf) // 16 * 16 + 16
    names = ("x", "residual", "rows", "k", "dtype", "stream_dtype", "post_weight", "post_eps", "gate", "div", "mod", "cols", "scale", "weight", "eps", "y", "h", "post_rstd", "rstd", "stream")
    right = dict(x=p, residual=p, rows=4, k=8, dtype=1, stream_dtype=1, post_weight=p, post_eps=0.0, gate=p, div=2, mod=2, cols=8, scale=1.0, weight=p, eps=0.0, y=p, h=p,
                 post_rstd=None, rstd=None, stream=None)
    call = lambda **k: lib.mxl_block_norm(*[{**right, **k}[n] for n in names])  # noqa: E731
    assert call() == -3 and call(rows=0, x=None) == 0 and call(gate=None, div=0, mod=0, cols=0) == -3 and call(cols=1) == -3 and call(post_weight=None) == -3
    assert call(weight=None, y=None) == -3 and call(stream_dtype=0) == -3 and call(k=16384, cols=16384) == -3 and call(div=1, mod=2) == -3
    for bad in (dict(x=None), dict(residual=None), dict(h=None), dict(y=None), dict(weight=None, post_weight=None), dict(k=0), dict(k=16385), dict(rows=-1), dict(rows=1 << 31),
                dict(dtype=3), dict(dtype=0, stream_dtype=1), dict(stream_dtype=2), dict(eps=-1.0), dict(post_eps=math.nan), dict(cols=2), dict(div=3), dict(mod=0), dict(div=0),
                dict(div=4), dict(mod=3, div=1)):
        assert call(**bad) == -1, bad
    ws = lib.mxl_block_norm_bwd_workspace_bytes
    need = ws(4, 8, 1, 1, 2, 2, 8, 1)
    assert need > 0 and ws(4, 16385, 1, 1, 1, 1, 0, 0) == -1 and ws(4, 8, 1, 1, 3, 2, 8, 1) == -1
    assert ws(0, 8, 1, 1, 0, 1, 8, 1) == 0 and ws(4, 8, 0, 0, 1, 1, 0, 0) == 0
    names = ("dy", "dh", "x", "h", "rows", "k", "dtype", "stream_dtype", "post_weight", "post_rstd", "gate", "div", "mod", "cols", "scale", "weight", "rstd", "dx", "dres", "dw", "dpw",
             "dgate", "ws", "bytes", "stream")
    right = dict(dy=p, dh=p, x=p, h=p, rows=4, k=8, dtype=1, stream_dtype=1, post_weight=p, post_rstd=p, gate=p, div=2, mod=2, cols=8, scale=1.0, weight=p, rstd=p, dx=p, dres=p, dw=p,
                 dpw=p, dgate=p, ws=p, bytes=need, stream=None)
    call = lambda **k: lib.mxl_block_norm_bwd(*[{**right, **k}[n] for n in names])  # noqa: E731
    assert call() == -3 and call(dh=None) == -3 and call(dx=None, dres=None) == -3 and call(post_weight=None, post_rstd=None, dpw=None) == -3
    assert call(weight=None, dy=None, h=None, rstd=None, dw=None, dres=None) == -3 and call(rows=0, dw=None, dpw=None) == 0
    for bad in (dict(dy=None), dict(x=None), dict(h=None), dict(rstd=None), dict(post_rstd=None), dict(gate=None), dict(ws=None), dict(bytes=need - 1), dict(ws=p + 8),
                dict(weight=None, dres=None), dict(weight=None, dw=None), dict(post_weight=None),
                dict(weight=None, post_weight=None, dw=None, dpw=None, dres=None), dict(mod=3), dict(k=0)):
        assert call(**bad) == -1, bad
    # lists
    spans = [(p, 10, 0), (p + 64, 7, 1)]
    ptr, n, dt = _arrays(spans)
    ws = lib.mxl_grad_norm_workspace_bytes(2)
    assert ws > 0 and lib.mxl_grad_norm_workspace_bytes(0) == 0 and lib.mxl_grad_norm_workspace_bytes(-1) == -1
    norm = lambda count=2, kind=0, out=p, w=p, wb=ws, d=dt, s=n: lib.mxl_grad_norm(ptr, s, d, count, kind, out, w, wb, None)  # noqa: E731
    assert norm() == -3 and norm(kind=1) == -3 and norm(count=0, w=None, wb=0) == -3
    for bad in (dict(kind=2), dict(out=None), dict(w=None), dict(wb=ws - 1), dict(count=-1), dict(d=(ctypes.c_int32 * 2)(0, 3)), dict(s=(ctypes.c_int64 * 2)(1, -1))):
        assert norm(**bad) == -1, bad

    def clip(ins, outs, max_norm=1.0, out=p + 32768):
        a, b = _arrays(ins), _arrays(outs)
        return lib.mxl_clip_grads(a[0], b[0], a[1], a[2], b[2], len(ins), max_norm, out, None)

    assert clip(spans, spans) == -3 and clip([], []) == -3 and clip([(p, 0, 0)] * 2, [(p, 0, 0)] * 2) == -3
    far = [(p + 4096, 10, 2), (p + 8192, 7, 0)]
    assert clip(spans, far) == -3 and clip([(p, 10, 0)] * 2, far[:1] + [(p + 8192, 10, 0)]) == -3
    assert clip(spans, far, max_norm=-1.0) == -1 and clip(spans, far, max_norm=math.nan) == -1 and clip(spans, far, out=None) == -1
    for ins, outs in (([(p, 10, 0)] * 2, [(p, 10, 0)] * 2), ([(p, 10, 0), (p + 36, 10, 0)],) * 2, ([(p, 10, 0)], [(p + 4, 10, 0)]), ([(p, 10, 1)], [(p, 10, 0)]),
                      (spans, [(p + 4096, 10, 0), (p + 4100, 7, 0)]), (spans, [(p + 4096, 10, 0), (p + 36, 7, 0)])):
        assert clip(ins, outs) == -1, (ins, outs)


def test_c_entry_refuses_to_sum_what_it_has_not():
    """A backward that sums h again: with a weight, x and a stream of 16 bits."""
    if torch.cuda.device_count() > 0:
        pytest.skip("a GPU is present: these calls would be real launches")
    lib = _lib.load()
    buf = ctypes.create_string_buffer(1 << 16)
    p = ctypes.addressof(buf) // 16 * 16 + 16
    need = lib.mxl_block_norm_bwd_workspace_bytes(4, 8, 1, 1, 1, 1, 0, 0)

    def call(x=p, dtype=1, stream=1, weight=p, post=None):
        pre = None if weight is None else p
        return lib.mxl_block_norm_bwd(pre, p, x, pre, 4, 8, dtype, stream | _lib.NORM_SUMMED, post, post, None, 1, 1, 0, 1.0, weight, pre, p, pre, pre, post, None, p, need, None)

    assert call() == -3 and call(dtype=2, stream=2) == -3 and call(post=p) == -3
    for bad in (dict(x=None), dict(stream=0), dict(dtype=0, stream=0), dict(weight=None, post=p), dict(stream=1 | 0x200), dict(stream=2)):
        assert call(**bad) == -1, bad
