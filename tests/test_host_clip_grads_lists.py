"""What the C entries of the gradient norm and clipping refuse about addresses, before anything is launched: checked without a GPU."""

import ctypes

import pytest
import torch

from primus_amd import _lib

FP, BF, HF = 0, 1, 2


@pytest.fixture()
def memory():
    if torch.cuda.device_count() > 0:
        pytest.skip("a GPU is present: calls that are right would be real launches")
    buf = ctypes.create_string_buffer(1 << 16)
    yield ctypes.addressof(buf) // 16 * 16 + 16


def _clip(ins, outs, norm):
    arrays = [[(ctypes.c_uint64 * len(s))(*[t[0] for t in s]), (ctypes.c_int64 * len(s))(*[t[1] for t in s]), (ctypes.c_int32 * len(s))(*[t[2] for t in s])] for s in (ins, outs)]
    return _lib.load().mxl_clip_grads(arrays[0][0], arrays[1][0], arrays[0][1], arrays[0][2], arrays[1][2], len(ins), 1.0, norm, None)


def test_norm_inside_what_is_written(memory):
    """Workgroups read the norm while others write: it may lie in no tensor that is written.  (-3: right, but no device here.)"""
    a, b = (memory, 10, FP), (memory + 4096, 10, BF)
    for norm in (memory, memory + 36):
        assert _clip([a], [a], norm) == -1
    for norm in (memory + 4096, memory + 4112):
        assert _clip([a], [b], norm) == -1
    assert _clip([a, (memory + 64, 0, FP)], [b, (memory + 64, 0, FP)], memory + 64) == -3
    for norm in (memory, memory + 36, memory + 40, memory + 4092, memory + 4116):      # in a gradient that is read, and beside both
        assert _clip([a], [b], norm) == -3


def _norm(spans, out, workspace):
    lib = _lib.load()
    a = [(ctypes.c_uint64 * len(spans))(*[t[0] for t in spans]), (ctypes.c_int64 * len(spans))(*[t[1] for t in spans]), (ctypes.c_int32 * len(spans))(*[t[2] for t in spans])]
    return lib.mxl_grad_norm(a[0], a[1], a[2], len(spans), 0, out, workspace, lib.mxl_grad_norm_workspace_bytes(len(spans)), None)


@pytest.mark.parametrize("dtype", [FP, BF, HF])
def test_addresses_between_elements(memory, dtype):
    """Sixteen-byte pieces are counted in elements from a tensor's address: it has to be an element's.  Of a tensor without elements it is not looked at."""
    size, norm = 4 if dtype == FP else 2, memory + 32768
    for off in range(1, 8):
        want = -3 if off % size == 0 else -1
        at = (memory + off, 10, dtype)
        assert _norm([at], norm, memory + 1024) == want
        assert _clip([at], [at], norm) == want and _clip([at], [(memory + 4096, 10, FP)], norm) == want and _clip([(memory + 4096, 10, FP)], [at], norm) == want
    assert _norm([(memory + 1, 0, dtype)], norm, memory + 1024) == -3 and _clip([(memory + 1, 0, dtype)] * 2, [(memory + 1, 0, dtype)] * 2, norm) == -3
    for off in (1, 2, 3):
        assert _norm([(memory, 10, dtype)], norm + off, memory + 1024) == -1 and _clip([(memory, 10, dtype)], [(memory, 10, dtype)], norm + off) == -1


class _Wrapped(torch.Tensor):
    """A tensor on the GPU by its looks, without memory of its own, as a sharded parameter's gradient is one."""

    @staticmethod
    def __new__(cls, shape):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=torch.float32, device="cuda:0")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(str(func))


def test_a_tensor_without_memory_is_no_overlap(memory, monkeypatch):
    from contextlib import nullcontext

    from primus_amd.pytorch import kernels as K

    monkeypatch.setattr(K, "_on", lambda device: nullcontext())
    monkeypatch.setattr(K, "_stream", lambda: None)
    w, norm = [_Wrapped((3, 5))], _Wrapped(())
    with pytest.raises(ValueError, match="memory of their own"):
        K.clip_grads_impl(w, w, 1.0, norm)
    for sizes, ptrs, why in (([0, 4], [0, 16], None), ([1 << 36], [16], "2\\^36"), ([3, 1], [16, 0], "memory of their own")):
        if why is None:
            K._why_refused(ptrs, sizes, "gradients")
            continue
        with pytest.raises(ValueError, match=why):
            K._why_refused(ptrs, sizes, "gradients")


_NO_MEMORY = """
import ctypes, resource, sys
sys.path.insert(0, {root!r})
from primus_amd import _lib
lib = _lib.load()
n = 1 << 22
ptr, size, kind = (ctypes.c_uint64 * n)(), (ctypes.c_int64 * n)(), (ctypes.c_int32 * n)()
norm = ctypes.c_float(1.0)
call = lambda: lib.mxl_clip_grads(ptr, ptr, size, kind, kind, n, 1.0, ctypes.byref(norm), None)
with open("/proc/self/statm") as f:
    now = int(f.read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (now + (32 << 20), resource.RLIM_INFINITY))      # (the spans take 24 bytes a tensor and direction: 201 MB)
first = call()
resource.setrlimit(resource.RLIMIT_AS, (resource.RLIM_INFINITY, resource.RLIM_INFINITY))
print(first, call(), lib.mxl_error_string(first).decode())
"""


def test_no_host_memory_is_no_overlap(memory):
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", _NO_MEMORY.format(root=root)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stderr[-2000:]
    assert out.stdout.split()[:2] == ["-6", "-3"] and "memory" in out.stdout
