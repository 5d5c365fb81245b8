"""A training step around the linears as it is run: norms between blocks on a residual stream in fp32, MXFP8 linears with the gated activation whose weight
gradients go into float32 ``main_grad``s, the norm behind the last block, then the global gradient norm and the clipping into the optimizer's
gradients.  Every norm of the run is held against its formulas on the inputs and gradients that it met, the norm of the gradients against float64;
a captured step is replayed on new inputs."""

import math

import pytest
import torch

from test_gpu_block_norm import BF, EPS, FP, _close, _reference
from test_gpu_grad_norm import _clipped, _exact_norm

pytestmark = pytest.mark.gpu

HIDDEN, FFN, BLOCKS = 256, 192, 2
MAX_NORM = 0.5


class Blocks(torch.nn.Module):
    def __init__(self, device):
        super().__init__()
        g = torch.Generator().manual_seed(4)
        param = lambda *s, scale=1.0, mean=0.0: torch.nn.Parameter((mean + scale * torch.randn(s, generator=g)).to(BF).to(device))  # noqa: E731
        self.pre = torch.nn.ParameterList([param(HIDDEN, scale=0.1, mean=1.0) for _ in range(BLOCKS)])
        self.post = torch.nn.ParameterList([param(HIDDEN, scale=0.1, mean=1.0) for _ in range(BLOCKS)])
        self.gate = torch.nn.ParameterList([param(HIDDEN, scale=0.3, mean=0.5) for _ in range(BLOCKS)])
        self.up = torch.nn.ParameterList([param(2 * FFN, HIDDEN, scale=HIDDEN ** -0.5) for _ in range(BLOCKS)])
        self.down = torch.nn.ParameterList([param(HIDDEN, FFN, scale=FFN ** -0.5) for _ in range(BLOCKS)])
        for w in list(self.up) + list(self.down):
            w.main_grad = torch.zeros(w.shape, device=device)
            w.grad_added_to_main_grad = False

    def forward(self, x, stream, calls=None):
        """``x``: the embedding's part, ``stream``: the residual stream it is added to."""
        from primus_amd.pytorch import ops
        from primus_amd.pytorch.core import Float8QuantConfig, ScaleDtype, ScalingGranularity

        cfg = Float8QuantConfig(granularity=ScalingGranularity.MX_BLOCKWISE, scale_dtype=ScaleDtype.E8M0, block_size=32)
        linear = lambda a, w: ops.gemm_fp8(a, w, config=cfg, fuse_bgrad_accum_pattern="megatron")  # noqa: E731
        out = x
        for i in range(BLOCKS):
            post, gate, scale = (None, None, 1.0) if i == 0 else (self.post[i - 1], self.gate[i - 1], 0.5)
            y, h = ops.add_rmsnorm(out, stream, self.pre[i], EPS, post_weight=post, gate=gate, scale=scale)
            if calls is not None:
                calls.append(dict(x=out, residual=stream, weight=self.pre[i], post_weight=post, gate=gate, scale=scale, y=y, h=h))
            stream = h
            out = linear(ops.swiglu_with_probs(linear(y, self.up[i]), torch.ones(len(y), device=y.device)), self.down[i])
        h = ops.rmsnorm_add(out, stream, self.post[-1], EPS, gate=self.gate[-1], scale=0.5)
        if calls is not None:
            calls.append(dict(x=out, residual=stream, weight=None, post_weight=self.post[-1], gate=self.gate[-1], scale=0.5, y=None, h=h))
        return h

    def gradients(self):
        small = list(self.pre) + list(self.post) + list(self.gate)
        return [w.main_grad for w in list(self.up) + list(self.down)] + [p.grad for p in small]


def _inputs(seed, device, tokens=100):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(tokens, HIDDEN, generator=g).to(BF).to(device), (2 * torch.randn(tokens, HIDDEN, generator=g)).to(device), torch.randn(tokens, HIDDEN, generator=g).to(device)


def _step(model, x, stream, dh, outs, calls=None):
    from primus_amd.pytorch import ops

    for w in list(model.up) + list(model.down):
        w.main_grad.zero_()
    for p in model.parameters():
        p.grad = None
    h = model(x, stream, calls)
    for c in calls or ():
        for n in ("x", "residual", "y", "h"):
            if c[n] is not None and c[n].requires_grad:
                c[n].retain_grad()
    h.backward(dh)
    return ops.clip_grads(model.gradients(), MAX_NORM, out=outs)


def test_step(gpu):
    model = Blocks(gpu)
    outs = [torch.empty(p.shape, device=gpu) for p in list(model.up) + list(model.down) + list(model.pre) + list(model.post) + list(model.gate)]
    x, stream, dh = _inputs(0, gpu)
    calls = []
    norm = _step(model, x.requires_grad_(), stream.requires_grad_(), dh, outs, calls)
    grads = model.gradients()
    want = _exact_norm(grads)
    assert all(w.grad_added_to_main_grad and w.main_grad.any() for w in list(model.up) + list(model.down))
    assert MAX_NORM < want and abs(norm.item() - want) <= (2.0 ** -24 + 1e-9) * want
    for o, g in zip(outs, grads):
        _clipped(o, g, MAX_NORM, norm)
    assert abs(_exact_norm(outs) - MAX_NORM) <= 1e-5 * MAX_NORM + 2e-6
    for i, c in enumerate(calls):
        pre = c["weight"] is not None
        # the stream's gradient that this norm was given is what the next one made of it (autograd holds the sum of both uses of y's block: one use of h)
        dh_in = calls[i + 1]["residual"].grad if i + 1 < len(calls) else dh
        ref = _reference(c, c["y"].grad if pre else None, dh_in, c["scale"], BF, FP, pre, eps=EPS, post_eps=EPS)
        for name in ("y", "h") if pre else ("h",):
            _close(c[name], ref[name], (name, c[name].dtype))
        for name in ("x", "residual"):
            _close(c[name].grad, ref[name], (name, c[name].dtype))
        for name in ("weight", "post_weight", "gate"):
            if c[name] is not None:     # (used by this call alone)
                _close(c[name].grad, ref[name], (name, BF))


def test_captured_step(gpu):
    model = Blocks(gpu)
    shapes = [p.shape for p in list(model.up) + list(model.down) + list(model.pre) + list(model.post) + list(model.gate)]
    x, stream, dh = _inputs(0, gpu)
    outs = [torch.empty(s, device=gpu) for s in shapes]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(model, x, stream, dh, outs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = _step(model, x, stream, dh, outs)
    for seed in range(1, 5):
        nx, ns, nd = _inputs(seed, gpu)
        x.copy_(nx), stream.copy_(ns), dh.copy_(nd)
        graph.replay()
        torch.cuda.synchronize()
        got = [norm.clone()] + [o.clone() for o in outs]
        eager = [torch.empty(s, device=gpu) for s in shapes]
        want = [_step(model, nx, ns, nd, eager)] + eager
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed
