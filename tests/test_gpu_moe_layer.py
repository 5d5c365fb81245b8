"""The operators around the expert MLP as a layer runs them: router, rows into the experts' order, experts, rows back, and a shared
expert whose last linear adds the routed output as its residual.  Against the layer written token by token in 64 bits on the same
bf16 weights; as a captured graph replayed with other tokens; through the Megatron-side expert MLP with a low-precision recipe.

Tolerance: every tensor between two steps is rounded to bf16 once, which moves it by at most 2^-8 of its 2-norm, and a product with a
random matrix hands a relative error of its operand on as it is.  Forward: x is exact; fc1, activation, fc2, the sum, the shared z
(its activation sees fp32), its output and the result: 7 steps.  Backward: at most as many again, and the saved ones: 14."""

import math
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu

HIDDEN, FFN, EXPERTS, TOPK, SHARED = 256, 192, 12, 3, 320


def _weights(gpu, seed):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=gen) * s[-1] ** -0.5).bfloat16().to(gpu).requires_grad_()  # noqa: E731
    w = SimpleNamespace(router=r(EXPERTS, HIDDEN), w1=r(EXPERTS, 2 * FFN, HIDDEN), w2=r(EXPERTS, HIDDEN, FFN), s1=r(SHARED, HIDDEN), b1=r(1, SHARED), s2=r(HIDDEN, SHARED))
    w.b1 = w.b1.detach()[0].clone().requires_grad_()
    w.bias = (torch.randn(EXPERTS, generator=gen) * 0.05).to(gpu)
    return w


def _layer(ops, x, w, mask, align):
    logits = x.float() @ w.router.float().t()
    probs, idx, counts = ops.topk_routing(logits, TOPK, score_function="sigmoid", expert_bias=w.bias, num_groups=4, group_topk=2, scaling_factor=1.5, token_mask=mask)
    rows, row_probs, lens, perm = ops.permute_tokens(x, idx, EXPERTS, probs=probs, align=align)
    h = ops.swiglu_with_probs(ops.grouped_gemm(rows, w.w1, lens), row_probs)
    routed = ops.unpermute_tokens(ops.grouped_gemm(h, w.w2, lens), perm)
    shared = ops.gemm_bias_act(x, w.s1, bias=w.b1, activation="silu")
    return ops.gemm_bias_act(shared, w.s2, residual=routed), idx, counts


def _by_token(x, w, idx):
    """The same from the given choice, in float64, one expert after the other."""
    d = {n: getattr(w, n).detach().double().requires_grad_() for n in ("router", "w1", "w2", "s1", "b1", "s2")}
    x = x.detach().double().requires_grad_()
    s = torch.sigmoid(x @ d["router"].t())
    chosen = torch.zeros_like(s, dtype=torch.bool)
    live = idx >= 0
    chosen[torch.nonzero(live)[:, 0], idx[live]] = True
    p = torch.where(chosen, s, 0.0)
    p = 1.5 * p / (p.sum(1, keepdim=True) + 1e-20)
    out = 0.0
    for e in range(EXPERTS):
        a = x @ d["w1"][e].t()
        g, u = a[:, :FFN], a[:, FFN:]
        out = out + (g * torch.sigmoid(g) * u * p[:, e:e + 1]) @ d["w2"][e].t()
    z = x @ d["s1"].t() + d["b1"]
    return out + (z * torch.sigmoid(z)) @ d["s2"].t(), x, d


def _rel(a, b):
    return float((a.detach().double() - b.detach()).norm() / b.detach().norm())


NAMES = ("router", "w1", "w2", "s1", "b1", "s2")


@pytest.mark.parametrize("tokens,align,masked", [(1, 1, False), (5, 32, False), (333, 1, True), (700, 32, True)])
def test_layer_against_float64(gpu, tokens, align, masked):
    from primus_amd.pytorch import ops

    w = _weights(gpu, 3)
    gen = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, HIDDEN, generator=gen).bfloat16().to(gpu).requires_grad_()
    dy = torch.randn(tokens, HIDDEN, generator=gen).bfloat16().to(gpu)
    mask = (torch.rand(tokens, generator=gen) < 0.8).to(gpu) if masked else None
    y, idx, counts = _layer(ops, x, w, mask, align)
    assert torch.equal(counts, torch.bincount(idx[idx >= 0], minlength=EXPERTS))
    if mask is not None:
        assert bool((idx[~mask] == -1).all()) and bool((idx[mask] >= 0).all())
    want, xd, d = _by_token(x, w, idx)
    assert _rel(y, want) <= 7 * 2.0 ** -8
    got = torch.autograd.grad(y, [x] + [getattr(w, n) for n in NAMES], dy)
    ref = torch.autograd.grad(want, [xd] + [d[n] for n in NAMES], dy.double())
    for name, a, b in zip(("x",) + NAMES, got, ref):
        assert _rel(a, b) <= 14 * 2.0 ** -8, (name, _rel(a, b))


def test_layer_in_a_graph(gpu):
    """Forward and backward captured once, replayed with other tokens, other routings and another mask, eager passes between."""
    from primus_amd.pytorch import ops

    w = _weights(gpu, 5)
    tokens = 200
    x = torch.randn(tokens, HIDDEN, device=gpu).bfloat16().requires_grad_()
    dy = torch.randn(tokens, HIDDEN, device=gpu).bfloat16()
    mask = torch.ones(tokens, dtype=torch.bool, device=gpu)

    def step():
        y, idx, counts = _layer(ops, x, w, mask, 32)
        return [y.detach(), idx, counts, *torch.autograd.grad(y, [x] + [getattr(w, n) for n in NAMES], dy)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(4):
        gen = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn(tokens, HIDDEN, generator=gen).bfloat16())
            dy.copy_(torch.randn(tokens, HIDDEN, generator=gen).bfloat16())
            mask.copy_(torch.rand(tokens, generator=gen) < (1.0, 0.5, 0.0, 0.9)[seed])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        want = step()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), (seed, i)


def test_two_graphs_and_eager_passes_do_not_share_anything(gpu):
    """Two captured graphs with split contractions (a workspace each) replayed in turn on two streams."""
    from primus_amd.pytorch import ops

    gen = torch.Generator(device=gpu).manual_seed(1)
    a = [torch.randn(70, 4096, generator=gen, device=gpu).bfloat16() for _ in range(2)]
    b = torch.randn(256, 4096, generator=gen, device=gpu).bfloat16()
    want = [ops.gemm_bias_act(t, b, activation="gelu") for t in a]
    graphs, outs = [], []
    for t in a:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.gemm_bias_act(t, b, activation="gelu"))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        assert torch.equal(ops.gemm_bias_act(a[0], b, activation="gelu"), want[0])
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert torch.equal(got, ref)


def test_expert_mlp_of_the_megatron_side(gpu):
    """PrimusGroupedMLP between the two moves, in MXFP8 with rows padded by the permutation, against its bf16 route: the bar the
    expert MLP's own test has (cosine 0.99)."""
    import contextlib

    from primus_amd.megatron import runtime
    from primus_amd.megatron.extensions import primus_turbo as pt
    from primus_amd.megatron.transformer.experts import PrimusGroupedMLP
    from primus_amd.pytorch import ops
    from primus_amd.pytorch.core import Format, ScaleDtype, ScalingGranularity

    pt.PrimusTurboLowPrecisionGlobalStateManager.reset()
    runtime.bind()
    runtime.set_args(enable_primus_turbo=True, use_turbo_gemm=True, use_turbo_grouped_gemm=True, use_turbo_fused_act_with_probs=True,
                     moe_router_padding_for_quantization=True)
    runtime.set_num_microbatches(1)
    try:
        torch.manual_seed(6)
        mlp = PrimusGroupedMLP(8, SimpleNamespace(
            params_dtype=torch.bfloat16, use_cpu_initialization=False, perform_initialization=True, tensor_model_parallel_size=1, gradient_accumulation_fusion=False,
            normalization="RMSNorm", layernorm_epsilon=1e-5, hidden_size=256, ffn_hidden_size=512, moe_ffn_hidden_size=512, gated_linear_unit=True,
            activation_func=torch.nn.functional.silu, fp8="e4m3", fp8_recipe="mxfp8", fp4=None, add_bias_linear=False))
        x = torch.randn(300, 256, device=gpu).bfloat16()
        logits = torch.randn(300, 8, device=gpu)
        dy = torch.randn(300, 256, device=gpu).bfloat16()
        cfg = pt.PrimusTurboQuantConfig(granularity=ScalingGranularity.MX_BLOCKWISE, format=Format.E4M3, block_size=32, scale_dtype=ScaleDtype.E8M0)

        def run(ctx, multiple):
            xi, li = x.clone().requires_grad_(), logits.clone().requires_grad_()
            probs, idx, _ = ops.topk_routing(li, 2)
            with ctx:
                align = pt.router_pad_multiple(True) or multiple
                rows, row_probs, lens, perm = ops.permute_tokens(xi, idx, 8, probs=probs, align=align)
                out, _ = mlp(rows, lens, row_probs)
            y = ops.unpermute_tokens(out, perm)
            return [y.detach(), *torch.autograd.grad(y, [xi, li, mlp.linear_fc1.weights, mlp.linear_fc2.weights], dy)], align

        ref, plain_align = run(contextlib.nullcontext(), 1)
        got, align = run(pt.primus_turbo_fp8_autocast(enabled=False, enabled_turbo=True, turbo_quant_config=cfg), 1)
        assert (plain_align, align) == (1, 32)
        for name, a, b in zip(("y", "dx", "dlogits", "dw1", "dw2"), got, ref):
            cos = torch.nn.functional.cosine_similarity(a.float().flatten(), b.float().flatten(), dim=0).item()
            assert math.isfinite(cos) and cos >= 0.99, (name, cos)
    finally:
        pt.PrimusTurboLowPrecisionGlobalStateManager.reset()
        runtime.set_args()
        runtime.set_num_microbatches(1)


def test_a_second_derivative_is_refused(gpu):
    """The gradients are kernels' outputs with no graph behind them: what depends on them through a second backward raises."""
    from primus_amd.pytorch import ops

    logits = torch.randn(40, 8, device=gpu, requires_grad=True)
    x = torch.randn(40, 64, device=gpu).bfloat16().requires_grad_()
    w = torch.randn(96, 64, device=gpu).bfloat16().requires_grad_()
    probs, idx, _ = ops.topk_routing(logits, 2)
    rows, _, _, order = ops.permute_tokens(x, idx, 8)
    outputs = [(probs, logits), (rows, x), (ops.unpermute_tokens(rows.detach().requires_grad_(), order, probs), logits),
               (ops.gemm_bias_act(x, w, activation="gelu"), x)]
    for y, leaf in outputs:
        dy = torch.ones_like(y).requires_grad_()
        (plain,) = torch.autograd.grad(y, leaf, dy.detach(), retain_graph=True)
        (g,) = torch.autograd.grad(y, leaf, dy, create_graph=True)
        assert torch.equal(g, plain)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


def test_saved_tensors_through_host_memory_and_with_other_strides(gpu):
    """What autograd kept may come back from hooks: the same values give the same gradients, other strides are refused."""
    from primus_amd.pytorch import ops

    gen = torch.Generator().manual_seed(11)
    logits, x, w = torch.randn(50, 8, generator=gen).to(gpu), torch.randn(50, 64, generator=gen).bfloat16().to(gpu), torch.randn(96, 64, generator=gen).bfloat16().to(gpu)
    with torch.no_grad():
        _, idx, _ = ops.topk_routing(logits, 2)
        probs = torch.rand(50, 2, generator=gen).to(gpu)
        rows, _, _, order = ops.permute_tokens(x, idx, 8, align=32)
    leaves = [t.clone().requires_grad_() for t in (logits, x, rows, probs, w)]
    runs = [(lambda: ops.topk_routing(leaves[0], 2)[0], leaves[:1]), (lambda: ops.permute_tokens(leaves[1], idx, 8)[0], leaves[1:2]),
            (lambda: ops.unpermute_tokens(leaves[2], order, leaves[3]), leaves[2:4]), (lambda: ops.gemm_bias_act(leaves[1], leaves[4], activation="silu"), [leaves[1], leaves[4]])]
    for run, inputs in runs:
        y = run()
        dy = torch.randn(y.shape, generator=gen).to(gpu).to(y.dtype)
        want = torch.autograd.grad(y, inputs, dy)
        with torch.autograd.graph.save_on_cpu():
            y = run()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, inputs, dy), want))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.t().contiguous(), lambda t: t.t()):
            y = run()
        with pytest.raises(ValueError):
            torch.autograd.grad(y, inputs, dy)
