"""What stands around the expert MLP and the unquantised linear of an MoE training or serving program, as cases that can
be timed and compared: the router's choice of experts (``ops.topk_routing``), the move of the tokens' rows into the
experts' order and back (``ops.permute_tokens`` / ``ops.unpermute_tokens``), and a dense bf16 linear with bias, activation
and residual in its epilogue (``ops.gemm_bias_act``).

``own`` False: every operator in its plain form, elementary torch operations in 32 bits (choices between experts that
depend on computed scores in 64); True: the calls a program makes of the framework.

A case holds ``op`` and the operator's sizes and options; ``backward``: the pass takes the gradients too.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- the cases ----------------------------------------------------------------------------------------------------
def _route(name, tokens, experts, topk, score="softmax", dtype="fp32", bias=False, groups=0, group_topk=0, renorm=True, scale=1.0, masked=0.0, backward=True):
    return dict(name=name, op="route", tokens=tokens, experts=experts, topk=topk, score=score, dtype=dtype, bias=bias, groups=groups,
                group_topk=group_topk, renorm=renorm, scale=scale, masked=masked, backward=backward)


def _move(name, op, tokens, experts, topk, hidden, dtype="bf16", align=1, probs=True, dropped=0.0, backward=True):
    return dict(name=name, op=op, tokens=tokens, experts=experts, topk=topk, hidden=hidden, dtype=dtype, align=align, probs=probs,
                dropped=dropped, backward=backward)


def _linear(name, m, n, k, bias=True, act="", residual=False, backward=True):
    return dict(name=name, op="linear", m=m, n=n, k=k, bias=bias, act=act, residual=residual, backward=backward)


def listed():
    return [
        # a decode step of GPT-OSS-120B's router: a few sequences, top 4 of 128
        _route("route_decode", 8, 128, 4, backward=False),
        # Mixtral-8x7B training: 16384 tokens, top 2 of 8
        _route("route_mixtral", 16384, 8, 2, dtype="bf16"),
        # DeepSeek-V3 training: sigmoid scores with the balancing bias, 4 of 8 groups, top 8 of 256
        _route("route_deepseek", 16384, 256, 8, score="sigmoid", bias=True, groups=8, group_topk=4, scale=2.5),
        # a padded batch of odd size, scores not renormalised
        _route("route_padded", 5003, 160, 6, renorm=False, scale=16.0, masked=0.1, dtype="bf16"),
        # serving GPT-OSS-120B: a few tokens into expert order
        _move("permute_decode", "permute", 32, 128, 4, 2880, backward=False),
        # Mixtral-8x7B training: 16384 tokens twice each
        _move("permute_mixtral", "permute", 16384, 8, 2, 4096),
        # a batch with padded tokens, rows padded to the MX block
        _move("unpermute_padded", "unpermute", 1801, 32, 6, 2880, align=32, dropped=0.07),
        # DeepSeek-V3: eight rows a token summed with their probabilities, and the gradients of both
        _move("unpermute_deepseek", "unpermute", 8192, 256, 8, 7168),
        # one token through a Llama-3-8B-sized projection: bound by the weight
        _linear("linear_decode", 1, 14336, 4096, act="silu", backward=False),
        # a short prompt of odd length through the projection back, residual added
        _linear("linear_short", 333, 4096, 14336, residual=True, backward=False),
        # odd rows and the GPT-OSS width, everything in the epilogue, fine-tuning
        _linear("linear_odd", 2051, 2880, 2880, act="gelu", residual=True),
        # Llama-3-8B-sized training: 8192 tokens
        _linear("linear_train", 8192, 14336, 4096, act="gelu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("route", "permute", "unpermute", "linear"))
    backward = rng.random() < 0.6
    if op == "linear":
        n, k = (32 * _log(rng, 4, 448) for _ in range(2))
        m = _log(rng, 1, max(1, min(16384, 8192 * 14336 * 4096 // (n * k))))
        c = _linear("", m, n, k, bias=rng.random() < 0.8, act=rng.choice(("", "silu", "gelu", "relu")), residual=rng.random() < 0.5, backward=backward)
    elif op == "route":
        topk = rng.randint(1, 10)
        experts = max(topk, _log(rng, 4, 512))
        groups, group_topk = 0, 0
        score = rng.choice(("softmax", "sigmoid"))
        if rng.random() < 0.4 and topk <= 8:
            groups = rng.choice((2, 4, 8))
            group_topk = rng.randint(1, groups)
            experts = groups * max(1, round(experts / groups), -(-topk // group_topk))
        c = _route("", _log(rng, 1, 16384 if experts <= 256 else 8192), experts, topk, score=score, dtype=rng.choice(("fp32", "bf16", "fp16")),
                   bias=rng.random() < 0.5, groups=groups, group_topk=group_topk, renorm=topk > 1 and rng.random() < 0.6,
                   scale=rng.choice((1.0, 2.5)), masked=rng.choice((0.0, 0.0, 0.2)), backward=backward)
    else:
        topk = rng.randint(1, 8)
        experts = max(topk, _log(rng, 4, 512))
        hidden = _log(rng, 64, 8192) if rng.random() < 0.3 else 32 * _log(rng, 2, 256)
        tokens = _log(rng, 1, max(1, min(32768, 8192 * 8 * 7168 // (topk * hidden))))
        c = _move("", op, tokens, experts, topk, hidden, dtype=rng.choice(("bf16", "bf16", "fp16")), align=rng.choice((1, 1, 16, 32)),
                  probs=rng.random() < 0.7, dropped=rng.choice((0.0, 0.0, 0.1)), backward=backward)
    del c["name"]
    return c


# ---- inputs -------------------------------------------------------------------------------------------------------
def _rows(c):
    return (c["tokens"] * c["topk"] + c["experts"] * (c["align"] - 1)) // c["align"] * c["align"]


def _pick_experts(c, gen):
    """[T, K] different experts a token, some experts busier than others; entries of padded tokens are -1."""
    dev = gen.device
    logits = torch.randn(c["tokens"], c["experts"], generator=gen, device=dev) + torch.randn(c["experts"], generator=gen, device=dev)
    idx = torch.topk(logits, c["topk"], dim=1).indices
    if c["dropped"]:
        idx[torch.rand(c["tokens"], generator=gen, device=dev) < c["dropped"]] = -1
    return idx


def _places(idx, experts, align):
    """Row of every entry (-1: dropped) and the rows of every expert, the last one's up to the buffer's end: a stable sort by expert."""
    flat = idx.reshape(-1)
    n = flat.numel()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    counts = (key[:, None] == torch.arange(experts, device=key.device)).sum(0) if n * experts <= 1 << 26 else torch.bincount(key, minlength=experts + 1)[:experts]
    padded = (counts + align - 1) // align * align
    off = torch.cumsum(padded, 0) - padded
    skip = torch.cumsum(counts, 0) - counts
    key_sorted, order = torch.sort(key, stable=True)
    live = key_sorted < experts
    e = key_sorted.clamp(max=experts - 1)
    row_sorted = torch.where(live, torch.arange(n, device=key.device) - skip[e] + off[e], -1)
    row = torch.empty_like(row_sorted)
    row[order] = row_sorted
    rows = (n + experts * (align - 1)) // align * align
    lens = padded.clone()
    lens[-1] = rows - off[-1]
    return row.view(idx.shape), lens


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    dev = gen.device
    s = {"case": c}

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dtype)

    if c["op"] == "route":
        t, e, k = c["tokens"], c["experts"], c["topk"]
        s["logits"] = (normal(t, e) + normal(e)).to(_DTYPES[c["dtype"]])
        s["bias"] = normal(e, scale=0.05) if c["bias"] else None
        s["mask"] = torch.rand(t, generator=gen, device=dev) >= c["masked"] if c["masked"] else None
        s["dprobs"] = normal(t, k) if c["backward"] else None
        if c["backward"]:
            s["logits"].requires_grad_(own)
    elif c["op"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        bf = torch.bfloat16
        s["a"], s["b"] = normal(m, k, dtype=bf), normal(n, k, dtype=bf, scale=k ** -0.5)
        s["bias"] = normal(n, dtype=bf, scale=0.5) if c["bias"] else None
        s["residual"] = normal(m, n, dtype=bf) if c["residual"] else None
        s["dy"] = normal(m, n, dtype=bf) if c["backward"] else None
        if c["backward"]:
            for name in ("a", "b", "bias", "residual"):
                if s[name] is not None:
                    s[name].requires_grad_(own)
    else:
        dt = _DTYPES[c["dtype"]]
        s["indices"] = _pick_experts(c, gen)
        s["probs"] = torch.rand(c["tokens"], c["topk"], generator=gen, device=dev) if c["probs"] else None
        if c["op"] == "permute":
            s["x"] = normal(c["tokens"], c["hidden"], dtype=dt)
            if c["backward"]:
                s["drows"] = normal(_rows(c), c["hidden"], dtype=dt)
                s["drow_probs"] = normal(_rows(c)) if c["probs"] else None
                s["x"].requires_grad_(own)
        else:
            # the experts' output, and where permute_tokens put every entry
            s["rows"] = normal(_rows(c), c["hidden"], dtype=dt)
            if own:
                from primus_amd.pytorch import ops

                s["permutation"] = ops.permute_tokens(s["rows"][:c["tokens"]], s["indices"], c["experts"], align=c["align"])[3]
            else:
                s["row_of"] = _places(s["indices"], c["experts"], c["align"])[0]
            if c["backward"]:
                s["dy"] = normal(c["tokens"], c["hidden"], dtype=dt)
                s["rows"].requires_grad_(own)
        if c["backward"] and c["probs"]:
            s["probs"].requires_grad_(own)
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _scores(logits, score):
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits))
    x = torch.exp(logits - logits.max(dim=1, keepdim=True).values)
    return x / x.sum(dim=1, keepdim=True)


def _choose(c, logits, bias):
    """Indices of the experts, best first, ties to the lower index.  Without bias and groups the order of the scores is that
    of the logits; otherwise the scores are compared in 64 bits."""
    k, groups = c["topk"], c["groups"]
    if bias is None and not groups:
        choice = logits.float()
    else:
        choice = _scores(logits.double(), c["score"])
        if bias is not None:
            choice = choice + bias.double()
        if groups:
            t, e = choice.shape
            inside = torch.sort(choice.view(t, groups, e // groups), dim=2, descending=True).values
            best = inside[:, :, :max(1, min(k // c["group_topk"], e // groups))].sum(2)
            order = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["group_topk"]]
            keep = torch.zeros(t, groups, dtype=torch.bool, device=choice.device)
            keep[torch.arange(t, device=choice.device)[:, None], order] = True
            choice = torch.where(keep[:, :, None].expand(t, groups, e // groups).reshape(t, e), choice, -math.inf)
    return torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :k].contiguous()


def _plain_route(s):
    c, logits, mask = s["case"], s["logits"], s["mask"]
    idx = _choose(c, logits, s["bias"])
    score = _scores(logits.float(), c["score"])
    w = score.gather(1, idx)
    total = w.sum(1, keepdim=True) + (1e-20 if c["score"] == "sigmoid" else 0.0)
    probs = (w / total if c["renorm"] else w) * c["scale"]
    live = torch.ones(logits.shape[0], dtype=torch.bool, device=logits.device) if mask is None else mask
    out_idx = torch.where(live[:, None], idx, -1)
    out = [torch.where(live[:, None], probs, 0.0), out_idx, (out_idx[:, :, None] == torch.arange(c["experts"], device=idx.device)).sum((0, 1))]
    if c["backward"]:
        g = s["dprobs"] * c["scale"]
        if c["renorm"]:
            g = (g - (g * (w / total)).sum(1, keepdim=True)) / total
        if c["score"] == "sigmoid":
            dl = torch.zeros_like(score).scatter(1, idx, g * w * (1.0 - w))
        else:
            dl = torch.zeros_like(score).scatter(1, idx, g * w) - score * (g * w).sum(1, keepdim=True)
        out.append(torch.where(live[:, None], dl, 0.0).to(logits.dtype))
    return out


def _plain_permute(s):
    c, x = s["case"], s["x"]
    row_of, lens = _places(s["indices"], c["experts"], c["align"])
    rows = x.new_zeros(_rows(c), c["hidden"])
    token, slot = torch.nonzero(row_of >= 0, as_tuple=True)
    at = row_of[token, slot]
    rows[at] = x[token]
    out = [rows, None, lens, row_of]
    if c["probs"]:
        out[1] = torch.zeros(_rows(c), device=x.device)
        out[1][at] = s["probs"][token, slot]
    if c["backward"]:
        dx = torch.zeros(c["tokens"], c["hidden"], device=x.device)
        for j in range(c["topk"]):
            dx += torch.where(row_of[:, j, None] >= 0, s["drows"][row_of[:, j].clamp(min=0)].float(), 0.0)
        out.append(dx.to(x.dtype))
        if c["probs"]:
            out.append(torch.where(row_of >= 0, s["drow_probs"][row_of.clamp(min=0)], 0.0))
    return out


def _plain_unpermute(s):
    c, rows, row_of = s["case"], s["rows"], s["row_of"]
    y = torch.zeros(c["tokens"], c["hidden"], device=rows.device)
    live, at = row_of >= 0, row_of.clamp(min=0)
    for j in range(c["topk"]):
        part = rows[at[:, j]].float()
        if c["probs"]:
            part = part * s["probs"][:, j, None]
        y += torch.where(live[:, j, None], part, 0.0)
    out = [y.to(rows.dtype)]
    if c["backward"]:
        dy = s["dy"].float()
        drows = torch.zeros_like(rows)
        dprobs = torch.zeros(c["tokens"], c["topk"], device=rows.device)
        for j in range(c["topk"]):
            part = dy * s["probs"][:, j, None] if c["probs"] else dy
            drows[at[live[:, j], j]] = part[live[:, j]].to(rows.dtype)
            if c["probs"]:
                dprobs[:, j] = torch.where(live[:, j], (rows[at[:, j]].float() * dy).sum(1), 0.0)
        out += [drows, dprobs] if c["probs"] else [drows]
    return out


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, 0.0)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return sig * (1.0 + z * (1.0 - sig))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    return torch.ones_like(z)


def _plain_linear(s):
    c, bf = s["case"], torch.bfloat16
    a, b = s["a"].float(), s["b"].float()
    z = a @ b.t()
    if c["bias"]:
        z = z + s["bias"].float()
    y = _act(z, c["act"])
    if c["residual"]:
        y = y + s["residual"].float()
    out = [y.to(bf)]
    if c["backward"]:
        dz = s["dy"].float() * _act_slope(z, c["act"])
        out += [(dz @ b).to(bf), (dz.t() @ a).to(bf)]
        if c["bias"]:
            out.append(dz.sum(0).to(bf))
        if c["residual"]:
            out.append(s["dy"])
    return out


# ---- the framework's calls ----------------------------------------------------------------------------------------
def _own_route(s):
    from primus_amd.pytorch import ops

    c = s["case"]
    probs, idx, counts = ops.topk_routing(s["logits"], c["topk"], score_function=c["score"], expert_bias=s["bias"], num_groups=c["groups"] or None,
                                          group_topk=c["group_topk"] or None, renormalize=c["renorm"], scaling_factor=c["scale"], token_mask=s["mask"])
    out = [probs.detach(), idx, counts]
    if c["backward"]:
        out += torch.autograd.grad(probs, s["logits"], s["dprobs"])
    return out


def _own_permute(s):
    from primus_amd.pytorch import ops

    c = s["case"]
    rows, row_probs, lens, permutation = ops.permute_tokens(s["x"], s["indices"], c["experts"], probs=s["probs"], align=c["align"])
    out = [rows.detach(), None if row_probs is None else row_probs.detach(), lens, permutation.row_of]
    if c["backward"]:
        if c["probs"]:
            out += torch.autograd.grad([rows, row_probs], [s["x"], s["probs"]], [s["drows"], s["drow_probs"]])
        else:
            out += torch.autograd.grad(rows, s["x"], s["drows"])
    return out


def _own_unpermute(s):
    from primus_amd.pytorch import ops

    c = s["case"]
    y = ops.unpermute_tokens(s["rows"], s["permutation"], probs=s["probs"])
    out = [y.detach()]
    if c["backward"]:
        out += torch.autograd.grad(y, [s["rows"], s["probs"]] if c["probs"] else s["rows"], s["dy"])
    return out


def _own_linear(s):
    from primus_amd.pytorch import ops

    c = s["case"]
    y = ops.gemm_bias_act(s["a"], s["b"], bias=s["bias"], activation=c["act"] or None, residual=s["residual"])
    out = [y.detach()]
    if c["backward"]:
        out += torch.autograd.grad(y, [s[name] for name in ("a", "b", "bias", "residual") if s[name] is not None], s["dy"])
    return out


_PLAIN = {"route": _plain_route, "permute": _plain_permute, "unpermute": _plain_unpermute, "linear": _plain_linear}
_OWN = {"route": _own_route, "permute": _own_permute, "unpermute": _own_unpermute, "linear": _own_linear}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "route":
        t, e, k = c["tokens"], c["experts"], c["topk"]
        size = 4 if c["dtype"] == "fp32" else 2
        nbytes = t * e * size + t * k * 12 + e * 8 + (e * 4 if c["bias"] else 0) + (t if c["masked"] else 0)
        if c["backward"]:
            # the probabilities' gradient in, the logits' out; the logits are read for the forward
            nbytes += t * k * 4 + t * e * size
        return {"bytes": nbytes, "flops": 4 * t * e * (2 if c["backward"] else 1)}
    if c["op"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        nbytes = 2 * (m * k + n * k + m * n * (2 if c["residual"] else 1) + (n if c["bias"] else 0))
        flops = 2 * m * n * k
        if c["backward"]:
            nbytes += 2 * (m * n + m * k + n * k + (n if c["bias"] else 0))
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    t, k, h, r = c["tokens"], c["topk"], c["hidden"], _rows(c)
    size = 4 if c["dtype"] == "fp32" else 2
    live = t * k * (1.0 - c["dropped"])
    if c["op"] == "permute":
        nbytes = t * h * size + r * h * size + t * k * 16 + (t * k * 4 + r * 4 if c["probs"] else 0)
        flops = 0
        if c["backward"]:
            nbytes += live * h * size + t * h * size + (r * 4 + t * k * 4 if c["probs"] else 0)
            flops = live * h
    else:
        nbytes = live * h * size + t * h * size + t * k * 8 + (t * k * 4 if c["probs"] else 0)
        flops = 2 * live * h
        if c["backward"]:
            nbytes += t * h * size + r * h * size + (t * k * 4 if c["probs"] else 0)
            flops += 3 * live * h
    return {"bytes": int(nbytes), "flops": int(flops)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def _exact_route(s):
    c = s["case"]
    k, eps = c["topk"], 1e-20 if c["score"] == "sigmoid" else 0.0
    parts = []
    for lo in range(0, c["tokens"], 1024):
        l = s["logits"].detach()[lo:lo + 1024].double()
        p = torch.sigmoid(l) if c["score"] == "sigmoid" else torch.softmax(l, 1)
        order = l if s["bias"] is None and not c["groups"] else p if s["bias"] is None else p + s["bias"].double()
        lower = torch.arange(c["experts"], device=l.device)
        if c["groups"]:
            g = order.view(len(l), c["groups"], -1)
            take = max(1, min(k // c["group_topk"], g.shape[2]))
            best = g.topk(take, dim=2).values.sum(2)
            gi = torch.arange(c["groups"], device=l.device)
            ahead = (best[:, None, :] > best[:, :, None]) | ((best[:, None, :] == best[:, :, None]) & (gi[None, :] < gi[:, None]))
            order = torch.where((ahead.sum(2) < c["group_topk"])[:, :, None], g, -math.inf).reshape(len(l), -1)
        # an expert's place is the number of experts ahead of it
        ahead = (order[:, None, :] > order[:, :, None]) | ((order[:, None, :] == order[:, :, None]) & (lower[None, :] < lower[:, None]))
        place = ahead.sum(2)
        idx = torch.stack([(place == j).to(torch.int8).argmax(1) for j in range(k)], 1)
        chosen = place < k
        w = torch.where(chosen, p, 0.0)
        total = w.sum(1, keepdim=True) + eps
        full = w / total if c["renorm"] else w
        probs = full.gather(1, idx) * c["scale"]
        dl = None
        if c["backward"]:
            g = torch.zeros_like(p).scatter(1, idx, s["dprobs"][lo:lo + 1024].double() * c["scale"])
            dp = torch.where(chosen, (g - (g * full).sum(1, keepdim=True)) / total, 0.0) if c["renorm"] else g
            dl = dp * p * (1 - p) if c["score"] == "sigmoid" else p * (dp - (dp * p).sum(1, keepdim=True))
        if s["mask"] is not None:
            live = s["mask"][lo:lo + 1024, None]
            idx, probs = torch.where(live, idx, -1), torch.where(live, probs, 0.0)
            dl = None if dl is None else torch.where(live, dl, 0.0)
        parts.append((probs, idx, dl))
    idx = torch.cat([x[1] for x in parts])
    out = [torch.cat([x[0] for x in parts]), idx, torch.bincount(idx[idx >= 0], minlength=c["experts"])]
    return out + [torch.cat([x[2] for x in parts])] if c["backward"] else out


def _exact_places(c, idx):
    """Expert after expert: where its entries stand in the list, in their order."""
    flat = idx.reshape(-1)
    row, lens, at = torch.full_like(flat, -1), [], 0
    for e in range(c["experts"]):
        where = torch.nonzero(flat == e).reshape(-1)
        row[where] = at + torch.arange(len(where), device=flat.device)
        lens.append(-(-len(where) // c["align"]) * c["align"])
        at += lens[-1]
    lens[-1] += _rows(c) - at
    return row, torch.tensor(lens, device=flat.device)


def _exact_move(s):
    c = s["case"]
    row, lens = _exact_places(c, s["indices"])
    entry = torch.nonzero(row >= 0).reshape(-1)
    at, token = row[entry], entry // c["topk"]
    w = s["probs"].detach().double().reshape(-1)[entry] if c["probs"] else None
    zeros = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device=row.device)  # noqa: E731
    if c["op"] == "permute":
        out = [zeros(_rows(c), c["hidden"]).index_copy(0, at, s["x"].detach().double()[token]), None, lens, row.view(c["tokens"], -1)]
        if c["probs"]:
            out[1] = zeros(_rows(c)).index_copy(0, at, w)
        if c["backward"]:
            out.append(zeros(c["tokens"], c["hidden"]).index_add(0, token, s["drows"][at].double()))
            if c["probs"]:
                out.append(zeros(c["tokens"] * c["topk"]).index_copy(0, entry, s["drow_probs"][at].double()).view(c["tokens"], -1))
        return out
    y, drows = zeros(c["tokens"], c["hidden"]), zeros(_rows(c), c["hidden"]) if c["backward"] else None
    dp = zeros(c["tokens"] * c["topk"])
    for lo in range(0, len(entry), 8192):
        e, r, t = entry[lo:lo + 8192], at[lo:lo + 8192], token[lo:lo + 8192]
        part = s["rows"].detach()[r].double()
        scale = w[lo:lo + 8192, None] if c["probs"] else 1.0
        y.index_add_(0, t, part * scale)
        if c["backward"]:
            d = s["dy"][t].double()
            drows[r] = d * scale
            dp[e] = (d * part).sum(1)
    if not c["backward"]:
        return [y]
    return [y, drows, dp.view(c["tokens"], -1)] if c["probs"] else [y, drows]


def _exact_linear(s):
    c = s["case"]
    a, b = s["a"].detach().double(), s["b"].detach().double()
    bias = s["bias"].detach().double() if c["bias"] else torch.zeros(c["n"], dtype=torch.float64, device=a.device)
    z = torch.addmm(bias, a, b.t())
    p = torch.sigmoid(z) if c["act"] == "silu" else 0.5 * torch.erfc(-z / math.sqrt(2.0)) if c["act"] == "gelu" else None
    y = z.clamp(min=0) if c["act"] == "relu" else z if p is None else z * p
    out = [y + s["residual"].detach().double() if c["residual"] else y]
    if c["backward"]:
        dz = s["dy"].double()
        if c["act"] == "relu":
            dz = dz * (z > 0)
        elif c["act"] == "silu":
            dz = dz * (p + z * p * (1 - p))
        elif c["act"] == "gelu":
            dz = dz * (p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
        out += [torch.mm(dz, b), torch.mm(dz.t(), a)]
        if c["bias"]:
            out.append(torch.mv(dz.t(), torch.ones(c["m"], dtype=torch.float64, device=a.device)))
        if c["residual"]:
            out.append(s["dy"].double())
    return out


def exact(case, seed):
    """What ``run`` returns for these inputs, from the definitions in 64 bits."""
    global own
    was, own = own, False       # the inputs without the framework's handle
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"route": _exact_route, "permute": _exact_move, "unpermute": _exact_move, "linear": _exact_linear}[case["op"]](s)
