"""The operators of a feed-forward block with experts, as measurable cases.

``residual_norm``   ``kernels.block_norm.residual_norm``: the norm after a block, its gate and residual scale, the
                    residual sum and the norm before the next block; alone (inference) or with the gradients of every
                    input (``"step": True``).
``expert_route``    ``kernels.experts.expert_route``: scores, choice of the k best experts of a token, their weights, and
                    the CSR of the experts' slots; with the gradient of the logits.
``expert_linear``   ``kernels.experts.expert_linear``: every slot's rows times its expert's matrix, with an optional gated
                    SiLU; with the gradients of rows and matrices.
``expert_combine``  ``kernels.experts.expert_combine``: the weighted sum of a token's slots; with both gradients.

With ``own`` false ``run`` computes the same from elementary torch operations.

A token has k slots, numbered token * k + j.  The dispatch lists them expert by expert: place p holds the slot
``order[p]``, expert e owns the places ``offsets[e]`` to ``offsets[e + 1]``, and ``slots[t, j]`` is the place of slot
(t, j).  A slot without an expert (-1) has no place: its entry of ``slots`` is -1, and so are the last entries of ``order``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1.0e-6


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # The smallest call: the pooled feature rows of 64 frames at inference.
        {"name": "norm_pooled", "op": "residual_norm", "rows": 64, "width": 64, "dtype": "float32",
         "residual": "float32", "gate": "none", "activation": "none", "post": True, "pre": True, "scale": "number", "step": False},
        # Node features [24576, 16 * 64] of one box in training, gated, with a learned residual scale.
        {"name": "norm_nodes_step", "op": "residual_norm", "rows": 24576, "width": 1024, "dtype": "float32",
         "residual": "float32", "gate": "full", "activation": "sigmoid", "post": True, "pre": True, "scale": "channels", "step": True},
        # A bfloat16 block on a float32 residual stream, an odd width, one gate a row, in training.
        {"name": "norm_odd_step", "op": "residual_norm", "rows": 30011, "width": 810, "dtype": "bfloat16",
         "residual": "float32", "gate": "row", "activation": "silu", "post": True, "pre": True, "scale": "channels", "step": True},
        # One frame of 192 atoms at inference, two of eight experts.
        {"name": "route_frame", "op": "expert_route", "tokens": 192, "experts": 8, "k": 2, "scores": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "dtype": "float32", "masked": 0.0, "step": False},
        # A box of 24,576 atoms in training: sigmoid scores, a bias for balance, 4 of 8 groups, 6 of 64 experts, padded rows.
        {"name": "route_box_step", "op": "expert_route", "tokens": 24576, "experts": 64, "k": 6, "scores": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "dtype": "float32", "masked": 0.05, "step": True},
        # 65,536 tokens over 256 experts, 8 of them each, bfloat16 logits, in training.
        {"name": "route_large_step", "op": "expert_route", "tokens": 65536, "experts": 256, "k": 8, "scores": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "dtype": "bfloat16", "masked": 0.0, "step": True},
        # Eight tokens through the first matrices of 32 experts, 4 each: what bounds it is reading the matrices.
        {"name": "linear_tokens", "op": "expert_linear", "tokens": 8, "inner": 1, "experts": 32, "k": 4, "k_in": 1024, "n_out": 2048,
         "source": "tokens", "gated": True, "dtype": "bfloat16", "masked": 0.0, "step": False},
        # Node features [24576, 16, 64] through two of eight experts in training, float32.
        {"name": "linear_nodes_step", "op": "expert_linear", "tokens": 24576, "inner": 16, "experts": 8, "k": 2, "k_in": 64,
         "n_out": 64, "source": "tokens", "gated": False, "dtype": "float32", "masked": 0.0, "step": True},
        # The largest: the first, gated matrices of 32 experts over 8,192 tokens, 4 experts each, in training.
        {"name": "linear_large_step", "op": "expert_linear", "tokens": 8192, "inner": 1, "experts": 32, "k": 4, "k_in": 1024,
         "n_out": 2048, "source": "tokens", "gated": True, "dtype": "bfloat16", "masked": 0.0, "step": True},
        # The second matrices at odd sizes, float16, some slots without an expert, in training.
        {"name": "linear_odd_step", "op": "expert_linear", "tokens": 3001, "inner": 9, "experts": 13, "k": 3, "k_in": 250,
         "n_out": 90, "source": "slots", "gated": False, "dtype": "float16", "masked": 0.1, "step": True},
        # The two slots of each of 192 atoms, [16, 64] rows, at inference.
        {"name": "combine_frame", "op": "expert_combine", "tokens": 192, "inner": 16, "experts": 8, "k": 2, "width": 64,
         "dtype": "float32", "masked": 0.0, "step": False},
        # Four slots each of 16,384 tokens in training.
        {"name": "combine_large_step", "op": "expert_combine", "tokens": 16384, "inner": 1, "experts": 32, "k": 4, "width": 1024,
         "dtype": "bfloat16", "masked": 0.02, "step": True},
    ]


def _log(rng, low, high):
    """An integer spread over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw(rng):
    op = rng.choice(["residual_norm", "expert_route", "expert_linear", "expert_linear", "expert_combine"])
    dtype, step = rng.choice(["float32", "bfloat16", "float16"]), rng.random() < 0.5
    if op == "residual_norm":
        gate = rng.choice(["none", "full", "row"])
        return {"op": op, "rows": _log(rng, 1, 65536), "width": _log(rng, 8, 8192), "dtype": dtype,
                "residual": rng.choice(["float32", dtype]), "gate": gate,
                "activation": "none" if gate == "none" else rng.choice(["none", "sigmoid", "silu"]),
                "post": rng.random() < 0.7, "pre": rng.random() < 0.9, "scale": rng.choice(["none", "number", "channels"]), "step": step}
    masked = rng.choice([0.0, 0.05, 0.3])
    if op == "expert_route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log(rng, 2, 512 // groups)
        top_groups = rng.randint(1, groups)
        return {"op": op, "tokens": _log(rng, 1, 65536), "experts": experts,
                "k": rng.randint(1, min(10, top_groups * (experts // groups))), "scores": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups, "dtype": dtype, "masked": masked, "step": step}
    inner, experts = rng.choice([1, 1, 1, 9, 16]), _log(rng, 1, 128)
    case = {"op": op, "tokens": _log(rng, 1, 32768), "inner": inner, "experts": experts, "k": rng.randint(1, min(8, experts))}
    if op == "expert_linear":
        return {**case, "k_in": _log(rng, 16, 4096), "n_out": _log(rng, 16, 4096), "source": rng.choice(["tokens", "slots"]),
                "gated": rng.random() < 0.4, "dtype": dtype, "masked": masked, "step": step}
    return {**case, "width": _log(rng, 16, 4096), "dtype": dtype, "masked": masked, "step": step}


def _cost(case):
    """About the time of a case: its bytes and its products."""
    w = work(case)
    return w["bytes"] / 4.0e12 + w["flops"] / (1.0e14 if case["dtype"] == "float32" else 1.0e15)


def draw(rng):
    most = max(_cost(case) for case in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= most and work(case)["flops"] <= 8.3e11 and work(case)["bytes"] <= 4.0e9:
            return case


def work(case):
    """Each input read once, each output written once."""
    size, step = (4 if case["dtype"] == "float32" else 2), case["step"]
    if case["op"] == "residual_norm":
        values, stream = case["rows"] * case["width"], (4 if case["residual"] == "float32" else 2)
        gate = {"none": 0, "full": values, "row": case["rows"]}[case["gate"]]
        y = case["pre"] * values * size
        # x, residual, gate; h, y.  And the gradients of these five
        moved = (2 if step else 1) * (values * (size + 2 * stream) + gate * size + y)
        return {"bytes": moved, "flops": values * (50 if step else 15)}
    tokens, k, experts = case["tokens"], case["k"], case["experts"]
    slots = tokens * k
    if case["op"] == "expert_route":
        # logits; weights, experts, order, slots.  And the gradients of weights and logits
        moved = tokens * experts * size * (2 if step else 1) + slots * (28 + 4 * step) + 8 * (experts + 1)
        return {"bytes": moved, "flops": tokens * experts * (30 if step else 20)}
    inner = case["inner"]
    if case["op"] == "expert_combine":
        # the slots' rows, weights, places; the sums.  And the gradients of all but the places
        moved = (2 if step else 1) * ((slots + tokens) * inner * case["width"] * size + 4 * slots) + 8 * slots
        return {"bytes": moved, "flops": slots * inner * case["width"] * (6 if step else 2)}
    halves = 2 if case["gated"] else 1
    entries = tokens if case["source"] == "tokens" else slots
    matrices = min(experts, slots) * halves * case["n_out"] * case["k_in"]
    moved = (2 if step else 1) * size * (inner * (entries * case["k_in"] + slots * case["n_out"]) + matrices) + 8 * slots
    return {"bytes": moved, "flops": (6 if step else 2) * slots * inner * case["k_in"] * halves * case["n_out"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _generator(seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    return generator


def _plain_dispatch(experts, n_experts):
    """``(offsets, order, slots)`` of the experts chosen, [tokens, k]."""
    flat = experts.reshape(-1)
    keys, order = torch.sort(torch.where(flat < 0, n_experts, flat), stable=True)
    offsets = torch.searchsorted(keys, torch.arange(n_experts + 1, device=flat.device))
    held = keys < n_experts
    places = torch.arange(flat.numel(), device=flat.device)
    slots = torch.empty_like(flat)
    slots[order] = torch.where(held, places, -1)
    return offsets, torch.where(held, order, -1), slots.view(experts.shape)


def _chosen(case, generator):
    """k different experts for each token, some experts more popular than others; -1 for a masked share of the tokens."""
    tokens, experts = case["tokens"], case["experts"]
    popular = torch.randn(experts, generator=generator, device="cuda") * 0.5
    noise = -torch.log(-torch.log(torch.rand(tokens, experts, generator=generator, device="cuda").clamp(1.0e-7, 1.0 - 1.0e-7)))
    chosen = torch.topk(popular + noise, case["k"], dim=1).indices
    off = torch.rand(tokens, generator=generator, device="cuda") < case["masked"]
    return torch.where(off[:, None], -1, chosen)


def prepare(case, seed):
    generator = _generator(seed)
    dtype, step = DTYPES[case["dtype"]], case["step"]
    state = {"case": case}

    def normal(*shape, by=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=generator, device="cuda") * by).to(dtype)

    if case["op"] == "residual_norm":
        shape, width, stream = (case["rows"], case["width"]), case["width"], DTYPES[case["residual"]]
        state["x"], state["residual"] = normal(*shape, by=1.7), normal(*shape, by=3.0, dtype=stream)
        state["post"] = (torch.rand(width, generator=generator, device="cuda") + 0.5) if case["post"] else None
        state["pre"] = (torch.rand(width, generator=generator, device="cuda") + 0.5) if case["pre"] else None
        state["gate"] = {"none": None, "full": normal(*shape), "row": normal(case["rows"], 1)}[case["gate"]]
        state["scale"] = {"none": None, "number": 0.7,
                          "channels": torch.rand(width, generator=generator, device="cuda") * 0.4 + 0.1}[case["scale"]]
        if step:
            state["dh"], state["dy"] = normal(*shape, by=0.3, dtype=stream), normal(*shape, by=0.5)
    elif case["op"] == "expert_route":
        tokens, experts = case["tokens"], case["experts"]
        logits = normal(tokens, experts, by=1.5, dtype=torch.float32) + torch.randn(experts, generator=generator, device="cuda") * 0.5
        if case["masked"]:    # experts that are out for some tokens, and padding, where every expert is
            out = torch.rand(tokens, experts, generator=generator, device="cuda") < case["masked"]
            out |= torch.rand(tokens, 1, generator=generator, device="cuda") < case["masked"]
            logits.masked_fill_(out, -math.inf)
        state["logits"] = logits.to(dtype)
        state["bias"] = torch.randn(experts, generator=generator, device="cuda") * 0.1 if case["bias"] else None
        if step:
            state["dw"] = normal(tokens, case["k"], dtype=torch.float32)
    else:
        offsets, order, slots = _plain_dispatch(_chosen(case, generator), case["experts"])
        entries, inner = case["tokens"] * case["k"], case["inner"]
        state.update(offsets=offsets, order=order, slots=slots)
        if case["op"] == "expert_linear":
            out = case["n_out"]
            rows = case["tokens"] if case["source"] == "tokens" else entries
            state["x"] = normal(rows, inner, case["k_in"])
            state["weight"] = normal(case["experts"], (2 if case["gated"] else 1) * out, case["k_in"], by=case["k_in"] ** -0.5)
            state["bounds"] = offsets.tolist()    # the plain form's loop over the experts runs on the host
            if step:
                state["dy"] = normal(entries, inner, out, by=0.3)
        else:
            state["y"] = normal(entries, inner, case["width"])
            state["weights"] = torch.softmax(normal(case["tokens"], case["k"], dtype=torch.float32), 1)
            if step:
                state["dout"] = normal(case["tokens"], inner, case["width"], by=0.3)
        if own:
            from bysj_amd.kernels import experts

            state["plan"] = experts.ExpertPlan(offsets, order, slots)
    if step:
        state["leaves"] = [state[name] for name in ("x", "residual", "gate", "post", "pre", "scale", "logits", "weight", "y", "weights")
                           if isinstance(state.get(name), torch.Tensor)]
        for leaf in state["leaves"]:
            leaf.requires_grad_(True)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _RUN_OWN[case["op"]](case, state)
    with torch.no_grad():
        return _RUN_PLAIN[case["op"]](case, state)


def _own_norm(case, state):
    from bysj_amd.kernels.block_norm import residual_norm

    h, y = residual_norm(state["x"], state["residual"], post_scale=state["post"], gate=state["gate"],
                         gate_activation=None if case["activation"] == "none" else case["activation"],
                         residual_scale=state["scale"], pre_scale=state["pre"], post_norm=case["post"], pre_norm=case["pre"], eps=EPS)
    outputs = (h, y) if case["pre"] else (h,)
    if not case["step"]:
        return outputs
    grads = torch.autograd.grad(outputs, state["leaves"], (state["dh"], state["dy"])[: len(outputs)])
    return (*(o.detach() for o in outputs), *grads)


def _act(name, gate):
    """The gate and its slope."""
    if name == "none":
        return gate, torch.ones_like(gate)
    s = 1.0 / (1.0 + torch.exp(-gate))
    return (s, s * (1.0 - s)) if name == "sigmoid" else (gate * s, s * (1.0 + gate * (1.0 - s)))


def _plain_norm(case, state):
    x, residual = state["x"].float(), state["residual"].float()
    post, pre, scale = state["post"], state["pre"], state["scale"]
    gate, slope = _act(case["activation"], state["gate"].float()) if state["gate"] is not None else (1.0, None)
    scale = 1.0 if scale is None else scale
    r = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS) if case["post"] else None
    a = x * r * post if case["post"] else x
    h = residual + scale * gate * a
    outputs = [h.to(state["residual"].dtype)]
    if case["pre"]:
        q = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
        outputs.append((h * q * pre).to(state["x"].dtype))
    if not case["step"]:
        return tuple(outputs)
    dh, d_pre = state["dh"].float(), None
    if case["pre"]:
        dy = state["dy"].float()
        d_pre = (dy * h * q).double().sum(0).float()
        u = dy * pre
        dh = dh + q * (u - h * (q * q) * (u * h).mean(1, keepdim=True))
    d_scale = (dh * gate * a).double().sum(0).float()
    d_gate = dh * scale * a
    if slope is not None:
        d_gate = d_gate * slope
    da = dh * scale * gate
    dx, d_post = da, None
    if case["post"]:
        d_post = (da * x * r).double().sum(0).float()
        u = da * post
        dx = r * (u - x * (r * r) * (u * x).mean(1, keepdim=True))
    outputs += [dx.to(state["x"].dtype), dh.to(state["residual"].dtype)]
    if case["gate"] != "none":
        outputs.append((d_gate.sum(1, keepdim=True) if case["gate"] == "row" else d_gate).to(state["gate"].dtype))
    outputs += [d for d, there in ((d_post, case["post"]), (d_pre, case["pre"]), (d_scale, case["scale"] == "channels")) if there]
    return tuple(outputs)


def _own_route(case, state):
    from bysj_amd.kernels.experts import expert_route

    weights, experts, plan = expert_route(state["logits"], case["k"], scores=case["scores"], bias=state["bias"], groups=case["groups"],
                                          top_groups=case["top_groups"], normalize=True, scale=1.5)
    outputs = (weights.detach(), experts, plan.offsets, plan.order, plan.slots)
    return (*outputs, *torch.autograd.grad(weights, state["leaves"], state["dw"])) if case["step"] else outputs


def _plain_route(case, state):
    logits, k, groups = state["logits"], case["k"], case["groups"]
    tokens, n = logits.shape
    there = logits > -math.inf

    def scores(values):
        if case["scores"] == "sigmoid":
            return 1.0 / (1.0 + torch.exp(-values))
        top = values.amax(1, keepdim=True).clamp(min=torch.finfo(values.dtype).min)
        e = torch.exp(values - top)
        return e / e.sum(1, keepdim=True).clamp(min=torch.finfo(values.dtype).tiny)

    # 64 bits for what is compared: two keys next to each other keep their order in any computation of them
    key = logits.double()
    if state["bias"] is not None or groups > 1:
        key = scores(key) + (0.0 if state["bias"] is None else state["bias"].double())
        key = torch.where(there, key, -math.inf)
    if groups > 1:
        split = key.view(tokens, groups, n // groups)
        best = torch.sort(split, dim=2, descending=True).values[:, :, :2]
        value = torch.where(best > -math.inf, best, 0.0).sum(2)
        value = torch.where(best[:, :, 0] > -math.inf, value, -math.inf)
        place = torch.sort(value, dim=1, descending=True, stable=True).indices[:, : case["top_groups"]]
        keep = torch.zeros(tokens, groups, dtype=torch.bool, device=logits.device).scatter_(1, place, True)
        key = torch.where(keep[:, :, None], split, -math.inf).view(tokens, n)
    ranked, place = torch.sort(key, dim=1, descending=True, stable=True)
    chosen = ranked[:, :k] > -math.inf
    place = place[:, :k]
    experts = torch.where(chosen, place, -1)
    s = scores(logits.float())
    picked = torch.where(chosen, s.gather(1, place), 0.0)
    total = picked.sum(1, keepdim=True) + 1.0e-20
    weights = 1.5 * picked / total
    outputs = (weights, experts, *_plain_dispatch(experts, n))
    if not case["step"]:
        return outputs
    dw = torch.where(chosen, state["dw"], 0.0)
    ds = torch.where(chosen, 1.5 / total * (dw - (dw * picked).sum(1, keepdim=True) / total), 0.0)
    if case["scores"] == "sigmoid":
        d = torch.zeros_like(s).scatter_add_(1, place, ds * picked * (1.0 - picked))
    else:
        d = s * (torch.zeros_like(s).scatter_add_(1, place, ds) - (ds * picked).sum(1, keepdim=True))
    return (*outputs, d.to(logits.dtype))


def _own_linear(case, state):
    from bysj_amd.kernels.experts import expert_linear

    y = expert_linear(state["x"], state["weight"], state["plan"], from_tokens=case["source"] == "tokens",
                      activation="silu_gate" if case["gated"] else None)
    return (y.detach(), *torch.autograd.grad(y, state["leaves"], state["dy"])) if case["step"] else y


def _plain_linear(case, state):
    x, weight, bounds, out = state["x"], state["weight"], state["bounds"], case["n_out"]
    y = torch.zeros(state["order"].numel(), *x.shape[1:-1], out, dtype=x.dtype, device=x.device)
    dx, dweight = torch.zeros(x.shape, device=x.device), torch.zeros_like(weight)
    for e in range(case["experts"]):
        a, b = bounds[e], bounds[e + 1]
        if a == b:
            continue
        entries = state["order"][a:b] // case["k"] if case["source"] == "tokens" else torch.arange(a, b, device=x.device)
        rows = x[entries].float().view(-1, case["k_in"])
        matrix = weight[e].float()
        z = rows @ matrix.t()
        if case["gated"]:
            gate, up = z[:, :out], z[:, out:]
            s, slope = _act("silu", gate)
            z = s * up
        y[a:b] = z.view(b - a, *x.shape[1:-1], out).to(y.dtype)
        if case["step"]:
            dz = state["dy"][a:b].float().reshape(-1, out)
            if case["gated"]:
                dz = torch.cat([dz * up * slope, dz * s], 1)
            dx.index_add_(0, entries, (dz @ matrix).view(b - a, *x.shape[1:]))    # a token comes once in each expert
            dweight[e] = (dz.t() @ rows).to(dweight.dtype)
    return (y, dx.to(x.dtype), dweight) if case["step"] else y


def _own_combine(case, state):
    from bysj_amd.kernels.experts import expert_combine

    out = expert_combine(state["y"], state["weights"], state["plan"])
    return (out.detach(), *torch.autograd.grad(out, state["leaves"], state["dout"])) if case["step"] else out


def _plain_combine(case, state):
    y, weights, slots = state["y"], state["weights"], state["slots"]
    held, place = slots >= 0, slots.clamp(min=0)
    w = torch.where(held, weights, 0.0)
    rows = torch.where(held[:, :, None, None], y[place].float(), 0.0)
    out = (w[:, :, None, None] * rows).sum(1).to(y.dtype)
    if not case["step"]:
        return out
    dout = state["dout"].float()
    dweights = (rows * dout[:, None]).sum((2, 3))
    spread = (w[:, :, None, None] * dout[:, None]).to(y.dtype).view(-1, *y.shape[1:])
    # rows of no slot get no gradient
    held_places = state["order"] >= 0
    dy = torch.where(held_places[:, None, None], spread[state["order"].clamp(min=0)], torch.zeros((), dtype=y.dtype, device=y.device))
    return out, dy, dweights


_RUN_OWN = {"residual_norm": _own_norm, "expert_route": _own_route, "expert_linear": _own_linear, "expert_combine": _own_combine}
_RUN_PLAIN = {"residual_norm": _plain_norm, "expert_route": _plain_route, "expert_linear": _plain_linear,
              "expert_combine": _plain_combine}


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        wide = {name: value.detach().double() if isinstance(value, torch.Tensor) and value.is_floating_point() else value
                for name, value in state.items()}
    return {"residual_norm": _exact_norm, "expert_route": _exact_route, "expert_linear": _exact_linear,
            "expert_combine": _exact_combine}[case["op"]](case, wide)


def _differentiated(outputs, leaves, seeds):
    """Outputs and gradients of leaves that take part."""
    return (*(o.detach() for o in outputs), *torch.autograd.grad(outputs, leaves, seeds))


def _exact_norm(case, state):
    leaves = [state[name].requires_grad_(case["step"]) for name in ("x", "residual", "gate", "post", "pre", "scale")
              if isinstance(state[name], torch.Tensor)]
    a = state["x"]
    if case["post"]:
        a = state["post"] * a / torch.linalg.vector_norm(a, dim=1, keepdim=True).square().div(case["width"]).add(EPS).sqrt()
    if state["gate"] is not None:
        gate = state["gate"]
        a = a * {"none": gate, "sigmoid": torch.special.expit(gate), "silu": gate * torch.special.expit(gate)}[case["activation"]]
    h = state["residual"] + a * (1.0 if state["scale"] is None else state["scale"])
    outputs = (h,)
    if case["pre"]:
        outputs = (h, state["pre"] * h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS))
    if not case["step"]:
        return outputs
    return _differentiated(outputs, leaves, (state["dh"], state["dy"])[: len(outputs)])


def _exact_route(case, state):
    logits = state["logits"].requires_grad_(case["step"])
    tokens, n = logits.shape
    k, groups = case["k"], case["groups"]
    out = torch.isneginf(logits)
    if case["scores"] == "softmax":
        s = torch.where(out.all(1, keepdim=True), 0.0, torch.softmax(torch.where(out.all(1, keepdim=True), 0.0, logits), 1))
    else:
        s = torch.special.expit(logits)
    with torch.no_grad():
        key = logits if state["bias"] is None and groups == 1 else s + (0.0 if state["bias"] is None else state["bias"])
        key = key.masked_fill(out, -math.inf).clone()
        if groups > 1:
            members = key.view(tokens, groups, -1)
            first, at = members.max(2)
            second = members.scatter(2, at[:, :, None], -math.inf).amax(2)
            value = first + second.masked_fill(torch.isneginf(second), 0.0)
            allowed = torch.zeros_like(value, dtype=torch.bool)
            for _ in range(case["top_groups"]):    # the best group left, the first of equal ones
                best = value.amax(1, keepdim=True)
                at = (value == best).to(torch.int8).argmax(1, keepdim=True)
                allowed.scatter_(1, at, True)
                value.scatter_(1, at, -math.inf)
            key.masked_fill_(~allowed.repeat_interleave(n // groups, 1), -math.inf)
        picks = []
        for _ in range(k):
            best = key.amax(1, keepdim=True)
            at = (key == best).to(torch.int8).argmax(1, keepdim=True)
            picks.append(torch.where(torch.isneginf(best), -1, at))
            key.scatter_(1, at, -math.inf)
        experts = torch.cat(picks, 1)
    picked = torch.where(experts >= 0, s.gather(1, experts.clamp(min=0)), 0.0)
    weights = 1.5 * picked / (picked.sum(1, keepdim=True) + 1.0e-20)
    flat = experts.reshape(-1)
    order = torch.full_like(flat, -1)
    slots = torch.full_like(flat, -1)
    offsets, at = [0], 0
    for e in range(n):
        mine = torch.nonzero(flat == e).view(-1)
        order[at: at + mine.numel()] = mine
        slots[mine] = torch.arange(at, at + mine.numel(), device=flat.device)
        at += mine.numel()
        offsets.append(at)
    whole = (experts, torch.tensor(offsets, device=flat.device), order, slots.view(tokens, k))
    if not case["step"]:
        return (weights, *whole)
    (grad,) = torch.autograd.grad(weights, logits, state["dw"])
    return (weights.detach(), *whole, torch.nan_to_num(grad))


def _exact_linear(case, state):
    x, weight, k = state["x"], state["weight"], case["k"]
    y = torch.zeros(state["order"].numel(), case["inner"], case["n_out"], dtype=torch.float64, device=x.device)
    dx, dweight = torch.zeros_like(x), torch.zeros_like(weight)
    for e, (a, b) in enumerate(zip(state["bounds"], state["bounds"][1:])):
        if a == b:
            continue
        at = state["order"][a:b].div(k, rounding_mode="floor") if case["source"] == "tokens" else slice(a, b)
        rows, matrix = x[at].detach().requires_grad_(case["step"]), weight[e].detach().requires_grad_(case["step"])
        with torch.set_grad_enabled(case["step"]):
            z = torch.matmul(rows.reshape(-1, case["k_in"]), matrix.transpose(0, 1))
            if case["gated"]:
                gate, up = z.chunk(2, 1)
                z = gate * torch.special.expit(gate) * up
            z = z.view(b - a, case["inner"], case["n_out"])
        y[a:b] = z.detach()
        if case["step"]:
            drows, dweight[e] = torch.autograd.grad(z, (rows, matrix), state["dy"][a:b])
            dx[at] += drows    # a token comes once in each expert
    return (y, dx, dweight) if case["step"] else y


def _exact_combine(case, state):
    y, weights = (state[name].requires_grad_(case["step"]) for name in ("y", "weights"))
    out = torch.zeros(case["tokens"], case["inner"], case["width"], dtype=torch.float64, device=y.device)
    for j in range(case["k"]):
        at = torch.nonzero(state["slots"][:, j] >= 0).view(-1)
        out = out.index_add(0, at, weights[at, j, None, None] * y[state["slots"][at, j]])
    return _differentiated((out,), [y, weights], (state["dout"],)) if case["step"] else out
