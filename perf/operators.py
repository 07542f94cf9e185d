"""The operators around the training of a DPA4/SeZM model, as measurable cases.

``group_norm``  ``kernels.group_norm.group_norm``: normalisation over the rows of a frame (or of a node's edges) and a
                group of channels, with scale, bias and an optional SiLU; alone (inference) or with the gradients of
                its input, scale and bias (``"step": True``).
``adamw``       ``kernels.optim.adamw_step``: one step over all tensors of a model, moments in 32 or in 8 bits.
``grad_norm``   ``kernels.optim.grad_norm``: the norm over all gradients and the factor that clips it.

With ``own`` false ``run`` computes the same from elementary torch operations.

The 8-bit moments: blocks of 32 consecutive elements of a tensor share a power of two, 2^(X - 127), the binade of the
largest magnitude after it is rounded up to three mantissa bits.  A code is a float with three mantissa bits in the
binades down from there, without subnormals: a sign and 16 binades for the first moment, 32 for the second.  Roundings to
fewer bits are stochastic with 16 random bits a value; the bits come from an integer mix of the seed, the step and the
element's position, where every tensor starts at a multiple of 32.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BETAS, EPS, DECAY, LR, MAX_NORM = (0.9, 0.999), 1.0e-8, 1.0e-2, 1.0e-3, 1.0
LARGEST_BYTES = 5.0e9    # no drawn case moves more than the largest listed one
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # The smallest call: the pooled feature rows of 64 frames, one row each, in front of a fitting net at inference.
        {"name": "norm_one_row", "op": "group_norm", "samples": 64, "rows": 64, "inner": 1, "channels": 64, "groups": 8,
         "lengths": "dense", "dtype": "float32", "silu": True, "step": False},
        # Node features [N, 16, 64] (lmax 3) of a batch of 32 frames of about 192 atoms at inference.
        {"name": "norm_frames", "op": "group_norm", "samples": 32, "rows": 6144, "inner": 16, "channels": 64,
         "groups": 8, "lengths": "even", "dtype": "float32", "silu": True, "step": False},
        # Edge features per destination node, 3,000 atoms with about 60 neighbours, in training.
        {"name": "norm_edges_step", "op": "group_norm", "samples": 3000, "rows": 181838, "inner": 1, "channels": 64,
         "groups": 4, "lengths": "even", "dtype": "float32", "silu": True, "step": True},
        # One large box, 24,576 atoms of 16 rows of 64 channels: a single sample, in training.
        {"name": "norm_box_step", "op": "group_norm", "samples": 1, "rows": 24576, "inner": 16, "channels": 64,
         "groups": 16, "lengths": "dense", "dtype": "float32", "silu": False, "step": True},
        # Eight boxes of very different sizes, 65,536 atoms together, 128 channels in bfloat16, at inference.
        {"name": "norm_boxes_bf16", "op": "group_norm", "samples": 8, "rows": 65536, "inner": 16, "channels": 128,
         "groups": 8, "lengths": "wild", "dtype": "bfloat16", "silu": True, "step": False},
        # Odd sizes: 90 channels in 6 groups, frames of any length (some empty), float16, in training.
        {"name": "norm_odd_step", "op": "group_norm", "samples": 257, "rows": 30011, "inner": 9, "channels": 90,
         "groups": 6, "lengths": "wild", "dtype": "float16", "silu": True, "step": True},
        # A model of 300 tensors, matrices of 64 to 256 rows among biases and scalars: what a step of it costs.
        {"name": "adamw_model", "op": "adamw", "tensors": 300, "width": 64, "dtype": "float32", "grad": "float32",
         "bits": 32, "factor": True},
        # The largest: a model of 72 million parameters, float32 with gradients in float32.
        {"name": "adamw_large", "op": "adamw", "tensors": 64, "width": 1009, "dtype": "float32", "grad": "float32",
         "bits": 32, "factor": True},
        # The 300 tensors with 8-bit moments.
        {"name": "adamw8_model", "op": "adamw", "tensors": 300, "width": 64, "dtype": "float32", "grad": "float32",
         "bits": 8, "factor": True},
        # The large model held in bfloat16 with 8-bit moments.
        {"name": "adamw8_large", "op": "adamw", "tensors": 64, "width": 1009, "dtype": "bfloat16", "grad": "bfloat16",
         "bits": 8, "factor": False},
        # Norm of the 300 tensors' gradients.
        {"name": "norm_of_model", "op": "grad_norm", "tensors": 300, "width": 64, "grad": "float32"},
        # Norm of the large model's gradients, in bfloat16.
        {"name": "norm_of_large", "op": "grad_norm", "tensors": 64, "width": 1009, "grad": "bfloat16"},
    ]


def _log(rng, low, high):
    """An integer spread over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw(rng):
    op = rng.choice(["group_norm", "group_norm", "group_norm", "adamw", "adamw", "grad_norm"])
    if op == "group_norm":
        groups = rng.choice([1, 2, 4, 6, 8, 16, 32])
        channels = groups * _log(rng, 2, 512 // groups)
        lengths = rng.choice(["dense", "even", "wild"])
        samples = _log(rng, 1, 4096)
        rows = samples * _log(rng, 1, max(1, 200000 // samples)) if lengths == "dense" else max(samples, _log(rng, 64, 200000))
        return {"op": op, "samples": samples, "rows": rows, "inner": rng.choice([1, 1, 4, 9, 16]), "channels": channels,
                "groups": groups, "lengths": lengths, "dtype": rng.choice(["float32", "float32", "bfloat16", "float16"]),
                "silu": rng.random() < 0.7, "step": rng.random() < 0.5}
    case = {"op": op, "tensors": _log(rng, 1, 400), "width": _log(rng, 8, 1009)}
    if op == "grad_norm":
        return {**case, "grad": rng.choice(["float32", "float32", "bfloat16"])}
    return {**case, "dtype": rng.choice(["float32", "float32", "bfloat16"]),
            "grad": rng.choice(["float32", "float32", "bfloat16"]), "bits": rng.choice([32, 8]),
            "factor": rng.random() < 0.5}


def draw(rng):
    while True:
        case = _draw(rng)
        if work(case)["bytes"] <= LARGEST_BYTES:
            return case


def _shapes(case):
    """The parameter shapes of a model: matrices, stacks of them, biases, norm scales and scalars, by turns."""
    w = case["width"]
    kinds = [(w, w), (w,), (4 * w, w), (1,), (w, 2 * w), (2 * w + 1,), (16, w), (3, w, w), (w + 1,)]
    return [kinds[i % len(kinds)] for i in range(case["tensors"])]


def _padded(shapes):
    """Where each tensor starts, at multiples of 32, and the end."""
    starts, at = [], 0
    for shape in shapes:
        starts.append(at)
        at += -(-math.prod(shape) // 32) * 32
    return starts, at


def work(case):
    """Each input read once, each output written once."""
    if case["op"] == "group_norm":
        size = 4 if case["dtype"] == "float32" else 2
        values = case["rows"] * case["inner"] * case["channels"]
        streams = 4 if case["step"] else 2    # x, y; and the gradients of both
        more = 8 * (case["samples"] + 1) * (case["lengths"] != "dense") + 4 * case["channels"] * (4 if case["step"] else 2)
        return {"bytes": values * size * streams + more, "flops": values * (40 if case["step"] else 12)}
    values = sum(math.prod(s) for s in _shapes(case))
    size = 2 if case["grad"] == "bfloat16" else 4
    if case["op"] == "grad_norm":
        return {"bytes": values * size + 8, "flops": 2 * values}
    each = 2 * (2 if case["dtype"] == "bfloat16" else 4) + size
    # 8 bits: codes and exponents in and out, and the moments' values out
    each += 16 if case["bits"] == 32 else 2 * (2 + 2 / 32) + 8
    return {"bytes": values * each, "flops": 15 * values}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _generator(seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    return generator


def _offsets(case, seed):
    """Rows of the samples: about even, or cut anywhere (lengths from none to several times the mean)."""
    r, rows, samples = random.Random(seed), case["rows"], case["samples"]
    if case["lengths"] == "even":
        cuts = [round((i + r.uniform(-0.3, 0.3)) * rows / samples) for i in range(1, samples)]
    else:
        cuts = [r.randrange(rows + 1) for _ in range(samples - 1)]
    return [0] + sorted(min(max(c, 0), rows) for c in cuts) + [rows]


def _views(flat, shapes):
    starts, _ = _padded(shapes)
    return [flat[a: a + math.prod(s)].view(s) for a, s in zip(starts, shapes)]


def _inside(shapes):
    """1 where the padded concatenation holds an element, 0 where it holds padding."""
    _, total = _padded(shapes)
    mask = torch.zeros(total, device="cuda")
    for view in _views(mask, shapes):
        view.fill_(1.0)
    return mask


def prepare(case, seed):
    generator = _generator(seed)
    if case["op"] == "group_norm":
        dtype, channels = DTYPES[case["dtype"]], case["channels"]
        shape = (case["rows"], case["inner"], channels)
        state = {"case": case, "offsets": None, "most": None}
        if case["lengths"] == "dense":
            shape = (case["samples"], case["rows"] // case["samples"] * case["inner"], channels)
        else:
            offsets = _offsets(case, seed)
            state["offsets"] = torch.tensor(offsets, device="cuda")
            state["most"] = max(b - a for a, b in zip(offsets, offsets[1:]))    # a program knows its largest frame
        # features after a linear layer: channels of different spread, some far from zero
        spread = torch.rand(channels, generator=generator, device="cuda") * 2.0 + 0.2
        centre = torch.randn(channels, generator=generator, device="cuda")
        state["x"] = (torch.randn(shape, generator=generator, device="cuda") * spread + centre).to(dtype)
        state["scale"] = torch.rand(channels, generator=generator, device="cuda") + 0.5
        state["bias"] = torch.randn(channels, generator=generator, device="cuda") * 0.1
        if case["step"]:
            state["dy"] = (torch.randn(shape, generator=generator, device="cuda") * 0.3).to(dtype)
            for name in ("x", "scale", "bias"):
                state[name].requires_grad_(True)
        return state
    shapes = _shapes(case)
    _, total = _padded(shapes)
    # gradients of a model in training: each tensor's of its own size
    size = torch.exp(torch.randn(len(shapes), generator=generator, device="cuda") * 1.5 - 6.0)
    grad = torch.randn(total, generator=generator, device="cuda")
    for k, view in enumerate(_views(grad, shapes)):
        view.mul_(size[k])
    state = {"case": case, "grad_flat": grad.to(DTYPES[case["grad"]]), "shapes": shapes}
    state["grads"] = _views(state["grad_flat"], shapes)
    if case["op"] == "grad_norm":
        return state
    inside = _inside(shapes)
    state["param_flat"] = (torch.randn(total, generator=generator, device="cuda") * 0.05 * inside).to(DTYPES[case["dtype"]])
    # moments after a thousand steps: the first a mean of noise, the second near the gradients' mean square
    first = torch.randn(total, generator=generator, device="cuda") * 0.23 * inside
    second = (torch.rand(total, generator=generator, device="cuda") * 0.6 + 0.7) * inside
    for k, (m, v) in enumerate(zip(_views(first, shapes), _views(second, shapes))):
        m.mul_(size[k])
        v.mul_(size[k] * size[k])
    if case["bits"] == 8:
        half = torch.full((total,), 0x8000, dtype=torch.int64, device="cuda")
        first, second = _coded(first, half, True), _coded(second, half, False)
    state.update(first_flat=first, second_flat=second, step=1000, seed=seed)
    state["factor"] = torch.full((), 0.37, device="cuda") if case["factor"] else None
    state["params"] = _views(state["param_flat"], shapes)
    state["first"], state["second"] = _views(first, shapes), _views(second, shapes)
    if own:
        from bysj_amd.kernels import optim

        state["plan"] = optim.adamw_plan(state["params"], state["first"], state["second"], step=1000, state_bits=case["bits"])
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return {"group_norm": _run_group_norm, "adamw": _run_adamw, "grad_norm": _run_grad_norm}[state["case"]["op"]](state)


def _run_group_norm(state):
    case, x, scale, bias = state["case"], state["x"], state["scale"], state["bias"]
    if own:
        from bysj_amd.kernels.group_norm import group_norm

        y = group_norm(x, case["groups"], scale, bias, offsets=state["offsets"], max_rows=state["most"], eps=1.0e-5,
                       activation="silu" if case["silu"] else None)
        if not case["step"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (x, scale, bias), state["dy"]))
    with torch.no_grad():
        return _plain_group_norm(case, x, scale, bias, state["offsets"], state.get("dy"))


def _plain_group_norm(case, x, scale, bias, offsets, dy):
    entries, inner, channels, groups = x.shape[0], x.shape[1], x.shape[2], case["groups"]
    grouped = (entries, inner, groups, channels // groups)
    if offsets is None:
        offsets = torch.arange(entries + 1, device=x.device)
    lengths = offsets[1:] - offsets[:-1]
    sample = torch.repeat_interleave(torch.arange(lengths.numel(), device=x.device), lengths, output_size=entries)
    count = (lengths * inner * (channels // groups)).clamp(min=1).double()[:, None]

    def mean(values):    # over a sample's rows and a group's channels, the long sums in 64 bits, one value per entry
        sums = torch.cat([torch.zeros(groups, 1, dtype=torch.float64, device=x.device),
                          values.double().sum((1, 3)).t().contiguous().cumsum(1)], 1)
        return ((sums[:, offsets[1:]] - sums[:, offsets[:-1]]).t() / count)[sample][:, None, :, None].float()

    x32 = x.float().view(grouped)
    weight, shift = scale.view(groups, -1), bias.view(groups, -1)
    centred = x32 - mean(x32)
    inverse = 1.0 / torch.sqrt(mean(centred * centred) + 1.0e-5)
    hat = centred * inverse
    z = hat * weight + shift
    gate = torch.sigmoid(z) if case["silu"] else None
    y = (z * gate if case["silu"] else z).to(x.dtype).view(x.shape)
    if dy is None:
        return y
    dz = dy.float().view(grouped)
    if case["silu"]:
        dz = dz * (gate * (1.0 + z * (1.0 - gate)))
    d_bias = dz.double().sum((0, 1)).float().view(-1)
    d_scale = (dz * hat).double().sum((0, 1)).float().view(-1)
    u = dz * weight
    dx = inverse * (u - mean(u) - hat * mean(u * hat))
    return y, dx.to(x.dtype).view(x.shape), d_scale, d_bias


def _run_adamw(state):
    case = state["case"]
    if own:
        from bysj_amd.kernels import optim

        optim.adamw_step(state["plan"], state["grads"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
                         grad_factor=state["factor"], seed=state["seed"])
        if case["bits"] == 8:
            optim.adamw_states(state["plan"], state["first"], state["second"])
    else:
        _plain_adamw(state, case)
    return state["param_flat"], state["first_flat"], state["second_flat"]


def _joined(tensors, shapes, flat):
    """The tensors of a list one after the other, each padded to a multiple of 32, in 32 bits."""
    zeros = torch.zeros(32, dtype=flat.dtype, device=flat.device)
    return torch.cat([piece for t, s in zip(tensors, shapes) for piece in (t.reshape(-1), zeros[: -math.prod(s) % 32])]).float()


def _plain_adamw(state, case):
    state["step"] += 1
    t, (beta1, beta2) = state["step"], BETAS
    p, g = _joined(state["params"], state["shapes"], state["param_flat"]), _joined(state["grads"], state["shapes"], state["grad_flat"])
    if state["factor"] is not None:
        g = g * state["factor"]
    m = state["first_flat"] * beta1 + g * (1.0 - beta1)
    v = state["second_flat"] * beta2 + (g * g) * (1.0 - beta2)
    denominator = v.sqrt() * (1.0 / math.sqrt(1.0 - beta2 ** t)) + EPS
    p = p * (1.0 - LR * DECAY) - (m / denominator) * (LR / (1.0 - beta1 ** t))
    if case["bits"] == 8 or case["dtype"] == "bfloat16":
        bits = _random_bits(state["seed"], t, p.numel())
    if case["bits"] == 8:
        m, v = _coded(m, bits & 0xFFFF, True), _coded(v, bits >> 16, False)
    if case["dtype"] == "bfloat16":
        word = p.view(torch.int32) + (_mix(bits + 0x9E3779B1) & 0xFFFF).int()
        p = (word & -65536).view(torch.float32).bfloat16()
    state["first_flat"].copy_(m)
    state["second_flat"].copy_(v)
    starts, _ = _padded(state["shapes"])
    torch._foreach_copy_(state["params"], [p[a: a + math.prod(s)].view(s) for a, s in zip(starts, state["shapes"])])


def _mix(x):
    """An integer mix of 32 bits (in int64)."""
    x = x & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x6A09E667) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _mix_one(x):
    return int(_mix(torch.tensor(x, dtype=torch.int64)))


def _random_bits(seed, t, count):
    """32 bits for each position: mix(position ^ key), the key a mix of seed, step and the position's upper half (here 0)."""
    key = _mix_one((seed & 0xFFFFFFFF) ^ _mix_one((seed >> 32) + _mix_one(t)))
    return _mix(torch.arange(count, device="cuda") ^ key)


def _coded(x, random16, signed):
    """The values that the 8-bit codes of `x` stand for."""
    word = x.abs().view(torch.int32).long()
    binades = 16 if signed else 32
    top = ((word + 0xFFFFF) >> 23).view(-1, 32).amax(1).clamp(min=binades)
    low = ((top - (binades - 1)) << 3).repeat_interleave(32)
    code = ((word + (random16 << 4)) >> 20) - low
    if signed:    # below the least code: up to it as often as the value's share of it
        least = ((low + 1) << 20).int().view(torch.float32)
        under = (x.abs() > least * (random16.float() * 2.0 ** -16)).long()
    else:         # a second moment that is not 0 never becomes 0
        under = (word > 0).long()
    code = torch.where(code < 1, under, code)
    value = torch.where(code > 0, ((code + low) << 20).int().view(torch.float32), torch.zeros_like(x))
    return torch.copysign(value, x) if signed else value


def _run_grad_norm(state):
    if own:
        from bysj_amd.kernels import optim

        return optim.grad_norm(state["grads"], MAX_NORM)
    flat = torch.cat([g.reshape(-1) for g in state["grads"]])
    norm = flat.double().square().sum().sqrt()
    return norm.float(), (MAX_NORM / (norm + 1.0e-6)).clamp(max=1.0).float()


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"group_norm": _exact_group_norm, "adamw": _exact_adamw, "grad_norm": _exact_grad_norm}[case["op"]](case, state)


def _exact_group_norm(case, state):
    x, groups = state["x"].detach().double(), case["groups"]
    weight, shift = state["scale"].detach().double(), state["bias"].detach().double()
    bounds = list(range(x.shape[0] + 1)) if state["offsets"] is None else state["offsets"].tolist()
    y = torch.zeros_like(x)
    dx, d_scale, d_bias = torch.zeros_like(x), torch.zeros_like(weight), torch.zeros_like(shift)
    for a, b in zip(bounds, bounds[1:]):
        if a == b:
            continue
        rows = x[a:b].reshape(-1, groups, case["channels"] // groups)
        variance, centre = torch.var_mean(rows, dim=(0, 2), correction=0, keepdim=True)
        root = torch.sqrt(variance + 1.0e-5)
        hat = ((rows - centre) / root).reshape(-1, case["channels"])
        z = hat * weight + shift
        slope = 1.0
        if case["silu"]:
            s = 1.0 / (1.0 + torch.exp(-z))
            y[a:b] = (z * s).view(x[a:b].shape)
            slope = s + z * s * (1.0 - s)
        else:
            y[a:b] = z.view(x[a:b].shape)
        if case["step"]:
            dz = state["dy"][a:b].double().reshape(-1, case["channels"]) * slope
            d_bias += dz.sum(0)
            d_scale += (dz * hat).sum(0)
            u, h = ((dz * weight).view(rows.shape), hat.view(rows.shape))
            inner = (u * h).mean((0, 2), keepdim=True)
            dx[a:b] = ((u - u.mean((0, 2), keepdim=True) - h * inner) / root).view(x[a:b].shape)
    return (y, dx, d_scale, d_bias) if case["step"] else y


def _exact_adamw(case, state):
    t, (beta1, beta2), total = 1001, BETAS, state["param_flat"].numel()
    p, g = state["param_flat"].double(), state["grad_flat"].double()
    g = g * _inside(state["shapes"])    # nothing happens in the padding
    if state["factor"] is not None:
        g = g * state["factor"].double()
    m = beta1 * state["first_flat"].double() + (1.0 - beta1) * g
    v = beta2 * state["second_flat"].double() + (1.0 - beta2) * g * g
    p = p - LR * DECAY * p - LR * (m / (1.0 - beta1 ** t)) / (torch.sqrt(v / (1.0 - beta2 ** t)) + EPS)
    if case["dtype"] == "bfloat16":
        # the step's own rounding: up where the fraction of a bfloat16 step and the random bits pass one
        noise = (_mix(_random_bits(seed=state["seed"], t=t, count=total) + 0x9E3779B1) & 0xFFFF).double() / 65536.0
        _, exponent = torch.frexp(p)
        unit = torch.ldexp(torch.ones_like(p), exponent - 8)
        p = torch.sign(p) * torch.floor(p.abs() / unit + noise) * unit
    if case["bits"] == 8:
        return p, None, None    # a moment next to a border of two codes has no value apart from the 32-bit sums
    return p, m, v


def _exact_grad_norm(case, state):
    total = sum(float(g.double().square().sum()) for g in state["grads"])
    norm = math.sqrt(total)
    return norm, min(1.0, MAX_NORM / (norm + 1.0e-6))
