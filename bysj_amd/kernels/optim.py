"""The optimiser step over all tensors of a model: gradient norm, AdamW, moments in 32 or in 8 bits.

The operators' backward passes give a model's gradients; these turn them into
a step in a few launches, whatever the number of tensors, without waiting for
the GPU:

    norm, factor = grad_norm(grads, max_norm=1.0)
    plan = adamw_plan(params, state_bits=8)                       # once
    adamw_step(plan, grads, lr=1e-3, grad_factor=factor)

or, as a ``torch.optim.Optimizer``, ``AdamW(params, lr=1e-3, max_norm=1.0)``.
No counterpart in the reference; not part of ``kernels.__all__``.

Moments in 8 bits take 2.06 bytes an element instead of 8.  Blocks of 32
consecutive elements of a tensor share a power of two, and a code is a float
with 3 mantissa bits in the 16 (first moment, with a sign) or 32 (second)
binades below it.  They are rounded stochastically, as bfloat16 parameters are: a
slow average moves by less than half a step at a time, which a nearest
rounding would lose every time.
"""
from __future__ import annotations

import math
import numbers
import operator

import torch

from .native import _extension, require_dcu

DTYPES = (torch.float32, torch.bfloat16)
STATE_BITS = (32, 8)

# A model has hundreds of tensors and a step a few kernels of some microseconds,
# so lists are checked attribute by attribute at the speed of map().
_DTYPE_OF, _SHAPE_OF, _DEVICE_OF = (operator.attrgetter(name) for name in ("dtype", "shape", "device"))


def _all_on(tensors, device) -> bool:
    if device.type == "cuda":  # an index says it all, at half the cost of a device
        return set(map(torch.Tensor.get_device, tensors)) == {device.index}
    return set(map(_DEVICE_OF, tensors)) == {device}


def _tensors(values, what: str, *, allow_none: bool = False) -> list:
    if isinstance(values, torch.Tensor) or not hasattr(values, "__iter__"):
        raise TypeError(f"{what} must be a sequence of tensors")
    values = list(values)
    for kind in set(map(type, values)):
        if not issubclass(kind, torch.Tensor) and not (allow_none and kind is type(None)):
            raise TypeError(f"{what} must be a sequence of tensors")
    return values


def _real(value, what: str, low: float, high: float = math.inf, *, above: bool = False) -> float:
    if isinstance(value, bool) or not isinstance(value, numbers.Real):
        raise TypeError(f"{what} must be a real number")
    value = float(value)
    if not math.isfinite(value) or value < low or value >= high or (above and value == low):
        raise ValueError(f"{what} is out of range: {value}")
    return value


def _scalar_tensor(value, what: str, device=None):
    if value.dtype != torch.float32 or value.numel() != 1:
        raise ValueError(f"{what} must be a float32 tensor of one element")
    if device is not None and value.device != device:
        raise ValueError(f"{what} must be on the parameters' device")
    return value


# ---------------------------------------------------------------------------
# gradient norm
# ---------------------------------------------------------------------------

def grad_norm(grads, max_norm: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(norm, factor)``: the norm over all gradients, and what they are to be multiplied with so that it is at most ``max_norm``.

    ``grads``: contiguous float32 or bfloat16 tensors on one device; None
    entries count as 0.  Both results are float32 tensors without dimensions
    on that device, without a gradient of their own; nothing waits for the GPU.
    The squares are summed in 64 bits in a fixed order.  ``factor`` is ``min(1, max_norm / (norm + 1e-6))``,
    1 without ``max_norm``, and NaN where the norm is not finite:
    ``adamw_step`` then takes no step.
    """
    grads = _tensors(grads, "grad_norm gradients", allow_none=True)
    if type(None) in set(map(type, grads)):
        grads = [g for g in grads if g is not None]
    if not grads:
        raise ValueError("grad_norm needs at least one gradient")
    limit = 0.0 if max_norm is None else _real(max_norm, "grad_norm max_norm", 0.0, above=True)
    dtypes = list(map(_DTYPE_OF, grads))
    if not set(dtypes) <= set(DTYPES):
        raise TypeError("grad_norm requires float32 or bfloat16 gradients")
    if not all(map(torch.Tensor.is_contiguous, grads)):
        raise ValueError("grad_norm gradients must be contiguous")
    if not _all_on(grads, grads[0].device):
        raise ValueError("grad_norm gradients must share a device")
    require_dcu(grads[0])
    return _extension("grad_norm").grad_norm(grads, limit, dtypes)


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------

def _refuse_overlaps(tensors) -> None:
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors if t.numel())
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError("AdamW parameters and moments must not overlap")


def _moments(values, shapes, device, what: str):
    values = _tensors(values, what)
    if len(values) != len(shapes):
        raise ValueError(f"{what}: expected one tensor per parameter")
    if set(map(_DTYPE_OF, values)) != {torch.float32}:
        raise TypeError(f"{what} must be float32")
    if list(map(_SHAPE_OF, values)) != shapes or not all(map(torch.Tensor.is_contiguous, values)) \
            or not _all_on(values, device):
        raise ValueError(f"{what} must be contiguous, of the parameters' shapes and device")
    return values


def adamw_plan(params, exp_avgs=None, exp_avg_sqs=None, *, step=0, state_bits: int = 32):
    """The tensors of ``adamw_step`` with their moments, listed once on the device.

    ``params``: contiguous tensors of one dtype (float32 or bfloat16) and
    device that do not overlap.  ``exp_avgs``, ``exp_avg_sqs``: float32
    tensors of their shapes, both or neither; with ``state_bits`` 32 they are
    the plan's moments, updated in place, with 8 the plan starts from their
    nearest codes.  ``step``: steps taken so far, one number or one per
    tensor.  Building a plan copies its table to the device and waits for it.
    """
    params = _tensors(params, "AdamW parameters")
    if not params:
        raise ValueError("AdamW needs at least one parameter")
    if isinstance(state_bits, bool) or state_bits not in STATE_BITS:
        raise ValueError(f"AdamW state_bits must be 32 or 8, got {state_bits!r}")
    for p in params:
        if p.dtype not in DTYPES:
            raise TypeError("AdamW requires float32 or bfloat16 parameters")
        if p.dtype != params[0].dtype or p.device != params[0].device:
            raise ValueError("the parameters of a plan must share a dtype and a device")
        if not p.is_contiguous():
            raise ValueError("AdamW parameters must be contiguous")
    if (exp_avgs is None) != (exp_avg_sqs is None):
        raise ValueError("AdamW moments: give both or neither")
    if exp_avgs is not None:
        shapes = list(map(_SHAPE_OF, params))
        exp_avgs = _moments(exp_avgs, shapes, params[0].device, "AdamW exp_avgs")
        exp_avg_sqs = _moments(exp_avg_sqs, shapes, params[0].device, "AdamW exp_avg_sqs")
    _refuse_overlaps(params + (exp_avgs or []) + (exp_avg_sqs or []))
    steps = [step] * len(params) if isinstance(step, numbers.Integral) else list(step)
    if len(steps) != len(params):
        raise ValueError("AdamW step: expected one number per parameter")
    for value in steps:
        if isinstance(value, bool) or not isinstance(value, numbers.Integral):
            raise TypeError("AdamW step must be an integer")
        if value < 0:
            raise ValueError("AdamW step must not be negative")
    require_dcu(params[0])
    return _extension("adamw_plan").adamw_plan(params, exp_avgs, exp_avg_sqs, steps, state_bits)


def adamw_step(plan, grads, *, lr, betas=(0.9, 0.999), eps: float = 1.0e-8, weight_decay: float = 1.0e-2,
               grad_factor: torch.Tensor | None = None, seed: int = 0) -> None:
    """One AdamW step over the tensors of ``plan``, in place.

        g = grad * grad_factor
        m = beta1 m + (1 - beta1) g,    v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

    every operation rounded to float32, so that a step equals the eager chain
    bit for bit.  ``grads``: one tensor per parameter (contiguous, of its
    shape; all float32 or all bfloat16) or None where it takes no step.
    ``lr``: a number, or a float32 tensor of one element on the device (read
    when the step runs, also in a captured graph).  ``grad_factor``: such a
    tensor; a NaN leaves parameters, moments and step counts as they are.
    ``seed``: of the stochastic roundings of bfloat16 parameters and 8-bit
    moments, which also depend on the step.  Calls on one plan must not
    overlap in time.
    """
    params = plan.params
    grads = _tensors(grads, "adamw_step gradients", allow_none=True)
    if len(grads) != len(params):
        raise ValueError(f"adamw_step: {len(params)} parameters, {len(grads)} gradients")
    if list(map(torch.Tensor.data_ptr, params)) != plan.addresses:
        raise RuntimeError("adamw_step: a parameter's memory has moved since the plan was built")
    given, shapes = grads, plan.shapes
    if type(None) in set(map(type, grads)):
        given, shapes = [g for g in grads if g is not None], [s for g, s in zip(grads, shapes) if g is not None]
        if not given:
            return
    dtypes = set(map(_DTYPE_OF, given))
    if len(dtypes) != 1 or not dtypes <= set(DTYPES):
        raise TypeError("adamw_step requires gradients of one dtype, float32 or bfloat16")
    if list(map(_SHAPE_OF, given)) != shapes:
        raise ValueError("adamw_step gradients must have their parameters' shapes")
    if not all(map(torch.Tensor.is_contiguous, given)):
        raise ValueError("adamw_step gradients must be contiguous")
    if not _all_on(given, plan.device):
        raise ValueError("adamw_step gradients must be on the parameters' device")
    lr_tensor = None
    if isinstance(lr, torch.Tensor):
        lr_tensor, lr = _scalar_tensor(lr, "adamw_step lr", plan.device), 0.0
    else:
        lr = _real(lr, "adamw_step lr", 0.0)
    if not isinstance(betas, (tuple, list)) or len(betas) != 2:
        raise TypeError("adamw_step betas must be a pair")
    beta1, beta2 = (_real(b, "adamw_step beta", 0.0, 1.0) for b in betas)
    eps = _real(eps, "adamw_step eps", 1.0e-38)
    weight_decay = _real(weight_decay, "adamw_step weight_decay", 0.0)
    if grad_factor is not None:
        if not isinstance(grad_factor, torch.Tensor):
            raise TypeError("adamw_step grad_factor must be a tensor or None")
        _scalar_tensor(grad_factor, "adamw_step grad_factor", plan.device)
    if isinstance(seed, bool) or not isinstance(seed, numbers.Integral):
        raise TypeError("adamw_step seed must be an integer")
    native = _extension("adamw_step")
    native.adamw_step(plan, grads, dtypes.pop(), lr, lr_tensor, beta1, beta2, eps, weight_decay, grad_factor,
                      int(seed))
    # the kernels write behind autograd's back: saved tensors and caches of derived data see it by the counter
    torch.autograd.graph.increment_version(params)


def adamw_states(plan, exp_avgs=None, exp_avg_sqs=None) -> tuple[list, list]:
    """The moments of ``plan`` as float32 tensors of the parameters' shapes: copies, or written into the tensors given.

    Tensors given must not overlap each other.
    """
    out = []
    for values, what in ((exp_avgs, "AdamW exp_avgs"), (exp_avg_sqs, "AdamW exp_avg_sqs")):
        out.append([torch.empty_like(p, dtype=torch.float32) for p in plan.params] if values is None
                   else _moments(values, plan.shapes, plan.device, what))
    if plan.state_bits == 32:
        for to, values in zip(out, (plan.exp_avgs, plan.exp_avg_sqs)):
            torch._foreach_copy_(to, values)
    else:
        _extension("adamw_read_states").adamw_read_states(plan, *out)
        for values in out:
            torch.autograd.graph.increment_version(values)
    return out[0], out[1]


class AdamW(torch.optim.Optimizer):
    """AdamW over all tensors at once, as a ``torch.optim.Optimizer``.

    ``lr`` (a number, or a float32 tensor of one element on the device),
    ``betas``, ``eps`` and ``weight_decay`` may differ between parameter
    groups; ``max_norm`` clips the norm over all gradients of all groups (or,
    where that norm is not finite, takes no step); ``state_bits`` is 32 or 8.
    Parameters are contiguous float32 or bfloat16 tensors on one device.
    After ``step`` the attribute ``norm`` is the gradients' norm before
    clipping, a tensor on the device, or None without ``max_norm``.

    The plans are built in the first step; later steps may be captured in a
    HIP graph (with ``lr`` a tensor where a schedule changes it between
    replays; a graph uses the plans it was captured with, which
    ``load_state_dict`` and parameters that move, come or go replace).  What is
    refused (a step, a group, a checkpoint) changes nothing.  Checkpoints hold each parameter's step count and moments; 8-bit
    moments are kept as their codes.  They come from ``state_dict``, and its
    hooks see them: ``state`` itself stays empty, for the moments live in the
    plans.
    """

    def __init__(self, params, lr=1.0e-3, betas=(0.9, 0.999), eps: float = 1.0e-8, weight_decay: float = 1.0e-2, *,
                 max_norm: float | None = None, state_bits: int = 32, seed: int = 0):
        if isinstance(state_bits, bool) or state_bits not in STATE_BITS:
            raise ValueError(f"AdamW state_bits must be 32 or 8, got {state_bits!r}")
        if isinstance(seed, bool) or not isinstance(seed, numbers.Integral):
            raise TypeError("AdamW seed must be an integer")
        self.max_norm = None if max_norm is None else _real(max_norm, "AdamW max_norm", 0.0, above=True)
        self.state_bits, self.seed, self.norm = state_bits, int(seed), None
        self._plans: dict = {}     # (group, dtype): plan
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, param_group) -> None:
        """As torch's; a group that is refused is not kept."""
        self._refuse_variants([{**self.defaults, **param_group}])
        super().add_param_group(param_group)
        try:
            self._check_group(self.param_groups[-1])
        except BaseException:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_options(group) -> None:
        if not {"lr", "betas", "eps", "weight_decay"} <= group.keys():
            raise ValueError("an AdamW parameter group has lr, betas, eps and weight_decay")
        if isinstance(group["lr"], torch.Tensor):
            _scalar_tensor(group["lr"], "AdamW lr")
        else:
            _real(group["lr"], "AdamW lr", 0.0)
        if not isinstance(group["betas"], (tuple, list)) or len(group["betas"]) != 2:
            raise TypeError("AdamW betas must be a pair")
        for beta in group["betas"]:
            _real(beta, "AdamW beta", 0.0, 1.0)
        _real(group["eps"], "AdamW eps", 1.0e-38)
        _real(group["weight_decay"], "AdamW weight_decay", 0.0)

    @classmethod
    def _check_group(cls, group) -> None:
        cls._check_options(group)
        for p in group["params"]:
            if p.device.type != "cpu":  # on the CPU they may still be on their way
                cls._check_place(group, p.device)
            if p.dtype not in DTYPES:
                raise TypeError("AdamW requires float32 or bfloat16 parameters")
            if not p.is_contiguous():
                raise ValueError("AdamW parameters must be contiguous")

    @staticmethod
    def _check_place(group, device) -> None:
        if isinstance(group["lr"], torch.Tensor) and group["lr"].device != device:
            raise ValueError("AdamW lr must be on the parameters' device")

    @staticmethod
    def _refuse_variants(groups) -> None:
        """Options of torch's optimisers that change the step, as their checkpoints and parameter groups hold them."""
        for group in groups:
            if group.get("amsgrad") or group.get("maximize"):
                raise ValueError("AdamW has neither amsgrad nor maximize")
            if not group.get("decoupled_weight_decay", True) and group["weight_decay"] != 0:
                raise ValueError("AdamW's weight decay is decoupled from the gradient")

    def _current(self) -> list:
        """``[(group index, dtype), parameters]`` as they are now: every parameter, or a refusal."""
        current = []
        for index, group in enumerate(self.param_groups):
            params = group["params"]
            kinds = set(map(_DTYPE_OF, params))
            if not kinds <= set(DTYPES):
                raise TypeError("AdamW requires float32 or bfloat16 parameters")
            current += [((index, dtype), params if kinds == {dtype} else [p for p in params if p.dtype == dtype])
                        for dtype in DTYPES]
        return current

    def _follow(self, current) -> None:
        """Rebuilds the plans if a parameter has moved, come or gone, or changed its dtype since they were built."""
        now = dict(current)
        for key, plan in self._plans.items():
            params = now.get(key, ())
            if not (len(plan.params) == len(params) and all(map(operator.is_, plan.params, params))
                    and list(map(torch.Tensor.data_ptr, params)) == plan.addresses):
                plans = self._plans.values()
                shapes = {p: shape for plan in plans for p, shape in zip(plan.params, plan.shapes)}
                if any([p.shape != shapes.get(p, p.shape) for _, params in current for p in params]):
                    raise ValueError("a parameter has another shape than its moments")
                self._plans = self._rebuilt({p: part for plan in plans for p, part in self._held(plan).items()})
                return

    def _rebuilt(self, held) -> dict:
        """New plans that go on from ``held``; the old ones stay until the caller replaces them."""
        return {key: self._build(params, held) for key, params in self._current() if any([p in held for p in params])}

    def _build(self, params, held):
        """A plan of ``params`` that goes on from ``held``: {parameter: its part of a checkpoint}."""
        known = {k: held[p] for k, p in enumerate(params) if p in held}
        steps = [int(known[k]["step"]) if k in known else 0 for k in range(len(params))]
        if self.state_bits == 32:
            moments = [[known[k][name].to(device=p.device, dtype=torch.float32).contiguous().clone()
                        if k in known else torch.zeros_like(p, dtype=torch.float32).detach()
                        for k, p in enumerate(params)] for name in ("exp_avg", "exp_avg_sq")]
            return adamw_plan(params, *moments, step=steps)
        plan = adamw_plan(params, step=steps, state_bits=8)
        for k, (codes, scales) in enumerate(plan.parts()):
            if k in known:
                codes.copy_(known[k]["codes"])
                scales.copy_(known[k]["scales"])
        return plan

    @staticmethod
    def _held(plan) -> dict:
        steps = plan.steps().tolist()
        if plan.state_bits == 32:
            return {p: {"step": t, "exp_avg": m, "exp_avg_sq": v}
                    for p, t, m, v in zip(plan.params, steps, plan.exp_avgs, plan.exp_avg_sqs)}
        return {p: {"step": t, "codes": codes, "scales": scales}
                for p, t, (codes, scales) in zip(plan.params, steps, plan.parts())}

    @torch.no_grad()
    def step(self, closure=None):
        """One step over the parameters that have a gradient; returns the closure's loss."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        current, work = self._current(), []
        self._follow(current)
        for key, params in current:
            grads = [p.grad for p in params]
            given = [g for g in grads if g is not None]
            if not all(map(torch.Tensor.is_contiguous, given)):
                grads = [None if g is None else g.contiguous() for g in grads]
            if given:
                plan = self._plans.get(key)
                if plan is None:
                    plan = self._plans[key] = self._build(params, {})
                index, dtype = key
                group = self.param_groups[index]
                self._check_options(group)  # all of them before the first group's step
                self._check_place(group, plan.device)
                work.append((group, plan, grads, index * 2 + (dtype == torch.bfloat16)))
        self.norm = factor = None
        if self.max_norm is not None and work:
            self.norm, factor = grad_norm([g for _, _, grads, _ in work for g in grads if g is not None], self.max_norm)
        for group, plan, grads, stream in work:
            adamw_step(plan, grads, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                       weight_decay=group["weight_decay"], grad_factor=factor, seed=self.seed + stream * 0x9E3779B97F4A7C15)
        return loss

    def __getstate__(self):
        raise TypeError("the moments live in plans on the device: save state_dict() instead")

    def state_dict(self) -> dict:
        """Groups, and each parameter's step count and moments; hooks see all of it."""
        def fill(_, result):
            numbers_of = {p: k for k, p in enumerate(p for group in self.param_groups for p in group["params"])}
            result["state"] = {numbers_of[p]: {name: value.clone() if isinstance(value, torch.Tensor) else value
                                               for name, value in part.items()}
                               for plan in self._plans.values() for p, part in self._held(plan).items() if p in numbers_of}
            result["state_bits"] = self.state_bits

        hook = self.register_state_dict_post_hook(fill, prepend=True)
        try:
            return super().state_dict()
        finally:
            hook.remove()

    def _check_part(self, p, part) -> None:
        """One parameter's part of a checkpoint."""
        if self.state_bits == 32:
            wanted = {"exp_avg": p.shape, "exp_avg_sq": p.shape}
        else:
            spans = -(-p.numel() // 32)
            wanted = {"codes": (2, spans * 32), "scales": (2, spans)}
        if not isinstance(part, dict) or not {"step", *wanted} <= part.keys():
            raise ValueError(f"the checkpoint's moments must have step, {' and '.join(wanted)}")
        if float(part["step"]) != int(part["step"]) or part["step"] < 0:
            raise ValueError(f"the checkpoint has a bad step count: {part['step']!r}")
        for name, shape in wanted.items():
            value = part[name]
            if not isinstance(value, torch.Tensor) or value.shape != shape:
                raise ValueError(f"the checkpoint's {name} must be a tensor of shape {tuple(shape)}")
            if value.dtype != torch.uint8 if self.state_bits == 8 else not value.is_floating_point():
                raise TypeError(f"the checkpoint's {name} has the wrong type: {value.dtype}")

    def _plans_of(self, state_dict) -> dict:
        """The plans of a checkpoint, all of which is checked."""
        bits = state_dict.get("state_bits", 32)  # torch's own AdamW does not say
        if bits != self.state_bits:
            raise ValueError(f"the checkpoint holds {bits}-bit moments, not {self.state_bits}-bit ones")
        groups = state_dict["param_groups"]
        if [len(group["params"]) for group in groups] != [len(group["params"]) for group in self.param_groups]:
            raise ValueError("the checkpoint's parameter groups are of other sizes")
        for group in groups:
            self._check_options(group)
        self._refuse_variants(groups)
        saved = (k for group in groups for k in group["params"])
        params = dict(zip(saved, (p for group in self.param_groups for p in group["params"])))
        held = {}
        for k, part in state_dict["state"].items():
            if int(k) not in params:
                raise ValueError(f"the checkpoint has moments of a parameter {k!r} that is in no group")
            self._check_part(params[int(k)], part)
            held[params[int(k)]] = part
        return self._rebuilt(held)

    def load_state_dict(self, state_dict) -> None:
        """Takes a checkpoint over; one that is refused leaves the optimiser as it was."""
        plans = {}

        def build(_, given):  # behind the hooks that may change the checkpoint, before anything is replaced
            plans.update(self._plans_of(given))
            groups = [{**saved, "lr": saved["lr"].to(group["params"][0].device)}
                      if isinstance(saved["lr"], torch.Tensor) and group["params"] else saved
                      for saved, group in zip(given["param_groups"], self.param_groups)]
            return {**given, "state": {}, "param_groups": groups}

        def replace(_):  # before the hooks that look at the result
            self._plans = plans

        hooks = [self.register_load_state_dict_pre_hook(build), self.register_load_state_dict_post_hook(replace, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()


__all__ = ["AdamW", "grad_norm", "adamw_plan", "adamw_step", "adamw_states", "DTYPES", "STATE_BITS"]
