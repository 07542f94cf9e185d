"""Layers of experts: routing, dispatch, the experts' products and their weighted sum.

Where nodes of different kinds (elements, environments) share a layer, each
token chooses k of E matrices instead of one:

    weights, experts, plan = expert_route(logits, k)          # [tokens, E] -> the k best of each token
    z = expert_linear(x, w_in, plan, activation="silu_gate")  # by token -> by place, expert after expert
    z = expert_linear(z, w_out, plan, from_tokens=False)      # by place
    out = expert_combine(z, weights, plan)                    # back, summed over a token's k slots

The reference has no such layer; the plan is the CSR its segment operators take
(python/kernels/segment.py:46-71): slot ``t * k + j`` is token t's j-th choice,
expert e owns the places ``offsets[e]`` to ``offsets[e + 1]``, place p holds slot
``order[p]``, and ``slots[t, j]`` is the place of a slot, -1 for one without an
expert.  Nothing here waits for the GPU.  Not part of ``kernels.__all__``.

Entries may have rows: ``[N, 16, C]`` goes through one matrix of its expert as
16 rows of C channels.  Routed by the l = 0 row alone, that keeps rotational
equivariance; the gated SiLU acts on components and does not, so it is one for
invariant rows.
"""
from __future__ import annotations

import math
import numbers
from typing import NamedTuple

import torch

from .native import apply_function, _extension, require_dcu

SCORES = ("softmax", "sigmoid")
ACTIVATIONS = (None, "silu_gate")
DTYPES = (torch.float32, torch.bfloat16, torch.float16)
MAX_EXPERTS = 1024
MAX_GROUPS = 64
MAX_CHANNELS = 65536   # of a product, whose sum over them is held in float32
_MOST = 2**31 - 1


class ExpertPlan(NamedTuple):
    """The CSR of the slots by expert: int64 ``offsets`` (E + 1,), ``order`` (tokens * k,), ``slots`` (tokens, k)."""

    offsets: torch.Tensor
    order: torch.Tensor
    slots: torch.Tensor


def _integer(value, what: str) -> int:
    if isinstance(value, bool) or not isinstance(value, numbers.Integral):
        raise TypeError(f"{what} must be an integer")
    return int(value)


def _floats(tensor, what: str) -> None:
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{what} must be a tensor")
    if tensor.dtype not in DTYPES:
        raise TypeError(f"{what} must be float32, bfloat16 or float16")
    if not tensor.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


def _check_plan(plan) -> tuple[int, int]:
    """(tokens, k) of a plan."""
    if not isinstance(plan, ExpertPlan):
        raise TypeError("the expert plan must be an ExpertPlan")
    for name, tensor, ndim in (("offsets", plan.offsets, 1), ("order", plan.order, 1), ("slots", plan.slots, 2)):
        if not isinstance(tensor, torch.Tensor):
            raise TypeError(f"expert plan {name} must be a tensor")
        if tensor.dtype != torch.int64:
            raise TypeError(f"expert plan {name} must be int64")
        if tensor.ndim != ndim or not tensor.is_contiguous():
            raise ValueError(f"expert plan {name} must be contiguous and {ndim}-dimensional")
    tokens, k = plan.slots.shape
    if k < 1 or plan.order.numel() != tokens * k:
        raise ValueError("expert plan order must have one entry for each of the slots (tokens, k)")
    if not 2 <= plan.offsets.numel() <= MAX_EXPERTS + 1:
        raise ValueError(f"expert plan offsets must be those of 1 to {MAX_EXPERTS} experts")
    return tokens, k


def _same_device(first, *others) -> None:
    for other in others:
        if other is not None and other.device != first.device:
            raise ValueError("the tensors of an expert operator must share a device")


# ---------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------

class _RouteFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, options):
        keep = ctx.needs_input_grad[0]
        native = _extension("expert_route_forward")
        weights, experts, statistics = native.expert_route_forward(logits, bias, options, keep and options[3] == 0)
        if keep:
            ctx.save_for_backward(logits, experts, statistics)
            ctx.mark_non_differentiable(experts)
            ctx.options = options
        return weights, experts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_weights, _):
        logits, experts, statistics = ctx.saved_tensors
        native = _extension("expert_route_backward")
        return native.expert_route_backward(grad_weights.contiguous(), logits, experts, statistics, ctx.options), None, None


def expert_route(logits: torch.Tensor, k: int, *, scores: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
                 top_groups: int | None = None, normalize: bool = True, scale: float = 1.0):
    """``(weights, experts, plan)``: the ``k`` best experts of each token, their weights, and the slots by expert.

    ``logits``: contiguous ``(tokens, E)`` in float32, bfloat16 or float16, at
    most 1,024 experts.  Scores are a softmax or a sigmoid of them; experts are
    ranked by ``score + bias`` (float32 ``(E,)``, which balances the load and does
    not enter the weights), compared in 64 bits, or without bias and groups by
    the logit.  With ``groups`` of ``E / groups`` neighbours only the
    ``top_groups`` groups with the largest sum of their two best keys take part.
    Equal keys go to the lowest index.  ``weights`` (float32 ``(tokens, k)``) are
    ``scale * score / (sum of the chosen scores + 1e-20)``, or with
    ``normalize=False`` ``scale * score``; ``experts`` (int64) is in the order of
    the keys.  A logit of -inf takes an expert out for that token (a bias of -inf
    for all): where fewer than k are left, the last entries are expert -1 with
    weight 0 and no place in the plan.  A NaN ranks behind every other logit, and
    a group with one among its two best behind the others; it makes the weights of
    its token NaN, with a sigmoid where it is chosen.

    Gradients of ``logits``, once; the bias has none (it only chooses).
    """
    _floats(logits, "expert route logits")
    if logits.ndim != 2:
        raise ValueError("expert route logits must have shape (tokens, experts)")
    tokens, n_experts = logits.shape
    if not 1 <= n_experts <= MAX_EXPERTS:
        raise ValueError(f"expert route takes 1 to {MAX_EXPERTS} experts, got {n_experts}")
    k, groups = _integer(k, "expert route k"), _integer(groups, "expert route groups")
    if groups < 1 or groups > MAX_GROUPS or n_experts % groups != 0:
        raise ValueError(f"expert route groups must divide the experts and be at most {MAX_GROUPS}")
    top_groups = groups if top_groups is None else _integer(top_groups, "expert route top_groups")
    if not 1 <= top_groups <= groups:
        raise ValueError("expert route top_groups must be 1 to groups")
    if not 1 <= k <= top_groups * (n_experts // groups):
        raise ValueError("expert route k must be 1 to the number of experts in top_groups groups")
    if tokens * k > _MOST:
        raise ValueError("expert route takes fewer than 2^31 slots")
    if scores not in SCORES:
        raise ValueError(f"expert route scores must be 'softmax' or 'sigmoid', got {scores!r}")
    if not isinstance(normalize, bool):
        raise TypeError("expert route normalize must be a bool")
    if isinstance(scale, bool) or not isinstance(scale, numbers.Real):
        raise TypeError("expert route scale must be a real number")
    scale = float(scale)
    if not math.isfinite(scale) or abs(scale) > 3.0e38:
        raise ValueError("expert route scale must be a finite float32 number")
    if bias is not None:
        if not isinstance(bias, torch.Tensor):
            raise TypeError("expert route bias must be a tensor or None")
        if bias.dtype != torch.float32:
            raise TypeError("expert route bias must be float32")
        if tuple(bias.shape) != (n_experts,) or not bias.is_contiguous():
            raise ValueError("expert route bias must be contiguous, of shape (experts,)")
        _same_device(logits, bias)
        if bias.requires_grad and torch.is_grad_enabled():
            raise ValueError("expert route bias only chooses and has no gradient: pass bias.detach()")
    require_dcu(logits, bias)
    options = k, groups, top_groups, SCORES.index(scores), normalize, scale
    weights, experts = apply_function(_RouteFunction, logits, bias, options)
    return weights, experts, ExpertPlan(*_extension("expert_dispatch").expert_dispatch(experts, n_experts))


def expert_dispatch(experts: torch.Tensor, n_experts: int) -> ExpertPlan:
    """The plan of experts chosen elsewhere (by element, say): contiguous int64 ``(tokens, k)``.

    Slots whose expert is outside ``0 .. n_experts - 1`` have no place.  A token
    may name an expert more than once.
    """
    if not isinstance(experts, torch.Tensor):
        raise TypeError("expert dispatch experts must be a tensor")
    if experts.dtype != torch.int64:
        raise TypeError("expert dispatch experts must be int64")
    if experts.ndim != 2 or experts.shape[1] < 1 or not experts.is_contiguous():
        raise ValueError("expert dispatch experts must be contiguous, of shape (tokens, k)")
    n_experts = _integer(n_experts, "expert dispatch n_experts")
    if not 1 <= n_experts <= MAX_EXPERTS:
        raise ValueError(f"expert dispatch takes 1 to {MAX_EXPERTS} experts, got {n_experts}")
    if experts.numel() > _MOST:
        raise ValueError("expert dispatch takes fewer than 2^31 slots")
    require_dcu(experts)
    return ExpertPlan(*_extension("expert_dispatch").expert_dispatch(experts, n_experts))


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------

class _LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets, order, slots, sizes, gated):
        keep = any(ctx.needs_input_grad)
        y, before = _extension("expert_linear_forward").expert_linear_forward(x, weight, offsets, order, sizes, gated, keep)
        if keep:
            ctx.save_for_backward(x, weight, before, offsets, order, slots)
            ctx.sizes = sizes
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, before, offsets, order, slots = ctx.saved_tensors
        want = ctx.needs_input_grad
        grads = _extension("expert_linear_backward").expert_linear_backward(
            grad.contiguous(), x, weight, before, offsets, order, slots, ctx.sizes, want[0], want[1])
        return (*grads, None, None, None, None, None)


def expert_linear(x: torch.Tensor, weight: torch.Tensor, plan: ExpertPlan, *, from_tokens: bool = True,
                  activation: str | None = None) -> torch.Tensor:
    """Every slot's rows times its expert's matrix: ``(tokens * k, ..., outputs)`` by place.

    ``x``: contiguous ``(tokens, ..., inputs)``, or with ``from_tokens=False``
    ``(tokens * k, ..., inputs)`` by place, in float32, bfloat16 or float16.
    ``weight``: ``(E, outputs, inputs)`` of its dtype, one matrix for each of
    the plan's experts.  ``activation="silu_gate"``: the first half of the outputs
    is a gate, ``silu(gate) * rest``, and the result has half of them.  At most
    65,536 inputs and outputs, whose sums are kept in float32.  Places behind
    ``plan.offsets[-1]`` give 0 and take no part in a gradient.  Gradients of ``x``
    (summed in float32 over a token's slots) and ``weight``, once; the gradient in
    front of the gate is held in float32 or two 16-bit parts (in float16 up to
    1.3e8), so that they are rounded once.
    """
    tokens, k = _check_plan(plan)
    _floats(x, "expert linear input")
    _floats(weight, "expert linear weight")
    if weight.dtype != x.dtype:
        raise TypeError("expert linear input and weight must be of one dtype")
    if not isinstance(from_tokens, bool):
        raise TypeError("expert linear from_tokens must be a bool")
    if activation not in ACTIVATIONS:
        raise ValueError(f"expert linear activation must be None or 'silu_gate', got {activation!r}")
    if x.ndim < 2:
        raise ValueError("expert linear input must have at least two dimensions")
    if weight.ndim != 3 or weight.shape[0] != plan.offsets.numel() - 1:
        raise ValueError("expert linear weight must have shape (experts, outputs, inputs) for the plan's experts")
    if weight.shape[2] != x.shape[-1]:
        raise ValueError("expert linear weight does not fit the input's last dimension")
    if not 1 <= weight.shape[1] <= MAX_CHANNELS or not 1 <= weight.shape[2] <= MAX_CHANNELS:
        raise ValueError(f"expert linear takes 1 to {MAX_CHANNELS} inputs and outputs")
    if activation is not None and weight.shape[1] % 2 != 0:
        raise ValueError("expert linear: a gate needs an even number of outputs")
    entries = tokens if from_tokens else tokens * k
    if x.shape[0] != entries:
        raise ValueError(f"expert linear input must have {entries} entries, one per {'token' if from_tokens else 'place'}")
    inner = math.prod(x.shape[1:-1])
    if tokens * k * inner >= 2**31 - 1024:
        raise ValueError("expert linear takes fewer than 2^31 - 1024 rows")
    _same_device(x, weight, *plan)
    require_dcu(x, weight, *plan)
    return apply_function(_LinearFunction, x, weight, plan.offsets, plan.order if from_tokens else None,
                          plan.slots if from_tokens else None, (tokens * k, k, inner), activation is not None)


# ---------------------------------------------------------------------------
# the weighted sum of a token's slots
# ---------------------------------------------------------------------------

class _CombineFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, offsets, slots):
        ctx.save_for_backward(y, weights, offsets, slots)
        return _extension("expert_combine_forward").expert_combine_forward(y, weights, slots)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        y, weights, offsets, slots = ctx.saved_tensors
        want = ctx.needs_input_grad
        grads = _extension("expert_combine_backward").expert_combine_backward(grad.contiguous(), y, weights, offsets, slots,
                                                                              want[0], want[1])
        return (*grads, None, None)


def expert_combine(y: torch.Tensor, weights: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """``out[t] = sum_j weights[t, j] * y[plan.slots[t, j]]``: ``(tokens, ...)``.

    ``y``: contiguous ``(tokens * k, ...)`` by place, float32, bfloat16 or float16;
    ``weights``: contiguous float32 ``(tokens, k)``.  Slots without a place add
    nothing, whatever their weight.  Summed in float32 in the order of the
    slots.  Gradients of both, once; a weight without a place has gradient 0.
    """
    tokens, k = _check_plan(plan)
    _floats(y, "expert combine input")
    if not isinstance(weights, torch.Tensor):
        raise TypeError("expert combine weights must be a tensor")
    if weights.dtype != torch.float32:
        raise TypeError("expert combine weights must be float32")
    if y.ndim < 2 or y.shape[0] != tokens * k:
        raise ValueError(f"expert combine input must have {tokens * k} entries, one per place, of at least one dimension")
    if tuple(weights.shape) != (tokens, k) or not weights.is_contiguous():
        raise ValueError("expert combine weights must be contiguous, of shape (tokens, k)")
    if tokens * k > _MOST or math.prod(y.shape[1:]) > _MOST:
        raise ValueError("expert combine takes fewer than 2^31 slots and elements of an entry")
    _same_device(y, weights, *plan)
    require_dcu(y, weights, *plan)
    return apply_function(_CombineFunction, y, weights, plan.offsets, plan.slots)


__all__ = ["ExpertPlan", "expert_route", "expert_dispatch", "expert_linear", "expert_combine", "ACTIVATIONS", "DTYPES",
           "MAX_CHANNELS", "MAX_EXPERTS", "MAX_GROUPS", "SCORES"]
