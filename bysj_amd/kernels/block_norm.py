"""The norms around a block of a model with its gate and residual sum, in one pass.

A block's output goes through a norm, a gate and a scale, is added to the
residual stream, and the sum is normed for the next block.  The reference has
the norm alone (python/kernels/rmsnorm.py), and counts the residual adds and
gates between its operators among the elementwise passes worth fusing
(docs/task2-hip-fusion-plan.md:280-300).  Here

    a = post_scale * x / sqrt(mean x^2 + eps)            the norm after the block
    h = residual + residual_scale * act(gate) * a        gate, scale and residual sum
    y = pre_scale * h / sqrt(mean h^2 + eps)             the norm before the next

with gradients of every input.  Not part of ``kernels.__all__``, which stays
the reference's list.

Over the whole row of a node, ``[N, 16 * C]``, the mean square is a norm of
spherical harmonics and does not depend on the frame's orientation; scales and
gates keep that only where the components of one degree share them.
"""
from __future__ import annotations

import math
import numbers

import torch

from .native import apply_function, _extension, require_dcu

GATE_ACTIVATIONS = (None, "sigmoid", "silu")
DTYPES = (torch.float32, torch.bfloat16, torch.float16)
MAX_CHANNELS = 8192

_GATE_NONE, _GATE_FULL, _GATE_ROW = 0, 1, 2


def _validate(x, residual, post_scale, gate, gate_activation, residual_scale, pre_scale, post_norm, pre_norm, eps):
    for name, tensor in (("input", x), ("residual", residual)):
        if not isinstance(tensor, torch.Tensor):
            raise TypeError(f"residual norm {name} must be a tensor")
        if tensor.dtype not in DTYPES:
            raise TypeError(f"residual norm requires a float32, bfloat16 or float16 {name}")
    if residual.dtype not in (x.dtype, torch.float32):
        raise TypeError("residual norm: the residual must be of the input's dtype or float32")
    if x.ndim < 1:
        raise ValueError("residual norm input must have at least one dimension")
    channels = x.shape[-1]
    if not 1 <= channels <= MAX_CHANNELS:
        raise ValueError(f"residual norm takes 1 to {MAX_CHANNELS} channels, got {channels}")
    if residual.shape != x.shape:
        raise ValueError("residual norm input and residual must have the same shape")
    kind = _GATE_NONE
    if gate is not None:
        if not isinstance(gate, torch.Tensor):
            raise TypeError("residual norm gate must be a tensor or None")
        if gate.dtype != x.dtype:
            raise TypeError("residual norm gate must be of the input's dtype")
        if gate.shape == x.shape:
            kind = _GATE_FULL
        elif gate.shape == (*x.shape[:-1], 1):
            kind = _GATE_ROW
        else:
            raise ValueError("residual norm gate must have the input's shape, or one value a row")
    elif gate_activation is not None:
        raise ValueError("residual norm gate_activation belongs to a gate")
    if gate_activation not in GATE_ACTIVATIONS:
        raise ValueError(f"residual norm gate_activation must be None, 'sigmoid' or 'silu', got {gate_activation!r}")
    for name, norm in (("post_norm", post_norm), ("pre_norm", pre_norm)):
        if not isinstance(norm, bool):
            raise TypeError(f"residual norm {name} must be a bool")
    factor = 1.0
    if residual_scale is not None and not isinstance(residual_scale, torch.Tensor):
        if isinstance(residual_scale, bool) or not isinstance(residual_scale, numbers.Real):
            raise TypeError("residual norm residual_scale must be a tensor, a real number or None")
        factor, residual_scale = float(residual_scale), None
        if not math.isfinite(factor) or abs(factor) > 3.0e38:
            raise ValueError("residual norm residual_scale must be a finite float32 number")
    for name, scale, used in (("post_scale", post_scale, post_norm), ("residual_scale", residual_scale, True),
                              ("pre_scale", pre_scale, pre_norm)):
        if scale is None:
            continue
        if not isinstance(scale, torch.Tensor):
            raise TypeError(f"residual norm {name} must be a tensor or None")
        if not used:
            raise ValueError(f"residual norm {name} belongs to a norm that is switched off")
        if scale.dtype != torch.float32:
            raise TypeError(f"residual norm {name} must be float32")
        if tuple(scale.shape) != (channels,):
            raise ValueError(f"residual norm {name} must have shape (channels,)")
    for name, tensor in (("input", x), ("residual", residual), ("gate", gate), ("post_scale", post_scale),
                         ("residual_scale", residual_scale), ("pre_scale", pre_scale)):
        if tensor is None:
            continue
        if tensor.device != x.device:
            raise ValueError(f"residual norm input and {name} must share a device")
        if not tensor.is_contiguous():
            raise ValueError(f"residual norm {name} must be contiguous")
    try:
        eps = float(eps)
    except (TypeError, ValueError) as error:
        raise ValueError("residual norm eps must be a finite positive number") from error
    if not 1.0e-45 < eps < 3.0e38:
        raise ValueError("residual norm eps must be a finite positive float32 number")
    rows = math.prod(x.shape[:-1])
    return residual_scale, (rows, channels, factor, eps, post_norm, pre_norm, kind, GATE_ACTIVATIONS.index(gate_activation))


class _ResidualNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gate, post_scale, residual_scale, pre_scale, options):
        keep = any(ctx.needs_input_grad)
        h, y, rstd = _extension("residual_norm_forward").residual_norm_forward(x, residual, gate, post_scale, residual_scale,
                                                                               pre_scale, options, keep)
        if keep:
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(x, residual, gate, post_scale, residual_scale, pre_scale, rstd)
            ctx.options = options
        return h if y is None else (h, y)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_h, grad_y=None):
        x, residual, gate, post_scale, residual_scale, pre_scale, rstd = ctx.saved_tensors
        if grad_h is None and grad_y is None:
            return (None,) * 7
        want = list(ctx.needs_input_grad[:6])
        given = want[1] and grad_y is None    # without the second norm the residual's gradient is h's
        want[1] = want[1] and not given
        grad_h, grad_y = (None if g is None else g.contiguous() for g in (grad_h, grad_y))
        grads = _extension("residual_norm_backward").residual_norm_backward(
            grad_h, grad_y, x, residual, gate, post_scale, residual_scale, pre_scale, rstd, ctx.options, want)
        if given:
            grads[1] = grad_h
        return (*grads, None)


def residual_norm(x: torch.Tensor, residual: torch.Tensor, *, post_scale: torch.Tensor | None = None,
                  gate: torch.Tensor | None = None, gate_activation: str | None = None,
                  residual_scale: torch.Tensor | float | None = None, pre_scale: torch.Tensor | None = None,
                  post_norm: bool = True, pre_norm: bool = True, eps: float = 1.0e-6):
    """``(h, y)``: the residual stream behind a block, and its norm for the next one.

    ``h = residual + residual_scale * act(gate) * rms(x) * post_scale`` and
    ``y = rms(h) * pre_scale``, where ``rms(v)`` is ``v / sqrt(mean(v^2) + eps)``
    over the last axis of up to 8,192 channels.  ``x``: contiguous float32,
    bfloat16 or float16; ``residual``: like it, or in float32.  ``gate``: like
    ``x``, or one value a row ``(..., 1)``, through ``gate_activation`` (None,
    ``"sigmoid"`` or ``"silu"``).  ``post_scale``, ``pre_scale`` and
    ``residual_scale``: float32 ``(channels,)`` or None; ``residual_scale`` may be
    a number.  ``post_norm=False`` adds ``x`` as it is, ``pre_norm=False`` returns
    None for ``y``.  ``h`` has the residual's type, ``y`` the input's; sums are
    kept in float32 and ``y`` is that of the unrounded ``h``.  The squares of a
    row must add up to less than float32's largest number (3e38).  Gradients of
    every tensor, once: a second derivative is refused.
    """
    residual_scale, options = _validate(x, residual, post_scale, gate, gate_activation, residual_scale, pre_scale, post_norm,
                                        pre_norm, eps)
    require_dcu(x, residual, gate, post_scale, residual_scale, pre_scale)
    out = apply_function(_ResidualNormFunction, x, residual, gate, post_scale, residual_scale, pre_scale, options)
    return out if pre_norm else (out, None)


__all__ = ["residual_norm", "DTYPES", "GATE_ACTIVATIONS", "MAX_CHANNELS"]
