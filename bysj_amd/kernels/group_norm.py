"""Group norm over samples of rows, channels last, with an optional SiLU.

The reference normalises single rows (python/kernels/rmsnorm.py).  A batch of
frames, or the edges of a node, is normalised over more than one row: a sample
is the rows of one frame (or one node), and the statistics run over these rows
and a group of neighbouring channels:

    h = (x - mean) / sqrt(var + eps),    y = act(h * scale + bias)

with ``groups`` = 1 a layer norm over each sample, with ``groups`` = channels
an instance norm.  Samples are given by CSR offsets, as in ``segment_sum``, or
are the entries of the first axis.  Gradients of the input, the scale and the
bias.  Not part of ``kernels.__all__``, which stays the reference's list.

It is a norm of invariant features.  Of spherical-harmonic components it may
run over the l = 0 row alone: a mean over the rows of l > 0, a bias on them or a
SiLU of them depends on the orientation of the frame.
"""
from __future__ import annotations

import math
import numbers

import torch

from .native import apply_function, _extension, require_dcu

ACTIVATIONS = (None, "silu")
DTYPES = (torch.float32, torch.bfloat16, torch.float16)
MAX_CHANNELS = 4096


def _validate(x, groups, scale, bias, offsets, max_rows, eps, activation) -> tuple[int, float]:
    if not isinstance(x, torch.Tensor):
        raise TypeError("group norm input must be a tensor")
    if x.dtype not in DTYPES:
        raise TypeError("group norm requires float32, bfloat16 or float16 input")
    if x.ndim < 2:
        raise ValueError("group norm input must have at least two dimensions")
    if not 1 <= x.shape[-1] <= MAX_CHANNELS:
        raise ValueError(f"group norm takes 1 to {MAX_CHANNELS} channels, got {x.shape[-1]}")
    if not x.is_contiguous():
        raise ValueError("group norm input must be contiguous")
    if isinstance(groups, bool) or not isinstance(groups, numbers.Integral):
        raise TypeError("group norm groups must be an integer")
    if groups < 1 or x.shape[-1] % groups != 0:
        raise ValueError("group norm groups must divide the channels")
    for name, tensor in (("scale", scale), ("bias", bias)):
        if tensor is None:
            continue
        if not isinstance(tensor, torch.Tensor):
            raise TypeError(f"group norm {name} must be a tensor or None")
        if tensor.dtype != torch.float32:
            raise TypeError(f"group norm {name} must be float32")
        if tuple(tensor.shape) != (x.shape[-1],):
            raise ValueError(f"group norm {name} must have shape (channels,)")
        if tensor.device != x.device:
            raise ValueError(f"group norm input and {name} must share a device")
        if not tensor.is_contiguous():
            raise ValueError(f"group norm {name} must be contiguous")
    if offsets is not None:
        if not isinstance(offsets, torch.Tensor):
            raise TypeError("group norm offsets must be a tensor or None")
        if offsets.dtype != torch.int64:
            raise TypeError("group norm offsets must be int64")
        if offsets.ndim != 1 or offsets.numel() < 1:
            raise ValueError("group norm offsets must be a one-dimensional exclusive prefix sum")
        if offsets.device != x.device:
            raise ValueError("group norm input and offsets must share a device")
        if not offsets.is_contiguous():
            raise ValueError("group norm offsets must be contiguous")
    if max_rows is not None:
        if isinstance(max_rows, bool) or not isinstance(max_rows, numbers.Integral):
            raise TypeError("group norm max_rows must be an integer or None")
        if max_rows < 0:
            raise ValueError("group norm max_rows must not be negative")
    if activation not in ACTIVATIONS:
        raise ValueError(f"group norm activation must be None or 'silu', got {activation!r}")
    try:
        eps = float(eps)
    except (TypeError, ValueError) as error:
        raise ValueError("group norm eps must be a finite positive number") from error
    if not math.isfinite(eps) or eps <= 0.0:
        raise ValueError("group norm eps must be a finite positive number")
    return int(groups), eps


class _GroupNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale, bias, offsets, groups, max_rows, eps, silu):
        native = _extension("group_norm_forward")
        shape = x.shape
        samples = shape[0] if offsets is None else offsets.numel() - 1
        sizes = samples, shape[0], math.prod(shape[1:-1]), shape[-1]
        y, statistics = native.group_norm_forward(x, groups, scale, bias, offsets, eps, silu, max_rows=max_rows, sizes=sizes)
        ctx.save_for_backward(x, scale, bias, offsets, statistics)
        ctx.arguments = groups, max_rows, silu, sizes
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        x, scale, bias, offsets, statistics = ctx.saved_tensors
        groups, max_rows, silu, sizes = ctx.arguments
        want = ctx.needs_input_grad
        native = _extension("group_norm_backward")
        grads = native.group_norm_backward(grad_output.contiguous(), x, groups, scale, bias, offsets, statistics, silu,
                                           want_x=want[0], want_scale=want[1], want_bias=want[2], max_rows=max_rows,
                                           sizes=sizes)
        return (*grads, None, None, None, None, None)


def group_norm(x: torch.Tensor, groups: int, scale: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
               offsets: torch.Tensor | None = None, max_rows: int | None = None, eps: float = 1.0e-5,
               activation: str | None = None) -> torch.Tensor:
    """``act((x - mean) / sqrt(var + eps) * scale + bias)`` with statistics per sample and group of channels.

    ``x``: contiguous ``(entries, ..., channels)`` in float32, bfloat16 or
    float16, at most 4,096 channels.  ``offsets`` (int64, ``samples + 1``):
    sample ``s`` is the entries ``offsets[s]`` to ``offsets[s + 1]`` with all
    their rows; entries of no sample give 0.  Without offsets every entry is a
    sample.  ``scale``, ``bias``: float32 ``(channels,)``.  ``max_rows``: the
    entries of the longest sample where the caller knows it; it only selects
    the schedule (one that is too small costs time).  ``activation``: None or
    ``"silu"``.  Statistics are kept in float32 or wider whatever the input's
    type; the squared deviations of a sample's group must add up to less than
    float32's largest number (3e38), else its rstd is 0.  The gradients have no
    gradients of their own: a second derivative is refused.
    """
    groups, eps = _validate(x, groups, scale, bias, offsets, max_rows, eps, activation)
    require_dcu(x, scale, bias, offsets)
    return apply_function(_GroupNormFunction, x, scale, bias, offsets, groups,
                          None if max_rows is None else int(max_rows), eps, activation == "silu")


__all__ = ["group_norm", "ACTIVATIONS", "DTYPES", "MAX_CHANNELS"]
