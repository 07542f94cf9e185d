"""CPU oracle of the group norm in 64 bits -- test infrastructure only.

A sample at a time, from the definition:  h = (x - mean) / sqrt(var + eps) per
group of channels,  y = act(h * scale + bias);  rows of no sample give 0.
"""
from __future__ import annotations

import torch


def _samples(x, offsets):
    bounds = list(range(x.shape[0] + 1)) if offsets is None else [min(max(int(o), 0), x.shape[0]) for o in offsets]
    return [(a, b) for a, b in zip(bounds, bounds[1:]) if a < b]


def _normed(part, groups, eps):
    """(h, 1 / sqrt(var + eps)) of one sample's rows as (rows, groups, channels per group)."""
    rows = part.reshape(-1, groups, part.shape[-1] // groups)
    centred = rows - rows.mean((0, 2), keepdim=True)
    inverse = 1.0 / torch.sqrt(centred.square().mean((0, 2), keepdim=True) + eps)
    return centred * inverse, inverse


def group_norm_reference(x, groups, scale=None, bias=None, offsets=None, eps=1.0e-5, activation=None):
    x = x.detach().double()
    channels = x.shape[-1]
    scale = torch.ones(channels, dtype=torch.float64) if scale is None else scale.detach().double()
    bias = torch.zeros(channels, dtype=torch.float64) if bias is None else bias.detach().double()
    y = torch.zeros_like(x)
    for a, b in _samples(x, offsets):
        h, _ = _normed(x[a:b], groups, eps)
        z = h.reshape(-1, channels) * scale + bias
        y[a:b] = (z * torch.sigmoid(z) if activation == "silu" else z).view(x[a:b].shape)
    return y


def group_norm_backward_reference(grad, x, groups, scale=None, bias=None, offsets=None, eps=1.0e-5, activation=None):
    """``(grad_x, grad_scale, grad_bias)`` by the closed form."""
    x, grad = x.detach().double(), grad.detach().double()
    channels = x.shape[-1]
    scale = torch.ones(channels, dtype=torch.float64) if scale is None else scale.detach().double()
    bias = torch.zeros(channels, dtype=torch.float64) if bias is None else bias.detach().double()
    grad_x, grad_scale, grad_bias = torch.zeros_like(x), torch.zeros_like(scale), torch.zeros_like(bias)
    for a, b in _samples(x, offsets):
        h, inverse = _normed(x[a:b], groups, eps)
        flat = h.reshape(-1, channels)
        z = flat * scale + bias
        gate = torch.sigmoid(z)
        dz = grad[a:b].reshape(-1, channels) * (gate * (1.0 + z * (1.0 - gate)) if activation == "silu" else 1.0)
        grad_scale += (dz * flat).sum(0)
        grad_bias += dz.sum(0)
        u = (dz * scale).view(h.shape)
        out = inverse * (u - u.mean((0, 2), keepdim=True) - h * (u * h).mean((0, 2), keepdim=True))
        grad_x[a:b] = out.reshape(x[a:b].shape)
    return grad_x, grad_scale, grad_bias
