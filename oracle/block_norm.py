"""CPU oracle of the norms around a block, in 64 bits -- test infrastructure only."""
from __future__ import annotations

import torch


def _gate(gate, activation):
    """act(gate) and its slope."""
    if activation is None:
        return gate, torch.ones_like(gate)
    s = torch.sigmoid(gate)
    return (s, s * (1.0 - s)) if activation == "sigmoid" else (gate * s, s * (1.0 + gate * (1.0 - s)))


def _prepared(x, residual, post_scale, gate, activation, residual_scale, pre_scale, post_norm, eps):
    x, residual = x.detach().double(), residual.detach().double()
    one = torch.ones(x.shape[-1], dtype=torch.float64)
    post = one if post_scale is None else post_scale.detach().double()
    pre = one if pre_scale is None else pre_scale.detach().double()
    if residual_scale is None:
        scale = one
    else:
        scale = residual_scale.detach().double() if isinstance(residual_scale, torch.Tensor) else one * float(residual_scale)
    act, slope = (one, None) if gate is None else _gate(gate.detach().double(), activation)
    r = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) if post_norm else torch.ones_like(x[..., :1])
    a = x * r * post
    h = residual + scale * act * a
    q = 1.0 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    return x, post, pre, scale, act, slope, r, a, h, q


def residual_norm_reference(x, residual, *, post_scale=None, gate=None, gate_activation=None, residual_scale=None, pre_scale=None,
                            post_norm=True, pre_norm=True, eps=1.0e-6):
    _, _, pre, _, _, _, _, _, h, q = _prepared(x, residual, post_scale, gate, gate_activation, residual_scale, pre_scale, post_norm, eps)
    return h, h * q * pre if pre_norm else None


def residual_norm_backward_reference(grad_h, grad_y, x, residual, *, post_scale=None, gate=None, gate_activation=None,
                                     residual_scale=None, pre_scale=None, post_norm=True, pre_norm=True, eps=1.0e-6):
    """Gradients of x, residual, gate, post_scale, residual_scale, pre_scale by the closed form (None without the input)."""
    x, post, pre, scale, act, slope, r, a, h, q = _prepared(x, residual, post_scale, gate, gate_activation, residual_scale, pre_scale,
                                                            post_norm, eps)
    g = torch.zeros_like(h) if grad_h is None else grad_h.detach().double()
    columns = tuple(range(x.ndim - 1))
    d_pre = torch.zeros(x.shape[-1], dtype=torch.float64)
    if pre_norm and grad_y is not None:
        dy = grad_y.detach().double()
        d_pre = (dy * h * q).sum(columns)
        u = dy * pre
        g = g + q * (u - h * q * q * (u * h).mean(-1, keepdim=True))
    d_scale = (g * act * a).sum(columns)
    d_gate = None
    if gate is not None:
        d_gate = g * scale * a * slope
        if gate.shape != x.shape:
            d_gate = d_gate.sum(-1, keepdim=True)
    b = g * scale * act
    d_post = (b * x * r).sum(columns)
    v = b * post
    dx = r * (v - x * r * r * (v * x).mean(-1, keepdim=True)) if post_norm else v
    return (dx, g, d_gate, None if post_scale is None else d_post, d_scale if isinstance(residual_scale, torch.Tensor) else None,
            None if pre_scale is None else d_pre)


def residual_norm_grad_x_operands(grad_h, grad_y, x, residual, **kwargs):
    """r (|v| + |x r mean(v x r)|): the magnitudes whose difference grad_x is."""
    post_scale, gate, eps = kwargs.get("post_scale"), kwargs.get("gate"), kwargs.get("eps", 1.0e-6)
    x, post, _, scale, act, _, r, _, _, _ = _prepared(x, residual, post_scale, gate, kwargs.get("gate_activation"),
                                                      kwargs.get("residual_scale"), kwargs.get("pre_scale"), True, eps)
    g = residual_norm_backward_reference(grad_h, grad_y, x, residual, **kwargs)[1]
    v = g * scale * act * post
    return r * (v.abs() + (x * r * (v * x * r).mean(-1, keepdim=True)).abs())
