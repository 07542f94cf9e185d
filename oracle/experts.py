"""CPU oracle of routing, dispatch, the experts' products and their sum, in 64 bits -- test infrastructure only.

Token by token and expert by expert, from the definitions.
"""
from __future__ import annotations

import math

import torch


def _scores(row, scores):
    if scores == "sigmoid":
        return [0.0 if v == -math.inf else (1.0 / (1.0 + math.exp(-v)) if v > -700.0 else 0.0) for v in row]
    top = max(row)
    if top == -math.inf:
        return [0.0] * len(row)
    e = [math.exp(v - top) for v in row]
    total = math.fsum(e)
    return [v / total for v in e]


def expert_route_reference(logits, k, *, scores="softmax", bias=None, groups=1, top_groups=None, normalize=True, scale=1.0):
    """``(weights, experts, scores)`` of logits without NaN or +inf, lists of rows as tensors."""
    n = logits.shape[1]
    top_groups = groups if top_groups is None else top_groups
    all_weights, all_experts, all_scores = [], [], []
    for row in logits.detach().double().tolist():
        s = _scores(row, scores)
        key = list(row) if bias is None and groups == 1 else [a + b for a, b in zip(s, [0.0] * n if bias is None else bias.double().tolist())]
        key = [-math.inf if v == -math.inf else u for v, u in zip(row, key)]
        members = n // groups
        values = []
        for g in range(groups):
            best = sorted(key[g * members: (g + 1) * members], reverse=True)[:2]
            there = [v for v in best if v > -math.inf]
            values.append(sum(there) if there else -math.inf)
        allowed = sorted(range(groups), key=lambda g: (-values[g], g))[:top_groups]
        order = sorted((e for e in range(n) if e // members in allowed and key[e] > -math.inf), key=lambda e: (-key[e], e))[:k]
        total = math.fsum(s[e] for e in order) + 1.0e-20
        w = [scale * s[e] / (total if normalize else 1.0) for e in order]
        all_weights.append(w + [0.0] * (k - len(w)))
        all_experts.append(order + [-1] * (k - len(order)))
        all_scores.append(s)
    return (torch.tensor(all_weights, dtype=torch.float64).view(-1, k), torch.tensor(all_experts, dtype=torch.int64).view(-1, k),
            torch.tensor(all_scores, dtype=torch.float64).view(-1, n))


def expert_route_backward_reference(grad_weights, logits, k, *, scores="softmax", normalize=True, scale=1.0, **kwargs):
    _, experts, s = expert_route_reference(logits, k, scores=scores, normalize=normalize, scale=scale, **kwargs)
    held = experts >= 0
    chosen = torch.where(held, s.gather(1, experts.clamp(min=0)), 0.0)
    dw = torch.where(held, grad_weights.detach().double(), 0.0)
    total = chosen.sum(1, keepdim=True) + 1.0e-20
    if normalize:    # dw - sum(dw s) / total, without its cancellation: (sum_i s_i (dw - dw_i) + 1e-20 dw) / total
        ds = scale / total.square() * ((chosen[:, None] * (dw[:, :, None] - dw[:, None])).sum(2) + 1.0e-20 * dw)
    else:
        ds = scale * dw
    ds = torch.where(held, ds, 0.0)
    dense = torch.zeros_like(s).scatter_add_(1, experts.clamp(min=0), ds)
    if scores == "sigmoid":
        return dense * s * (1.0 - s)
    return s * (dense - (ds * chosen).sum(1, keepdim=True))


def expert_dispatch_reference(experts, n_experts):
    """``(offsets, order, slots)``."""
    flat = experts.reshape(-1).tolist()
    offsets, order, slots = [0], [], [-1] * len(flat)
    for e in range(n_experts):
        for slot, expert in enumerate(flat):
            if expert == e:
                slots[slot] = len(order)
                order.append(slot)
        offsets.append(len(order))
    order += [-1] * (len(flat) - len(order))
    return (torch.tensor(offsets), torch.tensor(order, dtype=torch.int64),
            torch.tensor(slots, dtype=torch.int64).view(experts.shape))


def _entries(plan, e, from_tokens):
    offsets, order, slots = plan
    a, b = int(offsets[e]), int(offsets[e + 1])
    places = torch.arange(a, b)
    return places, order[a:b] // slots.shape[1] if from_tokens else places


def expert_linear_reference(x, weight, plan, *, from_tokens=True, activation=None, grad=None):
    """``y``, or with its gradient ``(y, dx, dweight, dx_bound, dweight_bound)``.

    The bounds are the sums of the magnitudes of the products that make up dx and
    dweight, by which the rounding of dz, the gate's gradient, is multiplied.
    """
    x, weight = x.detach().double(), weight.detach().double()
    n_out = weight.shape[1] // (1 if activation is None else 2)
    y = torch.zeros(plan[1].numel(), *x.shape[1:-1], n_out, dtype=torch.float64)
    dx, dw = torch.zeros_like(x), torch.zeros_like(weight)
    dx_bound, dw_bound = torch.zeros_like(x), torch.zeros_like(weight)
    for e in range(weight.shape[0]):
        places, entries = _entries(plan, e, from_tokens)
        if places.numel() == 0:
            continue
        z = x[entries] @ weight[e].t()
        if activation is not None:
            gate, up = z[..., :n_out], z[..., n_out:]
            s = torch.sigmoid(gate)
            y[places] = gate * s * up
        else:
            y[places] = z
        if grad is None:
            continue
        dz = grad.detach().double()[places]
        if activation is not None:
            dz = torch.cat([dz * up * s * (1.0 + gate * (1.0 - s)), dz * gate * s], -1)
        rows, flat = x[entries].reshape(-1, x.shape[-1]), dz.reshape(-1, dz.shape[-1])
        dx.index_add_(0, entries, dz @ weight[e])
        dx_bound.index_add_(0, entries, dz.abs() @ weight[e].abs())
        dw[e] = flat.t() @ rows
        dw_bound[e] = flat.abs().t() @ rows.abs()
    return y if grad is None else (y, dx, dw, dx_bound, dw_bound)


def expert_combine_reference(y, weights, plan, grad=None):
    """``out``, or with its gradient ``(out, dy, dweights)``."""
    y, weights = y.detach().double(), weights.detach().double()
    slots = plan[2]
    out = torch.zeros(slots.shape[0], *y.shape[1:], dtype=torch.float64)
    dy, dweights = torch.zeros_like(y), torch.zeros_like(weights)
    for t in range(slots.shape[0]):
        for j, place in enumerate(slots[t].tolist()):
            if place < 0:
                continue
            out[t] += weights[t, j] * y[place]
            if grad is not None:
                dy[place] += weights[t, j] * grad[t].double()
                dweights[t, j] = (grad[t].double() * y[place]).sum()
    return out if grad is None else (out, dy, dweights)
