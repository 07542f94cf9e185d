"""CPU oracle of the AdamW step -- test infrastructure only.

``adamw_chain`` restates the step as the chain of float32 operations that it
promises to equal bit for bit; ``adamw_f64`` is the definition in 64 bits.
Tensors are flat here.
"""
from __future__ import annotations

import math

import torch

SPAN = 32


def mix(x: torch.Tensor) -> torch.Tensor:
    """The integer mix of 32 bits, in int64."""
    x = x & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x6A09E667) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_bits(seed: int, t: int, positions: torch.Tensor) -> torch.Tensor:
    seed &= 0xFFFFFFFFFFFFFFFF
    high = positions >> 32
    step_key = mix(torch.tensor(t) + high * 0x9E3779B1)
    key = mix((seed & 0xFFFFFFFF) ^ mix((seed >> 32) + step_key))
    return mix((positions & 0xFFFFFFFF) ^ key)


def coded(x: torch.Tensor, random16: torch.Tensor, signed: bool) -> torch.Tensor:
    """The values that the 8-bit codes of a flat float32 tensor stand for; blocks of 32 from its start."""
    count = x.numel()
    pad = -count % SPAN
    x = torch.nn.functional.pad(x, (0, pad))
    random16 = torch.nn.functional.pad(random16, (0, pad))
    word = x.abs().view(torch.int32).long()
    binades = 16 if signed else 32
    top = ((word + 0xFFFFF) >> 23).view(-1, SPAN).amax(1).clamp(min=binades).repeat_interleave(SPAN)
    low = (top - binades + 1) << 3
    code = ((word + (random16 << 4)) >> 20) - low
    least = ((low + 1) << 20).int().view(torch.float32)
    under = x.abs() > least * (random16.float() / 65536.0) if signed else word > 0
    code = torch.where(code < 1, under.long(), code)
    value = torch.where(code > 0, ((code + low) << 20).int().view(torch.float32), torch.zeros_like(x))
    value = torch.copysign(value, x) if signed else value
    return torch.where(top >= 255, torch.full_like(value, float("nan")), value)[:count]


def to_bfloat16(x: torch.Tensor, random16: torch.Tensor) -> torch.Tensor:
    word = x.view(torch.int32).long() & 0xFFFFFFFF
    up = (word + random16) & 0xFFFF0000
    finite = (word & 0x7F800000) != 0x7F800000
    up = torch.where(up >= 0x80000000, up - 0x100000000, up).int().view(torch.float32)
    return torch.where(finite, up, x).bfloat16()


def adamw_chain(p, g, m, v, t, *, lr, betas, eps, weight_decay, factor=1.0, seed=0, position=0, bits=32):
    """``(p, m, v)`` after step ``t`` (from 1) of one flat tensor that starts at ``position`` of its plan."""
    beta1, beta2 = betas
    g = g.float() * torch.tensor(factor, dtype=torch.float32)
    m = m * beta1 + g * (1.0 - beta1)
    v = v * beta2 + (g * g) * (1.0 - beta2)
    denominator = v.sqrt() * (1.0 / math.sqrt(1.0 - beta2 ** t)) + eps
    new_p = p.float() * (1.0 - lr * weight_decay) - (m / denominator) * (lr / (1.0 - beta1 ** t))
    noise = random_bits(seed, t, position + torch.arange(p.numel(), device=p.device))
    if p.dtype == torch.bfloat16:
        new_p = to_bfloat16(new_p, mix(noise + 0x9E3779B1) & 0xFFFF)
    if bits == 8:
        m, v = coded(m, noise & 0xFFFF, True), coded(v, noise >> 16, False)
    return new_p, m, v


def adamw_f64(p, g, m, v, t, *, lr, betas, eps, weight_decay, factor=1.0):
    beta1, beta2 = betas
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * factor
    m = beta1 * m + (1.0 - beta1) * g
    v = beta2 * v + (1.0 - beta2) * g * g
    step = lr * (m / (1.0 - beta1 ** t)) / (torch.sqrt(v / (1.0 - beta2 ** t)) + eps)
    return p - lr * weight_decay * p - step, m, v
