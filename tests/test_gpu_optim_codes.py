"""GPU tests of what the 8-bit moments do with values that are not ordinary numbers."""
from __future__ import annotations

import pytest
import torch

from bysj_amd.kernels import optim
from oracle import optim as ref
from parity import announce, assert_bitwise

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)


def _nan_words(dtype):
    """NaN of both signs, quiet, with all bits set, and with the fewest."""
    if dtype == torch.float32:
        words = torch.tensor([-1, 0x7FFFFFFF, 0x7FC00000, -0x400000, -0x100000, -0xFFFFF, -0x100001], dtype=torch.int32)
    else:
        words = torch.tensor([-1, 0x7FFF, 0x7FC0, -0x40, -0x10, -0x11], dtype=torch.int16)
    values = words.view(dtype)
    assert torch.isnan(values).all()
    return values


@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_any_nan_turns_its_block_into_nan(dtype, grad):
    """One NaN gradient in a block of 32: both moments of the block become NaN, the neighbours' codes are the oracle's."""
    announce("nan", dtype, grad)
    values = _nan_words(grad)
    n = 96 * len(values) + 17
    generator = torch.Generator().manual_seed(0)
    g = (torch.randn(n, generator=generator) * 1e-3).to(grad)
    hit = torch.zeros(n, dtype=torch.bool)
    for k, value in enumerate(values):
        g[96 * k + 32 + 5 * k] = value
        hit[96 * k + 32: 96 * k + 64] = True
    p = (torch.randn(n, generator=generator) * 0.1).to(dtype).to(DEV)
    plan = optim.adamw_plan([p], state_bits=8)
    zero = torch.zeros(n)
    _, m_wanted, v_wanted = ref.adamw_chain(p.cpu(), g, zero, zero, 1, **HYPER, bits=8)
    optim.adamw_step(plan, [g.to(DEV)], **HYPER)
    (m,), (v,) = optim.adamw_states(plan)
    for actual, wanted in ((m.cpu(), m_wanted), (v.cpu(), v_wanted)):
        assert torch.isnan(actual[hit]).all()
        assert torch.isfinite(actual[~hit]).all()
        assert_bitwise(actual[~hit], wanted[~hit], "other blocks")


@pytest.mark.parametrize("n", [32, 100, 5000])
def test_second_moments_of_minus_zero_count_as_zero(n):
    generator = torch.Generator().manual_seed(n)
    m = torch.randn(n, generator=generator) * 1e-3
    v = torch.rand(n, generator=generator) * 1e-6
    v[::3] = -0.0
    half = torch.full((n,), 0x8000)
    plan = optim.adamw_plan([torch.zeros(n, device=DEV)], [m.to(DEV)], [v.to(DEV)], state_bits=8)
    (m_read,), (v_read,) = optim.adamw_states(plan)
    assert_bitwise(m_read, ref.coded(m, half, True), "first")
    assert_bitwise(v_read, ref.coded(v.abs(), half, False), "second")
    assert (v_read[::3] == 0).all() and torch.isfinite(v_read).all()


def test_second_moments_below_zero_turn_their_block_into_nan():
    """They have no code, and a root that is NaN: visible, as in 32 bits."""
    v = torch.full((96,), 1e-6)
    v[40] = -1e-6
    plan = optim.adamw_plan([torch.zeros(96, device=DEV)], [torch.zeros(96, device=DEV)], [v.to(DEV)], state_bits=8)
    _, (read,) = optim.adamw_states(plan)
    assert torch.isnan(read[32:64]).all() and torch.isfinite(read[:32]).all() and torch.isfinite(read[64:]).all()
