"""GPU tests of the optimiser step: gradient norm, AdamW with moments in 32 and in 8 bits.

A step promises the bits of the elementwise float32 chain, so it is compared
with that chain (run by torch on the same GPU) bit for bit, at every size and
type; the chain itself is compared with the definition in 64 bits: a moment
sums two products (three roundings), a parameter adds a quotient of about eight
roundings, so ten of 2^-24 (6e-7) of the largest term bound it.
"""
from __future__ import annotations

import copy
import math

import pytest
import torch

from bysj_amd.kernels import optim
from oracle import optim as ref
from parity import announce, assert_bitwise, assert_close_scaled

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)
SIZES = [1, 3, 31, 32, 33, 100, 4095, 4096, 4097, 0, 10000]


def _model(sizes, dtype=torch.float32, grad=torch.float32, seed=0):
    """Parameters, gradients and moments of a model in training, each tensor of its own scale."""
    generator = torch.Generator().manual_seed(seed)
    params, grads, first, second = [], [], [], []
    for k, n in enumerate(sizes):
        size = 10.0 ** (-k % 7 - 3)
        params.append((torch.randn(n, generator=generator) * 0.1).to(dtype))
        grads.append((torch.randn(n, generator=generator) * size).to(grad))
        first.append(torch.randn(n, generator=generator) * size * 0.3)
        second.append(torch.rand(n, generator=generator) * size * size)
    return tuple([t.to(DEV) for t in group] for group in (params, grads, first, second))


def _positions(sizes):
    at, out = 0, []
    for n in sizes:
        out.append(at)
        at += -(-n // 32) * 32
    return out


# ---------------------------------------------------------------------------
# gradient norm
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("sizes", [[1], [0, 5, 0], SIZES, [7] * 500, [8191, 8192, 8193], [20_000_001], [3] * 180, [9] * 181])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_grad_norm(sizes, dtype):
    announce("grad norm", len(sizes), sum(sizes), dtype)
    generator = torch.Generator(device=DEV).manual_seed(1)
    grads = [(torch.randn(n, generator=generator, device=DEV) * 0.1).to(dtype) for n in sizes]
    wanted = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    for limit in (None, 0.5, 1e9):
        norm, factor = optim.grad_norm(grads, limit)
        assert norm.shape == factor.shape == () and norm.device == DEV
        # 64-bit sums, rounded once
        assert abs(norm.item() - wanted) <= 2.0 ** -24 * 1.01 * wanted
        expected = 1.0 if limit is None else min(1.0, limit / (wanted + 1e-6))
        assert abs(factor.item() - expected) <= 2.0 ** -24 * 1.01 * expected
    again = optim.grad_norm(grads, 0.5)
    assert_bitwise(torch.stack(again), torch.stack(optim.grad_norm(grads, 0.5)), "again")


def test_grad_norm_of_mixed_views_and_missing_gradients():
    held = torch.arange(1, 1001, dtype=torch.float32, device=DEV)
    half = torch.ones(1001, dtype=torch.bfloat16, device=DEV)
    norm, factor = optim.grad_norm([held[1:8], None, half[3:], held[9:].view(-1, 1)], 10.0)
    wanted = math.sqrt(sum(k * k for k in range(2, 9)) + 998 + sum(k * k for k in range(10, 1001)))
    assert abs(norm.item() - wanted) <= 2.0 ** -24 * 1.01 * wanted
    assert abs(factor.item() - 10.0 / wanted) <= 1e-6 / wanted


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_grad_norm_that_is_not_finite(bad):
    grads = [torch.ones(5000, device=DEV), torch.ones(3, device=DEV)]
    grads[0][4321] = bad
    norm, factor = optim.grad_norm(grads, 1.0)
    assert not math.isfinite(norm.item()) and math.isnan(factor.item())
    # squares past float32's range are summed in 64 bits
    grads = [torch.full((4,), 1e30, device=DEV)]
    norm, factor = optim.grad_norm(grads, 1.0)
    assert abs(norm.item() / 2e30 - 1.0) < 1e-6 and abs(factor.item() / 5e-31 - 1.0) < 1e-6


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,grad", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                        (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)])
def test_steps_equal_the_chain(dtype, grad, bits):
    announce("adamw", dtype, grad, bits)
    params, grads, first, second = _model(SIZES, dtype, grad)
    factor = torch.tensor(0.37, device=DEV)
    expected = [[p.clone(), m.clone(), v.clone()] for p, m, v in zip(params, first, second)]
    if bits == 8:
        for part in expected:
            half = torch.full((part[0].numel(),), 0x8000, dtype=torch.int64, device=DEV)
            part[1], part[2] = ref.coded(part[1], half, True), ref.coded(part[2], half, False)
    plan = optim.adamw_plan(params, first, second, step=41, state_bits=bits)
    for step in range(42, 46):
        use_factor = step % 2 == 0
        optim.adamw_step(plan, grads, **HYPER, grad_factor=factor if use_factor else None, seed=12345678901)
        moments = (first, second) if bits == 32 else optim.adamw_states(plan)
        for k, (n, position) in enumerate(zip(SIZES, _positions(SIZES))):
            before = [t.clone() for t in expected[k]]
            expected[k] = list(ref.adamw_chain(*[expected[k][0], grads[k], expected[k][1], expected[k][2]], step, **HYPER,
                                               factor=0.37 if use_factor else 1.0, seed=12345678901, position=position,
                                               bits=bits))
            for name, actual, wanted in zip("pmv", (params[k], moments[0][k], moments[1][k]), expected[k]):
                assert_bitwise(actual, wanted, f"step {step} size {n} {name}")
            if bits == 32 and dtype == torch.float32 and n:
                truth = ref.adamw_f64(before[0], grads[k], before[1], before[2], step, **HYPER,
                                      factor=float(torch.tensor(0.37)) if use_factor else 1.0)
                for actual, wanted in zip((params[k], first[k], second[k]), truth):
                    assert_close_scaled(actual, wanted, rtol=6e-7, scale=6e-7, what=f"64 bits, size {n}")
    assert plan.steps().tolist() == [45 if n else 41 for n in SIZES]


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(bits):
    """More tensors than one list of pointers holds."""
    sizes = [1 + 37 * (k % 11) for k in range(1000)]
    params, grads, first, second = _model(sizes)
    plan = optim.adamw_plan(params, state_bits=bits)
    start = [p.clone() for p in params]
    optim.adamw_step(plan, grads, **HYPER, seed=5)
    for k, position in enumerate(_positions(sizes)):
        if k % 97 == 0 or k in (439, 440, 441, 999):
            zero = torch.zeros_like(start[k])
            wanted, _, _ = ref.adamw_chain(start[k], grads[k], zero, zero, 1, **HYPER, seed=5, position=position, bits=bits)
            assert_bitwise(params[k], wanted, f"tensor {k}")
    assert plan.steps().eq(1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_views_at_odd_offsets(bits):
    sizes = [5000, 77]
    for dtype in (torch.float32, torch.bfloat16):
        params, grads, first, second = _model(sizes, dtype, dtype)
        held = [torch.zeros(n + 8, dtype=dtype, device=DEV) for n in sizes for _ in range(2)]
        views = [h[3: 3 + n] for h, n in zip(held, [n for n in sizes for _ in range(2)])]
        odd_params, odd_grads = views[0::2], views[1::2]
        for to, value in zip(odd_params + odd_grads, params + grads):
            to.copy_(value)
        moved = [torch.zeros(n + 1, device=DEV)[1:].copy_(m) for n, m in zip(sizes, first)], second
        plan = optim.adamw_plan(params, [m.clone() for m in first], [v.clone() for v in second], state_bits=bits)
        odd = optim.adamw_plan(odd_params, *moved, state_bits=bits)
        for _ in range(2):
            optim.adamw_step(plan, grads, **HYPER)
            optim.adamw_step(odd, odd_grads, **HYPER)
        for a, b in zip(odd_params, params):
            assert_bitwise(a, b, "odd view")
        for h, n in zip(held, [n for n in sizes for _ in range(2)]):
            assert not h[:3].any() and not h[3 + n:].any()  # nothing around the views is written


@pytest.mark.parametrize("bits", [32, 8])
def test_missing_gradients_and_skipped_steps(bits):
    sizes = [100, 33, 5000]
    params, grads, first, second = _model(sizes)
    plan = optim.adamw_plan(params, first, second, step=[3, 4, 5], state_bits=bits)
    start = [t.clone() for t in params]
    optim.adamw_step(plan, [grads[0], None, grads[2]], **HYPER)
    assert plan.steps().tolist() == [4, 4, 6]
    assert_bitwise(params[1], start[1], "no gradient")
    assert not torch.equal(params[0], start[0]) and not torch.equal(params[2], start[2])
    held = [t.clone() for t in params] + [m.clone() for group in optim.adamw_states(plan) for m in group]
    optim.adamw_step(plan, grads, **HYPER, grad_factor=torch.tensor(float("nan"), device=DEV))
    for a, b in zip(params + [m for group in optim.adamw_states(plan) for m in group], held):
        assert_bitwise(a, b, "a factor of NaN")
    assert plan.steps().tolist() == [4, 4, 6]
    optim.adamw_step(plan, [None] * 3, **HYPER)
    assert plan.steps().tolist() == [4, 4, 6]


def test_learning_rate_on_the_device():
    sizes = [500, 40]
    params, grads, first, second = _model(sizes)
    other = [p.clone() for p in params]
    plan, twin = (optim.adamw_plan(group, state_bits=32) for group in (params, other))
    rate = torch.tensor(0.25, device=DEV)
    optim.adamw_step(plan, grads, **{**HYPER, "lr": rate})
    optim.adamw_step(twin, grads, **{**HYPER, "lr": 0.25})
    for a, b in zip(params, other):
        assert_bitwise(a, b, "lr")


def test_seeds_and_steps_draw_other_bits():
    params, grads, first, second = _model([4096], torch.bfloat16)
    results = []
    for seed in (1, 2, 1, 1 + (1 << 32)):
        p = [params[0].clone()]
        plan = optim.adamw_plan(p, state_bits=8)
        for _ in range(2):
            optim.adamw_step(plan, grads, **HYPER, seed=seed)
        results.append(p[0])
    assert torch.equal(results[0], results[2])
    assert not torch.equal(results[0], results[1]) and not torch.equal(results[0], results[3])


def test_eight_bit_averages_follow_the_exact_ones():
    """The stochastic roundings keep the averages' means: over 2^18 elements with gradients of one size, the mean of v
    stays with the exact average.  One element's rounding has a variance below step^2 f (1 - f) with a step of at most
    v / 8 and f the distance moved in steps; summed over t steps of decay 0.999 its relative variance stays below 0.08,
    so the mean of 2^18 elements is within 5 sqrt(0.08 / 2^18) = 0.3% of it."""
    n, beta2 = 1 << 18, 0.999
    p = [torch.zeros(n, device=DEV)]
    plan = optim.adamw_plan(p, state_bits=8)
    generator = torch.Generator(device=DEV).manual_seed(0)
    exact = torch.zeros(n, dtype=torch.float64, device=DEV)
    for _ in range(300):
        g = torch.randn(n, generator=generator, device=DEV) * 1e-3
        exact = exact * beta2 + g.double().square() * (1.0 - beta2)
        optim.adamw_step(plan, [g], **HYPER)
    _, (v,) = optim.adamw_states(plan)
    assert abs((v.double().mean() / exact.mean()).item() - 1.0) < 3e-3
    assert (v > 0).all()


def test_nonfinite_gradients_without_a_norm_poison_their_block_visibly():
    p = [torch.zeros(128, device=DEV)]
    plan = optim.adamw_plan(p, state_bits=8)
    g = torch.ones(128, device=DEV)
    g[70] = float("inf")
    optim.adamw_step(plan, [g], **HYPER)
    (m,), (v,) = optim.adamw_states(plan)
    assert torch.isnan(v[64:96]).all() and torch.isfinite(v[:64]).all() and torch.isfinite(v[96:]).all()
    assert torch.isnan(p[0][70]) and torch.isfinite(p[0][:70]).all()


def test_versions_move_with_the_parameters():
    params, grads, _, _ = _model([10])
    w = params[0].requires_grad_(True)
    y = (w * w).sum()
    before = w._version
    plan = optim.adamw_plan([w])
    optim.adamw_step(plan, grads, **HYPER)
    assert w._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_replay_the_eager_ones(bits):
    """Norm and step in a graph, replayed with new gradients and eager work in between, against an eager twin."""
    sizes = [1000, 33, 64 * 64, 1]
    params, grads, first, second = _model(sizes, torch.bfloat16, torch.bfloat16)
    twin = [p.clone() for p in params]
    plans = [optim.adamw_plan(group, [m.clone() for m in first], [v.clone() for v in second], state_bits=bits)
             for group in (params, twin)]
    rate = torch.tensor(1e-2, device=DEV)

    def once(plan):
        norm, factor = optim.grad_norm(grads, 0.01)
        optim.adamw_step(plan, grads, **{**HYPER, "lr": rate}, grad_factor=factor, seed=9)
        return norm

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        once(plans[0])
    torch.cuda.current_stream().wait_stream(stream)
    once(plans[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = once(plans[0])
    for turn in range(4):
        for g in grads:
            g.mul_(1.5)
        rate.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        assert_bitwise(norm, once(plans[1]), f"norm {turn}")
        for a, b in zip(params, twin):
            assert_bitwise(a, b, f"parameters {turn}")
        for a, b in zip(sum(optim.adamw_states(plans[0]), []), sum(optim.adamw_states(plans[1]), [])):
            assert_bitwise(a, b, f"moments {turn}")
    assert plans[0].steps().tolist() == plans[1].steps().tolist() == [5] * 4


def test_positions_past_32_bits():
    """A plan of more than 2^32 positions: its last tensor draws bits of the upper word, and lies past 2^32 bytes."""
    big = torch.zeros((1 << 32) + 64, dtype=torch.bfloat16, device=DEV)
    last = (torch.randn(100, generator=torch.Generator().manual_seed(0)) * 0.1).bfloat16().to(DEV)
    plan = optim.adamw_plan([big, last], state_bits=8)
    start = last.clone()
    g = torch.randn(100, device=DEV) * 1e-3
    optim.adamw_step(plan, [None, g], **HYPER, seed=3)
    zero = torch.zeros(100, device=DEV)
    wanted, m, v = ref.adamw_chain(start, g, zero, zero, 1, **HYPER, seed=3, position=big.numel(), bits=8)
    assert_bitwise(last, wanted, "parameter")


# ---------------------------------------------------------------------------
# the optimiser
# ---------------------------------------------------------------------------

def _optimiser(params, bits=32, **more):
    return optim.AdamW([{"params": params[:2], "weight_decay": 0.0}, {"params": params[2:], "lr": 1e-2}], lr=1e-3,
                       max_norm=0.5, state_bits=bits, **more)


@pytest.mark.parametrize("bits", [32, 8])
def test_optimiser_follows_the_functions(bits):
    sizes = [64, 64 * 64, 33, 500]
    params, grads, _, _ = _model(sizes)
    params[3] = params[3].bfloat16()
    twin = [p.clone() for p in params]
    for p in params:
        p.requires_grad_(True)
    optimiser = _optimiser(params, bits, seed=7)
    plans = [optim.adamw_plan(twin[:2], state_bits=bits), optim.adamw_plan(twin[2:3], state_bits=bits),
             optim.adamw_plan(twin[3:], state_bits=bits)]
    for step in range(3):
        for p, g in zip(params, grads):
            p.grad = (g * (step + 1)).to(p.dtype)
        loss = optimiser.step(lambda: torch.tensor(2.0))
        assert loss.item() == 2.0
        now = [p.grad for p in params]
        norm, factor = optim.grad_norm(now, 0.5)
        assert_bitwise(optimiser.norm, norm, "norm")
        weyl = 0x9E3779B97F4A7C15
        optim.adamw_step(plans[0], now[:2], lr=1e-3, weight_decay=0.0, grad_factor=factor, seed=7)
        optim.adamw_step(plans[1], now[2:3], lr=1e-2, grad_factor=factor, seed=7 + 2 * weyl)
        optim.adamw_step(plans[2], now[3:], lr=1e-2, grad_factor=factor, seed=7 + 3 * weyl)
        for a, b in zip(params, twin):
            assert_bitwise(a, b, f"step {step}")
        optimiser.zero_grad()


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoints_resume_bit_for_bit(bits, tmp_path):
    sizes = [64, 1000, 33, 500]
    params, grads, _, _ = _model(sizes)
    params[1] = params[1].bfloat16()
    for p, g in zip(params, grads):
        p.requires_grad_(True)
        p.grad = g.to(p.dtype)
    optimiser = _optimiser(params, bits)
    optimiser.step()
    torch.save(optimiser.state_dict(), tmp_path / "state.pt")
    resumed = [p.detach().clone().requires_grad_(True) for p in params]
    for p, g in zip(resumed, grads):
        p.grad = g.to(p.dtype)
    other = _optimiser(resumed, bits)
    other.load_state_dict(torch.load(tmp_path / "state.pt", weights_only=True))
    assert other.state_dict()["state"].keys() == {0, 1, 2, 3}
    for o in (optimiser, other):
        o.param_groups[0]["lr"] = 5e-4
        o.step()
        o.step()
    for a, b in zip(params, resumed):
        assert_bitwise(a, b, "resumed")
    with pytest.raises(ValueError, match="bit moments"):
        _optimiser([p.detach().clone() for p in params], 40 - bits).load_state_dict(optimiser.state_dict())


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_move_keep_their_moments(bits):
    params, grads, _, _ = _model([100, 40])
    twin = [p.clone() for p in params]
    pair = []
    for group in (params, twin):
        for p, g in zip(group, grads):
            p.requires_grad_(True)
            p.grad = g
        pair.append(optim.AdamW(group, state_bits=bits))
    for o in pair:
        o.step()
    plan = next(iter(pair[0]._plans.values()))
    held = params[0].data
    params[0].data = held.clone()
    with pytest.raises(RuntimeError, match="moved"):
        optim.adamw_step(plan, grads, **HYPER)
    for o in pair:
        o.step()
    for a, b in zip(params, twin):
        assert_bitwise(a, b, "moved")


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("changed", [slice(0, 1), slice(0, 2)])
def test_parameters_of_another_dtype_keep_their_moments(bits, changed):
    params, grads, _, _ = _model([100, 40])
    for p, g in zip(params, grads):
        p.requires_grad_(True)
        p.grad = g
    optimiser = optim.AdamW(params, state_bits=bits)
    optimiser.step()
    before = optimiser.state_dict()["state"]
    for p in params[changed]:
        p.grad = None
        p.data = p.data.to(torch.bfloat16)
    optimiser.step()  # nothing for those that changed: their moments are as they were
    after = optimiser.state_dict()["state"]
    assert sorted(after) == [0, 1]
    assert not [key for key, plan in optimiser._plans.items() if not plan.params or plan.params[0].dtype != key[1]]
    for k, p in enumerate(params):
        kept = p.dtype == torch.bfloat16
        assert after[k]["step"] == before[k]["step"] + (0 if kept else 1)
        if kept:
            for name in before[k]:
                if name != "step":
                    assert_bitwise(after[k][name], before[k][name], name)
    for p, g in zip(params, grads):
        p.grad = g.to(p.dtype)
    optimiser.step()
    assert [part["step"] for _, part in sorted(optimiser.state_dict()["state"].items())] == \
        [2 if p.dtype == torch.bfloat16 else 3 for p in params]


def test_a_checkpoint_of_torch_is_taken_over():
    params, grads, _, _ = _model([64, 33])
    twin = [p.clone().requires_grad_(True) for p in params]
    theirs = torch.optim.AdamW(twin, lr=0.01)
    for p, g in zip(twin, grads):
        p.grad = g
    theirs.step()
    mine = [p.detach().clone().requires_grad_(True) for p in twin]
    optimiser = optim.AdamW(mine, lr=0.01)
    optimiser.load_state_dict(theirs.state_dict())
    for p, g in zip(mine, grads):
        p.grad = g
    optimiser.step()
    theirs.step()
    for a, b in zip(mine, twin):
        # both in float32: a step of at most 0.01 and its quotient of about ten roundings on each side
        assert_close_scaled(a.detach(), b.detach(), rtol=2e-7, scale=2e-7, what="taken over")


def test_gradients_of_any_layout_and_moments_that_are_replaced():
    p = torch.randn(8, 16, generator=torch.Generator().manual_seed(0)).to(DEV).requires_grad_(True)
    twin = p.detach().clone().requires_grad_(True)
    g = torch.randn(16, 8, device=DEV)
    pair = [optim.AdamW([t], max_norm=0.5) for t in (p, twin)]
    p.grad, twin.grad = g.t(), g.t().contiguous()
    for o in pair:
        o.step()
    assert_bitwise(p.detach(), twin.detach(), "transposed gradient")
    m, v = torch.zeros(100, device=DEV), torch.zeros(100, device=DEV)
    w = [torch.zeros(100, device=DEV)]
    plan = optim.adamw_plan(w, [m], [v])
    m.data = torch.full((100,), 7.0, device=DEV)
    optim.adamw_step(plan, [torch.ones(100, device=DEV)], **HYPER)
    assert (m == 7.0).all() and (plan.exp_avgs[0] > 0).all()  # the plan keeps the memory that it was given


def test_an_optimiser_is_saved_by_its_state():
    optimiser = optim.AdamW([torch.zeros(3, device=DEV, requires_grad=True)])
    with pytest.raises(TypeError, match="state_dict"):
        copy.deepcopy(optimiser)


def test_scheduler_and_copies():
    params, grads, _, _ = _model([64])
    p = params[0].requires_grad_(True)
    p.grad = grads[0]
    optimiser = optim.AdamW([p], lr=0.1)
    scheduler = torch.optim.lr_scheduler.StepLR(optimiser, 1, 0.5)
    optimiser.step()
    scheduler.step()
    assert optimiser.param_groups[0]["lr"] == 0.05
    saved = copy.deepcopy(optimiser.state_dict())
    assert saved["state"][0]["step"] == 1
