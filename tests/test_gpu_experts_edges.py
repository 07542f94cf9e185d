"""GPU tests of the expert operators where a sum is long, a value extreme or a segment far from the mean.

Sums of n equal terms in sequence: each addition is off by at most half a step of the running sum, so together at most
n 2^-25 of the result, here with every second-level addition counted too.
"""
from __future__ import annotations

import math

import pytest
import torch

from bysj_amd.kernels.block_norm import residual_norm
from bysj_amd.kernels.experts import ExpertPlan, expert_combine, expert_dispatch, expert_linear, expert_route
from oracle.experts import expert_dispatch_reference, expert_linear_reference
from parity import announce, assert_bitwise, assert_close_scaled

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _half(dtype):
    return 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------
# the gated SiLU's gradient between the products
# ---------------------------------------------------------------------------

def _gated_gradients(plan, experts, inner, k_in, n_out, dtype, *, from_tokens, seed):
    announce("expert linear, gated gradients", tuple(plan[2].shape), experts, inner, k_in, n_out, dtype, from_tokens)
    generator = torch.Generator().manual_seed(seed)
    entries = plan[2].shape[0] if from_tokens else plan[2].numel()
    x = torch.randn(entries, *inner, k_in, generator=generator).to(dtype)
    weight = (torch.randn(experts, 2 * n_out, k_in, generator=generator) * k_in ** -0.5).to(dtype)
    dy = torch.randn(plan[2].numel(), *inner, n_out, generator=generator).to(dtype)
    leaves = x.to(DEV).requires_grad_(True), weight.to(DEV).requires_grad_(True)
    y = expert_linear(*leaves, ExpertPlan(*(t.to(DEV) for t in plan)), from_tokens=from_tokens, activation="silu_gate")
    grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    _, *wanted = expert_linear_reference(x, weight, plan, from_tokens=from_tokens, activation="silu_gate", grad=dy)
    # dz in two parts: bfloat16 2^-18 of each product, float16 2^-24, or 2^-25 of the other operand
    operands = (weight.double().abs().sum((0, 1)), x.double().abs().reshape(-1, k_in).sum(0))
    for got, value, products, operand, what in zip(grads, wanted[:2], wanted[2:], operands, ("dx", "dweight")):
        budget = (1e-5 + _half(dtype)) * value.abs() + 1e-5 * value.abs().max()
        budget = budget + (2.0 ** -18 * products if dtype == BF16 else 2.0 ** -24 * products + 2.0 ** -25 * (1.0 + operand))
        error = (got.detach().cpu().double() - value).abs()
        assert bool((error <= budget).all()), (what, float((error - budget).max()), float(value.abs().max()))


def _random_plan(tokens, k, experts, seed):
    generator = torch.Generator().manual_seed(seed)
    chosen = torch.randint(0, experts, (tokens, k), generator=generator)
    chosen[torch.rand(tokens, generator=generator) < 0.1] = -1
    return expert_dispatch_reference(chosen, experts)


# loads by piece and straight to LDS, ragged and whole rows, every tile; sums of one slice, of several, of an odd number
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("k_in,n_out", [(1, 1), (3, 5), (16, 20), (32, 32), (33, 31), (64, 64), (90, 65), (128, 96), (130, 200), (264, 33)])
def test_gated_gradients_round_once(k_in, n_out, dtype):
    for from_tokens in (True, False):
        _gated_gradients(_random_plan(61, 3, 5, seed=k_in), 5, (), k_in, n_out, dtype, from_tokens=from_tokens, seed=n_out)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,k,experts,inner,k_in,n_out", [(900, 2, 3, (), 256, 264), (900, 2, 3, (), 266, 130), (1, 1, 1, (), 48, 40),
                                                               (3000, 1, 2, (3,), 64, 48), (40, 2, 200, (), 48, 70)])
def test_gated_gradients_of_plans(tokens, k, experts, inner, k_in, n_out, dtype):
    """Tiles of 256 by 256 and of 128, one token, segments that dW cuts, more experts than rows."""
    for from_tokens in (True, False):
        _gated_gradients(_random_plan(tokens, k, experts, seed=tokens), experts, inner, k_in, n_out, dtype, from_tokens=from_tokens, seed=k)


@pytest.mark.parametrize("dtype,k_in,n_out", [(BF16, 8, 6), (F16, 10, 48), (BF16, 16, 96)])
def test_gated_gradients_of_many_rows(dtype, k_in, n_out):
    """So many rows that a workgroup takes a run of tiles; sums of one, two and three slices a part."""
    generator = torch.Generator().manual_seed(n_out)
    chosen = torch.multinomial(torch.tensor([0.5, 0.0, 0.3, 0.01, 0.19]), 26_000, replacement=True, generator=generator)[:, None]
    chosen[torch.rand(26_000, generator=generator) < 0.02] = -1
    plan = tuple(t.cpu() for t in expert_dispatch(chosen.to(DEV), 5))
    for from_tokens in (True, False):
        _gated_gradients(plan, 5, (33,), k_in, n_out, dtype, from_tokens=from_tokens, seed=1)


@pytest.mark.parametrize("rows", [1, 40, 700])
def test_gated_gradients_past_float16(rows):
    """dy * up * slope of 1.8e5: past float16, while the gradients of x and of the matrix fit."""
    announce("expert linear, gated gradients past float16", rows)
    k_in = 256
    x = torch.full((rows, k_in), 0.3, dtype=F16)
    weight = torch.full((1, 2, k_in), 0.53, dtype=F16)
    weight[0, 0] = 0.026
    dy = torch.zeros(rows, 1, dtype=F16)
    dy[rows // 2] = 4000.0
    plan = expert_dispatch_reference(torch.zeros(rows, 1, dtype=torch.int64), 1)
    leaves = x.to(DEV).requires_grad_(True), weight.to(DEV).requires_grad_(True)
    y = expert_linear(*leaves, ExpertPlan(*(t.to(DEV) for t in plan)), activation="silu_gate")
    grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    _, want_x, want_w, _, _ = expert_linear_reference(x, weight, plan, activation="silu_gate", grad=dy)
    assert float(want_x.abs().max()) < 65504.0 and float(want_w.abs().max()) < 65504.0
    for got, wanted in zip(grads, (want_x, want_w)):
        assert_close_scaled(got, wanted, rtol=1e-5 + _half(F16), what="gradient")


# ---------------------------------------------------------------------------
# sums of long segments among short ones
# ---------------------------------------------------------------------------

def _one_segment(rows, experts, k_in, n_out, dtype, only):
    """dW where one expert has every row and all terms are equal."""
    announce("expert linear, one segment of many", rows, experts, k_in, n_out, dtype)
    plan = expert_dispatch(torch.full((rows, 1), only, device=DEV), experts)
    x = torch.full((rows, k_in), 0.7, device=DEV, dtype=dtype)
    x[:, 1::2] = -0.35
    weight = torch.zeros(experts, n_out, k_in, device=DEV, dtype=dtype, requires_grad=True)
    y = expert_linear(x, weight, plan, from_tokens=False)
    dy = torch.full_like(y, 0.3)
    (dw,) = torch.autograd.grad(y, weight, dy)
    row = rows * x[0].cpu().double() * float(dy[0, 0])
    assert int(dw[:only].count_nonzero()) == 0 and int(dw[only + 1:].count_nonzero()) == 0
    # at most 32,768 rows in sequence: 2,048 additions of 16-bit operands, 256 and 64 of float32
    assert_close_scaled(dw[only], row.expand(n_out, k_in), rtol=(320 if dtype == F32 else 2048) * 2.0 ** -25 + 2.0 ** -24 + _half(dtype),
                        scale=0.0, what="dweight")


@pytest.mark.parametrize("dtype,rows,experts,k_in,n_out", [(F32, 131_000, 4, 1024, 2048), (BF16, 4_190_000, 128, 256, 256), (F32, 1_000_000, 32, 256, 512),
                                                           (F32, 520_000, 1024, 64, 40), (F32, 256_000, 500, 64, 40), (BF16, 256_000, 500, 24, 40),
                                                           (F16, 256_001, 501, 25, 40)])
def test_one_segment_of_many_experts(dtype, rows, experts, k_in, n_out):
    """Cuts go by a segment's own length: the mean is below 32,768 rows here, or below 512."""
    _one_segment(rows, experts, k_in, n_out, dtype, experts // 2)


@pytest.mark.parametrize("k_in,n_out", [(24, 40), (1024, 1032)])
def test_segments_around_the_cut(k_in, n_out):
    """Segments of 0, 1, 32,767 to 32,769, 65,536 and 65,537 rows, cut and uncut side by side, gradients against 64 bits."""
    lengths = [32_769, 0, 65_537, 1, 32_768, 65_536, 32_767, 300, 0]
    announce("expert linear, segments around the cut", k_in, n_out)
    chosen = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
    chosen = chosen[torch.randperm(chosen.numel(), generator=torch.Generator().manual_seed(1))]
    plan = expert_dispatch(chosen[:, None].to(DEV), len(lengths))
    for dtype in (F32, BF16):
        generator = torch.Generator().manual_seed(2)
        x = torch.randn(chosen.numel(), k_in, generator=generator).to(dtype).to(DEV)
        weight = torch.randn(len(lengths), n_out, k_in, generator=generator).to(dtype).to(DEV).requires_grad_(True)
        y = expert_linear(x, weight, plan)
        dy = torch.randn(y.shape, generator=generator).to(dtype).to(DEV)
        (dw,) = torch.autograd.grad(y, weight, dy)
        offsets = plan.offsets.tolist()
        for e in range(len(lengths)):
            a, b = offsets[e], offsets[e + 1]
            wanted = dy[a:b].double().t() @ x[plan.order[a:b]].double()
            assert_close_scaled(dw[e], wanted, rtol=1e-5 + _half(dtype), what=f"dweight {e} {dtype}")


@pytest.mark.parametrize("rows", [1, 16, 24])
@pytest.mark.parametrize("gated", [False, True])
def test_long_sums_of_few_rows(rows, gated):
    """65,536 inputs in float32 for a few rows: as exact as in tiles."""
    announce("expert linear, long sums of few rows", rows, gated)
    plan = expert_dispatch(torch.zeros(rows, 1, dtype=torch.int64, device=DEV), 1)
    x = torch.full((rows, 65536), 0.7, device=DEV)
    weight = (torch.arange(1, 71, device=DEV, dtype=F32) * 0.0137)[None, :, None].expand(1, 70, 65536).contiguous()
    product = float(x[0, 0]) * weight[0, :, 0].cpu().double()
    z = (product * 65536).expand(rows, 70)
    # four waves' sums, each of 512 products and 32 of these in sequence
    rtol = (512 + 32 + 4) * 2.0 ** -25 + 2.0 ** -24
    if gated:
        y = expert_linear(x, weight, plan, activation="silu_gate")
        assert_close_scaled(y, z[:, :35] * torch.sigmoid(z[:, :35]) * z[:, 35:], rtol=2 * rtol + 2.0 ** -22, scale=0.0, what="y")
    else:
        assert_close_scaled(expert_linear(x, weight, plan), z, rtol=rtol, scale=0.0, what="y")


# ---------------------------------------------------------------------------
# NaN, infinities and the lowest values
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [True, False])
def test_route_nan_with_groups(scores, bias):
    """A NaN ranks behind every other logit and in front of what is masked, in its group and among the groups."""
    announce("expert route, NaN with groups", scores, bias)
    nan, out = math.nan, -math.inf
    rows = [
        # logits of three groups of three, the experts chosen of two groups
        ([out, out, out, nan, nan, nan, out, out, out], [3, 4, 5]),     # NaN before empty groups
        ([out, out, out, nan, nan, nan, 1.0, 2.0, 0.5], [7, 6, 8]),     # behind a group without it
        ([nan, 3.0, 1.0, 0.0, -1.0, -2.0, -3.0, -4.0, -5.0], [1, 2, 3]),
        ([nan, 3.0, nan, 0.0, -1.0, -2.0, -3.0, -4.0, -5.0], [3, 4, 5]),  # its two best keys hold a NaN
        ([nan] * 9, [0, 1, 2]),
        ([out] * 9, [-1, -1, -1]),
        ([out, nan, out, out, out, out, out, out, out], [1, -1, -1]),
    ]
    logits = torch.tensor([r for r, _ in rows], device=DEV)
    weights, experts, plan = expert_route(logits, 3, scores=scores, groups=3, top_groups=2, bias=torch.zeros(9, device=DEV) if bias else None)
    assert experts.tolist() == [e for _, e in rows]
    held = torch.tensor([[e >= 0 for e in chosen] for _, chosen in rows])
    weights = weights.cpu()
    assert bool((weights[~held] == 0.0).all())
    for row in (0, 4, 6):
        assert bool(torch.isnan(weights[row][held[row]]).all())
    if scores == "softmax":    # one NaN is in every score of its row
        assert bool(torch.isnan(weights[:5]).all())
    assert plan.slots.cpu().ge(0).equal(held)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_nan_ranks_last_with_a_bias(scores):
    announce("expert route, NaN with a bias", scores)
    logits = torch.tensor([[math.nan, 1.0, 3.0, 2.0], [1.0, math.nan, -50.0, math.nan], [math.nan, -math.inf, 0.0, -math.inf],
                           [0.0, math.nan, 1.0, 2.0]], device=DEV)
    _, experts, _ = expert_route(logits, 3, scores=scores, bias=torch.zeros(4, device=DEV))
    assert experts.tolist() == [[2, 3, 1], [0, 2, 1], [2, 0, -1], [3, 2, 0]]
    # a bias of -inf takes an expert out, whatever its logit
    _, experts, _ = expert_route(logits, 4, scores=scores, bias=torch.tensor([0.0, -math.inf, 0.0, 0.0], device=DEV))
    assert experts.tolist() == [[2, 3, 0, -1], [0, 2, 3, -1], [2, 0, -1, -1], [3, 2, 0, -1]]


@pytest.mark.parametrize("kwargs", [{}, {"bias": torch.zeros(6)}, {"groups": 2}])
def test_route_infinite_logits_rank_first(kwargs):
    announce("expert route, +inf")
    logits = torch.tensor([[0.0, 1.0, math.inf, 2.0, -1.0, 5.0], [0.0, math.inf, 1.0, -math.inf, math.nan, math.inf]], device=DEV)
    on = {n: v.to(DEV) if isinstance(v, torch.Tensor) else v for n, v in kwargs.items()}
    weights, experts, _ = expert_route(logits, 2, **on)
    assert experts[:, 0].tolist() == [2, 1] and int(experts[1, 1]) == 5
    assert bool(torch.isnan(weights).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_gates_of_the_largest_size(dtype):
    """Gates of the type's lowest and largest value, as a mask leaves them: off and on, with slopes of 0 and 1."""
    announce("gates of the largest size", dtype)
    most = torch.finfo(dtype).max
    gate = torch.tensor([[-most, most, -1e4, 1e4, -200.0, 200.0, -most / 3, most / 3]], dtype=dtype, device=DEV).requires_grad_(True)
    x = torch.full_like(gate, 2.0 ** -20)
    for activation, value, slope in (("sigmoid", (gate > 0).double(), torch.zeros_like(gate).double()),
                                     ("silu", torch.where(gate > 0, gate, 0.0).double(), (gate > 0).double())):
        h, _ = residual_norm(x.detach(), torch.zeros_like(x), gate=gate, gate_activation=activation, post_norm=False, pre_norm=False)
        (grad,) = torch.autograd.grad(h, gate, torch.ones_like(h))
        for got, wanted in ((h, value), (grad, slope)):
            wanted = wanted.detach().cpu() * 2.0 ** -20
            error = (got.detach().cpu().double() - wanted).abs()
            assert bool((error <= (1e-5 + _half(dtype)) * wanted.abs() + 1e-30 + (2.0 ** -25 if dtype == F16 else 0.0)).all()), (activation, error)


@pytest.mark.parametrize("rows", [1, 40])
def test_gated_product_of_the_largest_gates(rows):
    """z of (+-3e38, 2^-20): silu(-3e38) is 0, and so is its slope."""
    announce("expert linear, gates of the largest size", rows)
    plan = expert_dispatch(torch.zeros(rows, 1, dtype=torch.int64, device=DEV), 1)
    for sign in (-1.0, 1.0):
        x = torch.ones(rows, 1, device=DEV, requires_grad=True)
        weight = torch.tensor([[[sign * 3e38], [2.0 ** -20]]], device=DEV, requires_grad=True)
        y = expert_linear(x, weight, plan, activation="silu_gate")
        (dw,) = torch.autograd.grad(y, weight, torch.full_like(y, 2.0 ** -10))
        on = 0.0 if sign < 0 else 1.0
        assert_close_scaled(y, torch.full((rows, 1), on * 3e38 * 2.0 ** -20, dtype=torch.float64), scale=0.0, what="y")
        wanted = torch.tensor([[[on * 2.0 ** -30], [on * 3e38 * 2.0 ** -10]]], dtype=torch.float64) * rows
        assert_close_scaled(dw, wanted, scale=0.0, what="dweight")


# ---------------------------------------------------------------------------
# runs of tiles
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,tokens,k_in,n_out,gated", [
    (F32, 64_003, 70, 128, False),      # 3 slices forward, 4 in dx; runs of 8
    (F32, 97_003, 100, 40, False),      # narrow columns; 4 slices forward, 2 in dx
    (BF16, 32_803, 150, 256, False),    # two columns of tiles; 3 and 4 slices
    (F16, 66_003, 256, 128, False),
    (BF16, 64_003, 140, 48, True),      # 3 slices forward, 2 of each part in dx
])
def test_runs_of_eight_tiles(dtype, tokens, k_in, n_out, gated):
    """Sums of up to four slices over so many rows that a workgroup takes eight tiles; an odd number of slices is padded."""
    announce("expert linear, runs of eight", tokens, k_in, n_out, dtype, gated)
    inner, experts = 33, 5
    generator = torch.Generator().manual_seed(k_in)
    chosen = torch.multinomial(torch.tensor([0.4, 0.0, 0.35, 0.01, 0.24]), tokens, replacement=True, generator=generator)[:, None]
    chosen[torch.rand(tokens, generator=generator) < 0.02] = -1
    plan = expert_dispatch(chosen.to(DEV), experts)
    offsets = plan.offsets.tolist()
    torch.manual_seed(n_out)
    for from_tokens in (True, False):
        x = torch.randn(tokens, inner, k_in, device=DEV).to(dtype).requires_grad_(True)
        weight = (torch.randn(experts, n_out * (2 if gated else 1), k_in, device=DEV) * k_in ** -0.5).to(dtype).requires_grad_(True)
        y = expert_linear(x, weight, plan, from_tokens=from_tokens, activation="silu_gate" if gated else None)
        dy = torch.randn_like(y)
        dx, dw = torch.autograd.grad(y, (x, weight), dy)
        rule = 1e-5 + _half(dtype)
        for e in range(experts):
            a, b = offsets[e], offsets[e + 1]
            at = plan.order[a:b] if from_tokens else slice(a, b)
            rows, matrix = x.detach()[at].double().view(-1, k_in), weight.detach()[e].double()
            dz = dy[a:b].double().view(-1, n_out)
            z = rows @ matrix.t()
            if gated:
                gate, up = z[:, :n_out], z[:, n_out:]
                s = torch.sigmoid(gate)
                dz = torch.cat([dz * up * s * (1.0 + gate * (1.0 - s)), dz * gate * s], 1)
                z = gate * s * up
            for got, wanted, what in ((y[a:b].reshape(-1, n_out), z, "y"), (dx[at].reshape(-1, k_in), dz @ matrix, "dx"), (dw[e], dz.t() @ rows, "dweight")):
                if wanted.numel() == 0:
                    continue
                # a gated dz loses 2^-18 of each of its products, at random signs as these have: 2^-18 of the root of the
                # sum of their squares, which the largest value is past; 16 deviations
                budget = rule * wanted.abs() + (1e-5 + (2.0 ** -14 if gated else 0.0)) * wanted.abs().max() + 2.0 ** -25
                error = (got.detach().double() - wanted).abs()
                assert bool((error <= budget).all()), (what, e, float((error - budget).max()))
        held = offsets[-1]
        assert int(y[held:].count_nonzero()) == 0
        if from_tokens:
            assert int(dx[(plan.slots[:, 0] < 0)].count_nonzero()) == 0
        else:
            assert int(dx[held:].count_nonzero()) == 0
        del x, y, dy, dx


# ---------------------------------------------------------------------------
# the weighted sum
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [40_000, 1_000_003, 4_194_304])
def test_long_sums_of_weights_gradients(dtype, size):
    """The gradient of a weight, a dot product of entries of up to 4M equal elements, at the rule of float32."""
    announce("expert combine, long sums", size, dtype)
    plan = expert_dispatch(torch.tensor([[0], [1], [0]], device=DEV), 2)
    y = torch.full((3, size), 0.7, device=DEV, dtype=dtype)
    weights = torch.ones(3, 1, device=DEV, requires_grad=True)
    out = expert_combine(y, weights, plan)
    dout = torch.full_like(out, 0.3)
    (grad,) = torch.autograd.grad(out, weights, dout)
    wanted = torch.full((3, 1), size * float(y[0, 0]) * float(dout[0, 0]), dtype=torch.float64)
    assert_close_scaled(grad, wanted, scale=0.0, what="dweights")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,inner", [(0, ()), (4, (0,))])
def test_gated_products_of_nothing(tokens, inner, dtype):
    """No tokens, and entries without rows: empty results, matrices' gradients of 0."""
    announce("expert linear, gated, empty", tokens, inner, dtype)
    plan = expert_dispatch(torch.zeros(tokens, 2, dtype=torch.int64, device=DEV), 3)
    for from_tokens in (True, False):
        x = torch.zeros(tokens if from_tokens else 2 * tokens, *inner, 5, device=DEV, dtype=dtype, requires_grad=True)
        weight = torch.ones(3, 14, 5, device=DEV, dtype=dtype, requires_grad=True)
        y = expert_linear(x, weight, plan, from_tokens=from_tokens, activation="silu_gate")
        assert y.shape == (2 * tokens, *inner, 7)
        dx, dw = torch.autograd.grad(y, (x, weight), torch.zeros_like(y))
        assert dx.shape == x.shape and dw.shape == weight.shape and int(dw.count_nonzero()) == 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,k_in,n_out", [(60, 40, 24), (900, 256, 264)])
def test_gated_gradients_keep_to_their_places(tokens, k_in, n_out, dtype):
    """NaN and infinities of rows of no place reach no gradient, and one gradient alone is that of both."""
    announce("expert linear, gated, NaN, single gradients", tokens, k_in, n_out, dtype)
    generator = torch.Generator().manual_seed(tokens)
    chosen = torch.randint(0, 3, (tokens, 2), generator=generator)
    chosen[torch.rand(tokens, generator=generator) < 0.3] = -1
    plan = expert_dispatch(chosen.to(DEV), 3)
    held, out = int(plan.offsets[-1]), (chosen < 0).all(1)
    weight = (torch.randn(3, 2 * n_out, k_in, generator=generator) * k_in ** -0.5).to(dtype).to(DEV)
    dy = torch.randn(2 * tokens, n_out, generator=generator).to(dtype)
    dirty_dy = dy.clone()
    dirty_dy[held:] = math.inf
    for from_tokens in (True, False):
        x = torch.randn(tokens if from_tokens else 2 * tokens, k_in, generator=generator).to(dtype)
        dirty = x.clone()
        dirty[out if from_tokens else slice(held, None)] = math.nan
        results = []
        for rows, seed, wanted in ((x, dy, (True, True)), (dirty, dirty_dy, (True, True)), (x, dy, (True, False)), (x, dy, (False, True))):
            leaves = [t.clone().requires_grad_(w) for t, w in zip((rows.to(DEV), weight), wanted)]
            y = expert_linear(*leaves, plan, from_tokens=from_tokens, activation="silu_gate")
            grads = torch.autograd.grad(y, [t for t, w in zip(leaves, wanted) if w], seed.to(DEV))
            results.append((y.detach(), *grads))
        for a, b in zip(results[0], results[1]):
            assert_bitwise(a, b)
        assert_bitwise(results[0][1], results[2][1])
        assert_bitwise(results[0][2], results[3][1])


def test_gated_gradients_past_32_bits():
    """A dz whose parts are of 4.9 GB each: rows on both sides of 2^31 and 2^32 bytes, and sums over all."""
    tokens, k_in, n_out = 600_003, 16, 2048
    announce("expert linear, gated, dz of twice 4.9 GB", tokens, k_in, n_out)
    torch.manual_seed(0)
    x = torch.randn(tokens, k_in, device=DEV).to(BF16).requires_grad_(True)
    weight = (torch.randn(2, 2 * n_out, k_in, device=DEV) * k_in ** -0.5).to(BF16).requires_grad_(True)
    plan = expert_dispatch((torch.arange(tokens, device=DEV) % 2)[:, None].contiguous(), 2)
    y = expert_linear(x, weight, plan, activation="silu_gate")
    dy = torch.randn_like(y)
    dx, dw = torch.autograd.grad(y, (x, weight), dy)

    def dz_of(rows, matrix, grad):
        z = rows @ matrix.t()
        gate, up = z[:, :n_out], z[:, n_out:]
        s = torch.sigmoid(gate)
        return torch.cat([grad * up * s * (1.0 + gate * (1.0 - s)), grad * gate * s], 1)

    rule = 1e-5 + _half(BF16)
    for e in range(2):
        matrix, begin, end = weight.detach()[e].double(), int(plan.offsets[e]), int(plan.offsets[e + 1])
        wanted = torch.zeros(2 * n_out, k_in, dtype=torch.float64, device=DEV)
        for first in range(begin, end, 50_000):
            places = slice(first, min(first + 50_000, end))
            at = plan.order[places]
            rows = x.detach()[at].double()
            dz = dz_of(rows, matrix, dy[places].double())
            wanted += dz.t() @ rows
            want_x = dz @ matrix
            # 2^-18 of each product, at most 2^-18 of their magnitudes
            budget = rule * want_x.abs() + 1e-5 * want_x.abs().max() + 2.0 ** -18 * (dz.abs() @ matrix.abs())
            assert bool(((dx[at].double() - want_x).abs() <= budget).all()), f"dx of places from {first}"
        error = (dw[e].double() - wanted).abs()
        # roundings of 2^-18 at random signs over 300,000 products of random sign: 16 deviations
        assert bool((error <= rule * wanted.abs() + (1e-5 + 2.0 ** -14) * wanted.abs().max()).all()), float(error.max())
