"""GPU parity of the group norm, forward and backward, against its definition in 64 bits.

Tolerances.  float32: the repository's rule, 1e-5 of the value plus 1e-5 of the
largest (about 170 roundings of 2^-24; the chain has about ten, and sums of up
to a few hundred terms per thread before they continue in 64 bits).  A mean far
from 0 adds the rounding of the mean itself, 2^-24 |mean| rstd |scale|.  16-bit
outputs add half a step, eps / 2 of the value.
"""
from __future__ import annotations

import itertools

import pytest
import torch

from bysj_amd.kernels import _C
from bysj_amd.kernels.group_norm import group_norm
from oracle.group_norm import group_norm_backward_reference, group_norm_reference
from parity import announce, assert_bitwise, assert_close_scaled

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _rtol(dtype):
    return 1e-5 + (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)


def _inputs(shape, dtype, seed=0, mean=0.5, affine=True):
    generator = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=generator) * 1.5 + mean).to(dtype)
    grad = torch.randn(shape, generator=generator).to(dtype)
    if not affine:
        return x, grad, None, None
    return x, grad, torch.rand(shape[-1], generator=generator) + 0.5, torch.randn(shape[-1], generator=generator)


def _offsets(lengths):
    return torch.tensor([0, *itertools.accumulate(lengths)], dtype=torch.int64)


def _on(t):
    return None if t is None else t.to(DEV)


def _check(x, grad, groups, scale, bias, offsets, activation, *, scale_of_bound=1e-5, max_rows=None, what=""):
    announce("group norm", what, tuple(x.shape), x.dtype, groups, activation)
    leaves = [_on(t) for t in (x, scale, bias)]
    for t in leaves:
        if t is not None:
            t.requires_grad_(True)
    y = group_norm(leaves[0], groups, leaves[1], leaves[2], offsets=_on(offsets), max_rows=max_rows, eps=1e-5,
                   activation=activation)
    given = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, given, _on(grad))
    rtol = _rtol(x.dtype)
    assert y.dtype == x.dtype and y.shape == x.shape
    assert_close_scaled(y, group_norm_reference(x, groups, scale, bias, offsets, 1e-5, activation), rtol=rtol,
                        scale=scale_of_bound, what=f"{what} y")
    wanted = group_norm_backward_reference(grad, x, groups, scale, bias, offsets, 1e-5, activation)
    assert_close_scaled(grads[0], wanted[0], rtol=rtol, scale=scale_of_bound, what=f"{what} grad_x")
    present = [(name, expected) for name, leaf, expected in zip(("scale", "bias"), leaves[1:], wanted[1:]) if leaf is not None]
    for (name, expected), actual in zip(present, grads[1:]):
        assert actual.dtype == torch.float32
        assert_close_scaled(actual, expected, scale=scale_of_bound, what=f"{what} grad_{name}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("channels,groups", [(1, 1), (2, 1), (3, 3), (5, 1), (8, 2), (12, 4), (64, 8), (64, 64), (90, 6),
                                             (96, 1), (130, 13), (513, 3), (520, 65), (1030, 2), (4095, 5), (4096, 32)])
def test_widths(channels, groups, dtype):
    """Every width: whole and ragged vectors, periods within and beyond a workgroup, groups inside and across vectors."""
    lengths = [1, 0, 7, 2, 29]
    x, grad, scale, bias = _inputs((sum(lengths), channels), dtype, seed=channels)
    _check(x, grad, groups, scale, bias, _offsets(lengths), "silu", what="widths")


@pytest.mark.parametrize("lengths", [[1], [0, 0, 1, 0], [1] * 70, [0, 300, 1, 0, 0, 2999, 5, 0], [40000], [3] * 4000,
                                     [20000, 1, 1, 1, 0, 15000, 2]])
@pytest.mark.parametrize("inner", [1, 3])
def test_samples_of_any_length(lengths, inner):
    x, grad, scale, bias = _inputs((sum(lengths), inner, 24), torch.float32, seed=len(lengths))
    _check(x, grad, 4, scale, bias, _offsets(lengths), "silu", what=str(lengths[:4]))
    _check(x, grad, 4, scale, bias, _offsets(lengths), None, max_rows=max(lengths), what=str(lengths[:4]))


@pytest.mark.parametrize("max_rows", [None, 0, 1, 40, 10**9])
def test_a_wrong_longest_sample_changes_nothing_but_the_schedule(max_rows):
    lengths = [1, 40, 0, 3000, 12, 700]
    x, grad, scale, bias = _inputs((sum(lengths), 32), torch.float32)
    _check(x, grad, 4, scale, bias, _offsets(lengths), "silu", max_rows=max_rows, what="max_rows")


@pytest.mark.parametrize("shape", [(1, 1, 64), (64, 64), (64, 1, 64), (5, 1000, 32), (2, 9, 7, 48), (1, 100000, 8), (0, 4, 8), (4, 0, 8)])
def test_entries_as_samples(shape):
    x, grad, scale, bias = _inputs(shape, torch.float32)
    _check(x, grad, 8, scale, bias, None, "silu", what="dense")


@pytest.mark.parametrize("activation", [None, "silu"])
def test_without_scale_and_bias(activation):
    x, grad, _, _ = _inputs((100, 48), torch.float32, affine=False)
    _check(x, grad, 3, None, None, _offsets([10, 60, 30]), activation, what="plain")
    scale = torch.rand(48) + 0.5
    _check(x, grad, 3, scale, None, _offsets([10, 60, 30]), activation, what="scale alone")
    _check(x, grad, 3, None, scale, _offsets([10, 60, 30]), activation, what="bias alone")


@pytest.mark.parametrize("mean", [30.0, -1000.0])
def test_means_far_from_zero(mean):
    lengths = [5000, 3, 800]
    x, grad, scale, bias = _inputs((sum(lengths), 40), torch.float32, mean=mean)
    # h is off by the rounding of the mean, 2^-24 |mean| / std, on values of up to about 4 (|grad_x| / rstd likewise)
    bound = 1e-5 + 2.0 ** -24 * abs(mean) * 4
    _check(x, grad, 5, scale, bias, _offsets(lengths), "silu", scale_of_bound=bound, what="far mean")


def test_rows_of_no_sample_give_zero():
    """A padded batch: rows before the first and behind the last sample are 0 in y and in the gradient, and count nowhere."""
    for channels in (7, 32):
        x, grad, scale, bias = _inputs((5000, 2, channels), torch.float32)
        x[:9], x[4000:] = float("nan"), float("inf")
        _check(x, grad, 1, scale, bias, torch.tensor([9, 9, 30, 4000]), "silu", what="padded")
        y = group_norm(x.to(DEV), 1, offsets=torch.tensor([9, 9, 30, 4000], device=DEV))
        assert not y[:9].any() and not y[4000:].any()
        nothing = group_norm(x.to(DEV), 1, offsets=torch.tensor([0], device=DEV))
        assert not nothing.any()


def test_malformed_offsets_stay_in_bounds():
    """Decreasing or far offsets give wrong values, never an access outside the tensors (offsets are clamped)."""
    x = torch.randn(200, 16, device=DEV)
    for offsets in ([0, 150, 40, 200], [-5, 1 << 40, 3, -7], [500, 600]):
        y = group_norm(x, 2, offsets=torch.tensor(offsets, device=DEV))
        assert y.shape == x.shape
    torch.cuda.synchronize()


def test_constant_and_nonfinite_samples():
    """A constant sample gives the bias; a NaN or infinity stays in its own sample and group."""
    for rows, channels, groups, value in ((30, 8, 2, 3.25), (77, 15, 3, 0.1), (5000, 30, 2, -1.7e5), (40000, 7, 7, 1e-3)):
        x = torch.full((rows, channels), value)
        bias = torch.arange(float(channels), device=DEV)
        y = group_norm(x.to(DEV), groups, None, bias, offsets=torch.tensor([0, rows], device=DEV))
        assert_bitwise(y, bias.cpu().expand(rows, channels), "constant")
    x = torch.randn(30, 8)
    clean = group_norm(x.to(DEV), 2, offsets=torch.tensor([0, 10, 20, 30], device=DEV))
    x[12, 5] = float("nan")
    x[25, 1] = float("inf")
    y = group_norm(x.to(DEV), 2, offsets=torch.tensor([0, 10, 20, 30], device=DEV)).cpu()
    hit = torch.zeros(30, 8, dtype=torch.bool)
    hit[10:20, 4:] = True
    hit[20:, :4] = True
    assert torch.isnan(y[hit]).all()
    assert_bitwise(y[~hit], clean.cpu()[~hit], "others")


@pytest.mark.parametrize("dtype,offset", [(torch.float32, 1), (torch.float16, 1), (torch.bfloat16, 3)])
def test_tensors_that_start_anywhere(dtype, offset):
    """Contiguous views at odd element offsets, also of the gradient."""
    lengths = [3, 70, 500]
    rows, channels = sum(lengths), 33
    x, grad, scale, bias = _inputs((rows, channels), dtype)
    held = [torch.zeros(rows * channels + 8, dtype=dtype, device=DEV) for _ in range(2)]
    views = [h[offset: offset + rows * channels].view(rows, channels) for h in held]
    views[0].copy_(x)
    views[1].copy_(grad)
    offsets = _on(_offsets(lengths))
    y, statistics = _C.group_norm_forward(views[0], 3, _on(scale), _on(bias), offsets, 1e-5, True)
    grads = _C.group_norm_backward(views[1], views[0], 3, _on(scale), _on(bias), offsets, statistics, True)
    assert_close_scaled(y, group_norm_reference(x, 3, scale, bias, _offsets(lengths), 1e-5, "silu"), rtol=_rtol(dtype))
    wanted = group_norm_backward_reference(grad, x, 3, scale, bias, _offsets(lengths), 1e-5, "silu")
    for actual, expected in zip(grads, wanted):
        assert_close_scaled(actual, expected, rtol=_rtol(dtype))


def test_gradients_wanted_one_by_one_equal_those_wanted_together():
    lengths = [100, 7, 4000]
    x, grad, scale, bias = (t.to(DEV) for t in _inputs((sum(lengths), 24), torch.float32))
    offsets = _on(_offsets(lengths))
    _, statistics = _C.group_norm_forward(x, 4, scale, bias, offsets, 1e-5, True)
    every = _C.group_norm_backward(grad, x, 4, scale, bias, offsets, statistics, True)
    for k, name in enumerate(("want_x", "want_scale", "want_bias")):
        wants = {n: n == name for n in ("want_x", "want_scale", "want_bias")}
        alone = _C.group_norm_backward(grad, x, 4, scale, bias, offsets, statistics, True, **wants)
        assert [a is None for a in alone] == [i != k for i in range(3)]
        assert_bitwise(alone[k], every[k], name)


def test_runs_are_bitwise_the_same_and_gradients_of_strided_outputs_work():
    lengths = [1000, 1, 30000, 60]
    x, grad, scale, bias = (t.to(DEV).requires_grad_(True) for t in _inputs((sum(lengths), 64), torch.float32))
    offsets = _on(_offsets(lengths))

    def once():
        y = group_norm(x, 8, scale, bias, offsets=offsets, activation="silu")
        return (y, *torch.autograd.grad(y.t(), (x, scale, bias), grad.detach().t()))

    first = once()
    for _ in range(3):
        for a, b in zip(first, once()):
            assert_bitwise(a, b, "again")


def test_gradients_against_differences():
    """The kernels' gradients against central differences of the oracle in 64 bits."""
    lengths = [4, 0, 9]
    x, grad, scale, bias = _inputs((13, 6), torch.float32, seed=3)
    offsets = _offsets(lengths)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, scale, bias)]
    y = group_norm(leaves[0], 2, leaves[1], leaves[2], offsets=offsets.to(DEV), activation="silu")
    grads = torch.autograd.grad(y, leaves, grad.to(DEV))
    step = 1e-5
    for which, (leaf, got) in enumerate(zip((x, scale, bias), grads)):
        differences = torch.zeros(leaf.numel(), dtype=torch.float64)
        for i in range(leaf.numel()):
            values = []
            for sign in (1.0, -1.0):
                args = [x.double(), scale.double(), bias.double()]
                moved = args[which].clone().view(-1)
                moved[i] += sign * step
                args[which] = moved.view(leaf.shape)
                values.append((group_norm_reference(args[0], 2, args[1], args[2], offsets, 1e-5, "silu") * grad.double()).sum())
            differences[i] = (values[0] - values[1]) / (2 * step)
        # differences are off by about step^2 * third derivative + 1e-16 / step: 1e-9; the rest is the float32 rule
        assert_close_scaled(got.reshape(-1), differences, what=f"leaf {which}")


def test_captured_graphs_replay_the_eager_results():
    """Forward and backward in two graphs of the same shapes, replayed in turn with new values in between."""
    lengths = [50, 4000, 0, 3]
    offsets = _on(_offsets(lengths))
    cases = []
    for seed in (1, 2):
        x, grad, scale, bias = (t.to(DEV) for t in _inputs((sum(lengths), 40), torch.float32, seed=seed))
        cases.append((x, grad, scale, bias))

    def both(x, grad, scale, bias):
        y, statistics = _C.group_norm_forward(x, 4, scale, bias, offsets, 1e-5, True)
        return (y, *_C.group_norm_backward(grad, x, 4, scale, bias, offsets, statistics, True))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for case in cases:
            both(*case)
    torch.cuda.current_stream().wait_stream(stream)
    graphs = []
    for case in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(*case)
        graphs.append((graph, out))
    for turn in range(4):
        for case in cases:
            case[0].add_(0.25 * turn)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for case, (_, out) in zip(cases, graphs):
            for a, b in zip(out, both(*case)):
                assert_bitwise(a, b, f"replay {turn}")


def test_another_stream():
    x, grad, scale, bias = (t.to(DEV) for t in _inputs((5000, 32), torch.float32))
    wanted = group_norm(x.view(5, 1000, 32), 4, scale, bias)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y = group_norm(x.view(5, 1000, 32), 4, scale, bias)
    stream.synchronize()
    assert_bitwise(y, wanted, "stream")


def test_inference_mode_and_empty_batches():
    with torch.inference_mode():
        y = group_norm(torch.randn(10, 16, device=DEV), 2)
    assert y.shape == (10, 16)
    x = torch.zeros(0, 16, device=DEV, requires_grad=True)
    scale = torch.ones(16, device=DEV, requires_grad=True)
    y = group_norm(x, 2, scale, offsets=torch.zeros(4, dtype=torch.int64, device=DEV))
    grads = torch.autograd.grad(y, (x, scale), torch.zeros_like(y))
    assert grads[0].shape == (0, 16) and not grads[1].any()


def test_launch_rows():
    """Grids of more than one row of blocks."""
    from bysj_amd.kernels import _lib

    lengths = [3] * 5000
    x, grad, scale, bias = _inputs((sum(lengths), 40), torch.float32)
    library = _lib.load()
    assert library.dpa4k_set_launch_row_limit(7) == _lib.OK
    try:
        _check(x, grad, 4, scale, bias, _offsets(lengths), "silu", what="rows of blocks")
    finally:
        assert library.dpa4k_set_launch_row_limit(0) == _lib.OK


def test_offsets_past_32_bits():
    """2.4e9 elements in bfloat16 (4.8 GB): the last sample lies behind 2^32 bytes and 2^31 elements."""
    rows, channels = 37_500_000, 64
    x = torch.zeros(rows, channels, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(5000, channels, generator=torch.Generator().manual_seed(0)).bfloat16()
    x[-5000:] = tail.to(DEV)
    offsets = torch.tensor([0, 1, rows - 5000, rows], device=DEV)
    y = group_norm(x, 8, offsets=offsets, activation="silu")
    wanted = group_norm_reference(tail, 8, activation="silu", offsets=torch.tensor([0, 5000]))
    assert_close_scaled(y[-5000:], wanted, rtol=_rtol(torch.bfloat16))
    assert not y[:-5000].any()
