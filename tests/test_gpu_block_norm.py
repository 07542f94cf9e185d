"""GPU parity of the norms around a block, forward and backward, against their definition in 64 bits.

Tolerances.  float32: the repository's rule, 1e-5 of the value plus 1e-5 of the
largest (about 170 roundings of 2^-24; the chain has some twenty and sums of
up to 8,192 terms in trees of at most 32 in sequence).  16-bit outputs add half
a step, eps / 2 of the value, and a subnormal step of float16, 2^-25.  Sums over
rows are float32 whatever the inputs' type.

grad_x is a difference, r (v - x r mean(v x r)), which comes out far below its
operands where one channel holds most of a row (always in a row of one channel,
where it is v eps r^3).  Each operand is the result of at most 40 roundings of
2^-24 (the chain up to v has some twenty, the mean a tree of as many again), so
the difference may be off by 40 * 2^-24 of their magnitudes, whatever is left.
"""
from __future__ import annotations

import pytest
import torch

from bysj_amd.kernels.block_norm import residual_norm
from oracle.block_norm import residual_norm_backward_reference, residual_norm_grad_x_operands, residual_norm_reference
from parity import announce, assert_bitwise, assert_close_scaled

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _rtol(dtype):
    return 1e-5 + (0.0 if dtype == F32 else torch.finfo(dtype).eps / 2)


def _case(shape, dtype, stream, *, gate=None, activation=None, post=True, pre=True, scale="channels", seed=0):
    generator = torch.Generator().manual_seed(seed)

    def normal(size, by, kind):
        return (torch.randn(size, generator=generator) * by).to(kind)

    c = shape[-1]
    kwargs = {"gate": None if gate is None else normal(shape if gate == "full" else (*shape[:-1], 1), 1.5, dtype),
              "post_scale": torch.rand(c, generator=generator) + 0.5 if post else None,
              "pre_scale": torch.rand(c, generator=generator) + 0.5 if pre else None,
              "residual_scale": torch.rand(c, generator=generator) * 0.5 if scale == "channels" else scale}
    tensors = {"x": normal(shape, 2.0, dtype), "residual": normal(shape, 3.0, stream), "dh": normal(shape, 0.5, stream),
               "dy": normal(shape, 1.0, dtype)}
    return tensors, kwargs, {"gate_activation": activation, "post_norm": post, "pre_norm": pre, "eps": 1e-6}


def _on(value):
    return value.to(DEV).requires_grad_(True) if isinstance(value, torch.Tensor) else value


def _check(tensors, kwargs, options, what=""):
    x, residual = tensors["x"], tensors["residual"]
    announce("residual norm", what, tuple(x.shape), x.dtype, residual.dtype, options)
    leaves = {"x": _on(x), "residual": _on(residual), **{name: _on(value) for name, value in kwargs.items()}}
    h, y = residual_norm(leaves["x"], leaves["residual"], **{name: leaves[name] for name in kwargs}, **options)
    want_h, want_y = residual_norm_reference(x, residual, **kwargs, **options)
    assert h.dtype == residual.dtype and h.shape == x.shape
    assert_close_scaled(h, want_h, rtol=_rtol(h.dtype), what=f"{what} h")
    outputs, seeds = [h], [tensors["dh"].to(DEV)]
    if options["pre_norm"]:
        assert y.dtype == x.dtype and y.shape == x.shape
        assert_close_scaled(y, want_y, rtol=_rtol(y.dtype), what=f"{what} y")
        outputs, seeds = [h, y], [*seeds, tensors["dy"].to(DEV)]
    else:
        assert y is None
    names = [name for name in ("x", "residual", "gate", "post_scale", "residual_scale", "pre_scale")
             if isinstance(leaves[name], torch.Tensor)]
    grads = torch.autograd.grad(outputs, [leaves[name] for name in names], seeds)
    wanted = residual_norm_backward_reference(tensors["dh"], tensors["dy"], x, residual, **kwargs, **options)
    wanted = dict(zip(("x", "residual", "gate", "post_scale", "residual_scale", "pre_scale"), wanted))
    for name, grad in zip(names, grads):
        assert grad.dtype == leaves[name].dtype and grad.shape == leaves[name].shape
        if name == "x" and x.shape[-1] == 1 and options["post_norm"]:
            operands = residual_norm_grad_x_operands(tensors["dh"], tensors["dy"], x, residual, **kwargs, **options)
            budget = _rtol(grad.dtype) * wanted[name].abs() + 40 * 2.0 ** -24 * operands + (2.0 ** -25 if grad.dtype == F16 else 0.0)
            assert bool(((grad.cpu().double() - wanted[name]).abs() <= budget).all()), f"{what} grad_x"
            continue
        assert_close_scaled(grad, wanted[name], rtol=_rtol(grad.dtype), what=f"{what} grad_{name}")


# every layout of a row (8 to 64 lanes, a workgroup of 256 and 512), whole and ragged chunks, both ends of each
@pytest.mark.parametrize("dtype,stream", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("width", [1, 2, 7, 8, 63, 64, 65, 90, 128, 129, 250, 256, 257, 511, 512, 513, 810, 1024, 1025, 2047, 2049,
                                   4096, 4099, 8191, 8192])
def test_widths(width, dtype, stream):
    _check(*_case((5, width), dtype, stream, gate="full", activation="sigmoid", seed=width), "widths")


@pytest.mark.parametrize("gate,activation", [(None, None), ("full", None), ("full", "silu"), ("row", None), ("row", "sigmoid"), ("row", "silu")])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("scale", [None, 0.3, "channels"])
def test_parts(gate, activation, post, pre, scale):
    for dtype, stream, width in ((F32, F32, 70), (BF16, F32, 1300)):
        _check(*_case((3, 4, width), dtype, stream, gate=gate, activation=activation, post=post, pre=pre, scale=scale, seed=width), "parts")


# one row, fewer and more rows than the resident workgroups have groups, and enough that a workgroup walks its most
@pytest.mark.parametrize("rows,width", [(1, 64), (31, 64), (33, 64), (5000, 40), (300_000, 8), (2100, 1024), (1030, 8192)])
def test_row_counts(rows, width):
    _check(*_case((rows, width), BF16, F32, gate="row", activation="silu", seed=rows), "rows")


def test_sums_of_one_sign_stay_exact():
    """A column's sum over 4M rows of equal terms: 32-bit sums of that length would be off by 1e-3, these by less than 1e-5."""
    rows, width = 4_000_000, 8
    announce("residual norm, long column sums", rows, width)
    x = torch.ones(rows, width, device=DEV)
    scale = torch.full((width,), 0.7, device=DEV, requires_grad=True)
    h, _ = residual_norm(x, torch.zeros_like(x), residual_scale=scale, pre_norm=False)
    (grad,) = torch.autograd.grad(h, scale, torch.full_like(h, 0.1))
    assert_close_scaled(grad, torch.full((width,), rows * 0.1 / (1.0 + 1e-6) ** 0.5, dtype=torch.float64), what="dscale")


def test_empty_and_unused():
    announce("residual norm, empty")
    scale = torch.ones(16, device=DEV, requires_grad=True)
    for shape in ((0, 16), (3, 0, 16)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        h, y = residual_norm(x, torch.zeros(shape, device=DEV), post_scale=scale)
        assert h.shape == y.shape == shape
        grads = torch.autograd.grad((h, y), (x, scale), (torch.ones_like(h), torch.ones_like(y)))
        assert grads[0].shape == shape and int(grads[1].count_nonzero()) == 0
    # one output alone, and neither of the streams' gradients
    tensors, kwargs, options = _case((6, 70), F32, F32, gate="full", activation="silu")
    leaves = [_on(tensors["x"]), _on(tensors["residual"])]
    scales = {name: _on(value) for name, value in kwargs.items()}
    h, y = residual_norm(*leaves, **scales, **options)
    for output, seeds in ((h, (tensors["dh"], torch.zeros_like(tensors["dy"]))), (y, (torch.zeros_like(tensors["dh"]), tensors["dy"]))):
        wanted = residual_norm_backward_reference(*seeds, tensors["x"], tensors["residual"], **kwargs, **options)
        seed = seeds[0] if output is h else seeds[1]
        names = ("post_scale", "residual_scale") + (("pre_scale",) if output is y else ())
        got = torch.autograd.grad(output, [*leaves, scales["gate"], *(scales[n] for n in names)], seed.to(DEV), retain_graph=True)
        for actual, expected in zip(got, wanted):
            assert_close_scaled(actual, expected, what="one output")


def test_non_finite_rows_stay_in_their_rows():
    tensors, kwargs, options = _case((64, 90), BF16, F32, gate="full", activation="sigmoid")
    announce("residual norm, infinities and NaN")
    clean = residual_norm(tensors["x"].to(DEV), tensors["residual"].to(DEV), **{k: v.to(DEV) for k, v in kwargs.items() if v is not None}, **options)
    x = tensors["x"].clone()
    x[3, 5], x[17, 0], x[40, 89] = float("nan"), float("inf"), float("-inf")
    dirty = residual_norm(x.to(DEV), tensors["residual"].to(DEV), **{k: v.to(DEV) for k, v in kwargs.items() if v is not None}, **options)
    rest = [r for r in range(64) if r not in (3, 17, 40)]
    for a, b in zip(dirty, clean):
        assert_bitwise(a[rest], b[rest])
        assert bool(torch.isnan(a[3]).all())


def test_unaligned_tensors_and_another_stream():
    """Tensors that start at any element, used on a side stream; results are the same bit for bit."""
    announce("residual norm, unaligned, side stream")
    for dtype in (F32, BF16):
        base = torch.randn(2, 40 * 130 + 3, device=DEV).to(dtype)
        x, residual = (base[i, 3:].view(40, 130) for i in range(2))
        expected = residual_norm(x.clone(), residual.clone())
        side = torch.cuda.Stream(DEV)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = residual_norm(x, residual)
        side.synchronize()
        for a, b in zip(got, expected):
            assert_bitwise(a, b)


def test_gradient_of_gates_near_one():
    """Sigmoid gates up to 1 - 1e-13: their slopes keep their digits."""
    announce("residual norm, gates near one")
    gate = torch.linspace(-30.0, 30.0, 512, device=DEV).view(8, 64).contiguous().requires_grad_(True)
    x, dh = torch.randn(8, 64, device=DEV), torch.randn(8, 64, device=DEV)
    h, _ = residual_norm(x, torch.zeros_like(x), gate=gate, gate_activation="sigmoid", post_norm=False, pre_norm=False)
    (grad,) = torch.autograd.grad(h, gate, dh)
    exact = gate.detach().cpu().double()
    wanted = dh.cpu().double() * x.cpu().double() * torch.sigmoid(exact) * torch.sigmoid(-exact)
    # two sigmoids and three products, each a few steps of 2^-24 off
    assert_close_scaled(grad, wanted, rtol=2e-6, scale=0.0, what="dgate")


@pytest.mark.parametrize("activation", ["sigmoid", "silu"])
def test_gates_near_zero(activation):
    """Gates of -120 to -80, whose exponential passes float32."""
    announce("residual norm, gates near zero", activation)
    gate = torch.linspace(-120.0, -80.0, 4096, device=DEV).view(64, 64).contiguous().requires_grad_(True)
    x = torch.ones(64, 64, device=DEV)
    h, _ = residual_norm(x, torch.zeros_like(x), gate=gate, gate_activation=activation, post_norm=False, pre_norm=False)
    (grad,) = torch.autograd.grad(h, gate, torch.ones_like(h))
    exact = gate.detach().cpu().double()
    s = torch.sigmoid(exact)
    value, slope = (s, s * (1.0 - s)) if activation == "sigmoid" else (exact * s, s * (1.0 + exact * (1.0 - s)))
    # where s is below float32's smallest normal number, 1.2e-38, it may be 0
    for got, wanted in ((h, value), (grad, slope)):
        assert ((got.detach().cpu().double() - wanted).abs() <= 1e-5 * wanted.abs() + 1.2e-38 * 121.0).all()


def test_second_derivative_is_refused():
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    h, y = residual_norm(x, torch.zeros_like(x))
    (grad,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.sum(), x)


def test_captured_step_replays():
    """Forward and backward captured once; replays follow new inputs, with eager work between them."""
    announce("residual norm, graph")
    shape = (777, 384)
    static = {name: torch.randn(shape, device=DEV) for name in ("x", "residual", "gate", "dh", "dy")}
    scale = torch.rand(384, device=DEV) + 0.5

    def step():
        leaves = [static["x"].detach().requires_grad_(True), static["residual"].detach().requires_grad_(True),
                  static["gate"].detach().requires_grad_(True), scale.detach().requires_grad_(True)]
        h, y = residual_norm(leaves[0], leaves[1], gate=leaves[2], gate_activation="silu", post_scale=leaves[3])
        return (h.detach(), y.detach(), *torch.autograd.grad((h, y), leaves, (static["dh"], static["dy"])))

    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = step()
    for seed in range(3):
        torch.manual_seed(seed)
        for tensor in static.values():
            tensor.copy_(torch.randn(shape, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outputs]
        for a, b in zip(got, step()):
            assert_bitwise(a, b)


@pytest.mark.parametrize("dtype,stream", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("width", [1, 2, 7, 8, 9, 63, 64, 65, 90, 128, 129, 250, 256, 257, 511, 512, 513, 810, 1024])
def test_whole_and_last_workgroups(width, dtype, stream):
    """70 rows: workgroups with rows behind them, whose loads need no guard, and the last one, whose do."""
    _check(*_case((70, width), dtype, stream, gate="full", activation="silu", seed=width), "workgroups")
