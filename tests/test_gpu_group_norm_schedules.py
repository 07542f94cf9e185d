"""GPU parity of the group norm on every workgroup that a sample's length selects, for every layout of channels.

A sample of up to 32 elements a thread is held by a workgroup of 64, 256, 512 or
(forward) 1,024 threads, longer ones are streamed or cut into tiles; a thread's
vector lies in one group (64 channels in 8), in two (90 in 6) or in any number of
them (12 in 4).  Tolerances are those of ``test_gpu_group_norm``.
"""
from __future__ import annotations

import pytest
import torch

from bysj_amd.kernels import _C
from bysj_amd.kernels.group_norm import group_norm
from parity import announce, assert_close_scaled
from test_gpu_group_norm import _check, _inputs, _offsets, _rtol

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)

LAYOUTS = [(64, 8), (90, 6), (12, 4)]
ELEMENTS = [1000, 5000, 12000, 30000, 200000]    # of a sample: 64, 256, 512 and 1,024 threads, tiles
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("elements", ELEMENTS)
@pytest.mark.parametrize("channels,groups", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_samples_of_one_length(dtype, channels, groups, elements):
    rows = elements // channels
    x, grad, scale, bias = _inputs((3, rows, channels), dtype, seed=elements)
    _check(x, grad, groups, scale, bias, None, "silu", what=f"{elements} elements")


@pytest.mark.parametrize("elements", ELEMENTS)
@pytest.mark.parametrize("channels,groups", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_samples_up_to_a_length(dtype, channels, groups, elements):
    rows = elements // channels
    lengths = [rows, 0, 1, rows // 2, rows - 1]
    x, grad, scale, bias = _inputs((sum(lengths), channels), dtype, seed=elements)
    for longest in (rows, None):
        _check(x, grad, groups, scale, bias, _offsets(lengths), None, max_rows=longest, what=f"up to {elements} elements")


@pytest.mark.parametrize("channels,groups", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_workgroups_that_take_several_samples(dtype, channels, groups):
    """More samples than workgroups of 512 threads are resident."""
    x, grad, scale, bias = _inputs((700, 12000 // channels, channels), dtype)
    _check(x, grad, groups, scale, bias, None, "silu", what="many")


@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("mean,threads", [(800, 64), (5000, 256), (8500, 512), (20000, 1024)])
@pytest.mark.parametrize("channels,groups", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_longer_samples_among_many(dtype, channels, groups, mean, threads, activation):
    """Workgroups for the mean: the longest sample is several times what they hold."""
    samples = 1100 if threads == 64 else 262144 // threads + 40
    rows = mean // channels
    lengths = [rows - (k * 7) % (rows // 3) for k in range(samples)]
    lengths[5], lengths[77] = 6 * rows, 0
    x, grad, scale, bias = _inputs((sum(lengths), channels), dtype, seed=mean)
    _check(x, grad, groups, scale, bias, _offsets(lengths), activation, max_rows=6 * rows, what=f"about {mean} elements")


@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("said", [500, 5000, 12000, 30000])
@pytest.mark.parametrize("channels,groups", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_samples_longer_than_said_among_others(dtype, channels, groups, said, activation):
    """Samples of the length that was said, of up to 16 times that, and of more, in turn."""
    rows = said // channels
    lengths = [rows, 20 * rows + 1, 0, 3 * rows, 1, 33 * rows - 1, rows // 2, rows, 17 * rows]
    x, grad, scale, bias = _inputs((sum(lengths), channels), dtype, seed=said)
    _check(x, grad, groups, scale, bias, _offsets(lengths), activation, max_rows=rows, what=f"said {said} elements")


# ---------------------------------------------------------------------------
# long sums
# ---------------------------------------------------------------------------
#
# Terms that are all alike do not average their roundings out: a running sum of n
# of them in 32 bits is off by up to n 2^-25 of it.  The rule of 1e-5 leaves room
# for about 300 in sequence.

def _even_gradients(x, groups, scale, bias, offsets, value, activation, max_rows):
    """(y, grad_x, grad_scale, grad_bias) for a gradient of ``value`` everywhere, the definition's in 64 bits on the GPU, and
    what the roundings of h leave of grad_scale."""
    leaves = [t.requires_grad_(True) for t in (x, scale, bias)]
    y = group_norm(x, groups, scale, bias, offsets=offsets, max_rows=max_rows, activation=activation)
    grad = torch.full_like(y, value)
    actual = torch.autograd.grad(y, leaves, grad)
    with torch.no_grad():
        rows = x.double().reshape(-1, groups, x.shape[-1] // groups)
        centred = rows - rows.mean((0, 2), keepdim=True)
        inverse = 1.0 / torch.sqrt(centred.square().mean((0, 2), keepdim=True) + 1e-5)
        hat = (centred * inverse).reshape(-1, x.shape[-1])
        z = hat * scale.double() + bias.double()
        gate = torch.sigmoid(z)
        dz = grad.double().reshape(hat.shape) * (gate * (1.0 + z * (1.0 - gate)) if activation else 1.0)
        wanted_y = (z * gate if activation else z).view(x.shape)
        u = (dz * scale.double()).view(rows.shape)
        h = hat.view(rows.shape)
        grad_x = inverse * (u - u.mean((0, 2), keepdim=True) - h * (u * h).mean((0, 2), keepdim=True))
        wanted = grad_x.view(x.shape), (dz * hat).sum(0), dz.sum(0)
        # grad_scale adds dz h over all rows, and its terms may cancel.  A row's h is off by 2^-24 (|mean| rstd + 2 |h|) at
        # most (the stored mean's rounding, the difference's, rstd's), whatever the sum does with its own roundings.
        far = (rows.mean((0, 2), keepdim=True).abs() * inverse).expand_as(h)
        slack = 2.0 ** -24 * (dz.abs() * (far + 2.0 * h.abs()).reshape(hat.shape)).sum(0)
    return (y, *actual), (wanted_y, *wanted), slack


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels,groups", LAYOUTS)
@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("said", [1, 5000, 12000, 30000])
def test_a_sample_much_longer_than_said(said, channels, groups, activation, dtype):
    """max_rows of ``said`` elements for a sample of 24 million: its sums stay as exact as others'."""
    announce("longer than said", said, channels, groups, activation, dtype)
    rows = 24_000_000 // channels
    generator = torch.Generator(device=DEV).manual_seed(channels)
    x = (torch.randn(rows, channels, generator=generator, device=DEV) * 1.5 + 0.5).to(dtype)
    scale = torch.rand(channels, generator=generator, device=DEV) + 0.5
    bias = torch.randn(channels, generator=generator, device=DEV)
    offsets = torch.tensor([0, rows], device=DEV)
    actual, wanted, slack = _even_gradients(x, groups, scale, bias, offsets, 0.1, activation, max(said // channels, 1))
    for name, a, b in zip(("y", "grad_x", "grad_scale", "grad_bias"), actual, wanted):
        if name == "grad_scale":
            bound = 1e-5 * b.abs() + 1e-5 * b.abs().max() + slack
            assert ((a.double() - b).abs() <= bound).all(), f"grad_scale: {((a.double() - b).abs() / bound).max()} of the bound"
        else:
            assert_close_scaled(a, b, rtol=_rtol(dtype) if name in ("y", "grad_x") else 1e-5, what=name)


def test_a_far_mean_of_a_sample_much_longer_than_said():
    rows, channels, mean = 375_000, 64, -1000.0
    generator = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(rows, channels, generator=generator, device=DEV) * 1.5 + mean
    y = group_norm(x, 8, offsets=torch.tensor([0, rows], device=DEV), max_rows=1)
    part = x.double().view(rows, 8, 8)
    centred = part - part.mean((0, 2), keepdim=True)
    wanted = centred / torch.sqrt(centred.square().mean((0, 2), keepdim=True) + 1e-5)
    # the rounding of the mean, 2^-24 |mean| / std on values of up to about 4
    assert_close_scaled(y, wanted.view(rows, channels), scale=1e-5 + 2.0 ** -24 * abs(mean) * 4, what="far mean")


@pytest.mark.parametrize("channels,groups", LAYOUTS)
@pytest.mark.parametrize("size", [0.3, 7.7])
def test_deviations_of_one_size_in_a_sample_much_longer_than_said(size, channels, groups):
    """Rows of +size and -size by turns: every batch adds the same to the squared deviations."""
    rows = 48_000_000 // channels // 2 * 2
    sign = torch.ones(rows, 1, device=DEV)
    sign[1::2] = -1.0
    x = (sign * size).expand(rows, channels).contiguous()
    y = group_norm(x, groups, offsets=torch.tensor([0, rows], device=DEV), max_rows=1)
    value = float(x[0, 0])
    assert_close_scaled(y, (sign.double() * (value / (value * value + 1e-5) ** 0.5)).expand(rows, channels), what="one size")


def test_gradients_summed_over_many_samples():
    """61 million samples of one row under gradients of one size: what a workgroup adds up stays short."""
    announce("many samples")
    samples, channels = 61_000_000, 8
    x = torch.randn(samples, channels, generator=torch.Generator(device=DEV).manual_seed(0), device=DEV)
    grad = torch.full_like(x, 0.1)
    _, statistics = _C.group_norm_forward(x, 1)
    _, _, grad_bias = _C.group_norm_backward(grad, x, 1, None, None, None, statistics, want_x=False, want_scale=False)
    assert_close_scaled(grad_bias, torch.full((channels,), samples * float(grad[0, 0]), dtype=torch.float64), what="grad_bias")


def test_gradients_summed_over_a_large_sample():
    """One sample of 4e9 elements (16 GB): the same for a tile's workgroup."""
    announce("large sample")
    rows, channels = 62_500_000, 64
    x = torch.randn(rows, channels, generator=torch.Generator(device=DEV).manual_seed(0), device=DEV)
    grad = torch.full_like(x, 0.1)
    offsets = torch.tensor([0, rows], device=DEV)
    _, statistics = _C.group_norm_forward(x, 8, None, None, offsets)
    _, _, grad_bias = _C.group_norm_backward(grad, x, 8, None, None, offsets, statistics, want_x=False, want_scale=False)
    assert_close_scaled(grad_bias, torch.full((channels,), rows * float(grad[0, 0]), dtype=torch.float64), what="grad_bias")
