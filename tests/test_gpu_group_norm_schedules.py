"""GPU parity of the group norm on every workgroup that a sample's length selects, for every layout of channels.

A sample of up to 32 elements a thread is held by a workgroup of 64, 256, 512 or
(forward) 1,024 threads, longer ones are streamed or cut into tiles; a thread's
vector lies in one group (64 channels in 8), in two (90 in 6) or in any number of
them (12 in 4).  Tolerances are those of ``test_gpu_group_norm``.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_group_norm import _check, _inputs, _offsets

pytestmark = pytest.mark.gpu

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
