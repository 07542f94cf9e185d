"""What the group norm and the optimiser refuse, on the CPU: no call here reaches a GPU.

Arguments are checked before the device, so a wrong one is named as such; right
ones end at the device gate (RuntimeError).  The C entry points check sizes and
pointers before any device call.
"""
from __future__ import annotations

import ctypes

import pytest
import torch

from bysj_amd.kernels import _lib, optim
from bysj_amd.kernels.group_norm import group_norm
from oracle.group_norm import group_norm_backward_reference, group_norm_reference
from oracle import optim as ref

BUILT = pytest.mark.skipif(not _lib.LIBRARY_PATH.exists(), reason="libdpa4k.so is not built")
X = torch.zeros(6, 8)


@pytest.mark.parametrize("error,args,kwargs", [
    (TypeError, ([1.0], 2), {}),
    (TypeError, (X.double(), 2), {}),
    (TypeError, (X.int(), 2), {}),
    (ValueError, (X[0], 2), {}),
    (ValueError, (X.t(), 2), {}),
    (ValueError, (torch.zeros(2, 0), 1), {}),
    (ValueError, (torch.zeros(2, 4097), 1), {}),
    (TypeError, (X, 2.0), {}),
    (TypeError, (X, True), {}),
    (ValueError, (X, 3), {}),
    (ValueError, (X, 0), {}),
    (ValueError, (X, -2), {}),
    (TypeError, (X, 2, [1.0] * 8), {}),
    (TypeError, (X, 2, torch.ones(8).double()), {}),
    (ValueError, (X, 2, torch.ones(4)), {}),
    (ValueError, (X, 2, torch.ones(16)[::2]), {}),
    (ValueError, (X, 2, None, torch.ones(8, 1)), {}),
    (TypeError, (X, 2), {"offsets": [0, 6]}),
    (TypeError, (X, 2), {"offsets": torch.tensor([0, 6], dtype=torch.int32)}),
    (ValueError, (X, 2), {"offsets": torch.tensor([], dtype=torch.int64)}),
    (ValueError, (X, 2), {"offsets": torch.zeros(2, 2, dtype=torch.int64)}),
    (ValueError, (X, 2), {"offsets": torch.zeros(4, dtype=torch.int64)[::2]}),
    (TypeError, (X, 2), {"max_rows": 2.5}),
    (ValueError, (X, 2), {"max_rows": -1}),
    (ValueError, (X, 2), {"activation": "relu"}),
    (ValueError, (X, 2), {"eps": 0.0}),
    (ValueError, (X, 2), {"eps": float("nan")}),
    (ValueError, (X, 2), {"eps": "small"}),
    (RuntimeError, (X, 2), {}),
])
def test_group_norm_refusals(error, args, kwargs):
    with pytest.raises(error):
        group_norm(*args, **kwargs)


P = [torch.zeros(4), torch.zeros(2, 3)]


@pytest.mark.parametrize("error,args,kwargs", [
    (TypeError, (torch.zeros(3),), {}),
    (TypeError, (3,), {}),
    (TypeError, ([1.0],), {}),
    (ValueError, ([],), {}),
    (ValueError, ([None],), {}),
    (TypeError, ([torch.zeros(3).double()],), {}),
    (ValueError, ([torch.zeros(4)[::2]],), {}),
    (ValueError, (P, 0.0), {}),
    (ValueError, (P, -1.0), {}),
    (ValueError, (P, float("inf")), {}),
    (TypeError, (P, "1"), {}),
    (RuntimeError, (P, 1.0), {}),
])
def test_grad_norm_refusals(error, args, kwargs):
    with pytest.raises(error):
        optim.grad_norm(*args, **kwargs)


@pytest.mark.parametrize("error,args,kwargs", [
    (TypeError, (torch.zeros(3),), {}),
    (ValueError, ([],), {}),
    (TypeError, ([None],), {}),
    (TypeError, ([torch.zeros(3).half()],), {}),
    (ValueError, ([torch.zeros(3), torch.zeros(3).bfloat16()],), {}),
    (ValueError, ([torch.zeros(4)[::2]],), {}),
    (ValueError, (P,), {"state_bits": 16}),
    (ValueError, (P,), {"state_bits": True}),
    (ValueError, (P, [torch.zeros(4), torch.zeros(2, 3)]), {}),
    (ValueError, (P, [torch.zeros(4)], [torch.zeros(4)]), {}),
    (ValueError, (P, [torch.zeros(4), torch.zeros(3, 2)], [torch.zeros(4), torch.zeros(2, 3)]), {}),
    (TypeError, (P, [torch.zeros(4).double(), torch.zeros(2, 3)], [torch.zeros(4), torch.zeros(2, 3)]), {}),
    (ValueError, (P,), {"step": -1}),
    (ValueError, (P,), {"step": [1]}),
    (TypeError, (P,), {"step": [1, 2.5]}),
    (RuntimeError, (P,), {}),
])
def test_adamw_plan_refusals(error, args, kwargs):
    with pytest.raises(error):
        optim.adamw_plan(*args, **kwargs)


def test_overlapping_parameters_are_refused():
    flat = torch.zeros(10)
    for params in ([flat, flat], [flat[:6], flat[5:]]):
        with pytest.raises(ValueError, match="overlap"):
            optim.adamw_plan(params)
    with pytest.raises(ValueError, match="overlap"):
        optim.adamw_plan([flat[:5]], [flat[5:]], [flat[5:]])
    with pytest.raises(RuntimeError):  # neighbours are fine; the device is not
        optim.adamw_plan([flat[:5], flat[5:]])


class _Plan:
    params = P
    addresses = [p.data_ptr() for p in P]
    shapes = [p.shape for p in P]
    device = torch.device("cpu")


@pytest.mark.parametrize("error,grads,kwargs", [
    (ValueError, P[:1], {}),
    (TypeError, [1.0, P[1]], {}),
    (TypeError, [p.double() for p in P], {}),
    (TypeError, [P[0], P[1].bfloat16()], {}),
    (ValueError, [P[0], torch.zeros(3, 2)], {}),
    (ValueError, [torch.zeros(8)[::2], P[1]], {}),
    (ValueError, [torch.zeros(4, device="meta"), None], {}),
    (ValueError, P, {"lr": -1.0}),
    (ValueError, P, {"lr": float("nan")}),
    (TypeError, P, {"lr": "1"}),
    (ValueError, P, {"lr": torch.zeros(2)}),
    (ValueError, P, {"lr": torch.zeros((), dtype=torch.float64)}),
    (TypeError, P, {"betas": 0.9}),
    (ValueError, P, {"betas": (1.0, 0.9)}),
    (ValueError, P, {"betas": (0.9, -0.1)}),
    (ValueError, P, {"eps": 0.0}),
    (ValueError, P, {"weight_decay": -1.0}),
    (TypeError, P, {"grad_factor": 0.5}),
    (ValueError, P, {"grad_factor": torch.ones(3)}),
    (TypeError, P, {"seed": 1.5}),
])
def test_adamw_step_refusals(error, grads, kwargs):
    with pytest.raises(error):
        optim.adamw_step(_Plan, grads, **{"lr": 1e-3, **kwargs})


def test_adamw_step_refuses_parameters_that_moved():
    class Moved(_Plan):
        addresses = [0, 0]

    with pytest.raises(RuntimeError, match="moved"):
        optim.adamw_step(Moved, P, lr=1e-3)
    assert optim.adamw_step(_Plan, [None, None], lr=1e-3) is None


@pytest.mark.parametrize("error,params,kwargs", [
    (ValueError, P, {"lr": -1.0}),
    (ValueError, P, {"betas": (0.9, 1.0)}),
    (ValueError, P, {"eps": -1.0}),
    (ValueError, P, {"weight_decay": -1.0}),
    (ValueError, P, {"max_norm": 0.0}),
    (ValueError, P, {"state_bits": 4}),
    (TypeError, [torch.zeros(3).double()], {}),
    (ValueError, [torch.zeros(4)[::2]], {}),
    (ValueError, [], {}),
])
def test_optimiser_refusals(error, params, kwargs):
    with pytest.raises(error):
        optim.AdamW(params, **kwargs)


@pytest.mark.parametrize("theirs,options", [
    (torch.optim.AdamW, {"amsgrad": True}),
    (torch.optim.AdamW, {"maximize": True}),
    (torch.optim.Adam, {"weight_decay": 0.1}),  # added to the gradient there
])
def test_optimiser_refuses_options_that_it_does_not_have(theirs, options):
    p = torch.nn.Parameter(torch.zeros(3))
    mine = optim.AdamW([p], lr=0.5)
    with pytest.raises(ValueError):
        mine.load_state_dict(theirs([p], **options).state_dict())
    assert mine.param_groups[0]["lr"] == 0.5
    with pytest.raises(ValueError):
        optim.AdamW([dict(theirs([p], **options).param_groups[0])])
    mine.load_state_dict(theirs([p], lr=0.25, weight_decay=0.0).state_dict())
    assert mine.param_groups[0]["lr"] == 0.25


@pytest.mark.parametrize("seed", [1.5, True, "1", None])
def test_optimiser_refuses_seeds_that_are_not_integers(seed):
    with pytest.raises(TypeError):
        optim.AdamW(P, seed=seed)


@BUILT
def test_c_entry_points_refuse_bad_sizes_before_any_device_call():
    lib = _lib.load()
    null, f32 = None, _lib.TYPE_F32
    eps = ctypes.c_float(1e-5)
    some = ctypes.c_void_p(256)  # never dereferenced

    def norm(*sizes, eps=eps, type_=f32, offsets=some, x=null):
        return lib.dpa4k_group_norm_forward(x, null, null, offsets, null, null, null, *sizes, -1, eps, 0, type_, null, 0, null)

    cases = [
        (norm(1, -1, 1, 8, 2), "negative"),
        (norm(1, 4, 1, 0, 1), "channels"),
        (norm(1, 4, 1, 4097, 1), "channels"),
        (norm(1, 4, 1, 8, 3), "divide"),
        (norm(1, 4, 1, 8, 2, type_=7), "unknown type"),
        (norm(3, 4, 1, 8, 2, offsets=null), "every entry"),
        (norm(1, 2**40, 2**30, 8, 2), "overflows"),
        (norm(2**61, 4, 1, 8, 2), "overflows"),
        (norm(1, 4, 1, 8, 2, eps=ctypes.c_float(0.0)), "eps"),
        (norm(1, 4, 1, 8, 2), "null pointer"),
    ]
    for status, _ in cases:
        assert status == _lib.EINVAL
    for call, (_, fragment) in zip((lambda: norm(1, 4, 1, 8, 3), lambda: norm(1, 4, 1, 8, 2)), ((0, "divide"), (0, "null"))):
        call()
        assert fragment in lib.dpa4k_last_error().decode()
    backward = lib.dpa4k_group_norm_backward(null, null, null, null, some, null, null, null, null, null, 1, 4, 1, 8, 2, -1, 0, f32,
                                             null, 0, null)
    assert backward == _lib.EINVAL
    status = lib.dpa4k_group_norm_forward(some, null, null, some, some, some, some, 1, 4, 1, 8, 2, -1, eps, 0, f32, null, 0, null)
    assert status == _lib.EWORKSPACE
    assert lib.dpa4k_group_norm_workspace_size(1, 4, 1, 8, 3, 1, -1, f32, 0) == 0
    for backward in (0, 1):
        small, large = (lib.dpa4k_group_norm_workspace_size(10, rows, 1, 64, 8, 1, -1, f32, backward) for rows in (100, 10**7))
        assert 0 < small <= large and large % 256 == 0

    counts, types = (ctypes.c_int64 * 1)(4), (ctypes.c_int32 * 1)(0)
    pointers = (ctypes.c_void_p * 1)(256)
    assert lib.dpa4k_grad_norm(pointers, counts, types, -1, 1.0, some, some, some, 256, null) == _lib.EINVAL
    assert lib.dpa4k_grad_norm(pointers, counts, types, 1, 1.0, null, some, some, 256, null) == _lib.EINVAL
    assert lib.dpa4k_grad_norm(pointers, counts, (ctypes.c_int32 * 1)(2), 1, 1.0, some, some, some, 256, null) == _lib.EINVAL
    assert lib.dpa4k_grad_norm(pointers, (ctypes.c_int64 * 1)(-4), types, 1, 1.0, some, some, some, 256, null) == _lib.EINVAL
    assert lib.dpa4k_grad_norm(pointers, counts, types, 1, 1.0, some, some, null, 0, null) == _lib.EWORKSPACE

    chunks = ctypes.c_int64(0)
    entry = (_lib.AdamwTensor * 1)()
    entry[0].count = 4
    host = (ctypes.c_char * 4096)()
    assert lib.dpa4k_adamw_plan(entry, 1, 32, host, 4096, ctypes.byref(chunks)) == _lib.EINVAL  # null pointers
    entry[0].param = entry[0].exp_avg = entry[0].exp_avg_sq = 256
    assert lib.dpa4k_adamw_plan(entry, 1, 32, host, 16, ctypes.byref(chunks)) == _lib.EWORKSPACE
    assert lib.dpa4k_adamw_plan(entry, 1, 16, host, 4096, ctypes.byref(chunks)) == _lib.EINVAL
    assert lib.dpa4k_adamw_plan(entry, 1, 8, host, 4096, ctypes.byref(chunks)) == _lib.EINVAL  # no scales
    assert lib.dpa4k_adamw_plan(entry, 1, 32, host, 4096, ctypes.byref(chunks)) == _lib.OK and chunks.value == 1
    entry[0].step = -1
    assert lib.dpa4k_adamw_plan(entry, 1, 32, host, 4096, ctypes.byref(chunks)) == _lib.EINVAL

    def step(plan=some, tensors=1, chunks=1, bits=32, p=0, g=0, grads=pointers, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0):
        return lib.dpa4k_adamw_step(plan, tensors, chunks, bits, p, g, grads, lr, null, b1, b2, eps, wd, null, 0, null)

    for bad in (dict(plan=null), dict(tensors=-1), dict(chunks=-1), dict(bits=4), dict(p=2), dict(g=2), dict(grads=null),
                dict(lr=-1.0), dict(lr=float("nan")), dict(b1=1.0), dict(b2=-0.5), dict(eps=0.0), dict(eps=1e-60),
                dict(wd=float("inf"))):
        assert step(**bad) == _lib.EINVAL, bad
    assert step(tensors=0, chunks=0, plan=null) == _lib.OK


# ---------------------------------------------------------------------------
# the oracles
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("activation", [None, "silu"])
def test_group_norm_oracle_against_autograd_and_torch(activation):
    generator = torch.Generator().manual_seed(0)
    x = torch.randn(12, 3, 8, generator=generator, dtype=torch.float64, requires_grad=True)
    scale = torch.rand(8, generator=generator, dtype=torch.float64).requires_grad_(True)
    bias = torch.randn(8, generator=generator, dtype=torch.float64).requires_grad_(True)
    grad = torch.randn(12, 3, 8, generator=generator, dtype=torch.float64)
    offsets = torch.tensor([0, 5, 5, 12])
    parts = []
    for a, b in ((0, 5), (5, 12)):
        rows = x[a:b].reshape(1, -1, 8).transpose(1, 2)
        z = torch.nn.functional.group_norm(rows, 2, scale, bias, 1e-5).transpose(1, 2).reshape(b - a, 3, 8)
        parts.append(torch.nn.functional.silu(z) if activation else z)
    y = torch.cat(parts)
    torch.testing.assert_close(group_norm_reference(x, 2, scale, bias, offsets, 1e-5, activation), y.detach(),
                               rtol=1e-12, atol=1e-12)
    wanted = torch.autograd.grad(y, (x, scale, bias), grad)
    for actual, expected in zip(group_norm_backward_reference(grad, x, 2, scale, bias, offsets, 1e-5, activation), wanted):
        torch.testing.assert_close(actual, expected, rtol=1e-11, atol=1e-11)


def test_adamw_oracle_against_torch():
    generator = torch.Generator().manual_seed(0)
    p = torch.randn(50, generator=generator, dtype=torch.float64)
    twin = torch.nn.Parameter(p.clone())
    optimiser = torch.optim.AdamW([twin], lr=0.01, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1, foreach=False)
    m = v = torch.zeros(50, dtype=torch.float64)
    for t in range(1, 5):
        g = torch.randn(50, generator=generator, dtype=torch.float64)
        twin.grad = g.clone()
        optimiser.step()
        p, m, v = ref.adamw_f64(p, g, m, v, t, lr=0.01, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)
        torch.testing.assert_close(p, twin.detach(), rtol=1e-12, atol=1e-12)


def test_code_oracle():
    """Codes are exact on their own values, off by at most a sixteenth elsewhere, never above the block's largest code, and
    a second moment that is not 0 never becomes 0."""
    generator = torch.Generator().manual_seed(0)
    x = torch.randn(32 * 300, generator=generator) * torch.exp(4.0 * torch.randn(32 * 300, generator=generator))
    half = torch.full((x.numel(),), 0x8000)
    for signed in (True, False):
        value = x if signed else x.square()
        once = ref.coded(value, half, signed)
        for noise in (0, 0xFFFF):
            assert torch.equal(ref.coded(once, torch.full((x.numel(),), noise), signed), once)
        top = value.abs().view(-1, 32).amax(1).repeat_interleave(32)
        near = value.abs() > top * 2.0 ** (-14 if signed else -30)
        assert ((once - value).abs()[near] <= value.abs()[near] / 16 * (1 + 2.0 ** -16)).all()
        if not signed:
            assert (once > 0).all()
    zero = torch.zeros(32)
    assert torch.equal(ref.coded(zero, half[:32], False), zero) and torch.equal(ref.coded(zero, half[:32], True), zero)
    # halfway between two codes: up and down equally often
    between = torch.full((32,), 1.0625)
    assert torch.equal(ref.coded(between, torch.arange(32) * 2048, True) > 1.0625, torch.arange(32) >= 16)
