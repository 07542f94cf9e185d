"""What the block norm and the expert operators refuse, and their oracles against autograd, on the CPU.

Arguments are checked before the device, so a wrong one is named as such; right
ones end at the device gate (RuntimeError).  The C entry points check sizes and
pointers before any device call.
"""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from bysj_amd.kernels import _lib
from bysj_amd.kernels.block_norm import residual_norm
from bysj_amd.kernels.experts import ExpertPlan, expert_combine, expert_dispatch, expert_linear, expert_route
from oracle.block_norm import residual_norm_backward_reference, residual_norm_reference
from oracle.experts import (expert_combine_reference, expert_dispatch_reference, expert_linear_reference,
                            expert_route_backward_reference, expert_route_reference)

BUILT = pytest.mark.skipif(not _lib.LIBRARY_PATH.exists(), reason="libdpa4k.so is not built")
X = torch.zeros(6, 8)
C8 = torch.ones(8)


@pytest.mark.parametrize("error,args,kwargs", [
    (TypeError, ([1.0], X), {}),
    (TypeError, (X, [1.0]), {}),
    (TypeError, (X.double(), X.double()), {}),
    (TypeError, (X, X.bfloat16()), {}),
    (TypeError, (X.half(), X.bfloat16()), {}),
    (ValueError, (X, X[:3]), {}),
    (ValueError, (torch.zeros(()), torch.zeros(())), {}),
    (ValueError, (torch.zeros(2, 0), torch.zeros(2, 0)), {}),
    (ValueError, (torch.zeros(1, 8193), torch.zeros(1, 8193)), {}),
    (ValueError, (torch.zeros(8, 6).t(), X), {}),
    (ValueError, (X, torch.zeros(8, 6).t()), {}),
    (TypeError, (X, X), {"gate": 1.0}),
    (TypeError, (X, X), {"gate": X.half()}),
    (ValueError, (X, X), {"gate": torch.zeros(8)}),
    (ValueError, (X, X), {"gate": torch.zeros(6)}),
    (ValueError, (X, X), {"gate": torch.zeros(8, 6).t()}),
    (ValueError, (X, X), {"gate_activation": "silu"}),
    (ValueError, (X, X), {"gate": X, "gate_activation": "tanh"}),
    (TypeError, (X, X), {"post_scale": 1.0}),
    (TypeError, (X, X), {"post_scale": C8.double()}),
    (ValueError, (X, X), {"post_scale": torch.ones(4)}),
    (ValueError, (X, X), {"post_scale": torch.ones(16)[::2]}),
    (ValueError, (X, X), {"post_scale": C8, "post_norm": False}),
    (ValueError, (X, X), {"pre_scale": C8, "pre_norm": False}),
    (TypeError, (X, X), {"pre_norm": 1}),
    (TypeError, (X, X), {"residual_scale": True}),
    (TypeError, (X, X), {"residual_scale": "small"}),
    (ValueError, (X, X), {"residual_scale": math.nan}),
    (ValueError, (X, X), {"residual_scale": 1e39}),
    (ValueError, (X, X), {"residual_scale": torch.ones(1)}),
    (ValueError, (X, X), {"eps": 0.0}),
    (ValueError, (X, X), {"eps": math.inf}),
    (ValueError, (X, X), {"eps": 1e-60}),
    (ValueError, (X, X), {"eps": "small"}),
    (RuntimeError, (X, X), {}),
    (RuntimeError, (X.half(), X), {"gate": torch.zeros(6, 1).half(), "post_scale": C8, "residual_scale": 0.5}),
])
def test_residual_norm_refusals(error, args, kwargs):
    with pytest.raises(error):
        residual_norm(*args, **kwargs)


@pytest.mark.parametrize("error,args,kwargs", [
    (TypeError, ([1.0], 2), {}),
    (TypeError, (X.double(), 2), {}),
    (ValueError, (X[0], 2), {}),
    (ValueError, (torch.zeros(8, 6).t(), 2), {}),
    (ValueError, (torch.zeros(4, 0), 1), {}),
    (ValueError, (torch.zeros(4, 1025), 1), {}),
    (TypeError, (X, 2.0), {}),
    (TypeError, (X, True), {}),
    (ValueError, (X, 0), {}),
    (ValueError, (X, 9), {}),
    (ValueError, (X, 5), {"groups": 4, "top_groups": 2}),
    (ValueError, (X, 2), {"groups": 3}),
    (ValueError, (X, 2), {"groups": 0}),
    (ValueError, (torch.zeros(4, 1024), 2), {"groups": 128}),
    (ValueError, (X, 2), {"groups": 2, "top_groups": 3}),
    (ValueError, (X, 2), {"groups": 2, "top_groups": 0}),
    (TypeError, (X, 2), {"groups": 2.0}),
    (ValueError, (X, 2), {"scores": "relu"}),
    (TypeError, (X, 2), {"normalize": 1}),
    (TypeError, (X, 2), {"scale": "1"}),
    (ValueError, (X, 2), {"scale": math.inf}),
    (TypeError, (X, 2), {"bias": [0.0] * 8}),
    (TypeError, (X, 2), {"bias": C8.double()}),
    (ValueError, (X, 2), {"bias": torch.ones(4)}),
    (ValueError, (X, 2), {"bias": torch.ones(16)[::2]}),
    (ValueError, (X, 2), {"bias": C8.clone().requires_grad_(True)}),
    (RuntimeError, (X, 2), {}),
    (RuntimeError, (X.bfloat16(), 2), {"bias": C8, "groups": 4, "top_groups": 1, "scores": "sigmoid"}),
])
def test_expert_route_refusals(error, args, kwargs):
    with pytest.raises(error):
        expert_route(*args, **kwargs)


CHOSEN = torch.tensor([[0, 1], [1, 2], [2, -1]])
PLAN = ExpertPlan(*expert_dispatch_reference(CHOSEN, 3))


@pytest.mark.parametrize("error,args", [
    (TypeError, ([[0]], 3)),
    (TypeError, (CHOSEN.int(), 3)),
    (ValueError, (CHOSEN[0], 3)),
    (ValueError, (CHOSEN.t(), 3)),
    (ValueError, (CHOSEN[:, :0], 3)),
    (TypeError, (CHOSEN, 3.0)),
    (ValueError, (CHOSEN, 0)),
    (ValueError, (CHOSEN, 1025)),
    (RuntimeError, (CHOSEN, 3)),
])
def test_expert_dispatch_refusals(error, args):
    with pytest.raises(error):
        expert_dispatch(*args)


W = torch.zeros(3, 4, 8)


@pytest.mark.parametrize("error,args,kwargs", [
    (TypeError, (X[:3], W, tuple(PLAN)), {}),
    (TypeError, (X[:3], W, PLAN._replace(offsets=[0, 1, 2, 3])), {}),
    (TypeError, (X[:3], W, PLAN._replace(order=PLAN.order.int())), {}),
    (ValueError, (X[:3], W, PLAN._replace(order=PLAN.order[:5])), {}),
    (ValueError, (X[:3], W, PLAN._replace(slots=PLAN.slots.view(-1))), {}),
    (ValueError, (X[:3], W, PLAN._replace(slots=PLAN.slots.t())), {}),
    (ValueError, (X[:3], W, PLAN._replace(offsets=PLAN.offsets[:1])), {}),
    (ValueError, (X[:3], W, PLAN._replace(offsets=PLAN.offsets[:3])), {}),
    (TypeError, ([1.0], W, PLAN), {}),
    (TypeError, (X[:3].double(), W.double(), PLAN), {}),
    (TypeError, (X[:3], W.half(), PLAN), {}),
    (ValueError, (X, W, PLAN), {}),
    (ValueError, (X[:3], W, PLAN), {"from_tokens": False}),
    (ValueError, (torch.zeros(8, 3).t(), W, PLAN), {}),
    (ValueError, (X[:3], W.transpose(1, 2).contiguous().transpose(1, 2), PLAN), {}),
    (ValueError, (X[:3], W[0], PLAN), {}),
    (ValueError, (X[:3], W[:2], PLAN), {}),
    (ValueError, (X[:3, :4].contiguous(), W, PLAN), {}),
    (ValueError, (X[:3], torch.zeros(3, 5, 8), PLAN), {"activation": "silu_gate"}),
    (ValueError, (X[:3], torch.zeros(3, 0, 8), PLAN), {}),
    (ValueError, (X[:3], W, PLAN), {"activation": "gelu"}),
    (TypeError, (X[:3], W, PLAN), {"from_tokens": 1}),
    (RuntimeError, (X[:3], W, PLAN), {}),
    (RuntimeError, (X, W, PLAN), {"from_tokens": False, "activation": "silu_gate"}),
])
def test_expert_linear_refusals(error, args, kwargs):
    with pytest.raises(error):
        expert_linear(*args, **kwargs)


WEIGHTS = torch.zeros(3, 2)


@pytest.mark.parametrize("error,args", [
    (TypeError, (X, WEIGHTS, None)),
    (TypeError, (X.double(), WEIGHTS, PLAN)),
    (TypeError, (X, WEIGHTS.half(), PLAN)),
    (TypeError, (X, 1.0, PLAN)),
    (ValueError, (X[:3], WEIGHTS, PLAN)),
    (ValueError, (torch.zeros(6), WEIGHTS, PLAN)),
    (ValueError, (torch.zeros(8, 6).t(), WEIGHTS, PLAN)),
    (ValueError, (X, WEIGHTS[:2], PLAN)),
    (ValueError, (X, torch.zeros(2, 3).t(), PLAN)),
    (RuntimeError, (X, WEIGHTS, PLAN)),
])
def test_expert_combine_refusals(error, args):
    with pytest.raises(error):
        expert_combine(*args)


@BUILT
def test_c_entry_points_refuse_bad_sizes_before_any_device_call():
    lib = _lib.load()
    null, some, f32 = None, ctypes.c_void_p(256), _lib.TYPE_F32   # never dereferenced

    def norm(rows=4, channels=8, eps=1e-6, gate=0, act=0, type_=f32, residual_type=f32, x=null):
        return lib.dpa4k_residual_norm_forward(x, some, null, null, null, null, some, some, null, null, rows, channels, 1.0, eps, 1, 1,
                                               gate, act, type_, residual_type, null)

    def route(tokens=4, n=8, k=2, groups=1, top=1, scores=0, type_=f32, logits=null):
        return lib.dpa4k_expert_route_forward(logits, null, some, some, null, tokens, n, k, groups, top, scores, 1, 1.0, type_, null)

    def linear(places=4, k=2, inner=1, n=3, k_in=8, n_out=8, gated=0, type_=f32, x=null):
        return lib.dpa4k_expert_linear_forward(x, some, some, null, some, null, places, k, inner, n, k_in, n_out, gated, type_, null)

    def combine(tokens=4, k=2, size=8, type_=f32, y=null):
        return lib.dpa4k_expert_combine_forward(y, some, some, some, tokens, k, size, type_, null)

    def dispatch(slots=4, n=8, offsets=some, experts=some, workspace=null):
        return lib.dpa4k_expert_dispatch(experts, slots, n, offsets, some, some, workspace, 0, null)

    cases = [
        (lambda: norm(rows=-1), "negative"), (lambda: norm(channels=0), "channels"), (lambda: norm(channels=8193), "channels"),
        (lambda: norm(type_=7), "unknown type"), (lambda: norm(residual_type=_lib.TYPE_F16), "residual's type"),
        (lambda: norm(eps=0.0), "eps"), (lambda: norm(eps=math.nan), "eps"), (lambda: norm(gate=3), "gate"),
        (lambda: norm(act=3), "activation"), (lambda: norm(rows=2**60), "overflows"), (lambda: norm(), "null pointer"),
        (lambda: route(tokens=-1), "negative"), (lambda: route(n=0), "experts"), (lambda: route(n=1025), "experts"),
        (lambda: route(groups=3), "groups"), (lambda: route(groups=2, top=3), "top_groups"), (lambda: route(k=9), "k must"),
        (lambda: route(k=0), "k must"), (lambda: route(scores=2), "scores"), (lambda: route(type_=9), "unknown type"),
        (lambda: route(tokens=2**31), "2^31"), (lambda: route(), "null pointer"),
        (lambda: linear(places=-2), "negative"), (lambda: linear(places=3), "k for each token"), (lambda: linear(n=0), "experts"),
        (lambda: linear(k_in=0), "channels"), (lambda: linear(gated=1, n_out=7), "even"), (lambda: linear(type_=5), "unknown type"),
        (lambda: linear(places=2**30, inner=4), "2^31"), (lambda: linear(), "null pointer"),
        (lambda: combine(tokens=-1), "bad sizes"), (lambda: combine(k=0), "bad sizes"), (lambda: combine(type_=4), "unknown type"),
        (lambda: combine(tokens=2**31), "2^31"), (lambda: combine(size=2**32), "2^31"), (lambda: combine(), "null pointer"),
        (lambda: dispatch(slots=-1), "negative"), (lambda: dispatch(slots=2**31), "2^31"), (lambda: dispatch(n=0), "experts"),
        (lambda: dispatch(offsets=null), "null pointer"), (lambda: dispatch(experts=null), "null pointer"),
    ]
    for call, fragment in cases:
        assert call() == _lib.EINVAL, fragment
        assert fragment in lib.dpa4k_last_error().decode(), (fragment, lib.dpa4k_last_error())
    assert dispatch(slots=100000) == _lib.EWORKSPACE
    assert lib.dpa4k_expert_dispatch_workspace_size(100, 8) == 0 < lib.dpa4k_expert_dispatch_workspace_size(100000, 8)
    assert lib.dpa4k_residual_norm_backward(some, some, some, some, null, null, null, null, some, some, some, some, null, some, null, null,
                                            4, 8, 1.0, 1, 1, 0, 0, f32, f32, null, 0, null) == _lib.EWORKSPACE
    assert lib.dpa4k_residual_norm_backward(some, some, some, null, null, null, null, null, some, some, some, some, null, null, null, null,
                                            4, 8, 1.0, 1, 1, 0, 0, f32, f32, null, 0, null) == _lib.EINVAL
    assert lib.dpa4k_expert_linear_backward(some, some, some, some, some, some, some, null, 4, 2, 1, 3, 8, 8, f32, null, 0,
                                            null) == _lib.EWORKSPACE
    assert lib.dpa4k_expert_linear_backward(some, some, some, some, some, null, some, null, 4, 2, 1, 3, 8, 8, f32, some, 4096,
                                            null) == _lib.EINVAL    # no slots
    assert lib.dpa4k_expert_route_backward(some, some, some, null, some, 4, 8, 2, 0, 1, 1.0, f32, null) == _lib.EINVAL
    assert lib.dpa4k_expert_combine_backward(some, some, some, some, null, some, some, 4, 2, 8, f32, null) == _lib.EINVAL
    # nothing to do is no error
    assert route(tokens=0) == linear(places=0) == combine(tokens=0) == norm(rows=0) == _lib.OK


# ---------------------------------------------------------------------------
# the oracles' closed forms against autograd
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("gate,activation", [(None, None), ("full", None), ("full", "sigmoid"), ("row", "silu")])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True)])
def test_residual_norm_oracle_against_autograd(gate, activation, post, pre):
    generator = torch.Generator().manual_seed(3)

    def normal(*shape):
        return torch.randn(*shape, generator=generator, dtype=torch.float64).requires_grad_(True)

    x, residual = normal(4, 3, 6), normal(4, 3, 6)
    g = None if gate is None else normal(4, 3, 6) if gate == "full" else normal(4, 3, 1)
    post_scale, pre_scale, scale = normal(6) if post else None, normal(6) if pre else None, normal(6)
    a = x if not post else x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * post_scale
    act = {None: lambda v: v, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu}[activation]
    h = residual + scale * (1.0 if g is None else act(g)) * a
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * pre_scale if pre else None
    kwargs = dict(post_scale=post_scale, gate=g, gate_activation=activation, residual_scale=scale, pre_scale=pre_scale, post_norm=post,
                  pre_norm=pre, eps=1e-6)
    got_h, got_y = residual_norm_reference(x, residual, **kwargs)
    torch.testing.assert_close(got_h, h.detach(), rtol=1e-12, atol=1e-12)
    dh, dy = torch.randn_like(h), torch.randn_like(h) if pre else None
    outputs, seeds = ((h, y), (dh, dy)) if pre else ((h,), (dh,))
    if pre:
        torch.testing.assert_close(got_y, y.detach(), rtol=1e-12, atol=1e-12)
    leaves = (x, residual, g, post_scale, scale, pre_scale)
    wanted = iter(torch.autograd.grad(outputs, [t for t in leaves if t is not None], seeds))
    for leaf, got in zip(leaves, residual_norm_backward_reference(dh, dy, x, residual, **kwargs)):
        assert (leaf is None) == (got is None)
        if leaf is not None:
            torch.testing.assert_close(got, next(wanted), rtol=1e-10, atol=1e-10)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [True, False])
def test_expert_route_oracle_against_autograd(scores, normalize):
    generator = torch.Generator().manual_seed(5)
    logits = torch.randn(7, 12, generator=generator, dtype=torch.float64)
    logits[1, :10] = -math.inf
    logits[2] = -math.inf
    kwargs = dict(scores=scores, bias=torch.randn(12, generator=generator) * 0.2, groups=3, top_groups=2, normalize=normalize, scale=2.5)
    weights, experts, s = expert_route_reference(logits, 4, **kwargs)
    assert experts[2].tolist() == [-1] * 4 and weights[2].tolist() == [0.0] * 4
    assert experts[1, :2].sort().values.tolist() == [10, 11] and experts[1, 2:].tolist() == [-1, -1]
    leaf = logits.clone().requires_grad_(True)
    shifted = torch.where(torch.isneginf(leaf).all(1, keepdim=True), torch.zeros_like(leaf), leaf)
    table = torch.softmax(shifted, 1) if scores == "softmax" else torch.sigmoid(leaf)
    chosen = torch.where(experts >= 0, table.gather(1, experts.clamp(min=0)), 0.0)
    expected = 2.5 * chosen / ((chosen.sum(1, keepdim=True) + 1e-20) if normalize else 1.0)
    torch.testing.assert_close(weights, expected.detach(), rtol=1e-12, atol=1e-12)
    dw = torch.randn(7, 4, generator=generator, dtype=torch.float64)
    (grad,) = torch.autograd.grad(expected, leaf, dw)
    torch.testing.assert_close(expert_route_backward_reference(dw, logits, 4, **kwargs), torch.nan_to_num(grad), rtol=1e-10, atol=1e-10)


@pytest.mark.parametrize("activation", [None, "silu_gate"])
@pytest.mark.parametrize("from_tokens", [True, False])
def test_expert_products_oracles_against_autograd(activation, from_tokens):
    generator = torch.Generator().manual_seed(6)
    chosen = torch.tensor([[0, 2], [2, -1], [-1, -1], [3, 0], [2, 3]])
    plan = expert_dispatch_reference(chosen, 4)
    x = torch.randn(5 if from_tokens else 10, 3, 6, generator=generator, dtype=torch.float64).requires_grad_(True)
    weight = torch.randn(4, 8, 6, generator=generator, dtype=torch.float64).requires_grad_(True)
    weights = torch.randn(5, 2, generator=generator, dtype=torch.float64).requires_grad_(True)
    n = 8 if activation is None else 4
    rows = []
    for p in range(10):
        slot = int(plan[1][p])
        if slot < 0:
            rows.append(torch.zeros(3, n, dtype=torch.float64))
            continue
        z = x[slot // 2 if from_tokens else p] @ weight[int(chosen.view(-1)[slot])].t()
        rows.append(z if activation is None else torch.nn.functional.silu(z[:, :4]) * z[:, 4:])
    y = torch.stack(rows)
    out = torch.stack([sum(weights[t, j] * y[plan[2][t, j]] for j in range(2) if plan[2][t, j] >= 0) + torch.zeros(3, n).double()
                       for t in range(5)])
    dy, dout = torch.randn(10, 3, n, generator=generator).double(), torch.randn(5, 3, n, generator=generator).double()
    got = expert_linear_reference(x, weight, plan, from_tokens=from_tokens, activation=activation, grad=dy)
    for actual, expected in zip(got, (y.detach(), *torch.autograd.grad(y, (x, weight), dy, retain_graph=True))):
        torch.testing.assert_close(actual, expected, rtol=1e-10, atol=1e-10)
    got = expert_combine_reference(y, weights, plan, dout)
    for actual, expected in zip(got, (out.detach(), *torch.autograd.grad(out, (y, weights), dout))):
        torch.testing.assert_close(actual, expected, rtol=1e-10, atol=1e-10)


@BUILT
def test_gated_backward_refuses_bad_sizes_before_any_device_call():
    lib = _lib.load()
    null, some, f32, bf16 = None, ctypes.c_void_p(256), _lib.TYPE_F32, _lib.TYPE_BF16   # never dereferenced

    def gated(grad=some, before=some, x=some, weight=some, offsets=some, order=some, slots=some, dx=some, dw=some, places=4, k=2, inner=1,
              n=3, k_in=8, n_out=8, type_=bf16, workspace=some, nbytes=1 << 30):
        return lib.dpa4k_expert_gated_backward(grad, before, x, weight, offsets, order, slots, dx, dw, places, k, inner, n, k_in, n_out,
                                               type_, workspace, nbytes, null)

    for call, fragment in [
        (lambda: gated(places=-2), "negative"), (lambda: gated(places=3), "k for each token"), (lambda: gated(n=0), "experts"),
        (lambda: gated(k_in=0), "channels"), (lambda: gated(n_out=7), "even"), (lambda: gated(type_=5), "unknown type"),
        (lambda: gated(places=2**30, inner=4), "2^31"), (lambda: gated(grad=null), "null pointer"), (lambda: gated(before=null), "null pointer"),
        (lambda: gated(x=null), "null pointer"), (lambda: gated(weight=null), "null pointer"), (lambda: gated(offsets=null), "null pointer"),
        (lambda: gated(slots=null), "null pointer"),
    ]:
        assert call() == _lib.EINVAL, fragment
        assert fragment in lib.dpa4k_last_error().decode(), (fragment, lib.dpa4k_last_error())
    sizes = 4, 2, 1, 3, 8, 8
    assert gated(workspace=null) == _lib.EWORKSPACE
    assert gated(nbytes=lib.dpa4k_expert_gated_workspace_size(*sizes, 1, 1, 1, bf16) - 1) == _lib.EWORKSPACE
    # dz lies in front of what the products need: two parts in 16 bits, one in 32
    rest = lib.dpa4k_expert_linear_workspace_size(*sizes, 1, 1, 1)
    assert lib.dpa4k_expert_gated_workspace_size(*sizes, 1, 1, 1, bf16) == rest + 2 * 256
    assert lib.dpa4k_expert_gated_workspace_size(*sizes, 1, 1, 1, f32) == rest + 256
    assert lib.dpa4k_expert_gated_workspace_size(0, *sizes[1:], 1, 1, 1, bf16) == 0
    assert gated(dx=null, dw=null, workspace=null) == gated(places=0, dw=null, workspace=null) == _lib.OK


@BUILT
def test_workspace_of_the_matrices_gradient():
    """Partial sums for as many chunks as segments of any lengths can have, none where no segment can be cut."""
    lib = _lib.load()

    def chunks(rows, experts, k_in=256, n_out=256):
        return lib.dpa4k_expert_linear_workspace_size(rows, 1, 1, experts, k_in, n_out, 0, 0, 1) // (4 * k_in * n_out)

    assert chunks(32768, 128) == 0                 # 32,768 rows are one chunk
    for rows, experts in ((32769, 128), (65536, 128), (65538, 128), (1_000_000, 128), (5_000_000, 128)):
        most = 0
        for cut in range(1, min(experts, rows // 32769) + 1):    # segments of one row more than a chunk, the last takes the rest
            lengths = [32769] * (cut - 1) + [rows - 32769 * (cut - 1)]
            most = max(most, sum(math.ceil(n / 32768) for n in lengths))
        assert most <= chunks(rows, experts) <= 2 * rows // 32768, (rows, most)
