"""What ``kernels.optim.AdamW`` does with its state when something is refused, on the CPU.

A stand-in takes the place of the GPU entry points: plans are the real ones (they are
host work), a step is the oracle's chain.  Each test ends with the state as it should be,
bit for bit, after the refusal.
"""
from __future__ import annotations

import pytest
import torch

from bysj_amd.kernels import _lib, optim
from oracle import optim as ref

pytestmark = pytest.mark.skipif(not _lib.LIBRARY_PATH.exists(), reason="libdpa4k.so is not built")


class _Native:
    """The entry points of ``kernels._C`` on CPU tensors."""

    def __init__(self):
        from bysj_amd.kernels import _C

        self.adamw_plan = _C.adamw_plan

    @staticmethod
    def grad_norm(grads, limit, dtypes):
        norm = torch.sqrt(sum(g.double().square().sum() for g in grads))
        return norm.float(), (limit / (norm + 1e-6)).clamp(max=1.0).float()

    @staticmethod
    def adamw_step(plan, grads, grad_dtype, lr, lr_tensor, beta1, beta2, eps, weight_decay, factor, seed):
        n = len(plan.params)
        steps = plan.words[: n * _lib.ADAMW_RECORD_BYTES].view(torch.int64).view(n, -1)[:, _lib.ADAMW_STEP_OFFSET // 8]
        for k, (p, g, part) in enumerate(zip(plan.params, grads, plan.parts() if plan.state_bits == 8 else [None] * n)):
            if g is None:
                continue
            steps[k] += 1
            if plan.state_bits == 8:    # anything that differs from step to step
                part[0].fill_(int(steps[k]))
                part[1].fill_(100 + int(steps[k]))
                continue
            m, v = plan.exp_avgs[k], plan.exp_avg_sqs[k]
            new = ref.adamw_chain(p.detach().view(-1), g.view(-1), m.view(-1), v.view(-1), int(steps[k]),
                                  lr=float(lr if lr_tensor is None else lr_tensor), betas=(beta1, beta2), eps=eps,
                                  weight_decay=weight_decay, factor=1.0 if factor is None else float(factor), seed=seed)
            for to, value in zip((p, m, v), new):
                to.detach().view(-1).copy_(value)


@pytest.fixture(autouse=True)
def native(monkeypatch):
    stand_in = _Native()
    monkeypatch.setattr(optim, "_extension", lambda name: stand_in)
    monkeypatch.setattr(optim, "require_dcu", lambda *tensors: None)
    return stand_in


def _trained(bits=32, **more):
    """An optimiser of two groups after two steps, and its parameters with gradients."""
    generator = torch.Generator().manual_seed(0)
    params = [torch.randn(2, 3, generator=generator).requires_grad_(True), torch.randn(40, generator=generator).requires_grad_(True)]
    optimiser = optim.AdamW([{"params": params[:1]}, {"params": params[1:], "lr": 1e-2}], state_bits=bits, **more)
    for p in params:
        p.grad = torch.randn(p.shape, generator=generator)
    optimiser.step()
    optimiser.step()
    return optimiser, params


def _same(a, b):
    assert type(a) is type(b) or (isinstance(a, (int, float)) and isinstance(b, (int, float)))
    if isinstance(a, torch.Tensor):
        assert a.dtype == b.dtype and torch.equal(a, b)
    elif isinstance(a, dict):
        assert a.keys() == b.keys()
        for key in a:
            _same(a[key], b[key])
    elif isinstance(a, (list, tuple)):
        assert len(a) == len(b)
        for x, y in zip(a, b):
            _same(x, y)
    else:
        assert a == b


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
@pytest.mark.parametrize("which", [[0], [0, 1]])
def test_a_step_refuses_parameters_of_a_dtype_it_does_not_have(dtype, which, bits):
    """After ``model.half()`` or ``model.double()``: no parameter is left out silently, no moment is lost."""
    optimiser, params = _trained(bits, max_norm=1.0)
    before, held = optimiser.state_dict(), [(p.data, p.grad) for p in params]
    for k in which:
        p = params[k]
        p.grad, p.data = None, p.data.to(dtype)
        p.grad = held[k][1].to(dtype)
    values = [p.detach().clone() for p in params]
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        optimiser.step()
    _same([p.detach() for p in params], values)
    for p, (data, grad) in zip(params, held):
        p.grad, p.data = None, data
        p.grad = grad
    _same(optimiser.state_dict(), before)
    optimiser.step()
    assert [optimiser.state_dict()["state"][k]["step"] for k in (0, 1)] == [3, 3]


@pytest.mark.parametrize("error,group", [
    (TypeError, {"params": [torch.zeros(3, dtype=torch.float16)]}),
    (ValueError, {"params": [torch.zeros(4)[::2]]}),
    (ValueError, {"params": [torch.zeros(3)], "lr": -1.0}),
    (TypeError, {"params": [torch.zeros(3)], "betas": 0.9}),
])
def test_a_refused_group_is_not_kept(error, group):
    optimiser, params = _trained()
    before = optimiser.state_dict()
    with pytest.raises(error):
        optimiser.add_param_group(group)
    assert [g["params"] for g in optimiser.param_groups] == [params[:1], params[1:]]
    _same(optimiser.state_dict(), before)
    optimiser.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_that_cannot_list_its_parameters_keeps_the_moments(bits):
    """A parameter's memory becomes strided: the step raises; with the layout put right training goes on where it was."""
    optimiser, params = _trained(bits)
    before = optimiser.state_dict()
    params[1].data = torch.randn(80)[::2]
    with pytest.raises(ValueError, match="contiguous"):
        optimiser.step()
    _same(optimiser.state_dict(), before)
    params[1].data = params[1].data.contiguous()
    optimiser.step()
    assert [optimiser.state_dict()["state"][k]["step"] for k in (0, 1)] == [3, 3]


def _without(part, name):
    return {key: value for key, value in part.items() if key != name}


@pytest.mark.parametrize("error,bits,change", [
    (ValueError, 32, lambda d: d["state"][1].update(exp_avg=torch.zeros(39))),
    (ValueError, 32, lambda d: d["state"][0].update(exp_avg=torch.zeros(3, 2))),    # as many elements
    (ValueError, 32, lambda d: d["state"][0].update(exp_avg_sq=torch.zeros(()))),
    (ValueError, 32, lambda d: d["state"].update({1: _without(d["state"][1], "exp_avg_sq")})),
    (ValueError, 32, lambda d: d["state"].update({1: _without(d["state"][1], "step")})),
    (ValueError, 32, lambda d: d["state"][1].update(step=-1)),
    (ValueError, 32, lambda d: d["state"][1].update(step=2.5)),
    (TypeError, 32, lambda d: d["state"][1].update(exp_avg=torch.zeros(40, dtype=torch.int32))),
    (ValueError, 32, lambda d: d["state"].update({2: d["state"][1]})),
    (ValueError, 8, lambda d: d["state"][1].update(codes=torch.zeros(2, 32, dtype=torch.uint8))),
    (ValueError, 8, lambda d: d["state"][1].update(codes=torch.zeros(1, dtype=torch.uint8))),    # would be broadcast
    (ValueError, 8, lambda d: d["state"][1].update(scales=torch.zeros(2, 1, dtype=torch.uint8))),
    (TypeError, 8, lambda d: d["state"][1].update(codes=torch.zeros(2, 64))),
    (ValueError, 32, lambda d: d.update(state_bits=8)),
    (ValueError, 32, lambda d: d["param_groups"][1].update(lr=-1.0)),
    (TypeError, 32, lambda d: d["param_groups"][1].update(betas=0.9)),
    (ValueError, 32, lambda d: d["param_groups"][1].pop("eps")),
    (ValueError, 32, lambda d: d["param_groups"][1].update(amsgrad=True)),
    (ValueError, 32, lambda d: d["param_groups"].pop()),
    (ValueError, 32, lambda d: d["param_groups"][1]["params"].append(2)),
])
def test_a_refused_checkpoint_changes_nothing(error, bits, change):
    optimiser, params = _trained(bits)
    twin, others = _trained(bits)
    before, checkpoint = optimiser.state_dict(), optimiser.state_dict()
    checkpoint["param_groups"][0]["lr"] = 0.5
    change(checkpoint)
    with pytest.raises(error):
        optimiser.load_state_dict(checkpoint)
    _same(optimiser.state_dict(), before)
    optimiser.step()
    twin.step()
    _same([p.detach() for p in params], [p.detach() for p in others])
    _same(optimiser.state_dict(), twin.state_dict())


@pytest.mark.parametrize("bits", [32, 8])
def test_a_checkpoint_that_cannot_be_listed_changes_nothing(bits, native, monkeypatch):
    """No memory for the new plans."""
    optimiser, _ = _trained(bits)
    before, checkpoint = optimiser.state_dict(), optimiser.state_dict()
    checkpoint["param_groups"][0]["lr"] = 0.5

    def refuse(*args):
        raise RuntimeError("out of memory")

    with monkeypatch.context() as patched:
        patched.setattr(native, "adamw_plan", refuse)
        with pytest.raises(RuntimeError, match="memory"):
            optimiser.load_state_dict(checkpoint)
    _same(optimiser.state_dict(), before)
    optimiser.load_state_dict(checkpoint)
    _same(optimiser.state_dict(), checkpoint)


@pytest.mark.parametrize("bits", [32, 8])
def test_hooks_see_the_whole_checkpoint(bits):
    optimiser, _ = _trained(bits)
    saved, given, loaded = [], [], []
    optimiser.register_state_dict_post_hook(lambda o, d: saved.append({**d}))
    checkpoint = optimiser.state_dict()
    assert saved[0].keys() == checkpoint.keys()
    _same(saved[0], checkpoint)
    assert sorted(checkpoint["state"]) == [0, 1]

    def longer(o, d):
        given.append(d["state"].keys())
        return {**d, "state": {k: {**part, "step": part["step"] + 5} for k, part in d["state"].items()}}

    optimiser.register_load_state_dict_pre_hook(longer)
    optimiser.register_load_state_dict_post_hook(lambda o: loaded.append(o.state_dict()))
    for turn in (1, 2):
        optimiser.load_state_dict(checkpoint)
        assert given == [{0, 1}] * turn
        assert [loaded[-1]["state"][k]["step"] for k in (0, 1)] == [7, 7]
    for name, value in checkpoint["state"][1].items():
        if name != "step":
            assert torch.equal(loaded[-1]["state"][1][name], value)


def test_hooks_of_a_refused_checkpoint_do_not_pile_up():
    optimiser, _ = _trained()
    checkpoint = optimiser.state_dict()
    for _ in range(2):
        with pytest.raises(ValueError):
            optimiser.load_state_dict({**checkpoint, "state_bits": 8})
    optimiser.load_state_dict(checkpoint)
    _same(optimiser.state_dict(), checkpoint)


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_taken_out_of_a_group_leave_the_checkpoint(bits):
    """Before the next step too, and with the whole last group."""
    optimiser, params = _trained(bits)
    before = optimiser.state_dict()["state"]
    group = optimiser.param_groups.pop()
    assert sorted(optimiser.state_dict()["state"]) == [0]
    _same(optimiser.state_dict()["state"][0], before[0])
    optimiser.step()
    assert sorted(optimiser.state_dict()["state"]) == [0] and len(optimiser._plans) == 1
    optimiser.add_param_group(group)    # begins from zero: its moments went with it
    optimiser.step()
    assert [optimiser.state_dict()["state"][k]["step"] for k in (0, 1)] == [4, 1]
    del optimiser.param_groups[1]["params"][0]
    assert sorted(optimiser.state_dict()["state"]) == [0]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_of_another_shape_is_refused(bits):
    """As many elements in another order: moments taken over by their place would belong to other elements."""
    optimiser, params = _trained(bits)
    before, p = optimiser.state_dict(), params[0]
    data, grad = p.data, p.grad
    p.grad, p.data = None, p.data.t().contiguous()
    p.grad = grad.t().contiguous()
    with pytest.raises(ValueError, match="shape"):
        optimiser.step()
    _same(optimiser.state_dict(), before)
    p.grad, p.data = None, data.clone()
    p.grad = grad
    optimiser.step()
    assert optimiser.state_dict()["state"][0]["step"] == 3


@pytest.mark.parametrize("bits", [32, 8])
def test_memory_that_a_plan_lists_is_not_given_to_others(bits):
    """A parameter lets go of its memory: nothing else may get that address while a plan would write to it."""
    p = torch.zeros(1000)
    plan, address = optim.adamw_plan([p], state_bits=bits), p.data_ptr()
    p.data = torch.empty(0)
    others = [torch.zeros(size) for size in [1000] * 40 + [900, 500, 100]]
    assert address not in [t.data_ptr() for t in others]
    p.data = others[0]
    with pytest.raises(RuntimeError, match="moved"):
        optim.adamw_step(plan, [torch.ones(1000)], lr=1.0)
    assert not any(t.any() for t in others)


def test_a_learning_rate_tensor_is_on_the_parameters_device():
    """Refused by the constructor, not by the first step; a checkpoint that was loaded to the CPU follows the parameters."""
    there = torch.zeros(3, device="meta")
    with pytest.raises(ValueError, match="device"):
        optim.AdamW([there], lr=torch.tensor(0.1))
    optimiser = optim.AdamW([there], lr=torch.tensor(0.1, device="meta"))
    checkpoint = optimiser.state_dict()
    checkpoint["param_groups"][0]["lr"] = torch.tensor(0.2)
    optimiser.load_state_dict(checkpoint)
    assert optimiser.param_groups[0]["lr"].device == there.device
    assert checkpoint["param_groups"][0]["lr"].device.type == "cpu"
    optim.AdamW([torch.zeros(3)], lr=torch.tensor(0.1, device="meta"))    # parameters that are still to be moved


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("error,option,value", [
    (ValueError, "lr", -1.0), (TypeError, "lr", "1"), (ValueError, "lr", torch.zeros(2)), (ValueError, "lr", torch.zeros((), device="meta")),
    (TypeError, "betas", 0.9), (ValueError, "betas", (0.9, 1.0)), (ValueError, "eps", 0.0), (ValueError, "weight_decay", -0.1),
])
def test_a_step_is_refused_whole(error, option, value, bits):
    """An option of the second group goes wrong between two steps: the first group takes no step either."""
    optimiser, params = _trained(bits)
    before, values = optimiser.state_dict(), [p.detach().clone() for p in params]
    held = optimiser.param_groups[1][option]
    optimiser.param_groups[1][option] = value
    with pytest.raises(error):
        optimiser.step()
    optimiser.param_groups[1][option] = held
    _same(optimiser.state_dict(), before)
    _same([p.detach() for p in params], values)
