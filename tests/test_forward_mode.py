"""Forward-mode tangents are refused, never lost: ``apply_function`` on the CPU with a function of its own."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from bysj_amd.kernels.native import apply_function


class _Twice(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, factor):
        ctx.save_for_backward(x)
        return x * factor + (0.0 if bias is None else bias)

    @staticmethod
    def backward(ctx, grad):
        return 2.0 * grad, None, None


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", [0, 1])
def test_a_tangent_is_refused(which, grad):
    args = [torch.randn(3), torch.randn(3), 2.0]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        assert torch.equal(apply_function(_Twice, *args), args[0] * 2.0 + args[1])    # no tangent among them
        args[which] = forward_ad.make_dual(args[which], torch.ones(3))
        with pytest.raises(NotImplementedError):
            apply_function(_Twice, *args)


def test_without_tangents_nothing_changes():
    x = torch.randn(3)
    assert torch.equal(apply_function(_Twice, x, None, 2.0), x * 2.0)
    with forward_ad.dual_level(), torch.inference_mode():    # where tangents do not exist
        assert torch.equal(apply_function(_Twice, forward_ad.make_dual(x, torch.ones(3)), None, 2.0), x * 2.0)
    y = apply_function(_Twice, x.requires_grad_(True), None, 2.0)
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], torch.full((3,), 2.0))
