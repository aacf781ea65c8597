"""Derivatives that the logits kernel does not have are refused instead of left out."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


def test_second_derivatives():
    from verl_omni_b200.ops.logits import process_logits

    x = torch.randn(2, 64, device="cuda", requires_grad=True)
    g = torch.randn(2, 64, device="cuda", requires_grad=True)
    y = process_logits(x, torch.zeros(2, 3, dtype=torch.int64, device="cuda"), repetition=1.5)
    (dx,) = torch.autograd.grad(y, x, g, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (dx.sum() + (x * x).sum()).backward()  # the second term alone has a graph


def test_tangents():
    from verl_omni_b200.ops.logits import process_logits

    x = torch.randn(2, 64, device="cuda")
    with fwd.dual_level():
        process_logits(x)
        with pytest.raises(ValueError, match="forward-mode"):
            process_logits(fwd.make_dual(x, torch.ones_like(x)))
        with pytest.raises((ValueError, RuntimeError)):
            process_logits(fwd.make_dual(x.clone().requires_grad_(True), torch.ones_like(x)))
