"""Derivatives that the rollout's operators do not have are refused (those of the CPU oracle of the logits are torch's)."""

import pytest
import torch
import torch.autograd.forward_ad as fwd


def test_attention_refuses_tangents():
    from verl_omni_b200.ops.paged8 import PagedKVCache8

    c = PagedKVCache8(1, 2, 1, 4, 16, "cpu")
    v = c.batch([c.add_sequence()]).views()[0]
    v.append(torch.randn(1, 1, 3, 16), torch.randn(1, 1, 3, 16))
    q = torch.randn(1, 2, 1, 16)
    with fwd.dual_level():
        v.attend(q)
        with pytest.raises(ValueError, match="forward-mode"):
            v.attend(fwd.make_dual(q, torch.ones_like(q)))


def test_cpu_logits_carry_tangents():
    from verl_omni_b200.ops.logits import process_logits

    x = torch.tensor([[2.0, -2.0, 1.0]])
    with fwd.dual_level():
        y = process_logits(fwd.make_dual(x, torch.ones_like(x)), torch.tensor([[0, 1]]), repetition=2.0)
        assert fwd.unpack_dual(y).tangent.tolist() == [[0.5, 2.0, 1.0]]
