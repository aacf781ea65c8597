"""Logits processing on the CPU: the oracle against a token-by-token definition, packing, refusals."""

import math

import pytest
import torch

from verl_omni_b200.ops.logits import pack_allowed, process_logits


def test_definition_token_by_token():
    x = torch.tensor([[2.0, -2.0, 0.5, -0.5, 1.0, -math.inf]])
    hist = torch.tensor([[0, 1, 1, 2, 9, -1, 2, 5]])
    lens, pl = torch.tensor([7], dtype=torch.int32), torch.tensor([2], dtype=torch.int32)
    y = process_logits(x, hist, lens, pl, repetition=2.0, presence=0.25, frequency=0.5, bias=torch.arange(6).float(),
                       allowed=pack_allowed(torch.tensor([[True, True, True, False, True, True]])))
    # token 0: prompt only; 1: prompt and once in the response; 2: twice in the response; 5 lies past the length
    assert y[0].tolist() == [1.0, -4.0 - 0.75 + 1, 0.25 - 1.25 + 2, -math.inf, 5.0, -math.inf]


def test_pack_allowed_round_trip():
    m = torch.rand(3, 70) < 0.5
    w = pack_allowed(m)
    assert w.shape == (3, 3) and w.dtype == torch.int32
    bits = (w[:, torch.arange(70) // 32] >> (torch.arange(70) % 32)) & 1
    assert torch.equal(bits == 1, m)


def test_gradient_and_rows():
    torch.manual_seed(0)
    x = torch.randn(4, 12, dtype=torch.float32, requires_grad=True)
    rows = torch.tensor([1, 0, 1, 5], dtype=torch.int32)  # the last names no sequence: no history
    hist = torch.randint(0, 12, (2, 6))
    lens = torch.tensor([6, 3, 0, 6], dtype=torch.int32)
    y = process_logits(x, hist, lens, rows=rows, repetition=1.5, allowed=pack_allowed(torch.rand(1, 12) < 0.8))
    g = torch.randn(4, 12)
    (dx,) = torch.autograd.grad(torch.where(y.isfinite(), y, 0.0), x, g)
    for r in range(4):
        seen = set(hist[int(rows[r])][:int(lens[r])].tolist()) if rows[r] < 2 else set()
        for v in range(12):
            f = (1 / 1.5 if x[r, v] > 0 else 1.5) if v in seen else 1.0
            want = 0.0 if y[r, v].isinf() else g[r, v] * f
            assert abs(float(dx[r, v]) - float(want)) < 1e-5
    torch.testing.assert_close(y[2:][y[2:].isfinite()], x[2:][y[2:].isfinite()])


def test_refusals():
    x, h = torch.randn(2, 64), torch.zeros(2, 4, dtype=torch.int64)
    i2 = torch.ones(2, dtype=torch.int32)
    for bad in (dict(x=x[0]), dict(history=h[:1]), dict(history=h.float()), dict(history=h, lens=i2.long()), dict(history=h, lens=i2[:1]),
                dict(repetition=torch.ones(3)), dict(presence=torch.ones(2).double()), dict(bias=torch.zeros(63)),
                dict(allowed=torch.zeros(2, 3, dtype=torch.int32)), dict(allowed=torch.zeros(2, 2, dtype=torch.int64)),
                dict(bias=torch.zeros(64, requires_grad=True))):
        with pytest.raises(ValueError):
            process_logits(**{"x": x, **bad})
