"""8-bit paged KV cache on the GPU: contiguous inputs that start off a 16-byte boundary."""

import pytest
import torch

from test_paged8_gpu import _pool, _table

pytestmark = pytest.mark.gpu


def _shifted(x, by=1):
    """The same numbers, contiguous, ``by`` elements past an allocation's start."""
    out = torch.empty(x.numel() + by, dtype=x.dtype, device=x.device)[by:].view(x.shape)
    return out.copy_(x)


@pytest.mark.parametrize("S,hd,bs", [(1, 128, 16), (3, 64, 64), (40, 128, 64), (1, 96, 16), (5, 48, 24)])
def test_inputs_off_a_16_byte_boundary(S, hd, bs):
    from verl_omni_b200.ops.paged8 import append_paged8, attend_paged8

    torch.manual_seed(0)
    B, Hk, rep, start = 3, 2, 4, 37
    width = -(-(start + S) // bs)
    pages = B * width + 2
    table = _table(B, width, pages)
    first = torch.full((B,), start, dtype=torch.int32, device="cuda")
    k, v = (torch.randn(B, Hk, S, hd, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(B, Hk * rep, S, hd, device="cuda").bfloat16()
    out = []
    for shift in (0, 1, 3, 4):
        (kp, ks), (vp, vs) = _pool(pages, Hk, bs, hd), _pool(pages, Hk, bs, hd, seed=1)
        a, b, c = ((_shifted(t, shift) if shift else t) for t in (k, v, q))
        assert a.is_contiguous() and (a.data_ptr() % 16 != 0) == (shift != 0)
        append_paged8(a, b, kp, vp, ks, vs, table, first)
        o = attend_paged8(c, kp, vp, ks, vs, table, first + S)
        out.append((kp.view(torch.uint8), vp.view(torch.uint8), ks, vs, o))
    for other in out[1:]:
        for x, y in zip(out[0], other):
            assert torch.equal(x, y)
