"""8-bit paged attention on the GPU: pages outside the pool read as zeros whatever their place in shared memory held before."""

import math

import pytest
import torch

from test_paged8_gpu import _agree, _attend64, _pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rep,S", [(4, 3), (1, 2), (5, 3), (8, 1), (16, 20)])
@pytest.mark.parametrize("hd", [64, 128])
def test_missing_pages_after_nan_values(hd, rep, S):
    """Two of three sequences hold only NaN values, the third one's last pages are outside the pool.  With three tiles a sequence and
    about twenty a block, the tile of those pages takes a place that held the values of a NaN sequence."""
    from verl_omni_b200.ops.paged8 import attend_paged8

    B, bs, n = 2000, 64, 384
    width = n // bs
    kp, ks = _pool(2 * width, 1, bs, hd)
    vp, vs = _pool(2 * width, 1, bs, hd, seed=1)
    vp.view(torch.uint8)[:width] = 0x7F
    table = torch.arange(width, dtype=torch.int32, device="cuda").repeat(B, 1)
    clean = torch.arange(2, B, 3, device="cuda")
    table[clean] += width
    table[clean, -2] = 2 * width
    table[clean, -1] = -1
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    q = torch.randn(B, rep, S, hd, device="cuda").bfloat16()
    got = attend_paged8(q, kp, vp, ks, vs, table, lens)
    assert bool(got[clean].isfinite().all())
    bad = torch.ones(B, dtype=torch.bool, device="cuda")
    bad[clean] = False
    assert bool(got[bad].isnan().all())
    pick = clean[:: max(1, len(clean) // 12)]
    want, tol = _attend64(q[pick], kp, vp, ks, vs, table[pick], lens[pick], None, hd ** -0.5)
    _agree(got[pick], want, tol)
    assert not math.isnan(float(want.sum()))
