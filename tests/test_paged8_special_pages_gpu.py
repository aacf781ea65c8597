"""8-bit paged attention on the GPU: pages that hold no finite value."""

import pytest
import torch

from test_paged8_gpu import _agree, _attend64, _pool, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,hd", [(1, 128), (3, 64), (1, 96), (40, 128), (40, 64), (300, 128)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_page_of_nan_alone_reaches_the_rows_that_see_it(which, S, hd):
    """Rows of NaN do not count for a page's scale: it is the smallest there is, far below those beside it."""
    from verl_omni_b200.ops.paged8 import append_paged8, attend_paged8

    torch.manual_seed(0)
    B, Hk, rep, bs, n = 2, 2, 4, 32, 320
    table = _table(B, n // bs, 24)
    (kp, ks), (vp, vs) = _pool(24, Hk, bs, hd), _pool(24, Hk, bs, hd, seed=1)
    k, v = (torch.randn(B, Hk, n, hd, device="cuda").bfloat16() for _ in range(2))
    (k if which == "k" else v)[1, :, 2 * bs:3 * bs] = float("nan")
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    append_paged8(k, v, kp, vp, ks, vs, table, zero)
    assert float((ks if which == "k" else vs)[int(table[1, 2]), 0]) == 2.0 ** -100
    q = torch.randn(B, Hk * rep, S, hd, device="cuda").bfloat16()
    got = attend_paged8(q, kp, vp, ks, vs, table, zero + n)
    want, tol = _attend64(q, kp, vp, ks, vs, table, zero + n, None, hd ** -0.5)
    assert bool(want[0].isfinite().all()) and bool(want[1, -1].isnan().all())
    _agree(got, want, tol)
