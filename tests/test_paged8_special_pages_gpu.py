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


@pytest.mark.parametrize("S,hd", [(1, 128), (3, 64), (1, 96), (40, 128), (40, 64)])
def test_page_scales_that_are_no_powers_of_two(S, hd):
    """Codes written elsewhere, with any positive scale (zero for a page of zero keys).  For many rows the f16 tiles hold
    code * scale / largest to 2^-11: twice (the factor and the product), of sum |q k| * scale for a score and of sum p |v|."""
    from verl_omni_b200.ops.paged8 import attend_paged8

    torch.manual_seed(0)
    B, Hk, rep, bs, n = 3, 2, 4, 16, 500
    table = _table(B, -(-n // bs), 100)
    (kp, ks), (vp, vs) = _pool(100, Hk, bs, hd), _pool(100, Hk, bs, hd, seed=1)
    ks, vs = (t * (1 + torch.rand(t.shape, device="cuda")) for t in (ks, vs))
    ks[int(table[0, 3])] = 0.0
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    q = torch.randn(B, Hk * rep, S, hd, device="cuda").bfloat16()
    scale = 0.2 * hd ** -0.5
    got = attend_paged8(q, kp, vp, ks, vs, table, lens, scale=scale)
    want, tol = _attend64(q, kp, vp, ks, vs, table, lens, None, scale)
    if S * rep > 16:
        plus = vp.view(torch.uint8).bitwise_and(0x7F).view(vp.dtype)
        weighed, _ = _attend64(q, kp, plus, ks, vs, table, lens, None, scale)  # sum p |v|
        terms = float((kp.float().abs() * ks[..., None, None]).sum(-1).amax() * q.float().abs().amax() * scale)
        tol = tol + (2 * terms + 1) * 2.0 ** -10 * weighed
    _agree(got, want, tol)
