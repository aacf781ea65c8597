"""8-bit paged attention on the GPU where weights span many orders of magnitude: a key far above the rest (the first token of
most language models) whose value is small, so that the output is made of the small weights."""

import math

import pytest
import torch

from test_paged8_gpu import E4M3, _agree, _table, _values

pytestmark = pytest.mark.gpu

TILE = 128  # keys whose weights share a reference in the kernel for few query rows


def _codes(x):
    """fp32 rows [pages, Hk, block, hd] -> e4m3 codes and power-of-two page scales."""
    amax = x.abs().amax((2, 3))
    scale = torch.exp2(torch.ceil(torch.log2(amax.clamp(min=2.0 ** -80) / 448)))
    return (x / scale[..., None, None]).to(E4M3), scale


def _case(B, Hk, rep, hd, bs, n, S, gap, sinks, seed=0):
    """``sinks`` leading keys ``gap`` nats above the others, their values zero."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = -(-n // bs)
    table = _table(B, width, B * width + 2, seed)
    k = torch.randn(B * width + 2, Hk, bs, hd, device="cuda", generator=g)
    v = torch.randn(B * width + 2, Hk, bs, hd, device="cuda", generator=g)
    q = torch.randn(B, Hk * rep, S, hd, device="cuda", generator=g) * 0.05  # scores of the others: spread of about half a nat
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    left = sinks
    for page in range(-(-sinks // bs)):
        m = min(bs, left)
        i = table[:, page].long()
        k[i, :, :m, :] = 0.0
        k[i, :, :m, 0] = gap / 8
        v[i, :, :m] = 0.0
        left -= m
    (kp, ks), (vp, vs) = _codes(k), _codes(v)
    return q.bfloat16(), kp, vp, ks, vs, table, torch.full((B,), n, dtype=torch.int32, device="cuda")


def _attend64(q, kp, vp, ks, vs, table, lens, scale, few):
    """(output, tolerance) in 64 bits.

    Output: bf16, 2^-8 of |o|.  Weights in the kernel for few rows: two e4m3 parts, 2^-8 each, and f16 between (2^-11): 1.25 * 2^-8 of
    sum p |v|; below, a step of 2^-14 on a weight of 256 for the reference, a rounding of 2^-23 of it.  The reference is the running
    maximum of the row, or, where the 128 keys of the tile lie more than 2^4 below, less than twice the largest of them; of the
    code at the tile's largest v scale.  For many rows: f16, 2^-11 (2^-10 with the fp32 sums) down to 2^-21, and a step of 2^-24
    on a weight of 2^7 at least: 2^-32 of the row's largest."""
    B, Hq, S, hd = q.shape
    Hk, bs = kp.shape[1:3]
    rep = Hq // Hk
    out = torch.zeros(B, S, Hq, hd, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = int(lens[b])
        ids = table[b, :-(-n // bs)].long()
        for h in range(Hk):
            code_k, code_v = (_values(p.view(torch.uint8)[ids, h]) for p in (kp, vp))  # [pages, bs, hd]
            sv = vs[ids, h].double()[:, None].expand(-1, bs).reshape(-1)[:n]
            k = (code_k * ks[ids, h].double()[:, None, None]).reshape(-1, hd)[:n]
            cv = code_v.reshape(-1, hd)[:n]
            v = cv * sv[:, None]
            pad = -n % TILE
            top_v = torch.nn.functional.pad(sv, (0, pad)).view(-1, TILE).amax(1)
            if not few:
                top_v = torch.full_like(top_v, float(sv.max()))
            coarse = torch.nn.functional.pad(cv.abs(), (0, 0, 0, pad)).view(-1, TILE, hd).sum(1) * top_v[:, None]  # [tiles, hd]
            for i in range(S):
                lim = n - S + i + 1
                z = torch.einsum("gd,td->gt", q[b, h * rep:(h + 1) * rep, i].double(), k[:lim]) * scale
                p = torch.softmax(z, -1)
                o = p @ v[:lim]
                a = p @ v[:lim].abs()
                pt = torch.nn.functional.pad(p, (0, n + pad - lim)).view(rep, -1, TILE).amax(-1)
                t = 2.0 ** -8 * o.abs()
                if few:
                    below = (p.amax(-1, keepdim=True) / pt.clamp(min=1e-300)).clamp(2.0, 16.0)
                    t = t + 1.25 * 2.0 ** -8 * a + 2.0 ** -23 * ((below * pt) @ coarse)
                else:
                    t = t + 2.0 ** -10 * a + 2.0 ** -32 * p.amax(-1, keepdim=True) * coarse.sum(0)
                out[b, i, h * rep:(h + 1) * rep] = o
                tol[b, i, h * rep:(h + 1) * rep] = t
    return out, tol


@pytest.mark.parametrize("gap,sinks", [(9.0, 1), (13.0, 1), (14.0, 1), (16.0, 128), (30.0, 256)])
@pytest.mark.parametrize("B,Hk,rep,hd,bs,n,S", [(32, 2, 8, 128, 64, 8191, 1), (24, 4, 4, 64, 16, 6000, 1), (1, 1, 16, 128, 128, 32768, 1),
                                                (24, 2, 5, 128, 16, 5001, 3), (1, 1, 2, 64, 8, 300, 1)])
def test_small_weights_behind_a_sink_few_rows(B, Hk, rep, hd, bs, n, S, gap, sinks):
    from verl_omni_b200.ops.paged8 import attend_paged8

    c = _case(B, Hk, rep, hd, bs, n, S, gap, sinks)
    got = attend_paged8(*c, scale=1.0)
    _agree(got, *_attend64(*c, 1.0, few=True))


@pytest.mark.parametrize("gap", [9.0, 13.0, 15.0, 16.0])
@pytest.mark.parametrize("B,Hk,rep,hd,bs,n,S", [(8, 2, 8, 128, 64, 8191, 33), (24, 2, 5, 64, 16, 3000, 60)])
def test_small_weights_behind_a_sink_many_rows(B, Hk, rep, hd, bs, n, S, gap):
    from verl_omni_b200.ops.paged8 import attend_paged8

    c = _case(B, Hk, rep, hd, bs, n, S, gap, 1)
    got = attend_paged8(*c, scale=1.0)
    _agree(got, *_attend64(*c, 1.0, few=False))


@pytest.mark.parametrize("rep,S", [(8, 1), (2, 1), (16, 1), (5, 3)])
@pytest.mark.parametrize("hd", [64, 128])
def test_queries_with_one_large_element(hd, rep, S):
    """Eight elements 2^14 below the largest, which meets zeros in every key: the scores come from the small ones.  Queries are two
    e4m3 numbers relative to a power of two 2^e with max |q| <= 448 * 2^e, the low one times 16: a rounding of 2^-14 * 2^e at most
    per element, so of that times sum |k| * scale per score, and of twice the largest of it times sum p |v| in the output."""
    from verl_omni_b200.ops.paged8 import attend_paged8

    torch.manual_seed(0)
    B, Hk, bs, n = 4, 2, 16, 500
    scale = 4 * 2.0 ** 14 / 8 ** 0.5  # scores with a spread of about 4
    q = torch.zeros(B, Hk * rep, S, hd, device="cuda")
    q[..., 3:11] = torch.randn(B, Hk * rep, S, 8, device="cuda") * 2.0 ** -14
    q[..., 0] = 1.0
    k = torch.randn(140, Hk, bs, hd, device="cuda")
    k[..., 0] = 0.0
    (kp, ks), (vp, vs) = _codes(k), _codes(torch.randn(140, Hk, bs, hd, device="cuda"))
    c = (q.bfloat16(), kp, vp, ks, vs, _table(B, -(-n // bs), 140), torch.full((B,), n, dtype=torch.int32, device="cuda"))
    want, tol = _attend64(*c, scale, few=True)
    keys = (_values(kp.view(torch.uint8)) * ks.double()[..., None, None])[..., 3:11].abs().sum(-1).amax()
    weighed, _ = _attend64(*c[:2], vp.view(torch.uint8).bitwise_and(0x7F).view(E4M3), *c[3:], scale, few=True)  # sum p |v|
    tol = tol + 2 * 2.0 ** -14 * 2.0 ** -8 * float(keys) * scale * weighed
    _agree(attend_paged8(*c, scale=scale), want, tol)
