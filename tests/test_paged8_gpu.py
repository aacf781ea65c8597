"""8-bit paged KV cache on the GPU: quantising append, attention over it and page copies against 64-bit definitions."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def _values(code):
    """e4m3 codes (uint8) as 64-bit numbers, from the format: sign, 4 exponent bits with bias 7, 3 fraction bits."""
    c = torch.arange(256, dtype=torch.int64)
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2((e - 10).double()))
    v = torch.where((c & 127) == 127, math.nan, v) * torch.where(c >= 128, -1.0, 1.0)
    return v.to(code.device)[code.long()]


def _nearest(x):
    """64-bit x, |x| <= 448, to the nearest e4m3 number (ties to even)."""
    e = (torch.frexp(x)[1] - 1).clamp(min=-6)
    step = torch.exp2((e - 3).double())
    return torch.round(x / step) * step


def _pool(pages, Hk, bs, hd, spread=3, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    code = torch.randint(0, 127, (pages, Hk, bs, hd), generator=g, device="cuda", dtype=torch.uint8)
    # codes up to 2^0: typical magnitudes around 1 and many small ones
    code = torch.where(code > 64, code - 63, code)
    code = code + 128 * torch.randint(0, 2, code.shape, generator=g, device="cuda", dtype=torch.uint8)
    scale = torch.exp2(torch.randint(-spread, 2, (pages, Hk), generator=g, device="cuda").float())
    return code.view(E4M3), scale


def _attend64(q, kp, vp, ks, vs, table, lens, q_lens, scale):
    """(output, tolerance) in 64 bits, row by row.

    The tolerance is the kernels' rounding: the bf16 output (unit roundoff 2^-8, of |o|), probabilities kept to 8 bits
    (2^-8 each, so 2^-8 of sum p|v| >= |o|) with a floor of 2^-18 of the largest one; the factor 2 on the last two
    covers the sums and the fp32 products."""
    B, Hq, S, hd = q.shape
    Hk, bs = kp.shape[1:3]
    rep = Hq // Hk
    out = torch.zeros(B, S, Hq, hd, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    K = _values(kp.view(torch.uint8)) * ks.double()[..., None, None]
    V = _values(vp.view(torch.uint8)) * vs.double()[..., None, None]
    for b in range(B):
        n = max(0, min(int(lens[b]), table.shape[1] * bs))
        m = S if q_lens is None else min(int(q_lens[b]), S)
        ids = table[b, :-(-n // bs)].long()
        bad = (ids < 0) | (ids >= kp.shape[0])
        ids = torch.where(bad, 0, ids)
        k, v = (torch.where(bad[:, None, None, None], 0.0, x[ids]).transpose(0, 1).reshape(Hk, -1, hd)[:, :n] for x in (K, V))
        for i in range(m):
            lim = n - m + i + 1
            if lim <= 0:
                continue
            kk, vv = k[:, :lim].repeat_interleave(rep, 0), v[:, :lim].repeat_interleave(rep, 0)
            z = torch.einsum("hd,htd->ht", q[b, :, i].double(), kk) * scale
            p = torch.softmax(z, -1)
            out[b, i] = torch.einsum("ht,htd->hd", p, vv)
            a = torch.einsum("ht,htd->hd", p, vv.abs())
            tol[b, i] = 2 * (2.0 ** -9 * out[b, i].abs() + 2.0 ** -8 * a + 2.0 ** -18 * p.amax(-1, keepdim=True) * vv.abs().sum(1))
    return out, tol


def _agree(got, want, tol):
    assert torch.equal(got.isnan(), want.isnan())
    err = (got.double() - want).abs()
    bad = (err > tol + 1e-30) & ~want.isnan()
    assert not bool(bad.any()), f"{int(bad.sum())} values off, worst {float((err / (tol + 1e-30))[~want.isnan()].max()):.2f} x tolerance"


def _table(B, width, pages, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[:B * width].view(B, width).to(torch.int32).cuda()


SHAPES = [
    # kv_heads, group, head_dim, block
    (4, 8, 128, 16), (4, 8, 128, 128), (2, 16, 128, 64), (8, 1, 128, 32), (3, 5, 128, 16), (1, 32, 128, 64), (2, 3, 128, 256),
    (4, 8, 64, 16), (2, 2, 64, 128), (1, 16, 64, 32), (2, 4, 128, 48), (2, 2, 16, 4), (1, 7, 96, 16), (1, 2, 256, 8), (2, 4, 128, 8),
]


@pytest.mark.parametrize("Hk,rep,hd,bs", SHAPES)
def test_attend_one_token(Hk, rep, hd, bs):
    from verl_omni_b200.ops.paged8 import attend_paged8

    lens = torch.tensor([1, 0, 700, 129, 127, 128, 33, 1], dtype=torch.int32, device="cuda")
    B, width = len(lens), -(-700 // bs)
    kp, ks = _pool(B * width + 2, Hk, bs, hd)
    vp, vs = _pool(B * width + 2, Hk, bs, hd, seed=1)
    table = _table(B, width, kp.shape[0])
    torch.manual_seed(0)
    q = torch.randn(B, Hk * rep, 1, hd, device="cuda").bfloat16()
    got = attend_paged8(q, kp, vp, ks, vs, table, lens)
    want, tol = _attend64(q, kp, vp, ks, vs, table, lens, None, hd ** -0.5)
    _agree(got, want, tol)
    assert not got[1].any()


@pytest.mark.parametrize("S", [2, 5, 17, 64, 150])
@pytest.mark.parametrize("Hk,rep,hd,bs", [(4, 8, 128, 16), (2, 5, 128, 128), (1, 16, 64, 64), (2, 2, 16, 4), (2, 1, 128, 64)])
def test_attend_several_tokens(Hk, rep, hd, bs, S):
    """Causal among the new tokens; ragged token counts; sequences shorter than their query count (empty rows)."""
    from verl_omni_b200.ops.paged8 import attend_paged8

    lens = torch.tensor([S, S + 300, 0, 1, 129, S + 1], dtype=torch.int32, device="cuda")
    q_lens = torch.tensor([S, S, S, S, max(1, S // 2), 0], dtype=torch.int32, device="cuda")
    B, width = len(lens), -(-(S + 300) // bs)
    kp, ks = _pool(B * width + 2, Hk, bs, hd)
    vp, vs = _pool(B * width + 2, Hk, bs, hd, seed=1)
    table = _table(B, width, kp.shape[0])
    torch.manual_seed(0)
    q = torch.randn(B, Hk * rep, S, hd, device="cuda").bfloat16()
    got = attend_paged8(q, kp, vp, ks, vs, table, lens, q_lens=q_lens)
    want, tol = _attend64(q, kp, vp, ks, vs, table, lens, q_lens, hd ** -0.5)
    _agree(got, want, tol)
    # no counts: every sequence has all S tokens
    whole = torch.full_like(q_lens, S)
    assert torch.equal(attend_paged8(q, kp, vp, ks, vs, table, lens), attend_paged8(q, kp, vp, ks, vs, table, lens, q_lens=whole))
    # a smaller batch is cut elsewhere: the same values within the tolerance
    _agree(attend_paged8(q[:2], kp, vp, ks, vs, table[:2].contiguous(), lens[:2].contiguous()), want[:2], tol[:2])


@pytest.mark.parametrize("hd", [64, 128])
def test_attend_long_and_many(hd):
    """Long caches split over many blocks, next to short ones, and more sequences than fit one wave."""
    from verl_omni_b200.ops.paged8 import attend_paged8

    Hk, rep, bs = 2, 4, 64
    lens = torch.tensor([20000, 1, 64, 5000] + [7 * i % 300 for i in range(200)], dtype=torch.int32, device="cuda")
    B = len(lens)
    width = -(-20000 // bs)
    pages = 1200
    kp, ks = _pool(pages, Hk, bs, hd)
    vp, vs = _pool(pages, Hk, bs, hd, seed=1)
    g = torch.Generator().manual_seed(3)
    table = torch.randint(0, pages, (B, width), generator=g, dtype=torch.int32).cuda()
    q = torch.randn(B, Hk * rep, 1, hd, device="cuda").bfloat16()
    got = attend_paged8(q, kp, vp, ks, vs, table, lens)
    want, tol = _attend64(q, kp, vp, ks, vs, table, lens, None, hd ** -0.5)
    _agree(got, want, tol)


@pytest.mark.parametrize("S,bs,hd", [(1, 16, 128), (1, 64, 64), (4, 128, 128), (4, 24, 128), (150, 64, 128), (150, 64, 64)])
def test_attend_garbage_past_the_rows(S, bs, hd):
    """NaN codes and NaN scales past a sequence's rows, out-of-pool pages and lengths past the table do not leak."""
    from verl_omni_b200.ops.paged8 import attend_paged8

    Hk, rep = 2, 4
    top = 5 * bs + S
    lens = torch.tensor([S + bs // 2, 3 * bs, top, 10 ** 6, -5], dtype=torch.int32, device="cuda")
    B, width = len(lens), -(-top // bs)
    kp, ks = _pool(B * width + 2, Hk, bs, hd)
    vp, vs = _pool(B * width + 2, Hk, bs, hd, seed=1)
    table = _table(B, width, kp.shape[0])
    table[2, 1] = 10 ** 6
    table[2, 2] = -1
    for b in range(2):
        for page in range(width):
            r = max(0, min(bs, int(lens[b]) - page * bs))
            i = int(table[b, page])
            kp.view(torch.uint8)[i, :, r:] = 0x7F
            vp.view(torch.uint8)[i, :, r:] = 0xFF
            if r == 0:
                ks[i] = math.nan
                vs[i] = math.nan
                table[b, page] = 2 ** 30 if page % 2 else i
    q = torch.randn(B, Hk * rep, S, hd, device="cuda").bfloat16()
    got = attend_paged8(q, kp, vp, ks, vs, table, lens)
    want, tol = _attend64(q, kp, vp, ks, vs, table, lens, None, hd ** -0.5)
    assert bool(got.isfinite().all()) and not got[4].any()
    _agree(got, want, tol)


@pytest.mark.parametrize("S,hd", [(3, 128), (3, 64), (3, 32), (140, 128), (140, 64)])
def test_attend_nan_row_reaches_only_rows_that_see_it(S, hd):
    from verl_omni_b200.ops.paged8 import attend_paged8

    Hk, rep, bs = 2, 4, 32
    n = 200
    kp, ks = _pool(20, Hk, bs, hd)
    vp, vs = _pool(20, Hk, bs, hd, seed=1)
    table = _table(2, 7, 20)
    lens = torch.tensor([n, n], dtype=torch.int32, device="cuda")
    t = n - 2  # the second to last new token
    vp.view(torch.uint8)[int(table[0, t // bs]), 1, t % bs, 5] = 0x7F  # one value of sequence 0, KV head 1
    kp.view(torch.uint8)[int(table[1, t // bs]), 0, t % bs, 3] = 0x7F  # one key of sequence 1, KV head 0
    q = torch.randn(2, Hk * rep, S, hd, device="cuda").bfloat16()
    got = attend_paged8(q, kp, vp, ks, vs, table, lens)
    want, tol = _attend64(q, kp, vp, ks, vs, table, lens, None, hd ** -0.5)
    assert bool(got[0, :-2].isfinite().all()) and bool(got[1, :-2].isfinite().all())
    assert bool(got[0, -2:, rep:, 5].isnan().all()) and bool(got[1, -2:, :rep].isnan().all())
    _agree(got, want, tol)


@pytest.mark.parametrize("magnitude", [1e-30, 1e-3, 1e3, 3e4])
def test_attend_scale_extremes(magnitude):
    """Queries and pages of very small and large magnitude (the softmax scale undoes them)."""
    from verl_omni_b200.ops.paged8 import attend_paged8

    Hk, rep, bs, hd = 2, 8, 16, 128
    kp, ks = _pool(40, Hk, bs, hd)
    vp, vs = _pool(40, Hk, bs, hd, seed=1)
    vs = vs * 2.0 ** 60
    table = _table(3, 12, 40)
    lens = torch.tensor([190, 64, 5], dtype=torch.int32, device="cuda")
    q = (torch.randn(3, Hk * rep, 1, hd, device="cuda") * magnitude).bfloat16()
    got = attend_paged8(q, kp, vp, ks, vs, table, lens, scale=hd ** -0.5 / magnitude)
    want, tol = _attend64(q, kp, vp, ks, vs, table, lens, None, hd ** -0.5 / magnitude)
    _agree(got, want, tol)


def test_attend_strides_streams_and_determinism():
    from verl_omni_b200.ops.paged8 import attend_paged8

    B, Hk, rep, bs, hd, S = 5, 4, 8, 16, 128, 3
    kp, ks = _pool(200, Hk, bs, hd)
    vp, vs = _pool(200, Hk, bs, hd, seed=1)
    table = _table(B, 40, 200)
    lens = torch.tensor([640, 3, 77, 500, 16], dtype=torch.int32, device="cuda")
    wide = torch.randn(B, S, 3 * Hk * rep * hd + 1, device="cuda").bfloat16()
    q = wide[..., Hk * rep * hd:2 * Hk * rep * hd].view(B, S, Hk * rep, hd).transpose(1, 2)  # odd token stride
    want = attend_paged8(q.contiguous(), kp, vp, ks, vs, table, lens)
    assert torch.equal(attend_paged8(q, kp, vp, ks, vs, table, lens), want)
    even = torch.randn(B, S, 2 * Hk * rep * hd, device="cuda").bfloat16()
    qe = even[..., Hk * rep * hd:].view(B, S, Hk * rep, hd).transpose(1, 2)
    assert torch.equal(attend_paged8(qe, kp, vp, ks, vs, table, lens), attend_paged8(qe.contiguous(), kp, vp, ks, vs, table, lens))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [attend_paged8(q, kp, vp, ks, vs, table, lens) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want) for g in got)


# ------------------------------------------------------------------------------------------------ append
def _append64(x, code, scale, table, start, counts):
    """The definition in 64 bits -> (values of the codes, scales); rows are cached page by page in order."""
    vals, sc = _values(code.view(torch.uint8)), scale.double().clone()
    bs = code.shape[2]
    for b in range(x.shape[0]):
        p0, n, done = int(start[b]), int(counts[b]), 0
        while done < n:
            page, r0 = divmod(p0 + done, bs)
            m = min(bs - r0, n - done)
            if page >= table.shape[1]:
                break
            i = int(table[b, page])
            if 0 <= i < code.shape[0]:
                rows = x[b, :, done:done + m].double()
                fin = torch.where(rows.isfinite(), rows.abs(), 0.0).amax((1, 2))
                e = torch.full_like(fin, -100.0)
                while bool((fin > 448 * torch.exp2(e)).any()):
                    e = torch.where(fin > 448 * torch.exp2(e), e + 1, e)
                now = torch.exp2(e)
                if r0:
                    now = torch.maximum(now, sc[i])
                    vals[i, :, :r0] = _nearest(vals[i, :, :r0] * (sc[i] / now)[:, None, None])
                vals[i, :, r0:r0 + m] = _nearest((rows / now[:, None, None]).clamp(-448, 448))
                sc[i] = now
            done += m
    return vals, sc


@pytest.mark.parametrize("S", [1, 2, 7, 100, 333])
@pytest.mark.parametrize("Hk,hd,bs", [(4, 128, 16), (2, 64, 128), (1, 16, 4), (3, 96, 24), (2, 128, 64), (1, 256, 256)])
def test_append(Hk, hd, bs, S):
    from verl_omni_b200.ops.paged8 import append_paged8

    torch.manual_seed(0)
    start = torch.tensor([0, 1, bs - 1, 2 * bs, bs + bs // 2, 5], dtype=torch.int32, device="cuda")
    counts = torch.tensor([S, S, S, 0, max(1, S // 2), min(1, S)], dtype=torch.int32, device="cuda")
    B, width = len(start), -(-(2 * bs + S) // bs) + 1
    kp, ks = _pool(B * width + 2, Hk, bs, hd)
    vp, vs = _pool(B * width + 2, Hk, bs, hd, seed=1)
    table = _table(B, width, kp.shape[0])
    k = (torch.randn(B, Hk, S, hd, device="cuda") * torch.exp2(torch.randint(-6, 12, (B, Hk, 1, 1), device="cuda").float())).bfloat16()
    v = torch.randn(B, S, 3 * Hk * hd, device="cuda").bfloat16()[..., 2 * Hk * hd:].view(B, S, Hk, hd).transpose(1, 2)
    if S > 1:
        k[0, 0, :] = 0  # a page of zeros
        v[1] *= 1e-36
    want = [_append64(x, c, s, table, start, counts) for x, c, s in ((k, kp, ks), (v, vp, vs))]
    append_paged8(k, v, kp, vp, ks, vs, table, start, counts=counts)
    for (code, scale), (vals, sc) in zip(((kp, ks), (vp, vs)), want):
        assert torch.equal(scale.double(), sc)
        assert torch.equal(_values(code.view(torch.uint8)), vals)


def test_append_amax_edges_and_non_finite():
    """448 * 2^e exactly and just above; infinities saturate, NaN stays NaN, neither sets the scale."""
    from verl_omni_b200.ops.paged8 import append_paged8

    bs, hd = 16, 64
    x = torch.zeros(6, 1, 1, hd, device="cuda")
    x[0, ..., 3] = 448.0
    x[1, ..., 3] = 450.0
    x[2, ..., 3] = -0.875 * 2.0 ** -40
    x[3, ..., 3:6] = torch.tensor([math.inf, -math.inf, 7.0], device="cuda")
    x[4, ..., 3:5] = torch.tensor([math.nan, 1.0], device="cuda")
    x[5, ..., 3] = 3.3e38
    x = x.bfloat16()
    kp, ks = _pool(8, 1, bs, hd)
    vp, vs = _pool(8, 1, bs, hd, seed=1)
    table = torch.arange(6, dtype=torch.int32, device="cuda")[:, None].contiguous()
    start = torch.zeros(6, dtype=torch.int32, device="cuda")
    append_paged8(x, x, kp, vp, ks, vs, table, start)
    assert ks[:6, 0].tolist() == [1.0, 2.0, 2.0 ** -49, 2.0 ** -6, 2.0 ** -8, 2.0 ** 120]
    got = kp.float()[:6, 0, 0] * ks[:6]
    assert got[3, 3:6].tolist() == [7.0, -7.0, 7.0]
    assert bool(got[4, 3].isnan()) and float(got[4, 4]) == 1.0 and int(got.isnan().sum()) == 1


def test_append_drops_what_the_table_does_not_hold():
    from verl_omni_b200.ops.paged8 import append_paged8

    kp, ks = _pool(6, 2, 8, 64)
    vp, vs = _pool(6, 2, 8, 64, seed=1)
    before = [t.clone() for t in (kp.view(torch.uint8), vp.view(torch.uint8), ks, vs)]
    x = torch.randn(4, 2, 20, 64, device="cuda").bfloat16()
    table = torch.tensor([[99, -1], [2 ** 31 - 1, 7], [-7, 6], [0, 1]], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 3, 100, -4], dtype=torch.int32, device="cuda")
    append_paged8(x, x, kp, vp, ks, vs, table, start)
    for t, b in zip((kp.view(torch.uint8), vp.view(torch.uint8), ks, vs), before):
        assert torch.equal(t, b)


def test_append_then_attend_equals_whole_append():
    """A prompt written in unlike chunks holds the rows of the last scale of each page: attention over it matches the
    64-bit attention over its own codes, and the values stay within the format's error of the inputs."""
    from verl_omni_b200.ops.paged8 import append_paged8, attend_paged8

    torch.manual_seed(0)
    B, Hk, rep, bs, hd = 2, 2, 8, 64, 128
    kp, ks = _pool(12, Hk, bs, hd)
    vp, vs = _pool(12, Hk, bs, hd, seed=1)
    table = _table(B, 5, 12)
    k, v = (torch.randn(B, Hk, 300, hd, device="cuda").bfloat16() for _ in range(2))
    start = torch.zeros(B, dtype=torch.int32, device="cuda")
    at = 0
    for n in (1, 2, 61, 1, 130, 105):
        append_paged8(k[:, :, at:at + n], v[:, :, at:at + n], kp, vp, ks, vs, table, start, offset=at)
        at += n
    ids = table.long()
    got = (kp.float()[ids] * ks[ids][..., None, None]).transpose(1, 2).reshape(B, Hk, -1, hd)[:, :, :300]
    # relative error of e4m3: 2^-4; subnormal step: 2^-10 of a unit of scale (ks <= 2^-6 here: |k| < 7)
    assert bool(((got - k.float()).abs() <= 2.0 ** -4 * k.float().abs() + 2.0 ** -10 * ks.max()).all())
    lens = torch.full((B,), 300, dtype=torch.int32, device="cuda")
    q = torch.randn(B, Hk * rep, 1, hd, device="cuda").bfloat16()
    _agree(attend_paged8(q, kp, vp, ks, vs, table, lens), *_attend64(q, kp, vp, ks, vs, table, lens, None, hd ** -0.5))


# ------------------------------------------------------------------------------------------------ pages
@pytest.mark.parametrize("layers,Hk,bs,hd", [(1, 1, 4, 16), (3, 4, 16, 128), (2, 3, 128, 128), (5, 2, 8, 96)])
@pytest.mark.parametrize("n", [0, 1, 9, 40])
def test_copy_pages(layers, Hk, bs, hd, n):
    from verl_omni_b200.ops.paged8 import copy_pages

    g = torch.Generator(device="cuda").manual_seed(0)
    pages = 2 * n + 3
    pools = [torch.randint(0, 256, (layers, pages, Hk, bs, hd), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
    pools += [torch.randn(layers, pages, Hk, device="cuda") for _ in range(2)]
    pools += [torch.randint(0, 256, (layers, pages, 5), generator=g, device="cuda", dtype=torch.uint8)]  # odd page size
    at = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()
    src, dst = at[:n], at[n:2 * n]
    want = [p.clone() for p in pools]
    for p in want:
        for i, j in zip(src, dst):
            p[:, j] = p[:, i]
    copies = [p.clone() for p in pools]
    copy_pages(pools, src, dst)
    t = [torch.tensor(x + [pages, -1], dtype=torch.int32, device="cuda") for x in (src, dst)]  # outside: skipped
    copy_pages(copies, *t)
    for p, c, w in zip(pools, copies, want):
        assert torch.equal(p, w) and torch.equal(c, w)


def test_pages_past_32_bit_offsets():
    """A pool of more than 2^31 bytes: append, attention and copies at its far end."""
    from verl_omni_b200.ops.paged8 import append_paged8, attend_paged8, copy_pages

    Hk, bs, hd = 4, 128, 128
    pages = 2 ** 31 // (Hk * bs * hd) + 40
    kp, vp = (torch.zeros(pages, Hk, bs, hd, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    ks, vs = (torch.ones(pages, Hk, device="cuda") for _ in range(2))
    far = torch.tensor([[pages - 1, pages - 3], [5, pages - 2]], dtype=torch.int32, device="cuda")
    x = torch.randn(2, Hk, 200, hd, device="cuda").bfloat16()
    append_paged8(x, x, kp, vp, ks, vs, far, torch.zeros(2, dtype=torch.int32, device="cuda"))
    near_k, near_s = kp[far.long().view(-1)].view(torch.uint8).clone().view(E4M3), ks[far.long().view(-1)].clone()
    lens = torch.tensor([200, 200], dtype=torch.int32, device="cuda")
    near = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    for S in (1, 70):
        q = torch.randn(2, Hk * 8, S, hd, device="cuda").bfloat16()
        got = attend_paged8(q, kp, vp, ks, vs, far, lens)
        assert torch.equal(got, attend_paged8(q, near_k, near_k, near_s, near_s, near, lens)) and bool(got.any())
    copy_pages([p.unsqueeze(0) for p in (kp, vp, ks, vs)], [pages - 1], [pages - 10])
    assert torch.equal(kp.view(torch.uint8)[pages - 10], kp.view(torch.uint8)[pages - 1])


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    from verl_omni_b200.ops.paged8 import append_paged8, attend_paged8, copy_pages

    kp, ks = _pool(8, 2, 16, 64)
    vp, vs = _pool(8, 2, 16, 64, seed=1)
    table = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    lens = torch.ones(3, dtype=torch.int32, device="cuda")
    q = torch.randn(3, 4, 1, 64, device="cuda").bfloat16()
    ok = (q, kp, vp, ks, vs, table, lens)
    attend_paged8(*ok)
    for i, bad in [(0, q.half()), (0, q[..., :32]), (0, q[:, :3]), (0, q[:2]), (0, q[0]), (1, kp.view(torch.uint8)), (1, kp[:, :1]),
                   (2, vp[:4]), (1, kp.transpose(1, 2)), (3, ks.half()), (4, vs[:, :1]), (5, table.long()), (5, table[:2]),
                   (6, lens.long()), (6, lens[:2]), (6, lens.cpu()), (5, table.cpu())]:
        with pytest.raises(ValueError):
            attend_paged8(*(bad if j == i else t for j, t in enumerate(ok)))
    with pytest.raises(ValueError):
        attend_paged8(*ok, q_lens=lens[:1])
    with pytest.raises(ValueError, match="no backward"):
        attend_paged8(q.clone().requires_grad_(True), *ok[1:])
    k = torch.randn(3, 2, 2, 64, device="cuda").bfloat16()
    okk = (k, k, kp, vp, ks, vs, table, lens)
    for i, bad in [(0, k.float()), (1, k[:, :1]), (0, k[:2]), (2, kp[..., :32]), (7, lens.long()), (6, table[0])]:
        with pytest.raises(ValueError):
            append_paged8(*(bad if j == i else t for j, t in enumerate(okk)))
    with pytest.raises(ValueError):
        append_paged8(*okk, counts=lens.float())
    pools = [kp.unsqueeze(0), ks.unsqueeze(0)]
    for src, dst in [([0], [8]), ([-1], [0]), ([0, 1], [2]), ([0, 1], [2, 2]), ([0, 1], [1, 2])]:
        with pytest.raises(ValueError):
            copy_pages(pools, src, dst)
    i32 = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bad in ([kp.unsqueeze(0), ks[:4].unsqueeze(0)], [kp.unsqueeze(0).transpose(1, 2)], []):
        with pytest.raises((ValueError, IndexError)):
            copy_pages(bad, i32, i32 + 1)
    with pytest.raises(ValueError):
        copy_pages(pools, i32.long(), i32.long() + 1)


def test_empty_calls():
    from verl_omni_b200.ops.paged8 import append_paged8, attend_paged8

    kp, ks = _pool(8, 2, 16, 64)
    vp, vs = _pool(8, 2, 16, 64, seed=1)
    z = torch.zeros(0, dtype=torch.int32, device="cuda")
    t = torch.zeros(0, 2, dtype=torch.int32, device="cuda")
    assert attend_paged8(torch.zeros(0, 4, 1, 64, device="cuda").bfloat16(), kp, vp, ks, vs, t, z).shape == (0, 1, 4, 64)
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    assert attend_paged8(torch.zeros(1, 4, 0, 64, device="cuda").bfloat16(), kp, vp, ks, vs, t.new_zeros(1, 2), one).shape == (1, 0, 4, 64)
    # a table of no pages: nothing is cached
    out = attend_paged8(torch.randn(1, 4, 1, 64, device="cuda").bfloat16(), kp, vp, ks, vs, t.new_zeros(1, 0), one)
    assert not out.any()
    append_paged8(torch.zeros(0, 2, 3, 64, device="cuda").bfloat16(), torch.zeros(0, 2, 3, 64, device="cuda").bfloat16(), kp, vp, ks, vs, t, z)


# ------------------------------------------------------------------------------------------------ rollout
def test_rollout_graph_groups_and_chunks(monkeypatch):
    """The thinker's rollout on the 8-bit cache: the decode step captured as a CUDA graph equals eager steps, shared
    prompt pages equal unshared ones, and penalties and a grammar mask run in the same loop."""
    from verl_omni_b200.models.moe_llm import MoEConfig, MoELLM
    from verl_omni_b200.ops._ext import ext
    from verl_omni_b200.ops.logits import pack_allowed
    from verl_omni_b200.ops.paged8 import PagedKVCache8
    from verl_omni_b200.utils.dataproto import DataProto
    from verl_omni_b200.workers.rollout.llm_rollout import LLMRolloutEngine

    torch.manual_seed(0)
    cfg = MoEConfig(vocab=2048, hidden=512, layers=2, q_heads=16, kv_heads=2, head_dim=128, experts=8, top_k=2,
                    expert_ffn=256, audio_layers=1, audio_dim=128, audio_mel=16, vision_layers=1, vision_dim=128,
                    vision_patch_dim=48, audio_token=2046, image_token=2047)
    m = MoELLM(cfg).to("cuda", torch.bfloat16).eval()
    ids = torch.randint(0, 2000, (2, 37)).repeat_interleave(3, 0)
    batch = DataProto({"input_ids": ids}, {})
    ban = torch.ones(1, 2048, dtype=torch.bool, device="cuda")
    ban[0, 100:] = False
    mask = pack_allowed(ban)
    kw = dict(max_new_tokens=40, temperature=0.0, device=torch.device("cuda"), kv_cache_dtype="fp8_e4m3", kv_block_size=16,
              repetition_penalty=1.2, presence_penalty=0.1, frequency_penalty=0.05, allowed_tokens=lambda said: mask)
    out = {}
    for graph in ("0", "1"):
        for group in (1, 3):
            monkeypatch.setenv("VO_DECODE_GRAPH", graph)
            out[graph, group] = LLMRolloutEngine(m, **kw).generate(batch, seed=0, group=group)
    torch.cuda.synchronize()
    assert ext().paged8_error(False) == 0
    ref = out["0", 1].batch
    assert bool((ref["responses"] < 100).all())
    for o in out.values():
        assert torch.equal(o.batch["responses"], ref["responses"])
        torch.testing.assert_close(o.batch["rollout_log_probs"], ref["rollout_log_probs"], rtol=1e-4, atol=1e-4)
    assert torch.equal(ref["responses"][0], ref["responses"][2]) and ref["responses"].shape == (6, 40)
    # a prompt continued in chunks against the cache stays near the whole prompt's hidden states (8-bit keys and values)
    c = PagedKVCache8(cfg.layers, 12, cfg.kv_heads, 16, cfg.head_dim, "cuda")
    views = c.batch([c.add_sequence(), c.add_sequence()]).views()
    p = torch.randint(0, 2000, (2, 90), device="cuda")
    with torch.no_grad():
        whole = m(p, return_hidden=True).float()
        part = torch.cat([m(p[:, a:b], caches=views, pos0=a, return_hidden=True).float() for a, b in ((0, 30), (30, 89), (89, 90))], 1)
    assert float((part - whole).norm() / whole.norm()) < 0.1
