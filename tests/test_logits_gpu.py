"""Logits processing on the GPU against a 64-bit definition, its gradient against the formula and differences."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _exact(x, hist, lens, pl, rows, rep, pres, freq, bias, allowed):
    """(y, dy/dx, size of the terms) in 64 bits, row by row."""
    R, V = x.shape
    y, d, size = (torch.zeros(R, V, dtype=torch.float64) for _ in range(3))
    x = x.detach().double().cpu()
    at = lambda p, r: float(p[r]) if isinstance(p, torch.Tensor) else p  # noqa: E731
    for r in range(R):
        h = [] if hist is None else hist[r if rows is None else int(rows[r])].tolist()
        n = len(h) if lens is None else max(0, min(int(lens[r]), len(h)))
        m = 0 if pl is None else int(pl[r])
        f = torch.ones(V, dtype=torch.float64)
        add = torch.zeros(V, dtype=torch.float64)
        for i, t in enumerate(h[:n]):
            if 0 <= t < V:
                rp = at(rep, r)
                f[t] = 1 / rp if x[r, t] > 0 else rp
                if i >= m:
                    if add[t] == 0:
                        add[t] += at(pres, r)
                    add[t] += at(freq, r)
        y[r] = x[r] * f - add
        size[r] = (x[r] * f).abs() + add.abs()
        if bias is not None:
            b = bias.double().cpu()
            b = b if b.dim() == 1 else b[r if b.shape[0] > 1 else 0]
            y[r] += b
            size[r] += b.abs()
        if allowed is not None:
            w = allowed[r if allowed.shape[0] > 1 else 0].cpu().long()
            bits = ((w[:, None] >> torch.arange(32)) & 1).flatten()[:V] == 1
            y[r] = torch.where(bits, y[r], -math.inf)
            f = torch.where(bits, f, 0.0)
        d[r] = f
    return y, d, size


def _close(got, want, size, dt):
    # at most five roundings to fp32 (2^-24 of the terms each; counted 8), and one to the output's type
    # (unit roundoff 2^-24 for 24 significand bits, 2^-8 for bf16's 8)
    unit = 2.0 ** -24 if dt == torch.float32 else 2.0 ** -8
    got = got.double().cpu()
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf])
    tol = 8 * 2.0 ** -24 * size + unit * want.abs() + 1e-40
    assert bool(((got - want).abs()[~inf] <= tol[~inf]).all())


CASES = [
    # rows, vocab, history
    (1, 151936, 513), (3, 512, 0), (5, 1, 7), (7, 4097, 60), (2, 33, 100), (4, 10000, 3001), (66, 130, 9),
]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("h64", [True, False])
@pytest.mark.parametrize("R,V,L", CASES)
def test_process_logits(R, V, L, h64, dt):
    from verl_omni_b200.ops.logits import pack_allowed, process_logits

    torch.manual_seed(R + V)
    x = (torch.randn(R, V + 3, device="cuda") * 4).to(dt)[:, 1:V + 1]  # odd row stride and offset
    x[0, V // 2] = -math.inf
    hist = (torch.rand(R, L, device="cuda") ** 3 * V).long()
    if L > 6:
        hist[:, 3] = -1
        hist[:, 5] = V + 2
        hist[0] = hist[0, 0]  # one token over and over
    hist = hist if h64 else hist.int()
    lens = torch.randint(0, L + 1, (R,), device="cuda", dtype=torch.int32)
    lens[0] = L
    pl = (lens * 0.4).int()
    rep = 1 + torch.rand(R, device="cuda")
    pres, freq = torch.rand(R, device="cuda"), torch.rand(R, device="cuda") - 0.3
    bias = torch.randn(V, device="cuda")
    mask = torch.rand(R, V, device="cuda") < 0.7
    mask[0] = R > 1  # a lone row whose mask allows nothing
    allowed = pack_allowed(mask)
    got = process_logits(x, hist, lens, pl, None, rep, pres, freq, bias, allowed)
    want, _, size = _exact(x, hist, lens, pl, None, rep, pres, freq, bias, allowed)
    assert got.dtype == dt
    _close(got, want, size, dt)
    # numbers for all rows, a bias per row, one mask for all rows, no prompt
    br = torch.randn(R, V, device="cuda")
    got = process_logits(x, hist, lens, repetition=1.2, presence=0.25, frequency=0.5, bias=br, allowed=allowed[-1:])
    want, _, size = _exact(x, hist, lens, None, None, 1.2, 0.25, 0.5, br, allowed[-1:])
    _close(got, want, size, dt)
    # nothing to do: the same numbers
    assert torch.equal(process_logits(x), x)


@pytest.mark.parametrize("R,V,L", [(3, 20000, 4096), (3, 20000, 4097), (2, 9001, 12000), (1, 2200000, 500), (700, 40, 4100), (300, 1000, 40)])
def test_long_history_wide_vocabulary_many_rows(R, V, L):
    """Histories and vocabularies past what one row's token table holds, rows past the CTAs, and their gradient."""
    from verl_omni_b200.ops.logits import pack_allowed, process_logits

    torch.manual_seed(R + L)
    x = (torch.randn(R, V, device="cuda") * 3).requires_grad_(True)
    hist = (torch.rand(R, L, device="cuda") ** 4 * V).long().clamp(max=V - 1)
    lens = torch.randint(L // 2, L + 1, (R,), device="cuda", dtype=torch.int32)
    allowed = pack_allowed(torch.rand(1, V, device="cuda") < 0.9)
    y = process_logits(x, hist, lens, lens // 3, repetition=1.5, presence=0.5, frequency=0.25, allowed=allowed)
    g = torch.randn(R, V, device="cuda")
    (dx,) = torch.autograd.grad(y, x, g)
    pick = sorted({0, R // 2, R - 1})
    want, d, size = _exact(x[pick], hist[pick], lens[pick], (lens // 3)[pick], None, 1.5, 0.5, 0.25, None, allowed)
    # the frequency penalty adds count * 0.25: exact in the oracle, one rounding of the sum here
    _close(y.detach()[pick], want, size, torch.float32)
    _close(dx[pick], g[pick].double().cpu() * d, (g[pick].double().cpu() * d).abs(), torch.float32)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [700, 5000])
def test_gradient(V, dt):
    """Training form: several positions of one sequence, each with its own history length."""
    from verl_omni_b200.ops.logits import pack_allowed, process_logits

    torch.manual_seed(0)
    N, L, R = 3, 50, 11
    rows = torch.tensor([0, 0, 0, 1, 1, 2, 2, 2, 2, 1, 0], dtype=torch.int32, device="cuda")
    hist = torch.randint(0, V // 4, (N, L), device="cuda")
    lens = torch.randint(0, L + 1, (R,), device="cuda", dtype=torch.int32)
    pl = torch.full((R,), 10, dtype=torch.int32, device="cuda")
    x = torch.randn(R, V, device="cuda")
    x = (x + 1.5 * torch.sign(x)).to(dt).requires_grad_(True)  # no logit within 1 of the kink at 0
    allowed = pack_allowed(torch.rand(R, V, device="cuda") < 0.8)
    kw = dict(history=hist, lens=lens, prompt_lens=pl, rows=rows, repetition=1.25, presence=0.3, frequency=0.2,
              bias=torch.randn(V, device="cuda"), allowed=allowed)
    y = process_logits(x, **kw)
    want, d, size = _exact(x, hist, lens, pl, rows, 1.25, 0.3, 0.2, kw["bias"], allowed)
    _close(y.detach(), want, size, dt)
    g = torch.randn(R, V, device="cuda").to(dt)
    (dx,) = torch.autograd.grad(y, x, g)
    _close(dx, g.double().cpu() * d, (g.double().cpu() * d).abs(), dt)
    if dt == torch.float32:
        # the map is linear away from the kink: a central difference of step 1/2 has the rounding of y alone
        with torch.no_grad():
            hi, lo = (process_logits(x + s, **kw).double().cpu() for s in (0.25, -0.25))
        ok = want.isfinite()
        diff = torch.where(ok, (hi - lo) * 2, 0.0)
        assert bool(((diff - d).abs()[ok] <= 4 * 10 * 2.0 ** -24 * (size + 1)[ok]).all())
    # a strided and a broadcast gradient
    gs = torch.randn(V, R, device="cuda").to(dt).t()
    y = process_logits(x, **kw)
    (dx,) = torch.autograd.grad(y, x, gs)
    _close(dx, gs.double().cpu() * d, (gs.double().cpu() * d).abs(), dt)
    y = process_logits(x, **{**kw, "allowed": None})
    (dx,) = torch.autograd.grad(y.float().sum(), x)
    _, d, _ = _exact(x, hist, lens, pl, rows, 1.25, 0.3, 0.2, kw["bias"], None)
    _close(dx, d, d.abs(), dt)


def test_masked_nan_and_many_rows():
    from verl_omni_b200.ops.logits import pack_allowed, process_logits

    x = torch.randn(2, 100, device="cuda")
    x[0, 3], x[0, 4], x[1, 5] = math.nan, math.inf, math.nan
    ok = torch.ones(2, 100, dtype=torch.bool, device="cuda")
    ok[0, 3:5] = False
    y = process_logits(x, allowed=pack_allowed(ok))
    assert y[0, 3:5].tolist() == [-math.inf, -math.inf] and int(y.isnan().sum()) == 1
    big = torch.randn(70000, 40, device="cuda").bfloat16()  # more rows than a launch's grid holds in one dimension
    hist = torch.randint(0, 40, (70000, 3), device="cuda")
    y = process_logits(big, hist, repetition=2.0)
    seen = torch.zeros(70000, 40, device="cuda").scatter(1, hist, 1.0) > 0
    want = torch.where(seen, torch.where(big > 0, big.float() / 2, big.float() * 2), big.float()).bfloat16()
    assert torch.equal(y, want)


def test_refusals():
    from verl_omni_b200.ops.logits import process_logits

    x = torch.randn(2, 64, device="cuda")
    h = torch.zeros(2, 4, dtype=torch.int64, device="cuda")
    i2 = torch.ones(2, dtype=torch.int32, device="cuda")
    for bad in (dict(x=x.half()), dict(x=x[0]), dict(history=h[:1]), dict(history=h.float()), dict(history=h, lens=i2.long()),
                dict(history=h, lens=i2[:1]), dict(history=h.cpu()), dict(repetition=torch.ones(3, device="cuda")),
                dict(presence=torch.ones(2, device="cuda").double()), dict(bias=torch.zeros(63, device="cuda")),
                dict(bias=torch.zeros(64, device="cuda").half()), dict(allowed=torch.zeros(2, 3, dtype=torch.int32, device="cuda")),
                dict(allowed=torch.zeros(2, 2, dtype=torch.int64, device="cuda")), dict(history=h, rows=i2.long()),
                dict(bias=torch.zeros(64, device="cuda", requires_grad=True))):
        with pytest.raises(ValueError):
            process_logits(**{"x": x, **bad})
    assert process_logits(x[:0]).shape == (0, 64)
