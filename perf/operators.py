"""Measured cases of the rollout's 8-bit paged KV cache and of its logits processing.

Four operators that one decode step of the language-model rollout runs one after the other:

* ``append``: new key / value rows are rounded to e4m3 with one power-of-two scale per (page, KV head) and written
  into the pages of their sequences; a page that was partly filled is brought to the larger scale;
* ``attend``: one or more new query tokens per sequence attend causally to the rows cached in such pages;
* ``pages``: whole pages of every layer are copied inside the pool (the partly filled last page of a forked prompt,
  the live pages that move down when a pool is compacted);
* ``logits``: repetition, presence and frequency penalties, a bias and a grammar bitmask on next-token logits, and
  their gradient.

``own`` false: the plain forms (elementary torch operations in 32 bits).  ``own`` true: the package's operators.
"""

import math

import numpy as np
import torch

own = False

FP8 = torch.float8_e4m3fn
E_MIN = -100  # smallest exponent of a page scale


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    thinker = {"kv_heads": 4, "group": 8, "head_dim": 128}
    return [
        # one sequence's next token against a short cache: latency of a single interactive request
        {"name": "attend-one", "op": "attend", "batch": 1, "queries": 1, "ctx": 1000, "ragged": False, "block": 16, **thinker},
        # the rollout's decode step: 64 sequences with 4096 cached positions each
        {"name": "attend-rollout", "op": "attend", "batch": 64, "queries": 1, "ctx": 4096, "ragged": False, "block": 128, **thinker},
        # continuous batching: lengths from nothing to long in one call, small pages
        {"name": "attend-ragged", "op": "attend", "batch": 96, "queries": 1, "ctx": 8191, "ragged": True, "block": 16, **thinker},
        # a prompt continued in chunks: 512 new tokens of each sequence against its cached prefix and themselves
        {"name": "attend-chunk", "op": "attend", "batch": 4, "queries": 512, "ctx": 8000, "ragged": False, "block": 128, **thinker},
        # the decode step's write: one token per sequence, into partly filled pages
        {"name": "append-step", "op": "append", "batch": 64, "tokens": 1, "start": 1000, "ragged": True, "block": 16, **thinker},
        # chunks of unlike length that start inside a page
        {"name": "append-ragged", "op": "append", "batch": 24, "tokens": 333, "start": 777, "ragged": True, "block": 64, **thinker},
        # the prompts of a rollout batch
        {"name": "append-prefill", "op": "append", "batch": 64, "tokens": 1024, "start": 0, "ragged": False, "block": 128, **thinker},
        # the last page of one prompt for each of its 8 samples, all 48 layers
        {"name": "pages-fork", "op": "pages", "layers": 48, "blocks": 256, "pairs": 7, "block": 16, "kv_heads": 4, "head_dim": 128},
        # a pool whose live pages move to its low end
        {"name": "pages-compact", "op": "pages", "layers": 8, "blocks": 1000, "pairs": 400, "block": 128, "kv_heads": 4, "head_dim": 128},
        # one request's next-token logits
        {"name": "logits-one", "op": "logits", "rows": 1, "vocab": 151936, "history": 512, "dtype": "float32", "mask": True, "bias": True, "grad": False},
        # the rollout batch's logits, prompt and response so far as the history
        {"name": "logits-rollout", "op": "logits", "rows": 64, "vocab": 151936, "history": 1536, "dtype": "float32", "mask": True, "bias": False, "grad": False},
        # a training micro-batch whose log-probs are taken under the processed distribution
        {"name": "logits-train", "op": "logits", "rows": 512, "vocab": 151936, "history": 1536, "dtype": "bfloat16", "mask": False, "bias": True, "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "pages", "logits"])
    if op == "attend":
        kv, group = rng.choice([(4, 8), (2, 16), (8, 1), (2, 4), (4, 2), (1, 8), (3, 5)])
        queries = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 500)])
        ctx = max(queries, _log(rng, 1, 8000)) | 1
        batch = _log(rng, 1, 128)
        batch = max(1, min(batch, 64 * 4096 * 4 // (ctx * kv), 4 * 512 * 8000 * 32 // (queries * ctx * kv * group)))
        return {"op": op, "batch": batch, "queries": queries, "ctx": ctx, "ragged": rng.random() < 0.6,
                "block": rng.choice([16, 32, 64, 128]), "kv_heads": kv, "group": group, "head_dim": rng.choice([128, 128, 64])}
    if op == "append":
        tokens = rng.choice([1, 1, _log(rng, 2, 1000)])
        return {"op": op, "batch": max(1, min(_log(rng, 1, 128), 64000 // tokens)), "tokens": tokens, "start": rng.choice([0, _log(rng, 1, 2000)]),
                "ragged": rng.random() < 0.6, "block": rng.choice([16, 32, 64, 128]), "kv_heads": rng.choice([1, 2, 4, 8]),
                "group": 1, "head_dim": rng.choice([64, 128])}
    if op == "pages":
        block, layers = rng.choice([16, 32, 64, 128]), rng.choice([1, 8, 48])
        pairs = max(1, min(_log(rng, 1, 400), 400 * 128 * 8 // (block * layers)))
        return {"op": op, "layers": layers, "blocks": 2 * pairs + rng.randint(1, 40), "pairs": pairs, "block": block,
                "kv_heads": rng.choice([1, 2, 4]), "head_dim": rng.choice([64, 128])}
    grad = rng.random() < 0.4
    vocab = rng.choice([151936, 151936, 512, _log(rng, 400, 150000)])
    return {"op": op, "rows": max(1, min(_log(rng, 1, 500), 512 * 151936 // (2 * vocab))), "vocab": vocab, "history": _log(rng, 1, 4000) | 1,
            "dtype": rng.choice(["float32", "bfloat16"]), "mask": rng.random() < 0.6, "bias": rng.random() < 0.5, "grad": grad}


# ---------------------------------------------------------------------------------------------------- shapes
def _spread(n, top):
    """n whole numbers from 0 to top, unlike and in no order, the same for every seed; the first is top, then 1 and 0."""
    v = [int(top * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]
    return ([top, min(1, top), 0] + v[3:])[:n]


def _lengths(case):
    """Cached rows (the new ones among them) and new query tokens of each sequence."""
    n, top, s = case["batch"], case["ctx"], case["queries"]
    lens = _spread(n, top) if case["ragged"] else [top] * n
    return lens, [min(s, length) for length in lens]


def _starts(case):
    """First position and number of the new rows of each sequence."""
    n, s, t = case["batch"], case["start"], case["tokens"]
    if not case["ragged"]:
        return [s] * n, [t] * n
    return [s + 5 * i for i in range(n)], ([t] * n if t == 1 else _spread(n, t))


def _pages_of(n, block):
    return -(-n // block)


def work(case):
    if case["op"] == "attend":
        lens, q = _lengths(case)
        hk, hd = case["kv_heads"], case["head_dim"]
        hq, pages = hk * case["group"], sum(_pages_of(n, case["block"]) for n in lens)
        seen = sum(k * (2 * n - k + 1) // 2 for n, k in zip(lens, q))  # (query token, key) pairs that the mask leaves
        return {"bytes": 2 * hk * hd * sum(lens) + pages * (4 + 8 * hk) + 2 * 2 * hq * hd * case["batch"] * case["queries"],
                "flops": 4 * seen * hq * hd}
    if case["op"] == "append":
        starts, counts = _starts(case)
        rows = sum(counts) * case["kv_heads"] * case["head_dim"]
        pages = sum(_pages_of(s + n, case["block"]) - s // case["block"] for s, n in zip(starts, counts) if n)
        return {"bytes": 2 * rows * (2 + 1) + pages * (4 + 2 * 4 * case["kv_heads"]), "flops": 4 * rows}
    if case["op"] == "pages":
        page = case["kv_heads"] * (case["block"] * case["head_dim"] + 4)
        return {"bytes": 2 * 2 * case["layers"] * case["pairs"] * page + 8 * case["pairs"], "flops": 0}
    r, v = case["rows"], case["vocab"]
    size = 4 if case["dtype"] == "float32" else 2
    passes = 4 if case["grad"] else 2
    return {"bytes": passes * size * r * v + 8 * r * case["history"] + (r * v // 8 if case["mask"] else 0) + (4 * v if case["bias"] else 0),
            "flops": 3 * r * v}


# ---------------------------------------------------------------------------------------------------- inputs
def _scale_of(amax):
    """The smallest power of two 2^e, e >= E_MIN, with amax <= 448 * 2^e."""
    m, x = torch.frexp(amax)
    e = torch.where(m > 0.875, x - 8, x - 9)
    e = torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(min=E_MIN)
    return torch.ldexp(torch.ones_like(amax), e)


def _pool(case, pages, table, fill, gen):
    """A pool [pages, kv_heads, block, head_dim] with ``fill[b]`` rows of each sequence's pages written, and its scales."""
    hk, bs, hd = case["kv_heads"], case["block"], case["head_dim"]
    x = torch.randn(pages, hk, bs, hd, device="cuda", generator=gen)
    x *= torch.exp2(torch.randint(-1, 2, (pages, hk, 1, 1), device="cuda", generator=gen).float())
    at = torch.arange(table.shape[1] * bs, device="cuda").view(1, -1, bs)
    live = torch.zeros(pages, bs, dtype=torch.bool, device="cuda")
    has = at[:, :, 0] < fill[:, None]
    live[table.long()[has]] = (at < fill[:, None, None])[has]
    x *= live[:, None, :, None]
    scale = _scale_of(x.abs().amax((2, 3)))
    return (x / scale[..., None, None]).to(FP8), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] in ("attend", "append"):
        n, hk, hd, bs = case["batch"], case["kv_heads"], case["head_dim"], case["block"]
        if case["op"] == "attend":
            lens, q_lens = _lengths(case)
            fill, need = lens, [max(1, x) for x in lens]
        else:
            starts, counts = _starts(case)
            fill, need = starts, [max(1, s + c) for s, c in zip(starts, counts)]
        width = _pages_of(max(need), bs)
        own_pages = torch.tensor([_pages_of(x, bs) for x in need], device="cuda")
        used = int(own_pages.sum())
        pages = used + 3
        order = torch.randperm(pages, device="cuda", generator=g)[:used].to(torch.int32)
        has = torch.arange(width, device="cuda")[None] < own_pages[:, None]
        table = torch.zeros(n, width, dtype=torch.int32, device="cuda")
        table[has] = order
        fill_t = torch.tensor(fill, dtype=torch.int32, device="cuda")
        k_pool, k_scale = _pool(case, pages, table, fill_t, g)
        v_pool, v_scale = _pool(case, pages, table, fill_t, g)
        st = {"case": case, "k_pool": k_pool, "v_pool": v_pool, "k_scale": k_scale, "v_scale": v_scale, "table": table}
        if case["op"] == "attend":
            q = torch.randn(n, hk * case["group"], case["queries"], hd, device="cuda", generator=g).bfloat16()
            return {**st, "q": q, "lens": fill_t, "q_lens": torch.tensor(q_lens, dtype=torch.int32, device="cuda")}
        # keys as the rotary kernel writes them; values a strided view of the fused key / value projection's output
        k = torch.randn(n, hk, case["tokens"], hd, device="cuda", generator=g).bfloat16()
        v = torch.randn(n, case["tokens"], 2 * hk * hd, device="cuda", generator=g).bfloat16()
        v = v[..., hk * hd:].view(n, case["tokens"], hk, hd).transpose(1, 2)
        return {**st, "k": k, "v": v, "start": fill_t, "counts": torch.tensor(counts, dtype=torch.int32, device="cuda")}
    if case["op"] == "pages":
        shape = (case["layers"], case["blocks"], case["kv_heads"])
        body = shape + (case["block"], case["head_dim"])
        code = [(torch.randint(0, 127, body, device="cuda", generator=g, dtype=torch.uint8)
                 + 128 * torch.randint(0, 2, body, device="cuda", generator=g, dtype=torch.uint8)).view(FP8) for _ in range(2)]
        scale = [torch.exp2(torch.randint(-12, 3, shape, device="cuda", generator=g).float()) for _ in range(2)]
        at = torch.randperm(case["blocks"], device="cuda", generator=g).to(torch.int32)
        return {"case": case, "pools": code + scale, "src": at[:case["pairs"]].contiguous(),
                "dst": at[case["pairs"]:2 * case["pairs"]].contiguous()}
    r, v, h = case["rows"], case["vocab"], case["history"]
    dt = getattr(torch, case["dtype"])
    x = (torch.randn(r, v, device="cuda", generator=g) * 3).to(dt)
    # frequent tokens come often
    hist = (torch.rand(r, h, device="cuda", generator=g).pow(4) * v).long().clamp(max=v - 1)
    lens = torch.randint((h + 1) // 2, h + 1, (r,), device="cuda", generator=g, dtype=torch.int32)
    st = {"case": case, "x": x.requires_grad_(case["grad"]), "history": hist, "lens": lens, "prompt_lens": lens // 3,
          "repetition": 1 + 0.3 * torch.rand(r, device="cuda", generator=g), "presence": torch.rand(r, device="cuda", generator=g),
          "frequency": 0.5 * torch.rand(r, device="cuda", generator=g), "bias": None, "allowed": None, "g": None}
    if case["bias"]:
        st["bias"] = torch.randn(v, device="cuda", generator=g)
    if case["mask"]:
        st["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (r, _pages_of(v, 32)), device="cuda", generator=g).to(torch.int32)
    if case["grad"]:
        st["g"] = (torch.randn(r, v, device="cuda", generator=g) / v).to(dt)
    return st


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_attend(s):
    q, table, lens, q_lens = s["q"], s["table"].long(), s["lens"], s["q_lens"]
    b, hq, sq, hd = q.shape
    hk, bs = s["k_pool"].shape[1:3]
    n = table.shape[1] * bs
    k = s["k_pool"].view(torch.uint8)[table].view(FP8).float() * s["k_scale"][table][..., None, None]
    v = s["v_pool"].view(torch.uint8)[table].view(FP8).float() * s["v_scale"][table][..., None, None]
    k, v = (x.permute(0, 2, 1, 3, 4).reshape(b, hk, n, hd) for x in (k, v))
    at = torch.arange(n, device=q.device)
    # query token i of sequence b stands at position lens[b] - q_lens[b] + i and sees the rows up to its own
    row = torch.arange(sq, device=q.device)
    last = torch.where(row < q_lens[:, None], (lens - q_lens)[:, None] + row, -1)
    see = (at <= last[:, :, None])[:, None, None]  # [b, 1, 1, sq, n]
    z = torch.matmul(q.float().reshape(b, hk, -1, hd), k.transpose(-1, -2)).view(b, hk, -1, sq, n) / math.sqrt(hd)
    z = torch.where(see, z, -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.matmul(p.view(b, hk, -1, n), v).view(b, hq, sq, hd)
    return o.transpose(1, 2).contiguous().to(q.dtype)


def _plain_append_one(pool, scale, x, table, start, counts):
    b, hk, s, hd = x.shape
    bs = pool.shape[2]
    touched_most = (s + bs - 2) // bs + 1
    page = (start // bs)[:, None] + torch.arange(touched_most, device=x.device)  # [b, t]
    at = page[..., None] * bs + torch.arange(bs, device=x.device)  # [b, t, bs]
    first, end = start[:, None, None], (start + counts)[:, None, None]
    new = (at >= first) & (at < end)
    hit = new.any(-1)
    ids = table.long().gather(1, page.clamp(max=table.shape[1] - 1).long())
    rows = (at - first).clamp(0, s - 1).view(b, 1, -1, 1).expand(b, hk, -1, hd)
    y = x.float().gather(2, rows.long()).view(b, hk, -1, bs, hd).transpose(1, 2) * new[:, :, None, :, None]  # [b, t, hk, bs, hd]
    was = torch.where(((at[..., 0] < start[:, None]))[..., None], scale[ids], 0.0)
    now = torch.maximum(was, _scale_of(y.abs().amax((3, 4))))
    had = pool.view(torch.uint8)[ids].view(FP8).float()
    kept = torch.where((at < first)[:, :, None, :, None], had * (was / now)[..., None, None], had)
    y = torch.where(new[:, :, None, :, None], y / now[..., None, None], kept).to(FP8)
    pool.view(torch.uint8)[ids[hit]] = y.view(torch.uint8)[hit]
    scale[ids[hit]] = now[hit]


def _plain_logits(s):
    x = s["x"].detach().float()
    r, v = x.shape
    h = s["history"]
    at = torch.arange(h.shape[1], device=x.device)
    seen = torch.zeros(r, v, device=x.device).scatter_add_(1, h, (at < s["lens"][:, None]).float()) > 0
    said = torch.zeros(r, v, device=x.device).scatter_add_(1, h, ((at < s["lens"][:, None]) & (at >= s["prompt_lens"][:, None])).float())
    rep = s["repetition"][:, None]
    y = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    y = y - (s["frequency"][:, None] * said + s["presence"][:, None] * (said > 0))
    if s["bias"] is not None:
        y = y + s["bias"]
    ok = None
    if s["allowed"] is not None:
        at = torch.arange(v, device=x.device)
        ok = (s["allowed"][:, at // 32] >> (at % 32)) & 1 == 1
        y = torch.where(ok, y, -math.inf)
    y = y.to(s["x"].dtype)
    if s["g"] is None:
        return y
    dx = s["g"].float() * torch.where(seen, torch.where(x > 0, 1 / rep, rep), 1.0)
    if ok is not None:
        dx = torch.where(ok, dx, 0.0)
    return y, dx.to(s["x"].dtype)


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from verl_omni_b200.ops.logits import process_logits
        from verl_omni_b200.ops.paged8 import append_paged8, attend_paged8, copy_pages
    if op == "attend":
        if not own:
            return _plain_attend(s)
        return attend_paged8(s["q"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"], s["table"], s["lens"], q_lens=s["q_lens"])
    if op == "append":
        if not own:
            _plain_append_one(s["k_pool"], s["k_scale"], s["k"], s["table"], s["start"], s["counts"])
            _plain_append_one(s["v_pool"], s["v_scale"], s["v"], s["table"], s["start"], s["counts"])
        else:
            append_paged8(s["k"], s["v"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"], s["table"], s["start"], counts=s["counts"])
        # the pages hold e4m3 numbers: they and their scales are the state
        return s["k_pool"], s["k_scale"], s["v_pool"], s["v_scale"]
    if op == "pages":
        if own:
            copy_pages(s["pools"], s["src"], s["dst"])
            return s["pools"]
        src, dst = s["src"].long(), s["dst"].long()
        k, v = (p.view(torch.uint8) for p in s["pools"][:2])
        k[:, dst] = k[:, src]
        v[:, dst] = v[:, src]
        s["pools"][2][:, dst] = s["pools"][2][:, src]
        s["pools"][3][:, dst] = s["pools"][3][:, src]
        return s["pools"]
    if not own:
        return _plain_logits(s)
    y = process_logits(s["x"], history=s["history"], lens=s["lens"], prompt_lens=s["prompt_lens"], repetition=s["repetition"],
                       presence=s["presence"], frequency=s["frequency"], bias=s["bias"], allowed=s["allowed"])
    return y if s["g"] is None else (y.detach(), torch.autograd.grad(y, s["x"], s["g"])[0])


# ---------------------------------------------------------------------------------------------------- 64 bits
def _e4m3_values(code):
    """The number that each e4m3 code stands for, from the format: sign, 4 exponent bits (bias 7), 3 fraction bits."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v) * np.where(c >= 128, -1, 1)
    return torch.tensor(v, device=code.device)[code.view(torch.uint8).long()]


def _e4m3_round(x):
    """x (64 bits, at most 448 in magnitude) to the nearest e4m3 number, ties to an even fraction."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _exact_attend(s):
    q = s["q"].double()
    out = torch.zeros(q.shape[0], q.shape[2], q.shape[1], q.shape[3], dtype=torch.float64, device=q.device)
    group, bs = s["case"]["group"], s["case"]["block"]
    for b, (n, m) in enumerate(zip(*_lengths(s["case"]))):
        if not m:
            continue
        ids = s["table"][b, :_pages_of(n, bs)].long()
        for h in range(s["case"]["kv_heads"]):
            k, v = ((_e4m3_values(s[p][ids, h]) * s[c][ids, h].double()[:, None, None]).flatten(0, 1)[:n] for p, c in (("k_pool", "k_scale"), ("v_pool", "v_scale")))
            for i in range(0, m, 128):
                j = min(m, i + 128)
                end = n - m + j
                z = torch.einsum("gsd,td->gst", q[b, h * group:(h + 1) * group, i:j], k[:end]) * q.shape[3] ** -0.5
                late = torch.arange(end, device=q.device)[None] > torch.arange(n - m + i, end, device=q.device)[:, None]
                z.masked_fill_(late, -math.inf)
                out[b, i:j, h * group:(h + 1) * group] = torch.einsum("gst,td->sgd", torch.softmax(z, -1), v[:end])
    return out


def _exact_append(s):
    """Row by row over the sequences, from the operator's definition: the page's scale is the larger of what its earlier
    rows had and what the new rows need."""
    bs, res = s["case"]["block"], []
    for p, c, x in (("k_pool", "k_scale", s["k"]), ("v_pool", "v_scale", s["v"])):
        pool, scale = _e4m3_values(s[p]), s[c].double()
        for b, (start, n) in enumerate(zip(*_starts(s["case"]))):
            done = 0
            while done < n:
                page, r0 = (start + done) // bs, (start + done) % bs
                m = min(bs - r0, n - done)
                i = int(s["table"][b, page])
                rows = x[b, :, done:done + m].double()
                amax = rows.abs().amax((1, 2))
                need = torch.exp2(torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448)).clamp(min=E_MIN))
                new = torch.maximum(scale[i], need) if r0 else need
                pool[i, :, :r0] = _e4m3_round(pool[i, :, :r0] * (scale[i] / new)[:, None, None])
                pool[i, :, r0:r0 + m] = _e4m3_round(rows / new[:, None, None])
                scale[i] = new
                done += m
        res += [pool, scale]
    return tuple(res)


def _exact_logits(s):
    x, v = s["x"].detach().double(), s["case"]["vocab"]
    y, dx = torch.empty_like(x), torch.empty_like(x) if s["g"] is not None else None
    for r, (n, m) in enumerate(zip(s["lens"].tolist(), s["prompt_lens"].tolist())):
        seen = torch.bincount(s["history"][r, :n], minlength=v) > 0
        said = torch.bincount(s["history"][r, m:n], minlength=v)
        rep = s["repetition"][r].double()
        factor = torch.ones(v, dtype=torch.float64, device=x.device)
        factor[seen & (x[r] > 0)] = 1 / rep
        factor[seen & (x[r] <= 0)] = rep
        y[r] = x[r] * factor - s["frequency"][r].double() * said - s["presence"][r].double() * said.clamp(max=1)
        if s["bias"] is not None:
            y[r] += s["bias"].double()
        if s["allowed"] is not None:
            bits = (s["allowed"][r].long()[:, None] >> torch.arange(32, device=x.device)) & 1
            banned = bits.flatten()[:v] == 0
            y[r, banned], factor[banned] = -math.inf, 0
        if dx is not None:
            dx[r] = s["g"][r].double() * factor
    return y if dx is None else (y, dx)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "pages":
        pools = [_e4m3_values(p) if p.dtype == FP8 else p.double() for p in s["pools"]]
        for i, j in zip(s["src"].tolist(), s["dst"].tolist()):
            for p in pools:
                p[:, j] = p[:, i]
        return pools
    return _exact_logits(s)
