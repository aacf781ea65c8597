"""Paged KV cache held in 8 bits: quantising append, attention over it, page copies, and the block manager.

Keys and values are e4m3 numbers with one power-of-two scale per (page, KV head): the smallest ``2^e``
(``e >= -100``) with ``amax <= 448 * 2^e``.  A cached value is ``code * scale``; half the bytes of a bf16 cache.

* :func:`append_paged8` -- new bf16 rows into the pages of their sequences.  A page that already holds rows keeps the
  larger of its scale and the new rows' (its codes are brought to it: an exponent shift); ``+-inf`` is stored as the
  largest number of the page, NaN as NaN, and neither counts for the scale;
* :func:`attend_paged8` -- one or more query tokens per sequence, causal among the new tokens, grouped heads;
* :func:`copy_pages` -- pages of every layer copied inside their pools in one launch (forks, compaction);
* :class:`PagedKVCache8` / :class:`PagedBatch8` / :class:`Paged8View` -- pools of all layers, a host block manager with
  shared (reference-counted) pages, and what one model layer receives as its cache.

CUDA tensors run ``csrc/paged8.cu`` (and the tcgen05 kernels next to it); CPU tensors an fp32 torch oracle.
Counterpart of vLLM's fp8 ``kv_cache_dtype`` and block manager under the reference's AR rollout
(``verl_omni/workers/rollout/vllm_rollout/vllm_omni_async_server.py:537-579``).
"""

from __future__ import annotations

import math
from typing import Optional, Sequence, Union

import torch
from torch.autograd.forward_ad import unpack_dual

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
MIN_EXP = -100


def _ext():
    from verl_omni_b200.ops._ext import ext

    return ext()


# ---------------------------------------------------------------------------------------------- oracles
def page_scale(amax: torch.Tensor) -> torch.Tensor:
    """Smallest power of two ``2^e >= amax / 448`` with ``e >= MIN_EXP`` (fp32)."""
    m, x = torch.frexp(amax.float())
    e = torch.where(m > 0.875, x - 8, x - 9)  # 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXP)).clamp(min=MIN_EXP)
    return torch.ldexp(torch.ones_like(amax, dtype=torch.float32), e)


def _to_e4m3(x: torch.Tensor) -> torch.Tensor:
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)  # clamp keeps NaN


def _check(kp, vp, ks, vs, table, B: int) -> None:
    """The oracle's checks (CUDA tensors are checked by the extension)."""
    if kp.dim() != 4 or kp.dtype != E4M3 or vp.shape != kp.shape or vp.dtype != E4M3:
        raise ValueError("pools: float8_e4m3fn [pages, kv_heads, block, head_dim]")
    if any(s.shape != kp.shape[:2] or s.dtype != torch.float32 for s in (ks, vs)):
        raise ValueError("scales: float32 [pages, kv_heads]")
    if table.dim() != 2 or table.shape[0] != B or table.dtype != torch.int32:
        raise ValueError("block_table: int32 [batch, max_pages]")


def append_paged8_reference(k, v, k_pool, v_pool, k_scale, v_scale, block_table, start, counts=None, offset: int = 0) -> None:
    B, Hk, S, hd = k.shape
    _check(k_pool, v_pool, k_scale, v_scale, block_table, B)
    if v.shape != k.shape or k_pool.shape[1] != Hk or k_pool.shape[3] != hd or start.shape != (B,):
        raise ValueError("k, v: [batch, kv_heads, tokens, head_dim] of the pools; start [batch]")
    bs = k_pool.shape[2]
    for b in range(B):
        p0 = int(start[b]) + offset
        n = S if counts is None else max(0, min(int(counts[b]), S))
        done = 0
        while p0 >= 0 and done < n and (p0 + done) // bs < block_table.shape[1]:
            page, r0 = divmod(p0 + done, bs)
            m = min(bs - r0, n - done)
            i = int(block_table[b, page])
            if 0 <= i < k_pool.shape[0]:
                for pool, scale, x in ((k_pool, k_scale, k), (v_pool, v_scale, v)):
                    rows = x[b, :, done:done + m].float()  # [Hk, m, hd]
                    now = page_scale(torch.where(rows.isfinite(), rows.abs(), 0.0).amax((1, 2)))
                    if r0:
                        now = torch.maximum(scale[i], now)
                        pool[i, :, :r0] = _to_e4m3(pool[i, :, :r0].float() * (scale[i] / now)[:, None, None])
                    pool[i, :, r0:r0 + m] = _to_e4m3(rows / now[:, None, None])
                    scale[i] = now
            done += m


def gather_paged8(pool: torch.Tensor, scale: torch.Tensor, table: torch.Tensor, n: int) -> torch.Tensor:
    """fp32 ``[B, Hk, n, hd]`` copy of the first ``n`` rows of every sequence; rows of pages outside the pool are zero."""
    bs = pool.shape[2]
    W = -(-n // bs)
    t = table[:, :W].long()
    inside = (t >= 0) & (t < pool.shape[0])
    t = torch.where(inside, t, 0)
    x = pool.view(torch.uint8)[t].view(E4M3).float() * scale[t][..., None, None]
    x = torch.where(inside[:, :, None, None, None], x, 0.0)
    return x.permute(0, 2, 1, 3, 4).reshape(t.shape[0], pool.shape[1], W * bs, -1)[:, :, :n]


def attend_paged8_reference(q, k_pool, v_pool, k_scale, v_scale, block_table, lens, q_lens=None,
                            scale: Optional[float] = None, len_add: int = 0) -> torch.Tensor:
    B, Hq, S, hd = q.shape
    _check(k_pool, v_pool, k_scale, v_scale, block_table, B)
    Hk, bs = k_pool.shape[1:3]
    if Hq % Hk or k_pool.shape[3] != hd or lens.shape != (B,):
        raise ValueError("q: head_dim of the pools, q_heads a multiple of kv_heads; lens [batch]")
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    out = torch.zeros(B, S, Hq, hd, dtype=torch.float32, device=q.device)
    for b in range(B):
        n = max(0, min(int(lens[b]) + len_add, block_table.shape[1] * bs))
        m = S if q_lens is None else max(0, min(int(q_lens[b]), S))
        if not n or not m:
            continue
        k, v = (gather_paged8(p, s, block_table[b:b + 1], n)[0].repeat_interleave(Hq // Hk, 0)
                for p, s in ((k_pool, k_scale), (v_pool, v_scale)))
        for i in range(m):
            lim = n - m + i + 1
            if lim > 0:
                z = torch.einsum("hd,htd->ht", q[b, :, i].float(), k[:, :lim]) * scale
                out[b, i] = torch.einsum("ht,htd->hd", torch.softmax(z, -1), v[:, :lim])
    return out.to(q.dtype)


# ---------------------------------------------------------------------------------------------- operators
def append_paged8(k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, block_table: torch.Tensor, start: torch.Tensor,
                  counts: Optional[torch.Tensor] = None, offset: int = 0) -> None:
    """Writes k / v ``[B, Hk, S, hd]`` (any strides) at positions ``start[b] + offset + i`` (``i < counts[b]``, all
    ``S`` without ``counts``) of each sequence, in place.

    Pools ``[pages, Hk, block, hd]`` e4m3, scales ``[pages, Hk]`` fp32, ``block_table [B, max_pages]``, ``start`` and
    ``counts [B]`` int32.  Rows past the table and pages outside the pool are dropped.  A page belongs to one sequence
    of the call: two rows of ``block_table`` that write to the same page give an undefined page.  On the GPU k and v
    are bf16."""
    if not k.is_cuda:
        return append_paged8_reference(k, v, k_pool, v_pool, k_scale, v_scale, block_table, start, counts, offset)
    _ext().paged8_append(k, v, k_pool, v_pool, k_scale, v_scale, block_table, start, counts, offset)


def attend_paged8(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                  q_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None, len_add: int = 0) -> torch.Tensor:
    """q ``[B, Hq, S, hd]`` (any strides) against the cached rows -> ``[B, S, Hq, hd]``.

    Pools ``[pages, Hk, block, hd]`` e4m3, positive scales ``[pages, Hk]`` fp32 (powers of two as :func:`append_paged8`
    writes them; with others more than 16 query rows take codes times scale in 11 bits), ``block_table [B, max_pages]``,
    ``lens [B]`` int32.  ``lens[b] + len_add`` rows of sequence b are cached, the new tokens' among them; query token ``i`` of its
    ``q_lens[b]`` (all ``S`` without) stands at position ``lens[b] + len_add - q_lens[b] + i`` and sees the rows up to
    its own.  Rows past ``q_lens`` and rows that see no key are zero; pages outside the pool read as zeros.
    Repeated calls agree bit for bit; a sequence's rounding may change with the lengths of the others, which decide
    where its keys are cut into parts.  Weights keep 8 bits down to 2^-9 of the largest among the 128 keys of a tile (up
    to 16 query rows: tokens times heads of a group) or 2^-24 of the row's largest so far (more), below in steps of
    2^-18 and 2^-31 of it; a value page's scale below the largest beside it counts as a smaller weight there.
    Inference only (no gradient).  Waits inside the kernels are bounded: :func:`raise_on_timeout` tells whether one ran out."""
    if q.requires_grad and torch.is_grad_enabled():
        raise ValueError("attention over the 8-bit cache has no backward: call it under torch.no_grad()")
    if unpack_dual(q).tangent is not None:
        raise ValueError("attention over the 8-bit cache has no forward-mode derivative")
    if not q.is_cuda:
        return attend_paged8_reference(q, k_pool, v_pool, k_scale, v_scale, block_table, lens, q_lens, scale, len_add)
    return _ext().paged8_attend(q, k_pool, v_pool, k_scale, v_scale, block_table, lens, q_lens,
                                1.0 / math.sqrt(q.shape[-1]) if scale is None else scale, len_add)


def raise_on_timeout(device) -> None:
    """Raises a RuntimeError if a bounded wait of the attention kernels ran out on ``device`` since the last call: what they
    wrote is then not an attention output.  Waits for the current stream; for the end of a rollout or a step, where results
    are read anyway."""
    device = torch.device(device)
    if device.type != "cuda":
        return
    with torch.cuda.device(device):
        torch.cuda.current_stream().synchronize()
        code = _ext().paged8_error(True)
    if code:
        raise RuntimeError(f"8-bit attention: a wait inside the kernel ran out (code {code}), its outputs are invalid")


def copy_pages(pools: Sequence[torch.Tensor], src: Union[torch.Tensor, Sequence[int]],
               dst: Union[torch.Tensor, Sequence[int]]) -> None:
    """Page ``dst[i]`` of every layer of every pool ``[layers, pages, ...]`` becomes a copy of page ``src[i]``.

    ``src`` / ``dst``: int32 tensors on the pools' device, or host lists (checked: inside the pool, no page written
    twice, none both read and written; tensors must hold the same, pages outside the pool are skipped)."""
    if not isinstance(src, torch.Tensor):
        src, dst = [int(i) for i in src], [int(i) for i in dst]
        n = pools[0].shape[1]
        if len(src) != len(dst) or any(not 0 <= i < n for i in src + dst):
            raise ValueError(f"copy_pages: as many sources as destinations, pages in [0, {n})")
        if len(set(dst)) != len(dst) or set(dst) & set(src):
            raise ValueError("copy_pages: a page is written twice, or both read and written")
        if not src:
            return
        both = torch.tensor([src, dst], dtype=torch.int32).to(pools[0].device)
        src, dst = both[0], both[1]
    if not pools[0].is_cuda:
        s, d = src.long(), dst.long()
        ok = (s >= 0) & (s < pools[0].shape[1]) & (d >= 0) & (d < pools[0].shape[1])
        for p in pools:
            b = p.view(torch.uint8) if p.dtype == E4M3 else p
            b[:, d[ok]] = b[:, s[ok]]
        return
    _ext().copy_pages(list(pools), src, dst)


# ---------------------------------------------------------------------------------------------- block manager
class PagedKVCache8:
    """Pools of all layers ``[layers, pages, Hk, block, hd]`` (K and V, e4m3) with their scales
    ``[layers, pages, Hk]``, and the host block manager: a free list, per-sequence page lists and a reference count per
    page.  Sequences forked from one another share their full pages; a page that may still be written has one owner.

    Attention at head_dim 64 / 128 over pages of 8 to 128 rows that divide 128, or multiples of 128, runs on the tensor cores;
    other sizes run a much slower kernel."""

    def __init__(self, layers: int, num_blocks: int, kv_heads: int, block_size: int, head_dim: int, device):
        if min(layers, num_blocks, kv_heads, block_size) < 1:
            raise ValueError("layers, num_blocks, kv_heads and block_size are at least 1")
        if head_dim < 16 or head_dim > 256 or head_dim % 16:
            raise ValueError(f"head_dim: a multiple of 16 up to 256, got {head_dim}")
        shape = (layers, num_blocks, kv_heads)
        self.k = torch.zeros(shape + (block_size, head_dim), dtype=torch.uint8, device=device).view(E4M3)
        self.v = torch.zeros(shape + (block_size, head_dim), dtype=torch.uint8, device=device).view(E4M3)
        self.k_scale = torch.full(shape, 2.0 ** MIN_EXP, device=device)
        self.v_scale = torch.full(shape, 2.0 ** MIN_EXP, device=device)
        self.block = block_size
        self.free: list[int] = list(range(num_blocks - 1, -1, -1))
        self.refs = [0] * num_blocks
        self.blocks: dict[int, list[int]] = {}
        self.length: dict[int, int] = {}
        self.version = 0  # moves when a sequence's pages change: batches then refresh their tables
        self._next = 0

    @property
    def pools(self) -> list[torch.Tensor]:
        return [self.k, self.v, self.k_scale, self.v_scale]

    def _take(self) -> int:
        i = self.free.pop()
        self.refs[i] = 1
        return i

    def add_sequence(self) -> int:
        sid, self._next = self._next, self._next + 1
        self.blocks[sid], self.length[sid] = [], 0
        return sid

    def free_sequence(self, sid: int) -> None:
        """Drops the sequence; a page returns to the free list with its last owner."""
        for i in reversed(self.blocks.pop(sid)):
            self.refs[i] -= 1
            if not self.refs[i]:
                self.free.append(i)
        del self.length[sid]
        self.version += 1

    def reserve(self, sids: Sequence[int], n: int) -> None:
        """Pages for ``n`` more rows of every listed sequence (all of them, or a RuntimeError and no change)."""
        need = [max(0, -(-(self.length[s] + n) // self.block) - len(self.blocks[s])) for s in sids]
        if sum(need) > len(self.free):
            raise RuntimeError(f"8-bit KV cache out of pages ({sum(need)} needed, {len(self.free)} free)")
        for s, m in zip(sids, need):
            self.blocks[s].extend(self._take() for _ in range(m))
        self.version += any(need)

    def fork(self, sids: Sequence[int], n: int) -> list[list[int]]:
        """``n`` children of every listed sequence, with its rows: full pages are shared, a partly filled last page is
        copied (one launch for all sequences and layers); pages reserved ahead of the rows stay with the parent."""
        part = [s for s in sids if self.length[s] % self.block]
        if n * len(part) > len(self.free):
            raise RuntimeError(f"8-bit KV cache out of pages ({n * len(part)} needed, {len(self.free)} free)")
        src, dst, out = [], [], []
        for s in sids:
            full, rest = divmod(self.length[s], self.block)
            kids = []
            for _ in range(n):
                c = self.add_sequence()
                pages = self.blocks[s][:full]
                for i in pages:
                    self.refs[i] += 1
                if rest:
                    pages = pages + [self._take()]
                    src.append(self.blocks[s][full])
                    dst.append(pages[-1])
                self.blocks[c], self.length[c] = pages, self.length[s]
                kids.append(c)
            out.append(kids)
        self.version += 1
        copy_pages(self.pools, src, dst)
        return out

    def compact(self) -> int:
        """Moves the pages in use to the low end of the pools (one launch) and returns their number: pages from there
        on are free, so the pools' head can be saved or handed on."""
        used = [i for i, r in enumerate(self.refs) if r]
        n = len(used)
        src = [i for i in used if i >= n]
        dst = [i for i in range(n) if not self.refs[i]]
        to = dict(zip(src, dst))
        if src:
            copy_pages(self.pools, src, dst)
            for s, d in to.items():
                self.refs[d], self.refs[s] = self.refs[s], 0
            self.blocks = {s: [to.get(i, i) for i in b] for s, b in self.blocks.items()}
            self.free = list(range(len(self.refs) - 1, n - 1, -1))
            self.version += 1
        return n

    def batch(self, sids: Sequence[int], max_len: int = 0) -> "PagedBatch8":
        return PagedBatch8(self, list(sids), max_len)


class PagedBatch8:
    """The sequences of one batch: their block table and row counts on the device, shared by the layers' views.

    ``max_len``: rows that the table covers (at least what is reserved); it grows when more are needed, until a step has been
    captured in a CUDA graph, which reads the table at its address: from then on more is a RuntimeError.  While a batch is in
    use, only it appends to its sequences."""

    def __init__(self, cache: PagedKVCache8, sids: list[int], max_len: int = 0):
        if len(set(sids)) != len(sids):
            raise ValueError("a sequence appears twice in the batch")
        self.cache, self.sids = cache, sids
        self.base = [cache.length[s] for s in sids]
        dev = cache.k.device
        width = max([1, -(-max_len // cache.block)] + [len(cache.blocks[s]) for s in sids])
        self.table = torch.zeros(len(sids), width, dtype=torch.int32, device=dev)
        self.lens = torch.tensor(self.base, dtype=torch.int32, device=dev)  # rows when the batch was made
        self.pos = self.lens.clone()  # position of the next row in steps that read it on the device
        self.off = 0  # rows appended since
        self.captured = False  # a CUDA graph holds the table's address
        self._seen = -1
        self._refresh()

    def _refresh(self) -> None:
        if self._seen == self.cache.version:
            return
        blocks = [self.cache.blocks[s] for s in self.sids]
        if max(len(b) for b in blocks) > self.table.shape[1]:
            self._fits(max(len(b) for b in blocks))
            self.table = torch.zeros(len(blocks), max(len(b) for b in blocks), dtype=torch.int32, device=self.table.device)
        t = torch.zeros(self.table.shape, dtype=torch.int32)
        for i, b in enumerate(blocks):
            t[i, :len(b)] = torch.tensor(b, dtype=torch.int32)
        self.table.copy_(t)
        self._seen = self.cache.version

    def _fits(self, pages: int) -> None:
        if self.captured and pages > self.table.shape[1]:
            raise RuntimeError(f"the block table holds {self.table.shape[1]} pages a sequence and a captured step reads it: "
                               f"make the batch with max_len for {pages}")

    def _reserve(self, n: int) -> None:
        c = self.cache
        self._fits(max(max(len(c.blocks[s]), -(-(c.length[s] + n) // c.block)) for s in self.sids))  # before anything changes
        c.reserve(self.sids, n)

    def grow(self, off: int) -> None:
        """The batch's sequences hold ``off`` rows more than when it was made (pages are reserved as needed)."""
        if off > self.off:
            self._reserve(off - self.off)
            for s in self.sids:
                self.cache.length[s] += off - self.off
            self.off = off
        self._refresh()

    def reserve(self, n: int) -> None:
        """Pages for ``n`` rows more than now, so that later steps change no table."""
        self._reserve(n)
        self._refresh()

    def at(self, off: int) -> None:
        """Points ``pos`` at row ``base + off`` and counts it as held: before a device-position step."""
        self.grow(off + 1)
        torch.add(self.lens, off, out=self.pos)

    def views(self) -> list["Paged8View"]:
        return [Paged8View(self, i) for i in range(self.cache.k.shape[0])]


class Paged8View:
    """One layer of a :class:`PagedBatch8` (what a model layer receives as its cache)."""

    def __init__(self, batch: PagedBatch8, layer: int):
        c = batch.cache
        self.batch, self.layer = batch, layer
        self.off = batch.off
        self._pools = (c.k[layer], c.v[layer], c.k_scale[layer], c.v_scale[layer])

    @property
    def len(self) -> int:
        return max(self.batch.base) + self.off

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """k / v ``[B, Hk, S, hd]``: the next S rows of every sequence."""
        S = k.shape[2]
        self.batch.grow(self.off + S)
        append_paged8(k, v, *self._pools, self.batch.table, self.batch.lens, None, self.off)
        self.off += S

    def attend(self, q: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
        """q ``[B, Hq, S, hd]`` of the S rows appended last -> ``[B, S, Hq, hd]``."""
        return attend_paged8(q, *self._pools, self.batch.table, self.batch.lens, None, scale, self.off)

    def append_at(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """One row per sequence at the batch's device position (nothing is read on the host: the step can be captured in
        a CUDA graph; :meth:`PagedBatch8.at` moves the position between replays)."""
        self._note_capture()
        append_paged8(k, v, *self._pools, self.batch.table, self.batch.pos)

    def attend_at(self, q: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
        self._note_capture()
        return attend_paged8(q, *self._pools, self.batch.table, self.batch.pos, None, scale, 1)

    def _note_capture(self) -> None:
        if self.batch.table.is_cuda and torch.cuda.is_current_stream_capturing():
            self.batch.captured = True
